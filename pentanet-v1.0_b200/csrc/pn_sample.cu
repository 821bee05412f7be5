// pn_sample.cu -- one token per row of logits from given uniform numbers, after
// temperature, top-k, min-p and top-p.
//
// With w_i = exp((x_i - max) / T): keep the k largest logits (ties: the lowest
// index first), of them those with w_i >= min_p, of them the smallest prefix in
// that order whose sum reaches top_p of the sum of all that are left; the token
// is the first index whose running sum of kept w exceeds u times their total.
//
// Weights are held as 45-bit fixed-point fractions of the largest, computed in
// fp64 (an error of 2^-24 per weight would move the borders of the draw far
// enough to change about one token in 10^3 over a 50 k vocabulary).  Integer
// sums do not depend on their order, so the result is that of the formula and
// the same on every run.  Weights below 2^-46 of the largest count as zero;
// 2^18 weights of 2^45 fit 64 bits, hence the limit on the vocabulary.
//
// Shape.  A cluster of up to eight blocks takes a row, each with a run of it in
// shared memory (read from memory once).  Few rows: as many blocks as there are,
// for latency; many: as few as hold the row, two rows' blocks to an SM.
//
// No sort.  Logits within 2^-12 of the largest weight are the candidates: a few
// hundred in a model's distribution.  They are brought to the first block,
// which finds the k-th largest and the border of top-p by a histogram over 2048
// buckets of (max - x) / T (64 to a unit; beyond 32 units a weight is zero) and
// then among the few logits of one bucket.  Where the candidates do not reach
// the border, or do not fit (flat distributions, large k), every block
// histograms its run instead, and the border's bucket is searched by bisection on
// the logits' ordered bit patterns: on a list of them or, where one bucket holds
// too many (all logits nearly alike), over the runs themselves.
#include <cooperative_groups.h>

#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

namespace cg = cooperative_groups;

struct SampleArgs {
    const void* x;
    int64_t ld;   // elements between rows
    int V;
    int steps;    // 16-byte chunks per thread
    const float* u;
    const float* t;      // per row, or null: t0
    const int32_t* k;
    const float* p;
    const float* m;
    float t0, p0, m0;
    int32_t k0;
    int64_t* out;
};

constexpr int kSmpThreads = 512;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kSmpBuckets = 2048;
constexpr int kSmpList = 4096;
constexpr int kSmpBlocks = 8;  // of a cluster, at most
constexpr int64_t kSmpMaxVocab = 1 << 18;
constexpr double kSmpOne = 35184372088832.0;  // 2^45
constexpr float kSmpCut = 8.3f * 64.0f;       // candidates lie before this bucket: 12 ln 2 units

struct SampleShared {
    double table[64];  // 2^(j / 64 + 45)
    uint32_t lo[kSmpBuckets], hi[kSmpBuckets];  // 64-bit sums in two halves (shared memory adds 32 bits natively)
    float list[kSmpList];
    uint64_t red[kSmpWarps];
    uint32_t redc[kSmpWarps];
    float redf[kSmpWarps];
    // one entry per block of the cluster, written by that block
    uint64_t of_sum[2][kSmpBlocks];
    uint64_t of_cand[kSmpBlocks];
    uint32_t of_n[kSmpBlocks];
    float of_max[kSmpBlocks];
    // the first block's findings
    uint64_t sum, before, total;
    uint32_t bucket, ties;
    float key;
    uint32_t n;  // entries of list
    float few[32];
    uint32_t n_few;
};

__device__ __forceinline__ uint32_t order_bits(float v) {  // monotone in v
    const uint32_t b = __float_as_uint(v);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_order(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the block, the same in every thread.
__device__ __forceinline__ uint64_t block_sum(SampleShared& s, uint64_t v) {
    v = warp_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s.red[threadIdx.x % kSmpWarps];
#pragma unroll
    for (int o = kSmpWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One row's rule.  A logit is kept when it lies above `key`, or equals it and is
// among the first `ties` such in index order, and its weight is not zero.
struct SampleRow {
    const double* table;
    float max;
    double c;       // 64 log2(e) / T
    float per;      // buckets per unit of max - x
    uint64_t floor; // min-p as a weight (at least 1)
    float key;
    uint32_t ties;

    __device__ __forceinline__ float place(float x) const { return (max - x) * per; }  // NaN: a NaN logit, or greedy
    __device__ __forceinline__ int bucket(float x) const {  // monotone; kSmpBuckets: no weight
        return x == max ? 0 : (int)fminf(place(x), (float)kSmpBuckets);
    }
    // round(2^45 exp((x - max) / T)), 0 below the floor; for x in a bucket.  With
    // s = 64 log2(e) (x - max) / T = n + f: 2^(n / 64) from the table, 2^(f / 64) from its
    // series (|f| <= 1/2, so the fifth term is below 2^-44 of the sum).
    __device__ __forceinline__ uint64_t weight(float x) const {
        if (x == max) return (uint64_t)kSmpOne;
        constexpr double kShift = 6755399441055744.0;  // 1.5 * 2^52
        constexpr double a1 = 0.010830424696249145, a2 = a1 * a1 / 2, a3 = a2 * a1 / 3, a4 = a3 * a1 / 4;  // ln 2 / 64
        const double d = ((double)x - (double)max) * c, r = d + kShift, f = d - (r - kShift);
        const int n = __double2loint(r);
        const double p = fma(f, fma(f, fma(f, fma(f, a4, a3), a2), a1), 1.0);
        double t = table[n & 63];
        t = __hiloint2double(__double2hiint(t) + ((n >> 6) << 20), __double2loint(t));
        const uint64_t w = (uint64_t)__double_as_longlong(fma(t, p, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
        return w >= floor ? w : 0;
    }
};

// 16 bytes of logits as fp32.
template <typename T>
struct SmpChunk;
template <>
struct SmpChunk<float> {
    static constexpr int N = 4;
    static constexpr uint32_t kNone = 0xFF800000u;  // -inf
    static __device__ __forceinline__ void get(const uint4& u, float (&v)[N]) {
        v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ float max(const uint4& u) {
        return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    }
    static __device__ __forceinline__ void drop(uint4& u, int i) { (&u.x)[i] = kNone; }
};
template <>
struct SmpChunk<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr uint32_t kNone = 0xFF80FF80u;
    static __device__ __forceinline__ void get(const uint4& u, float (&v)[N]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float max(const uint4& u) {  // a NaN loses, as with fmaxf
        const uint32_t m = max2(max2(u.x, u.y), max2(u.z, u.w));
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
    }
    static __device__ __forceinline__ void drop(uint4& u, int i) {
        uint32_t& w = (&u.x)[i >> 1];
        w = i & 1 ? (w & 0xFFFFu) | 0xFF800000u : (w & 0xFFFF0000u) | 0xFF80u;
    }
};

__device__ __forceinline__ void hist_clear(SampleShared& s) {
    for (int i = threadIdx.x; i < kSmpBuckets; i += kSmpThreads) s.lo[i] = s.hi[i] = 0;
    __syncthreads();
}
__device__ __forceinline__ void hist_add(SampleShared& s, int b, uint64_t w) {
    const uint32_t old = atomicAdd(&s.lo[b], (uint32_t)w);
    const uint32_t h = (uint32_t)(w >> 32) + (old + (uint32_t)w < old ? 1 : 0);
    if (h) atomicAdd(&s.hi[b], h);
}

// The bucket in which the running sum reaches `need` (the first with inclusive sum
// >= need) and the sum before it, in s.bucket and s.before.  All buckets together
// hold at least `need`.
template <typename F>
__device__ __forceinline__ void find_bucket(SampleShared& s, F&& value, uint64_t need) {
    constexpr int per = kSmpBuckets / kSmpThreads;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    uint64_t v[per], sum = 0;
#pragma unroll
    for (int i = 0; i < per; ++i) sum += v[i] = value(tid * per + i);
    uint64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t n = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += n;
    }
    __syncthreads();
    if (lane == 31) s.red[w] = inc;
    __syncthreads();
    uint64_t before = inc - sum;
    for (int i = 0; i < w; ++i) before += s.red[i];
#pragma unroll
    for (int i = 0; i < per; ++i) {
        if (before < need && before + v[i] >= need) {
            s.bucket = tid * per + i;
            s.before = before;
        }
        before += v[i];
    }
    __syncthreads();
}

// Of the listed logits in `bucket`: the smallest key v (not below r.key) for which
// the sum of value(x) over x > v is below `need`; that sum goes to s.sum.
template <typename F>
__device__ __forceinline__ float list_border(SampleShared& s, const SampleRow& r, int n, int bucket, uint64_t need, F&& value) {
    const int tid = threadIdx.x;
    if (tid == 0) s.n_few = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSmpThreads) {
        const float v = s.list[i];
        if (r.bucket(v) == bucket && value(v) != 0) {
            const uint32_t at = atomicAdd(&s.n_few, 1);
            if (at < 32) s.few[at] = v;
        }
    }
    __syncthreads();
    const int few = (int)s.n_few;
    if (few <= 32) {
        // the border is the largest listed key with sum over x >= key of at least need, or r.key
        if (tid < 32) {
            const float mine = tid < few ? s.few[tid] : -INFINITY;
            const uint64_t w = tid < few ? value(mine) : 0;
            uint64_t above = 0, with = 0;
            for (int i = 0; i < few; ++i) {
                const float v = __shfl_sync(0xffffffffu, mine, i);
                const uint64_t q = __shfl_sync(0xffffffffu, w, i);
                if (v > mine) above += q;
                if (v >= mine) with += q;
            }
            const bool is = tid < few && above < need && with >= need;
            const uint32_t b = __ballot_sync(0xffffffffu, is);
            const uint64_t all = warp_sum_u64(w);
            if (b ? tid == __ffs(b) - 1 : tid == 0) {
                s.key = b ? mine : r.key;
                s.sum = b ? above : all;
            }
        }
        __syncthreads();
        return s.key;
    }
    uint32_t lo = order_bits(r.key), hi = order_bits(r.max);  // the answer is in [lo, hi]
    uint64_t above = 0;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        uint64_t sum = 0;
        for (int i = tid; i < n; i += kSmpThreads) {
            const float v = s.list[i];
            if (order_bits(v) > mid && r.bucket(v) == bucket) sum += value(v);
        }
        sum = block_sum(s, sum);
        if (sum < need) {
            hi = mid;
            above = sum;
        } else {
            lo = mid + 1;
        }
    }
    if (tid == 0) s.sum = above;
    __syncthreads();
    return from_order(lo);
}

template <typename T>
__global__ void __launch_bounds__(kSmpThreads, 2) sample_kernel(const SampleArgs a) {
    using K = SmpChunk<T>;
    asm volatile("griddepcontrol.launch_dependents;");
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint4* raw = reinterpret_cast<uint4*>(smem_raw);
    SampleShared& s = *reinterpret_cast<SampleShared*>(smem_raw + (size_t)a.steps * kSmpThreads * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / blocks;
    auto sync = [&]() {
        if (blocks > 1)
            cluster.sync();
        else
            __syncthreads();
    };
    // s.*entry of every block of the cluster, for this block's value (block-uniform)
    auto tell = [&](auto* entry, auto value) {
        if (tid < blocks) *cluster.map_shared_rank(entry, tid) = value;
    };

    // ---- the block's run of the row, in shared memory; chunks start on 16 bytes
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    const int shift = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    const uint4* src = reinterpret_cast<const uint4*>(x - shift);
    const int chunks = (a.V + shift + K::N - 1) / K::N;
    const int chunk0 = (rank * kSmpWarps + warp) * a.steps * 32 + lane;  // index order: block, warp, step, lane
    uint4* mine = raw + warp * a.steps * 32 + lane;
    float mx = -INFINITY;
#pragma unroll 4
    for (int j = 0; j < a.steps; ++j) {
        const int c = chunk0 + j * 32;
        uint4 u = make_uint4(K::kNone, K::kNone, K::kNone, K::kNone);
        if (c < chunks) {
            u = __ldg(src + c);
            if (c == 0 || c == chunks - 1) {  // what lies beside the row in its first and last chunk
                for (int i = 0; i < K::N; ++i) {
                    const int at = c * K::N - shift + i;
                    if (at < 0 || at >= a.V) K::drop(u, i);
                }
            }
        }
        mine[j * 32] = u;
        mx = fmaxf(mx, K::max(u));
    }
    if (tid < 64) s.table[tid] = exp2((double)tid / 64.0) * kSmpOne;
    if (tid == 0) s.n = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) s.redf[warp] = mx;
    __syncthreads();
    mx = s.redf[tid % kSmpWarps];
#pragma unroll
    for (int o = kSmpWarps / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (blocks > 1) {
        cluster.sync();  // every block runs before its shared memory is written from outside
        tell(&s.of_max[rank], mx);
        cluster.sync();
        for (int i = 0; i < blocks; ++i) mx = fmaxf(mx, s.of_max[i]);
    }
    if (mx == -INFINITY) {  // nothing to draw from
        if (rank == 0 && tid == 0) a.out[row] = -1;
        return;
    }

    const float temp = a.t ? __ldg(a.t + row) : a.t0, top_p = a.p ? __ldg(a.p + row) : a.p0,
                min_p = a.m ? __ldg(a.m + row) : a.m0;
    int k = a.k ? __ldg(a.k + row) : a.k0;
    SampleRow r;
    r.table = s.table;
    r.max = mx;
    // T <= 0 (and NaN) takes the first largest logit
    const bool greedy = !(temp > 0.0f);
    r.c = greedy ? 0.0 : 92.332482616893657 / (double)temp;
    r.per = greedy ? INFINITY : 64.0f / temp;
    r.floor = min_p > 0.0f ? max((uint64_t)__double2ull_ru(fmin((double)min_p, 1.0) * kSmpOne), (uint64_t)1) : 1;
    r.key = -INFINITY;
    r.ties = 0;
    if (greedy) k = 1;
    const bool by_k = k > 0 && k < a.V, by_p = top_p < 1.0f && !greedy;
    const double p = fmax((double)top_p, 0.0);
    // kept while the sum before an element is < top_p * total: need = ceil(top_p * total), at least 1
    auto share = [&](uint64_t total) { return max((uint64_t)ceil(p * (double)total), (uint64_t)1); };
    auto one = [](float) { return (uint64_t)1; };

    // Every element of the block's run that may have weight: f(x).
    auto each = [&](auto&& f) {
#pragma unroll 1
        for (int j = 0; j < a.steps; ++j) {
            const uint4 u = mine[j * 32];
            float v[K::N];
            K::get(u, v);
#pragma unroll
            for (int i = 0; i < K::N; ++i) f(v[i]);
        }
    };
    auto push = [&](float v) {
        const uint32_t at = atomicAdd(&s.n, 1);
        if (at < kSmpList) s.list[at] = v;
    };
    // The blocks' lists, joined in the first block's: how many; more than
    // kSmpList: they do not fit, and nothing is joined.
    auto join_lists = [&]() {
        __syncthreads();
        const uint32_t n = s.n;
        tell(&s.of_n[rank], n);
        sync();
        uint32_t at = 0, all = 0;
        for (int i = 0; i < blocks; ++i) {
            if (i < rank) at += s.of_n[i];
            all += s.of_n[i];
        }
        if (blocks > 1) {
            if (rank > 0 && all <= kSmpList) {
                float* to = cluster.map_shared_rank(s.list, 0) + at;
                for (uint32_t i = tid; i < n; i += kSmpThreads) to[i] = s.list[i];
            }
            cluster.sync();
        }
        return all;
    };
    // The first block's findings, for all.
    auto publish = [&](float key, uint32_t ties) {
        __syncthreads();
        if (rank == 0) {
            tell(&s.key, key);
            tell(&s.ties, ties);
        }
        sync();
        r.key = s.key;
        r.ties = s.ties;
        sync();
    };

    // The border by a histogram over the runs: sets r.key and r.ties so that value
    // (of logits above the present r.key; that border's own ties weigh tie_value
    // together) is kept up to need(total).  All blocks.
    auto dense = [&](auto&& value, uint64_t tie_value, auto&& need_of) {
        hist_clear(s);
        each([&](float v) {
            const int b = r.bucket(v);
            if (b < kSmpBuckets && v > r.key) {
                const uint64_t w = value(v);
                if (w) hist_add(s, b, w);
            }
        });
        if (rank == 0 && tid == 0 && tie_value) hist_add(s, r.bucket(r.key), tie_value);
        sync();
        if (rank == 0) {
            uint64_t sum = 0;
            for (int b = tid * 4; b < kSmpBuckets; b += kSmpThreads * 4) {
                uint64_t w[4] = {};
                for (int i = 0; i < blocks; ++i) {
                    const uint4 l = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(s.lo, i) + b);
                    const uint4 h = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(s.hi, i) + b);
                    w[0] += (uint64_t)h.x << 32 | l.x, w[1] += (uint64_t)h.y << 32 | l.y;
                    w[2] += (uint64_t)h.z << 32 | l.z, w[3] += (uint64_t)h.w << 32 | l.w;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s.lo[b + i] = (uint32_t)w[i], s.hi[b + i] = (uint32_t)(w[i] >> 32);
                    sum += w[i];
                }
            }
            const uint64_t total = block_sum(s, sum), need = need_of(total);
            if (need < total) find_bucket(s, [&](int b) { return (uint64_t)s.hi[b] << 32 | s.lo[b]; }, need);
            const uint64_t before = s.before;
            const uint32_t bucket = s.bucket;
            __syncthreads();
            tell(&s.total, total);
            if (need < total) {
                tell(&s.bucket, bucket);
                tell(&s.before, before);
            }
        }
        if (tid == 0) s.n = 0;
        sync();
        const uint64_t total = s.total, need = need_of(total);
        if (need >= total) {
            sync();
            return;
        }
        const int bucket = (int)s.bucket;
        const uint64_t left = need - s.before;
        each([&](float v) {
            if (r.bucket(v) == bucket && v > r.key && value(v) != 0) push(v);
        });
        const uint32_t n = join_lists();
        float key;
        uint64_t above;
        if (n <= kSmpList) {
            key = r.key, above = 0;
            if (rank == 0) {
                key = list_border(s, r, (int)n, bucket, left, value);
                above = s.sum;
            }
        } else {  // over the runs: all blocks see the same sums and take the same steps
            uint32_t lo = order_bits(r.key), hi = order_bits(r.max);
            above = 0;
            for (int step = 0; lo < hi; step ^= 1) {
                const uint32_t mid = lo + (hi - lo) / 2;
                uint64_t sum = 0;
                each([&](float v) {
                    if (order_bits(v) > mid && r.bucket(v) == bucket) sum += value(v);
                });
                sum = block_sum(s, sum);
                tell(&s.of_sum[step][rank], sum);
                sync();
                sum = 0;
                for (int i = 0; i < blocks; ++i) sum += s.of_sum[step][i];
                if (sum < left) {
                    hi = mid;
                    above = sum;
                } else {
                    lo = mid + 1;
                }
            }
            key = from_order(lo);
        }
        const uint64_t w = value(key), rest = left - above;
        uint32_t ties = w ? (uint32_t)min((rest + w - 1) / w, (uint64_t)0xffffffffu) : 0;
        if (key == r.key) ties = min(ties, r.ties);  // at the earlier border, whose ties come last
        publish(key, ties);
    };

    // ---- top-k and top-p
    if (by_k || by_p) {
        const bool all_weights = by_p && !by_k;  // top-p of the whole row: its sum is needed
        uint64_t sum = 0, cand = 0;
        if (all_weights) {
            each([&](float v) {
                const float at = r.place(v);
                if (at < (float)kSmpBuckets || v == r.max) {
                    const uint64_t w = r.weight(v);
                    sum += w;
                    if (w && (at < kSmpCut || v == r.max)) {
                        cand += w;
                        push(v);
                    }
                }
            });
            sum = block_sum(s, sum);
            cand = block_sum(s, cand);
        } else {
#pragma unroll 1
            for (int j = 0; j < a.steps; ++j) {
                const uint4 u = mine[j * 32];
                const float top = K::max(u);
                if (r.place(top) < kSmpCut || top == r.max) {
                    float v[K::N];
                    K::get(u, v);
#pragma unroll
                    for (int i = 0; i < K::N; ++i)
                        if (r.place(v[i]) < kSmpCut || v[i] == r.max) push(v[i]);
                }
            }
        }
        tell(&s.of_sum[0][rank], sum);
        tell(&s.of_cand[rank], cand);
        const uint32_t n = join_lists();
        sum = cand = 0;
        for (int i = 0; i < blocks; ++i) sum += s.of_sum[0][i], cand += s.of_cand[i];
        bool done_k = !by_k, done_p = !by_p;
        if (n <= kSmpList && (by_k ? n >= (uint32_t)k : cand >= share(sum))) {
            // the borders are among the candidates: the first block finds them
            float key = r.key;
            uint32_t ties = 0;
            if (rank == 0) {
                if (by_k) {
                    hist_clear(s);
                    for (int i = tid; i < (int)n; i += kSmpThreads) atomicAdd(&s.lo[r.bucket(s.list[i])], 1u);
                    __syncthreads();
                    find_bucket(s, [&](int b) { return (uint64_t)s.lo[b]; }, (uint64_t)k);
                    const uint64_t left = k - s.before;
                    key = list_border(s, r, (int)n, (int)s.bucket, left, one);
                    ties = (uint32_t)(left - s.sum);
                    r.key = key, r.ties = ties;
                }
                if (by_p) {
                    auto value = [&](float v) { return v > r.key ? r.weight(v) : (uint64_t)0; };
                    hist_clear(s);
                    uint64_t listed = 0;
                    for (int i = tid; i < (int)n; i += kSmpThreads) {
                        const float v = s.list[i];
                        const uint64_t w = value(v);
                        if (w) hist_add(s, r.bucket(v), w);
                        listed += w;
                    }
                    if (tid == 0 && r.ties) {
                        const uint64_t w = r.weight(r.key) * r.ties;
                        if (w) hist_add(s, r.bucket(r.key), w);
                        listed += w;
                    }
                    if (by_k) sum = block_sum(s, listed);
                    __syncthreads();
                    const uint64_t need = share(sum);
                    if (need < sum) {
                        find_bucket(s, [&](int b) { return (uint64_t)s.hi[b] << 32 | s.lo[b]; }, need);
                        const uint64_t left = need - s.before;
                        key = list_border(s, r, (int)n, (int)s.bucket, left, value);
                        const uint64_t rest = left - s.sum, w = r.weight(key);
                        ties = w ? (uint32_t)min((rest + w - 1) / w, (uint64_t)0xffffffffu) : 0;
                        if (key == r.key) ties = min(ties, r.ties);
                    }
                }
                __syncthreads();
            }
            publish(key, ties);
            done_k = done_p = true;
        }
        if (!done_k)  // (no cut where there are not more than k logits with weight)
            dense(one, 0, [&](uint64_t total) { return min((uint64_t)k, total); });
        if (!done_p) {
            const float key = r.key;
            dense([&](float v) { return r.weight(v); }, r.ties ? r.weight(key) * r.ties : 0, share);
        }
    }

    // ---- draw
    uint64_t sum = 0;
    uint32_t ties = 0;
#pragma unroll 1
    for (int j = 0; j < a.steps; ++j) {
        const uint4 u = mine[j * 32];
        if (K::max(u) >= r.key) {
            float v[K::N];
            K::get(u, v);
#pragma unroll
            for (int i = 0; i < K::N; ++i) {
                if (v[i] > r.key && (r.place(v[i]) < (float)kSmpBuckets || v[i] == r.max)) sum += r.weight(v[i]);
                if (r.ties && v[i] == r.key) ++ties;
            }
        }
    }
    sum = warp_sum_u64(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    __syncthreads();
    if (lane == 0) s.redc[warp] = ties, s.red[warp] = sum;
    __syncthreads();
    uint64_t of_block = 0, before = 0;  // without ties
    uint32_t ties_of_block = 0, ties_before = 0;
    for (int i = 0; i < kSmpWarps; ++i) {
        if (i < warp) before += s.red[i], ties_before += s.redc[i];
        of_block += s.red[i], ties_of_block += s.redc[i];
    }
    uint64_t total = of_block;
    uint32_t all_ties = ties_of_block;
    if (blocks > 1) {
        tell(&s.of_sum[0][rank], of_block);
        tell(&s.of_n[rank], ties_of_block);
        cluster.sync();
        total = 0, all_ties = 0;
        for (int i = 0; i < blocks; ++i) {
            if (i < rank) before += s.of_sum[0][i], ties_before += s.of_n[i];
            total += s.of_sum[0][i], all_ties += s.of_n[i];
        }
    }
    const uint64_t wk = r.ties ? r.weight(r.key) : 0;
    const uint32_t quota = r.ties > ties_before ? min(r.ties - ties_before, ties) : 0;  // this warp's kept ties
    before += min(ties_before, r.ties) * wk;
    total += min(all_ties, r.ties) * wk;
    sum += quota * wk;
    const double ud = fmin(fmax((double)__ldg(a.u + row), 0.0), 1.0);
    // first index whose running sum exceeds u * total; u = 1 takes the last kept one
    const uint64_t target = min((uint64_t)(ud * (double)total), total - 1);
    if (target >= before && target < before + sum) {  // one warp of the cluster
        uint32_t left = quota;
        uint64_t at = before;
        for (int j = 0; j < a.steps; ++j) {
            const uint4 u = mine[j * 32];
            if (!__any_sync(0xffffffffu, K::max(u) >= r.key)) continue;
            float v[K::N];
            K::get(u, v);
            uint64_t w[K::N], own = 0;
            uint32_t eq = 0;
#pragma unroll
            for (int i = 0; i < K::N; ++i) {
                w[i] = v[i] > r.key && (r.place(v[i]) < (float)kSmpBuckets || v[i] == r.max) ? r.weight(v[i]) : 0;
                eq += r.ties && v[i] == r.key ? 1 : 0;
            }
            uint32_t eq_before = eq;  // ties in lower lanes
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t n = __shfl_up_sync(0xffffffffu, eq_before, o);
                if (lane >= o) eq_before += n;
            }
            const uint32_t eq_all = __shfl_sync(0xffffffffu, eq_before, 31);
            eq_before -= eq;
#pragma unroll
            for (int i = 0; i < K::N; ++i) {
                if (r.ties && v[i] == r.key && eq_before++ < left) w[i] = wk;
                own += w[i];
            }
            left -= min(left, eq_all);
            uint64_t inc = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t n = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += n;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, at + inc > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    uint64_t run = at + inc - own;
                    int token = -1;
#pragma unroll
                    for (int i = 0; i < K::N; ++i) {
                        run += w[i];
                        if (token < 0 && run > target) token = (chunk0 + j * 32) * K::N - shift + i;
                    }
                    a.out[row] = token;
                }
                break;
            }
            at += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    if (blocks > 1) cluster.sync();  // no block leaves while another may write to it
}

template <typename T>
static cudaError_t launch_sample(SampleArgs a, int64_t rows, cudaStream_t s) {
    // chunks of a row, wherever its first byte lies
    const int64_t chunks = (a.V + 2 * SmpChunk<T>::N - 2) / SmpChunk<T>::N;
    const int64_t sms = device_sm_count() > 0 ? device_sm_count() : 148;
    // Blocks per row: at least what holds it at 8 chunks per thread (64 KB, two
    // blocks per SM) or, beyond eight blocks, more chunks per thread; more blocks
    // while a row more or less would leave SMs idle, down to one chunk per thread.
    int64_t blocks = (chunks + 8 * kSmpThreads - 1) / (8 * kSmpThreads);
    const int64_t most = (chunks + kSmpThreads - 1) / kSmpThreads;
    while (blocks < most && blocks < kSmpBlocks && rows * (blocks + 1) <= 2 * sms) ++blocks;
    if (blocks > kSmpBlocks) blocks = kSmpBlocks;
    a.steps = (int)((chunks + blocks * kSmpThreads - 1) / (blocks * kSmpThreads));
    const size_t smem = (size_t)a.steps * kSmpThreads * 16 + sizeof(SampleShared);
    static bool done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) done[dev] = true;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * blocks));
    cfg.blockDim = dim3(kSmpThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
}

}  // namespace pn

extern "C" int pn_sample_tokens(const void* logits, int x_dtype, int64_t rows, int64_t vocab, int64_t ld, const float* u,
                                const float* temperature, float temperature0, const int32_t* top_k, int32_t top_k0,
                                const float* top_p, float top_p0, const float* min_p, float min_p0, int64_t* tokens,
                                void* stream) {
    if (x_dtype != PN_F32 && x_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "pn_sample_tokens: dtype %d", x_dtype);
    if (rows < 0 || rows > 0x7fffffff / pn::kSmpBlocks || vocab < 1 || vocab > pn::kSmpMaxVocab || ld < vocab)
        return fail(PN_ERR_SHAPE, "pn_sample_tokens: rows=%lld vocab=%lld (at most %lld) ld=%lld", (long long)rows,
                    (long long)vocab, (long long)pn::kSmpMaxVocab, (long long)ld);
    if (rows > 0 && (!logits || !u || !tokens)) return fail(PN_ERR_ARG, "pn_sample_tokens: null pointer");
    if (!aligned(logits, x_dtype == PN_F32 ? 4 : 2) || !aligned(u, 4) || !aligned(temperature, 4) || !aligned(top_k, 4) ||
        !aligned(top_p, 4) || !aligned(min_p, 4) || !aligned(tokens, 8))
        return fail(PN_ERR_ALIGN, "pn_sample_tokens: misaligned pointer");
    if (int st = check_device()) return st;
    if (rows == 0) return ok();
    const pn::SampleArgs a = {logits, ld, (int)vocab, 0, u, temperature, top_k, top_p, min_p, temperature0, top_p0, min_p0, top_k0,
                              tokens};
    const cudaError_t e = x_dtype == PN_F32 ? pn::launch_sample<float>(a, rows, (cudaStream_t)stream)
                                            : pn::launch_sample<__nv_bfloat16>(a, rows, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "pn_sample_tokens");
}
