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
// No sort.  The candidates, a few hundred in a model's distribution, are for top-k
// the logits not below the k-th largest of some block's per-thread maxima (there
// are k such at least), for top-p alone those within 2^-12 of the largest weight.
// They are brought to the first block, which finds the k-th largest and the border
// of top-p by a histogram over (max - x) / T, 32 buckets to an octave of weight, and
// then among the few logits of one bucket.  Where the candidates do not reach the
// border, or do not fit (flat distributions, k above 256), the histogram is taken
// over the blocks' runs instead, and the border's bucket is searched by bisection on
// the logits' ordered bit patterns: on a list of them or, where one bucket holds too
// many (all logits nearly alike), over the runs themselves.
//
// What bounds it: the chain of short steps, each behind a barrier of the block or the
// cluster (1 to 2 us); in large batches over flat distributions also the weights, about
// thirty instructions each (six of them fp64; the split into table index and rest runs in
// fp32), computed up to three times (sum, histogram, draw: 84 instructions per logit, 45 % of
// the issue slots used), and the histogram's atomics.  One bf16 row of 50257, top-k 50
// and top-p: 18.6 us; 64 fp32 rows with settings of their own: 25.6 us; 256 rows of 131071
// with top-p alone over a flat distribution: 219 us, five waves of clusters (a histogram of
// all weights in the first pass: 302 us; candidates down to 2^-16 of the largest: 236 us).
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
constexpr int kSmpUnits = 46 * 256;  // (max - x) / T in 1/256 octaves from which a weight is zero; eight units to a bucket
constexpr int kSmpList = 4096;
constexpr int kSmpBlocks = 8;  // of a cluster, at most
constexpr int64_t kSmpMaxVocab = 1 << 18;
constexpr double kSmpOne = 35184372088832.0;  // 2^45
constexpr float kSmpCut = 12 * 256;           // top-p's candidates lie within 12 octaves of the largest weight
constexpr int kSmpKMost = kSmpThreads / 2;    // top-k of at most so many takes its candidates by the threads' maxima

// One row's rule.  A logit is kept when it lies above `key`, or equals it and is
// among the first `ties` such in index order, and its weight is not zero.
struct SampleRow {
    float max;
    float per;       // 256 log2(e) / T
    double c;        // the same in fp64
    uint64_t floor;  // min-p as a weight (at least 1)
    bool flat;       // all weights are zero or one: T <= 0, or a maximum of +inf
    float key;
    uint32_t ties;

    // (max - x) / T in 1/256 octaves, monotone; kSmpUnits and more: no weight.  (The
    // products that are NaN belong to the maximum itself: 0 * inf, inf - inf.)
    __device__ __forceinline__ float place(float x) const { return fmaxf((max - x) * per, 0.0f); }
    __device__ __forceinline__ int bucket(float x) const { return (int)fminf(place(x), (float)kSmpUnits) >> 3; }
    static constexpr int kNone = kSmpUnits >> 3;  // the bucket of logits without weight
};

struct SampleFound {
    float key;
    uint32_t ties;
    uint32_t ok;  // the candidates sufficed
};

struct SampleShared {
    double table[256];  // 2^(45 - j / 256)
    uint32_t lo[kSmpBuckets], hi[kSmpBuckets];  // 64-bit sums in two halves (shared memory adds 32 bits natively)
    float list[kSmpList];
    SampleRow row;
    uint64_t red[kSmpWarps];
    uint32_t redc[kSmpWarps];
    float redf[kSmpWarps];
    // read by the other blocks of the cluster between two of its barriers
    float max, kth;
    uint32_t n;  // logits pushed to list (those past kSmpList are not held)
    uint64_t sum;
    uint64_t part[2];
    uint64_t kept;
    uint32_t kept_ties;
    // written by the first block
    SampleFound found[3];
    uint64_t total[2], before[2];
    uint32_t bucket[2];
    // within the block
    uint64_t b_sum, b_before;
    uint32_t b_bucket;
    float b_key;
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

// 2^45 exp((x - max) / T) + 2^52 rounded to a whole number, as its bit pattern, for a
// logit of weight at `place`: the weight is what exceeds kSmpBase.  With (x - max) / T =
// (f - n) / 256 octaves, n = rint(place): 2^(45 - n / 256) from the table and the exponent,
// 2^(f / 256) from its series (|f| <= 0.51, so the fourth term is below 2^-42 of the sum).
constexpr uint64_t kSmpBase = 0x4330000000000000ull;
__device__ __forceinline__ uint64_t smp_weight52(const double* table, float x, float place, double max, double c) {
    constexpr double a1 = 0.0027076061740622863, a2 = a1 * a1 / 2, a3 = a2 * a1 / 3;  // ln 2 / 256
    const float m = place + 12582912.0f;  // 1.5 * 2^23: the low bits are n
    const int n = __float_as_int(m) & 0x3FFFFF;
    const double f = fma((double)x - max, c, (double)(m - 12582912.0f));
    const double p = fma(f, fma(f, fma(f, a3, a2), a1), 1.0);
    const double t = table[n & 255];
    return (uint64_t)__double_as_longlong(fma(__hiloint2double(__double2hiint(t) - ((n >> 8) << 20), __double2loint(t)), p, 4503599627370496.0));
}

// The weights of N logits, those without one as 0.
template <int N>
__device__ __forceinline__ void smp_weights(const SampleShared& s, const float (&v)[N], uint64_t (&w)[N]) {
    const SampleRow& r = s.row;
    const double max = (double)r.max, c = r.c;
    const float mx = r.max, per = r.per;
    const bool flat = r.flat;
    const uint64_t floor = r.floor;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float at = fmaxf((mx - v[i]) * per, 0.0f);
        const bool in = at < (float)kSmpUnits;
        const uint64_t q = flat ? (uint64_t)kSmpOne : smp_weight52(s.table, in ? v[i] : mx, in ? at : 0.0f, max, c) - kSmpBase;
        w[i] = in && q >= floor ? q : 0;
    }
}
// The weight of a logit of weight, 0 below the floor.
__device__ __noinline__ uint64_t smp_weight(const SampleShared& s, float x) {
    if (s.row.flat) return (uint64_t)kSmpOne;
    const uint64_t w = smp_weight52(s.table, x, s.row.place(x), (double)s.row.max, s.row.c) - kSmpBase;
    return w >= s.row.floor ? w : 0;
}

// 16 bytes of logits as fp32.  clean: a NaN becomes -inf, and -0 becomes +0 (the sum
// with +0), so that equal logits have one bit pattern and the order of patterns is that of
// the logits.
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
    static __device__ __forceinline__ uint32_t clean(uint32_t w) {
        return __float_as_uint(__fadd_rn(fmaxf(__uint_as_float(w), -INFINITY), 0.0f));
    }
    static __device__ __forceinline__ void set_none(uint8_t* p) { *reinterpret_cast<uint32_t*>(p) = kNone; }
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
    static __device__ __forceinline__ uint32_t clean(uint32_t w) {
        uint32_t r;
        asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(max2(w, kNone)), "r"(0));
        return r;
    }
    static __device__ __forceinline__ void set_none(uint8_t* p) { *reinterpret_cast<uint16_t*>(p) = 0xFF80; }
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
// >= need) and the sum before it, in s.b_bucket and s.b_before.  All buckets together
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
            s.b_bucket = tid * per + i;
            s.b_before = before;
        }
        before += v[i];
    }
    __syncthreads();
}

// What is summed: the number of logits, or their weights, above the row's present key.
__device__ __forceinline__ uint64_t smp_value(const SampleShared& s, float x, bool weights) {
    return x <= s.row.key ? 0 : weights ? smp_weight(s, x) : 1;
}

// Of the n listed logits in `bucket`: the smallest key v (not below the present one)
// for which the sum of values over x > v is below `need`; that sum goes to s.b_sum.
// While more than a warp's logits are in question, a histogram over their ordered
// bit patterns leaves those of one of 2048 equal parts of their range.
__device__ __noinline__ float list_border(SampleShared& s, int n, int bucket, uint64_t need, bool weights) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const SampleRow& r = s.row;
    auto value = [&](float v) { return smp_value(s, v, weights); };
    uint32_t from = 0, to = 0xffffffffu;  // the patterns in question
    uint64_t done = 0;                    // sum of the values above them
#pragma unroll 1
    while (true) {
        uint32_t least = 0xffffffffu, most = 0, count = 0;
        __syncthreads();
        if (tid == 0) s.n_few = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kSmpThreads) {
            const float v = s.list[i];
            const uint32_t o = order_bits(v);
            if (v > r.key && r.bucket(v) == bucket && o >= from && o <= to) {
                least = min(least, o), most = max(most, o);
                ++count;
                const uint32_t at = atomicAdd(&s.n_few, 1);
                if (at < 32) s.few[at] = v;
            }
        }
        least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) s.redc[warp] = least, s.red[warp] = most;
        __syncthreads();
        least = __reduce_min_sync(0xffffffffu, s.redc[tid % kSmpWarps]);
        most = __reduce_max_sync(0xffffffffu, (uint32_t)s.red[tid % kSmpWarps]);
        const int few = (int)s.n_few;
        if (few <= 32) {
            // the border is the largest of them with sum over x >= key of at least need, or the present key
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
                    s.b_key = b ? mine : r.key;
                    s.b_sum = done + (b ? above : all);
                }
            }
            __syncthreads();
            return s.b_key;
        }
        if (least == most) {  // one key, many times
            const uint64_t all = block_sum(s, value(from_order(least)) * count);
            if (tid == 0) s.b_sum = all >= need ? done : done + all;
            __syncthreads();
            return all >= need ? from_order(least) : r.key;
        }
        const int shift = max(32 - __clz(most - least) - 11, 0);
        hist_clear(s);
        uint64_t all = 0;
        for (int i = tid; i < n; i += kSmpThreads) {
            const float v = s.list[i];
            const uint32_t o = order_bits(v);
            if (v > r.key && r.bucket(v) == bucket && o >= least && o <= most) {
                const uint64_t w = value(v);
                if (w) hist_add(s, (int)((most - o) >> shift), w);
                all += w;
            }
        }
        all = block_sum(s, all);
        if (all < need) {  // the border is the present key
            if (tid == 0) s.b_sum = done + all;
            __syncthreads();
            return r.key;
        }
        find_bucket(s, [&](int b) { return (uint64_t)s.hi[b] << 32 | s.lo[b]; }, need);
        const uint32_t b = s.b_bucket;
        done += s.b_before, need -= s.b_before;
        to = most - (b << shift);
        from = to - least >= (1u << shift) ? to - (1u << shift) + 1 : least;
    }
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
    // another block's entry of s
    auto of = [&](auto* entry, int i) { return *cluster.map_shared_rank(entry, i); };
    // after a barrier: the sum of the blocks' entries
    auto total_of = [&](auto* entry) {
        auto v = of(entry, lane < blocks ? lane : 0);
        if (lane >= blocks) v = 0;
#pragma unroll
        for (int o = kSmpBlocks / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return __shfl_sync(0xffffffffu, v, 0);
    };
    // writes the first block's value to every block's entry
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
    const float t_in = a.t ? __ldg(a.t + row) : a.t0, temp = t_in > 1e30f ? 1e30f : t_in,  // (all finite logits weigh the same)
                top_p = a.p ? __ldg(a.p + row) : a.p0,
                min_p = a.m ? __ldg(a.m + row) : a.m0;
    int k = a.k ? __ldg(a.k + row) : a.k0;
    const double ud = fmin(fmax((double)__ldg(a.u + row), 0.0), 1.0);
    // T <= 0 (and NaN) takes the first largest logit
    const bool greedy = !(temp > 0.0f);
    if (greedy) k = 1;
    const bool by_k = k > 0 && k < a.V, by_p = top_p < 1.0f && !greedy;
    float mx = -INFINITY;
#pragma unroll 4
    for (int j = 0; j < a.steps; ++j) {
        const int c = chunk0 + j * 32;
        uint4 u = make_uint4(K::kNone, K::kNone, K::kNone, K::kNone);
        if (c < chunks) {
            u = __ldg(src + c);
            u.x = K::clean(u.x), u.y = K::clean(u.y), u.z = K::clean(u.z), u.w = K::clean(u.w);
        }
        mine[j * 32] = u;
        if (c == 0 || c == chunks - 1) {  // what lies beside the row in its first and last chunk
#pragma unroll 1
            for (int i = 0; i < K::N; ++i) {
                const int at = c * K::N - shift + i;
                if (at < 0 || at >= a.V) K::set_none(reinterpret_cast<uint8_t*>(mine + j * 32) + i * sizeof(T));
            }
            u = mine[j * 32];
        }
        mx = fmaxf(mx, K::max(u));
    }
    if (tid < 256) s.table[tid] = exp2(45.0 - (double)tid / 256.0);
    if (tid == 0) s.n = 0;
    const float own = mx;
    auto warp_max = [](float v, int lanes) {
        for (int o = lanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    };
    mx = warp_max(mx, 32);
    if (lane == 0) s.redf[warp] = mx;
    __syncthreads();
    mx = warp_max(s.redf[tid % kSmpWarps], kSmpWarps);
    float kth = -INFINITY;  // not above the k-th largest logit
    if (by_k && k <= kSmpKMost && mx > -INFINITY) {
        uint32_t lo = order_bits(-INFINITY), hi = order_bits(mx);  // k threads or more are not below lo
        if (k == 1) lo = hi;
        // the 14 bits below the first in which the border can differ settle it well enough
        const uint32_t from = order_bits(own);
        const float least = mx - 64.0f * fabsf(mx) - 64.0f;
        if (__syncthreads_count(own >= least) >= k) lo = max(lo, order_bits(least));
#pragma unroll 1
        for (int i = 0; i < 16 && lo < hi; ++i) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            if (__syncthreads_count(from >= mid) >= k)
                lo = mid;
            else
                hi = mid - 1;
        }
        kth = from_order(lo);
    }
    if (blocks > 1) {
        if (tid == 0) s.max = mx, s.kth = kth;
        cluster.sync();
        const int i = lane < blocks ? lane : 0;
        mx = of(&s.max, i), kth = of(&s.kth, i);
        mx = __shfl_sync(0xffffffffu, warp_max(mx, kSmpBlocks), 0);
        kth = __shfl_sync(0xffffffffu, warp_max(kth, kSmpBlocks), 0);
    }
    SampleRow& r = s.row;
    if (tid == 0) {
        r.max = mx;
        r.per = greedy ? INFINITY : fmaxf(369.32993f / temp, 1.2e-38f);
        r.c = greedy ? 0.0 : 369.32993046757463 / (double)temp;
        r.floor = min_p > 0.0f ? max((uint64_t)__double2ull_ru(fmin((double)min_p, 1.0) * kSmpOne), (uint64_t)1) : 1;
        r.flat = greedy || mx == INFINITY;
        r.key = -INFINITY;
        r.ties = 0;
    }
    __syncthreads();
    const double p = fmax((double)top_p, 0.0);
    // kept while the sum before an element is < top_p * total: need = ceil(top_p * total), at least 1
    auto share = [&](uint64_t total) { return max((uint64_t)ceil(p * (double)total), (uint64_t)1); };

    // Every logit of the thread's part of the run: f(x).
    auto each = [&](auto&& f) {
#pragma unroll 1
        for (int j = 0; j < a.steps; ++j) {
            const T* e = reinterpret_cast<const T*>(mine + j * 32);
#pragma unroll 1
            for (int i = 0; i < K::N; ++i) f((float)e[i]);
        }
    };
    auto push = [&](float v) {
        if (*const_cast<volatile uint32_t*>(&s.n) > kSmpList) return;  // too many: how many does not matter
        const uint32_t at = atomicAdd(&s.n, 1);
        if (at < kSmpList) s.list[at] = v;
    };
    // After a barrier: all blocks' lists into the first block's (they fit).  The first block.
    auto pull_lists = [&]() {
        if (blocks > 1) {
            const uint32_t n = of(&s.n, lane < blocks ? lane : 0);
            const int from = 1 + warp % (blocks - 1);  // a warp or more per block
            const uint32_t at = __reduce_add_sync(0xffffffffu, lane < from ? n : 0), count = __shfl_sync(0xffffffffu, n, from);
            const float* list = cluster.map_shared_rank(s.list, from);
            const int warps = (kSmpWarps - from) / (blocks - 1) + 1;
            for (uint32_t e = warp / (blocks - 1) * 32 + lane; e < count; e += warps * 32) s.list[at + e] = list[e];
        }
        __syncthreads();
    };
    // The first block's findings, for all.
    auto publish = [&](int slot, float key, uint32_t ties, uint32_t ok) {
        __syncthreads();
        if (rank == 0) tell(&s.found[slot], SampleFound{key, ties, ok});
        sync();
        if (tid == 0) r.key = s.found[slot].key, r.ties = s.found[slot].ties;
        __syncthreads();
        return s.found[slot].ok != 0;
    };
    // How many of a border's ties are kept when `rest` is still missing above it.
    auto ties_for = [&](float key, uint64_t rest, bool weights) {
        const uint64_t w = weights ? smp_weight(s, key) : 1;
        uint32_t ties = w ? (uint32_t)min((rest + w - 1) / w, (uint64_t)0xffffffffu) : 0;
        if (key == r.key) ties = min(ties, r.ties);  // at the earlier border, whose own ties come last
        return ties;
    };

    // ---- top-k and top-p
    if ((by_k || by_p) && mx > -INFINITY) {
        uint64_t sum = 0;
        const bool try_list = !by_k || k <= kSmpKMost;
        bool done = false;
        if (try_list) {
            uint64_t part = 0;
            const float cut = by_k ? (float)kSmpUnits : kSmpCut;
#pragma unroll 1
            for (int j = 0; j < a.steps; ++j) {
                const uint4 u = mine[j * 32];
                const float top = K::max(u), top_at = r.place(top);
                if (!(top >= kth && top_at < (float)kSmpUnits)) continue;
                float v[K::N];
                K::get(u, v);
                if (!by_k) {  // top-p of the whole row: its sum is needed
                    uint64_t w[K::N];
                    smp_weights(s, v, w);
#pragma unroll
                    for (int i = 0; i < K::N; ++i) part += w[i];
                    if (top_at >= kSmpCut) continue;
                }
#pragma unroll
                for (int i = 0; i < K::N; ++i)
                    if (v[i] >= kth && r.place(v[i]) < cut) push(v[i]);
            }
            if (!by_k) {
                sum = block_sum(s, part);
                if (tid == 0) s.sum = sum;
            }
            sync();
            const uint32_t n = total_of(&s.n);
            if (!by_k) sum = total_of(&s.sum);
            if (n <= kSmpList) {  // the first block looks for the borders among the candidates
                bool ok = true;
                if (rank == 0) {
                    pull_lists();
                    if (by_k && n > (uint32_t)k) {  // (fewer: all with any weight are candidates, and are kept)
                        hist_clear(s);
                        for (int i = tid; i < (int)n; i += kSmpThreads) atomicAdd(&s.lo[r.bucket(s.list[i])], 1u);
                        __syncthreads();
                        find_bucket(s, [&](int b) { return (uint64_t)s.lo[b]; }, (uint64_t)k);
                        const uint64_t left = k - s.b_before;
                        const float key = list_border(s, (int)n, (int)s.b_bucket, left, false);
                        if (tid == 0) r.key = key, r.ties = (uint32_t)(left - s.b_sum);
                    } else if (by_k && n == (uint32_t)k) {  // all candidates, and nothing below them
                        float low = INFINITY;
                        for (int i = tid; i < (int)n; i += kSmpThreads) low = fminf(low, s.list[i]);
                        low = -warp_max(-low, 32);
                        if (lane == 0) s.redf[warp] = low;
                        __syncthreads();
                        low = -warp_max(-s.redf[tid % kSmpWarps], kSmpWarps);
                        uint64_t same = 0;
                        for (int i = tid; i < (int)n; i += kSmpThreads) same += s.list[i] == low;
                        same = block_sum(s, same);
                        if (tid == 0) r.key = low, r.ties = (uint32_t)same;
                    }
                    __syncthreads();
                    if (by_p) {
                        uint64_t listed = 0;
                        for (int i = tid; i < (int)n; i += kSmpThreads) listed += smp_value(s, s.list[i], true);
                        if (tid == 0 && r.ties) listed += smp_weight(s, r.key) * r.ties;
                        listed = block_sum(s, listed);
                        if (by_k) sum = listed;
                        const uint64_t need = share(sum);
                        ok = listed >= need;
                        if (ok && need < sum) {
                            hist_clear(s);
                            for (int i = tid; i < (int)n; i += kSmpThreads) {
                                const uint64_t w = smp_value(s, s.list[i], true);
                                if (w) hist_add(s, r.bucket(s.list[i]), w);
                            }
                            if (tid == 0 && r.ties) {
                                const uint64_t w = smp_weight(s, r.key) * r.ties;
                                if (w) hist_add(s, r.bucket(r.key), w);
                            }
                            __syncthreads();
                            find_bucket(s, [&](int b) { return (uint64_t)s.hi[b] << 32 | s.lo[b]; }, need);
                            const uint64_t left = need - s.b_before;
                            const float key = list_border(s, (int)n, (int)s.b_bucket, left, true);
                            const uint32_t ties = ties_for(key, left - s.b_sum, true);
                            __syncthreads();
                            if (tid == 0) r.key = key, r.ties = ties;
                        }
                    }
                    __syncthreads();
                }
                done = publish(0, r.key, r.ties, ok);
            }
        }
        // By a histogram over the runs, first for top-k, then for top-p: all blocks.
#pragma unroll 1
        for (int pass = 0; pass < 2 && !done; ++pass) {
            const bool weights = pass == 1;
            if (!(weights ? by_p : by_k)) continue;
            hist_clear(s);
#pragma unroll 1
            for (int j = 0; j < a.steps; ++j) {
                const uint4 u = mine[j * 32];
                const float top = K::max(u);
                if (!(top > r.key && r.place(top) < (float)kSmpUnits)) continue;
                float v[K::N];
                K::get(u, v);
                if (weights) {
                    uint64_t w[K::N];
                    smp_weights(s, v, w);
#pragma unroll
                    for (int i = 0; i < K::N; ++i)
                        if (v[i] > r.key && w[i]) hist_add(s, r.bucket(v[i]), w[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < K::N; ++i) {
                        const int b = r.bucket(v[i]);
                        if (v[i] > r.key && b < SampleRow::kNone) atomicAdd(&s.lo[b], 1u);
                    }
                }
            }
            if (rank == 0 && tid == 0 && r.ties) {  // (top-p behind top-k) the earlier border's own ties
                const uint64_t w = smp_weight(s, r.key) * r.ties;
                if (w) hist_add(s, r.bucket(r.key), w);
            }
            sync();
            auto need_of = [&](uint64_t total) { return weights ? share(total) : min((uint64_t)k, total); };
            if (rank == 0) {
                uint64_t all = 0;
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
                        all += w[i];
                    }
                }
                all = block_sum(s, all);
                const uint64_t need = need_of(all);
                if (need < all) {
                    find_bucket(s, [&](int b) { return (uint64_t)s.hi[b] << 32 | s.lo[b]; }, need);
                    tell(&s.bucket[pass], s.b_bucket);
                    tell(&s.before[pass], s.b_before);
                }
                tell(&s.total[pass], all);
            }
            if (tid == 0) s.n = 0;
            sync();
            const uint64_t total = s.total[pass], need = need_of(total);
            if (need >= total) continue;  // no cut
            const int bucket = (int)s.bucket[pass];
            const uint64_t left = need - s.before[pass];
#pragma unroll 1
            for (int j = 0; j < a.steps; ++j) {
                const uint4 u = mine[j * 32];
                if (r.bucket(K::max(u)) > bucket) continue;
                float v[K::N];
                K::get(u, v);
#pragma unroll
                for (int i = 0; i < K::N; ++i)
                    if (v[i] > r.key && r.bucket(v[i]) == bucket) push(v[i]);
            }
            sync();
            const uint32_t n = total_of(&s.n);
            float key = r.key;
            uint64_t above = 0;
            if (n <= kSmpList) {
                if (rank == 0) {
                    pull_lists();
                    key = list_border(s, (int)n, bucket, left, weights);
                    above = s.b_sum;
                }
            } else {  // over the runs: all blocks see the same sums and take the same steps
                uint32_t lo = order_bits(r.key), hi = order_bits(r.max);
#pragma unroll 1
                for (int step = 0; lo < hi; step ^= 1) {
                    const uint32_t mid = lo + (hi - lo) / 2;
                    uint64_t part = 0;
                    each([&](float v) {
                        if (order_bits(v) > mid && r.bucket(v) == bucket) part += smp_value(s, v, weights);
                    });
                    part = block_sum(s, part);
                    if (tid == 0) s.part[step] = part;
                    sync();
                    part = total_of(&s.part[step]);
                    if (part < left) {
                        hi = mid;
                        above = part;
                    } else {
                        lo = mid + 1;
                    }
                }
                key = from_order(lo);
            }
            publish(1 + pass, key, ties_for(key, left - above, weights), 1);
        }
    }

    // ---- draw
    const float key = r.key;
    const uint32_t key_ties = r.ties;
    uint64_t sum = 0;
    uint32_t ties = 0;
#pragma unroll 1
    for (int j = 0; j < a.steps; ++j) {
        const uint4 u = mine[j * 32];
        const float top = K::max(u);
        if (top < key || !(r.place(top) < (float)kSmpUnits)) continue;
        float v[K::N];
        uint64_t w[K::N];
        K::get(u, v);
        smp_weights(s, v, w);
#pragma unroll
        for (int i = 0; i < K::N; ++i) {
            sum += v[i] > key ? w[i] : 0;
            ties += key_ties && v[i] == key ? 1 : 0;
        }
    }
    sum = warp_sum_u64(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) s.redc[warp] = ties, s.red[warp] = sum;
    __syncthreads();
    // sums without ties: before this warp, of all
    uint64_t total = lane < kSmpWarps ? s.red[lane] : 0, before = lane < warp ? total : 0;
    uint32_t all_ties = lane < kSmpWarps ? s.redc[lane] : 0, ties_before = lane < warp ? all_ties : 0;
    before = warp_sum_u64(before), ties_before = __reduce_add_sync(0xffffffffu, ties_before);
    total = warp_sum_u64(total), all_ties = __reduce_add_sync(0xffffffffu, all_ties);
    if (blocks > 1) {
        if (tid == 0) s.kept = total, s.kept_ties = all_ties;
        cluster.sync();
        const int i = lane < blocks ? lane : 0;
        total = of(&s.kept, i), all_ties = of(&s.kept_ties, i);
        if (lane >= blocks) total = 0, all_ties = 0;
        before += warp_sum_u64(lane < rank ? total : 0);
        ties_before += __reduce_add_sync(0xffffffffu, lane < rank ? all_ties : 0);
        total = warp_sum_u64(total), all_ties = __reduce_add_sync(0xffffffffu, all_ties);
        // no block leaves while another may read from it
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    const uint64_t wk = key_ties ? smp_weight(s, key) : 0;
    const uint32_t quota = key_ties > ties_before ? min(key_ties - ties_before, ties) : 0;  // this warp's kept ties
    before += min(ties_before, key_ties) * wk;
    total += min(all_ties, key_ties) * wk;
    sum += quota * wk;
    if (mx == -INFINITY) {  // nothing to draw from
        if (rank == 0 && tid == 0) a.out[row] = -1;
        total = sum = 0;
    }
    // first index whose running sum exceeds u * total; u = 1 takes the last kept one
    const uint64_t target = total ? min((uint64_t)(ud * (double)total), total - 1) : 0;
    if (target >= before && target < before + sum) {  // one warp of the cluster
        uint32_t left = quota;
        uint64_t at = before;
#pragma unroll 1
        for (int j = 0; j < a.steps; ++j) {
            const float top = K::max(mine[j * 32]);
            if (!__any_sync(0xffffffffu, top >= key && r.place(top) < (float)kSmpUnits)) continue;
            const T* e = reinterpret_cast<const T*>(mine + j * 32);
            auto weigh = [&](float v, uint32_t& eq, uint32_t ahead) -> uint64_t {
                if (v > key) return r.place(v) < (float)kSmpUnits ? smp_weight(s, v) : 0;
                if (!key_ties || v != key) return 0;
                return ahead + eq++ < left ? wk : 0;
            };
            uint32_t eq = 0, eq_before = 0;  // ties of this lane; of lower lanes
#pragma unroll 1
            for (int i = 0; i < K::N; ++i) eq += key_ties && (float)e[i] == key ? 1 : 0;
            eq_before = eq;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t n = __shfl_up_sync(0xffffffffu, eq_before, o);
                if (lane >= o) eq_before += n;
            }
            const uint32_t eq_all = __shfl_sync(0xffffffffu, eq_before, 31);
            eq_before -= eq;
            uint64_t own = 0;
            eq = 0;
#pragma unroll 1
            for (int i = 0; i < K::N; ++i) own += weigh((float)e[i], eq, eq_before);
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
                    eq = 0;
                    int i = 0;
#pragma unroll 1
                    for (; i < K::N; ++i) {
                        run += weigh((float)e[i], eq, eq_before);
                        if (run > target) break;
                    }
                    a.out[row] = (chunk0 + j * 32) * K::N - shift + i;
                }
                break;
            }
            left -= min(left, eq_all);
            at += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    if (blocks > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

template <typename T>
static cudaError_t launch_sample(SampleArgs a, int64_t rows, cudaStream_t s) {
    // chunks of a row, wherever its first byte lies
    const int64_t chunks = (a.V + 2 * SmpChunk<T>::N - 2) / SmpChunk<T>::N;
    const int64_t sms = sm_count();
    // Blocks per row: at least what holds it at 8 chunks per thread (64 KB, two
    // blocks per SM) or, beyond eight blocks, more chunks per thread; more blocks
    // while a row more or less would leave SMs idle, down to one chunk per thread.
    int64_t blocks = (chunks + 8 * kSmpThreads - 1) / (8 * kSmpThreads);
    const int64_t most = (chunks + kSmpThreads - 1) / kSmpThreads;
    while (blocks < most && blocks < kSmpBlocks && rows * (blocks + 1) <= 2 * sms) ++blocks;
    if (blocks > kSmpBlocks) blocks = kSmpBlocks;
    a.steps = (int)((chunks + blocks * kSmpThreads - 1) / (blocks * kSmpThreads));
    const size_t smem = (size_t)a.steps * kSmpThreads * 16 + sizeof(SampleShared);
    static std::atomic<bool> done[64];  // false at first
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
