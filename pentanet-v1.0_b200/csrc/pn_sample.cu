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
// No sort: the k-th largest logit and the border of top-p are found by a
// histogram over 2048 buckets of (max - x) / T, 64 to a unit (beyond 32 units
// a weight is zero), and then among the logits of one bucket by bisection on
// their ordered bit patterns.
#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

struct SampleArgs {
    const void* x;
    int64_t ld;   // elements between rows
    int64_t V;
    const float* u;
    const float* t;      // per row, or null: t0
    const int32_t* k;
    const float* p;
    const float* m;
    float t0, p0, m0;
    int32_t k0;
    int64_t* out;
};

constexpr int kSmpThreads = 1024;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kSmpBuckets = 2048;
constexpr int kSmpList = 4096;
constexpr int64_t kSmpMaxVocab = 1 << 18;
constexpr double kSmpOne = 35184372088832.0;  // 2^45

struct SampleShared {
    uint32_t cnt[kSmpBuckets];
    uint32_t lo[kSmpBuckets], hi[kSmpBuckets];  // 64-bit sums in two halves (shared memory adds 32 bits natively)
    float list[kSmpList];
    uint64_t red[kSmpWarps];
    uint32_t redc[kSmpWarps];
    float redf[kSmpWarps];
    uint64_t sum;
    uint64_t before;
    uint32_t bucket;
    uint32_t n;
    int token;
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
    v = threadIdx.x % 32 < kSmpWarps ? s.red[threadIdx.x & 31] : 0;
    return warp_sum_u64(v);
}

// One row's rule.  An element is kept when it lies above `key`, or equals it
// and is among the first `ties` such in index order, and its weight is at
// least `floor`.
struct SampleRow {
    float max;
    double inv_t;   // 1 / T
    float per;      // buckets per unit of max - x
    uint64_t floor; // min-p as a weight (at least 1)
    float key;
    uint32_t ties;

    __device__ __forceinline__ int bucket(float x) const {  // monotone; kSmpBuckets: no weight
        return x == max ? 0 : (int)fminf((max - x) * per, (float)kSmpBuckets);
    }
    __device__ __forceinline__ uint64_t weight(float x) const {
        if (x == max) return (uint64_t)kSmpOne;
        const uint64_t w = (uint64_t)__double2ull_rn(exp(((double)x - (double)max) * inv_t) * kSmpOne);
        return w >= floor ? w : 0;
    }
};

template <typename T>
__device__ __forceinline__ float smp_ld(const T* x, int64_t i) {
    const float v = ld_elem(x, i);
    return v == v ? v : -INFINITY;  // a NaN is never drawn
}

// The bucket in which the running sum over buckets reaches `need` (first with
// inclusive sum >= need), and the sum before it.  All buckets together hold at
// least `need`.
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

template <typename T>
__global__ void __launch_bounds__(kSmpThreads) sample_kernel(const SampleArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    const int V = (int)a.V;
    const float temp = a.t ? a.t[row] : a.t0, top_p = a.p ? a.p[row] : a.p0, min_p = a.m ? a.m[row] : a.m0;
    int k = a.k ? a.k[row] : a.k0;

    // ---- the largest logit
    float mx = -INFINITY;
    for (int i = tid; i < V; i += kSmpThreads) mx = fmaxf(mx, smp_ld(x, i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) s.redf[warp] = mx;
    __syncthreads();
    mx = s.redf[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (mx == -INFINITY) {  // nothing to draw from
        if (tid == 0) a.out[row] = -1;
        return;
    }
    SampleRow r;
    r.max = mx;
    // T <= 0 (and NaN) takes the first largest logit
    const bool greedy = !(temp > 0.0f);
    r.inv_t = greedy ? (double)INFINITY : 1.0 / (double)temp;
    r.per = greedy ? INFINITY : 64.0f / temp;
    r.floor = min_p > 0.0f ? max((uint64_t)__double2ull_ru(fmin((double)min_p, 1.0) * kSmpOne), (uint64_t)1) : 1;
    r.key = -INFINITY;
    r.ties = 0;
    if (greedy) k = 1;

    // Of one bucket's logits, by bisection: the smallest key v for which
    // sum over x > v of value(x) < need, with that sum in s.sum.
    auto select = [&](int bucket, uint64_t need, auto&& value) {
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        for (int i = tid; i < V; i += kSmpThreads) {
            const float v = smp_ld(x, i);
            if (r.bucket(v) == bucket && value(v) != 0) {
                const uint32_t at = atomicAdd(&s.n, 1);
                if (at < kSmpList) s.list[at] = v;
            }
        }
        __syncthreads();
        const int n = (int)s.n;
        uint32_t lo = order_bits(r.key), hi = order_bits(r.max);  // the answer is in [lo, hi]
        uint64_t above = 0;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            uint64_t sum = 0;
            if (n <= kSmpList) {
                for (int i = tid; i < n; i += kSmpThreads)
                    if (order_bits(s.list[i]) > mid) sum += value(s.list[i]);
            } else {
                for (int i = tid; i < V; i += kSmpThreads) {
                    const float v = smp_ld(x, i);
                    if (r.bucket(v) == bucket && order_bits(v) > mid) sum += value(v);
                }
            }
            sum = block_sum(s, sum);
            if (sum < need) {
                hi = mid;
                above = sum;
            } else {
                lo = mid + 1;
            }
        }
        __syncthreads();
        if (tid == 0) s.sum = above;
        __syncthreads();
        return from_order(lo);
    };

    // ---- top-k: by count
    if (k > 0 && k < V) {
        for (int i = tid; i < kSmpBuckets; i += kSmpThreads) s.cnt[i] = 0;
        __syncthreads();
        uint32_t mine = 0;
        for (int i = tid; i < V; i += kSmpThreads) {
            const float v = smp_ld(x, i);
            const int b = r.bucket(v);
            if (b < kSmpBuckets) {
                atomicAdd(&s.cnt[b], 1u);
                ++mine;
            }
        }
        const uint64_t have = block_sum(s, mine);
        if (have > (uint64_t)k) {
            find_bucket(s, [&](int b) { return (uint64_t)s.cnt[b]; }, (uint64_t)k);
            const int bk = (int)s.bucket;
            const uint64_t before = s.before;
            r.key = select(bk, (uint64_t)k - before, [](float) { return (uint64_t)1; });
            r.ties = (uint32_t)((uint64_t)k - before - s.sum);
        }
    }

    // ---- top-p: by weight, over what is left
    if (top_p < 1.0f && !greedy) {
        const float kkey = r.key;
        const uint32_t kties = r.ties;
        for (int i = tid; i < kSmpBuckets; i += kSmpThreads) s.lo[i] = s.hi[i] = 0;
        __syncthreads();
        uint64_t mine = 0;
        auto add = [&](int b, uint64_t w) {
            const uint32_t old = atomicAdd(&s.lo[b], (uint32_t)w);
            const uint32_t carry = old + (uint32_t)w < old ? 1 : 0;
            const uint32_t h = (uint32_t)(w >> 32) + carry;
            if (h) atomicAdd(&s.hi[b], h);
        };
        for (int i = tid; i < V; i += kSmpThreads) {
            const float v = smp_ld(x, i);
            const int b = r.bucket(v);
            if (b < kSmpBuckets && v > kkey) {
                const uint64_t w = r.weight(v);
                if (w) {
                    add(b, w);
                    mine += w;
                }
            }
        }
        if (tid == 0 && kties > 0) {
            const uint64_t w = r.weight(kkey) * kties;
            if (w) add(r.bucket(kkey), w);
            mine += w;
        }
        const uint64_t total = block_sum(s, mine);
        // kept while the sum before an element is < top_p * total: need = ceil(top_p * total), at least 1
        const uint64_t need = max((uint64_t)ceil(fmax((double)top_p, 0.0) * (double)total), (uint64_t)1);
        if (need < total) {
            find_bucket(s, [&](int b) { return (uint64_t)s.hi[b] << 32 | s.lo[b]; }, need);
            const int bp = (int)s.bucket;
            const uint64_t before = s.before;
            const float key = select(bp, need - before, [&](float v) { return v > kkey ? r.weight(v) : (uint64_t)0; });
            // `select` sees what lies above the top-k border; the border's own ties come last
            const uint64_t left = need - before - s.sum;
            const uint64_t w = r.weight(key);
            r.key = key;
            r.ties = w ? (uint32_t)min((left + w - 1) / w, (uint64_t)0xffffffffu) : 0;
            if (key == kkey) r.ties = min(r.ties, kties);
        }
    }

    // ---- draw.  Every warp owns a run of the row, 32 elements a step.
    const int steps = (V + 32 * kSmpWarps - 1) / (32 * kSmpWarps);
    const int begin = warp * steps * 32;
    uint64_t sum = 0;
    uint32_t ties = 0;
    for (int j = 0; j < steps; ++j) {
        const int i = begin + j * 32 + lane;
        const float v = i < V ? smp_ld(x, i) : -INFINITY;
        if (v > r.key && r.bucket(v) < kSmpBuckets) sum += r.weight(v);
        if (r.ties && v == r.key) ++ties;
    }
    sum = warp_sum_u64(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) s.redc[warp] = ties;
    __syncthreads();
    const uint64_t wk = r.ties ? r.weight(r.key) : 0;
    uint32_t before_ties = 0;
    for (int i = 0; i < warp; ++i) before_ties += s.redc[i];
    const uint32_t quota = r.ties > before_ties ? min(r.ties - before_ties, ties) : 0;  // this warp's kept ties
    sum += quota * wk;
    __syncthreads();
    if (lane == 0) s.red[warp] = sum;
    if (tid == 0) s.token = -1;
    __syncthreads();
    uint64_t total = 0, before = 0;
    for (int i = 0; i < kSmpWarps; ++i) {
        if (i < warp) before += s.red[i];
        total += s.red[i];
    }
    const double ud = fmin(fmax((double)a.u[row], 0.0), 1.0);
    // first index whose running sum exceeds u * total; u = 1 takes the last kept one
    const uint64_t target = min((uint64_t)(ud * (double)total), total - 1);
    if (target >= before && target < before + sum) {
        uint32_t left = quota;
        uint64_t at = before;
        for (int j = 0; j < steps; ++j) {
            const int i = begin + j * 32 + lane;
            const float v = i < V ? smp_ld(x, i) : -INFINITY;
            uint64_t w = v > r.key && r.bucket(v) < kSmpBuckets ? r.weight(v) : 0;
            const uint32_t eq = __ballot_sync(0xffffffffu, r.ties && v == r.key);
            if (eq) {
                if ((eq >> lane & 1u) && (uint32_t)__popc(eq & ((1u << lane) - 1u)) < left) w = wk;
                left -= min(left, (uint32_t)__popc(eq));
            }
            if (!__any_sync(0xffffffffu, w != 0)) continue;
            uint64_t inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t n = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += n;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, at + inc > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) a.out[row] = i;
                break;
            }
            at += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
}

template <typename T>
static cudaError_t launch_sample(const SampleArgs& a, int64_t rows, cudaStream_t s) {
    const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)sizeof(SampleShared));
    if (e != cudaSuccess) return e;
    sample_kernel<T><<<(unsigned)rows, kSmpThreads, sizeof(SampleShared), s>>>(a);
    return cudaGetLastError();
}

}  // namespace pn

extern "C" int pn_sample_tokens(const void* logits, int x_dtype, int64_t rows, int64_t vocab, int64_t ld, const float* u,
                                const float* temperature, float temperature0, const int32_t* top_k, int32_t top_k0,
                                const float* top_p, float top_p0, const float* min_p, float min_p0, int64_t* tokens,
                                void* stream) {
    if (x_dtype != PN_F32 && x_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "pn_sample_tokens: dtype %d", x_dtype);
    if (rows < 0 || rows > 0x7fffffff || vocab < 1 || vocab > pn::kSmpMaxVocab || ld < vocab)
        return fail(PN_ERR_SHAPE, "pn_sample_tokens: rows=%lld vocab=%lld (at most %lld) ld=%lld", (long long)rows,
                    (long long)vocab, (long long)pn::kSmpMaxVocab, (long long)ld);
    if (rows > 0 && (!logits || !u || !tokens)) return fail(PN_ERR_ARG, "pn_sample_tokens: null pointer");
    if (!aligned(logits, x_dtype == PN_F32 ? 4 : 2) || !aligned(u, 4) || !aligned(temperature, 4) || !aligned(top_k, 4) ||
        !aligned(top_p, 4) || !aligned(min_p, 4) || !aligned(tokens, 8))
        return fail(PN_ERR_ALIGN, "pn_sample_tokens: misaligned pointer");
    if (int st = check_device()) return st;
    if (rows == 0) return ok();
    const pn::SampleArgs a = {logits, ld, vocab, u, temperature, top_k, top_p, min_p, temperature0, top_p0, min_p0, top_k0,
                              tokens};
    const cudaError_t e = x_dtype == PN_F32 ? pn::launch_sample<float>(a, rows, (cudaStream_t)stream)
                                            : pn::launch_sample<__nv_bfloat16>(a, rows, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "pn_sample_tokens");
}
