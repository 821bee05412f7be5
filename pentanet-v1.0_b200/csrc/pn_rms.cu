// pn_rms.cu -- root-mean-square norm with the residual's addition, the output
// in the input type of the next projection.
//
// h = T(x + r) (the residual stream, rounded to its own type T and written
// out), rstd = float(1 / sqrt(mean(h^2) + eps)), y = (h * rstd) * w in fp32
// with one rounding per product.  Output: y as bf16 or fp32, or quantised per
// row as quantize_activations_i8 does (s = max|y| / 127, 1 for an all-zero
// row; q = rint(y / s), IEEE division, ties to even) with the row sum that the
// int8 product needs.
//
// The sum of squares runs in fp64.  A sum in fp32 would leave rstd a few ulp
// from the correctly rounded value, depending on the order of the additions,
// and with it move values across the quantiser's rounding borders; in fp64
// every order rounds to the same rstd (but for one row in about 2^25), so the
// codes are those of the formula.
//
// A row holding an inf or NaN gives s = NaN (codes 0), so that the product
// after it shows the fault instead of hiding it behind finite codes.
#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

struct RmsArgs {
    const void* x;
    const void* r;        // residual, or null
    const void* w;        // weight, or null
    int w_f32;
    double eps, inv_c;    // inv_c = 1 / C
    int64_t M, C;
    void* h;              // x + r (not null when r is given)
    void* y;              // bf16 / fp32 output, or null
    int y_f32;
    int8_t* xq;           // int8 output, or null
    int64_t pitch;
    float* s_x;
    int32_t* rowsum;
};

// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// float(1 / sqrt(v)).  In fp32's comfortable range from rsqrtf by two Newton
// steps (relative error e -> 1.5 e^2: 2^-22, 2^-43, below 2^-52): nine fp64
// operations where the library's root and division take over a hundred.
__device__ __forceinline__ float rms_rstd(double v) {
    if (!(v > 1e-30 && v < 1e30)) return (float)(1.0 / sqrt(v));
    double r = (double)rsqrtf((float)v);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = fma(0.5 * r, fma(-(v * r), r, 1.0), r);
    return (float)r;
}

// s and whether the row can be quantised (s finite).
__device__ __forceinline__ float rms_scale(float amax) {
    const float s = __fdiv_rn(amax, 127.0f);
    return s == 0.0f ? 1.0f : s < INFINITY ? s : __int_as_float(0x7fc00000);
}

template <typename T>
__device__ __forceinline__ float ld_weight(const RmsArgs& a, int64_t c) {
    return !a.w ? 1.0f : a.w_f32 ? static_cast<const float*>(a.w)[c] : __bfloat162float(static_cast<const __nv_bfloat16*>(a.w)[c]);
}

template <typename T>
__device__ __forceinline__ T rms_round(float v);
template <>
__device__ __forceinline__ float rms_round<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 rms_round<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

constexpr int kRmsThreads = 256;

// Any width and alignment: one block per row, strided passes over the row (the
// second and third from L1 or L2).  1021 fp32 rows of 1001 to bf16: 6.6 us (the
// bytes alone 0.9 us): two passes, each a chain of reduction and barrier.
template <typename T>
__global__ void __launch_bounds__(kRmsThreads) rms_any_kernel(const RmsArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    __shared__ double red_d[kRmsThreads / 32];
    __shared__ float red_f[kRmsThreads / 32];
    __shared__ int red_i[kRmsThreads / 32];
    const int64_t m = blockIdx.x;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + m * a.C;
    const T* src = x;
    double sum = 0.0;
    if (a.r) {
        const T* r = static_cast<const T*>(a.r) + m * a.C;
        T* h = static_cast<T*>(a.h) + m * a.C;
        for (int64_t c = tid; c < a.C; c += kRmsThreads) {
            const T v = rms_round<T>(ld_elem(x, c) + ld_elem(r, c));
            h[c] = v;  // each thread reads back only what it wrote
            const double d = (double)(float)v;
            sum = fma(d, d, sum);
        }
        src = h;
    } else {
        for (int64_t c = tid; c < a.C; c += kRmsThreads) {
            const double d = (double)ld_elem(x, c);
            sum = fma(d, d, sum);
        }
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((tid & 31) == 0) red_d[tid >> 5] = sum;
    __syncthreads();
    sum = red_d[0];
#pragma unroll
    for (int i = 1; i < kRmsThreads / 32; ++i) sum += red_d[i];
    const float rstd = rms_rstd(fma(sum, a.inv_c, a.eps));
    auto value = [&](int64_t c) { return __fmul_rn(__fmul_rn(ld_elem(src, c), rstd), ld_weight<T>(a, c)); };
    if (!a.xq) {
        for (int64_t c = tid; c < a.C; c += kRmsThreads) {
            if (a.y_f32)
                static_cast<float*>(a.y)[m * a.C + c] = value(c);
            else
                static_cast<__nv_bfloat16*>(a.y)[m * a.C + c] = __float2bfloat16_rn(value(c));
        }
        return;
    }
    float amax = 0.0f;
    for (int64_t c = tid; c < a.C; c += kRmsThreads) amax = max_nan(amax, fabsf(value(c)));
    for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((tid & 31) == 0) red_f[tid >> 5] = amax;
    __syncthreads();
    amax = red_f[0];
#pragma unroll
    for (int i = 1; i < kRmsThreads / 32; ++i) amax = max_nan(amax, red_f[i]);
    const float s = rms_scale(amax);
    int8_t* q = a.xq + m * a.pitch;
    int total = 0;
    for (int64_t c = tid; c < a.pitch; c += kRmsThreads) {
        int v = 0;
        if (c < a.C && s == s) v = (int)fminf(fmaxf(rintf(__fdiv_rn(value(c), s)), -128.0f), 127.0f);
        q[c] = (int8_t)v;
        total += v;
    }
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if ((tid & 31) == 0) red_i[tid >> 5] = total;
    __syncthreads();
    if (tid == 0) {
        total = 0;
        for (int i = 0; i < kRmsThreads / 32; ++i) total += red_i[i];
        a.rowsum[m] = total;
        a.s_x[m] = s;
    }
}

// Rows of C % 8 == 0 elements on 16-byte boundaries, held in registers in their
// own type: TPT threads per row, PC pieces of eight elements each, one read of x
// and of the residual.
//
// What bounds it: the bytes of wide batches, and close behind the instructions (a
// wide int8 row moves 7 bytes per element; an SM has issue slots for about 40
// instructions per element in that time), so the passes over the registers are kept
// to about 20: the quantiser checks eight elements at once for a quotient next to a
// rounding border, packs bytes with PRMT and sums them with DP4A.  4096 bf16 rows of
// 8192 with a residual to int8: 45.6 us, 5.2 TB/s (35.9 us at the copy's rate;
// two pieces per thread 59.6 us).  Few rows are latency: one of 768 takes 2.2 us, most
// of it the launch.
__device__ __forceinline__ void ld_weight8(const RmsArgs& a, int c, float (&w)[8]) {
    if (!a.w) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 1.0f;
    } else if (a.w_f32) {
        Vec8<float>::load(static_cast<const float*>(a.w) + c, w);
    } else {
        Vec8<__nv_bfloat16>::load(static_cast<const __nv_bfloat16*>(a.w) + c, w);
    }
}

__device__ __forceinline__ uint4 pack8_bf16(const float (&v)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
        u[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// Two fp32 operations in one instruction, each rounded as the single one.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// Eight elements as they lie in memory.
template <typename T>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
    uint4 u;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = u; }
    __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) { u = pack8_bf16(v); }
};
template <>
struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ void store(float* p) const {
        reinterpret_cast<float4*>(p)[0] = a;
        reinterpret_cast<float4*>(p)[1] = b;
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        a = make_float4(v[0], v[1], v[2], v[3]);
        b = make_float4(v[4], v[5], v[6], v[7]);
    }
};

// quant1 of eight finite values with |v / s| <= 127 (their row's own scale), as
// eight bytes; their sum is added to total.  t = v / s + 1.5 * 2^23 rounds to the
// nearest integer; v * (1/s) is within 2 ulp of v / s, so only a value within
// 2^-14 of a half-integer can round otherwise: then all eight take the division
// (as they do where s is so small that 1/s, or s itself, is inexact).
__device__ __forceinline__ uint2 quant8(const float (&v)[8], float s, float rs, int& total) {
    uint32_t t[8];
    float far = 0.0f;
    const float2 rs2 = make_float2(rs, rs), up = make_float2(kRoundMagic, kRoundMagic),
                 down = make_float2(-kRoundMagic, -kRoundMagic), neg = make_float2(-rs, -rs);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float2 u = make_float2(v[j], v[j + 1]), m = fma2(u, rs2, up);
        const float2 d = fma2(u, neg, add2(m, down));  // the integer - v / s
        far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
        t[j] = __float_as_uint(m.x), t[j + 1] = __float_as_uint(m.y);
    }
    if (far > 0.5f - 0x1p-14f || s < 0x1p-100f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(v[j], s)), -128.0f), 127.0f);
    }
    uint2 b;
    b.x = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
    b.y = __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410);
    total = __dp4a((int)b.x, 0x01010101, total);
    total = __dp4a((int)b.y, 0x01010101, total);
    return b;
}

// Reduces over the TPT threads of a row: within warps by shuffles, across them
// through `red` (one entry per warp of the block).
template <int TPT, typename V, typename F>
__device__ __forceinline__ V rms_reduce(V v, V* red, F&& op) {
    constexpr int kWarps = TPT / 32;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (kWarps > 1) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) red[warp] = v;
        __syncthreads();
        v = red[warp / kWarps * kWarps + lane % kWarps];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}

template <typename T, int TPT, int PC, bool I8>
__global__ void __launch_bounds__(TPT < 256 ? 256 : TPT, TPT <= 256 ? 4 : TPT == 512 ? 2 : 1)
    rms_vec_kernel(const RmsArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    constexpr int kBlock = TPT < 256 ? 256 : TPT, kRows = kBlock / TPT;
    __shared__ double red_d[kBlock / 32];
    __shared__ float red_f[kBlock / 32];
    __shared__ int red_i[kBlock / 32];
    const int t = threadIdx.x % TPT;
    const int64_t m = (int64_t)blockIdx.x * kRows + threadIdx.x / TPT;
    const bool live = m < a.M;
    const int pieces = live ? (int)(a.C / 8) : 0;
    const T* x = static_cast<const T*>(a.x) + m * a.C;
    Raw8<T> h[PC];
#pragma unroll
    for (int i = 0; i < PC; ++i) {
        const int c = t + i * TPT;
        if (c < pieces)
            h[i].load(x + c * 8);
        else
            h[i].zero();
    }
    // one piece per thread: its weights come along with the row
    float w1[8];
    if constexpr (PC == 1)
        if (t < pieces) ld_weight8(a, t * 8, w1);
    double sum = 0.0;
    Raw8<T> r[PC];
    if (a.r) {
        const T* rp = static_cast<const T*>(a.r) + m * a.C;
#pragma unroll
        for (int i = 0; i < PC; ++i)
            if (t + i * TPT < pieces) r[i].load(rp + (t + i * TPT) * 8);
    }
#pragma unroll
    for (int i = 0; i < PC; ++i) {
        const int c = t + i * TPT;
        float v[8];
        if (a.r && c < pieces) {
            float u[8];
            h[i].get(v);
            r[i].get(u);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += u[j];
            h[i].set(v);
            h[i].store(static_cast<T*>(a.h) + m * a.C + c * 8);
        }
        h[i].get(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double d = (double)v[j];
            sum = fma(d, d, sum);
        }
    }
    sum = rms_reduce<TPT>(sum, red_d, [](double p, double q) { return p + q; });
    const float rstd = rms_rstd(fma(sum, a.inv_c, a.eps));
    auto values = [&](int i, float (&v)[8]) {
        float w[8];
        if constexpr (PC == 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = w1[j];
        } else {
            ld_weight8(a, (t + i * TPT) * 8, w);
        }
        h[i].get(v);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float2 y = mul2(mul2(make_float2(v[j], v[j + 1]), make_float2(rstd, rstd)), make_float2(w[j], w[j + 1]));
            v[j] = y.x, v[j + 1] = y.y;
        }
    };
    if constexpr (!I8) {
#pragma unroll
        for (int i = 0; i < PC; ++i) {
            const int c = t + i * TPT;
            if (c >= pieces) continue;
            float v[8];
            values(i, v);
            if (a.y_f32) {
                Raw8<float> o;
                o.set(v);
                o.store(static_cast<float*>(a.y) + m * a.C + c * 8);
            } else {
                Raw8<__nv_bfloat16> o;
                o.set(v);
                o.store(static_cast<__nv_bfloat16*>(a.y) + m * a.C + c * 8);
            }
        }
    } else {
        float amax = 0.0f;
        float y[PC][8];
#pragma unroll
        for (int i = 0; i < PC; ++i)
            if (t + i * TPT < pieces) {
                values(i, y[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(y[i][j]));
            }
        amax = rms_reduce<TPT>(amax, red_f, [](float p, float q) { return max_nan(p, q); });
        const float s = rms_scale(amax);
        const bool fine = s == s;
        const float rs = __frcp_rn(s);
        const int out_pieces = live ? (int)(a.pitch / 8) : 0;
        int8_t* q = a.xq + m * a.pitch;
        int total = 0;
#pragma unroll
        for (int i = 0; i < PC; ++i) {
            const int c = t + i * TPT;
            if (c >= out_pieces) continue;
            uint2 b = make_uint2(0, 0);
            if (c < pieces && fine) b = quant8(y[i], s, rs, total);
            *reinterpret_cast<uint2*>(q + c * 8) = b;
        }
        total = rms_reduce<TPT>(total, red_i, [](int p, int q) { return p + q; });
        if (live && t == 0) {
            a.rowsum[m] = total;
            a.s_x[m] = s;
        }
    }
}

template <typename T, int TPT, int PC, bool I8>
static void go_rms(const RmsArgs& a, cudaStream_t s) {
    constexpr int kBlock = TPT < 256 ? 256 : TPT, kRows = kBlock / TPT;
    rms_vec_kernel<T, TPT, PC, I8><<<(unsigned)((a.M + kRows - 1) / kRows), kBlock, 0, s>>>(a);
}

template <typename T, int PC, bool I8>
static void go_rms_tpt(int tpt, const RmsArgs& a, cudaStream_t s) {
    switch (tpt) {
        case 32: go_rms<T, 32, PC, I8>(a, s); break;
        case 64: go_rms<T, 64, PC, I8>(a, s); break;
        case 128: go_rms<T, 128, PC, I8>(a, s); break;
        case 256: go_rms<T, 256, PC, I8>(a, s); break;
        case 512: go_rms<T, 512, PC, I8>(a, s); break;
        default: go_rms<T, 1024, PC, I8>(a, s); break;
    }
}

template <typename T, bool I8>
static cudaError_t launch_rms_t(const RmsArgs& a, cudaStream_t s) {
    auto a16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) % 16) == 0; };
    const bool vec = a.C % 8 == 0 && a16(a.x) && a16(a.r) && a16(a.h) && a16(a.w) && a16(a.y);
    const int64_t pieces = I8 ? a.pitch / 8 : a.C / 8;
    // Few rows: a piece per thread, for latency.  Many: 64 bytes per thread
    // (fewer threads to reduce over, as many loads in flight).
    constexpr int kMany = sizeof(T) == 2 ? 4 : 2;
    const int64_t sms = sm_count();
    int pc = a.M <= 2 * sms ? 1 : kMany;
    if (pieces > 1024 * pc) pc = kMany;
    int tpt = 32;
    while (tpt < 1024 && (int64_t)tpt * pc < pieces) tpt *= 2;
    if (!vec || (int64_t)tpt * pc < pieces) {
        rms_any_kernel<T><<<(unsigned)a.M, kRmsThreads, 0, s>>>(a);
    } else if (pc == 1) {
        go_rms_tpt<T, 1, I8>(tpt, a, s);
    } else {
        go_rms_tpt<T, kMany, I8>(tpt, a, s);
    }
    return cudaGetLastError();
}

static cudaError_t launch_rms(const RmsArgs& a, int x_dtype, cudaStream_t s) {
    if (a.M == 0) return cudaSuccess;
    if (x_dtype == PN_F32) return a.xq ? launch_rms_t<float, true>(a, s) : launch_rms_t<float, false>(a, s);
    return a.xq ? launch_rms_t<__nv_bfloat16, true>(a, s) : launch_rms_t<__nv_bfloat16, false>(a, s);
}

}  // namespace pn

static int check_rms(const char* name, const void* x, int x_dtype, const void* residual, const void* weight, int w_dtype,
                     double eps, int64_t M, int64_t C, const void* h) {
    if (x_dtype != PN_F32 && x_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "%s: x dtype %d", name, x_dtype);
    if (weight && w_dtype != PN_F32 && w_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "%s: weight dtype %d", name, w_dtype);
    if (M < 0 || C < 1 || M > 0x7fffffff || C > 0x7fffffff)
        return fail(PN_ERR_SHAPE, "%s: M=%lld C=%lld", name, (long long)M, (long long)C);
    if (!(eps >= 0.0)) return fail(PN_ERR_ARG, "%s: eps must not be negative", name);
    if (M > 0 && !x) return fail(PN_ERR_ARG, "%s: null pointer", name);
    if ((residual != nullptr) != (h != nullptr)) return fail(PN_ERR_ARG, "%s: residual and h go together", name);
    const size_t e = x_dtype == PN_F32 ? 4 : 2;
    if (!aligned(x, e) || !aligned(residual, e) || !aligned(h, e) || !aligned(weight, w_dtype == PN_F32 ? 4 : 2))
        return fail(PN_ERR_ALIGN, "%s: misaligned pointer", name);
    return PN_OK;
}

extern "C" {

int pn_rms_norm(const void* x, int x_dtype, const void* residual, int64_t M, int64_t C, const void* weight, int w_dtype,
                double eps, void* h, void* y, int y_dtype, void* stream) {
    if (int st = check_rms("pn_rms_norm", x, x_dtype, residual, weight, w_dtype, eps, M, C, h)) return st;
    if (y_dtype != PN_F32 && y_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "pn_rms_norm: y dtype %d", y_dtype);
    if (M > 0 && !y) return fail(PN_ERR_ARG, "pn_rms_norm: null pointer");
    if (!aligned(y, y_dtype == PN_F32 ? 4 : 2)) return fail(PN_ERR_ALIGN, "pn_rms_norm: misaligned pointer");
    if (int st = check_device()) return st;
    const pn::RmsArgs a = {x, residual, weight, w_dtype == PN_F32, eps, 1.0 / (double)C, M, C, h, y, y_dtype == PN_F32, nullptr, 0, nullptr,
                           nullptr};
    const cudaError_t e = pn::launch_rms(a, x_dtype, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "pn_rms_norm");
}

int pn_rms_norm_i8(const void* x, int x_dtype, const void* residual, int64_t M, int64_t C, const void* weight,
                   int w_dtype, double eps, void* h, int8_t* xq, int64_t xq_pitch, float* s_x, int32_t* rowsum,
                   void* stream) {
    if (int st = check_rms("pn_rms_norm_i8", x, x_dtype, residual, weight, w_dtype, eps, M, C, h)) return st;
    if (xq_pitch < C || xq_pitch % 16 != 0)
        return fail(PN_ERR_SHAPE, "pn_rms_norm_i8: pitch=%lld (must be >= C=%lld, a multiple of 16)", (long long)xq_pitch,
                    (long long)C);
    if (M > 0 && (!xq || !s_x || !rowsum)) return fail(PN_ERR_ARG, "pn_rms_norm_i8: null pointer");
    if (!aligned(xq, 16) || !aligned(s_x, 4) || !aligned(rowsum, 4))
        return fail(PN_ERR_ALIGN, "pn_rms_norm_i8: misaligned pointer");
    if (int st = check_device()) return st;
    const pn::RmsArgs a = {x, residual, weight, w_dtype == PN_F32, eps, 1.0 / (double)C, M, C, h, nullptr, 0, xq, xq_pitch, s_x, rowsum};
    const cudaError_t e = pn::launch_rms(a, x_dtype, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "pn_rms_norm_i8");
}

int pn_dequant_act_i8(const int8_t* xq, int64_t xq_pitch, const float* s_x, int64_t M, int64_t K, void* y, int y_dtype,
                      void* stream) {
    if (M > 0 && (!xq || !s_x || !y)) return fail(PN_ERR_ARG, "pn_dequant_act_i8: null pointer");
    if (y_dtype != PN_F32 && y_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "pn_dequant_act_i8: dtype %d", y_dtype);
    if (M < 0 || K < 1 || xq_pitch < K || xq_pitch % 16 != 0 || K > 0x7fffffff || (double)M * (K / 16 + 1) > 5e11)
        return fail(PN_ERR_SHAPE, "pn_dequant_act_i8: M=%lld K=%lld pitch=%lld (pitch must be >= K, multiple of 16)",
                    (long long)M, (long long)K, (long long)xq_pitch);
    if (!aligned(xq, 16) || !aligned(s_x, 4) || !aligned(y, y_dtype == PN_F32 ? 4 : 2))
        return fail(PN_ERR_ALIGN, "pn_dequant_act_i8: misaligned pointer");
    if (int st = check_device()) return st;
    const cudaError_t e = pn::launch_dequant_act_i8(xq, xq_pitch, s_x, M, K, y, y_dtype, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "pn_dequant_act_i8");
}

}  // extern "C"
