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
    double eps;
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

__device__ __forceinline__ float rms_rstd(double sum, int64_t C, double eps) {
    return (float)(1.0 / sqrt(sum / (double)C + eps));
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

// Any width and alignment: one block per row, strided passes over the row.
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
    const float rstd = rms_rstd(sum, a.C, a.eps);
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
        if (c < a.C && s == s) v = (int)rintf(__fdiv_rn(value(c), s));
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

static cudaError_t launch_rms(const RmsArgs& a, int x_dtype, cudaStream_t s) {
    if (a.M == 0) return cudaSuccess;
    if (x_dtype == PN_F32)
        rms_any_kernel<float><<<(unsigned)a.M, kRmsThreads, 0, s>>>(a);
    else
        rms_any_kernel<__nv_bfloat16><<<(unsigned)a.M, kRmsThreads, 0, s>>>(a);
    return cudaGetLastError();
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
    const pn::RmsArgs a = {x, residual, weight, w_dtype == PN_F32, eps, M, C, h, y, y_dtype == PN_F32, nullptr, 0, nullptr,
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
    const pn::RmsArgs a = {x, residual, weight, w_dtype == PN_F32, eps, M, C, h, nullptr, 0, xq, xq_pitch, s_x, rowsum};
    const cudaError_t e = pn::launch_rms(a, x_dtype, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "pn_rms_norm_i8");
}

}  // extern "C"
