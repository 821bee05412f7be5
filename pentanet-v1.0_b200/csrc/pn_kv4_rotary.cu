// pn_kv4_rotary.cu -- rotating positions into queries and keys, and storing keys and
// values in the 4-bit paged cache (layout and quantiser: pn_kv4.cu), in one pass over a
// projection's output.
//
// Mathematics.  A row at position p of its sequence has the angle of entry p + offset of
// the tables.  Of the first R dims of a head, pair (a, b) becomes
//   (a cos - b sin, b cos + a sin),
// each product and sum rounded to fp32 in that order (no fused operation), so that the
// result does not depend on how it is compiled: a code next to a border is the same as
// that of the elementwise operations.  Queries are rounded once, to their type; keys go to the
// quantiser as fp32, which costs them no rounding to bf16.
#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

struct Kv4RotaryArgs {
    Kv4Seq s;
    const void* x[3];                // queries, keys, values
    int64_t sb[3], sl[3], sh[3];     // their strides in elements: sequence, row, head
    int vec;                         // 16-byte loads allowed
    int H;                           // query heads
    const float *cos, *sin;          // (n_pos, ld): one column per pair
    int64_t n_pos, ld;
    int table_vec;
    int rotated, interleaved;
    const int32_t* offsets;          // (B), or null
    void* out;                       // (T, H, D), the inputs' type
    uint8_t* cache;
    int zero_rest;                   // queries of rows of no sequence become zeros
    int parts;                       // warps that share a row
};
constexpr int kRotaryThreads = 128;

// The warp's row: where it lies in the inputs, the cache and the tables.
struct RotaryRow {
    int64_t src[3];
    uint8_t* page;    // null: keys and values are not stored
    int tok;
    int64_t angle;    // -1: the queries become zeros
};

__device__ __forceinline__ bool rotary_row(const Kv4RotaryArgs& a, int64_t row, int64_t block, RotaryRow& r) {
    int64_t b, i, first, n;
    if (!kv4_find(a.s, row, b, i)) return false;
    kv4_rows(a.s, b, first, n);
    const int64_t pos = (int64_t)kv4_len(a.s, b) - n + i;
    r.page = nullptr;
    r.tok = 0;
    r.angle = -1;
    if (pos >= 0) {
        const int64_t angle = pos + (a.offsets ? __ldg(a.offsets + b) : 0);
        if (angle >= 0 && angle < a.n_pos) {
            r.angle = angle;
            const int64_t page = kv4_page(a.s, b, (int)pos);
            if (page >= 0) r.page = a.cache + page * a.s.Hk * 2 * block;
            r.tok = (int)pos % a.s.page;
        } else {
            record_status(PN_ERR_ARG);
        }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) r.src[k] = a.s.cu ? row * a.sl[k] : b * a.sb[k] + i * a.sl[k];
    return true;
}

// Rotates sixteen values: with halves v[0 .. 8) meet v[8 .. 16), else neighbours meet.
__device__ __forceinline__ void rotate16(float (&v)[16], const float (&c)[8], const float (&s)[8], bool interleaved) {
    if (interleaved) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = v[2 * j], y = v[2 * j + 1];
            v[2 * j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
            v[2 * j + 1] = __fadd_rn(__fmul_rn(y, c[j]), __fmul_rn(x, s[j]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = v[j], y = v[j + 8];
            v[j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
            v[j + 8] = __fadd_rn(__fmul_rn(y, c[j]), __fmul_rn(x, s[j]));
        }
    }
}

// Scale and zero of a vector whose lanes hold sixteen values each (VT lanes).
template <int VT>
__device__ __forceinline__ void rotary_scale(const float (&v)[16], float& s, float& z) {
    float lo = v[0], hi = v[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) {
        lo = min_nan(lo, v[j]);
        hi = max_nan(hi, v[j]);
    }
#pragma unroll
    for (int o = VT / 2; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    z = floor_bf16(lo);
    s = ceil_bf16_pos(__fdiv_rn(__fsub_rn(hi, z), 15.0f));
    if (!(s < INFINITY) || !(fabsf(z) < INFINITY)) {  // an inf or NaN in the vector: all of it reads back as NaN
        s = 0.0f;
        z = __int_as_float(0x7fc00000);
    }
}

// D / 16 lanes per vector, two pieces of eight dims each: of rotated halves a lane holds the
// two that meet, so that no value crosses lanes and a lane needs eight angles, which it
// keeps for all heads of its row.  A warp takes a row (or one of `parts` shares of its
// vectors, where there are few rows), no block-wide step anywhere.  Its loads of the next step are in
// flight during this one; six blocks to an SM spill 4 to 32 bytes, but have more of them: 7 ragged prompts of up to 2047
// rows, 32 + 2 x 8 heads of 128 dims: 53 us (five blocks, no spills: 58; eight: 64), reading and writing once 31.
template <typename T, int D>
__global__ void __launch_bounds__(kRotaryThreads, 6) kv4_rotary_kernel(const Kv4RotaryArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int VT = D / 16, VP = 32 / VT;  // lanes per vector, vectors per step
    const int lane = threadIdx.x & 31, l = lane % VT, sub = lane / VT;
    const int64_t unit = (int64_t)blockIdx.x * (kRotaryThreads / 32) + (threadIdx.x >> 5);
    const int64_t row = unit / a.parts;
    const int part = (int)(unit - row * a.parts);
    if (row >= a.s.T) return;
    const int64_t block = (int64_t)a.s.page * (D / 2 + 4);
    RotaryRow r;
    if (!rotary_row(a, row, block, r)) {
        if (!a.zero_rest) return;
        const int64_t n = (int64_t)a.H * D * sizeof(T) / 16, from = n * part / a.parts, to = n * (part + 1) / a.parts;
        for (int64_t i = from + lane; i < to; i += 32) static_cast<uint4*>(a.out)[row * n + i] = make_uint4(0, 0, 0, 0);
        return;
    }

    // the lane's two pieces of eight dims
    const bool turns = l * 16 < a.rotated;
    const bool halves = turns && !a.interleaved;
    const int p0 = halves ? l : 2 * l, p1 = halves ? l + a.rotated / 16 : 2 * l + 1;
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = 1.0f, s[j] = 0.0f;
    if (turns && r.angle >= 0) {
        kv4_load8(a.cos + r.angle * a.ld + l * 8, a.table_vec, c);
        kv4_load8(a.sin + r.angle * a.ld + l * 8, a.table_vec, s);
    }
    // steps: VP query heads each, then key heads, then value heads
    const int nq = (a.H + VP - 1) / VP, nk = (a.s.Hk + VP - 1) / VP, steps = nq + 2 * nk;
    const int from = (int)((int64_t)steps * part / a.parts), to = (int)((int64_t)steps * (part + 1) / a.parts);
    auto load = [&](int step, Raw8<T> (&x)[2]) {
        x[0].zero();
        x[1].zero();
        const int kind = step < nq ? 0 : step < nq + nk ? 1 : 2;
        const int head = (step - (kind == 0 ? 0 : kind == 1 ? nq : nq + nk)) * VP + sub;
        if (step >= to || head >= (kind == 0 ? a.H : a.s.Hk) || (kind == 0 ? r.angle < 0 : !r.page)) return;
        const T* p = static_cast<const T*>(kind == 0 ? a.x[0] : kind == 1 ? a.x[1] : a.x[2]) +
                     (kind == 0 ? r.src[0] : kind == 1 ? r.src[1] : r.src[2]) +
                     head * (kind == 0 ? a.sh[0] : kind == 1 ? a.sh[1] : a.sh[2]);
        const int i0 = kind == 2 ? 2 * l : p0, i1 = kind == 2 ? 2 * l + 1 : p1;
        if (a.vec) {
            x[0].load(p + i0 * 8);
            x[1].load(p + i1 * 8);
        } else {
            float v[8];
            kv4_load8(p + i0 * 8, false, v);
            x[0].set(v);
            kv4_load8(p + i1 * 8, false, v);
            x[1].set(v);
        }
    };
    Raw8<T> x[2];
    load(from, x);
    for (int step = from; step < to; ++step) {
        const Raw8<T> now[2] = {x[0], x[1]};
        load(step + 1, x);
        float v[16];
        {
            float u[8];
            now[0].get(u);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = u[j];
            now[1].get(u);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[8 + j] = u[j];
        }
        if (step < nq + nk && turns) rotate16(v, c, s, a.interleaved);
        float lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] = v[j], hi[j] = v[8 + j];
        if (step < nq) {
            const int head = step * VP + sub;
            if (head < a.H) {
                T* y = static_cast<T*>(a.out) + (row * a.H + head) * D;
                Raw8<T> o;
                o.set(lo);
                o.store(y + p0 * 8);
                o.set(hi);
                o.store(y + p1 * 8);
            }
            continue;
        }
        const bool kv = step >= nq + nk;
        const int head = (step - (kv ? nq + nk : nq)) * VP + sub;
        float sc, z;
        rotary_scale<VT>(v, sc, z);
        if (head >= a.s.Hk || !r.page) continue;
        uint32_t w0 = 0, w1 = 0;
        if (sc > 0.0f) {
            w0 = kv4_codes8(lo, sc, z);
            w1 = kv4_codes8(hi, sc, z);
        }
        uint8_t* blk = r.page + (int64_t)(2 * head + kv) * block;
        if (!kv) {
            uint32_t* p = reinterpret_cast<uint32_t*>(blk + r.tok * (D / 2));
            p[p0] = w0;
            p[p1] = w1;
        } else {
            uint16_t* p = reinterpret_cast<uint16_t*>(blk + (r.tok >> 1) * D + l * 16 + (r.tok & 1) * 2);
            p[0] = (uint16_t)w0, p[2] = (uint16_t)(w0 >> 16);
            p[4] = (uint16_t)w1, p[6] = (uint16_t)(w1 >> 16);
        }
        if (l == 0)
            *reinterpret_cast<uint32_t*>(blk + a.s.page * (D / 2) + r.tok * 4) =
                (__float_as_uint(sc) >> 16) | (__float_as_uint(z) & 0xFFFF0000u);
    }
}

template <typename T, int D>
static cudaError_t launch_rotary(Kv4RotaryArgs& a, cudaStream_t s) {
    constexpr int VP = 32 / (D / 16);
    const int steps = (a.H + VP - 1) / VP + 2 * ((a.s.Hk + VP - 1) / VP);
    // few rows: a warp for each step
    const int64_t warps = (int64_t)sm_count() * 32;
    a.parts = (int)std::min<int64_t>(std::max<int64_t>(warps / a.s.T, 1), steps);
    constexpr int per = kRotaryThreads / 32;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.s.T * a.parts + per - 1) / per));
    cfg.blockDim = dim3(kRotaryThreads);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_rotary_kernel<T, D>, a);
}

}  // namespace pn

extern "C" {

int pn_kv4_append_rotary(const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh, int64_t q_heads, const void* k, int64_t k_sb,
                         int64_t k_sl, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_sl, int64_t v_sh, int dtype,
                         const float* cos, const float* sin, int64_t n_pos, int64_t table_stride, int64_t rotated,
                         int interleaved, const int32_t* offsets, void* cache, int64_t n_pages, int64_t kv_heads, int64_t page,
                         int64_t head_dim, const int32_t* block_table, int64_t table_ld, int64_t table_w,
                         const int32_t* seq_lens, const int32_t* cu_q, int64_t B, int64_t T, void* q_out, int zero_rest,
                         void* stream) {
    const char* name = "pn_kv4_append_rotary";
    pn::Kv4RotaryArgs a{};
    if (int st = check_kv4(name, cache, n_pages, kv_heads, page, head_dim, block_table, table_ld, table_w, seq_lens, cu_q, B, T,
                           &a.s))
        return st;
    if (dtype != PN_F32 && dtype != PN_BF16) return fail(PN_ERR_DTYPE, "%s: dtype %d", name, dtype);
    if (q_heads < 1 || q_heads > 65536) return fail(PN_ERR_SHAPE, "%s: %lld query heads", name, (long long)q_heads);
    if (rotated < 16 || rotated % 16 != 0 || rotated > head_dim)
        return fail(PN_ERR_SHAPE, "%s: %lld dims to rotate (a multiple of 16 up to head_dim)", name, (long long)rotated);
    if (n_pos < 0 || table_stride < rotated / 2)
        return fail(PN_ERR_SHAPE, "%s: tables of %lld positions, %lld apart", name, (long long)n_pos, (long long)table_stride);
    const size_t e = dtype == PN_F32 ? 4 : 2;
    if (T > 0 && B > 0 && (!q || !k || !v || !q_out || ((!cos || !sin) && n_pos > 0)))
        return fail(PN_ERR_ARG, "%s: null pointer", name);
    if (!aligned(q, e) || !aligned(k, e) || !aligned(v, e) || !aligned(cos, 4) || !aligned(sin, 4) || !aligned(offsets, 4) ||
        !aligned(q_out, 16))
        return fail(PN_ERR_ALIGN, "%s: misaligned pointer", name);
    if ((double)T * 64 > 4e9) return fail(PN_ERR_SHAPE, "%s: %lld rows are too much for one call", name, (long long)T);
    if (int st = check_device()) return st;
    if (T == 0 || B == 0) return ok();
    a.x[0] = q, a.sb[0] = q_sb, a.sl[0] = q_sl, a.sh[0] = q_sh;
    a.x[1] = k, a.sb[1] = k_sb, a.sl[1] = k_sl, a.sh[1] = k_sh;
    a.x[2] = v, a.sb[2] = v_sb, a.sl[2] = v_sl, a.sh[2] = v_sh;
    const int64_t n = 16 / (int64_t)e;
    a.vec = 1;
    for (int i = 0; i < 3; ++i)
        a.vec &= aligned(a.x[i], 16) && a.sb[i] % n == 0 && a.sl[i] % n == 0 && a.sh[i] % n == 0;
    a.H = (int)q_heads;
    a.cos = cos, a.sin = sin, a.n_pos = n_pos, a.ld = table_stride;
    a.table_vec = aligned(cos, 16) && aligned(sin, 16) && table_stride % 4 == 0;
    a.rotated = (int)rotated, a.interleaved = interleaved != 0, a.offsets = offsets;
    a.out = q_out;
    a.zero_rest = zero_rest != 0;
    a.cache = static_cast<uint8_t*>(cache);
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t err;
    if (dtype == PN_F32)
        err = head_dim == 64 ? pn::launch_rotary<float, 64>(a, s) : pn::launch_rotary<float, 128>(a, s);
    else
        err = head_dim == 64 ? pn::launch_rotary<__nv_bfloat16, 64>(a, s) : pn::launch_rotary<__nv_bfloat16, 128>(a, s);
    return err == cudaSuccess ? ok() : cuda_fail(err, name);
}

}  // extern "C"
