// pn_kv4.cu -- a paged cache of keys and values held in 4 bits: storing new
// tokens and reading tokens back (attention over it: pn_kv4_attn.cu).
//
// One vector of d values (a token's key or value in one head) is held as
// c = clamp(rint((x - z) / s), 0, 15) with z the vector's minimum rounded down
// to bf16 and s = (max - z) / 15 rounded up to bf16, so that every value lies
// within s / 2 of s * c + z: half a byte per value and four bytes per vector,
// 3.8x (d = 128) or 3.6x (d = 64) below bf16.  One pair per vector keeps the
// codes raw small integers in the attention's matrix products: scale and zero
// are applied to whole sums, not to elements.  bf16 pairs keep the exponent
// range of the activations.
//
// A page block (one page, one kv head, keys or values) is page * d / 2 bytes
// of codes, then page * 4 bytes of (scale, zero) pairs:
//   keys    token-major; word j of a token holds dims 8j .. 8j+7, dim 8j+n in
//           bits 4n..4n+3
//   values  tokens 2i and 2i+1 share a block of d bytes; its word j holds dims
//           4j .. 4j+3 of token 2i in the low half, of token 2i+1 in the high
//           half, dim 4j+n in bits 4n..4n+3 of the half
// A 32-bit word masked with 0x000F000F is thus a pair of matrix operands that
// sit next to each other along the summed axis: two dims of a key, two tokens
// of a value.
#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

// Where the rows of a call live: sequence b's newest rows are its last L_b
// positions (its length includes them).
struct Kv4Seq {
    const int32_t* table;  // (B, table_ld): page of tokens [i * page, (i + 1) * page)
    int64_t table_ld;
    int table_w;           // pages per sequence in the table
    const int32_t* lens;   // (B)
    const int32_t* cu;     // (B + 1) first row of each sequence, or null: L rows each
    int64_t B, T;          // sequences, rows
    int64_t L;
    int64_t n_pages;
    int Hk, page;
};

__device__ __forceinline__ int kv4_len(const Kv4Seq& s, int64_t b) {
    const int64_t cap = (int64_t)s.table_w * s.page;
    return (int)min(max((int64_t)__ldg(s.lens + b), (int64_t)0), cap);
}

// First row and number of rows of sequence b.
__device__ __forceinline__ void kv4_rows(const Kv4Seq& s, int64_t b, int64_t& first, int64_t& n) {
    if (!s.cu) {
        first = b * s.L;
        n = s.L;
        return;
    }
    first = min(max((int64_t)__ldg(s.cu + b), (int64_t)0), s.T);
    n = min(max((int64_t)__ldg(s.cu + b + 1), first), s.T) - first;
}

// The sequence of a row and the row's index there; false behind the last one.
__device__ __forceinline__ bool kv4_find(const Kv4Seq& s, int64_t row, int64_t& b, int64_t& i) {
    if (!s.cu) {
        b = row / s.L;
        i = row - b * s.L;
        return true;
    }
    int64_t lo = 0, hi = s.B;  // the last b with cu[b] <= row
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        if (__ldg(s.cu + mid) <= row)
            lo = mid;
        else
            hi = mid;
    }
    b = lo;
    int64_t first, n;
    kv4_rows(s, b, first, n);
    i = row - first;
    return i >= 0 && i < n;
}

// The page block that holds position pos of sequence b, or -1 (and the device
// status word) when the table's entry is no page of the cache.
__device__ __forceinline__ int64_t kv4_page(const Kv4Seq& s, int64_t b, int pos) {
    const int p = __ldg(s.table + b * s.table_ld + pos / s.page);
    if (p >= 0 && p < s.n_pages) return p;
    record_status(PN_ERR_ARG);
    return -1;
}

__device__ __forceinline__ float floor_bf16(float v) {  // towards -infinity
    const int bits = __float_as_int(v);
    int cut = bits & 0xFFFF0000;
    if (cut != bits && bits < 0) cut += 0x10000;
    return v == v ? __int_as_float(cut) : v;
}
__device__ __forceinline__ float ceil_bf16_pos(float v) {  // v >= 0
    const int bits = __float_as_int(v);
    const int cut = bits & 0xFFFF0000;
    return v == v ? __int_as_float(cut != bits ? cut + 0x10000 : cut) : v;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float m;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

template <typename T>
__device__ __forceinline__ void kv4_load8(const T* p, bool vec, float (&v)[8]) {
    if (vec) {
        Vec8<T>::load(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = ld_elem(p, j);
    }
}

struct Kv4AppendArgs {
    Kv4Seq s;
    const void* x[2];           // keys, values
    int64_t sb[2], sl[2], sh[2];  // their strides in elements: sequence, row, head
    int vec;                    // 16-byte loads allowed
    uint8_t* cache;
};

constexpr int kKv4Threads = 256;

// D / 8 lanes per vector, eight dims each.
template <typename T, int D>
__global__ void __launch_bounds__(kKv4Threads) kv4_append_kernel(const Kv4AppendArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    constexpr int VT = D / 8;
    const int64_t vec = ((int64_t)blockIdx.x * kKv4Threads + threadIdx.x) / VT;
    const int l = threadIdx.x % VT;
    const int kv = (int)(vec & 1);
    const int64_t rh = vec >> 1;
    const int64_t row = rh / a.s.Hk;
    const int head = (int)(rh - row * a.s.Hk);
    int64_t b = 0, i = 0;
    bool live = row < a.s.T && kv4_find(a.s, row, b, i);
    int64_t page = -1;
    int pos = -1;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (live) {
        int64_t first, n;
        kv4_rows(a.s, b, first, n);
        pos = (int)(kv4_len(a.s, b) - n + i);
        if (pos >= 0) page = kv4_page(a.s, b, pos);
        const T* x = static_cast<const T*>(a.x[kv]) + (a.s.cu ? row * a.sl[kv] : b * a.sb[kv] + i * a.sl[kv]) +
                     head * a.sh[kv] + l * 8;
        kv4_load8(x, a.vec, v);
    }
    float lo = v[0], hi = v[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
        lo = min_nan(lo, v[j]);
        hi = max_nan(hi, v[j]);
    }
#pragma unroll
    for (int o = VT / 2; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (page < 0) return;
    float z = floor_bf16(lo);
    float s = ceil_bf16_pos(__fdiv_rn(__fsub_rn(hi, z), 15.0f));
    if (!(s < INFINITY) || !(fabsf(z) < INFINITY)) {  // an inf or NaN in the vector: all of it reads back as NaN
        s = 0.0f;
        z = __int_as_float(0x7fc00000);
    }
    uint32_t w = 0;
    if (s > 0.0f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float q = rintf(__fdiv_rn(__fsub_rn(v[j], z), s));
            w |= (uint32_t)fminf(fmaxf(q, 0.0f), 15.0f) << (4 * j);
        }
    }
    const int tok = pos % a.s.page;
    const int64_t block = (int64_t)a.s.page * (D / 2 + 4);
    uint8_t* blk = a.cache + ((page * a.s.Hk + head) * 2 + kv) * block;
    if (kv == 0) {
        *reinterpret_cast<uint32_t*>(blk + tok * (D / 2) + l * 4) = w;
    } else {
        uint8_t* p = blk + (tok >> 1) * D + l * 8 + (tok & 1) * 2;
        *reinterpret_cast<uint16_t*>(p) = (uint16_t)w;
        *reinterpret_cast<uint16_t*>(p + 4) = (uint16_t)(w >> 16);
    }
    if (l == 0)
        *reinterpret_cast<uint32_t*>(blk + (int64_t)a.s.page * (D / 2) + tok * 4) =
            (__float_as_uint(s) >> 16) | (__float_as_uint(z) & 0xFFFF0000u);
}

struct Kv4GatherArgs {
    Kv4Seq s;
    const uint8_t* cache;
    void* y[2];
    int y_f32;
};

template <int D>
__global__ void __launch_bounds__(kKv4Threads) kv4_gather_kernel(const Kv4GatherArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    constexpr int VT = D / 8;
    const int64_t vec = ((int64_t)blockIdx.x * kKv4Threads + threadIdx.x) / VT;
    const int l = threadIdx.x % VT;
    const int kv = (int)(vec & 1);
    const int64_t rh = vec >> 1;
    const int64_t row = rh / a.s.Hk;
    const int head = (int)(rh - row * a.s.Hk);
    int64_t b, i;
    if (row >= a.s.T || !kv4_find(a.s, row, b, i)) return;
    int64_t first, n;
    kv4_rows(a.s, b, first, n);
    const int pos = (int)(kv4_len(a.s, b) - n + i);
    const int64_t page = pos >= 0 ? kv4_page(a.s, b, pos) : -1;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (page >= 0) {
        const int tok = pos % a.s.page;
        const int64_t block = (int64_t)a.s.page * (D / 2 + 4);
        const uint8_t* blk = a.cache + ((page * a.s.Hk + head) * 2 + kv) * block;
        const uint32_t pair = *reinterpret_cast<const uint32_t*>(blk + (int64_t)a.s.page * (D / 2) + tok * 4);
        uint32_t w;
        if (kv == 0) {
            w = *reinterpret_cast<const uint32_t*>(blk + tok * (D / 2) + l * 4);
        } else {
            const uint8_t* p = blk + (tok >> 1) * D + l * 8 + (tok & 1) * 2;
            w = *reinterpret_cast<const uint16_t*>(p) | (uint32_t) * reinterpret_cast<const uint16_t*>(p + 4) << 16;
        }
        const float s = __uint_as_float(pair << 16), z = __uint_as_float(pair & 0xFFFF0000u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fmaf(s, (float)(w >> (4 * j) & 15u), z);  // s * c is exact: one rounding
    }
    const int64_t at = (row * a.s.Hk + head) * D + l * 8;
    void* out = kv ? a.y[1] : a.y[0];
    if (a.y_f32) {
        float4* y = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
        y[0] = make_float4(v[0], v[1], v[2], v[3]);
        y[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
            u[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + at) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

}  // namespace pn

// The arguments that the cache's entry points share.
static int check_kv4(const char* name, const void* cache, int64_t n_pages, int64_t Hk, int64_t page, int64_t D,
                     const int32_t* table, int64_t table_ld, int64_t table_w, const int32_t* lens, const int32_t* cu,
                     int64_t B, int64_t T, pn::Kv4Seq* s) {
    if (D != 64 && D != 128) return fail(PN_ERR_SHAPE, "%s: head_dim=%lld (64 or 128)", name, (long long)D);
    if (page < 16 || page % 16 != 0 || page > 65536)
        return fail(PN_ERR_SHAPE, "%s: page=%lld (a multiple of 16 up to 65536)", name, (long long)page);
    if (n_pages < 0 || n_pages > 0x7fffffff || Hk < 1 || Hk > 65536 || B < 0 || T < 0 || T > 0x7fffffff || B > 0x7ffffffe)
        return fail(PN_ERR_SHAPE, "%s: pages=%lld kv heads=%lld sequences=%lld rows=%lld", name, (long long)n_pages,
                    (long long)Hk, (long long)B, (long long)T);
    if (table_w < 0 || table_ld < table_w || table_w > (1 << 30) / page)
        return fail(PN_ERR_SHAPE, "%s: block table width=%lld stride=%lld", name, (long long)table_w, (long long)table_ld);  // positions stay below 2^30
    if (!cu && B > 0 && T % B != 0)
        return fail(PN_ERR_SHAPE, "%s: %lld rows over %lld sequences need cu_q", name, (long long)T, (long long)B);
    if (T > 0 && B > 0 && ((!cache && n_pages > 0) || (!table && table_w > 0) || !lens))
        return fail(PN_ERR_ARG, "%s: null pointer", name);
    if (!aligned(cache, 16)) return fail(PN_ERR_ALIGN, "%s: the cache needs 16-byte alignment", name);
    if (!aligned(table, 4) || !aligned(lens, 4) || !aligned(cu, 4)) return fail(PN_ERR_ALIGN, "%s: misaligned pointer", name);
    *s = pn::Kv4Seq{table, table_ld, (int)table_w, lens, cu, B, T, B > 0 ? T / B : 0, n_pages, (int)Hk, (int)page};
    return PN_OK;
}

extern "C" {

int64_t pn_kv4_block_bytes(int64_t page, int64_t head_dim) { return page * (head_dim / 2 + 4); }

int pn_kv4_append(const void* k, int64_t k_sb, int64_t k_sl, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_sl,
                  int64_t v_sh, int kv_dtype, void* cache, int64_t n_pages, int64_t kv_heads, int64_t page,
                  int64_t head_dim, const int32_t* block_table, int64_t table_ld, int64_t table_w,
                  const int32_t* seq_lens, const int32_t* cu_q, int64_t B, int64_t T, void* stream) {
    pn::Kv4AppendArgs a{};
    if (int st = check_kv4("pn_kv4_append", cache, n_pages, kv_heads, page, head_dim, block_table, table_ld, table_w,
                           seq_lens, cu_q, B, T, &a.s))
        return st;
    if (kv_dtype != PN_F32 && kv_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "pn_kv4_append: dtype %d", kv_dtype);
    const size_t e = kv_dtype == PN_F32 ? 4 : 2;
    if (T > 0 && B > 0 && (!k || !v)) return fail(PN_ERR_ARG, "pn_kv4_append: null pointer");
    if (!aligned(k, e) || !aligned(v, e)) return fail(PN_ERR_ALIGN, "pn_kv4_append: misaligned pointer");
    if (int st = check_device()) return st;
    if (T == 0 || B == 0) return ok();
    if (n_pages == 0 || table_w == 0) return ok();  // no room for any token
    a.x[0] = k, a.sb[0] = k_sb, a.sl[0] = k_sl, a.sh[0] = k_sh;
    a.x[1] = v, a.sb[1] = v_sb, a.sl[1] = v_sl, a.sh[1] = v_sh;
    a.cache = static_cast<uint8_t*>(cache);
    auto whole = [&](int i) {  // every row of 8 dims starts on a 16-byte boundary
        const int64_t n = 16 / (int64_t)e;
        return aligned(a.x[i], 16) && a.sb[i] % n == 0 && a.sl[i] % n == 0 && a.sh[i] % n == 0;
    };
    a.vec = whole(0) && whole(1);
    const int64_t blocks = (T * kv_heads * 2 * (head_dim / 8) + pn::kKv4Threads - 1) / pn::kKv4Threads;
    if (blocks > 0x7fffffff) return fail(PN_ERR_SHAPE, "pn_kv4_append: too many rows");
    const unsigned g = (unsigned)blocks;
    const cudaStream_t s = (cudaStream_t)stream;
    if (kv_dtype == PN_F32) {
        if (head_dim == 64) pn::kv4_append_kernel<float, 64><<<g, pn::kKv4Threads, 0, s>>>(a);
        else pn::kv4_append_kernel<float, 128><<<g, pn::kKv4Threads, 0, s>>>(a);
    } else {
        if (head_dim == 64) pn::kv4_append_kernel<__nv_bfloat16, 64><<<g, pn::kKv4Threads, 0, s>>>(a);
        else pn::kv4_append_kernel<__nv_bfloat16, 128><<<g, pn::kKv4Threads, 0, s>>>(a);
    }
    const cudaError_t err = cudaGetLastError();
    return err == cudaSuccess ? ok() : cuda_fail(err, "pn_kv4_append");
}

int pn_kv4_gather(const void* cache, int64_t n_pages, int64_t kv_heads, int64_t page, int64_t head_dim,
                  const int32_t* block_table, int64_t table_ld, int64_t table_w, const int32_t* seq_lens,
                  const int32_t* cu_q, int64_t B, int64_t T, void* k, void* v, int kv_dtype, void* stream) {
    pn::Kv4GatherArgs a{};
    if (int st = check_kv4("pn_kv4_gather", cache, n_pages, kv_heads, page, head_dim, block_table, table_ld, table_w,
                           seq_lens, cu_q, B, T, &a.s))
        return st;
    if (kv_dtype != PN_F32 && kv_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "pn_kv4_gather: dtype %d", kv_dtype);
    if (T > 0 && B > 0 && (!k || !v)) return fail(PN_ERR_ARG, "pn_kv4_gather: null pointer");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(PN_ERR_ALIGN, "pn_kv4_gather: k and v need 16-byte alignment");
    if (int st = check_device()) return st;
    if (T == 0 || B == 0) return ok();
    if (n_pages == 0) a.s.table_w = 0;  // every length counts as zero
    a.cache = static_cast<const uint8_t*>(cache);
    a.y[0] = k;
    a.y[1] = v;
    a.y_f32 = kv_dtype == PN_F32;
    const int64_t blocks = (T * kv_heads * 2 * (head_dim / 8) + pn::kKv4Threads - 1) / pn::kKv4Threads;
    if (blocks > 0x7fffffff) return fail(PN_ERR_SHAPE, "pn_kv4_gather: too many rows");
    const cudaStream_t s = (cudaStream_t)stream;
    if (head_dim == 64) pn::kv4_gather_kernel<64><<<(unsigned)blocks, pn::kKv4Threads, 0, s>>>(a);
    else pn::kv4_gather_kernel<128><<<(unsigned)blocks, pn::kKv4Threads, 0, s>>>(a);
    const cudaError_t err = cudaGetLastError();
    return err == cudaSuccess ? ok() : cuda_fail(err, "pn_kv4_gather");
}

}  // extern "C"
