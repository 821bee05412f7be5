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
    int table_w;           // pages per sequence in the table; 0 where there are no pages at all
    const int32_t* lens;   // (B)
    const int32_t* cu;     // (B + 1) first row of each sequence, or null: L rows each
    int64_t B, T;          // sequences, rows
    int64_t L;
    int64_t n_pages;
    int Hk, page;
    int64_t table_hd;    // entries between the tables of a sequence's kv heads; 0: they share one
    // Shared prefixes: the B "sequences" are prefixes, with a table and a length each, whose
    // rows are those of sequences [grp[b], grp[b + 1]) of `grouped` (grp null: equally many
    // each).  0: the sequences are themselves.
    int64_t grouped;
    const int32_t* grp;  // (B + 1)
};

// An entry of a table or a length.  kMore: they may be what the kernel before wrote, and this one may have
// begun while it did (a dependent launch): memory that changes under a grid is not for __ldg, whose loads
// need not stay behind the grid's wait.
template <bool kMore>
__device__ __forceinline__ int kv4_load(const int32_t* p) {
    if constexpr (kMore)
        return *p;
    else
        return __ldg(p);
}
// The length of sequence b, and how much of it its table has room for.
template <bool kMore = false>
__device__ __forceinline__ int kv4_len(const Kv4Seq& s, int64_t b) { return min(max(kv4_load<kMore>(s.lens + b), 0), 1 << 30); }
template <bool kMore = false>
__device__ __forceinline__ int kv4_held(const Kv4Seq& s, int64_t b) { return min(kv4_len<kMore>(s, b), s.table_w * s.page); }

// First row and number of rows of sequence b (kMore: which may be a prefix).
template <bool kMore = false>
__device__ __forceinline__ void kv4_rows(const Kv4Seq& s, int64_t b, int64_t& first, int64_t& n) {
    if (kMore && s.grouped) {
        int64_t b0 = b * (s.grouped / s.B), b1 = b0 + s.grouped / s.B;
        if (s.grp) {
            b0 = min(max((int64_t)__ldg(s.grp + b), (int64_t)0), s.grouped);
            b1 = min(max((int64_t)__ldg(s.grp + b + 1), b0), s.grouped);
        }
        first = s.cu ? min(max((int64_t)__ldg(s.cu + b0), (int64_t)0), s.T) : b0 * s.L;
        n = (s.cu ? min(max((int64_t)__ldg(s.cu + b1), first), s.T) : b1 * s.L) - first;
        return;
    }
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
// status word) when the table has no entry for it, or one that is no page of the
// cache.  (A table without any entry is no mistake of an index: nothing is reported.)
__device__ __forceinline__ int64_t kv4_page(const Kv4Seq& s, int64_t b, int pos) {
    const int p = pos < s.table_w * s.page ? __ldg(s.table + b * s.table_ld + pos / s.page) : -1;
    if (p >= 0 && p < s.n_pages) return p;
    if (s.table_w > 0) record_status(PN_ERR_ARG);
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

// Where a row lives, looked up once per row and block.
struct Kv4Row {
    int64_t src[2];  // first element of its keys and values in the inputs
    int64_t dst;     // its page's first byte in the cache; -1: none
    int tok;         // its place in the page
};
constexpr int kKv4Threads = 256;
constexpr int kKv4MaxRows = 8;  // rows per block

// A block's vectors are numbered row by row, a row's keys before its values; a
// thread steps from one to the next without a division.
struct Kv4Step {
    int block;    // bytes of a page block
    int per_row;  // 2 * kv heads
    int dr, dh;   // the vectors of a block at once, as whole rows and the rest
};
struct Kv4At {
    int r, hv;  // row in the block; head, or Hk + head
    __device__ __forceinline__ Kv4At(const Kv4Step& s, int vec) : r(vec / s.per_row), hv(vec - r * s.per_row) {}
    __device__ __forceinline__ void next(const Kv4Step& s) {
        r += s.dr;
        hv += s.dh;
        if (hv >= s.per_row) {
            hv -= s.per_row;
            ++r;
        }
    }
};

__device__ __forceinline__ void kv4_rows_of_block(const Kv4Seq& s, int64_t row0, int n, const int64_t* sb, const int64_t* sl,
                                                  const Kv4Step& step, Kv4Row* rows) {
    if ((int)threadIdx.x < n) {
        Kv4Row r;
        const int64_t row = row0 + threadIdx.x;
        int64_t b, i;
        r.dst = -1;
        r.tok = 0;
        if (kv4_find(s, row, b, i)) {
            int64_t first, count;
            kv4_rows(s, b, first, count);
            const int pos = (int)(kv4_len(s, b) - count + i);
            if (pos >= 0) {
                const int64_t page = kv4_page(s, b, pos);
                if (page >= 0) r.dst = page * step.per_row * step.block;
                r.tok = pos % s.page;
            }
            if (sb)
                for (int kv = 0; kv < 2; ++kv) r.src[kv] = s.cu ? row * sl[kv] : b * sb[kv] + i * sl[kv];
        }
        rows[threadIdx.x] = r;
    }
    __syncthreads();
}

struct Kv4AppendArgs {
    Kv4Seq s;
    const void* x[2];             // keys, values
    int64_t sb[2], sl[2], sh[2];  // their strides in elements: sequence, row, head
    int vec;                      // 16-byte loads allowed
    int rows;                     // per block
    Kv4Step step;
    uint8_t* cache;
};

// Eight codes of a vector as nibbles: c_j = rint((v_j - z) / s), IEEE division,
// ties to even.  With bf16 inputs quotients that are exact half-integers are
// common (about one in 10^2), so the borders are decided exactly, without a
// division: h is the quotient in half steps, e = d - h * s / 2 is exact (h * s has
// 13 bits and cancels the head of d), and h / 2 + e / s, rounded to an integer,
// goes the way that the sign of e says, or to even where e is 0.  (s has 8 bits, so
// a quotient that is no half-integer lies at least ulp(d) / s away from one: more
// than half an ulp of the quotient, neither the rounding of h / 2 + e / s nor that
// of the IEEE quotient reaches the border.)  s >= (max - z) / 15 keeps c within
// 0 .. 15.
__device__ __forceinline__ uint32_t kv4_codes8(const float (&v)[8], float s, float z) {
    float rs;  // within an ulp
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rs) : "f"(s));
    const float2 up = make_float2(kRoundMagic, kRoundMagic), down = make_float2(-kRoundMagic, -kRoundMagic);
    float2 q[4];
    if (rs >= 0x1p-125f && rs <= 0x1p125f) {
        const float2 z2 = make_float2(-z, -z), rs1 = make_float2(rs, rs), rs2 = make_float2(2.0f * rs, 2.0f * rs);
        const float2 half_s = make_float2(-0.5f * s, -0.5f * s), half = make_float2(0.5f, 0.5f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 d = add2(make_float2(v[j], v[j + 4]), z2);
            const float2 h = add2(fma2(d, rs2, up), down);
            const float2 e = fma2(h, half_s, d);
            q[j] = add2(add2(fma2(e, rs1, mul2(h, half)), up), down);
        }
    } else {  // 1/s or its neighbours are no normal numbers
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            q[j].x = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(v[j], z), s)), 0.0f), 15.0f);
            q[j].y = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(v[j + 4], z), s)), 0.0f), 15.0f);
        }
    }
    // q0 + 16 (q1 + 16 (q2 + 16 q3)): exact below 2^16, and the integer is in the low bits of a sum with 2^23
    const float2 sixteen = make_float2(16.0f, 16.0f);
    const float2 w = add2(fma2(fma2(fma2(q[3], sixteen, q[2]), sixteen, q[1]), sixteen, q[0]),
                          make_float2(8388608.0f, 8388608.0f));
    return __byte_perm(__float_as_uint(w.x), __float_as_uint(w.y), 0x5410);
}

// The range of VT lanes' values, a NaN among them kept: (min, max).
template <int VT>
__device__ __forceinline__ float2 kv4_range(const Raw8<float> (&x)[2]) {
    float v[2][8];
    x[0].get(v[0]);
    x[1].get(v[1]);
    float lo = v[0][0], hi = v[0][0];
#pragma unroll
    for (int j = 1; j < 16; ++j) {
        lo = min_nan(lo, v[j >> 3][j & 7]);
        hi = max_nan(hi, v[j >> 3][j & 7]);
    }
#pragma unroll
    for (int o = VT / 2; o > 0; o >>= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    return make_float2(lo, hi);
}
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// bf16: (min, -max) share a register, one shuffle and one minimum per step.
template <int VT>
__device__ __forceinline__ float2 kv4_range(const Raw8<__nv_bfloat16> (&x)[2]) {
    constexpr uint32_t kNeg = 0x80008000u;
    const uint4 u = x[0].u, v = x[1].u;
    const uint32_t lo = min2_nan(min2_nan(min2_nan(u.x, u.y), min2_nan(u.z, u.w)), min2_nan(min2_nan(v.x, v.y), min2_nan(v.z, v.w)));
    const uint32_t hi = max2_nan(max2_nan(max2_nan(u.x, u.y), max2_nan(u.z, u.w)), max2_nan(max2_nan(v.x, v.y), max2_nan(v.z, v.w))) ^ kNeg;
    uint32_t r = min2_nan(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
#pragma unroll
    for (int o = VT / 2; o > 0; o >>= 1) r = min2_nan(r, __shfl_xor_sync(0xffffffffu, r, o));
    return make_float2(__uint_as_float(r << 16), __uint_as_float((r & 0xFFFF0000u) ^ 0x80000000u));
}

// D / 16 lanes per vector, sixteen dims each; a block takes a few rows with all
// their heads, the next vector's values in flight while one is stored.  One read
// of the inputs; what bounds it beside the bytes is the instructions per vector
// (the range's shuffles, scale, codes and addresses: 61 % of the issue slots) and the
// barrier behind each block's look-up, its largest stall.  9723 bf16 rows of 8 heads,
// d = 128: 21 us, 2.4 TB/s (8 us at the copy's rate); with eight dims per lane, 233
// instructions per eight values, it took 26 us.
template <typename T, int D>
__global__ void __launch_bounds__(kKv4Threads) kv4_append_kernel(const Kv4AppendArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    constexpr int VT = D / 16, kVecs = kKv4Threads / VT;
    __shared__ Kv4Row rows[kKv4MaxRows];
    const int64_t row0 = (int64_t)blockIdx.x * a.rows;
    const int n_rows = (int)min((int64_t)a.rows, a.s.T - row0);
    kv4_rows_of_block(a.s, row0, n_rows, a.sb, a.sl, a.step, rows);
    const int l = threadIdx.x % VT;

    Kv4At at(a.step, threadIdx.x / VT);
    auto load = [&](Raw8<T> (&x)[2]) {
        x[0].zero();
        x[1].zero();
        if (at.r >= n_rows || rows[at.r].dst < 0) return;
        const bool kv = at.hv >= a.s.Hk;
        const T* p = static_cast<const T*>(kv ? a.x[1] : a.x[0]) + rows[at.r].src[kv] + l * 16 +
                     (kv ? (at.hv - a.s.Hk) * a.sh[1] : at.hv * a.sh[0]);
        if (a.vec) {
            x[0].load(p);
            x[1].load(p + 8);
        } else {
            float v[8];
            kv4_load8(p, false, v);
            x[0].set(v);
            kv4_load8(p + 8, false, v);
            x[1].set(v);
        }
    };
    Raw8<T> x[2];
    load(x);
    for (int base = 0; base < n_rows * a.step.per_row; base += kVecs) {
        const Raw8<T> now[2] = {x[0], x[1]};
        const Kv4At was = at;
        at.next(a.step);
        load(x);
        const float2 range = kv4_range<VT>(now);
        if (was.r >= n_rows || rows[was.r].dst < 0) continue;
        const bool kv = was.hv >= a.s.Hk;
        float z = floor_bf16(range.x);
        float s = ceil_bf16_pos(__fdiv_rn(__fsub_rn(range.y, z), 15.0f));
        if (!(s < INFINITY) || !(fabsf(z) < INFINITY)) {  // an inf or NaN in the vector: all of it reads back as NaN
            s = 0.0f;
            z = __int_as_float(0x7fc00000);
        }
        uint2 w = make_uint2(0, 0);
        if (s > 0.0f) {
            float v[8];
            now[0].get(v);
            w.x = kv4_codes8(v, s, z);
            now[1].get(v);
            w.y = kv4_codes8(v, s, z);
        }
        const int tok = rows[was.r].tok;
        uint8_t* blk = a.cache + rows[was.r].dst + (int64_t)(kv ? 2 * (was.hv - a.s.Hk) + 1 : 2 * was.hv) * a.step.block;
        if (!kv) {
            *reinterpret_cast<uint2*>(blk + tok * (D / 2) + l * 8) = w;
        } else {
            uint16_t* p = reinterpret_cast<uint16_t*>(blk + (tok >> 1) * D + l * 16 + (tok & 1) * 2);
            p[0] = (uint16_t)w.x, p[2] = (uint16_t)(w.x >> 16);
            p[4] = (uint16_t)w.y, p[6] = (uint16_t)(w.y >> 16);
        }
        if (l == 0)
            *reinterpret_cast<uint32_t*>(blk + a.s.page * (D / 2) + tok * 4) =
                (__float_as_uint(s) >> 16) | (__float_as_uint(z) & 0xFFFF0000u);
    }
}

struct Kv4GatherArgs {
    Kv4Seq s;
    const uint8_t* cache;
    void* y[2];
    int y_f32;
    int rows;  // per block
    Kv4Step step;
};

// The reverse, zeros for rows that are not there: a code is masked into the low
// bits of 2^23, one fma per value.  Bound by latency: the rows' look-up, a barrier and the
// codes' loads stand before a block's first store (43 % of the issue slots used); the same
// rows 15.2 us, 3.4 TB/s.
template <int D>
__global__ void __launch_bounds__(kKv4Threads) kv4_gather_kernel(const Kv4GatherArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    constexpr int VT = D / 16;
    __shared__ Kv4Row rows[kKv4MaxRows];
    const int64_t row0 = (int64_t)blockIdx.x * a.rows;
    const int n_rows = (int)min((int64_t)a.rows, a.s.T - row0);
    kv4_rows_of_block(a.s, row0, n_rows, nullptr, nullptr, a.step, rows);
    const int l = threadIdx.x % VT;
    Kv4At at(a.step, threadIdx.x / VT);
    uint2 w = make_uint2(0, 0);  // the next vector's codes and (scale, zero)
    uint32_t pair = 0;
    auto load = [&]() {
        w = make_uint2(0, 0);  // stands for zeros
        pair = 0;
        if (at.r >= n_rows || rows[at.r].dst < 0) return;
        const bool kv = at.hv >= a.s.Hk;
        const int tok = rows[at.r].tok;
        const uint8_t* blk = a.cache + rows[at.r].dst + (int64_t)(kv ? 2 * (at.hv - a.s.Hk) + 1 : 2 * at.hv) * a.step.block;
        // (written out: the compiler puts its loads where they are used, 17.6 us for 15.2)
        asm volatile("ld.global.u32 %0, [%1];" : "=r"(pair) : "l"(blk + a.s.page * (D / 2) + tok * 4));
        if (!kv) {
            asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "l"(blk + tok * (D / 2) + l * 8));
        } else {
            uint4 two;
            asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(two.x), "=r"(two.y), "=r"(two.z), "=r"(two.w)
                         : "l"(blk + (tok >> 1) * D + l * 16));
            const uint32_t which = tok & 1 ? 0x7632 : 0x5410;
            w = make_uint2(__byte_perm(two.x, two.y, which), __byte_perm(two.z, two.w, which));
        }
    };
    load();
    while (at.r < n_rows) {
        const uint2 now = w;
        const uint32_t now_pair = pair;
        const Kv4At was = at;
        at.next(a.step);
        load();
        const bool kv = was.hv >= a.s.Hk;
        const float s = __uint_as_float(now_pair << 16), z = __uint_as_float(now_pair & 0xFFFF0000u);
        const int64_t to = ((row0 + was.r) * a.s.Hk + was.hv - (kv ? a.s.Hk : 0)) * D + l * 16;
        void* out = kv ? a.y[1] : a.y[0];
        // masked into the low bits of 2^23 a code reads as 2^23 + 16^j c; s * c is exact (12 bits), so one rounding
        const float2 z2 = make_float2(z, z), down = make_float2(-8388608.0f, -8388608.0f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t c8 = i ? now.y : now.x;
            float v[8], sj = s;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 c = make_float2(__uint_as_float((c8 & (15u << (4 * j))) | 0x4B000000u),
                                             __uint_as_float(((c8 >> 16) & (15u << (4 * j))) | 0x4B000000u));
                const float2 y = fma2(add2(c, down), make_float2(sj, sj), z2);
                v[j] = y.x, v[j + 4] = y.y;
                sj *= 0.0625f;
            }
            if (a.y_f32) {
                Raw8<float> o;
                o.set(v);
                o.store(static_cast<float*>(out) + to + i * 8);
            } else {
                Raw8<__nv_bfloat16> o;
                o.set(v);
                o.store(static_cast<__nv_bfloat16*>(out) + to + i * 8);
            }
        }
    }
}

// Rows per block: as many as leave eight blocks to an SM (each looks its rows up
// first), one where there are few.  (9723 rows: 21 us with 8 rows to a block, 23
// with 4, 28 with 2.)
static int kv4_block_rows(int64_t T) {
    const int64_t sms = sm_count();
    int r = 1;
    while (r < kKv4MaxRows && T / (2 * r) >= 8 * sms) r *= 2;
    return r;
}
static Kv4Step kv4_step(int Hk, int64_t page, int64_t D) {
    const int vecs = kKv4Threads / (int)(D / 16), per_row = 2 * Hk;
    return {(int)(page * (D / 2 + 4)), per_row, vecs / per_row, vecs % per_row};
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
    *s = pn::Kv4Seq{table, table_ld, n_pages > 0 ? (int)table_w : 0, lens, cu, B, T, B > 0 ? T / B : 0, n_pages, (int)Hk, (int)page};
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
    a.x[0] = k, a.sb[0] = k_sb, a.sl[0] = k_sl, a.sh[0] = k_sh;
    a.x[1] = v, a.sb[1] = v_sb, a.sl[1] = v_sl, a.sh[1] = v_sh;
    a.cache = static_cast<uint8_t*>(cache);
    auto whole = [&](int i) {  // every row of 8 dims starts on a 16-byte boundary
        const int64_t n = 16 / (int64_t)e;
        return aligned(a.x[i], 16) && a.sb[i] % n == 0 && a.sl[i] % n == 0 && a.sh[i] % n == 0;
    };
    a.vec = whole(0) && whole(1);
    a.rows = pn::kv4_block_rows(T);
    a.step = pn::kv4_step((int)kv_heads, page, head_dim);
    const unsigned g = (unsigned)((T + a.rows - 1) / a.rows);
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
    if (T > 0 && (!k || !v)) return fail(PN_ERR_ARG, "pn_kv4_gather: null pointer");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(PN_ERR_ALIGN, "pn_kv4_gather: k and v need 16-byte alignment");
    if (int st = check_device()) return st;
    if (T == 0) return ok();
    if (B == 0) {  // every row lies behind the last sequence
        const size_t bytes = (size_t)T * kv_heads * head_dim * (kv_dtype == PN_F32 ? 4 : 2);
        for (void* y : {k, v}) {
            const cudaError_t err = cudaMemsetAsync(y, 0, bytes, (cudaStream_t)stream);
            if (err != cudaSuccess) return cuda_fail(err, "pn_kv4_gather");
        }
        return ok();
    }
    a.cache = static_cast<const uint8_t*>(cache);
    a.y[0] = k;
    a.y[1] = v;
    a.y_f32 = kv_dtype == PN_F32;
    a.rows = pn::kv4_block_rows(T);
    a.step = pn::kv4_step((int)kv_heads, page, head_dim);
    const unsigned g = (unsigned)((T + a.rows - 1) / a.rows);
    const cudaStream_t s = (cudaStream_t)stream;
    if (head_dim == 64) pn::kv4_gather_kernel<64><<<g, pn::kKv4Threads, 0, s>>>(a);
    else pn::kv4_gather_kernel<128><<<g, pn::kKv4Threads, 0, s>>>(a);
    const cudaError_t err = cudaGetLastError();
    return err == cudaSuccess ? ok() : cuda_fail(err, "pn_kv4_gather");
}

}  // extern "C"
