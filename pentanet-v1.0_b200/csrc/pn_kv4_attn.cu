// pn_kv4_attn.cu -- causal attention of each sequence's newest rows over its
// 4-bit paged cache (layout: pn_kv4.cu).
//
// Mathematics.  With key c_k * s_k + z_k and value c_v * s_v + z_v per token,
//   logit = scale * (s_k * (q . c_k) + z_k * sum(q))
//   out   = (sum_t p_t s_v c_v + sum_t p_t z_v) / sum_t p_t,  p_t = 2^(logit_t - m)
// so both matrix products run on the raw codes.  A code is brought to fp16 by
// a mask alone: 0x000c read as fp16 is the subnormal c * 2^-24, 0x00c0 is
// c * 2^-20, both exact, and the products are summed in fp32; the powers of
// two are taken out again in fp32 (odd operands carry 2^4 more: on the key side
// the query is divided by 16 there, on the value side the output is).  Five
// integer operations give four fp16 pairs.  A row's query is scaled by a power
// of two to a largest magnitude in [2^14, 2^15), so bf16 queries stay exact in fp16 down
// to 2^-32 of the largest (fp32 queries are rounded to 11 bits).  The weights
// p_t * s_v are rounded to fp16 (11 bits, more than the bf16 output keeps)
// relative to the largest s_v seen; sums, the softmax's maximum and total, and
// the z term are fp32.
//
// Shape of the decode kernel.  Keys are the 16-row operand of m16n8k16 (16
// tokens), the query rows of one kv head (group x new tokens) its 8 columns,
// so one product serves a whole group and wastes no more than 8 - rows
// columns.  Each warp streams 16-token pieces of its own, with its own running
// maximum, total and output in registers: no block-wide step inside the loop;
// the four warps of a block are joined in shared memory at the end of a
// segment.  The pieces come through a ring of cp.async copies private to the
// warp.
//
// Work split.  The units (64 tokens of one row tile, kv head and sequence) of
// the whole call are laid end to end and every block takes an equal run of
// them, so ragged batches and single long sequences alike fill the SMs without
// the host knowing any length.  A block's run may start or end inside a row
// tile: such partial results go to the workspace and a second kernel joins
// them in a fixed order, so results do not depend on timing.
#include <cuda_fp16.h>

#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

struct Kv4AttnArgs {
    Kv4Seq s;
    const void* q;
    int q_f32, q_vec;
    int64_t q_sb, q_sl, q_sh;
    const uint8_t* cache;
    int G;            // query heads per kv head
    float scale_log2; // softmax scale * log2(e)
    void* out;        // (T, Hk * G, D), q's type
    int64_t* prefix;  // workspace: units before each sequence (B + 1)
    float* part;      // workspace: partial results of two segments per block
};

constexpr int kAttnTokens = 64;  // tokens of a unit
constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;

__device__ __forceinline__ float ex2f(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^e for e in [-126, 127].
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// Row tiles of RT query rows and the units of sequence b (every row tile is
// walked over all of the sequence's tokens; what a tile may not see is skipped
// when it is met).
__device__ __forceinline__ int64_t attn_units(const Kv4AttnArgs& a, int64_t b, int rt_rows, int& nt) {
    int64_t first, n;
    kv4_rows(a.s, b, first, n);
    nt = max((kv4_len(a.s, b) + kAttnTokens - 1) / kAttnTokens, 1);
    return (n * a.G + rt_rows - 1) / rt_rows * nt * a.s.Hk;
}

// Units before sequence b for every b, and the sequence that holds `want`:
// all threads of the block; block 0 leaves the sums for the joining kernel.
__device__ __forceinline__ int64_t attn_plan(const Kv4AttnArgs& a, int rt_rows, int64_t* sh_sum, int64_t& total) {
    // thread t takes sequences [t * per, (t + 1) * per)
    const int64_t per = (a.s.B + kAttnThreads - 1) / kAttnThreads;
    const int64_t b0 = min(threadIdx.x * per, a.s.B), b1 = min(b0 + per, a.s.B);
    int64_t sum = 0;
    int nt;
    for (int64_t b = b0; b < b1; ++b) sum += attn_units(a, b, rt_rows, nt);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) sh_sum[w] = inc;
    __syncthreads();
    int64_t before = inc - sum;
    total = 0;
#pragma unroll
    for (int i = 0; i < kAttnWarps; ++i) {
        if (i < w) before += sh_sum[i];
        total += sh_sum[i];
    }
    if (blockIdx.x == 0) {
        int64_t at = before;
        for (int64_t b = b0; b < b1; ++b) {
            a.prefix[b] = at;
            at += attn_units(a, b, rt_rows, nt);
        }
        if (threadIdx.x == 0) a.prefix[a.s.B] = total;
    }
    return before;
}

// Block c's first unit.
__device__ __forceinline__ int64_t attn_begin(int64_t total, int64_t blocks, int64_t c) {
    return total / blocks * c + min(c, total % blocks);
}

__device__ __forceinline__ void store_out(const Kv4AttnArgs& a, int64_t at, const float4& y, float inv) {
    if (a.q_f32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    } else {
        const __nv_bfloat162 u = __floats2bfloat162_rn(y.x * inv, y.y * inv), v = __floats2bfloat162_rn(y.z * inv, y.w * inv);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
    }
}

// A row's query operands: scaled to the power of two that brings the row's
// largest magnitude to [2^14, 2^15), dims base + {0,4}, {1,5} / 16, {2,6}, {3,7} / 16
// of each word of eight dims that this thread holds (words t * W ..).
template <int D>
__device__ __forceinline__ void load_query(const Kv4AttnArgs& a, const char* row, int t, uint32_t (&qb)[D / 8], float& ca,
                                           float& cb) {
    constexpr int W = D / 32;
    float v[W * 8];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        float u[8];
        if (!row) {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = 0.0f;
        } else if (a.q_f32) {
            kv4_load8(reinterpret_cast<const float*>(row) + (t * W + i) * 8, a.q_vec, u);
        } else {
            kv4_load8(reinterpret_cast<const __nv_bfloat16*>(row) + (t * W + i) * 8, a.q_vec, u);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i * 8 + j] = u[j];
    }
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < W * 8; ++j) amax = max_nan(amax, fabsf(v[j]));
    amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // exponent of the scaling, kept where 2^e and 2^(24 - e) are normal numbers
    int e = 14 - ((int)(__float_as_uint(amax) >> 23) - 127);
    e = amax > 0.0f ? min(max(e, -100), 126) : 0;
    const float up = pow2i(e);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = v[i * 8 + j] * up;
        const uint32_t p[4] = {pack_f16(u[0], u[4]), pack_f16(u[1] * 0.0625f, u[5] * 0.0625f), pack_f16(u[2], u[6]),
                               pack_f16(u[3] * 0.0625f, u[7] * 0.0625f)};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            qb[i * 4 + k] = p[k];
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[k]));
            sum += (f.x + f.y) * (k & 1 ? 16.0f : 1.0f);
        }
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    ca = a.scale_log2 * pow2i(24 - e);
    cb = a.scale_log2 * (sum * pow2i(-e));
}

template <int D, int NT>
struct AttnCfg {
    static constexpr int W = D / 32;             // words per thread and token
    static constexpr int kRows = 8 * NT;         // query rows of a row tile
    static constexpr int kStages = 4;
    static constexpr int kCodes = 16 * (D / 2);  // bytes of one 16-token piece of keys or values
    static constexpr int kStage = 2 * kCodes + 128;
    static constexpr int kRing = kAttnWarps * kStages * kStage;
    static constexpr int kPitch = D + 8;         // floats per row of the join buffer
    static constexpr int kJoin = kAttnWarps * kRows * kPitch * 4;
    static constexpr int kSmem = kRing + kJoin + kAttnWarps * kRows * 8;
    static constexpr int kPart = kRows * (D + 2);  // floats of one partial result
};

// Byte position of 16-byte chunk j of token pair p inside a piece's values:
// rotated so that the eight lanes of one shared-memory phase (two dim groups x
// four pairs) meet eight different bank groups.
template <int D>
__device__ __forceinline__ int v_chunk(int p, int j) {
    return D == 128 ? p * 128 + ((j + 2 * p) & 7) * 16 : p * 64 + ((j + (p & 2)) & 3) * 16;
}

template <int D, int NT>
__global__ void __launch_bounds__(kAttnThreads, NT == 1 ? 4 : NT == 2 ? 3 : 2) kv4_decode_kernel(const Kv4AttnArgs a) {
    using C = AttnCfg<D, NT>;
    constexpr int W = C::W, RT = C::kRows, ST = C::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t sh_sum[kAttnWarps];
    __shared__ int64_t sh_start[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * ST * C::kStage;
    const uint32_t ring_u = smem_u32(ring);
    float* join = reinterpret_cast<float*>(smem + C::kRing);
    float* join_ml = reinterpret_cast<float*>(smem + C::kRing + C::kJoin);
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    int64_t total;
    const int64_t before = attn_plan(a, RT, sh_sum, total);
    const int64_t begin = attn_begin(total, gridDim.x, blockIdx.x), end = attn_begin(total, gridDim.x, blockIdx.x + 1);
    if (begin >= end) return;
    {   // the sequence that holds unit `begin`
        const int64_t per = (a.s.B + kAttnThreads - 1) / kAttnThreads;
        const int64_t b0 = min(tid * per, a.s.B), b1 = min(b0 + per, a.s.B);
        int64_t at = before;
        int nt;
        for (int64_t b = b0; b < b1; ++b) {
            const int64_t n = attn_units(a, b, RT, nt);
            if (begin >= at && begin < at + n) {
                sh_start[0] = b;
                sh_start[1] = begin - at;
            }
            at += n;
        }
        __syncthreads();
    }
    int64_t b = sh_start[0], in_seq = sh_start[1], unit = begin;
    const int64_t block = (int64_t)a.s.page * (D / 2 + 4);

    while (unit < end) {
        int nt;
        while (in_seq >= attn_units(a, b, RT, nt)) {  // past the sequence (or one without rows)
            in_seq -= attn_units(a, b, RT, nt);
            ++b;
        }
        // a row tile's units are consecutive: (head, row tile, token tile)
        int64_t row0, n_rows;
        kv4_rows(a.s, b, row0, n_rows);
        const int len = kv4_len(a.s, b);
        const int64_t q_rows = n_rows * a.G, n_rt = (q_rows + RT - 1) / RT;
        const int64_t tile_id = in_seq / nt;
        const int head = (int)(tile_id / n_rt);
        const int64_t r0 = (tile_id - head * n_rt) * RT;  // first query row of the tile
        const int rows = (int)min((int64_t)RT, q_rows - r0);
        const int t0 = (int)(in_seq - tile_id * nt);
        const int t1 = (int)min((int64_t)nt, t0 + (end - unit));
        // positions: row r sees tokens up to len - n_rows + r / G
        const int64_t pos0 = len - n_rows;
        const int kv_end = (int)max(pos0 + (r0 + rows - 1) / a.G + 1, (int64_t)0);  // seen by the tile's last row
        const int lim_min = (int)(pos0 + r0 / a.G);                                  // ... by its first
        const int used = min(t1, (kv_end + kAttnTokens - 1) / kAttnTokens);           // tiles behind it are skipped

        // ---- queries
        uint32_t qb[NT][D / 8];
        float ca[NT][2], cb[NT][2];
        int lim[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int64_t r = r0 + n * 8 + g;
            const char* row = nullptr;
            if (n * 8 + g < rows) {
                const int64_t i = r / a.G, at = (a.s.cu ? (row0 + i) * a.q_sl : b * a.q_sb + i * a.q_sl) +
                                                (head * a.G + r % a.G) * a.q_sh;
                row = static_cast<const char*>(a.q) + at * (a.q_f32 ? 4 : 2);
            }
            float fa, fb;
            load_query<D>(a, row, t, qb[n], fa, fb);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                ca[n][k] = __shfl_sync(0xffffffffu, fa, (2 * t + k) * 4);
                cb[n][k] = __shfl_sync(0xffffffffu, fb, (2 * t + k) * 4);
                const int rl = n * 8 + 2 * t + k;
                lim[n][k] = rl < rows ? (int)(pos0 + (r0 + rl) / a.G) : kv_end - 1;
            }
        }

        // ---- the warp's pieces: tokens [64 * tile + 16 * warp, + 16)
        const int count = used - t0;
        uint32_t bad = 0;  // ring of flags: the piece is not there
        int page_id = 0, page_off = 0;
        auto issue = [&](int i) {
            if ((i & 31) == 0) {  // lane l looks up piece i + l
                const int tok = (t0 + i + lane) * kAttnTokens + warp * 16;
                page_id = -1;
                if (i + lane < count && tok < kv_end) {
                    const int p = __ldg(a.s.table + b * a.s.table_ld + tok / a.s.page);
                    page_off = tok % a.s.page;
                    if (p >= 0 && p < a.s.n_pages)
                        page_id = p;
                    else
                        record_status(PN_ERR_ARG);
                }
            }
            const int p = __shfl_sync(0xffffffffu, page_id, i & 31), off = __shfl_sync(0xffffffffu, page_off, i & 31);
            const uint32_t bit = 1u << (i & 31);
            if (i < count && p >= 0) {
                bad &= ~bit;
                const uint8_t* kb = a.cache + ((int64_t)p * a.s.Hk + head) * 2 * block;
                const uint8_t* vb = kb + block;
                const uint32_t dst = ring_u + (i % ST) * C::kStage;
#pragma unroll
                for (int c = lane; c < C::kCodes / 16; c += 32) {
                    cp_async16(dst + c * 16, kb + off * (D / 2) + c * 16);
                    cp_async16(dst + C::kCodes + v_chunk<D>(c / (D / 16), c % (D / 16)), vb + off * (D / 2) + c * 16);
                }
                if (lane < 8)
                    cp_async16(dst + 2 * C::kCodes + lane * 16,
                               (lane < 4 ? kb : vb) + (int64_t)a.s.page * (D / 2) + off * 4 + (lane & 3) * 16);
            } else {
                bad |= bit;
            }
            cp_commit();
        };

        float m[NT][2], l[NT][2], zs[NT][2], o[NT][D / 16][4];
        float S = 0.0f, inv_S = 0.0f;  // power of two not below the largest value scale seen, and its inverse
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int k = 0; k < 2; ++k) m[n][k] = -INFINITY, l[n][k] = 0.0f, zs[n][k] = 0.0f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[n][j][k] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) issue(i);
        for (int i = 0; i < count; ++i) {
            issue(i + ST - 1);
            cp_wait<ST - 1>();
            __syncwarp();
            const int tok0 = (t0 + i) * kAttnTokens + warp * 16;
            if (!(bad >> (i & 31) & 1u)) {
                const uint8_t* st = ring + (i % ST) * C::kStage;
                // ---- logits: 16 tokens x 8 rows per n
                float acc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[n][k] = 0.0f;
                uint32_t ka[W], kb[W];
                if constexpr (W == 4) {
                    const uint4 u = *reinterpret_cast<const uint4*>(st + g * (D / 2) + t * 16);
                    const uint4 v = *reinterpret_cast<const uint4*>(st + (g + 8) * (D / 2) + t * 16);
                    ka[0] = u.x, ka[1] = u.y, ka[2] = u.z, ka[3] = u.w;
                    kb[0] = v.x, kb[1] = v.y, kb[2] = v.z, kb[3] = v.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(st + g * (D / 2) + t * 8);
                    const uint2 v = *reinterpret_cast<const uint2*>(st + (g + 8) * (D / 2) + t * 8);
                    ka[0] = u.x, ka[1] = u.y, kb[0] = v.x, kb[1] = v.y;
                }
#pragma unroll
                for (int w = 0; w < W; ++w) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t u = h ? ka[w] >> 8 : ka[w], v = h ? kb[w] >> 8 : kb[w];
                        const uint32_t a0 = u & 0x000F000Fu, a1 = v & 0x000F000Fu, a2 = u & 0x00F000F0u, a3 = v & 0x00F000F0u;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_f16(acc[n], a0, a1, a2, a3, qb[n][w * 4 + h * 2], qb[n][w * 4 + h * 2 + 1]);
                    }
                }
                uint32_t kp[2], vp[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    kp[k] = *reinterpret_cast<const uint32_t*>(st + 2 * C::kCodes + (g + 8 * k) * 4);
                    vp[k] = *reinterpret_cast<const uint32_t*>(st + 2 * C::kCodes + 64 + (g + 8 * k) * 4);
                    if (tok0 + g + 8 * k >= kv_end) vp[k] = 0;  // whatever lies behind the sequence
                }
                bool grow = false;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float ks = __uint_as_float(kp[k] << 16), kz = __uint_as_float(kp[k] & 0xFFFF0000u);
                    grow |= __uint_as_float(vp[k] << 16) > S;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float& x = acc[n][2 * k + j];
                            x = fmaf(ks, x * ca[n][j], kz * cb[n][j]);
                        }
                }
                if (tok0 + 15 > lim_min) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (tok0 + g + 8 * (k >> 1) > lim[n][k & 1]) acc[n][k] = -INFINITY;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) grow |= acc[n][k] > m[n][k & 1] + 8.0f;
                // The maximum need not be exact: a weight may exceed 1 by up to 2^8
                // before the sums are rescaled (fp16 holds 2^15), so most pieces
                // skip this.
                if (__any_sync(0xffffffffu, grow)) {
                    float vs = fmaxf(__uint_as_float(vp[0] << 16), __uint_as_float(vp[1] << 16));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) vs = fmaxf(vs, __shfl_xor_sync(0xffffffffu, vs, d));
                    float fs = 1.0f;
                    if (vs > S) {
                        // next power of two, kept where the inverse and 2^24 times it are normal numbers
                        const int e = min(max((int)(__float_as_uint(vs) >> 23) - 126, -100), 102);
                        const float was = S;
                        S = pow2i(e);
                        inv_S = pow2i(-e);
                        fs = was * inv_S;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float f[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float x = fmaxf(acc[n][k], acc[n][2 + k]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                            const float mn = fmaxf(m[n][k], x);
                            f[k] = mn == m[n][k] ? 1.0f : ex2f(m[n][k] - mn);
                            m[n][k] = mn;
                            l[n][k] *= f[k];
                            zs[n][k] *= f[k];
                            f[k] *= fs;
                        }
#pragma unroll
                        for (int j = 0; j < D / 16; ++j)
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[n][j][k] *= f[k & 1];
                    }
                }
                // ---- weights
                uint32_t pb[NT][2];
                const float vn[2] = {__uint_as_float(vp[0] << 16) * inv_S, __uint_as_float(vp[1] << 16) * inv_S};
                const float vz[2] = {__uint_as_float(vp[0] & 0xFFFF0000u), __uint_as_float(vp[1] & 0xFFFF0000u)};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float wgt[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        // a token that a row does not see adds nothing, whatever its pair holds
                        const bool none = acc[n][k] == -INFINITY;
                        const float p = none ? 0.0f : ex2f(acc[n][k] - m[n][k & 1]);
                        l[n][k & 1] += p;
                        zs[n][k & 1] += none ? 0.0f : p * vz[k >> 1];
                        wgt[k] = none ? 0.0f : p * vn[k >> 1];
                    }
                    pb[n][0] = movmatrix_t(pack_f16(wgt[0], wgt[1]));
                    pb[n][1] = movmatrix_t(pack_f16(wgt[2], wgt[3]));
                }
                // ---- output: dims x rows
                uint32_t va[W], vb[W];
                const uint8_t* sv = st + C::kCodes;
                if constexpr (W == 4) {
                    const uint4 u = *reinterpret_cast<const uint4*>(sv + v_chunk<D>(t, g));
                    const uint4 v = *reinterpret_cast<const uint4*>(sv + v_chunk<D>(t + 4, g));
                    va[0] = u.x, va[1] = u.y, va[2] = u.z, va[3] = u.w;
                    vb[0] = v.x, vb[1] = v.y, vb[2] = v.z, vb[3] = v.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(sv + v_chunk<D>(t, g >> 1) + (g & 1) * 8);
                    const uint2 v = *reinterpret_cast<const uint2*>(sv + v_chunk<D>(t + 4, g >> 1) + (g & 1) * 8);
                    va[0] = u.x, va[1] = u.y, vb[0] = v.x, vb[1] = v.y;
                }
#pragma unroll
                for (int w = 0; w < W; ++w) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t u = h ? va[w] >> 8 : va[w], v = h ? vb[w] >> 8 : vb[w];
                        const uint32_t a0 = u & 0x000F000Fu, a1 = u & 0x00F000F0u, a2 = v & 0x000F000Fu, a3 = v & 0x00F000F0u;
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_f16(o[n][w * 2 + h], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                    }
                }
            }
            __syncwarp();  // every lane has read the stage before it is filled again
        }

        // ---- join the four warps
        const float up = S * 16777216.0f;  // the codes' 2^-24 and the weights' scale
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], d);
                    zs[n][k] += __shfl_xor_sync(0xffffffffu, zs[n][k], d);
                }
                const int r = n * 8 + 2 * t + k;
                float* dst = join + (warp * RT + r) * C::kPitch;
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
                    *reinterpret_cast<float2*>(dst + 4 * (g * W + j / 2) + 2 * (j & 1)) =
                        make_float2(fmaf(o[n][j][k], up, zs[n][k]), fmaf(o[n][j][2 + k], up * 0.0625f, zs[n][k]));
                if (g == 0) {
                    join_ml[(warp * RT + r) * 2] = m[n][k];
                    join_ml[(warp * RT + r) * 2 + 1] = l[n][k];
                }
            }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == nt;
        float* part = a.part + ((int64_t)blockIdx.x * 2 + (unit == begin ? 0 : 1)) * C::kPart;
        for (int idx = tid; idx < rows * (D / 4); idx += kAttnThreads) {
            const int r = idx / (D / 4), d = (idx - r * (D / 4)) * 4;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) mx = fmaxf(mx, join_ml[(w * RT + r) * 2]);
            float sum = 0.0f;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) {
                const float mw = join_ml[(w * RT + r) * 2], lw = join_ml[(w * RT + r) * 2 + 1];
                if (mw == -INFINITY && lw == 0.0f) continue;  // the warp saw nothing
                const float f = ex2f(mw - mx);
                sum = fmaf(f, lw, sum);
                const float4 u = *reinterpret_cast<const float4*>(join + (w * RT + r) * C::kPitch + d);
                y.x = fmaf(f, u.x, y.x), y.y = fmaf(f, u.y, y.y), y.z = fmaf(f, u.z, y.z), y.w = fmaf(f, u.w, y.w);
            }
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int64_t rr = r0 + r;
                store_out(a, ((row0 + rr / a.G) * a.s.Hk * a.G + head * a.G + rr % a.G) * D + d, y, inv);
            } else {
                *reinterpret_cast<float4*>(part + r * D + d) = y;
                if (d == 0) part[RT * D + r * 2] = mx, part[RT * D + r * 2 + 1] = sum;
            }
        }
        __syncthreads();
        unit += t1 - t0;
        in_seq += t1 - t0;
    }
}

// Joins the partial results of row tiles that several blocks share: a warp per
// query row and head.
template <int D>
__global__ void __launch_bounds__(128) kv4_join_kernel(const Kv4AttnArgs a, int rt_rows, int64_t blocks) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int Hq = a.s.Hk * a.G;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t row = id / Hq;
    const int hq = (int)(id - row * Hq);
    int64_t b, i;
    if (row >= a.s.T || !kv4_find(a.s, row, b, i)) return;
    int64_t row0, n_rows;
    kv4_rows(a.s, b, row0, n_rows);
    const int head = hq / a.G;
    const int64_t rr = i * a.G + hq % a.G, n_rt = (n_rows * a.G + rt_rows - 1) / rt_rows;
    const int nt = max((kv4_len(a.s, b) + kAttnTokens - 1) / kAttnTokens, 1);
    const int64_t total = __ldcg(a.prefix + a.s.B);
    const int64_t u0 = __ldcg(a.prefix + b) + (head * n_rt + rr / rt_rows) * nt;
    // the block that holds unit u: the first `rem` blocks hold one more
    const int64_t each = total / blocks, rem = total % blocks;
    auto owner = [&](int64_t u) { return u < (each + 1) * rem ? u / (each + 1) : rem + (u - (each + 1) * rem) / each; };
    const int64_t c0 = owner(u0), c1 = owner(u0 + nt - 1);
    if (c0 == c1) return;
    const int r = (int)(rr % rt_rows);
    const int64_t size = (int64_t)rt_rows * (D + 2);
    auto slot = [&](int64_t c) { return a.part + (c * 2 + (attn_begin(total, blocks, c) < u0 ? 1 : 0)) * size; };
    float mx = -INFINITY;
    for (int64_t c = c0 + lane; c <= c1; c += 32) mx = fmaxf(mx, __ldcg(slot(c) + rt_rows * D + r * 2));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    constexpr int E = D / 32;
    float y[E], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.0f;
    for (int64_t c = c0; c <= c1; ++c) {
        const float* p = slot(c);
        const float mc = __ldcg(p + rt_rows * D + r * 2), lc = __ldcg(p + rt_rows * D + r * 2 + 1);
        if (mc == -INFINITY && lc == 0.0f) continue;
        const float f = ex2f(mc - mx);
        sum = fmaf(f, lc, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = fmaf(f, __ldcg(p + r * D + lane * E + e), y[e]);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t at = (row * Hq + hq) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (a.q_f32)
            static_cast<float*>(a.out)[at + e] = y[e] * inv;
        else
            static_cast<__nv_bfloat16*>(a.out)[at + e] = __float2bfloat16_rn(y[e] * inv);
    }
}

// 8 NT query rows per tile: the fewest that hold a sequence's rows on average.
static int attn_nt(int64_t B, int64_t T, int64_t G) {
    const int64_t rows = (T + B - 1) / B * G;
    return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}
static int attn_blocks(int nt) {  // blocks that the device holds at once
    const int sms = device_sm_count();
    return (sms > 0 ? sms : 148) * (nt == 1 ? 4 : nt == 2 ? 3 : 2);
}
static size_t attn_prefix_bytes(int64_t B) { return ((size_t)(B + 1) * 8 + 255) / 256 * 256; }
static size_t attn_workspace(int64_t B, int64_t T, int64_t G, int64_t D) {
    if (B == 0 || T == 0) return 0;
    const int nt = attn_nt(B, T, G);
    return attn_prefix_bytes(B) + (size_t)attn_blocks(nt) * 2 * (8 * nt) * (D + 2) * 4;
}

template <int D, int NT>
static cudaError_t launch_attn(const Kv4AttnArgs& a, cudaStream_t s) {
    using C = AttnCfg<D, NT>;
    static bool done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   C::kSmem);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) done[dev] = true;
    }
    const int blocks = attn_blocks(NT);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kAttnThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_decode_kernel<D, NT>, a);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned)((a.s.T * a.s.Hk * a.G + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D>, a, C::kRows, (int64_t)blocks);
}

}  // namespace pn

extern "C" {

size_t pn_kv4_attention_workspace_size(int64_t B, int64_t T, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
    if (B < 0 || T < 0 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1) return 0;
    return pn::attn_workspace(B, T, q_heads / kv_heads, head_dim);
}

int pn_kv4_attention(const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh, int q_dtype, int64_t q_heads,
                     const void* cache, int64_t n_pages, int64_t kv_heads, int64_t page, int64_t head_dim,
                     const int32_t* block_table, int64_t table_ld, int64_t table_w, const int32_t* seq_lens,
                     const int32_t* cu_q, int64_t B, int64_t T, float scale, void* out, void* workspace,
                     size_t workspace_bytes, void* stream) {
    pn::Kv4AttnArgs a{};
    if (int st = check_kv4("pn_kv4_attention", cache, n_pages, kv_heads, page, head_dim, block_table, table_ld, table_w,
                           seq_lens, cu_q, B, T, &a.s))
        return st;
    if (q_dtype != PN_F32 && q_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "pn_kv4_attention: dtype %d", q_dtype);
    if (q_heads < 1 || q_heads % kv_heads != 0 || q_heads > 65536)
        return fail(PN_ERR_SHAPE, "pn_kv4_attention: %lld query heads over %lld kv heads", (long long)q_heads,
                    (long long)kv_heads);
    if (T > 0 && B > 0 && (!q || !out)) return fail(PN_ERR_ARG, "pn_kv4_attention: null pointer");
    const size_t e = q_dtype == PN_F32 ? 4 : 2;
    if (!aligned(q, e) || !aligned(out, 16)) return fail(PN_ERR_ALIGN, "pn_kv4_attention: misaligned pointer");
    if ((T * q_heads + 3) / 4 > 0x7fffffff) return fail(PN_ERR_SHAPE, "pn_kv4_attention: too many rows");
    if (int st = check_device()) return st;
    if (T == 0 || B == 0) return ok();
    const size_t need = pn::attn_workspace(B, T, q_heads / kv_heads, head_dim);
    if (!workspace || workspace_bytes < need)
        return fail(PN_ERR_WORKSPACE, "pn_kv4_attention: workspace needs %zu bytes", need);
    if (!aligned(workspace, 256)) return fail(PN_ERR_ALIGN, "pn_kv4_attention: the workspace needs 256-byte alignment");
    if (n_pages == 0) a.s.table_w = 0;  // every length counts as zero
    a.q = q, a.q_f32 = q_dtype == PN_F32, a.q_sb = q_sb, a.q_sl = q_sl, a.q_sh = q_sh;
    const int64_t n = 16 / (int64_t)e;
    a.q_vec = aligned(q, 16) && q_sb % n == 0 && q_sl % n == 0 && q_sh % n == 0;
    a.cache = static_cast<const uint8_t*>(cache);
    a.G = (int)(q_heads / kv_heads);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.out = out;
    a.prefix = static_cast<int64_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + pn::attn_prefix_bytes(B));
    const cudaStream_t s = (cudaStream_t)stream;
    const int nt = pn::attn_nt(B, T, a.G);
    cudaError_t err;
    if (head_dim == 64)
        err = nt == 1 ? pn::launch_attn<64, 1>(a, s) : nt == 2 ? pn::launch_attn<64, 2>(a, s) : pn::launch_attn<64, 4>(a, s);
    else
        err = nt == 1 ? pn::launch_attn<128, 1>(a, s) : nt == 2 ? pn::launch_attn<128, 2>(a, s) : pn::launch_attn<128, 4>(a, s);
    return err == cudaSuccess ? ok() : cuda_fail(err, "pn_kv4_attention");
}

}  // extern "C"
