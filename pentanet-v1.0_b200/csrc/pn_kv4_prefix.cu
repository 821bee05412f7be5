// pn_kv4_prefix.cu -- causal attention of sequences that share long prefixes by groups, over
// the 4-bit paged cache (layout: pn_kv4.cu): a prefix's tokens are read, unpacked and
// multiplied once for the rows of all its sequences.
//
// Mathematics.  A row sees the prefix and then its own sequence; with (y_i, lse_i) the
// results over either part and the logarithms (base 2) of their softmax totals,
//   y = sum_i 2^(lse_i - M) y_i / sum_i 2^(lse_i - M).
// Three kernels: the rows over their own sequences (those of pn_kv4_attn.cu), the rows over
// the prefixes (here), and one that joins whatever partial results either left.
//
// The rows of a group are the first operand of tcgen05 products, 128 at a time, codes the
// second.  A code is brought to fp16 centred: with z' = z + 8 s
//   key   = (c - 8) s + z',   logit = scale * (sum_d q_d (c_d - 8) s + z' sum(q)),
// where (c - 8) s, at most eleven bits long, is exact in fp16 once the tile's largest s is
// scaled to [2^11, 2^12), and z' sum(q) is added in fp32;
//   value = (c - 8) s + z', rounded once to fp16 relative to a power of two that keeps
// the largest value seen in [2^12, 2^15).  Centred codes keep the sums small: with raw ones
// (0 .. 15, and z sum(p) taken off) outputs over 131071 tokens moved by 0.0015 of their norm, the
// tensor core's sums being truncated.  Weights are fp16 relative to a power of two
// that keeps a row's largest between 2^6 and 2^14; totals are fp32.
#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

// A row tile is two of the products' tiles of 128 rows, which share the tokens' operands
// ("paired"); where a tile has 128 rows or fewer, the two take alternate tokens instead.  A
// unit of work is 128 tokens of a paired tile, 256 of one that is not: two products either way.
//
// Seventeen warps: two groups of four for the softmax of either product (a thread has a row),
// four that spread keys, four that spread values, and one that issues the products.  The
// groups meet at mbarriers only, so that products, exponentials and unpacking of different
// steps run side by side.  Tensor memory, all 512 columns: for either product 128 of logits, the
// weights taking the place of the first half once they are read, and D of output.
template <int D>
struct PrefixCfg {
    static constexpr bool kPaired = true;
    static constexpr int kRows = 256, kTile = 128, kTokens = 128, kThreads = 17 * 32;
    static constexpr int kOp = 128 * D * 2;  // bytes of an operand: rows of 128 bytes, boxes of 64 columns
    static constexpr int kSmem = 6 * kOp + 1024;  // queries of two tiles, keys and values twice (+ alignment)
    static constexpr int kPart = kTile * (D + 1);  // floats of a tile's partial result: rows, then their logarithms
    static constexpr uint32_t kColO = 128, kColNext = 256, kCols = 512;
    static constexpr uint32_t kIdescS = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
    static constexpr uint32_t kIdescO = (1u << 4) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
};

// One segment: a run of units of one row tile.  (The fields that attn_note reads are AttnSeg's.)
struct PrefixSeg {
    uint32_t b, nt, t0, t1;
    int head, rows;
    int64_t row0, r0;
    bool paired;
    int tok0, end, steps;  // first token, one behind the last, steps of 128 tokens

    template <int D>
    __device__ __forceinline__ PrefixSeg(const Kv4AttnArgs& a, const PrefixCfg<D>&, uint32_t& seq, uint32_t& in_seq,
                                         uint32_t left) {
        using C = PrefixCfg<D>;
        uint32_t last_nt, n = attn_units<C>(a, seq, last_nt);
        while (in_seq >= n) {
            in_seq -= n;
            ++seq;
            n = attn_units<C>(a, seq, last_nt);
        }
        b = seq;
        int64_t n_rows;
        kv4_rows(a.s, b, row0, n_rows);
        const uint32_t q_rows = (uint32_t)n_rows * a.G, tiles = (q_rows + C::kRows - 1) / C::kRows;
        const int held = kv4_held(a.s, b);
        const uint32_t full_nt = max((held + C::kTokens - 1) / C::kTokens, 1), per_head = (tiles - 1) * full_nt + last_nt;
        head = (int)(in_seq / per_head);
        const uint32_t at = in_seq - head * per_head, tile = min(at / full_nt, tiles - 1);
        r0 = (int64_t)tile * C::kRows;
        rows = (int)min((uint32_t)C::kRows, q_rows - (uint32_t)r0);
        paired = rows > C::kTile;
        nt = tile == tiles - 1 ? last_nt : full_nt;
        t0 = at - tile * full_nt;
        t1 = min(nt, t0 + left);
        const int unit = paired ? C::kTokens : 2 * C::kTokens;
        tok0 = (int)t0 * unit;
        end = (int)min((int64_t)held, (int64_t)t1 * unit);
        steps = max((end - tok0 + C::kTokens - 1) / C::kTokens, 0);
        if (t0 == 0 && threadIdx.x == 0 && a.s.table_w > 0 && kv4_len(a.s, b) > held) record_status(PN_ERR_ARG);
    }
    __device__ __forceinline__ int products() const { return paired ? 2 * steps : steps; }
    // The products of either tile.
    __device__ __forceinline__ int products_of(int t) const { return paired ? steps : (steps + 1 - t) >> 1; }
};

// What the softmax needs to know of a step's tokens.
struct __align__(16) PrefixInfo {
    float kz[128];              // z' of the keys, in units of 2^ek
    __half vs[128], vz[128];    // s and z' of the values, in units of 2^ev
    uint32_t valid[4];          // bits: the token is there
    int ek, ev;
};
constexpr int kPrefixInfos = 4;

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
// The wait for it, tied to its registers.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                   "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 h2_of(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
// Pairs of codes, less eight each: of bits 0-3 (1024 + c as fp16) or 4-7 (64 + c) of either half.
__device__ __forceinline__ __half2 codes_lo(uint32_t w) {
    return __hadd2(h2_of((w & 0x000F000Fu) | 0x64006400u), h2_of(0xE408E408u));  // - 1032
}
__device__ __forceinline__ __half2 codes_hi(uint32_t w) {
    return __hadd2(h2_of((w & 0x00F000F0u) | 0x54005400u), h2_of(0xD480D480u));  // - 72
}
// W consecutive words of codes, zeros where there is no page.
template <int W>
__device__ __forceinline__ void ldg_words(const uint8_t* p, bool there, uint32_t (&w)[W]) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0;
    if (!there) return;
    if constexpr (W == 4) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = u.x, w[1] = u.y;
    }
}
// Where the pieces of 16 tokens of a step are: lane 8 i + j holds piece j of step (base + i), four steps at once.
struct PrefixPages {
    AttnPages pages;
    __device__ __forceinline__ void look_up(const Kv4AttnArgs& a, const PrefixSeg& sg, int64_t block, int step) {
        const int tok = sg.tok0 + (step + (int)(threadIdx.x >> 3 & 3)) * 128 + (int)(threadIdx.x & 7) * 16;
        pages.look_up(a, sg.b, sg.head, block, tok, tok < sg.end);
    }
    __device__ __forceinline__ const uint8_t* page(int step, int piece) const {
        return reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, pages.addr, (step & 3) * 8 + piece));
    }
    __device__ __forceinline__ int off(int step, int piece) const {
        return __shfl_sync(0xffffffffu, pages.off, (step & 3) * 8 + piece);
    }
};

template <int D>
__global__ void __launch_bounds__(PrefixCfg<D>::kThreads, 1) kv4_prefix_kernel(const Kv4AttnArgs a) {
    using C = PrefixCfg<D>;
    constexpr int W = D / 32;  // words of codes that a spreading thread loads at once
    extern __shared__ uint8_t smem_base[];
    __shared__ PrefixInfo info[kPrefixInfos];
    __shared__ __align__(16) __half ks[128];
    __shared__ uint32_t red[2][4];
    __shared__ uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2], o_full[2],
        info_full[kPrefixInfos];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    uint8_t* qop = smem_base + (1024 - smem_u32(smem_base) % 1024) % 1024;
    uint8_t* kop = qop + 2 * C::kOp;
    uint8_t* vop = kop + 2 * C::kOp;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;");
    // (tensor memory is taken only when the grid before this one is done: it may hold some)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 16) {
        tmem_alloc(&s_tmem, C::kCols);
        tmem_relinquish();
    }
    if (tid == 0) {
        mbar_init(&q_full, 256);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 128);
            mbar_init(&v_full[i], 128);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < kPrefixInfos; ++i) mbar_init(&info_full[i], 128);
        fence_barrier_init();
        s_abort = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = s_tmem;
    volatile int* abort = &s_abort;
    const int64_t block = (int64_t)a.s.page * (D / 2 + 4);

    const AttnRun run = attn_plan<C>(a);
    uint32_t seq = run.seq, in_seq = run.in_seq;
    uint32_t step0 = 0;              // steps of the segments before
    uint32_t done[2] = {0, 0};       // products of either tile in them
    uint32_t some = 0, ends[2] = {0, 0};  // segments with products, of any and of either tile
    for (uint32_t unit = run.begin; unit < run.end;) {
        const PrefixSeg sg(a, C{}, seq, in_seq, run.end - unit);
        if (warp < 8) {
            // ---- softmax: tile t's row `row` is query row r
            const int t = warp >> 2, row = (warp & 3) * 32 + lane, r = (sg.paired ? t * 128 : 0) + row;
            const bool mine = r < sg.rows;
            const uint32_t ts = tm + t * C::kColNext + ((uint32_t)((warp & 3) * 32) << 16), to = ts + C::kColO;
            float ca = 0.0f, cb = 0.0f;
            if (sg.steps > 0) {
                // the row's query, scaled, as an operand (dims of a word of codes in their order there)
                const char* q = nullptr;
                if (mine) q = static_cast<const char*>(a.q) + attn_query(a, sg.b, sg.row0, sg.r0, sg.head, r) * (a.q_f32 ? 4 : 2);
                auto load = [&](int i, float (&v)[8]) {
                    if (!mine) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
                    } else if (a.q_f32) {
                        kv4_load8(reinterpret_cast<const float*>(q) + i * 8, a.q_vec, v);
                    } else {
                        kv4_load8(reinterpret_cast<const __nv_bfloat16*>(q) + i * 8, a.q_vec, v);
                    }
                };
                float amax = 0.0f, v[8];
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    load(i, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[j]));
                }
                const int e = query_exponent(amax);
                const float up = pow2i(e);
#pragma unroll 4
                for (int i = 0; i < D / 8; ++i) {
                    load(i, v);
                    uint32_t p[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        p[k] = pack_f16(v[k] * up, v[k + 4] * up);
                        const float2 f = __half22float2(h2_of(p[k]));
                        cb += f.x + f.y;
                    }
                    if (sg.paired || t == 0)
                        *reinterpret_cast<uint4*>(qop + t * C::kOp + (i >> 3) * 16384 + row * 128 + (((i & 7) ^ (row & 7)) * 16)) =
                            make_uint4(p[0], p[1], p[2], p[3]);
                }
                ca = a.scale_log2 * pow2i(-e);
                proxy_fence();
                mbar_arrive(&q_full);
            }
            float neg_r = 0.0f;  // the row's reference is 2^-neg_r; a whole number
            bool unset = true;   // nothing was seen yet
            float2 l2 = make_float2(0.0f, 0.0f);
            int ev = 0;
            const bool some_rows = __any_sync(0xffffffffu, mine);
            const int products = sg.products();
            // Multiplies the output so far, and the weights of the step's first `chunks` runs of 32 tokens, by f.
            auto rescale = [&](float f, bool output, int chunks) {
                if (output) {
#pragma unroll 1
                    for (int h = 0; h < D / 16; ++h) {
                        uint32_t u[16];
                        tmem_ld16(to + h * 16, u);
                        tmem_wait_ld16(u);
#pragma unroll
                        for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(__uint_as_float(u[k]) * f);
                        tmem_st16(to + h * 16, u);
                    }
                }
                const __half2 f2 = __float2half2_rn(f);
#pragma unroll 1
                for (int h = 0; h < chunks; ++h) {
                    uint32_t u[16];
                    tmem_ld16(ts + h * 16, u);
                    tmem_wait_ld16(u);
#pragma unroll
                    for (int k = 0; k < 16; ++k) u[k] = h2_bits(__hmul2(h2_of(u[k]), f2));
                    tmem_st16(ts + h * 16, u);
                }
                tmem_wait_st();
            };
            for (int j = t; j < products; j += 2) {
                const uint32_t step = step0 + (sg.paired ? j >> 1 : j);
                const PrefixInfo& in = info[step % kPrefixInfos];
                mbar_wait(&info_full[step % kPrefixInfos], (step / kPrefixInfos) & 1, abort);
                mbar_wait(&s_full[t], (done[t] + (j >> 1)) & 1, abort);
                __syncwarp();
                tc_fence_after();
                if (some_rows) {
                    if (in.ev != ev) {  // (the same for all rows)
                        if (j >= 2) rescale(pow2i(max(ev - in.ev, -126)), true, 0);
                        ev = in.ev;
                    }
                    const float cs = ca * pow2i(in.ek);
                    const bool full = (in.valid[0] & in.valid[1] & in.valid[2] & in.valid[3]) == 0xffffffffu;
                    uint32_t next[2][16];  // the next 32 logits, asked for as the registers of these come free
                    tmem_ld16(ts, next[0]);
                    tmem_ld16(ts + 16, next[1]);
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        float2 x[16];
                        tmem_wait_ld16(next[0]);
                        tmem_wait_ld16(next[1]);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            x[k] = make_float2(__uint_as_float(next[k >> 3][2 * (k & 7)]), __uint_as_float(next[k >> 3][2 * (k & 7) + 1]));
                        const float2 cb2 = make_float2(cb, cb), cs2 = make_float2(cs, cs);
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            const float4 z = *reinterpret_cast<const float4*>(in.kz + c * 32 + 2 * k);
                            x[k] = fma2(make_float2(z.x, z.y), cb2, x[k]);
                            x[k + 1] = fma2(make_float2(z.z, z.w), cb2, x[k + 1]);
                        }
                        if (!full) {
                            const uint32_t bits = in.valid[c];
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                if (!(bits >> (2 * k) & 1)) x[k].x = -INFINITY;
                                if (!(bits >> (2 * k + 1) & 1)) x[k].y = -INFINITY;
                            }
                        }
                        float top = -INFINITY;
#pragma unroll
                        for (int k = 0; k < 16; ++k) top = fmaxf(top, fmaxf(x[k].x, x[k].y));
                        top = fmaf(top, cs, neg_r);
                        if (__any_sync(0xffffffffu, top > 14.0f || unset)) {  // seldom
                            float f = 1.0f;
                            if (top > 14.0f || (unset && top > -INFINITY)) {
                                const float by = ceilf(top) - 6.0f;  // the largest weight so far becomes 2^5 to 2^6
                                neg_r -= by;
                                if (!unset) f = ex2f(-by);
                                unset = false;
                            }
                            l2 = mul2(l2, make_float2(f, f));
                            if (__any_sync(0xffffffffu, f != 1.0f)) rescale(f, j >= 2, c);
                        }
                        const float2 r2 = make_float2(neg_r, neg_r);
                        uint32_t pw[16];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int k = 8 * h; k < 8 * h + 8; ++k) {
                                const float2 d = fma2(x[k], cs2, r2);
                                const float2 p = make_float2(ex2f(d.x), ex2f(d.y));
                                l2 = add2(l2, p);
                                pw[k] = pack_f16(p.x, p.y);
                            }
                            if (c < 3) tmem_ld16(ts + (c + 1) * 32 + h * 16, next[h]);
                        }
                        tmem_st16(ts + c * 16, pw);
                    }
                    tmem_wait_st();
                }
                tc_fence_before();
                mbar_arrive(&p_full[t]);
            }
            // ---- results
            const bool whole = sg.t0 == 0 && sg.t1 == sg.nt, any = sg.products_of(t) > 0;
            if (any) {
                mbar_wait(&o_full[t], ends[t] & 1, abort);
                __syncwarp();
                tc_fence_after();
            }
            const float l = l2.x + l2.y, inv = l == 0.0f ? 0.0f : pow2i(ev) / l;
            const uint32_t rr = (uint32_t)sg.r0 + r, ri = rr / a.G;
            const int64_t out_row = ((sg.row0 + ri) * a.s.Hk + sg.head) * a.G + rr - ri * a.G + (sg.paired ? 0 : t * a.s.T * a.s.Hk * a.G);
            float* part = a.part + (((int64_t)blockIdx.x * 2 + (unit == run.begin ? 0 : 1)) * 2 + t) * C::kPart;
            float* y = whole ? static_cast<float*>(a.out) + out_row * D : part + row * D;
            if (any && some_rows) {
#pragma unroll 1
                for (int h = 0; h < D / 32; ++h) {
                    uint32_t u[32];
                    tmem_ld32(to + h * 32, u);
                    tmem_wait_ld32(u);
                    if (mine) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            *reinterpret_cast<float4*>(y + h * 32 + k) =
                                make_float4(__uint_as_float(u[k]) * inv, __uint_as_float(u[k + 1]) * inv, __uint_as_float(u[k + 2]) * inv,
                                            __uint_as_float(u[k + 3]) * inv);
                    }
                }
            }
            if (mine) (whole ? a.lse[out_row] : part[C::kTile * D + row]) = !any ? -INFINITY : attn_lse(-neg_r, l);
            if (tid == 0) attn_note(a, run, sg, unit);
            tc_fence_before();
        } else if (warp < 12) {
            // ---- keys, and what is to be known of a step's tokens
            const int k = tid - 256, of = k >> 2;  // a token's four quarters side by side
            PrefixPages pages;
            uint32_t ahead[4][W], kp = 0, vp = 0;
            bool there = false;
            auto fetch = [&](int i) {  // step i, if there is one
                if (i >= sg.steps) return;
                if ((i & 3) == 0) pages.look_up(a, sg, block, i);
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const int piece = 2 * p + (of >> 4);
                    const uint8_t* at = pages.page(i, piece);
                    const int off = pages.off(i, piece);
                    ldg_words<W>(at + (off + (of & 15)) * (D / 2) + (k & 3) * W * 4, at != nullptr, ahead[p]);
                }
                const uint8_t* at = pages.page(i, k >> 4);
                const int off = pages.off(i, k >> 4);
                there = at && sg.tok0 + i * 128 + k < sg.end;
                kp = vp = 0;
                if (there) {
                    at += (uint32_t)a.s.page * (D / 2) + (off + (k & 15)) * 4;
                    kp = __ldg(reinterpret_cast<const uint32_t*>(at));
                    vp = __ldg(reinterpret_cast<const uint32_t*>(at + block));
                }
            };
            fetch(0);
            int ev = 0;
            for (int i = 0; i < sg.steps; ++i) {
                const uint32_t step = step0 + i, b = step & 1;
                uint32_t w[4][W];
#pragma unroll
                for (int p = 0; p < 4; ++p)
#pragma unroll
                    for (int c = 0; c < W; ++c) w[p][c] = ahead[p][c];
                const float ksf = pair_lo(kp), kzf = fmaf(8.0f, ksf, pair_hi(kp)), vsf = pair_lo(vp), vzf = pair_hi(vp);
                const float loud = fmaxf(0.0f, fmaxf(fabsf(vzf), fabsf(fmaf(15.0f, vsf, vzf))));  // (a NaN does not count)
                // (a zero far above the scale counts too, so that it stays a number in units of the scale)
                const int kze = kzf == kzf ? (int)(__float_as_uint(fabsf(kzf)) >> 23) - 20 : 0;
                const uint32_t ke = __reduce_max_sync(0xffffffffu, (uint32_t)max((int)(__float_as_uint(ksf) >> 23), kze));
                const uint32_t ve = __reduce_max_sync(0xffffffffu, __float_as_uint(loud) >> 23);
                const uint32_t bits = __ballot_sync(0xffffffffu, there);
                fetch(i + 1);
                if (lane == 0) red[0][warp - 8] = ke, red[1][warp - 8] = ve;
                mbar_wait(&k_empty[b], ((step >> 1) & 1) ^ 1, abort);
                asm volatile("bar.sync 1, 128;" ::: "memory");
                const int ke4 = max(max(red[0][0], red[0][1]), max(red[0][2], red[0][3]));
                const int ve4 = max(max(red[1][0], red[1][1]), max(red[1][2], red[1][3]));
                const int ek = min(max(ke4 - 127, -100), 126) - 11, want = min(max(ve4 - 127, -100), 126) - 14;
                if (i == 0 || want > ev) ev = want + 2;
                const float kd = pow2i(-ek), vd = pow2i(-ev);
                PrefixInfo& in = info[step % kPrefixInfos];
                in.kz[k] = kzf * kd;
                in.vs[k] = __float2half_rn(vsf * vd);
                in.vz[k] = __float2half_rn(fmaf(8.0f, vsf, vzf) * vd);
                ks[k] = __float2half_rn(ksf * kd);
                if (lane == 0) in.valid[warp - 8] = bits;
                if (k == 0) in.ek = ek, in.ev = ev;
                mbar_arrive(&info_full[step % kPrefixInfos]);
                asm volatile("bar.sync 1, 128;" ::: "memory");
                uint8_t* op = kop + b * C::kOp;
                const bool swap = W == 4 && (k & 2);  // so that the eight lanes of a store's phase meet different banks
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const int tok = p * 32 + of;
                    const __half2 s2 = __half2half2(ks[tok]);
#pragma unroll
                    for (int c = 0; c < W; ++c) {
                        const int j = (k & 3) * W + (swap ? c ^ 2 : c);
                        const uint32_t x = swap ? w[p][c ^ (W / 2)] : w[p][c], y = x >> 8;
                        *reinterpret_cast<uint4*>(op + (j >> 3) * 16384 + tok * 128 + (((j & 7) ^ (tok & 7)) * 16)) =
                            make_uint4(h2_bits(__hmul2(codes_lo(x), s2)), h2_bits(__hmul2(codes_hi(x), s2)),
                                       h2_bits(__hmul2(codes_lo(y), s2)), h2_bits(__hmul2(codes_hi(y), s2)));
                    }
                }
                proxy_fence();
                mbar_arrive(&k_full[b]);
            }
        } else if (warp < 16) {
            // ---- values: eight tokens, W words of four dims
            const int q = (lane & 7) + 8 * (warp & 1), col = (lane >> 3) + 4 * ((warp - 12) >> 1);
            PrefixPages pages;
            uint32_t ahead[4][W];
            auto fetch = [&](int i) {
                if (i >= sg.steps) return;
                if ((i & 3) == 0) pages.look_up(a, sg, block, i);
                const uint8_t* at = pages.page(i, q >> 1);
                const int off = pages.off(i, q >> 1);
#pragma unroll
                for (int p = 0; p < 4; ++p)
                    ldg_words<W>(at + block + ((off >> 1) + 4 * (q & 1) + p) * D + col * W * 4, at != nullptr, ahead[p]);
            };
            fetch(0);
            for (int i = 0; i < sg.steps; ++i) {
                const uint32_t step = step0 + i, b = step & 1;
                const PrefixInfo& in = info[step % kPrefixInfos];
                uint32_t w[4][W];
#pragma unroll
                for (int p = 0; p < 4; ++p)
#pragma unroll
                    for (int c = 0; c < W; ++c) w[p][c] = ahead[p][c];
                fetch(i + 1);
                mbar_wait(&info_full[step % kPrefixInfos], (step / kPrefixInfos) & 1, abort);
                mbar_wait(&v_empty[b], ((step >> 1) & 1) ^ 1, abort);
                const uint4 s = *reinterpret_cast<const uint4*>(in.vs + 8 * q), z = *reinterpret_cast<const uint4*>(in.vz + 8 * q);
                const __half2 s2[4] = {h2_of(s.x), h2_of(s.y), h2_of(s.z), h2_of(s.w)};
                const __half2 z2[4] = {h2_of(z.x), h2_of(z.y), h2_of(z.z), h2_of(z.w)};
                uint8_t* op = vop + b * C::kOp + (q >> 3) * (D * 128);
#pragma unroll
                for (int c = 0; c < W; ++c) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int r = 4 * (col * W + c) + n;
                        uint32_t u[4];
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            const uint32_t x = n & 2 ? w[p][c] >> 8 : w[p][c];
                            u[p] = h2_bits(__hfma2(n & 1 ? codes_hi(x) : codes_lo(x), s2[p], z2[p]));
                        }
                        *reinterpret_cast<uint4*>(op + r * 128 + (((q & 7) ^ (r & 7)) * 16)) = make_uint4(u[0], u[1], u[2], u[3]);
                    }
                }
                proxy_fence();
                mbar_arrive(&v_full[b]);
            }
        } else if (sg.steps > 0) {
            // ---- products
            const uint32_t q_lo = desc_lo(qop), k_lo = desc_lo(kop), v_lo = desc_lo(vop);
            const int products = sg.products();
            auto logits = [&](int j) {
                const uint32_t step = step0 + (sg.paired ? j >> 1 : j), b = step & 1, t = j & 1;
                if (!sg.paired || t == 0) warp_wait(&k_full[b], (step >> 1) & 1, abort);
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < D / 64; ++h)
                    mma4_ss_warp(tm + t * C::kColNext, q_lo + ((sg.paired ? t * C::kOp : 0) + h * 16384 >> 4),
                                 k_lo + (b * C::kOp + h * 16384 >> 4), C::kIdescS, h);
                tc_commit_warp(&s_full[t]);
                if (!sg.paired || t == 1) tc_commit_warp(&k_empty[b]);
            };
            warp_wait(&q_full, some & 1, abort);
            logits(0);
            if (products > 1) logits(1);
            for (int j = 0; j < products; ++j) {
                const uint32_t step = step0 + (sg.paired ? j >> 1 : j), b = step & 1, t = j & 1;
                if (!sg.paired || t == 0) warp_wait(&v_full[b], (step >> 1) & 1, abort);
                warp_wait(&p_full[t], (done[t] + (j >> 1)) & 1, abort);
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    mma4_ts_warp(tm + t * C::kColNext + C::kColO, tm + t * C::kColNext + h * 32,
                                 v_lo + (b * C::kOp + h * (D * 128) >> 4), C::kIdescO, j >= 2 || h);
                if (!sg.paired || t == 1) tc_commit_warp(&v_empty[b]);
                // (the next logits of this tile take the place of the weights just read: products run in order)
                if (j + 2 < products)
                    logits(j + 2);
                else
                    tc_commit_warp(&o_full[t]);
            }
        }
        some += sg.steps > 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            done[t] += sg.products_of(t);
            ends[t] += sg.products_of(t) > 0;
        }
        step0 += sg.steps;
        unit += sg.t1 - sg.t0;
        in_seq += sg.t1 - sg.t0;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        tmem_dealloc(tm, C::kCols);
    }
}

// ---- joining ----------------------------------------------------------------

struct Kv4MergeArgs {
    Kv4Seq s;                  // the sequences
    const int32_t* grp;        // shares of the prefixes, or null
    int64_t P;
    int G;
    const float* y[3];         // whole results: own, and of either product over a prefix
    const float* lse[3];
    const Kv4Where* where[2];  // own, prefix
    const float* part[2];
    int tile;                  // rows of the own pass's row tiles
    void* out;
    int out_f32;
    int zero_rest;             // rows of no sequence get zeros
};
constexpr int kMergeWarps = 8;

// A warp per row and head: the lanes look up the totals of up to 32 partial results at
// once, then all read each result in turn, with its weight.
template <int D>
__global__ void __launch_bounds__(kMergeWarps * 32) kv4_merge_kernel(const Kv4MergeArgs a) {
    constexpr int E = D / 32;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, H = a.s.Hk * a.G, h = blockIdx.y * kMergeWarps + (threadIdx.x >> 5);
    const int64_t row = blockIdx.x;
    bool falls = false;  // nothing was computed
    if (a.s.cu)
        for (int b = threadIdx.x; b < a.s.B; b += kMergeWarps * 32) falls |= __ldg(a.s.cu + b + 1) < __ldg(a.s.cu + b);
    if (a.grp)
        for (int b = threadIdx.x; b < a.P; b += kMergeWarps * 32) falls |= __ldg(a.grp + b + 1) < __ldg(a.grp + b);
    falls = __syncthreads_or(falls);
    if (h >= H) return;
    const int64_t at = row * H + h;
    int64_t b, i;
    const bool found = !falls && kv4_find(a.s, row, b, i);
    if (!found && !a.zero_rest) return;
    float mx = -INFINITY, sum = 0.0f, y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.0f;
    if (found) {
        const int hk = h / a.G, gq = h - hk * a.G;
        // own results
        const int64_t r = i * a.G + gq, r0 = r / a.tile * a.tile;
        const Kv4Where own = a.where[0][((row - i + r0 / a.G) * a.s.Hk + hk) * a.G + r0 % a.G];
        const int n_own = own.last < 0 ? 1 : own.last - own.first + 1;
        // the prefix's
        Kv4Where pre = {};
        int n_pre = 0, slots = 1, slot = 0;
        int64_t pr = 0;
        Kv4Seq p = a.s;
        p.B = a.P, p.grouped = a.s.B, p.grp = a.grp;
        int64_t g = -1;
        if (!a.grp) {
            g = b / (a.s.B / a.P);
        } else {
            int64_t lo = 0, hi = a.P;  // the last g with grp[g] <= b
            while (hi - lo > 1) {
                const int64_t mid = (lo + hi) / 2;
                if (__ldg(a.grp + mid) <= b)
                    lo = mid;
                else
                    hi = mid;
            }
            if (b >= __ldg(a.grp + lo) && b < __ldg(a.grp + lo + 1)) g = lo;
        }
        if (g >= 0) {
            int64_t first, n;
            kv4_rows(p, g, first, n);
            pr = (row - first) * a.G + gq;
            const int64_t t0 = pr / 256 * 256;
            pre = a.where[1][((first + t0 / a.G) * a.s.Hk + hk) * a.G + t0 % a.G];
            pr -= t0;
            if (n * a.G - t0 > 128) {
                slot = (int)(pr >> 7);
                pr &= 127;
            } else {
                slots = 2;
            }
            n_pre = (pre.last < 0 ? 1 : pre.last - pre.first + 1) * slots;
        }
        for (int base = 0; base < n_own + n_pre; base += 32) {
            const int n = min(n_own + n_pre - base, 32), j = base + lane;
            const float* from = nullptr;
            float m = -INFINITY, l = 0.0f;
            if (j < n_own) {
                if (own.last < 0) {
                    from = a.y[0] + at * D;
                    m = a.lse[0][at], l = 1.0f;
                } else {
                    const int c = own.first + j;
                    const float* p0 = a.part[0] + ((int64_t)c * 2 + (j == 0 ? own.first_slot : 0)) * a.tile * (D + 2);
                    from = p0 + (r - r0) * D;
                    const float2 ml = *reinterpret_cast<const float2*>(p0 + a.tile * D + (r - r0) * 2);
                    m = ml.x, l = ml.y;
                }
            } else if (lane < n) {
                const int k = (j - n_own) / slots, t = slots == 2 ? (j - n_own) & 1 : slot;
                if (pre.last < 0) {
                    const int which = slots == 2 ? t : 0;
                    from = a.y[1 + which] + at * D;
                    m = a.lse[1 + which][at];
                } else {
                    const float* p0 = a.part[1] + (((int64_t)(pre.first + k) * 2 + (k == 0 ? pre.first_slot : 0)) * 2 + t) * PrefixCfg<D>::kPart;
                    from = p0 + pr * D;
                    m = p0[128 * D + pr];
                }
                l = 1.0f;
            }
            if (m == -INFINITY) l = 0.0f;
            if (l == 0.0f) m = -INFINITY;  // (a total of 0: nothing was seen)
            float top = m;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (top == -INFINITY) top = __any_sync(0xffffffffu, m != m) ? 0.0f : top;  // (totals that are NaN)
            if (top == -INFINITY) continue;
            const float mn = fmaxf(mx, top), f = ex2f(mx - mn), w = l == 0.0f ? 0.0f : ex2f(m - mn);
            float lw = l * w;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
            sum = fmaf(sum, f, lw);
            mx = mn;
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] *= f;
            const uint32_t some = __ballot_sync(0xffffffffu, l != 0.0f);
#pragma unroll 4
            for (int k = 0; k < n; ++k) {
                const float wk = __shfl_sync(0xffffffffu, w, k);
                const float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(from), k));
                if (!(some >> k & 1)) continue;
                float u[E];
                if constexpr (E == 4) {
                    const float4 v = reinterpret_cast<const float4*>(src)[lane];
                    u[0] = v.x, u[1] = v.y, u[2] = v.z, u[3] = v.w;
                } else {
                    const float2 v = reinterpret_cast<const float2*>(src)[lane];
                    u[0] = v.x, u[1] = v.y;
                }
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = fmaf(wk, u[e], y[e]);
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (a.out_f32)
            static_cast<float*>(a.out)[at * D + lane * E + e] = y[e] * inv;
        else
            static_cast<__nv_bfloat16*>(a.out)[at * D + lane * E + e] = __float2bfloat16_rn(y[e] * inv);
    }
}

// Parts of the workspace.
struct PrefixLayout {
    size_t y, lse, where[2], attn, part, total;
    PrefixLayout(int64_t B, int64_t T, int64_t Hk, int64_t G, int64_t D) {
        const size_t rows = (size_t)T * Hk * G;
        y = 0;  // of the own pass, and of either product over the prefixes
        lse = y + round256(3 * rows * D * 4);
        where[0] = lse + round256(3 * rows * 4);
        where[1] = where[0] + round256(rows * sizeof(Kv4Where));
        attn = where[1] + round256(rows * sizeof(Kv4Where));
        part = attn + round256(attn_workspace(B, T, Hk, G, D));
        total = part + (size_t)sm_count() * 4 * 128 * (D + 1) * 4;
    }
};

template <int D>
static cudaError_t launch_prefix(const Kv4AttnArgs& p, const Kv4MergeArgs& m, cudaStream_t s) {
    using C = PrefixCfg<D>;
    static std::atomic<bool> set[64];  // false at first
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_prefix_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)sm_count());
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_prefix_kernel<D>, p);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned)m.s.T, (unsigned)((m.s.Hk * m.G + kMergeWarps - 1) / kMergeWarps));
    cfg.blockDim = dim3(kMergeWarps * 32);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, kv4_merge_kernel<D>, m);
}

}  // namespace pn

extern "C" {

size_t pn_kv4_prefix_attention_workspace_size(int64_t B, int64_t T, int64_t n_prefixes, int64_t q_heads, int64_t kv_heads,
                                              int64_t head_dim) {
    if (B < 1 || T < 1 || n_prefixes < 0 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1) return 0;
    if (n_prefixes == 0) return pn_kv4_attention_workspace_size(B, T, q_heads, kv_heads, head_dim);
    return pn::PrefixLayout(B, T, kv_heads, q_heads / kv_heads, head_dim).total;
}

int pn_kv4_prefix_attention(const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh, int q_dtype, int64_t q_heads,
                            const void* cache, int64_t n_pages, int64_t kv_heads, int64_t page, int64_t head_dim,
                            const int32_t* block_table, int64_t table_ld, int64_t table_w, const int32_t* seq_lens,
                            const int32_t* cu_q, int64_t B, int64_t T, const int32_t* prefix_table, int64_t prefix_ld,
                            int64_t prefix_w, const int32_t* prefix_lens, const int32_t* cu_prefix, int64_t n_prefixes,
                            float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "pn_kv4_prefix_attention";
    pn::Kv4AttnArgs a{}, p{};
    if (int st = check_kv4(name, cache, n_pages, kv_heads, page, head_dim, block_table, table_ld, table_w, seq_lens, cu_q, B, T,
                           &a.s))
        return st;
    if (int st = check_attn(name, q, q_sb, q_sl, q_sh, q_dtype, q_heads, cache, scale, out, &a)) return st;
    // (the rows of a prefix are any number of sequences': cu_q or not is the sequences' matter)
    if (int st = check_kv4(name, cache, n_pages, kv_heads, page, head_dim, prefix_table, prefix_ld, prefix_w, prefix_lens, cu_prefix,
                           n_prefixes, n_prefixes > 0 ? T / n_prefixes * n_prefixes : T, &p.s))
        return st;
    if (!cu_prefix && n_prefixes > 0 && B % n_prefixes != 0)
        return fail(PN_ERR_SHAPE, "%s: %lld sequences over %lld prefixes need cu_prefix", name, (long long)B, (long long)n_prefixes);
    if (T > 0 && B > 0 && n_prefixes > 0 && (!prefix_lens || (!prefix_table && prefix_w > 0)))
        return fail(PN_ERR_ARG, "%s: null pointer", name);
    if (n_prefixes == 0)
        return pn_kv4_attention(q, q_sb, q_sl, q_sh, q_dtype, q_heads, cache, n_pages, kv_heads, page, head_dim, block_table,
                                table_ld, table_w, seq_lens, cu_q, B, T, scale, out, workspace, workspace_bytes, stream);
    if (int st = check_attn_units(name, a.s, a.G, table_w * page)) return st;
    const pn::Kv4Seq own = a.s;
    p.s.T = T, p.s.cu = cu_q, p.s.L = own.L, p.s.grouped = B, p.s.grp = cu_prefix;
    if (int st = check_attn_units(name, p.s, a.G, prefix_w * page)) return st;
    if (int st = check_device()) return st;
    if (T == 0 || B == 0) return ok();
    const pn::PrefixLayout lay(B, T, kv_heads, a.G, head_dim);
    if (!workspace || workspace_bytes < lay.total) return fail(PN_ERR_WORKSPACE, "%s: workspace needs %zu bytes", name, lay.total);
    if (!aligned(workspace, 256)) return fail(PN_ERR_ALIGN, "%s: the workspace needs 256-byte alignment", name);
    const cudaStream_t s = (cudaStream_t)stream;
    char* ws = static_cast<char*>(workspace);
    const int64_t rows = T * q_heads;
    float *y = reinterpret_cast<float*>(ws + lay.y), *lse = reinterpret_cast<float*>(ws + lay.lse);
    a.grp = cu_prefix, a.n_grp = (int)n_prefixes;
    a.out_f32 = 1;
    const pn::Kv4Seq prefixes = p.s;
    p = a;
    // the rows over their own sequences
    a.out = y, a.lse = lse, a.where = reinterpret_cast<pn::Kv4Where*>(ws + lay.where[0]);
    const pn::AttnKind kind = pn::attn_kind(B, T, kv_heads, a.G);
    cudaError_t err = pn::attn_pass(a, kind, head_dim, ws + lay.attn, s);
    if (err != cudaSuccess) return cuda_fail(err, name);
    // and over the prefixes
    p.s = prefixes;
    p.q_l = cu_q ? 0 : own.L;
    p.out = y + rows * head_dim, p.lse = lse + rows, p.where = reinterpret_cast<pn::Kv4Where*>(ws + lay.where[1]);
    p.part = reinterpret_cast<float*>(ws + lay.part);
    pn::Kv4MergeArgs m{};
    m.s = own, m.grp = cu_prefix, m.P = n_prefixes, m.G = a.G;
    for (int i = 0; i < 3; ++i) m.y[i] = y + i * rows * head_dim, m.lse[i] = lse + i * rows;
    m.where[0] = a.where, m.where[1] = p.where;
    m.part[0] = a.part, m.part[1] = p.part;
    constexpr int tile[4] = {8, 16, 64, 128};
    m.tile = tile[kind];
    m.out = out, m.out_f32 = q_dtype == PN_F32;
    err = head_dim == 64 ? pn::launch_prefix<64>(p, m, s) : pn::launch_prefix<128>(p, m, s);
    return err == cudaSuccess ? ok() : cuda_fail(err, name);
}

}  // extern "C"
