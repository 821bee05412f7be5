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
// to 2^-28 of the largest (fp32 queries are rounded to 11 bits).  The weights
// p_t * s_v are rounded to fp16 (11 bits, more than the bf16 output keeps)
// relative to the largest s_v that the row has seen; sums, the softmax's maximum
// and total, and the z term are fp32.
//
// Long walks.  sum p s_v c grows with the tokens while the result is its small
// difference from sum p z_v, and the tensor core cuts off what its products lose
// against a large sum: all one way, as codes and weights are not negative.  Left
// to grow over 131072 tokens the sums put the result off by 6 (decode kernel) to
// 25 % (tcgen05) of its norm, normal random data.  So the sums are kept near zero:
// every kCentre steps what they have reached (the middle one of three dims, so that
// a loud dim does not lead the others away) is taken out of a row's sums and joins,
// with the z term of these steps, a base that stays small, as its two parts cancel
// in one fma.  To 262144 tokens the error is now that of the rounded weights alone,
// 5e-4 to 8e-4 of the result's norm in every kernel.  What a product of 16 tokens
// loses against the sums that are left is up to 2^-24 of the result: over a million
// tokens that one block walks the error is 6e-4 to 9e-4 (decode), 17e-4 (chunk) and
// 27e-4 (tcgen05).  (With the middle
// code, 7.5, taken out of each value instead, which the tcgen05 kernel could do as
// it spreads them, that is 3e-4, but dims of low codes are less exact than now, and
// values to one side drift as before.)
//
// Shape of the decode kernel.  Keys are the 16-row operand of m16n8k16 (16
// tokens), the query rows of one kv head (group x new tokens) its 8 columns,
// so one product serves a whole group and wastes no more than 8 - rows
// columns.  Each warp streams runs of 32 tokens of its own (two 16-token pieces,
// whose products are interleaved), with its own running maximum, total and
// output in registers: no block-wide step inside the loop; the four warps of a
// block are joined in shared memory at the end of a segment.  The pieces come
// through a ring of cp.async copies private to the warp.
//
// Work split.  The units (128 tokens of one row tile, kv head and sequence) of
// the whole call are laid end to end and every block takes an equal run of
// them, so ragged batches and single long sequences alike fill the SMs without
// the host knowing any length.  A block's run may start or end inside a row
// tile: such partial results go to the workspace, with a note by the block that
// holds the tile's last unit, and a second kernel joins them in a fixed order,
// so results do not depend on timing.
#include <cuda_fp16.h>

#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

// What the joining kernel needs to know of a row tile whose last unit a block
// holds and whose first unit another one does.
struct Kv4Join {
    int rows;        // query rows of the tile; 0: nothing to join
    int first;       // the block with the tile's first unit ..
    int first_slot;  // .. and which of its two partial results that is
    int G;
    int64_t row0;    // first row of the tile's sequence
    int64_t r0;      // first query row of the tile
    int64_t head;
};

// Where a row tile's results are, at its first row: in `out` (last < 0), or in the partial results
// of blocks [first, last], the first's being its first_slot-th.
struct Kv4Where {
    int first, first_slot, last, pad;
};

struct Kv4AttnArgs {
    Kv4Seq s;
    const void* q;
    int q_f32, q_vec;
    int64_t q_sb, q_sl, q_sh;
    int64_t q_l;       // rows between the strides q_sb where the call's "sequences" are not those of q; 0: they are
    const uint8_t* cache;
    int G;             // query heads per kv head
    float scale_log2;  // softmax scale * log2(e)
    void* out;         // (T, Hk * G, D), q's type
    int out_f32;
    Kv4Join* notes;    // workspace: one per block
    float* part;       // workspace: partial results of two segments per block
    // A pass whose results another kernel joins with those of a second pass: out is fp32, with the
    // logarithms (base 2) of the rows' totals in lse, and a record per row tile says where
    // its results are.  (T, Hk * G) each; null: the pass is all there is.
    float* lse;
    Kv4Where* where;
    const int32_t* grp;  // (n_grp + 1) or null: shares of prefixes that may fall, where nothing is computed
    int n_grp;
};

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
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float middle3(float a, float b, float c) { return fmaxf(fminf(a, b), fminf(fmaxf(a, b), c)); }
// 2^e for e in [-126, 127].
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// A row's reference, 2^m S: m its running maximum, S a power of two 2^6 to 2^7 below the
// largest value scale of the tokens that it has seen (and of no others: what a row may not
// see must not cost it bits).  Weights, totals and outputs are relative to it.  neg_r is minus
// its logarithm.  The maximum need not be exact: a weight may exceed 1 / S by up to 2^8 before
// the sums are rescaled, so most tokens skip that; weights times value scales then stay below
// 2^15 in fp16, with the smallest ones as far above its last bit, 2^-24, as that allows.
// `limit`, 8 - log2 S, is what a logit may exceed the reference by.
constexpr int kScaleLeast = -60, kScaleMost = 100;  // exponents of S: sums of weights over 2^30 tokens stay normal numbers
constexpr float kFirstLimit = 8 - kScaleLeast;
// The value scale from which on S is raised.
__device__ __forceinline__ float loud_of(float limit) { return pow2i(15 - (int)limit); }
constexpr float kFirstLoud = 0x1p-53f;  // loud_of(kFirstLimit)
// Takes the logit x and the value scale vt into a row's reference; returns the factor that
// brings earlier sums to it.
__device__ __forceinline__ float raise_reference(float x, float vt, float& neg_r, float& limit) {
    const float neg_m = neg_r + (8.0f - limit);
    const bool louder = vt >= loud_of(limit);
    if (!louder && !(-x < neg_m)) return 1.0f;
    if (louder) limit = (float)(8 - min(max((int)(__float_as_uint(vt) >> 23) - 133, kScaleLeast), kScaleMost));
    const float was = neg_r;
    neg_r = fminf(neg_m, -x) - (8.0f - limit);
    return neg_r == was ? 1.0f : ex2f(neg_r - was);
}

// Row tiles and the units of sequence b (every row tile is
// walked over all of the sequence's tokens; what a tile may not see is skipped
// when it is met).  The host has checked that all units together fit 31 bits.
// C: the kernel's configuration, with kRows query rows to a row tile and kTokens tokens to a unit.
template <typename C>
__device__ __forceinline__ uint32_t attn_units(const Kv4AttnArgs& a, int64_t b, uint32_t& nt) {
    int64_t first, n;
    kv4_rows<C::kMore>(a.s, b, first, n);
    if (C::kMore && a.s.table_hd && kv4_load<true>(a.s.lens + b) < 0) n = 0;  // (of chosen pages: a row that is no sequence's)
    nt = max((kv4_held<C::kMore>(a.s, b) + C::kTokens - 1) / C::kTokens, 1);
    return ((uint32_t)n * a.G + C::kRows - 1) / C::kRows * nt * a.s.Hk;
}

// The units of the call, and this block's run [begin, end): all threads of the
// block.  seq, in_seq: the sequence that holds `begin` and the unit's place in it.
struct AttnRun {
    uint32_t total, begin, end, seq, in_seq;
};
__device__ __forceinline__ uint32_t attn_begin(uint32_t total, uint32_t blocks, uint32_t c) {
    return total / blocks * c + min(c, total % blocks);
}
template <typename C>
__device__ __forceinline__ AttnRun attn_plan(const Kv4AttnArgs& a) {
    constexpr int kWarps = C::kThreads / 32;
    __shared__ uint32_t sums[kWarps], start[2];
    // thread t takes sequences [t * per, (t + 1) * per)
    const uint32_t B = (uint32_t)a.s.B, per = (B + C::kThreads - 1) / C::kThreads;
    const uint32_t b0 = min(threadIdx.x * per, B), b1 = min(b0 + per, B);
    uint32_t sum = 0, nt;
    bool falls = false;  // cu_q does: its rows, and so the units, may be more than the host counted on
    for (uint32_t b = b0; b < b1; ++b) {
        sum += attn_units<C>(a, b, nt);
        falls |= !(C::kMore && a.s.grouped) && a.s.cu && __ldg(a.s.cu + b + 1) < __ldg(a.s.cu + b);
    }
    if (C::kMore && a.s.grouped && a.s.cu)
        for (uint32_t b = threadIdx.x; b < a.s.grouped; b += C::kThreads) falls |= __ldg(a.s.cu + b + 1) < __ldg(a.s.cu + b);
    if (C::kMore && a.grp)
        for (uint32_t b = threadIdx.x; b < (uint32_t)a.n_grp; b += C::kThreads) falls |= __ldg(a.grp + b + 1) < __ldg(a.grp + b);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) sums[w] = inc;
    AttnRun run;
    run.total = 0;
    if (__syncthreads_or(falls)) {  // nothing is computed
        if (threadIdx.x == 0) record_status(PN_ERR_ARG);
        run.begin = run.end = run.seq = run.in_seq = 0;
        return run;
    }
    uint32_t at = inc - sum;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        if (i < w) at += sums[i];
        run.total += sums[i];
    }
    run.begin = attn_begin(run.total, gridDim.x, blockIdx.x);
    run.end = attn_begin(run.total, gridDim.x, blockIdx.x + 1);
    if (run.begin >= at && run.begin < at + sum) {
        uint32_t b = b0;
        for (; b < b1; ++b) {
            const uint32_t n = attn_units<C>(a, b, nt);
            if (run.begin < at + n) break;
            at += n;
        }
        start[0] = b;
        start[1] = run.begin - at;
    }
    __syncthreads();
    run.seq = start[0];
    run.in_seq = start[1];
    return run;
}

// One segment: a run of units of one row tile.
struct AttnSeg {
    uint32_t b, nt, t0, t1;  // sequence; token tiles of it, and the segment's [t0, t1)
    int head, rows;          // kv head; query rows in the tile
    int64_t row0, r0;        // first row of the sequence; first query row of the tile
    int pos0;                // query row r sees positions up to pos0 + r / G (of a prefix: all)
    int kv_end;              // tokens that the tile's last row sees (and the table has room for)
    int lim_min;             // the last position that its first row sees (at most kv_end - 1)

    // Advances `in_seq` to its sequence first.
    template <typename C>
    __device__ __forceinline__ AttnSeg(const Kv4AttnArgs& a, const C&, uint32_t& seq, uint32_t& in_seq, uint32_t left) {
        uint32_t n = attn_units<C>(a, seq, nt);
        while (in_seq >= n) {  // past the sequence (or one without rows)
            in_seq -= n;
            ++seq;
            n = attn_units<C>(a, seq, nt);
        }
        b = seq;
        // a row tile's units are consecutive: (head, row tile, token tile)
        int64_t n_rows;
        kv4_rows<C::kMore>(a.s, b, row0, n_rows);
        const uint32_t q_rows = (uint32_t)n_rows * a.G, n_rt = (q_rows + C::kRows - 1) / C::kRows;
        const uint32_t tile = in_seq / nt;
        head = (int)(tile / n_rt);
        // first and last row tiles in turn: of a long prompt the first see few tokens, the last many
        const uint32_t i = tile - head * n_rt;
        r0 = (i & 1 ? n_rt - 1 - (i >> 1) : i >> 1) * C::kRows;
        rows = (int)min((uint32_t)C::kRows, q_rows - (uint32_t)r0);
        t0 = in_seq - tile * nt;
        t1 = min(nt, t0 + left);
        const bool all = C::kMore && a.s.grouped;
        pos0 = kv4_len<C::kMore>(a.s, b) - (int)n_rows;
        kv_end = all ? kv4_held<C::kMore>(a.s, b) : min(max(pos0 + (int)(((uint32_t)r0 + rows - 1) / a.G) + 1, 0), kv4_held<C::kMore>(a.s, b));
        if (t0 == 0 && threadIdx.x == 0 && a.s.table_w > 0 && pos0 + (int)n_rows > kv4_held<C::kMore>(a.s, b)) record_status(PN_ERR_ARG);
        lim_min = all ? kv_end - 1 : min(pos0 + (int)((uint32_t)r0 / a.G), kv_end - 1);
    }
    // Where query row r of the tile (r < rows) lies in q, in elements.
    template <typename C>
    __device__ __forceinline__ int64_t query(const Kv4AttnArgs& a, const C&, int r) const {
        const uint32_t rr = (uint32_t)r0 + r, i = rr / a.G;
        int64_t at = a.s.cu ? (row0 + i) * a.q_sl : b * a.q_sb + i * a.q_sl;
        if (C::kMore && !a.s.cu && a.q_l) {
            const int64_t of = (row0 + i) / a.q_l;
            at = of * a.q_sb + (row0 + i - of * a.q_l) * a.q_sl;
        }
        return at + (head * a.G + (rr - i * a.G)) * a.q_sh;
    }
};

// Leaves the joining kernel a note where a row tile ends in this block and began
// in an earlier one.
template <typename C>
__device__ __forceinline__ void attn_note(const Kv4AttnArgs& a, const C&, const AttnRun& run, const AttnSeg& sg, uint32_t unit) {
    if (sg.t1 != sg.nt) return;
    const bool where = C::kMore && a.where;
    if (sg.t0 == 0 && !where) return;
    const uint32_t i0 = (uint32_t)sg.r0 / a.G;
    const int64_t row = ((sg.row0 + i0) * a.s.Hk + sg.head) * a.G + (uint32_t)sg.r0 - i0 * a.G;
    if (sg.t0 == 0) {
        a.where[row] = {0, 0, -1, 0};
        return;
    }
    // the block that holds the tile's first unit: the first `rem` blocks hold one more
    const uint32_t u0 = unit - sg.t0, each = run.total / gridDim.x, rem = run.total % gridDim.x;
    const uint32_t c0 = u0 < (each + 1) * rem ? u0 / (each + 1) : rem + (u0 - (each + 1) * rem) / each;
    const int slot = attn_begin(run.total, gridDim.x, c0) < u0 ? 1 : 0;
    if (where)
        a.where[row] = {(int)c0, slot, (int)blockIdx.x, 0};
    else
        a.notes[blockIdx.x] = {sg.rows, (int)c0, slot, a.G, sg.row0, sg.r0, sg.head};
}

// Looks up the pages of a sequence, 32 pieces of 16 tokens at a time: lane l
// holds where piece (base + l)'s keys begin.
struct AttnPages {
    uint64_t addr;  // the page block of the keys; 0: not there
    int off;        // the piece's first token in its page

    template <typename C>
    __device__ __forceinline__ void look_up(const Kv4AttnArgs& a, const C&, uint32_t b, int head, int64_t block, int tok, bool want) {
        addr = 0;
        off = 0;
        if (!want) return;
        const uint32_t i = (uint32_t)tok / (uint32_t)a.s.page;
        const int p = kv4_load<C::kMore>(a.s.table + b * a.s.table_ld + (C::kMore ? head * a.s.table_hd : 0) + i);
        off = tok - (int)i * a.s.page;
        if (p >= 0 && p < a.s.n_pages)
            addr = (uint64_t)(a.cache + ((int64_t)p * a.s.Hk + head) * 2 * block);
        else
            record_status(PN_ERR_ARG);
    }
};

// The logarithm of a row's total `sum`, which is relative to 2^m.
__device__ __forceinline__ float attn_lse(float m, float sum) { return sum == 0.0f ? -INFINITY : m + log2f(sum); }
__device__ __forceinline__ void store_out(const Kv4AttnArgs& a, int64_t at, const float4& y, float inv) {
    if (a.out_f32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    } else {
        const __nv_bfloat162 u = __floats2bfloat162_rn(y.x * inv, y.y * inv), v = __floats2bfloat162_rn(y.z * inv, y.w * inv);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&u), *reinterpret_cast<const uint32_t*>(&v));
    }
}

// The exponent of a query row's scaling, which brings its largest magnitude to
// [2^14, 2^15), kept where 2^e and 2^(24 - e) are normal numbers.
__device__ __forceinline__ int query_exponent(float amax) {
    const int e = 14 - ((int)(__float_as_uint(amax) >> 23) - 127);
    return amax > 0.0f ? min(max(e, -100), 126) : 0;
}
// Eight dims (a word of codes) as the operands that meet the masked codes: dims
// {0,4}, {1,5} / 16, {2,6}, {3,7} / 16, times `up`.  Returns the sum of the rounded eight.
__device__ __forceinline__ float pack_query(const float* v, float up, uint32_t (&p)[4]) {
    float u[8], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = v[j] * up;
    p[0] = pack_f16(u[0], u[4]);
    p[1] = pack_f16(u[1] * 0.0625f, u[5] * 0.0625f);
    p[2] = pack_f16(u[2], u[6]);
    p[3] = pack_f16(u[3] * 0.0625f, u[7] * 0.0625f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[k]));
        sum += (f.x + f.y) * (k & 1 ? 16.0f : 1.0f);
    }
    return sum;
}

// A row's query operands for the words t * W .. that this thread holds.
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
    const int e = query_exponent(amax);
    const float up = pow2i(e);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        uint32_t p[4];
        sum += pack_query(v + i * 8, up, p);
#pragma unroll
        for (int k = 0; k < 4; ++k) qb[i * 4 + k] = p[k];
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    ca = a.scale_log2 * pow2i(24 - e);
    cb = a.scale_log2 * (sum * pow2i(-e));
}

// What bounds the decode kernel: neither the cache's bytes nor a pipe, but latency.  A
// piece of 16 tokens takes a warp about 260 instructions (d = 128, up to 8 rows: 64 masks
// and shifts, 32 products, the softmax of 16 x 8 logits), each waiting for the one
// before, and the registers leave room for twelve warps to an SM: they issue 1.9
// instructions of four possible per cycle, the ALU pipe is 44 % and the tensor
// pipe 23 % busy.
// 32 sequences of up to 8191 tokens, 8 heads: 50 us, 3.3 TB/s; one of 131072: 42 us,
// 3.4 TB/s (half of the copy's rate).  Three blocks of six stages per SM: two, four or
// five blocks, and more stages in two, are all slower.  With 16 rows at d = 128 the
// registers do not suffice (404 bytes spilled per thread).
template <int D, int NT, bool M>
struct AttnCfg {
    static constexpr bool kMore = M;
    static constexpr int W = D / 32;             // words per thread and token
    static constexpr int kRows = 8 * NT;         // query rows of a row tile
    static constexpr int kTokens = 128;          // tokens of a unit: 32 per warp
    // Runs between two centrings.  64 sequences of 4096 tokens, 8 heads of 8 rows: 71.7 us with 4, 71.3 with 8, 69.0
    // with none.
    static constexpr int kCentre = 4;
    static constexpr int kThreads = kAttnThreads;
    static constexpr int kStages = 6;
    static constexpr int kCodes = 16 * (D / 2);  // bytes of one 16-token piece of keys or values
    static constexpr int kStage = 2 * kCodes + 128;
    static constexpr int kRing = kStages * kStage;  // per warp
    static constexpr int kSmem = kAttnWarps * kRing;
    static constexpr int kPitch = D + 8;         // floats per row of the join buffer (over the warp's own ring)
    static constexpr int kPart = kRows * (D + 2);  // floats of one partial result
    static constexpr int kBlocks = 3;  // per SM
    static_assert(kRows * kPitch * 4 <= kRing, "the join buffer lies over the ring");
};

// Byte position of 16-byte chunk j of token pair p inside a piece's values:
// rotated so that the eight lanes of one shared-memory phase (two dim groups x
// four pairs) meet eight different bank groups.
template <int D>
__device__ __forceinline__ int v_chunk(int p, int j) {
    return D == 128 ? p * 128 + ((j + 2 * p) & 7) * 16 : p * 64 + ((j + (p & 2)) & 3) * 16;
}

// W words of a row of codes.
template <int W>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[W]) {
    if constexpr (W == 4) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x, w[1] = u.y;
    }
}
__device__ __forceinline__ float pair_lo(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float pair_hi(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }

template <int D, int NT, bool M>
__global__ void __launch_bounds__(kAttnThreads, AttnCfg<D, NT, M>::kBlocks) kv4_decode_kernel(const Kv4AttnArgs a) {
    using C = AttnCfg<D, NT, M>;
    constexpr int W = C::W, RT = C::kRows, ST = C::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float join_ml[kAttnWarps * RT * 2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * C::kRing;
    const uint32_t ring_u = smem_u32(ring);
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    AttnRun run = attn_plan<C>(a);
    if (tid == 0) a.notes[blockIdx.x].rows = 0;
    const int64_t block = (int64_t)a.s.page * (D / 2 + 4);
    // a lane's part of a piece: 16-byte chunks of codes, and of the pairs (lanes 0-3 keys, 4-7 values)
    const uint32_t pair_off = (uint32_t)a.s.page * (D / 2) + (lane & 3) * 16 + (lane & 4 ? (uint32_t)block : 0u);
    // (a second chunk of a lane lies four pairs on: the same rotation, 512 bytes further)
    const uint32_t dst_k = ring_u + lane * 16, dst_v = ring_u + C::kCodes + v_chunk<D>(lane / (D / 16), lane % (D / 16)),
                   dst_p = ring_u + 2 * C::kCodes + lane * 16;

    uint32_t seq = run.seq, in_seq = run.in_seq;
    for (uint32_t unit = run.begin; unit < run.end;) {
        const AttnSeg sg(a, C{}, seq, in_seq, run.end - unit);

        // ---- the warp's runs: tokens [128 * tile + 32 * warp, + 32), two pieces each
        const int used = min((int)sg.t1, (sg.kv_end + C::kTokens - 1) / C::kTokens);  // tiles behind it are skipped
        const int count = used - (int)sg.t0;
        const int tok_base = (int)sg.t0 * C::kTokens + warp * 32;
        AttnPages pages;
        uint32_t dead = 0;  // ring of flags: the piece is not there
        auto issue = [&](int i, uint32_t slot) {  // run i; slot: its first stage's offset in the ring
            if ((i & 15) == 0) {  // lane 2 k + j looks up piece j of run i + k
                const int k = i + (lane >> 1), tok = tok_base + k * C::kTokens + (lane & 1) * 16;
                pages.look_up(a, C{}, sg.b, sg.head, block, tok, k < count && tok < sg.kv_end);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int from = 2 * (i & 15) + j;
                const uint64_t addr = __shfl_sync(0xffffffffu, pages.addr, from);
                const uint32_t off = __shfl_sync(0xffffffffu, pages.off, from);
                const uint32_t bit = 1u << from;
                if (addr) {
                    dead &= ~bit;
                    const uint8_t* kc = reinterpret_cast<const uint8_t*>(addr) + (off * (D / 2) + lane * 16);
                    const uint8_t* vc = kc + block;
                    const uint32_t st = slot + j * C::kStage;
#pragma unroll
                    for (int c = 0; c < C::kCodes / 512; ++c) {
                        cp_async16(dst_k + st + c * 512, kc + c * 512);
                        cp_async16(dst_v + st + c * 512, vc + c * 512);
                    }
                    if (lane < 8) cp_async16(dst_p + st, reinterpret_cast<const uint8_t*>(addr) + (pair_off + off * 4));
                } else {
                    dead |= bit;
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < ST / 2 - 1; ++i) issue(i, 2 * i * C::kStage);

        // ---- queries
        uint32_t qb[NT][D / 8];
        float2 ca[NT], cb[NT];
        int lim[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const char* row = nullptr;
            if (n * 8 + g < sg.rows) row = static_cast<const char*>(a.q) + sg.query(a, C{}, n * 8 + g) * (a.q_f32 ? 4 : 2);
            float fa, fb;
            load_query<D>(a, row, t, qb[n], fa, fb);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float va = __shfl_sync(0xffffffffu, fa, (2 * t + k) * 4), vb = __shfl_sync(0xffffffffu, fb, (2 * t + k) * 4);
                if (k == 0)
                    ca[n].x = va, cb[n].x = vb;
                else
                    ca[n].y = va, cb[n].y = vb;
                const int rl = n * 8 + 2 * t + k;
                lim[n][k] = rl < sg.rows && !(C::kMore && a.s.grouped) ? sg.pos0 + (int)(((uint32_t)sg.r0 + rl) / a.G) : sg.kv_end - 1;
            }
        }

        float o[NT][D / 16][4];
        float2 base[NT];  // what was taken out of o, and the z term with it
        float2 neg_r[NT], limit[NT], l[NT], zs[NT];  // the rows' references; totals of p and of p z (this lane's tokens)
        float loud = kFirstLoud;  // the least of the rows'
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            neg_r[n] = make_float2(INFINITY, INFINITY), limit[n] = make_float2(kFirstLimit, kFirstLimit);
            l[n] = zs[n] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[n][j][k] = 0.0f;
            base[n] = make_float2(0.0f, 0.0f);
        }

        // The two pieces of run i.  kMask: some token of them is not seen by some row.
        auto pieces = [&](int i, uint32_t slot, auto mask) {
            constexpr bool kMask = decltype(mask)::value;
            const uint8_t* st[2] = {ring + slot, ring + slot + C::kStage};
            // ---- logits: 16 tokens x 8 rows per piece and n
            float acc[2][NT][4];
            uint32_t vp[2][2], ka[2][W], kb[2][W];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[j][n][k] = 0.0f;
                lds_words<W>(st[j] + g * (D / 2) + t * 4 * W, ka[j]);
                lds_words<W>(st[j] + (g + 8) * (D / 2) + t * 4 * W, kb[j]);
            }
            // the two pieces' products in turn: each is a chain over the dims
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t u = h ? ka[j][w] >> 8 : ka[j][w], v = h ? kb[j][w] >> 8 : kb[j][w];
                        const uint32_t a0 = u & 0x000F000Fu, a1 = v & 0x000F000Fu, a2 = u & 0x00F000F0u, a3 = v & 0x00F000F0u;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_f16(acc[j][n], a0, a1, a2, a3, qb[n][w * 4 + h * 2], qb[n][w * 4 + h * 2 + 1]);
                    }
            float rel[2][NT][4], vtop = 0.0f;  // rel: logit - reference
            float2 top[NT];                    // a row's largest
#pragma unroll
            for (int n = 0; n < NT; ++n) top[n] = make_float2(-INFINITY, -INFINITY);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int tok0 = tok_base + i * C::kTokens + j * 16;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t kp = *reinterpret_cast<const uint32_t*>(st[j] + 2 * C::kCodes + (g + 8 * k) * 4);
                    vp[j][k] = *reinterpret_cast<const uint32_t*>(st[j] + 2 * C::kCodes + 64 + (g + 8 * k) * 4);
                    const bool none = kMask && ((dead >> (2 * (i & 15) + j) & 1u) || tok0 + g + 8 * k >= sg.kv_end);
                    if (kMask && none) vp[j][k] = 0;  // whatever lies behind the sequence
                    const float2 ks = make_float2(pair_lo(kp), pair_lo(kp)), kz = make_float2(pair_hi(kp), pair_hi(kp));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float2 x = make_float2(acc[j][n][2 * k], acc[j][n][2 * k + 1]);
                        x = fma2(ks, mul2(x, ca[n]), mul2(kz, cb[n]));
                        if constexpr (kMask) {
                            if (none || tok0 + g + 8 * k > lim[n][0]) x.x = -INFINITY;
                            if (none || tok0 + g + 8 * k > lim[n][1]) x.y = -INFINITY;
                        }
                        acc[j][n][2 * k] = x.x, acc[j][n][2 * k + 1] = x.y;
                        x = add2(x, neg_r[n]);
                        rel[j][n][2 * k] = x.x, rel[j][n][2 * k + 1] = x.y;
                        top[n] = make_float2(fmaxf(top[n].x, x.x), fmaxf(top[n].y, x.y));
                    }
                    vtop = fmaxf(vtop, pair_lo(vp[j][k]));
                }
            }
            bool raise = vtop >= loud;
#pragma unroll
            for (int n = 0; n < NT; ++n) raise |= top[n].x > limit[n].x || top[n].y > limit[n].y;
            if (__any_sync(0xffffffffu, raise)) {  // (for the first piece it is true: m is -inf there)
                loud = INFINITY;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float f[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float x = fmaxf(fmaxf(acc[0][n][k], acc[0][n][2 + k]), fmaxf(acc[1][n][k], acc[1][n][2 + k]));
                        float vt = kMask ? 0.0f : vtop;
                        if constexpr (kMask) {  // of the tokens that the row sees
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int c = 0; c < 2; ++c)
                                    if (acc[j][n][2 * c + k] != -INFINITY) vt = fmaxf(vt, pair_lo(vp[j][c]));
                        }
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) {
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                            vt = fmaxf(vt, __shfl_xor_sync(0xffffffffu, vt, d));
                        }
                        f[k] = k ? raise_reference(x, vt, neg_r[n].y, limit[n].y) : raise_reference(x, vt, neg_r[n].x, limit[n].x);
                        loud = fminf(loud, loud_of(k ? limit[n].y : limit[n].x));
                        const float now = k ? neg_r[n].y : neg_r[n].x;
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int c = 0; c < 2; ++c) rel[j][n][2 * c + k] = acc[j][n][2 * c + k] + now;
                    }
                    l[n] = mul2(l[n], make_float2(f[0], f[1]));
                    zs[n] = mul2(zs[n], make_float2(f[0], f[1]));
#pragma unroll
                    for (int j = 0; j < D / 16; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[n][j][k] *= f[k & 1];
                    base[n] = mul2(base[n], make_float2(f[0], f[1]));
                }
            }
            // ---- weights, then dims x rows of the output
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t pb[NT][2];
                const float vs[2] = {pair_lo(vp[j][0]), pair_lo(vp[j][1])};
                const float vz[2] = {pair_hi(vp[j][0]), pair_hi(vp[j][1])};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t wgt[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float2 p = make_float2(ex2f(rel[j][n][2 * k]), ex2f(rel[j][n][2 * k + 1]));
                        float2 pz = p, pv = p;
                        if constexpr (kMask) {  // a token that a row does not see adds nothing, whatever its pair holds
                            const bool n0 = acc[j][n][2 * k] == -INFINITY, n1 = acc[j][n][2 * k + 1] == -INFINITY;
                            p.x = n0 ? 0.0f : p.x, p.y = n1 ? 0.0f : p.y;
                            pz = make_float2(n0 ? 0.0f : p.x * vz[k], n1 ? 0.0f : p.y * vz[k]);
                            pv = make_float2(n0 ? 0.0f : p.x * vs[k], n1 ? 0.0f : p.y * vs[k]);
                            zs[n] = add2(zs[n], pz);
                        } else {
                            zs[n] = fma2(p, make_float2(vz[k], vz[k]), zs[n]);
                            pv = mul2(p, make_float2(vs[k], vs[k]));
                        }
                        l[n] = add2(l[n], p);
                        wgt[k] = pack_f16(pv.x, pv.y);
                    }
                    pb[n][0] = movmatrix_t(wgt[0]);
                    pb[n][1] = movmatrix_t(wgt[1]);
                }
                uint32_t va[W], vb[W];
                const uint8_t* sv = st[j] + C::kCodes;
                lds_words<W>(sv + (W == 4 ? v_chunk<D>(t, g) : v_chunk<D>(t, g >> 1) + (g & 1) * 8), va);
                lds_words<W>(sv + (W == 4 ? v_chunk<D>(t + 4, g) : v_chunk<D>(t + 4, g >> 1) + (g & 1) * 8), vb);
#pragma unroll
                for (int w = 0; w < W; ++w)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t u = h ? va[w] >> 8 : va[w], v = h ? vb[w] >> 8 : vb[w];
                        const uint32_t a0 = u & 0x000F000Fu, a1 = u & 0x00F000F0u, a2 = v & 0x000F000Fu, a3 = v & 0x00F000F0u;
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_f16(o[n][w * 2 + h], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                    }
            }
        };
        // A row's sums back to about zero (all dims of a lane share the base).
        auto centre = [&]() {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 r = make_float2(middle3(o[n][0][0], o[n][1][0], o[n][2][0]), middle3(o[n][0][1], o[n][1][1], o[n][2][1]));
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    zs[n].x += __shfl_xor_sync(0xffffffffu, zs[n].x, d);
                    zs[n].y += __shfl_xor_sync(0xffffffffu, zs[n].y, d);
                }
                base[n] = add2(base[n], fma2(r, make_float2(16777216.0f, 16777216.0f), zs[n]));
                zs[n] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
#pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        const float up = k ? -16.0f : -1.0f;
                        const float2 y = fma2(r, make_float2(up, up), make_float2(o[n][j][k], o[n][j][k + 1]));
                        o[n][j][k] = y.x, o[n][j][k + 1] = y.y;
                    }
            }
        };
        uint32_t slot = 0, fill = (ST - 2) * C::kStage;  // stages of runs i and i + ST / 2 - 1
        for (int i = 0; i < count; ++i) {
            issue(i + ST / 2 - 1, fill);
            if (i % C::kCentre == 0 && i > 0) centre();
            cp_wait<ST / 2 - 1>();
            __syncwarp();
            const bool mask = (dead >> (2 * (i & 15)) & 3u) || tok_base + i * C::kTokens + 31 > sg.lim_min;
            if (mask)
                pieces(i, slot, std::true_type{});
            else
                pieces(i, slot, std::false_type{});
            __syncwarp();  // every lane has read the stages before they are filled again
            fill = slot;
            slot = slot == (ST - 2) * C::kStage ? 0 : slot + 2 * C::kStage;
        }

        centre();  // (what is left of the z term joins the base)

        // ---- join the four warps
        float* mine = reinterpret_cast<float*>(ring);  // nothing is in flight
        const float up = 16777216.0f;                  // the codes' 2^-24
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l[n].x += __shfl_xor_sync(0xffffffffu, l[n].x, d);
                l[n].y += __shfl_xor_sync(0xffffffffu, l[n].y, d);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = n * 8 + 2 * t + k;
                const float z = k ? base[n].y : base[n].x;
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
                    *reinterpret_cast<float2*>(mine + r * C::kPitch + 4 * (g * W + j / 2) + 2 * (j & 1)) =
                        make_float2(fmaf(o[n][j][k], up, z), fmaf(o[n][j][2 + k], up * 0.0625f, z));
                if (g == 0) {
                    join_ml[(warp * RT + r) * 2] = k ? -neg_r[n].y : -neg_r[n].x;
                    join_ml[(warp * RT + r) * 2 + 1] = k ? l[n].y : l[n].x;
                }
            }
        }
        __syncthreads();
        const bool whole = sg.t0 == 0 && sg.t1 == sg.nt;
        float* part = a.part + ((int64_t)blockIdx.x * 2 + (unit == run.begin ? 0 : 1)) * C::kPart;
        for (int idx = tid; idx < sg.rows * (D / 4); idx += kAttnThreads) {
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
                const float4 u = *reinterpret_cast<const float4*>(smem + w * C::kRing + (r * C::kPitch + d) * 4);
                y.x = fmaf(f, u.x, y.x), y.y = fmaf(f, u.y, y.y), y.z = fmaf(f, u.z, y.z), y.w = fmaf(f, u.w, y.w);
            }
            if (whole) {
                const uint32_t rr = (uint32_t)sg.r0 + r, i = rr / a.G;
                const int64_t at = ((sg.row0 + i) * a.s.Hk + sg.head) * a.G + rr - i * a.G;
                store_out(a, at * D + d, y, sum == 0.0f ? 0.0f : 1.0f / sum);
                if (C::kMore && a.lse && d == 0) a.lse[at] = attn_lse(mx, sum);
            } else {
                *reinterpret_cast<float4*>(part + r * D + d) = y;
                if (d == 0) part[RT * D + r * 2] = mx, part[RT * D + r * 2 + 1] = sum;
            }
        }
        if (tid == 0) attn_note(a, C{}, run, sg, unit);
        __syncthreads();
        unit += sg.t1 - sg.t0;
        in_seq += sg.t1 - sg.t0;
    }
}

// Prompts and chunks of them: 64 query rows per block, 16 per warp, which share
// the tokens' pieces in shared memory.  Here the rows are the 16-row operand, the
// codes the 8-column one: the same words and masks give it (the first operand's
// registers are two of the second's).  A block steps through 64 tokens at a time,
// a warp through 32 of them at once; rows meet the softmax as they lie in the
// accumulators, and their weights go back in as they come out.
//
// What bounds it: m16n8k16 runs at one per ten cycles on each quarter of an SM
// (measured; 460 TFLOP/s over the device), 128 of them to a warp's 64 tokens at
// d = 128, and 320 mask and shift instructions; but the tensor pipe is only 33 % busy
// and 41 % of the issue slots are used: as in the decode kernel the warps (twelve to
// an SM) wait for their own last instruction.  64 sequences x 64 rows x 4 heads over 1024
// tokens: 70 us (two blocks to an SM: 2 % slower than three); 180 bytes spilled per thread.
template <int D, bool M>
struct ChunkCfg {
    static constexpr bool kMore = M;
    static constexpr int W = D / 32;
    static constexpr int kRows = 64, kTokens = 64, kThreads = kAttnThreads;
    static constexpr int kCentre = 4;  // tiles between two centrings (8: the same time)
    static constexpr int kStages = 3;
    static constexpr int kCodes = 16 * (D / 2);
    static constexpr int kPiece = 2 * kCodes + 128;  // 16 tokens, as in AttnCfg
    static constexpr int kTile = 4 * kPiece;
    static constexpr int kSmem = kStages * kTile;
    static constexpr int kPart = kRows * (D + 2);
    static constexpr int kBlocks = 3;  // per SM
};

template <int D, bool M>
__global__ void __launch_bounds__(kAttnThreads, ChunkCfg<D, M>::kBlocks) kv4_chunk_kernel(const Kv4AttnArgs a) {
    using C = ChunkCfg<D, M>;
    constexpr int W = C::W, ST = C::kStages;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint8_t dead[ST][4];  // the piece is not there
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const AttnRun run = attn_plan<C>(a);
    if (tid == 0) a.notes[blockIdx.x].rows = 0;
    const int64_t block = (int64_t)a.s.page * (D / 2 + 4);
    const uint32_t pair_off = (uint32_t)a.s.page * (D / 2) + (lane & 3) * 16 + (lane & 4 ? (uint32_t)block : 0u);
    const uint32_t base_u = smem_u32(smem) + warp * C::kPiece;  // this warp copies piece `warp` of every tile
    const uint32_t dst_k = base_u + lane * 16, dst_v = base_u + C::kCodes + v_chunk<D>(lane / (D / 16), lane % (D / 16)),
                   dst_p = base_u + 2 * C::kCodes + lane * 16;

    uint32_t seq = run.seq, in_seq = run.in_seq;
    for (uint32_t unit = run.begin; unit < run.end;) {
        const AttnSeg sg(a, C{}, seq, in_seq, run.end - unit);
        const int used = min((int)sg.t1, (sg.kv_end + C::kTokens - 1) / C::kTokens);
        const int count = used - (int)sg.t0;
        const int tok_base = (int)sg.t0 * C::kTokens;
        AttnPages pages;
        auto issue = [&](int i, int stage) {
            if ((i & 31) == 0) {
                const int tok = tok_base + (i + lane) * C::kTokens + warp * 16;
                pages.look_up(a, C{}, sg.b, sg.head, block, tok, i + lane < count && tok < sg.kv_end);
            }
            const uint64_t addr = __shfl_sync(0xffffffffu, pages.addr, i & 31);
            const uint32_t off = __shfl_sync(0xffffffffu, pages.off, i & 31);
            if (lane == 0) dead[stage][warp] = addr == 0;
            if (addr) {
                const uint8_t* kc = reinterpret_cast<const uint8_t*>(addr) + (off * (D / 2) + lane * 16);
                const uint8_t* vc = kc + block;
                const uint32_t st = stage * C::kTile;
#pragma unroll
                for (int c = 0; c < C::kCodes / 512; ++c) {
                    cp_async16(dst_k + st + c * 512, kc + c * 512);
                    cp_async16(dst_v + st + c * 512, vc + c * 512);
                }
                if (lane < 8) cp_async16(dst_p + st, reinterpret_cast<const uint8_t*>(addr) + (pair_off + off * 4));
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) issue(i, i);

        // ---- this warp's rows: g and g + 8
        const int w_rows = min(sg.rows - warp * 16, 16);  // none: the warp only copies
        uint32_t qa[D / 8], qc[D / 8];
        float ca[2], cb[2];
        int lim[2], w_end = 0, w_min = 0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int r = warp * 16 + k * 8 + g;
            const char* row = nullptr;
            if (r < sg.rows) row = static_cast<const char*>(a.q) + sg.query(a, C{}, r) * (a.q_f32 ? 4 : 2);
            load_query<D>(a, row, t, k ? qc : qa, ca[k], cb[k]);
            lim[k] = r < sg.rows && !(C::kMore && a.s.grouped) ? sg.pos0 + (int)(((uint32_t)sg.r0 + r) / a.G) : sg.kv_end - 1;
        }
        if (w_rows > 0) {
            w_min = C::kMore && a.s.grouped ? sg.kv_end - 1 : sg.pos0 + (int)(((uint32_t)sg.r0 + warp * 16) / a.G);
            w_end = C::kMore && a.s.grouped ? sg.kv_end : max(sg.pos0 + (int)(((uint32_t)sg.r0 + warp * 16 + w_rows - 1) / a.G) + 1, 0);
            // a padding row sees what the warp's last one does
            if (warp * 16 + g >= sg.rows) lim[0] = w_end - 1;
            if (warp * 16 + 8 + g >= sg.rows) lim[1] = w_end - 1;
        }

        float o[D / 8][4], neg_r[2] = {INFINITY, INFINITY}, limit[2] = {kFirstLimit, kFirstLimit}, loud = kFirstLoud;
        float2 l[2], zs[2];
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[j][k] = 0.0f;
        l[0] = l[1] = zs[0] = zs[1] = make_float2(0.0f, 0.0f);

        float base[2] = {};  // what was taken out of o, and the z term with it
        // 32 tokens from tok on, pieces `st` and the next.
        auto half = [&](const uint8_t* st, int tok, bool dead0, bool dead1, auto mask) {
            constexpr bool kMask = decltype(mask)::value;
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[j][k] = 0.0f;
            }
#pragma unroll
            for (int w = 0; w < W; w += 2) {  // two words of each token at a time, the tokens' chains in turn
                uint32_t kw[4][2];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint2 u = *reinterpret_cast<const uint2*>(st + (j >> 1) * C::kPiece + ((j & 1) * 8 + g) * (D / 2) + t * 4 * W + w * 4);
                    kw[j][0] = u.x, kw[j][1] = u.y;
                }
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t u = h ? kw[j][x] >> 8 : kw[j][x];
                            const int q = (w + x) * 4 + h * 2;
                            mma_f16(acc[j], qa[q], qc[q], qa[q + 1], qc[q + 1], u & 0x000F000Fu, u & 0x00F000F0u);
                        }
            }
            // ---- logits; columns 2t, 2t + 1 of n-tile j are tokens 8 j + 2 t, + 1
            float top[2] = {-INFINITY, -INFINITY}, vtop = 0.0f;  // as in the decode kernel
            uint2 vp[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint8_t* pairs = st + (j >> 1) * C::kPiece + 2 * C::kCodes + ((j & 1) * 8 + 2 * t) * 4;
                const uint2 kp = *reinterpret_cast<const uint2*>(pairs);
                vp[j] = *reinterpret_cast<const uint2*>(pairs + 64);
                const int tk = tok + j * 8 + 2 * t;
                const bool gone = kMask && (j < 2 ? dead0 : dead1);
                if constexpr (kMask) {
                    if (gone || tk >= w_end) vp[j].x = 0;  // whatever lies behind the sequence
                    if (gone || tk + 1 >= w_end) vp[j].y = 0;
                }
                const float2 ks = make_float2(pair_lo(kp.x), pair_lo(kp.y)), kz = make_float2(pair_hi(kp.x), pair_hi(kp.y));
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float2 x = make_float2(acc[j][2 * k], acc[j][2 * k + 1]);
                    x = fma2(ks, mul2(x, make_float2(ca[k], ca[k])), mul2(kz, make_float2(cb[k], cb[k])));
                    if constexpr (kMask) {
                        if (gone || tk > lim[k]) x.x = -INFINITY;
                        if (gone || tk + 1 > lim[k]) x.y = -INFINITY;
                    }
                    acc[j][2 * k] = x.x, acc[j][2 * k + 1] = x.y;
                    const float2 d = add2(x, make_float2(neg_r[k], neg_r[k]));
                    top[k] = fmaxf(top[k], fmaxf(d.x, d.y));
                }
                vtop = fmaxf(vtop, fmaxf(pair_lo(vp[j].x), pair_lo(vp[j].y)));
            }
            if (__any_sync(0xffffffffu, top[0] > limit[0] || top[1] > limit[1] || vtop >= loud)) {  // seldom
                loud = INFINITY;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float x = -INFINITY, vt = kMask ? 0.0f : vtop;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x = fmaxf(x, fmaxf(acc[j][2 * k], acc[j][2 * k + 1]));
                        if constexpr (kMask) {  // of the tokens that the row sees
                            if (acc[j][2 * k] != -INFINITY) vt = fmaxf(vt, pair_lo(vp[j].x));
                            if (acc[j][2 * k + 1] != -INFINITY) vt = fmaxf(vt, pair_lo(vp[j].y));
                        }
                    }
#pragma unroll
                    for (int d = 1; d < 4; d <<= 1) {
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        vt = fmaxf(vt, __shfl_xor_sync(0xffffffffu, vt, d));
                    }
                    const float f = raise_reference(x, vt, neg_r[k], limit[k]);
                    loud = fminf(loud, loud_of(limit[k]));
                    l[k] = mul2(l[k], make_float2(f, f));
                    zs[k] = mul2(zs[k], make_float2(f, f));
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) o[j][2 * k] *= f, o[j][2 * k + 1] *= f;
                    base[k] *= f;
                }
            }
            // ---- weights, in place as the first operand of the output's products
            uint32_t pa[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 vs = make_float2(pair_lo(vp[j].x), pair_lo(vp[j].y));
                const float2 vz = make_float2(pair_hi(vp[j].x), pair_hi(vp[j].y));
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float2 d = add2(make_float2(acc[j][2 * k], acc[j][2 * k + 1]), make_float2(neg_r[k], neg_r[k]));
                    float2 p = make_float2(ex2f(d.x), ex2f(d.y)), pv;
                    if constexpr (kMask) {  // a token that a row does not see adds nothing, whatever its pair holds
                        const bool n0 = acc[j][2 * k] == -INFINITY, n1 = acc[j][2 * k + 1] == -INFINITY;
                        p = make_float2(n0 ? 0.0f : p.x, n1 ? 0.0f : p.y);
                        zs[k] = add2(zs[k], make_float2(n0 ? 0.0f : p.x * vz.x, n1 ? 0.0f : p.y * vz.y));
                        pv = make_float2(n0 ? 0.0f : p.x * vs.x, n1 ? 0.0f : p.y * vs.y);
                    } else {
                        zs[k] = fma2(p, vz, zs[k]);
                        pv = mul2(p, vs);
                    }
                    l[k] = add2(l[k], p);
                    pa[j][k] = pack_f16(pv.x, pv.y);
                }
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // 16 tokens each
                uint32_t va[W], vb[W];
                const uint8_t* sv = st + x * C::kPiece + C::kCodes;
                lds_words<W>(sv + (W == 4 ? v_chunk<D>(t, g) : v_chunk<D>(t, g >> 1) + (g & 1) * 8), va);
                lds_words<W>(sv + (W == 4 ? v_chunk<D>(t + 4, g) : v_chunk<D>(t + 4, g >> 1) + (g & 1) * 8), vb);
#pragma unroll
                for (int w = 0; w < W; ++w)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t u = h ? va[w] >> 8 : va[w], v = h ? vb[w] >> 8 : vb[w];
                        mma_f16(o[w * 4 + h * 2], pa[2 * x][0], pa[2 * x][1], pa[2 * x + 1][0], pa[2 * x + 1][1], u & 0x000F000Fu,
                                v & 0x000F000Fu);
                        mma_f16(o[w * 4 + h * 2 + 1], pa[2 * x][0], pa[2 * x][1], pa[2 * x + 1][0], pa[2 * x + 1][1],
                                u & 0x00F000F0u, v & 0x00F000F0u);
                    }
            }
        };
        auto centre = [&]() {  // as in the decode kernel
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float r = middle3(o[0][2 * k], o[2][2 * k], o[4][2 * k]);
                float z = zs[k].x + zs[k].y;
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
                base[k] += fmaf(r, 16777216.0f, z);
                zs[k] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    const float up = j & 1 ? -16.0f : -1.0f;
                    const float2 y = fma2(make_float2(r, r), make_float2(up, up), make_float2(o[j][2 * k], o[j][2 * k + 1]));
                    o[j][2 * k] = y.x, o[j][2 * k + 1] = y.y;
                }
            }
        };
        int stage = 0;
        for (int i = 0; i < count; ++i) {
            if (i % C::kCentre == 0 && i > 0) centre();
            cp_wait<ST - 2>();
            __syncthreads();  // tile i is there for all; all are done with the stage that is filled next
            issue(i + ST - 1, stage == 0 ? ST - 1 : stage - 1);
            const uint8_t* tile = smem + stage * C::kTile;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
                const int tok = tok_base + i * C::kTokens + h * 32;
                if (tok >= w_end) break;
                const bool d0 = dead[stage][2 * h], d1 = dead[stage][2 * h + 1];
                if (d0 || d1 || tok + 31 > w_min)
                    half(tile + 2 * h * C::kPiece, tok, d0, d1, std::true_type{});
                else
                    half(tile + 2 * h * C::kPiece, tok, false, false, std::false_type{});
            }
            stage = stage == ST - 1 ? 0 : stage + 1;
        }

        centre();

        // ---- results: row g's columns 2t and 2t + 1 are 4 W dims each
        const bool whole = sg.t0 == 0 && sg.t1 == sg.nt;
        float* part = a.part + ((int64_t)blockIdx.x * 2 + (unit == run.begin ? 0 : 1)) * C::kPart;
        const float up = 16777216.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float sum = l[k].x + l[k].y, z = base[k];
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const int r = warp * 16 + k * 8 + g;
            if (r >= sg.rows) continue;
            const uint32_t rr = (uint32_t)sg.r0 + r, i = rr / a.G;
            const int64_t row = ((sg.row0 + i) * a.s.Hk + sg.head) * a.G + rr - i * a.G, at = row * D;
            const float inv = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const int d = 4 * ((2 * t + c) * W + w);
                    const float4 y = make_float4(fmaf(o[w * 4][2 * k + c], up, z), fmaf(o[w * 4 + 1][2 * k + c], up * 0.0625f, z),
                                                 fmaf(o[w * 4 + 2][2 * k + c], up, z), fmaf(o[w * 4 + 3][2 * k + c], up * 0.0625f, z));
                    if (whole)
                        store_out(a, at + d, y, inv);
                    else
                        *reinterpret_cast<float4*>(part + r * D + d) = y;
                }
            if (C::kMore && whole && a.lse && t == 0) a.lse[row] = attn_lse(-neg_r[k], sum);
            if (!whole && t == 0) part[C::kRows * D + r * 2] = -neg_r[k], part[C::kRows * D + r * 2 + 1] = sum;
        }
        if (tid == 0) attn_note(a, C{}, run, sg, unit);
        __syncthreads();  // nobody reads a stage any more
        unit += sg.t1 - sg.t0;
        in_seq += sg.t1 - sg.t0;
    }
}

// Long prompts: 128 query rows per block on tcgen05, two blocks to an SM.  The
// block's eight warps spread 64 tokens' codes into fp16 operands in shared memory
// (128-byte swizzle; a code is still only masked), one thread has the tensor core
// form output += P V of one tile and logits = Q K^T of the next, with both results
// and P in tensor memory, and the warps do the softmax: thread (row, half) takes 32
// tokens of a row.
//
// Here a row's logits stay in units of its query's scaling until the exponent (the
// factor joins the reference in one fma).
//
// A step waits for the products of the one before, so operands and logits need no
// second buffer; the other block of the SM fills the wait.  (One block of 16 warps
// with doubled buffers and 128 tokens per step took 278 us where this takes 223 us,
// chunks of 1 to 512 tokens: its warps met at five barriers per step with
// nothing else to run.)
//
// What bounds it: the latency of the softmax's and the spreading's instructions, about
// 500 per thread and step, which all warps do in turn between the block's barriers (3500 to
// 4500 cycles for an SM's two blocks, 47 % of the issue slots used); the products take
// 512 cycles of a step at the tensor core's rate.  16 sequences x 512 rows x 8
// heads over 1024 tokens: 114 us (the chunk kernel 144).
template <int D, bool M>
struct TcCfg {
    static constexpr bool kMore = M;
    static constexpr int kRows = 128, kTokens = 64, kThreads = 256;
    static constexpr int kCentre = 8;  // tiles between two centrings, at most (2 % slower than with none; 4: 4 %)
    static constexpr int kStages = 3;
    static constexpr int kRawK = kTokens * (D / 2);      // codes of a tile's keys (or values)
    static constexpr int kRaw = 2 * kRawK + 8 * kTokens; // and the pairs: the keys', then the values'
    static constexpr int kQ = kRows * D * 2;             // operands: rows of 128 bytes, in boxes of 64 columns
    static constexpr int kK = kTokens * D * 2, kV = D * kTokens * 2;
    static constexpr int kPairs = 4 * kTokens * 4;       // key scales, key zeros, value scales, value zeros as fp32
    static constexpr int kSmem = kQ + kK + kV + kStages * kRaw + 2 * kPairs + 1024;  // (+ alignment)
    static constexpr int kPart = kRows * (D + 2);
    static constexpr int kBlocks = 2;  // per SM
    // tensor memory columns: logits, weights, output
    static constexpr uint32_t kColS = 0, kColP = 64, kColO = 128, kCols = 256;
    // instruction descriptors, f16 x f16 -> f32, 128 rows: 64 tokens (logits), D dims (output)
    static constexpr uint32_t kIdescS = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
    static constexpr uint32_t kIdescO = (1u << 4) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
};

__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Four K-steps over one 64-column box from a converged warp, kind::f16, with one
// election and 32-bit descriptor arithmetic (an election and a 64-bit descriptor per
// product took 58 cycles each, on the path of every step): D[tmem] (+)= A B^T, B in
// shared memory, A in shared memory (ss) or tensor memory (ts).  a, b: low words of
// the descriptors, or A's column; the steps lie 32 bytes, or 8 columns, apart.
__device__ __forceinline__ void mma4_ss_warp(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 r, a1, a2, a3, b1, b2, b3;\n\t.reg .b64 x0, x1, x2, x3, y0, y1, y2, y3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "add.u32 a1, %1, 2;\n\tadd.u32 a2, %1, 4;\n\tadd.u32 a3, %1, 6;\n\t"
        "add.u32 b1, %2, 2;\n\tadd.u32 b2, %2, 4;\n\tadd.u32 b3, %2, 6;\n\t"
        "mov.b64 x0, {%1, %5};\n\tmov.b64 x1, {a1, %5};\n\tmov.b64 x2, {a2, %5};\n\tmov.b64 x3, {a3, %5};\n\t"
        "mov.b64 y0, {%2, %5};\n\tmov.b64 y1, {b1, %5};\n\tmov.b64 y2, {b2, %5};\n\tmov.b64 y3, {b3, %5};\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x0, y0, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x1, y1, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x2, y2, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x3, y3, %3, 1;\n\t}" ::"r"(d_tmem),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHiSW128)
        : "memory");
}
__device__ __forceinline__ void mma4_ts_warp(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b32 r, a1, a2, a3, b1, b2, b3;\n\t.reg .b64 y0, y1, y2, y3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
        "add.u32 b1, %2, 2;\n\tadd.u32 b2, %2, 4;\n\tadd.u32 b3, %2, 6;\n\t"
        "mov.b64 y0, {%2, %5};\n\tmov.b64 y1, {b1, %5};\n\tmov.b64 y2, {b2, %5};\n\tmov.b64 y3, {b3, %5};\n\t"
        "elect.sync r|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y0, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], y1, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], y2, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], y3, %3, 1;\n\t}" ::"r"(d_tmem),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHiSW128)
        : "memory");
}
// The low word of a 128-byte swizzled operand's descriptor.
__device__ __forceinline__ uint32_t desc_lo(const void* p) { return 1u << 16 | (smem_u32(p) >> 4 & 0x3FFFu); }

template <int D, bool M>
__global__ void __launch_bounds__(256, 2) kv4_long_kernel(const Kv4AttnArgs a) {
    using C = TcCfg<D, M>;
    constexpr int ST = C::kStages;
    constexpr int kDims = D / 2;  // dims of a row per thread
    extern __shared__ uint8_t smem_base[];
    __shared__ uint64_t bar;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ uint8_t dead[ST][4];     // pieces that are not there
    __shared__ uint32_t v_top[2][2];    // largest value scale of a tile's halves (bits)
    __shared__ float ex[3][2][128];     // exchange between a row's two threads
    uint8_t* qop = smem_base + (1024 - smem_u32(smem_base) % 1024) % 1024;
    uint8_t* kop = qop + C::kQ;
    uint8_t* vop = kop + C::kK;
    uint8_t* raw = vop + C::kV;
    float* pairs = reinterpret_cast<float*>(raw + ST * C::kRaw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int quad = warp & 3, tq = warp >> 2;  // tensor-memory lanes 32 quad ..; half of the tile's tokens
    const int row = quad * 32 + lane;
    asm volatile("griddepcontrol.launch_dependents;");
    // Tensor memory is taken only when the grid before this one is done: one that allocates
    // after its own trigger (the product kernel does) could otherwise wait for columns that
    // this block holds while it waits for that grid.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) {
        tmem_alloc(&s_tmem, C::kCols);
        tmem_relinquish();  // (the SM's other block allocates too)
    }
    if (tid == 0) {
        mbar_init(&bar, 1);
        fence_barrier_init();
        s_abort = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = s_tmem;
    const uint32_t tl = tm + ((uint32_t)(quad * 32) << 16);  // this warp's lanes
    volatile int* abort = &s_abort;
    const uint32_t q_lo = desc_lo(qop), k_lo = desc_lo(kop), v_lo = desc_lo(vop);

    const AttnRun run = attn_plan<C>(a);
    if (tid == 0) a.notes[blockIdx.x].rows = 0;
    const int64_t block = (int64_t)a.s.page * (D / 2 + 4);
    uint32_t phase = 0;  // of bar

    uint32_t seq = run.seq, in_seq = run.in_seq;
    for (uint32_t unit = run.begin; unit < run.end;) {
        const AttnSeg sg(a, C{}, seq, in_seq, run.end - unit);
        const int used = min((int)sg.t1, (sg.kv_end + C::kTokens - 1) / C::kTokens);
        const int count = used - (int)sg.t0;
        const int tok_base = (int)sg.t0 * C::kTokens;

        // ---- copies: warps 0-3 a piece's keys, warps 4-7 a piece's values
        const int piece = warp & 3;
        AttnPages pages;
        auto issue = [&](int i, int stage) {
            if ((i & 31) == 0) {
                const int tok = tok_base + (i + lane) * C::kTokens + piece * 16;
                pages.look_up(a, C{}, sg.b, sg.head, block, tok, i + lane < count && tok < sg.kv_end);
            }
            const uint64_t addr = __shfl_sync(0xffffffffu, pages.addr, i & 31);
            const uint32_t off = __shfl_sync(0xffffffffu, pages.off, i & 31);
            if (warp < 4 && lane == 0) dead[stage][piece] = addr == 0;
            if (addr) {
                const uint8_t* from = reinterpret_cast<const uint8_t*>(addr) + (warp < 4 ? 0 : block);
                const uint32_t to = smem_u32(raw) + stage * C::kRaw;
#pragma unroll
                for (int c = 0; c < D / 64; ++c)  // 16 tokens of D / 2 bytes
                    cp_async16(to + (warp < 4 ? 0 : C::kRawK) + piece * 8 * D + (lane + 32 * c) * 16,
                               from + off * (D / 2) + (lane + 32 * c) * 16);
                if (lane < 4)
                    cp_async16(to + 2 * C::kRawK + (warp < 4 ? 0 : 4 * C::kTokens) + piece * 64 + lane * 16,
                               from + (uint32_t)a.s.page * (D / 2) + off * 4 + lane * 16);
            }
            cp_commit();
        };
        issue(0, 0);
        issue(1, 1);

        // ---- the row's query, scaled, as an operand: rows of 128 bytes, 64 dims each
        float ca, cb;  // logit = ca * (s_k * S + z_k * cb)
        {
            float v[kDims];
            if (row < sg.rows) {
                const char* q = static_cast<const char*>(a.q) + (sg.query(a, C{}, row) + tq * kDims) * (a.q_f32 ? 4 : 2);
#pragma unroll
                for (int i = 0; i < kDims / 8; ++i) {
                    float u[8];
                    if (a.q_f32)
                        kv4_load8(reinterpret_cast<const float*>(q) + i * 8, a.q_vec, u);
                    else
                        kv4_load8(reinterpret_cast<const __nv_bfloat16*>(q) + i * 8, a.q_vec, u);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[i * 8 + j] = u[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < kDims; ++j) v[j] = 0.0f;
            }
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < kDims; ++j) amax = max_nan(amax, fabsf(v[j]));
            ex[0][tq][row] = amax;
            __syncthreads();
            amax = max_nan(ex[0][0][row], ex[0][1][row]);
            const int e = query_exponent(amax);
            const float up = pow2i(e);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < kDims / 8; ++i) {
                uint32_t p[4];
                sum += pack_query(v + i * 8, up, p);
                const int j = tq * (kDims / 8) + i;
                *reinterpret_cast<uint4*>(qop + (j >> 3) * 16384 + row * 128 + (((j & 7) ^ (row & 7)) * 16)) =
                    make_uint4(p[0], p[1], p[2], p[3]);
            }
            ex[1][tq][row] = sum;
            __syncthreads();
            sum = ex[1][0][row] + ex[1][1][row];
            ca = a.scale_log2 * pow2i(24 - e);
            cb = sum * 0x1p-24f;
        }
        const int lim = row < sg.rows && !(C::kMore && a.s.grouped) ? sg.pos0 + (int)(((uint32_t)sg.r0 + row) / a.G) : sg.kv_end - 1;

        // ---- spreading of a tile's codes
        auto spread_keys = [&](int i, int stage) {
            const uint8_t* st = raw + stage * C::kRaw;
            constexpr int kQuads = D / 32;  // groups of four words (32 dims) per token
            if (tid < C::kTokens * kQuads) {
                const int tok = tid / kQuads, qr = tid % kQuads;
                uint4 u = *reinterpret_cast<const uint4*>(st + tok * (D / 2) + qr * 16);
                // lanes of one store phase: two tokens, all quads; the upper two write their words in
                // the order 2, 3, 0, 1, so that all eight meet different banks
                const bool swap = qr & 2;
                if (swap) u = make_uint4(u.z, u.w, u.x, u.y);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int j = qr * 4 + (swap ? k ^ 2 : k);  // the word: eight dims, one 16-byte chunk
                    const uint32_t x = w[k], y = x >> 8;
                    *reinterpret_cast<uint4*>(kop + (j >> 3) * (C::kTokens * 128) + tok * 128 + (((j & 7) ^ (tok & 7)) * 16)) =
                        make_uint4(x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u);
                }
            }
            // the pairs as fp32: 64 threads the keys', 64 the values'
            if (tid < 2 * C::kTokens) {
                const int tok = tid % C::kTokens, kv = tid / C::kTokens;
                const uint32_t p = *reinterpret_cast<const uint32_t*>(st + 2 * C::kRawK + kv * 4 * C::kTokens + tok * 4);
                float* to = pairs + (i & 1) * 4 * C::kTokens + kv * 2 * C::kTokens + tok;
                const bool none = dead[stage][tok >> 4] || tok_base + i * C::kTokens + tok >= sg.kv_end;
                to[0] = none ? 0.0f : pair_lo(p);  // whatever lies behind the sequence
                // (a dead piece's tokens are told by a zero of +inf: their logits are dropped)
                to[C::kTokens] = !none ? pair_hi(p) : !kv && dead[stage][tok >> 4] ? INFINITY : 0.0f;
                if (kv) {
                    const float top = none ? 0.0f : fmaxf(pair_lo(p), 0.0f);  // (a NaN does not count)
                    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
                    if (lane == 0) v_top[i & 1][tok / 32] = bits;  // (a warp has one half's tokens)
                }
            }
        };
        auto spread_values = [&](int stage) {
            const uint8_t* st = raw + stage * C::kRaw + C::kRawK;
            constexpr int kWords = D / 4;  // words (four dims) of a token pair
            if (tid < 8 * kWords) {
                const int j = tid % kWords, q = tid / kWords;  // dims 4 j .. 4 j + 3, tokens 8 q .. 8 q + 7
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = *reinterpret_cast<const uint32_t*>(st + (4 * q + k) * D + j * 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int n = (k + (j >> 1)) & 3;  // the dims in turn, so that eight lanes meet different banks
                    const uint32_t sh = (n & 2) * 4, mask = n & 1 ? 0x00F000F0u : 0x000F000Fu;
                    const int r = 4 * j + n;
                    *reinterpret_cast<uint4*>(vop + r * 128 + ((q ^ (r & 7)) * 16)) =
                        make_uint4(w[0] >> sh & mask, w[1] >> sh & mask, w[2] >> sh & mask, w[3] >> sh & mask);
                }
            }
        };
        auto logits = [&]() {  // warp 0
#pragma unroll
            for (int k = 0; k < D / 64; ++k)
                mma4_ss_warp(tm + C::kColS, q_lo + k * (16384 >> 4), k_lo + k * (C::kTokens * 128 >> 4), C::kIdescS, k);
        };

        float neg_r = INFINITY, limit = kFirstLimit, loud = kFirstLoud;  // the row's reference
        float2 l2 = make_float2(0.0f, 0.0f), z2 = make_float2(0.0f, 0.0f);  // sums over this thread's tokens
        float base = 0.0f;  // what was taken out of its dims' sums, and the z term with it
        float2 x[16];
        // weights of tile i into tensor memory; kMask: some token is not seen by some row
        auto weights = [&](const float* pk, auto mask) {
            constexpr bool kMask = decltype(mask)::value;
            const float2 m2 = make_float2(neg_r, neg_r), ca2 = make_float2(ca, ca);
            uint32_t pw[16];
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
                const float4 vs = *reinterpret_cast<const float4*>(pk + 2 * C::kTokens + 2 * k),
                             vz = *reinterpret_cast<const float4*>(pk + 3 * C::kTokens + 2 * k);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float2 y = x[k + c], d = fma2(y, ca2, m2);
                    float2 p = make_float2(ex2f(d.x), ex2f(d.y));
                    const float2 s2 = c ? make_float2(vs.z, vs.w) : make_float2(vs.x, vs.y);
                    const float2 zz = c ? make_float2(vz.z, vz.w) : make_float2(vz.x, vz.y);
                    float2 pv;
                    if constexpr (kMask) {  // a token that a row does not see adds nothing, whatever its pair holds
                        const bool n0 = y.x == -INFINITY, n1 = y.y == -INFINITY;
                        p = make_float2(n0 ? 0.0f : p.x, n1 ? 0.0f : p.y);
                        z2 = add2(z2, make_float2(n0 ? 0.0f : p.x * zz.x, n1 ? 0.0f : p.y * zz.y));
                        pv = make_float2(n0 ? 0.0f : p.x * s2.x, n1 ? 0.0f : p.y * s2.y);
                    } else {
                        z2 = fma2(p, zz, z2);
                        pv = mul2(p, s2);
                    }
                    l2 = add2(l2, p);
                    pw[k + c] = pack_f16(pv.x, pv.y);
                }
            }
            tmem_st16(tl + C::kColP + tq * 16, pw);
            tmem_wait_st();
        };
        if (count > 0) {
            cp_wait<1>();
            __syncthreads();  // tile 0 is there for all
            spread_keys(0, 0);
            proxy_fence();
            tc_fence_before();
            __syncthreads();
            if (warp == 0) {
                tc_fence_after();
                logits();
                tc_commit_warp(&bar);
            }
        }
        int stage = 0, ahead = 1, fill = 2;  // of tiles i, i + 1, i + 2
        for (int i = 0; i < count; ++i) {
            const int b = i & 1;
            issue(i + 2, fill);  // (the stage of tile i - 1, done with before the last barrier)
            // ---- softmax of tile i, once its logits and the output of tile i - 1 are there
            mbar_wait(&bar, phase & 1, abort);
            ++phase;
            __syncwarp();
            tc_fence_after();
            {
                uint32_t u[2][16];
                tmem_ld16(tl + C::kColS + tq * 32, u[0]);
                tmem_ld16(tl + C::kColS + tq * 32 + 16, u[1]);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    x[k] = make_float2(__uint_as_float(u[k >> 3][2 * (k & 7)]), __uint_as_float(u[k >> 3][2 * (k & 7) + 1]));
            }
            const float* pk = pairs + b * 4 * C::kTokens + tq * 32;
            const int tok = tok_base + i * C::kTokens + tq * 32;
            float top = -INFINITY, vt = __uint_as_float(v_top[b][tq]);
            const float2 cb2 = make_float2(cb, cb);
            const bool lost = pk[C::kTokens] == INFINITY || pk[C::kTokens + 16] == INFINITY;
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
                const float4 ks = *reinterpret_cast<const float4*>(pk + 2 * k), kz = *reinterpret_cast<const float4*>(pk + C::kTokens + 2 * k);
                x[k] = fma2(make_float2(ks.x, ks.y), x[k], mul2(make_float2(kz.x, kz.y), cb2));
                x[k + 1] = fma2(make_float2(ks.z, ks.w), x[k + 1], mul2(make_float2(kz.z, kz.w), cb2));
            }
            const bool mask = lost || tok + 31 > sg.lim_min;  // the warp's threads agree
            if (mask) {
                const bool d0 = pk[C::kTokens] == INFINITY, d1 = pk[C::kTokens + 16] == INFINITY;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const bool none = k < 8 ? d0 : d1;
                    if (none || tok + 2 * k > lim) x[k].x = -INFINITY;
                    if (none || tok + 2 * k + 1 > lim) x[k].y = -INFINITY;
                }
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) top = fmaxf(top, fmaxf(x[k].x, x[k].y));
            top *= ca;
            cp_wait<1>();  // tile i + 1 (visible to all behind the barrier)
            if (__syncthreads_or(top + neg_r > limit || vt >= loud || (i > 0 && i % C::kCentre == 0))) {  // seldom
                if (mask) {  // the scales of the tokens that the row sees
                    vt = 0.0f;
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float2 vs = *reinterpret_cast<const float2*>(pk + 2 * C::kTokens + 2 * k);
                        if (x[k].x != -INFINITY) vt = fmaxf(vt, vs.x);
                        if (x[k].y != -INFINITY) vt = fmaxf(vt, vs.y);
                    }
                }
                ex[0][tq][row] = top;
                ex[1][tq][row] = vt;
                ex[2][tq][row] = z2.x + z2.y;
                __syncthreads();
                top = fmaxf(ex[0][0][row], ex[0][1][row]);
                vt = fmaxf(ex[1][0][row], ex[1][1][row]);
                const float f = raise_reference(top, vt, neg_r, limit);
                loud = loud_of(limit);
                l2 = mul2(l2, make_float2(f, f));
                z2 = make_float2(0.0f, 0.0f);
                if (i > 0) {  // the output so far, and back to about zero
                    float r = 0.0f;
#pragma unroll 1
                    for (int h = 0; h < kDims / 16; ++h) {
                        uint32_t u[16];
                        tmem_ld16(tl + C::kColO + tq * kDims + h * 16, u);
                        tmem_wait_ld();
                        if (h == 0) {
                            r = f * middle3(__uint_as_float(u[0]), __uint_as_float(u[2]), __uint_as_float(u[4]));
                            base = fmaf(base, f, fmaf(r, 16777216.0f, f * (ex[2][0][row] + ex[2][1][row])));
                        }
#pragma unroll
                        for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(fmaf(__uint_as_float(u[k]), f, k & 1 ? -16.0f * r : -r));
                        tmem_st16(tl + C::kColO + tq * kDims + h * 16, u);
                    }
                    tmem_wait_st();
                }
            }
            if (mask)
                weights(pk, std::true_type{});
            else
                weights(pk, std::false_type{});
            // ---- the operands of the next products
            spread_values(stage);
            if (i + 1 < count) spread_keys(i + 1, ahead);
            proxy_fence();
            tc_fence_before();
            __syncthreads();
            if (warp == 0) {
                tc_fence_after();
                mma4_ts_warp(tm + C::kColO, tm + C::kColP, v_lo, C::kIdescO, i > 0);
                if (i + 1 < count) logits();
                tc_commit_warp(&bar);
            }
            const int done = stage;
            stage = ahead, ahead = fill, fill = done;
        }

        // ---- results
        if (count > 0) {
            mbar_wait(&bar, phase & 1, abort);
            ++phase;
            __syncwarp();
            tc_fence_after();
        }
        ex[0][tq][row] = l2.x + l2.y;
        ex[1][tq][row] = z2.x + z2.y;
        __syncthreads();
        const float l = ex[0][0][row] + ex[0][1][row], zs = base + (ex[1][0][row] + ex[1][1][row]);
        const bool whole = sg.t0 == 0 && sg.t1 == sg.nt;
        float* part = a.part + ((int64_t)blockIdx.x * 2 + (unit == run.begin ? 0 : 1)) * C::kPart;
        const float up = 16777216.0f, inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        const uint32_t rr = (uint32_t)sg.r0 + row, ri = rr / a.G;
        const int64_t out_row = ((sg.row0 + ri) * a.s.Hk + sg.head) * a.G + rr - ri * a.G, at = out_row * D + tq * kDims;
#pragma unroll
        for (int h = 0; h < kDims / 16; ++h) {
            uint32_t u[16];
            if (count > 0) {
                tmem_ld16(tl + C::kColO + tq * kDims + h * 16, u);
                tmem_wait_ld();
            } else {
#pragma unroll
                for (int k = 0; k < 16; ++k) u[k] = 0;
            }
            if (row < sg.rows) {
#pragma unroll
                for (int k = 0; k < 16; k += 4) {
                    const float4 y = make_float4(fmaf(__uint_as_float(u[k]), up, zs), fmaf(__uint_as_float(u[k + 1]), up * 0.0625f, zs),
                                                 fmaf(__uint_as_float(u[k + 2]), up, zs), fmaf(__uint_as_float(u[k + 3]), up * 0.0625f, zs));
                    if (whole)
                        store_out(a, at + h * 16 + k, y, inv);
                    else
                        *reinterpret_cast<float4*>(part + row * D + tq * kDims + h * 16 + k) = y;
                }
            }
        }
        if (C::kMore && whole && a.lse && tq == 0 && row < sg.rows) a.lse[out_row] = attn_lse(-neg_r, l);
        if (!whole && tq == 0 && row < sg.rows) part[C::kRows * D + row * 2] = -neg_r, part[C::kRows * D + row * 2 + 1] = l;
        if (tid == 0) attn_note(a, C{}, run, sg, unit);
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        unit += sg.t1 - sg.t0;
        in_seq += sg.t1 - sg.t0;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tm, C::kCols);
    }
}

// Joins the partial results of a row tile that several blocks share: block c of
// this grid those of the tile that ends in block c of the other, gridDim.y blocks
// sharing its rows.  The warps of a block are shared out over its rows; those of
// one row take its partial results in turn, then meet in shared memory.
constexpr int kJoinWarps = 8;  // at most
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) kv4_join_kernel(const Kv4AttnArgs a, int rt_rows) {
    constexpr int E = D / 32;  // dims per lane
    __shared__ float sh[kJoinWarps][D + 2];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int c1 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Kv4Join j = a.notes[c1];
    const int share = (rt_rows + gridDim.y - 1) / gridDim.y, from = blockIdx.y * share, to = min(from + share, j.rows);
    if (from >= to) return;
    const int warps = blockDim.x >> 5;
    int per_row = warps;  // of them per row
    while (per_row > 1 && warps / per_row < to - from && per_row > c1 - j.first) per_row /= 2;
    const int at_once = warps / per_row, part = warp % per_row;
    const int64_t size = (int64_t)rt_rows * (D + 2);
    for (int base = from; base < to; base += at_once) {
        const int r = base + warp / per_row;
        float mx = -INFINITY, sum = 0.0f, y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = 0.0f;
        if (r < to) {
#pragma unroll 8
            for (int c = j.first + part; c <= c1; c += per_row) {
                const float* p = a.part + ((int64_t)c * 2 + (c == j.first ? j.first_slot : 0)) * size;
                const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + rt_rows * D + r * 2));
                float u[E];
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] = __ldcg(p + r * D + e * 32 + lane);
                if (ml.x == -INFINITY && ml.y == 0.0f) continue;
                const float mn = fmaxf(mx, ml.x), f = mx == mn ? 1.0f : ex2f(mx - mn), k = ex2f(ml.x - mn);
                mx = mn;
                sum = fmaf(k, ml.y, sum * f);
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = fmaf(k, u[e], y[e] * f);
            }
        }
        if (per_row > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) sh[warp][e * 32 + lane] = y[e];
            if (lane == 0) sh[warp][D] = mx, sh[warp][D + 1] = sum;
            __syncthreads();
            if (part != 0) continue;
            float top = mx;
            for (int w = 1; w < per_row; ++w) top = fmaxf(top, sh[warp + w][D]);
            sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = 0.0f;
            for (int w = 0; w < per_row; ++w) {
                const float mw = sh[warp + w][D], lw = sh[warp + w][D + 1];
                if (mw == -INFINITY && lw == 0.0f) continue;
                const float f = ex2f(mw - top);
                sum = fmaf(f, lw, sum);
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = fmaf(f, sh[warp + w][e * 32 + lane], y[e]);
            }
        }
        if (r >= to) continue;
        const uint32_t rr = (uint32_t)j.r0 + r, i = rr / j.G;
        const int64_t at = (((j.row0 + i) * a.s.Hk + j.head) * j.G + rr - i * j.G) * D + lane;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (a.out_f32)
                static_cast<float*>(a.out)[at + e * 32] = y[e] * inv;
            else
                static_cast<__nv_bfloat16*>(a.out)[at + e * 32] = __float2bfloat16_rn(y[e] * inv);
        }
    }
}

// The kernel by the query rows that a sequence has on average for one kv head, and
// by the row tiles that this makes of the call.  A small tile reads and unpacks the
// cache more often, but gives the SMs more to share: up to four tiles of 16 rows
// per SM the 16-row kernel wins whatever the number of rows, from eight per SM
// on the larger one of the others.  In us for d = 128 (16 rows / chunk / tcgen05):
//   4 sequences x 128 rows x 8 heads of 2048 tokens (256 tiles)      46 /  61 /  93
//   one prompt of 500 tokens, 8 heads (256 tiles)                    28 /  43 /  36
//   8 x 144 x 8 heads of 2048 tokens (576 tiles)                     75 /  78 /  80
//   one prompt of 768 tokens, 12 heads (576 tiles)                   40 /  40 /  71
//   64 x 96 x 2 heads of 1024 tokens (768 tiles)                     65 /  63 /  66
//   32 prompts of 24 tokens, 12 heads (768 tiles)                    23 /  12 /  20
//   64 x 64 x 4 heads of 1024 tokens (1024 tiles)                    84 /  70 /  76
//   64 x 96 x 4 heads of 1024 tokens (1536 tiles)                   111 /  91 /  80
//   16 x 512 x 8 heads of 1024 tokens (4096 tiles)                  233 / 144 / 114
// and at 8 rows 23 against 34 (64 heads of 4096 tokens: the 8-row kernel, the 16-row
// one).  Where the rule is wrong: few tiles over very long sequences (290
// tokens x 4 behind 8192, 584 tiles: 196 / 179 / 152), many prompts of 128 to 512
// tokens (32 x 128, 12 heads: 81 / 38 / 52; d = 64, 16 x 512: 125 / 67 / 75), and a
// prompt among single tokens, whose sequences all go to the kernel that their mean
// asks for; the host knows neither lengths nor rows.
enum AttnKind { kAttn8, kAttn16, kAttnChunk, kAttnLong };
static AttnKind attn_kind(int64_t B, int64_t T, int64_t Hk, int64_t G) {
    const int64_t rows = (T + B - 1) / B * G, tiles = (rows + 15) / 16 * B * Hk;
    const int64_t sms = sm_count();
    if (rows <= 16 || tiles <= 4 * sms) return rows <= 8 ? kAttn8 : kAttn16;
    return rows <= 64 || tiles <= 8 * sms ? kAttnChunk : kAttnLong;
}
static int attn_blocks(AttnKind kind) {  // blocks that the device holds at once
    return sm_count() * (kind == kAttnLong ? TcCfg<128, false>::kBlocks : AttnCfg<128, 1, false>::kBlocks);
}
static size_t attn_notes_bytes(int blocks) { return ((size_t)blocks * sizeof(Kv4Join) + 255) / 256 * 256; }
static size_t attn_part_bytes(AttnKind kind, int64_t D) {
    constexpr int rows[4] = {8, 16, 64, 128};
    return (size_t)attn_blocks(kind) * 2 * rows[kind] * (D + 2) * 4;
}
// Bytes of the notes and partial results of one pass.
static size_t attn_workspace(AttnKind kind, int64_t D) {
    return attn_notes_bytes(attn_blocks(kind)) + attn_part_bytes(kind, D);
}
static size_t attn_workspace(int64_t B, int64_t T, int64_t Hk, int64_t G, int64_t D) {
    return B == 0 || T == 0 ? 0 : attn_workspace(attn_kind(B, T, Hk, G), D);
}

template <int D, typename C>
static cudaError_t launch_attn(void (*kernel)(Kv4AttnArgs), const Kv4AttnArgs& a, AttnKind kind, cudaStream_t s) {
    static std::atomic<bool> done[64];  // false at first
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) done[dev] = true;
    }
    const int blocks = attn_blocks(kind);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess || a.where) return e;
    // Few tiles have many partial results each: more blocks and warps per tile.
    // Many tiles: fewer, most blocks find nothing to join.  (8 tiles of 55
    // partial results: 41 us with 8 x 8 warps, 47 us with 4 x 4; 256 tiles of 2:
    // 52 us and 47 us.)
    const int64_t tiles = (a.s.B + a.s.T * a.G / C::kRows) * a.s.Hk;
    const bool few = tiles * 8 <= blocks;
    cfg.gridDim = dim3((unsigned)blocks, few ? 8 : 4);
    cfg.blockDim = dim3(few ? kJoinWarps * 32 : kJoinWarps * 16);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D>, a, (int)C::kRows);
}

// One pass: its kernel and (where no other kernel does) the one that joins, with notes and partial
// results at ws.  M: whether the rows or tables are other than pn_kv4_attention's; that is a matter of the kernels'
// type, since the tests for it made that one 3 to 10 % slower (one row of 12 heads over 513 tokens: 9.3 and 10.2 us).
template <bool M>
static cudaError_t attn_pass(Kv4AttnArgs& a, AttnKind kind, int64_t head_dim, void* ws, cudaStream_t s) {
    a.notes = static_cast<Kv4Join*>(ws);
    a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + attn_notes_bytes(attn_blocks(kind)));
    auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        switch (kind) {
            case kAttn8: return launch_attn<D, AttnCfg<D, 1, M>>(kv4_decode_kernel<D, 1, M>, a, kind, s);
            case kAttn16: return launch_attn<D, AttnCfg<D, 2, M>>(kv4_decode_kernel<D, 2, M>, a, kind, s);
            case kAttnChunk: return launch_attn<D, ChunkCfg<D, M>>(kv4_chunk_kernel<D, M>, a, kind, s);
            default: return launch_attn<D, TcCfg<D, M>>(kv4_long_kernel<D, M>, a, kind, s);
        }
    };
    return head_dim == 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

}  // namespace pn

// The queries and outputs of an attention call, a.s being there already.
static int check_attn(const char* name, const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh, int q_dtype, int64_t q_heads,
                      const void* cache, float scale, void* out, pn::Kv4AttnArgs* a) {
    const pn::Kv4Seq& s = a->s;
    if (q_dtype != PN_F32 && q_dtype != PN_BF16) return fail(PN_ERR_DTYPE, "%s: dtype %d", name, q_dtype);
    if (q_heads < 1 || q_heads % s.Hk != 0 || q_heads > 65536)
        return fail(PN_ERR_SHAPE, "%s: %lld query heads over %d kv heads", name, (long long)q_heads, s.Hk);
    if (s.T > 0 && s.B > 0 && (!q || !out)) return fail(PN_ERR_ARG, "%s: null pointer", name);
    if (!(scale > 0.0f && scale < INFINITY)) return fail(PN_ERR_ARG, "%s: scale must be positive", name);
    const size_t e = q_dtype == PN_F32 ? 4 : 2;
    if (!aligned(q, e) || !aligned(out, 16)) return fail(PN_ERR_ALIGN, "%s: misaligned pointer", name);
    a->q = q, a->q_f32 = a->out_f32 = q_dtype == PN_F32, a->q_sb = q_sb, a->q_sl = q_sl, a->q_sh = q_sh;
    const int64_t n = 16 / (int64_t)e;
    a->q_vec = aligned(q, 16) && q_sb % n == 0 && q_sl % n == 0 && q_sh % n == 0;
    a->cache = static_cast<const uint8_t*>(cache);
    a->G = (int)(q_heads / s.Hk);
    a->scale_log2 = scale * 1.4426950408889634f;
    a->out = out;
    return PN_OK;
}
// Upper bounds on the rows and units that the kernels count in 31 bits.
static int check_attn_units(const char* name, const pn::Kv4Seq& s, int64_t G, int64_t tokens) {
    if (s.B > 0 && ((double)s.T * G > 2e9 || ((double)s.T * G / 8 + s.B) * s.Hk * ((double)tokens / 64 + 1) > 2e9))
        return fail(PN_ERR_SHAPE, "%s: %lld rows over tables of %lld tokens are too much for one call", name, (long long)s.T,
                    (long long)tokens);
    return PN_OK;
}

extern "C" {

size_t pn_kv4_attention_workspace_size(int64_t B, int64_t T, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
    if (B < 0 || T < 0 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1) return 0;
    return pn::attn_workspace(B, T, kv_heads, q_heads / kv_heads, head_dim);
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
    if (int st = check_attn("pn_kv4_attention", q, q_sb, q_sl, q_sh, q_dtype, q_heads, cache, scale, out, &a)) return st;
    if (int st = check_attn_units("pn_kv4_attention", a.s, a.G, table_w * page)) return st;
    if (int st = check_device()) return st;
    if (T == 0 || B == 0) return ok();
    const pn::AttnKind kind = pn::attn_kind(B, T, kv_heads, a.G);
    const size_t need = pn::attn_workspace(kind, head_dim);
    if (!workspace || workspace_bytes < need)
        return fail(PN_ERR_WORKSPACE, "pn_kv4_attention: workspace needs %zu bytes", need);
    if (!aligned(workspace, 256)) return fail(PN_ERR_ALIGN, "pn_kv4_attention: the workspace needs 256-byte alignment");
    const cudaError_t err = pn::attn_pass<false>(a, kind, head_dim, workspace, (cudaStream_t)stream);
    return err == cudaSuccess ? ok() : cuda_fail(err, "pn_kv4_attention");
}

}  // extern "C"
