// pn_kv4_prefix.cu -- causal attention of sequences that share long prefixes by groups, over
// the 4-bit paged cache (layout: pn_kv4.cu): a prefix's tokens are read, unpacked and
// multiplied once for the rows of all its sequences.
//
// Mathematics.  A row sees the prefix and then its own sequence; with (y_i, lse_i) the
// results over either part and the logarithms (base 2) of their softmax totals,
//   y = sum_i 2^(lse_i - M) y_i / sum_i 2^(lse_i - M),  M = max lse_i.
//
// Three kernels.  The rows over the prefixes and the rows over their own sequences go through the
// kernels of pn_kv4_attn.cu: there a prefix is a "sequence" whose rows, those of all its
// sequences, see all of it.  Both leave fp32 results in the workspace, and those of tiles that
// were split over blocks in parts.  The third kernel (here) joins whatever either left, so
// that no pass needs a joining kernel of its own.
//
// What bounds it: over the prefix, that a step's softmax and the spreading of its codes stand between
// the block's barriers (issue slots 40 %, tensor pipe 16 %), and that the passes run one behind the
// other.  64 sequences x 8 heads of 128 dims x 8 rows a head over 8192 tokens: 65 us over the prefix,
// the rows' own 1000 tokens 39, the joining 13, together 107 as each begins before the one in front has
// ended.  A kernel for the prefix alone was built too (256 rows to a tile,
// warps by task, the logits of a step formed while the softmax of the one before ran): 75 us
// there and 186 over one prefix of 131071 tokens for 64 rows a head, where the chunk kernel
// took 148; its five kinds of warps did not fit the instruction cache, and it was given up.
#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

struct Kv4MergeArgs {
    Kv4Seq s;                  // the sequences
    const int32_t* grp;        // shares of the prefixes, or null
    int64_t P;
    int G;
    // of the passes over the sequences and over the prefixes
    const float* y[2];         // whole results
    const float* lse[2];
    const Kv4Where* where[2];
    const float* part[2];
    int tile[2];               // rows of their row tiles
    void* out;
    int out_f32;
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
    if (falls || !kv4_find(a.s, row, b, i)) return;
    float mx = -INFINITY, sum = 0.0f, y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.0f;
    const int hk = h / a.G, gq = h - hk * a.G;
    // own results
    const int64_t r = i * a.G + gq, r0 = r / a.tile[0] * a.tile[0];
    const Kv4Where own = a.where[0][((row - i + r0 / a.G) * a.s.Hk + hk) * a.G + r0 % a.G];
    const int n_own = own.last < 0 ? 1 : own.last - own.first + 1;
    // the prefix's
    Kv4Where pre = {};
    int n_pre = 0;
    int64_t pr = 0;  // the row in its row tile
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
        kv4_rows<true>(p, g, first, n);
        pr = (row - first) * a.G + gq;
        const int64_t t0 = pr / a.tile[1] * a.tile[1];
        pre = a.where[1][((first + t0 / a.G) * a.s.Hk + hk) * a.G + t0 % a.G];
        pr -= t0;
        n_pre = pre.last < 0 ? 1 : pre.last - pre.first + 1;
    }
    for (int base = 0; base < n_own + n_pre; base += 32) {
        const int n = min(n_own + n_pre - base, 32), j = base + lane;
        const float* from = a.y[0];  // (somewhere, for lanes without one)
        float m = -INFINITY, l = 0.0f;
        if (lane < n) {
            const int which = j < n_own ? 0 : 1, k = which ? j - n_own : j;
            const Kv4Where w = which ? pre : own;
            if (w.last < 0) {
                from = a.y[which] + at * D;
                m = a.lse[which][at], l = 1.0f;
            } else {
                const int tile = a.tile[which];
                const int64_t tr = which ? pr : r - r0;
                const float* p0 = a.part[which] + ((int64_t)(w.first + k) * 2 + (k == 0 ? w.first_slot : 0)) * tile * (D + 2);
                from = p0 + tr * D;
                const float2 ml = *reinterpret_cast<const float2*>(p0 + tile * D + tr * 2);
                m = ml.x, l = ml.y;
            }
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
        // Results are read so many at once, no load behind a branch or behind another's use: 512 rows of 55, the longest
        // lists, 23 us (37 where the compiler orders them, four at a time), 768 rows of two to four 27 (33 with eight for all).
        auto add = [&](auto at_once) {
            constexpr int N = decltype(at_once)::value;
#pragma unroll 1
            for (int k = 0; k < n; k += N) {
                float u[N][E];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(from), k + j));
                    if constexpr (E == 4)
                        asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(u[j][0]), "=f"(u[j][1]), "=f"(u[j][2]), "=f"(u[j][3]) : "l"(src + lane * 4));
                    else
                        asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(u[j][0]), "=f"(u[j][1]) : "l"(src + lane * 2));
                }
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const bool on = some >> (k + j) & 1;  // (what weighs nothing may be no number)
                    const float wk = __shfl_sync(0xffffffffu, w, k + j);
#pragma unroll
                    for (int e = 0; e < E; ++e) y[e] = on ? fmaf(wk, u[j][e], y[e]) : y[e];
                }
            }
        };
        if (n <= 2)
            add(std::integral_constant<int, 2>{});
        else if (n <= 4)
            add(std::integral_constant<int, 4>{});
        else
            add(std::integral_constant<int, 8>{});
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

// The kernel for the rows over the prefixes, which walk long sequences together; the host knows no
// more of the lengths than the table's width.
// Not attn_kind's rule: the tiles are few, but their walks long.  A call in us with the kernels for 8, 16, 64 and
// 128 rows, 8 heads of 128 dims:
//   64 rows a head over 131071 tokens      - / 202 / 185 / 174
//   128 rows over 8192 tokens              - /  58 /  59 /  58
//   32, 16, 8 rows there                  36 /  47 /  52 /  48,  34 / 41 / 50 / 46,  33 / 40 / 46 / 45
// Where the rule is wrong: few rows over a prefix of some thousand tokens (the 8-row kernel leads up to 32), 64
// rows over very long ones (the tcgen05 kernel does), and shares that are not alike, as it knows their mean: of eight
// prefixes of 8192 tokens with 500 rows behind one the chunk kernel is taken, 154 (tcgen05 124).
static AttnKind prefix_kind(int64_t P, int64_t T, int64_t Hk, int64_t G) {
    const int64_t rows = (T + P - 1) / P * G;
    if (rows <= 16) return rows <= 8 ? kAttn8 : kAttn16;
    return rows <= 64 ? kAttnChunk : kAttnLong;
}

// Parts of the workspace.
struct PrefixLayout {
    AttnKind own, prefix;
    size_t y, lse, where[2], pass[2], total;
    PrefixLayout(int64_t B, int64_t T, int64_t P, int64_t Hk, int64_t G, int64_t D)
        : own(attn_kind(B, T, Hk, G)), prefix(prefix_kind(P, T, Hk, G)) {
        const size_t rows = (size_t)T * Hk * G;
        y = 0;  // of either pass
        lse = y + round256(2 * rows * D * 4);
        where[0] = lse + round256(2 * rows * 4);
        where[1] = where[0] + round256(rows * sizeof(Kv4Where));
        pass[0] = where[1] + round256(rows * sizeof(Kv4Where));
        pass[1] = pass[0] + round256(attn_workspace(own, D));
        total = pass[1] + attn_workspace(prefix, D);
    }
};

template <int D>
static cudaError_t launch_merge(const Kv4MergeArgs& m, cudaStream_t s) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)m.s.T, (unsigned)((m.s.Hk * m.G + kMergeWarps - 1) / kMergeWarps));
    cfg.blockDim = dim3(kMergeWarps * 32);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_merge_kernel<D>, m);
}

}  // namespace pn

extern "C" {

size_t pn_kv4_prefix_attention_workspace_size(int64_t B, int64_t T, int64_t n_prefixes, int64_t q_heads, int64_t kv_heads,
                                              int64_t head_dim) {
    if (B < 1 || T < 1 || n_prefixes < 0 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1) return 0;
    if (n_prefixes == 0) return pn_kv4_attention_workspace_size(B, T, q_heads, kv_heads, head_dim);
    return pn::PrefixLayout(B, T, n_prefixes, kv_heads, q_heads / kv_heads, head_dim).total;
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
    const pn::PrefixLayout lay(B, T, n_prefixes, kv_heads, a.G, head_dim);
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
    // the rows over the prefixes
    p.s = prefixes;
    p.q_l = cu_q ? 0 : own.L;
    p.out = y + rows * head_dim, p.lse = lse + rows, p.where = reinterpret_cast<pn::Kv4Where*>(ws + lay.where[1]);
    cudaError_t err = pn::attn_pass<true>(p, lay.prefix, head_dim, ws + lay.pass[1], s);
    if (err != cudaSuccess) return cuda_fail(err, name);
    // and over their own sequences
    a.out = y, a.lse = lse, a.where = reinterpret_cast<pn::Kv4Where*>(ws + lay.where[0]);
    err = pn::attn_pass<true>(a, lay.own, head_dim, ws + lay.pass[0], s);
    if (err != cudaSuccess) return cuda_fail(err, name);
    constexpr int tile[4] = {8, 16, 64, 128};
    pn::Kv4MergeArgs m{};
    m.s = own, m.grp = cu_prefix, m.P = n_prefixes, m.G = a.G;
    m.y[0] = y, m.y[1] = y + rows * head_dim;
    m.lse[0] = lse, m.lse[1] = lse + rows;
    m.where[0] = a.where, m.where[1] = p.where;
    m.part[0] = a.part, m.part[1] = p.part;
    m.tile[0] = tile[lay.own], m.tile[1] = tile[lay.prefix];
    m.out = out, m.out_f32 = q_dtype == PN_F32;
    err = head_dim == 64 ? pn::launch_merge<64>(m, s) : pn::launch_merge<128>(m, s);
    return err == cudaSuccess ? ok() : cuda_fail(err, name);
}

}  // extern "C"
