// pn_kv4_sparse.cu -- attention over chosen pages of the 4-bit paged cache (layout:
// pn_kv4.cu): the mean key of each page, a score of the means for each row, the choice,
// and the attention kernels of pn_kv4_attn.cu over the pages chosen.
//
// Mathematics.  A page's mean key in a head is (sum_t s_t c_t + z_t) / n over its n tokens,
// rounded to bf16; page i scores (sum of the group's queries) . mean_i for a row.  The
// first and the last pages that the row sees are taken, and of the others the `top` largest
// scores, ties by the lowest page.  Two scores that are close decide which page is read,
// so sums and scores are fp64: a choice then depends on no order of summing short of
// scores that agree to 2^-45 or so, and is the formula's.
//
// The chosen pages become a block table of the row's own, one for each kv head, in ascending
// order, so the row's last page is the last and the only one that it may see in part;
// the attention kernels walk it as any table, a row as a sequence of one.
#include "pn_common.cuh"
#include "pn_internal.h"

namespace pn {

// ---- means ------------------------------------------------------------------

struct Kv4MeansArgs {
    Kv4Seq s;
    const uint8_t* cache;
    __nv_bfloat16* means;  // (n_pages, Hk, D)
    int rows;              // per block
};
constexpr int kMeansThreads = 128;
constexpr int kMeansRows = 64;  // per block, at most

// A block looks at a few rows: one that is its sequence's last, or whose successor starts a
// page, stands for its page.  The block's warps share the tokens of each such page, lane
// (token parity, word of eight dims), in fp64.  A code times its scale is exact in fp32, where a sixteenth of
// the largest scales keeps it below the largest number.  (Products in fp64, whose conversions from integers are
// slow: a page of 256 tokens 11.7 us, 7.7 so.)
template <int D>
__global__ void __launch_bounds__(kMeansThreads) kv4_means_kernel(const Kv4MeansArgs a) {
    constexpr int WORDS = D / 8, TP = 32 / WORDS, WARPS = kMeansThreads / 32;  // words of a key, tokens per warp and step
    __shared__ int64_t at[kMeansRows];
    __shared__ int held[kMeansRows];
    __shared__ int count;
    __shared__ double sums[WARPS * TP][D + 1];
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) count = 0;
    __syncthreads();
    const int64_t row = (int64_t)blockIdx.x * a.rows + tid;
    int64_t b, i;
    if (tid < a.rows && row < a.s.T && kv4_find(a.s, row, b, i)) {
        int64_t first, n;
        kv4_rows(a.s, b, first, n);
        const int len = kv4_len(a.s, b);
        const int64_t pos = len - n + i;
        if (pos >= 0 && (i == n - 1 || (pos + 1) % a.s.page == 0)) {
            const int64_t page = kv4_page(a.s, b, (int)pos);
            if (page >= 0) {
                const int k = atomicAdd(&count, 1);  // (pages are done one by one: their order does not matter)
                at[k] = page;
                held[k] = (int)min((int64_t)a.s.page, len - pos / a.s.page * a.s.page);
            }
        }
    }
    __syncthreads();
    const int64_t block = (int64_t)a.s.page * (D / 2 + 4);
    const int word = lane % WORDS, sub = warp * TP + lane / WORDS;
    for (int k = 0; k < count; ++k) {
        const int64_t head = at[k] * a.s.Hk + blockIdx.y;
        const uint8_t* p = a.cache + head * 2 * block;
        const int n = held[k];
        double acc[8], zeros = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.0;
#pragma unroll 4
        for (int t = sub; t < n; t += WARPS * TP) {
            const uint32_t c = *reinterpret_cast<const uint32_t*>(p + t * (D / 2) + word * 4);
            const uint32_t pair = *reinterpret_cast<const uint32_t*>(p + a.s.page * (D / 2) + t * 4);
            const float s = __uint_as_float(pair << 16), z = __uint_as_float(pair & 0xFFFF0000u);
            const bool large = s >= 0x1p123f;
            const float less = large ? s * 0.0625f : s;
            const double up = large ? 16.0 : 1.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fma((double)(less * (float)(c >> (4 * j) & 15)), up, acc[j]);
            zeros += (double)z;
        }
        __syncthreads();  // the sums of the page before are read
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[sub][word * 8 + j] = acc[j] + zeros;
        __syncthreads();
        for (int d = tid; d < D; d += kMeansThreads) {
            double sum = 0.0;
#pragma unroll
            for (int w = 0; w < WARPS * TP; ++w) sum += sums[w][d];
            a.means[head * D + d] = __float2bfloat16_rn(__double2float_rn(sum / n));
        }
    }
}

// ---- scores -----------------------------------------------------------------

// Scores as keys whose order as integers is theirs as numbers; 0: a NaN, or a page that is not
// there, taken last.
__device__ __forceinline__ uint64_t score_key(double v) {
    if (v != v) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);  // -0 counts as 0
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

struct Kv4SelectArgs {
    Kv4Seq s;
    const void* q;
    int q_f32;
    int64_t q_sb, q_sl, q_sh;
    int G;
    const __nv_bfloat16* means;
    int first, last, top;
    int width;            // first + last + top
    int list;             // pages of a row's table: as many, or all that the block table has
    int64_t row0, row1;   // the rows of this launch
    uint64_t* keys;       // workspace (row1 - row0, Hk, table_w): scores
    int32_t* pages;       // workspace (T, Hk, list): the chosen pages, as entries of the block table
    int32_t* lens;        // workspace (T): tokens of them; -1: no row
    int32_t* chosen;      // (T, Hk, width): their numbers in the sequence, or null
    int tile;             // rows of a block of the score kernel
    int splits;           // blocks that share the pages
};
constexpr int kScoreThreads = 128;
constexpr int kScoreTile = 8;

// Where a row is: its sequence, and the pages [0, first), [first, free_end) and
// [free_end, seen) that are taken, may be chosen, and are taken.
struct SelectRow {
    int64_t b, i;
    int seen, free_end, len;  // len: tokens that the row sees; -1: no row
    bool over;                // the table has no room for all of them
    __device__ __forceinline__ SelectRow(const Kv4SelectArgs& a, int64_t row)
        : b(0), i(0), seen(0), free_end(0), len(-1), over(false) {
        if (row >= a.row1 || !kv4_find(a.s, row, b, i)) return;
        int64_t at, n;
        kv4_rows(a.s, b, at, n);
        const int64_t pos = (int64_t)kv4_len(a.s, b) - n + i;
        len = (int)min(max(pos + 1, (int64_t)0), (int64_t)a.s.table_w * a.s.page);
        over = pos >= (int64_t)a.s.table_w * a.s.page && a.s.table_w > 0;
        seen = (len + a.s.page - 1) / a.s.page;
        free_end = max(seen - a.last, 0);
    }
};

// A block scores some pages for up to `tile` rows of one kv head.  Four lanes share a page's
// mean, held as fp64 for all rows of a sequence; the group's queries are summed once per
// block.  Rows are taken four at a time: one by one the kernel waits for their loads from
// shared memory (251 rows of 250 pages and 157 of 138, 8 heads: 65 us, 79 one by one; the fp64 units
// are busy for a fourteenth of it).
template <int D>
__global__ void __launch_bounds__(kScoreThreads) kv4_score_kernel(const Kv4SelectArgs a) {
    constexpr int E = D / 4;  // dims per lane: chunks of 8, four lanes in turn
    __shared__ double q[kScoreTile][D];
    __shared__ int seq[kScoreTile], to[kScoreTile];
    __shared__ int64_t base[kScoreTile];
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row0 = a.row0 + (int64_t)blockIdx.x * a.tile;
    const int head = blockIdx.y;
    if (tid < a.tile) {
        const SelectRow at(a, row0 + tid);
        seq[tid] = max(at.free_end - a.first, 0) > a.top ? (int)at.b : -1;  // (with fewer pages all are taken)
        to[tid] = at.free_end;
        base[tid] = a.s.cu ? (row0 + tid) * a.q_sl : at.b * a.q_sb + at.i * a.q_sl;
    }
    __syncthreads();
#pragma unroll 4
    for (int k = tid; k < a.tile * D; k += kScoreThreads) {
        const int r = k / D, d = k % D;
        if (seq[r] < 0) continue;
        double sum = 0.0;
        for (int g = 0; g < a.G; ++g) {
            const int64_t p = base[r] + (int64_t)(head * a.G + g) * a.q_sh + d;
            sum += (double)(a.q_f32 ? static_cast<const float*>(a.q)[p]
                                    : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[p]));
        }
        q[r][d] = sum;
    }
    __syncthreads();
    const int part = lane & 3, sub = warp * 8 + (lane >> 2);
    for (int r0 = 0; r0 < a.tile;) {
        if (seq[r0] < 0) {
            ++r0;
            continue;
        }
        int r1 = r0 + 1, hi = to[r0];
        for (; r1 < a.tile && seq[r1] == seq[r0]; ++r1) hi = max(hi, to[r1]);
        const int64_t b = seq[r0];
        // the pages [first, hi) in runs of 32 to a block
        for (int run = a.first + blockIdx.z * 32; run < hi; run += a.splits * 32) {
            const int i = run + sub;
            const int p = i < hi ? __ldg(a.s.table + b * a.s.table_ld + i) : -1;
            const bool there = p >= 0 && p < a.s.n_pages;
            double m[E];
            const uint4* src = reinterpret_cast<const uint4*>(a.means + ((int64_t)p * a.s.Hk + head) * D);
#pragma unroll
            for (int c = 0; c < E / 8; ++c) {
                const uint4 u = there ? src[c * 4 + part] : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    m[c * 8 + 2 * j] = (double)__uint_as_float(w[j] << 16);
                    m[c * 8 + 2 * j + 1] = (double)__uint_as_float(w[j] & 0xFFFF0000u);
                }
            }
            auto part_of = [&](int r) {  // this lane's part of the score of row r
                double sum = 0.0, sum2 = 0.0;
#pragma unroll
                for (int c = 0; c < E / 8; ++c)
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const double2 x = *reinterpret_cast<const double2*>(&q[r][(c * 4 + part) * 8 + j]);
                        sum = fma(x.x, m[c * 8 + j], sum);
                        sum2 = fma(x.y, m[c * 8 + j + 1], sum2);
                    }
                return sum + sum2;
            };
            auto put = [&](int r, double sum) {
                if (i < to[r]) a.keys[((row0 - a.row0 + r) * a.s.Hk + head) * a.s.table_w + i] = there ? score_key(sum) : 0;
            };
            if (r1 - r0 == 1) {
                double sum = part_of(r0);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if (part == 0) put(r0, sum);
                continue;
            }
            // four rows at once: their loads and sums do not wait for one another, and each lane ends with one row
            for (int r = r0; r < r1; r += 4) {
                double s[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) s[k] = part_of(min(r + k, r1 - 1));
                const bool odd = part & 1, high = part & 2;
                const double two[2] = {(odd ? s[1] : s[0]) + __shfl_xor_sync(0xffffffffu, odd ? s[0] : s[1], 1),
                                       (odd ? s[3] : s[2]) + __shfl_xor_sync(0xffffffffu, odd ? s[2] : s[3], 1)};
                const double sum = (high ? two[1] : two[0]) + __shfl_xor_sync(0xffffffffu, high ? two[0] : two[1], 2);
                if (r + part < r1) put(r + part, sum);
            }
        }
        r0 = r1;
    }
}

// ---- choice -----------------------------------------------------------------

constexpr int kSelectBins = 2048;
constexpr int kSelectFew = 256;  // keys that are ranked one against another

// The score of a key, to fp32 (which keeps their order).
__device__ __forceinline__ float score_of(uint64_t k) {
    return __double2float_rn(__longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k)));
}
// Bin of a key, from evenly spaced ones between the least and the largest finite score (which are at
// lo and lo + 2047 / each): never higher for a smaller key.
__device__ __forceinline__ int score_bin(uint64_t k, float lo, float each) {
    if (k == 0) return 0;
    const float v = score_of(k);
    if (!(v < INFINITY)) return kSelectBins - 1;
    return (int)fminf(fmaxf((v - lo) * each, 0.0f), (float)(kSelectBins - 1));
}

// Counts from above: the bin where they reach `need`, and how many of it are needed.
template <int THREADS>
__device__ __forceinline__ void select_border(const int* bins, int need, int* warp_sums, int* border) {
    constexpr int PER = kSelectBins / THREADS;  // thread t has bins [PER (THREADS - 1 - t), + PER)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) mine += bins[(THREADS - 1 - tid) * PER + j];
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    for (int w = 0; w < warp; ++w) inc += warp_sums[w];
    int above = inc - mine;
    if (above < need && need <= inc) {
        int j = PER - 1;
        for (;; --j) {
            const int c = bins[(THREADS - 1 - tid) * PER + j];
            if (above + c >= need) break;
            above += c;
        }
        border[0] = (THREADS - 1 - tid) * PER + j;
        border[1] = need - above;
    }
    __syncthreads();
}

// A row's list in one kv head, and what of it does not depend on the scores.
struct SelectList {
    SelectRow at;
    int64_t row, unit;
    int head, n;   // n: pages that may be chosen
    bool choose;   // not all of them are
    const uint64_t* keys;
    const int32_t* table;
    __device__ __forceinline__ SelectList(const Kv4SelectArgs& a, int64_t u)  // u: of this launch's rows
        : at(a, a.row0 + u / a.s.Hk), row(a.row0 + u / a.s.Hk), unit(a.row0 * a.s.Hk + u), head((int)(unit - row * a.s.Hk)) {}
    // falls: so do row starts, and nothing is computed
    __device__ __forceinline__ void settle(const Kv4SelectArgs& a, bool falls, bool speaks) {
        if (falls) at.len = -1, at.seen = at.free_end = 0, at.over = true;
        if (at.over && head == 0 && speaks) record_status(PN_ERR_ARG);
        n = max(at.free_end - a.first, 0);
        choose = n > a.top;
        keys = a.keys + (unit - a.row0 * a.s.Hk) * a.s.table_w + a.first;
        table = a.s.table + at.b * a.s.table_ld;
    }
    __device__ __forceinline__ void put(const Kv4SelectArgs& a, int slot, int i) const {
        a.pages[unit * a.list + slot] = i < a.s.table_w ? __ldg(table + i) : -1;
        if (a.chosen) a.chosen[unit * a.width + slot] = i;
    }
    // The first and the last pages (or all), the rest of the list, and the row's length; by thread `me` of `of`.
    __device__ __forceinline__ void frame(const Kv4SelectArgs& a, int me, int of) const {
        const int taken = choose ? a.first + a.top : at.seen, last = choose ? at.free_end : at.seen, kept = taken + at.seen - last;
        for (int i = me; i < (choose ? a.first : taken); i += of) put(a, i, i);
        for (int i = me; i < at.seen - last; i += of) put(a, taken + i, last + i);
        for (int i = kept + me; i < a.list; i += of) a.pages[unit * a.list + i] = -1;
        for (int i = kept + me; i < a.width && a.chosen; i += of) a.chosen[unit * a.width + i] = -1;
        if (head == 0 && me == 0)  // all pages but the last are whole
            a.lens[row] = at.len <= 0 ? at.len : (kept - 1) * a.s.page + at.len - (at.seen - 1) * a.s.page;
    }
};

// The threshold of the `top` largest of n keys.  A histogram over evenly spaced bins leaves few
// keys in the bin where the count from above reaches `top`; those are ranked one against
// another.  Where that bin holds more than kSelectFew (scores that are equal, or far from evenly
// spread), or there are few keys at all, they are taken digit by digit from the highest instead,
// until the digits are out or a bin is taken whole.  Then the pages above the threshold and the
// first `need` of those at it are written in order.  One block per row and kv head; the threads
// keep HELD keys each in registers from pass to pass (more are read again), and what is counted
// per warp is joined once for all of them: what bounds the kernel is how often it waits (8 rows of
// 4096 pages, 1024 threads: 13 us; 256 threads, keys read for each pass, by digits alone and with
// counts joined for 256 pages at a time: 22 us).
template <int THREADS, int HELD>
__global__ void __launch_bounds__(THREADS) kv4_select_kernel(const Kv4SelectArgs a) {
    __shared__ int bins[kSelectBins];
    __shared__ int warp_sums[THREADS / 32];
    __shared__ int border[2];  // the bin, and how many of it are needed
    __shared__ float range[2][THREADS / 32];
    __shared__ int counts[HELD * (THREADS / 32)];
    __shared__ uint64_t few[kSelectFew];
    __shared__ uint64_t found[2];  // the threshold, and how many of those at it are needed
    __shared__ int n_few;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    SelectList to(a, blockIdx.x);
    bool falls = false;
    if (a.s.cu)
        for (int b = tid; b < a.s.B; b += THREADS) falls |= __ldg(a.s.cu + b + 1) < __ldg(a.s.cu + b);
    to.settle(a, __syncthreads_or(falls), tid == 0);
    to.frame(a, tid, THREADS);
    const int n = to.n;
    const uint64_t* keys = to.keys;
    uint64_t edge = 0;  // taken: keys whose digits above `shift` exceed it, and `need` of those that equal it
    int shift = 0, need = 0;
    if (to.choose && a.top > 0) {
        constexpr int RUN = THREADS * HELD;
        const int runs = (n + RUN - 1) / RUN;
        uint64_t k[HELD];
        auto load = [&](int run) {
#pragma unroll
            for (int j = 0; j < HELD; ++j) {
                const int i = run * RUN + j * THREADS + tid;
                k[j] = i < n ? keys[i] : 0;
            }
        };
        // f(key) for all keys
        auto each_key = [&](auto f) {
            for (int run = 0; run < runs; ++run) {
                if (runs > 1) load(run);
#pragma unroll
                for (int j = 0; j < HELD; ++j) {
                    const int i = run * RUN + j * THREADS + tid;
                    if (i < n) f(k[j]);
                }
            }
        };
        load(0);
        bool digits = true;
        if constexpr (HELD > 2) {  // (with fewer keys that is more work than the digits')
            float lo = INFINITY, hi = -INFINITY;
            each_key([&](uint64_t key) {
                const float v = score_of(key);
                if (key != 0 && fabsf(v) < INFINITY) lo = fminf(lo, v), hi = fmaxf(hi, v);
            });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            if (lane == 0) range[0][warp] = lo, range[1][warp] = hi;
            for (int i = tid; i < kSelectBins; i += THREADS) bins[i] = 0;
            if (tid == 0) n_few = 0;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < THREADS / 32; ++w) lo = fminf(lo, range[0][w]), hi = fmaxf(hi, range[1][w]);
            float each = (kSelectBins - 1) / (hi - lo);
            if (!(hi > lo) || !(each < INFINITY)) lo = 0.0f, each = 0.0f;  // (one bin but for infinities)
            each_key([&](uint64_t key) { atomicAdd(&bins[score_bin(key, lo, each)], 1); });
            __syncthreads();
            select_border<THREADS>(bins, a.top, warp_sums, border);
            const int bin = border[0], m = bins[bin];
            need = border[1];
            if (m <= kSelectFew) {
                each_key([&](uint64_t key) {
                    if (score_bin(key, lo, each) == bin) few[atomicAdd(&n_few, 1)] = key;
                });
                __syncthreads();
                if (tid < m) {
                    const uint64_t key = few[tid];
                    int above = 0, same = 0;
                    for (int j = 0; j < m; ++j) {
                        above += few[j] > key;
                        same += few[j] == key;
                    }
                    // (equal keys write the same)
                    if (above < need && need <= above + same) found[0] = key, found[1] = need - above;
                }
                __syncthreads();
                edge = found[0];
                need = (int)found[1];
                digits = false;
            }
            __syncthreads();  // the border is read
        }
        if (digits) {
            need = a.top;
            shift = 64;
            for (int width = 11; shift > 0; shift -= width) {
                if (shift < width) width = shift;
                for (int i = tid; i < kSelectBins; i += THREADS) bins[i] = 0;
                __syncthreads();
                const int low = shift - width;
                each_key([&](uint64_t key) {
                    if (shift == 64 || key >> shift == edge) atomicAdd(&bins[(key >> low) & ((1 << width) - 1)], 1);
                });
                __syncthreads();
                select_border<THREADS>(bins, need, warp_sums, border);
                edge = (shift == 64 ? 0 : edge << width) | (uint32_t)border[0];
                need = border[1];
                const bool whole = bins[border[0]] == need;
                __syncthreads();
                if (whole) {
                    shift = low;
                    break;
                }
            }
        }
        // those chosen, in order
        int done = 0, equal = 0;  // keys above the edge and at it in the runs before
        for (int run = 0; run < runs; ++run) {
            if (runs > 1) load(run);
            // how many of either a warp has in each of its rows of keys: those above in the low half
            int before[HELD];
            uint32_t takes = 0, ties = 0;
            __syncthreads();  // the counts of the run before are read
#pragma unroll
            for (int j = 0; j < HELD; ++j) {
                const bool there = run * RUN + j * THREADS + tid < n;
                const uint64_t digits = k[j] >> shift;
                const bool take = there && digits > edge, tie = there && digits == edge;
                const uint32_t m_take = __ballot_sync(0xffffffffu, take), m_tie = __ballot_sync(0xffffffffu, tie);
                const uint32_t under = (1u << lane) - 1;
                before[j] = __popc(m_take & under) | __popc(m_tie & under) << 16;
                takes |= (uint32_t)take << j, ties |= (uint32_t)tie << j;
                if (lane == 0) counts[j * (THREADS / 32) + warp] = __popc(m_take) | __popc(m_tie) << 16;
            }
            __syncthreads();
            // the counts before each, and their sum
            constexpr int ALL = HELD * (THREADS / 32), PER = (ALL + 31) / 32;
            if (warp == 0) {
                int mine[PER], sum = 0;
#pragma unroll
                for (int j = 0; j < PER; ++j) sum += mine[j] = lane * PER + j < ALL ? counts[lane * PER + j] : 0;
                int inc = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += v;
                }
                int at = inc - sum;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    if (lane * PER + j < ALL) counts[lane * PER + j] = at;
                    at += mine[j];
                }
                if (lane == 31) border[0] = inc;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < HELD; ++j) {
                const int v = counts[j * (THREADS / 32) + warp] + before[j];
                const int above = done + (v & 0xFFFF), same = equal + (v >> 16);
                if ((takes >> j & 1) || ((ties >> j & 1) && same < need))
                    to.put(a, a.first + above + min(same, need), a.first + run * RUN + j * THREADS + tid);
            }
            done += border[0] & 0xFFFF;
            equal += border[0] >> 16;
        }
    }
}

// The same for tables of up to kSmallPages pages and many rows: a warp per row and kv head, its keys
// in registers, the threshold found bit by bit from the highest in which two keys differ, until exactly
// `top` are at or above it or the bits are out.  251 rows of 250 pages and 157 of 138, 8 heads: 16 us, 35 with a
// block for each; few rows wait for its steps, though (32 x 8 of up to 512: 12 us, 9 with blocks).
constexpr int kWarpHeld = 16, kSmallPages = 32 * kWarpHeld, kWarpSelects = 4;
__global__ void __launch_bounds__(kWarpSelects * 32) kv4_select_warp_kernel(const Kv4SelectArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * kWarpSelects + (threadIdx.x >> 5);
    if (unit >= (a.row1 - a.row0) * a.s.Hk) return;
    SelectList to(a, unit);
    bool falls = false;
    if (a.s.cu)
        for (int b = lane; b < a.s.B; b += 32) falls |= __ldg(a.s.cu + b + 1) < __ldg(a.s.cu + b);
    to.settle(a, __any_sync(0xffffffffu, falls), lane == 0);
    to.frame(a, lane, 32);
    if (!to.choose || a.top == 0) return;
    uint64_t k[kWarpHeld], lo = ~0ull, hi = 0;
#pragma unroll
    for (int j = 0; j < kWarpHeld; ++j) k[j] = j * 32 + lane < to.n ? to.keys[j * 32 + lane] : 0;
#pragma unroll
    for (int j = 0; j < kWarpHeld; ++j)
        if (j * 32 + lane < to.n) lo = min(lo, k[j]), hi = max(hi, k[j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, (uint64_t)__shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, (uint64_t)__shfl_xor_sync(0xffffffffu, hi, o));
    }
    // `edge`: the largest number that at least `top` keys reach (those that are not there are 0, and reach none)
    int bit = 64 - __clzll((long long)(lo ^ hi)), above = 0;
    uint64_t edge = bit == 64 ? 0 : hi >> bit << bit;
    for (bool exact = false; bit > 0 && !exact;) {
        const uint64_t next = edge | 1ull << --bit;
        int reach = 0;
#pragma unroll
        for (int j = 0; j < kWarpHeld; ++j) reach += k[j] >= next;
        reach = __reduce_add_sync(0xffffffffu, reach);
        if (reach >= a.top) edge = next;
        exact = reach == a.top;
    }
#pragma unroll
    for (int j = 0; j < kWarpHeld; ++j) above += k[j] > edge;
    const int need = a.top - __reduce_add_sync(0xffffffffu, above);  // of those at the edge, the first
    int done = a.first, equal = 0;
    const uint32_t under = (1u << lane) - 1;
#pragma unroll
    for (int j = 0; j < kWarpHeld; ++j) {
        const bool there = j * 32 + lane < to.n, take = there && k[j] > edge, tie = there && k[j] == edge;
        const uint32_t m_take = __ballot_sync(0xffffffffu, take), m_tie = __ballot_sync(0xffffffffu, tie);
        const int same = equal + __popc(m_tie & under);
        if (take || (tie && same < need)) to.put(a, done + __popc(m_take & under) + min(same, need), a.first + j * 32 + lane);
        done += __popc(m_take);
        equal += __popc(m_tie);
    }
}

// The scores' share of the workspace: calls that need more take their rows in turn.
constexpr size_t kKeyBytes = (size_t)256 << 20;

struct SparseLayout {  // of the workspace
    bool scored;   // else every page is taken, of any row
    int list;      // pages of a row's table
    int64_t rows;  // whose scores are held at once
    size_t keys, pages, lens, attn, total;
    SparseLayout(int64_t T, int64_t Hk, int64_t G, int64_t D, int64_t table_w, int64_t width)
        : scored(table_w > width), list((int)std::max<int64_t>(std::min(table_w, width), 1)), rows(T) {
        keys = 0;
        const size_t row = (size_t)Hk * table_w * 8;
        if (scored && T * row > kKeyBytes) rows = std::max<int64_t>(kKeyBytes / row / kScoreTile * kScoreTile, 1);
        pages = keys + (scored ? round256(std::min(rows, T) * row) : 0);
        lens = pages + round256((size_t)T * Hk * list * 4);
        attn = lens + round256((size_t)T * 4);
        total = attn + attn_workspace(T, T, Hk, G, D);
    }
};

template <typename... Args>
static cudaError_t launch_dependent(void (*kernel)(Args...), dim3 grid, unsigned threads, cudaStream_t s, const Args&... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace pn

extern "C" {

int pn_kv4_page_means(const void* cache, int64_t n_pages, int64_t kv_heads, int64_t page, int64_t head_dim,
                      const int32_t* block_table, int64_t table_ld, int64_t table_w, const int32_t* seq_lens,
                      const int32_t* cu_q, int64_t B, int64_t T, void* means, void* stream) {
    const char* name = "pn_kv4_page_means";
    pn::Kv4MeansArgs a{};
    if (int st = check_kv4(name, cache, n_pages, kv_heads, page, head_dim, block_table, table_ld, table_w, seq_lens, cu_q, B, T,
                           &a.s))
        return st;
    if (T > 0 && B > 0 && !means && n_pages > 0) return fail(PN_ERR_ARG, "%s: null pointer", name);
    if (!aligned(means, 16)) return fail(PN_ERR_ALIGN, "%s: means needs 16-byte alignment", name);
    if (kv_heads > 65535) return fail(PN_ERR_SHAPE, "%s: %lld kv heads", name, (long long)kv_heads);
    if (int st = check_device()) return st;
    if (T == 0 || B == 0) return ok();
    a.cache = static_cast<const uint8_t*>(cache);
    a.means = static_cast<__nv_bfloat16*>(means);
    // as many rows to a block as leave four blocks to an SM
    a.rows = pn::kMeansRows;
    while (a.rows > 1 && T / a.rows * kv_heads < 4 * pn::sm_count()) a.rows /= 2;
    const dim3 grid((unsigned)((T + a.rows - 1) / a.rows), (unsigned)kv_heads);
    const cudaError_t err = head_dim == 64 ? pn::launch_dependent(pn::kv4_means_kernel<64>, grid, pn::kMeansThreads, (cudaStream_t)stream, a)
                                           : pn::launch_dependent(pn::kv4_means_kernel<128>, grid, pn::kMeansThreads, (cudaStream_t)stream, a);
    return err == cudaSuccess ? ok() : cuda_fail(err, name);
}

size_t pn_kv4_sparse_attention_workspace_size(int64_t T, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t table_w,
                                              int64_t width) {
    if (T < 1 || kv_heads < 1 || q_heads < kv_heads || head_dim < 1 || table_w < 0 || width < 1) return 0;
    return pn::SparseLayout(T, kv_heads, q_heads / kv_heads, head_dim, table_w, width).total;
}

int pn_kv4_sparse_attention(const void* q, int64_t q_sb, int64_t q_sl, int64_t q_sh, int q_dtype, int64_t q_heads,
                            const void* cache, const void* means, int64_t n_pages, int64_t kv_heads, int64_t page,
                            int64_t head_dim, const int32_t* block_table, int64_t table_ld, int64_t table_w,
                            const int32_t* seq_lens, const int32_t* cu_q, int64_t B, int64_t T, int64_t first_pages,
                            int64_t last_pages, int64_t top_pages, float scale, void* out, int32_t* chosen, void* workspace,
                            size_t workspace_bytes, void* stream) {
    const char* name = "pn_kv4_sparse_attention";
    pn::Kv4AttnArgs a{};
    if (int st = check_kv4(name, cache, n_pages, kv_heads, page, head_dim, block_table, table_ld, table_w, seq_lens, cu_q, B, T,
                           &a.s))
        return st;
    if (int st = check_attn(name, q, q_sb, q_sl, q_sh, q_dtype, q_heads, cache, scale, out, &a)) return st;
    if (first_pages < 0 || last_pages < 1 || top_pages < 0 || first_pages > 1 << 30 || last_pages > 1 << 30 || top_pages > 1 << 30)
        return fail(PN_ERR_SHAPE, "%s: first=%lld last=%lld top=%lld pages", name, (long long)first_pages, (long long)last_pages,
                    (long long)top_pages);
    const int64_t width = first_pages + last_pages + top_pages;
    if (width > (1 << 30) / page) return fail(PN_ERR_SHAPE, "%s: %lld pages to a row", name, (long long)width);
    if (T > 0 && B > 0 && !means && n_pages > 0) return fail(PN_ERR_ARG, "%s: null pointer", name);
    if (!aligned(means, 16)) return fail(PN_ERR_ALIGN, "%s: means needs 16-byte alignment", name);
    if (!aligned(chosen, 4)) return fail(PN_ERR_ALIGN, "%s: misaligned pointer", name);
    if (kv_heads > 65535 || (double)T * kv_heads > 2e9) return fail(PN_ERR_SHAPE, "%s: %lld rows of %lld kv heads", name, (long long)T, (long long)kv_heads);
    if ((double)T * kv_heads * std::min(width, table_w) * 4 > 3e10 || (double)kv_heads * table_w * 8 > 3e10)
        return fail(PN_ERR_SHAPE, "%s: %lld rows over tables of %lld pages are too much for one call", name, (long long)T, (long long)table_w);
    pn::Kv4Seq each = a.s;  // (every row a sequence of its own)
    each.B = T;
    if (int st = check_attn_units(name, each, a.G, std::min(width, table_w) * page)) return st;
    if (int st = check_device()) return st;
    if (T == 0 || B == 0) return ok();
    const pn::SparseLayout lay(T, kv_heads, a.G, head_dim, a.s.table_w, width);
    if (!workspace || workspace_bytes < lay.total) return fail(PN_ERR_WORKSPACE, "%s: workspace needs %zu bytes", name, lay.total);
    if (!aligned(workspace, 256)) return fail(PN_ERR_ALIGN, "%s: the workspace needs 256-byte alignment", name);
    char* ws = static_cast<char*>(workspace);
    pn::Kv4SelectArgs c{};
    c.s = a.s;
    c.q = q, c.q_f32 = a.q_f32, c.q_sb = q_sb, c.q_sl = q_sl, c.q_sh = q_sh, c.G = a.G;
    c.means = static_cast<const __nv_bfloat16*>(means);
    c.first = (int)first_pages, c.last = (int)last_pages, c.top = (int)top_pages, c.width = (int)width, c.list = lay.list;
    c.keys = reinterpret_cast<uint64_t*>(ws + lay.keys);
    c.pages = reinterpret_cast<int32_t*>(ws + lay.pages);
    c.lens = reinterpret_cast<int32_t*>(ws + lay.lens);
    c.chosen = chosen;
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t err = cudaSuccess;
    const bool scored = lay.scored && top_pages > 0;
    c.tile = 1;
    while (c.tile < pn::kScoreTile && 2 * c.tile <= T / B) c.tile *= 2;
    for (c.row0 = 0; c.row0 < T; c.row0 = c.row1) {
        c.row1 = scored ? std::min(c.row0 + lay.rows, T) : T;
        const int64_t rows = c.row1 - c.row0, units = rows * kv_heads;
        if (scored) {
            const int64_t tiles = (rows + c.tile - 1) / c.tile, runs = (a.s.table_w + 31) / 32;
            c.splits = (int)std::min<int64_t>(std::max<int64_t>(8 * pn::sm_count() / (tiles * kv_heads), 1), std::min<int64_t>(runs, 65535));
            const dim3 grid((unsigned)tiles, (unsigned)kv_heads, (unsigned)c.splits);
            err = head_dim == 64 ? pn::launch_dependent(pn::kv4_score_kernel<64>, grid, pn::kScoreThreads, s, c)
                                 : pn::launch_dependent(pn::kv4_score_kernel<128>, grid, pn::kScoreThreads, s, c);
            if (err != cudaSuccess) return cuda_fail(err, name);
        }
        const dim3 blocks((unsigned)units);
        // (for few rows the passes of each are what takes the time)
        if (a.s.table_w > pn::kSmallPages)
            err = units <= pn::sm_count() ? pn::launch_dependent(pn::kv4_select_kernel<1024, 8>, blocks, 1024, s, c)
                                          : pn::launch_dependent(pn::kv4_select_kernel<256, 8>, blocks, 256, s, c);
        else if (units <= 8 * pn::sm_count())
            err = pn::launch_dependent(pn::kv4_select_kernel<256, 2>, blocks, 256, s, c);
        else
            err = pn::launch_dependent(pn::kv4_select_warp_kernel, dim3((unsigned)((units + pn::kWarpSelects - 1) / pn::kWarpSelects)),
                                       pn::kWarpSelects * 32, s, c);
        if (err != cudaSuccess) return cuda_fail(err, name);
    }
    // every row a sequence of its own
    a.q_l = cu_q ? T : a.s.L;  // (with cu_q rows lie one after another)
    a.s.table = c.pages, a.s.table_hd = lay.list, a.s.table_ld = kv_heads * lay.list, a.s.table_w = n_pages > 0 ? lay.list : 0;
    a.s.lens = c.lens, a.s.cu = nullptr, a.s.B = T, a.s.L = 1;
    err = pn::attn_pass<true>(a, pn::attn_kind(T, T, kv_heads, a.G), head_dim, ws + lay.attn, s);
    return err == cudaSuccess ? ok() : cuda_fail(err, name);
}

}  // extern "C"
