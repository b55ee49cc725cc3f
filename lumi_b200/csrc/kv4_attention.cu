// Attention over a paged cache in 4 bits: y = softmax(scale q K^T) V for the rows of sequences of different lengths, with an optional sliding window and an optional sink (one more
// score, 0, without a value).  Row i of a sequence's n new rows stands at position tokens - n + i and sees the positions up to its own.
//
// kv4_step_kernel (few rows per sequence): the work is a line of pages, unit after unit; a unit is a sequence's head of the cache with up to 4, 8 or 16 columns, a column being a row and a query
// head that reads that cache head.  CTAs, and within them warps, take equal runs of that line, whatever the lengths.  A page's block comes by one bulk copy into the warp's ring, and a warp
// needs no other one until its run ends: then the parts of a unit are joined, first within the CTA, then by the CTA that arrives last.
//
// Products are m16n8k16 of warps: tokens (scores) and numbers of a head (values) in the rows of A, straight from the words of codes, columns in B.  A page of 64 tokens has too few columns
// per cache head to fill a tcgen05 tile's 128 rows, and its codes would have to go to shared memory once more.
// Scores S^T = K q: q times a power of two per column as fp16; codes of keys of bf16 rows as subnormals n 2^-24 (an AND), those of a word's second pair as 16 n 2^-24 against q / 16; the
// accumulator starts at -8 sum q.  A fp32 multiply-add per score and group brings the scale in.  fp32 rows: two fp16 terms of q, codes as n - 8.
// Values O^T = V^T P: codes less 8 in A (the transposing matrix load gives them), softmax weights times the group's scale in B, kept in fp16's range by 2^7 / (largest scale so far).
// fp32 rows: two fp16 terms of p s, in products of their own or, up to four columns, in the other four columns; bf16 rows: one term (2^-12 of a weight, beside 2^-9 of y).
//
// Bound by memory on paper (18 bytes per 32 numbers), by the issue of instructions in fact (a page of 128 + 128 numbers is 9216 bytes and about 850 warp instructions), and for short lines by
// latency: a page alone takes 10 us, launch, first instructions, copies and joins.  8 sequences of 32000 tokens, 64 / 8 bf16 heads of 128: 83 us, 3.6 TB/s; of 128000: 260 us, 4.6 TB/s;
// 64 sequences of 90 to 8192 tokens, 32 / 8 heads of 128: 60 us; 256 sequences in windows of 1024, 16 fp32 heads of 80: 106 us; one of 4000 tokens, 16 / 4 fp32 heads of 64: 14.7 us.
#include "device_args.h"
#include "kv4.cuh"
#include "rows.cuh"

#include <algorithm>

namespace lumi {
namespace {

constexpr int kMaxCtas = 296;                              // of the step kernel: places for parts
// Fewer pages than these for each CTA are taken by fewer CTAs (us of one sequence of 4000 tokens and four heads of 64, and of 8 x 1000 and eight of 128): 4 pages 16.8, 19.7; 6 16.5, 19.6;
// 8 15.1, 16.7; 12 18.0, 20.3.
constexpr int kCtaPages = 8;
// What a unit's beginning and end (queries in, results out) cost, in pages: where units are many, each begins with so many places without a page on the line that is split.  us of 256 sequences
// of 32 to 1024 visible tokens, 16 fp32 heads of 80 each, and of 64 of 90 to 8192, 8 bf16 heads of 128: none 150, 75; one 112, 63; two 113, 60; three 116, 59.
constexpr int kUnitCost = 1;
// Columns of a sequence up to which this kernel takes it, the one of prompts beyond.  us here and there, of 16 sequences of 4000 tokens and eight heads of 128 (bf16; fp32), and of 64 of 500 and
// four of 64 (bf16): 32 columns 86, 115; 106, 156; 32, 47.  48 columns 118, 117; 143, 158; 39, 48.  64 columns 146, 117; 187, 158; 49, 53.
constexpr int kFewColumns = 48;

// Matrix loads may be moved as the arithmetic around them allows; what orders them is their address, which comes from pinned() behind what they have to wait for.
__device__ __forceinline__ uint32_t pinned(uint32_t a) {
    uint32_t b;
    asm volatile("mov.u32 %0, %1;" : "=r"(b) : "r"(a) : "memory");
    return b;
}
__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&r)[4]) {
    asm("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t a, uint32_t (&r)[4]) {
    asm("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma16(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}
// Two codes less 8 as halves, of bits 0 .. 3 and 16 .. 19 of a word; 16 times that, of bits 4 .. 7 and 20 .. 23.  NORMAL: by way of 1024 + n, as numbers n - 8.  Else as subnormals (n - 8) 2^-24,
// an AND and an addition; but sums of such products are aligned by their exponents, which promise more than subnormals hold, and keep only about 17 bits: enough for bf16 rows, and 5 % faster
// (8 sequences of 32000 tokens 83 us against 87).  fp32 rows, 4000 tokens: 3e-7 off against 7e-6.
__device__ __forceinline__ uint32_t less(uint32_t x, uint32_t c) {
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool NORMAL>
__device__ __forceinline__ uint32_t signed_code(uint32_t w) { return NORMAL ? less((w & 0x000f000fu) | 0x64006400u, 0x64086408u) : less(w & 0x000f000fu, 0x00080008u); }
template <bool NORMAL>
__device__ __forceinline__ uint32_t signed_code16(uint32_t w) { return NORMAL ? less((w & 0x00f000f0u) | 0x64006400u, 0x64806480u) : less(w & 0x00f000f0u, 0x00800080u); }
// An 8 x 8 matrix of 16-bit numbers, one row per four lanes, two numbers each, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t u) {
    uint32_t v;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(v) : "r"(u));
    return v;
}
// Pages that any of its rows sees, and units of `cols` columns.  Nothing of a sequence that is left out, or that is another kernel's.
__device__ __forceinline__ Sequence step_sequence(const AttendArgs& a, int s, int cols, bool& bad) {
    Sequence q;
    const bool fits = lengths_of(a, s, q);
    bad = !fits;
    q.page0 = q.pages = q.units = 0;
    if (!fits || q.n <= 0 || q.n > a.max_new || (long)q.n * a.group > a.few) return q;
    const int lo = a.window > 0 ? max(0, q.total - q.n - a.window + 1) : 0;
    q.page0 = lo / kPage;
    q.pages = (q.total - 1) / kPage - q.page0 + 1;
    q.units = (q.n * a.group + cols - 1) / cols * a.kv_heads;
    return q;
}

// ---- few rows per sequence --------------------------------------------------------------------------------------
// MODE 0: up to 8 columns of bf16 rows; 1: up to 16; 2: up to 8 columns of fp32 rows, as two terms; 3: up to 4, whose second terms are the other columns of the same products.
template <int NG, int MODE>
struct StepShape {
    static constexpr int kCols = MODE == 1 ? 16 : MODE == 3 ? 4 : 8;
    // registers: accumulators of values 4 NG per eight columns and number block, of their offsets, scores, q
    static constexpr int kWarps = NG == 8 ? 6 : MODE == 1 ? (NG == 4 ? 8 : 12) : (NG == 4 ? 12 : 16);
};

// One part of a unit: columns' largest score m (in units of log2), sum l and numbers o [column][dv], all relative to 2^m.  Where parts lie: m [cols], l [cols], o [cols][pad].
__host__ __device__ inline int part_floats(int cols, int dv) { return cols * (2 + kv4_groups(dv) * kGroup); }

struct Open { long long lo, hi; int s, unit; };

template <typename T, int NG, int MODE>
__global__ void __launch_bounds__(StepShape<NG, MODE>::kWarps * 32, 1) kv4_step_kernel(const AttendArgs a) {
    using Shape = StepShape<NG, MODE>;
    constexpr int W = Shape::kWarps, COLS = Shape::kCols, THREADS = W * 32, NT = MODE == 1 ? 2 : 1;
    constexpr bool SIGNED = MODE >= 2;                     // codes of keys too are n - 8, and all of them numbers that are not subnormal
    constexpr bool TWO = MODE == 2, PAIRED = MODE == 3;    // two terms of q and of the weights: products of their own; columns c and 4 + c
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ long long before[THREADS + 1], units_before[THREADS + 1];      // pages and units of the sequences ahead of each thread's
    __shared__ uint64_t full[W][4];
    __shared__ long long warp_pages[W], warp_units[W];
    __shared__ Open heads_s[W], tails_s[W];                // units that began ahead of a warp's run and end in it; that its run ends with and that it does not hold whole
    __shared__ int lost_s, n_open_s;
    __shared__ int4 opens_s[2 * W], shared_s[2];
    __shared__ long long line_s[3 + W];                    // places of the line, the CTA's first page and its end, runs' first ones: not kept in registers over the pages
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i8 = lane >> 2, j4 = lane & 3;
    uint8_t* const ring = sm + (size_t)warp * a.slots * a.slot_bytes;
    const int gk = kv4_groups(a.dk), gv = kv4_groups(a.dv), part = kv4_part(a.dk), block = kv4_block(a.dk, a.dv);
    const int rec = part_floats(COLS, a.dv), pad = gv * kGroup;

    if (lane < 4) mbar_init(&full[warp][lane], 1);
    if (lane == 0) heads_s[warp].lo = tails_s[warp].lo = -1;
    if (tid == 0) lost_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_release();
    pdl_sync();

    // ---- the line of pages: each thread sums up a run of sequences
    const int each = (a.nseq + THREADS - 1) / THREADS, s_lo = min(a.nseq, tid * each), s_hi = min(a.nseq, s_lo + each);
    long long mine = 0, my_units = 0;
    bool any_bad = false;
    for (int s = s_lo; s < s_hi; ++s) {
        bool bad;
        const Sequence q = step_sequence(a, s, COLS, bad);
        any_bad |= bad;
        mine += (long long)q.pages * q.units;
        my_units += q.units;
    }
    if (any_bad && blockIdx.x == 0 && a.status != nullptr) atomicOr(a.status, kBadPage);
    long long run = mine, run_units = my_units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, run, o), u = __shfl_up_sync(0xffffffffu, run_units, o);
        if (lane >= o) { run += t; run_units += u; }
    }
    if (lane == 31) { warp_pages[warp] = run; warp_units[warp] = run_units; }
    __syncthreads();
    long long ahead = 0, total = 0, units_ahead = 0, units = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const long long p = warp_pages[w], u = warp_units[w];
        if (w < warp) { ahead += p; units_ahead += u; }
        total += p;
        units += u;
    }
    before[tid] = ahead + run - mine;
    units_before[tid] = units_ahead + run_units - my_units;
    if (tid == THREADS - 1) { before[THREADS] = total; units_before[THREADS] = units; }
    __syncthreads();
    // CTAs that get work: some pages each.  Where units are many, each begins with places without a page on the line that is split, so that short ones are not taken for cheap ones.
    const int ctas = (int)min((long long)gridDim.x, quotient(total + kCtaPages - 1, kCtaPages)), cta = blockIdx.x;
    if (cta >= ctas) return;
    const int extra = units > ctas ? kUnitCost : 0;
    const long long places = total + units * extra;
    const long long c_lo = quotient(places * cta, ctas), c_hi = quotient(places * (cta + 1), ctas);
    const int runs = (int)min((long long)W, c_hi - c_lo);    // runs that are not empty come first
    auto warp_from = [&](int w) { return c_lo + quotient((c_hi - c_lo) * min(w, runs), runs); };
    // the first page at or behind a place
    auto page_at = [&](long long x) {
        int lo = 0, hi = THREADS;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (before[mid] + extra * units_before[mid] <= x) lo = mid; else hi = mid; }
        long long at = before[lo], rel = x - at - extra * units_before[lo];
        for (int s = lo * each; s < min(a.nseq, (lo + 1) * each); ++s) {
            bool bad;
            const Sequence q = step_sequence(a, s, COLS, bad);
            const int per = q.pages + extra;
            if (rel < (long long)per * q.units) {
                const long long unit = quotient(rel, per);
                return at + unit * q.pages + max(0, (int)(rel - unit * per) - extra);
            }
            rel -= (long long)per * q.units;
            at += (long long)q.pages * q.units;
        }
        return at;
    };
    long long edge_of = lane == 0 ? warp_from(warp) : lane == 1 ? warp_from(warp + 1) : lane == 2 ? c_lo : c_hi;
    if (extra != 0 && lane < 4) edge_of = page_at(edge_of);
    __syncwarp();
    const int run_n = (int)(__shfl_sync(0xffffffffu, edge_of, 1) - __shfl_sync(0xffffffffu, edge_of, 0));
    if (lane == 0) line_s[3 + warp] = edge_of;
    if (warp == 0 && lane == 2) { line_s[0] = places; line_s[1] = edge_of; }
    if (warp == 0 && lane == 3) line_s[2] = edge_of;
    __syncwarp();
    volatile const long long* const x_lo_s = line_s + 3 + warp;

    // where page x of the line lies: sequence, unit, page of the unit's
    struct Spot { int s, unit, p, page; };
    auto find = [&](long long x) {
        int lo = 0, hi = THREADS;
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (before[mid] <= x) lo = mid; else hi = mid; }
        long long at = before[lo];
        Spot r{0, 0, 0, -1};
        for (int s = lo * each; s < min(a.nseq, (lo + 1) * each); ++s) {
            bool bad;
            const Sequence q = step_sequence(a, s, COLS, bad);
            const long long n = (long long)q.pages * q.units;
            if (x < at + n) {
                const long long rel = x - at;
                r.s = s;
                r.unit = (int)quotient(rel, q.pages);
                r.p = (int)(rel - (long long)r.unit * q.pages);
                r.page = a.table[(size_t)s * a.width + q.page0 + r.p];
                if (r.page < 0 || r.page >= a.n_pages) {
                    r.page = -1;
                    if (a.status != nullptr) atomicOr(a.status, kBadPage);
                }
                break;
            }
            at += n;
        }
        return r;
    };

    // ---- state of the unit at hand.  Lane 4 i + j: columns 2 j and 2 j + 1 of each eight, tokens i of each eight, numbers 4 i .. 4 i + 3 of each group.
    float O[NT][2 * NG][4], m[NT][2], l[NT][2];
    uint32_t Q[NT][2 * NG][TWO ? 4 : 2];                   // q as B, first and second term
    float QC[NT][NG][2];                                   // -8 sum q of each group: what the scores' accumulators start at
    float cx[NT][2];                                       // factor from accumulators to scores in units of log2
    int lo_pos[NT][2], hi_pos[NT][2];                      // positions that the column sees: lo .. hi
    int e_v = 0;                                           // scales of values are below 2^e_v so far
    int first_full = 0, last_full = 0;                     // positions that every column sees
    bool dead = false;                                     // a wait gave up
    const float sign = a.scale < 0.f ? -1.f : 1.f;
    const float second = j4 >= 2 ? -1.f : 0.f;             // (PAIRED) the lane's columns are second terms

    auto begin_unit = [&](const Sequence& q, int unit) {
        const int cols = q.n * a.group, tile = unit / a.kv_heads, head = unit - tile * a.kv_heads, col0 = tile * COLS;
        first_full = 0; last_full = 0x7fffffff;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int col = col0 + nt * 8 + (PAIRED ? i8 & 3 : i8), row = min(col, cols - 1) / a.group, h = min(col, cols - 1) - row * a.group;
            const T* const p = (const T*)a.q + (long)(q.first + row) * a.ldq + (long)(head * a.group + h) * a.dk + j4 * 8;
            float raw[NG][8];                              // numbers 8 j .. 8 j + 7 of each group of column i
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int n = col < cols ? a.dk - g * kGroup - j4 * 8 : 0;
                if (a.wide_q) eight_numbers(p + g * kGroup, n, raw[g]);
                else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) raw[g][e] = e < n ? number(p + g * kGroup + e) : 0.f;
                }
            }
            // times a power of two that brings the column's largest to 2^13 .. 2^14
            uint32_t top = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(raw[g][e]) & 0x7fffffffu);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float by = power_of_two(top >= 0x7f800000u || top == 0 ? 0 : min(126, 13 + 127 - (int)(top >> 23)));
            const float c = fminf(fmaxf(__fdiv_rn(fabsf(a.scale) * kLog2e, by) * (SIGNED ? 1.f : 16777216.f), 1e-37f), 3.4e38f);      // (not 0: hidden scores are -inf)
            const int pos = q.total - q.n + row, lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                cx[nt][e] = __shfl_sync(0xffffffffu, c, 8 * j4 + 4 * e);
                hi_pos[nt][e] = __shfl_sync(0xffffffffu, pos, 8 * j4 + 4 * e);
                lo_pos[nt][e] = __shfl_sync(0xffffffffu, lo, 8 * j4 + 4 * e);
                m[nt][e] = -INFINITY;
                l[nt][e] = 0.f;
            }
            last_full = min(last_full, __reduce_min_sync(0xffffffffu, pos));
            first_full = max(first_full, __reduce_max_sync(0xffffffffu, lo));
            const float f = by * sign, f16 = f * 0.0625f;  // the second pair of a step meets codes that are 16 times as large
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int step = 0; step < 2; ++step) {
                    const float(&v)[8] = raw[g];
                    const float v0 = v[step * 4] * f, v1 = v[step * 4 + 1] * f, v2 = v[step * 4 + 2] * f16, v3 = v[step * 4 + 3] * f16;
                    auto& to = Q[nt][2 * g + step];
                    to[0] = halves(v0, v1);
                    to[1] = halves(v2, v3);
                    if (PAIRED) {
                        const float2 h0 = unhalves(to[0]), h1 = unhalves(to[1]);
                        if (i8 >= 4) { to[0] = halves(v0 - h0.x, v1 - h0.y); to[1] = halves(v2 - h1.x, v3 - h1.y); }
                    }
                    if constexpr (TWO) {
                        const float2 h0 = unhalves(to[0]), h1 = unhalves(to[1]);
                        to[2] = halves(v0 - h0.x, v1 - h0.y);
                        to[3] = halves(v2 - h1.x, v3 - h1.y);
                    }
                }
#pragma unroll
            for (int g = 0; g < NG && !SIGNED; ++g) {
                float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int step = 0; step < 2; ++step) {
                    const auto& b = Q[nt][2 * g + step];
                    mma16(t, 0x80088008u, 0x80088008u, 0x80808080u, 0x80808080u, b[0], b[1]);                // -8 2^-24 and -128 2^-24
                }
                QC[nt][g][0] = t[0]; QC[nt][g][1] = t[1];
            }
#pragma unroll
            for (int t = 0; t < 2 * NG; ++t) O[nt][t][0] = O[nt][t][1] = O[nt][t][2] = O[nt][t][3] = 0.f;
        }
        e_v = -90;
    };
    // ---- one page of the unit
    auto work_page = [&](uint8_t* slot, int pos0) {
        const bool edge = pos0 < first_full || pos0 + kPage - 1 > last_full;
        if (edge) {
            // scales of tokens that no column sees may be any bits: they become 0
            int lo = lo_pos[0][0], hi = hi_pos[0][0];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) { lo = min(lo, min(lo_pos[nt][0], lo_pos[nt][1])); hi = max(hi, max(hi_pos[nt][0], hi_pos[nt][1])); }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
            uint16_t* const sv = reinterpret_cast<uint16_t*>(slot + part + gv * kPlane);
            for (int k = lane; k < gv * kPage; k += 32) {
                const int pos = pos0 + k % kPage;
                if (pos < lo || pos > hi) sv[k] = 0;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        }
        const uint32_t base = pinned(smem_u32(slot));
        // scales of a pair of groups, of tokens i of four eights: the transposing load finds the pair's planes in its odd and even rows
        auto pair_scales = [&](uint32_t scales, int g, int groups, int h, uint32_t (&sc)[4]) {
            ldmatrix4_trans(scales + min(g + lane % 2, groups - 1) * kScales + h * 64 + (lane / 8) * 16, sc);
        };
        float S[NT][8][2];                                 // token i of each eight
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int t = 0; t < 8; ++t) S[nt][t][0] = S[nt][t][1] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t sc[4];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (g >= gk) break;
                if (g % 2 == 0) pair_scales(base + gk * kPlane, g, gk, h, sc);
                uint32_t w[4];
                ldmatrix4(base + g * kPlane + lane * 16 + h * 512, w);
                float d[NT][2][4];                         // (products that do not wait for one another side by side)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        uint32_t a0 = w[2 * k] & 0x000f000fu, a1 = w[2 * k + 1] & 0x000f000fu, a2 = w[2 * k] & 0x00f000f0u, a3 = w[2 * k + 1] & 0x00f000f0u;
                        if (SIGNED) { a0 = signed_code<SIGNED>(w[2 * k]); a1 = signed_code<SIGNED>(w[2 * k + 1]); a2 = signed_code16<SIGNED>(w[2 * k]); a3 = signed_code16<SIGNED>(w[2 * k + 1]); }
                        const auto& q = Q[nt][2 * g];
                        const float c0 = SIGNED ? 0.f : QC[nt][g][0], c1 = SIGNED ? 0.f : QC[nt][g][1];
                        mma16(d[nt][k], a0, a1, a2, a3, q[0], q[1], c0, c1, c0, c1);
                        if constexpr (TWO) mma16(d[nt][k], a0, a1, a2, a3, q[2], q[3]);
                    }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint32_t u0 = w[2 * k] >> 8, u1 = w[2 * k + 1] >> 8;
                        uint32_t a0 = u0 & 0x000f000fu, a1 = u1 & 0x000f000fu, a2 = u0 & 0x00f000f0u, a3 = u1 & 0x00f000f0u;
                        if (SIGNED) { a0 = signed_code<SIGNED>(u0); a1 = signed_code<SIGNED>(u1); a2 = signed_code16<SIGNED>(u0); a3 = signed_code16<SIGNED>(u1); }
                        const auto& q = Q[nt][2 * g + 1];
                        mma16(d[nt][k], a0, a1, a2, a3, q[0], q[1]);
                        if constexpr (TWO) mma16(d[nt][k], a0, a1, a2, a3, q[2], q[3]);
                    }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float s0 = g % 2 ? high_bf16(sc[2 * k]) : low_bf16(sc[2 * k]), s1 = g % 2 ? high_bf16(sc[2 * k + 1]) : low_bf16(sc[2 * k + 1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float(&x)[2] = S[nt][4 * h + 2 * k], (&y)[2] = S[nt][4 * h + 2 * k + 1];
                        x[0] = fmaf(d[nt][k][0], s0, x[0]); x[1] = fmaf(d[nt][k][1], s0, x[1]);
                        y[0] = fmaf(d[nt][k][2], s1, y[0]); y[1] = fmaf(d[nt][k][3], s1, y[1]);
                    }
                }
            }
        }
        if constexpr (PAIRED) {                            // both terms' scores, in lanes of both
#pragma unroll
            for (int t = 0; t < 8; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) S[0][t][e] += __shfl_xor_sync(0xffffffffu, S[0][t][e], 2);
        }
        if (edge) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int pos = pos0 + t * 8 + i8;
                        if (pos < lo_pos[nt][e] || pos > hi_pos[nt][e]) S[nt][t][e] = -INFINITY;
                    }
        }
        // the largest scale of values: a lane looks at eight of them
        auto top_scale = [&]() {
            uint32_t top = 0;
            const uint4* const sv = reinterpret_cast<const uint4*>(slot + part + gv * kPlane);
#pragma unroll
            for (int k = 0; k < (NG + 3) / 4; ++k) {
                const int at = k * 32 + lane;
                if (at < gv * 8) {
                    const uint4 u = sv[at];
                    const __nv_bfloat162* const b = reinterpret_cast<const __nv_bfloat162*>(&u);
                    const __nv_bfloat162 x = __hmax2_nan(__hmax2_nan(b[0], b[1]), __hmax2_nan(b[2], b[3]));
                    const uint32_t bits = *reinterpret_cast<const uint32_t*>(&x);
                    top = max(top, max(bits & 0x7fffu, bits >> 16 & 0x7fffu));
                }
            }
            return top;
        };
        uint32_t top_bits = top_scale();
        if (__any_sync(0xffffffffu, top_bits >= 0x7f80u)) {
            // (rare) tokens with values that are no numbers: a column that sees one is none, and the others do not meet them
            uint16_t* const sv = reinterpret_cast<uint16_t*>(slot + part + gv * kPlane);
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                bool none = false;                         // token half * 32 + lane
#pragma unroll 1
                for (int g = 0; g < gv; ++g) {
                    uint16_t& b = sv[g * kPage + half * 32 + lane];
                    if ((b & 0x7fffu) >= 0x7f80u) { b = 0; none = true; }
                }
#pragma unroll 1
                for (uint32_t at = __ballot_sync(0xffffffffu, none); at != 0; at &= at - 1) {
                    const int pos = pos0 + half * 32 + __ffs(at) - 1;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (pos >= lo_pos[nt][e] && pos <= hi_pos[nt][e]) l[nt][e] = __uint_as_float(0x7fc00000u);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            top_bits = top_scale();
        }
        const int e_top = min(127, (int)(top_bits >> 7) - 126);      // the largest is below 2^e
        const uint32_t vals = pinned(smem_u32(slot) + part);
        // weights are relative to the running maximum, which moves where it would have to by more than 2^8, and to 2^(e_v - 7)
        bool moves = e_top > e_v;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float t = S[nt][0][e];
#pragma unroll
                for (int k = 1; k < 8; ++k) t = fmaxf(t, S[nt][k][e]);
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                top[nt][e] = t * cx[nt][e];
                moves |= top[nt][e] > m[nt][e] + 8.f || (m[nt][e] == -INFINITY && top[nt][e] > -INFINITY);
            }
        if (__any_sync(0xffffffffu, moves)) {
            const int to_e = max(e_v, __reduce_max_sync(0xffffffffu, e_top));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float to = fmaxf(m[nt][e], top[nt][e]);
                    top[nt][e] = m[nt][e] == -INFINITY ? 0.f : exp2_fast(0.5f * (m[nt][e] - to + (float)(e_v - to_e)));      // (nothing so far: the numbers are 0)
                    m[nt][e] = to;
                }
            e_v = to_e;
#pragma unroll 1
            for (int twice = 0; twice < 2; ++twice)        // the factor's root: scales of values may differ by more than fp32's range
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float f0 = top[nt][0], f1 = top[nt][1];
#pragma unroll
                    for (int t = 0; t < 2 * NG; ++t) { O[nt][t][0] *= f0; O[nt][t][1] *= f1; O[nt][t][2] *= f0; O[nt][t][3] *= f1; }
                    l[nt][0] *= f0; l[nt][1] *= f1;
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float up = (float)(7 - e_v), off0 = m[nt][0] == -INFINITY ? 0.f : up - m[nt][0], off1 = m[nt][1] == -INFINITY ? 0.f : up - m[nt][1];
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                float(&x)[2] = S[nt][t];
                fma2(x[0], x[1], x[0], x[1], cx[nt][0], cx[nt][1], off0, off1);
                x[0] = exp2_fast(x[0]);
                x[1] = exp2_fast(x[1]);
                add2(l[nt][0], l[nt][1], x[0], x[1]);
            }
        }
        // values: 32 tokens, then group after group, so that products into the same accumulators lie apart
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t sc[4];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (g >= gv) break;
                if (g % 2 == 0) pair_scales(vals + gv * kPlane, g, gv, h, sc);
                uint32_t w[4];
                ldmatrix4_trans(vals + g * kPlane + lane * 16 + h * 512, w);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t r0 = w[2 * k], r1 = w[2 * k + 1], u0 = r0 >> 8, u1 = r1 >> 8;
                    const uint32_t a0 = signed_code<SIGNED>(r0), a1 = signed_code16<SIGNED>(r0), a2 = signed_code<SIGNED>(r1), a3 = signed_code16<SIGNED>(r1);
                    const uint32_t a4 = signed_code<SIGNED>(u0), a5 = signed_code16<SIGNED>(u0), a6 = signed_code<SIGNED>(u1), a7 = signed_code16<SIGNED>(u1);
                    const float s0 = g % 2 ? high_bf16(sc[2 * k]) : low_bf16(sc[2 * k]), s1 = g % 2 ? high_bf16(sc[2 * k + 1]) : low_bf16(sc[2 * k + 1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float(&x)[2] = S[nt][4 * h + 2 * k], (&y)[2] = S[nt][4 * h + 2 * k + 1];
                        const float v0 = x[0] * s0, v1 = x[1] * s0, v2 = y[0] * s1, v3 = y[1] * s1;
                        uint32_t p0 = halves(v0, v1), p1 = halves(v2, v3);
                        if constexpr (PAIRED) {
                            const float2 h0 = unhalves(p0), h1 = unhalves(p1);
                            p0 = halves(fmaf(h0.x, second, v0), fmaf(h0.y, second, v1));
                            p1 = halves(fmaf(h1.x, second, v2), fmaf(h1.y, second, v3));
                        }
#pragma unroll
                        for (int term = 0; term < (TWO ? 2 : 1); ++term) {
                            uint32_t b0 = p0, b1 = p1;
                            if (term == 1) {
                                const float2 h0 = unhalves(p0), h1 = unhalves(p1);
                                b0 = halves(v0 - h0.x, v1 - h0.y);
                                b1 = halves(v2 - h1.x, v3 - h1.y);
                            }
                            b0 = transposed(b0);
                            b1 = transposed(b1);
                            mma16(O[nt][2 * g], a0, a1, a2, a3, b0, b1);
                            mma16(O[nt][2 * g + 1], a4, a5, a6, a7, b0, b1);
                        }
                    }
                }
            }
        }
        // the slot's numbers have been read when these are known
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int t = 0; t < 2 * NG; ++t) asm volatile("" : "+f"(O[nt][t][0]), "+f"(O[nt][t][1]), "+f"(O[nt][t][2]), "+f"(O[nt][t][3]) : : "memory");
        }
    };

    // ---- what a unit leaves: numbers 4 i .. 4 i + 3 of each group, of columns 2 j and 2 j + 1, before the division by the sum
    auto over_tokens = [&](float v) {
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        return v + __shfl_xor_sync(0xffffffffu, v, 16);
    };
    auto number_at = [&](int nt, int g, int t, int e) { return O[nt][2 * g + (t >> 1)][(t & 1) * 2 + e] * ((t & 1) ? 0.0625f : 1.f); };
    // to == nullptr: the whole unit was this warp's, rows of y; else a part of it
    auto leave_unit = [&](int s, int unit, float* to) {
        Sequence q;
        lengths_of(a, s, q);
        const int cols = q.n * a.group, tile = unit / a.kv_heads, head = unit - tile * a.kv_heads;
        const float by = power_of_two(e_v / 2), by2 = power_of_two(e_v - e_v / 2);          // back from 2^(7 - e_v)
        if constexpr (PAIRED) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int t = 0; t < 2 * NG; ++t) {
                    O[0][t][e] += __shfl_xor_sync(0xffffffffu, O[0][t][e], 2);
                    O[0][t][2 + e] += __shfl_xor_sync(0xffffffffu, O[0][t][2 + e], 2);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = over_tokens(l[nt][e]) * 0.0078125f * by * by2;
                if (to == nullptr && a.sink && m[nt][e] != -INFINITY) sum += exp2_fast(-m[nt][e]);
                if (dead) sum = __uint_as_float(0x7fc00000u);
                const float f = to != nullptr ? 1.f : m[nt][e] == -INFINITY && sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
                const int c8 = nt * 8 + 2 * j4 + e, col = tile * COLS + c8, row = col / a.group, h = col - row * a.group;
                const bool puts = !PAIRED || j4 < 2;       // (all lanes take part in the shuffles)
                if (to != nullptr && i8 == 0 && puts) { to[c8] = m[nt][e]; to[COLS + c8] = sum; }
                T* const y = (T*)a.y + (long)(q.first + row) * a.ldy + (long)(head * a.group + h) * a.dv;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (g >= gv) break;
                    float v[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) v[t] = number_at(nt, g, t, e) * (SIGNED ? 0.0078125f : 131072.f) * by * by2 * f;
                    const int d = g * kGroup + 4 * i8;
                    if (to != nullptr && puts) *reinterpret_cast<float4*>(to + 2 * COLS + c8 * pad + d) = make_float4(v[0], v[1], v[2], v[3]);
                    if (to == nullptr && puts && col < cols) put_four(y + d, a.dv - d, a.wide_y, v);
                }
            }
    };

    // ---- the warp's run
    float* const head_part = a.parts + (size_t)kMaxCtas * 2 * rec + ((size_t)cta * W + warp) * rec;
    uint32_t pending = 0, phases = 0;                      // bits of slots: a copy is on its way; parity of the next one's end
    Spot now{0, 0, 0, -1}, then{0, 0, 0, -1};              // of the 32 pages at hand, one per lane, and of the next 32
    auto issue = [&](int x, int slot, int page, int unit) {      // (uniform)
        if (page < 0) return;
        pending |= 1u << slot;
        if (lane == 0) {
            mbar_expect_tx(&full[warp][slot], block);
            if (a.skip < 0 || *x_lo_s + x != a.skip) bulk_copy(smem_u32(ring) + slot * a.slot_bytes, a.kv + ((size_t)page * a.kv_heads + unit % a.kv_heads) * block, block, &full[warp][slot]);
        }
    };
    int s = 0, unit = 0, pages = 0, page0 = 0;             // the unit at hand
    int unit_lo = 0, unit_hi = 0;                          // its pages, counted from the run's first
    if (run_n > 0) {
        int batch = 0, asked = 0, slot = 0;
        for (int x = 0; x < run_n; ++x) {
            const int k = x - batch;
            if (x == 0 || k == 8) {                        // places of the first 32 pages; of the 32 behind these
                const int at = x == 0 ? 0 : batch + 32;
                Spot found{0, 0, 0, -1};
                if (at + lane < run_n) found = find(*x_lo_s + at + lane);
                __syncwarp();
                if (x == 0) {
                    now = found;
#pragma unroll 1
                    for (; asked < min(run_n, a.slots); ++asked) issue(asked, asked, __shfl_sync(0xffffffffu, now.page, asked), __shfl_sync(0xffffffffu, now.unit, asked));
                } else then = found;
            }
            const int p = __shfl_sync(0xffffffffu, now.p, k);
            if (x == 0 || p == 0) {
                s = __shfl_sync(0xffffffffu, now.s, k);
                unit = __shfl_sync(0xffffffffu, now.unit, k);
                bool bad;
                const Sequence q = step_sequence(a, s, COLS, bad);
                pages = q.pages; page0 = q.page0;
                unit_lo = x - p; unit_hi = unit_lo + pages;
                begin_unit(q, unit);
            }
            if (pending >> slot & 1) {
                if (!dead) dead = __any_sync(0xffffffffu, !mbar_wait(&full[warp][slot], phases >> slot & 1, a.wait_ns));
                if (!dead) {
                    pending &= ~(1u << slot);
                    phases ^= 1u << slot;
                    work_page(ring + slot * a.slot_bytes, (page0 + p) * kPage);
                    __syncwarp();
                }
            }
            // the unit ends here, or the run does
            if (p == pages - 1 || x == run_n - 1) {
                float* to = nullptr;
                if (unit_lo < 0 || p < pages - 1) {
                    to = x + 1 < run_n ? head_part : reinterpret_cast<float*>(ring);
                    if (x == run_n - 1)                    // (only after a wait gave up: copies in flight land before their places are used again)
#pragma unroll 1
                        for (int i = 0; i < a.slots; ++i) if (pending >> i & 1) mbar_wait(&full[warp][i], phases >> i & 1, a.wait_ns);
                    if (lane == 0) (x + 1 < run_n ? heads_s : tails_s)[warp] = Open{*x_lo_s + unit_lo, *x_lo_s + unit_hi, s, unit};
                }
                leave_unit(s, unit, to);
            }
            // the slot is free for the page `slots` further on
            if (asked < run_n && !dead) {
                const int kk = asked - batch;
                const int page = __shfl_sync(0xffffffffu, kk < 32 ? now.page : then.page, kk & 31), u = __shfl_sync(0xffffffffu, kk < 32 ? now.unit : then.unit, kk & 31);
                issue(asked, slot, page, u);
                ++asked;
            }
            if (k == 31) { now = then; batch += 32; }
            slot = slot + 1 == a.slots ? 0 : slot + 1;
        }
        if (dead) {
#pragma unroll 1
            for (int i = 0; i < a.slots; ++i) if (pending >> i & 1) mbar_wait(&full[warp][i], phases >> i & 1, a.wait_ns);
            if (lane == 0) {
                lost_s = 1;
                if (a.status != nullptr) atomicOr(a.status, STATUS_TIMEOUT);
            }
        }
    }
    __syncthreads();

    // ---- parts of units, joined, four numbers of a column at a time
    // Open units of the CTA in their order: each begins with a head of a run (only the first run's, of a unit of CTAs ahead) or with a tail, goes on with tails and may end with a head.
    if (warp == 0) {
        bool first = false;
        int last_tail = -1, last_head = -1;
        const int w = lane / 2, tail = lane % 2;
        if (w < W) {
            const long long lo = tail ? tails_s[w].lo : heads_s[w].lo;
            first = lo >= 0;
            for (int v = 0; v < w; ++v) first &= tails_s[v].lo != lo;
            for (int v = w; v < W; ++v) {
                if (tails_s[v].lo == lo) last_tail = v;
                if ((v > w || !tail) && heads_s[v].lo == lo) last_head = v;
            }
        }
        const uint32_t all = __ballot_sync(0xffffffffu, first);
        if (first) opens_s[__popc(all & ((1u << lane) - 1))] = make_int4(w, tail ? last_tail : w - 1, last_head, 0);
        if (lane == 0) n_open_s = __popc(all);
    }
    __syncthreads();
    const int n_open = n_open_s, items = COLS * pad / 4;
    const long long all_places = line_s[0], cta_lo = line_s[1], cta_hi = line_s[2];
    auto open_unit = [&](int k) { const int4 o = opens_s[k]; return o.y < o.x ? heads_s[o.z] : tails_s[o.x]; };
    auto put_numbers = [&](const Open& u, int col, int d, float4 v, float m, float sum) {      // sums over all of the unit
        Sequence q;
        lengths_of(a, u.s, q);
        const int cols = q.n * a.group, tile = u.unit / a.kv_heads, head = u.unit - tile * a.kv_heads;
        col += tile * COLS;
        if (col >= cols) return;
        if (a.sink && m != -INFINITY) sum += exp2_fast(-m);
        const float f = lost_s ? __uint_as_float(0x7fc00000u) : m == -INFINITY && sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
        const int row = col / a.group, h = col - row * a.group;
        const float t[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
        put_four((T*)a.y + (long)(q.first + row) * a.ldy + (long)(head * a.group + h) * a.dv + d, a.dv - d, a.wide_y, t);
    };
    // (a part that has seen nothing counts for nothing, unless its sum is no number)
    auto weight = [](float pm, float m) { return pm == -INFINITY ? 0.f : exp2_fast(pm - m); };
    auto add_part = [](float& sum, float4& o, float w, float ps, float4 po) {
        sum += ps == ps ? ps * w : ps;
        o.x = fmaf(po.x, w, o.x); o.y = fmaf(po.y, w, o.y); o.z = fmaf(po.z, w, o.z); o.w = fmaf(po.w, w, o.w);
    };
    for (int x = tid; x < n_open * items; x += THREADS) {
        const int k = x / items, i = x - k * items, col = i * 4 / pad, d = i * 4 - col * pad;
        const int4 parts = opens_s[k];                     // tails x .. y, head z
        const Open u = open_unit(k);
        const float* const head = a.parts + (size_t)kMaxCtas * 2 * rec + ((size_t)cta * W + max(parts.z, 0)) * rec;
        auto tail = [&](int v) { return reinterpret_cast<const float*>(sm + v * a.slots * a.slot_bytes); };
        float m = parts.z >= 0 ? head[col] : -INFINITY, sum = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int v = parts.x; v <= parts.y; ++v) m = fmaxf(m, tail(v)[col]);
#pragma unroll 4
        for (int v = parts.x; v <= parts.y; ++v) add_part(sum, o, weight(tail(v)[col], m), tail(v)[COLS + col], *reinterpret_cast<const float4*>(tail(v) + 2 * COLS + i * 4));
        if (parts.z >= 0) add_part(sum, o, weight(head[col], m), head[COLS + col], *reinterpret_cast<const float4*>(head + 2 * COLS + i * 4));
        if (u.lo >= cta_lo && u.hi <= cta_hi) put_numbers(u, col, d, o, m, sum);
        else {
            float* const to = a.parts + ((size_t)cta * 2 + (u.lo < cta_lo ? 0 : 1)) * rec;
            *reinterpret_cast<float4*>(to + 2 * COLS + i * 4) = o;
            if (d == 0) { to[col] = m; to[COLS + col] = lost_s ? __uint_as_float(0x7fc00000u) : sum; }
        }
    }
    // ---- units that CTAs share: who arrives last joins them, in their order.  They are the CTA's first and last open ones.
    if (n_open == 0) return;
    const Open ends[2] = {open_unit(0), open_unit(n_open - 1)};
    const bool shared[2] = {ends[0].lo < cta_lo, ends[1].lo >= cta_lo && ends[1].hi > cta_hi};
    if (!shared[0] && !shared[1]) return;
    __threadfence();
    __syncthreads();
    if (tid < 2 && shared[tid]) {
        const Open u = ends[tid];
        const int sharers = (int)min((long long)gridDim.x, quotient(before[THREADS] + kCtaPages - 1, kCtaPages));
        long long ahead_of = 0;                            // places without a page ahead of the unit's first page
        if (units_before[THREADS] > sharers) {
            const int t = u.s / each;
            ahead_of = units_before[t] + u.unit + 1;
            for (int s = t * each; s < u.s; ++s) { bool bad; ahead_of += step_sequence(a, s, COLS, bad).units; }
            ahead_of *= kUnitCost;
        }
        const int c0 = (int)quotient((u.lo + ahead_of + 1) * sharers - 1, all_places), c1 = (int)quotient((u.hi + ahead_of) * sharers - 1, all_places);
        const bool last = atomicAdd(a.tickets + c0, 1) == c1 - c0;
        if (last) a.tickets[c0] = 0;
        shared_s[tid] = make_int4(c0, c1, last, 0);
    }
    __syncthreads();
    __threadfence();
    for (int place = 0; place < 2; ++place) {
        if (!shared[place] || !shared_s[place].z) continue;
        const Open u = ends[place];
        const int c0 = shared_s[place].x, c1 = shared_s[place].y;
        for (int i = tid; i < items; i += THREADS) {
            const int col = i * 4 / pad, d = i * 4 - col * pad;
            float m = -INFINITY, sum = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            auto place_of = [&](int c) { return a.parts + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * rec; };
#pragma unroll 8
            for (int c = c0; c <= c1; ++c) m = fmaxf(m, __ldcg(place_of(c) + col));
#pragma unroll 8
            for (int c = c0; c <= c1; ++c) {
                const float* const p = place_of(c);
                add_part(sum, o, weight(__ldcg(p + col), m), __ldcg(p + COLS + col), __ldcg(reinterpret_cast<const float4*>(p + 2 * COLS + i * 4)));
            }
            put_numbers(u, col, d, o, m, sum);
        }
    }
}

template <typename T, int NG, int MODE>
int32_t launch_step(AttendArgs a, uint64_t work, cudaStream_t st) {
    using Shape = StepShape<NG, MODE>;
    constexpr int W = Shape::kWarps;
    const int rec = part_floats(Shape::kCols, a.dv) * 4;
    a.slot_bytes = (std::max(kv4_block(a.dk, a.dv), rec) + 127) / 128 * 128;
    // 232448 bytes of shared memory per CTA, less what is declared in the kernel
    a.slots = std::min(4, (int)((232448 - 1024 - W * 704) / (W * a.slot_bytes)));
    a.tickets = (int32_t*)work;
    a.parts = (float*)(work + 4096);
    const size_t smem = (size_t)W * a.slots * a.slot_bytes;
    LUMI_CUDA(cudaFuncSetAttribute(kv4_step_kernel<T, NG, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    const int ctas = std::min(kMaxCtas, sm_count());
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // the launch itself overlaps the kernel in front
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    LUMI_CUDA(cudaLaunchKernelEx(&cfg, kv4_step_kernel<T, NG, MODE>, a));
    return LUMI_OK;
}

template <typename T>
int32_t step(const AttendArgs& a, uint64_t work, cudaStream_t st) {
    const int groups = std::max(kv4_groups(a.dk), kv4_groups(a.dv));
    if constexpr (sizeof(T) == 4) {
        const bool many = (long)a.group * a.max_new > 4;
        if (groups <= 2) return many ? launch_step<T, 2, 2>(a, work, st) : launch_step<T, 2, 3>(a, work, st);
        if (groups <= 4) return many ? launch_step<T, 4, 2>(a, work, st) : launch_step<T, 4, 3>(a, work, st);
        return many ? launch_step<T, 8, 2>(a, work, st) : launch_step<T, 8, 3>(a, work, st);
    } else {
        const bool many = (long)a.group * a.max_new > 8;
        if (groups <= 2) return many ? launch_step<T, 2, 1>(a, work, st) : launch_step<T, 2, 0>(a, work, st);
        if (groups <= 4) return many ? launch_step<T, 4, 1>(a, work, st) : launch_step<T, 4, 0>(a, work, st);
        return launch_step<T, 8, 0>(a, work, st);
    }
}

}  // namespace
}  // namespace lumi

using namespace lumi;

extern "C" int32_t lumi_k_kv4_attention_work_bytes(int32_t heads, int32_t kv_heads, int32_t dk, int32_t dv, int64_t* bytes) {
    if (!bytes || kv_heads <= 0 || heads <= 0 || heads % kv_heads || dk <= 0 || dv <= 0) return fail(LUMI_E_INVALID, "bad argument to lumi_k_kv4_attention_work_bytes");
    if (dk > kMaxHead || dv > kMaxHead || heads > 65535)
        return fail(LUMI_E_UNSUPPORTED, "lumi_k_kv4_attention_work_bytes: %d heads of %d and %d numbers (at most %d)", heads, dk, dv, kMaxHead);
    *bytes = 64 << 20;                                     // of both kernels' parts at their largest: 320 of 256 columns and 130 numbers
    return LUMI_OK;
}

namespace {

int32_t check_and_run(const char* what, uint64_t q, int32_t ldq, int32_t dtype, uint64_t kv, int32_t n_pages, uint64_t page_table, int32_t pages_per_seq, uint64_t row_start,
                      uint64_t tokens, uint64_t y, int32_t ldy, int32_t heads, int32_t kv_heads, int32_t dk, int32_t dv, int32_t window, float scale, int32_t sink, int32_t nseq,
                      int32_t rows, int32_t max_new, uint64_t work, uint64_t work_bytes, uint64_t status, uint64_t wait_ns, int32_t skip, cudaStream_t st) {
    const bool f32 = dtype == LUMI_DTYPE_F32;
    if (!q || !kv || !page_table || !row_start || !tokens || !y || !work || (!f32 && dtype != LUMI_DTYPE_BF16) || n_pages <= 0 || pages_per_seq <= 0 || heads <= 0 || kv_heads <= 0 ||
        heads % kv_heads || dk <= 0 || dv <= 0 || window < 0 || !(scale >= -3.4e38f && scale <= 3.4e38f) || nseq < 0 || rows < 0 || max_new < 0 || ldq < (long)heads * dk ||
        ldy < (long)heads * dv)
        return fail(LUMI_E_INVALID, "bad argument to %s", what);
    if ((kv & 15) || (work & 15) || ((page_table | row_start | tokens | status) & 3) || ((q | y) & (f32 ? 3 : 1)))
        return fail(LUMI_E_INVALID, "%s: cache and work area have to begin on 16-byte boundaries, numbers on their own", what);
    if (dk > kMaxHead || dv > kMaxHead || n_pages > kMaxPages || pages_per_seq > kMaxPages || heads > 65535 || rows > kMaxRows)
        return fail(LUMI_E_UNSUPPORTED, "%s: heads of %d and %d numbers (at most %d), %d heads, %d pages (at most %d), %d rows (at most %d)", what, dk, dv, kMaxHead, heads, n_pages,
                    kMaxPages, rows, kMaxRows);
    if ((long)std::min(rows, max_new) * (heads / kv_heads) > 1 << 30)      // columns of a sequence are 32-bit numbers
        return fail(LUMI_E_UNSUPPORTED, "%s: %d rows of %d heads on %d", what, std::min(rows, max_new), heads, kv_heads);
    int64_t need = 0;
    LUMI_TRY(lumi_k_kv4_attention_work_bytes(heads, kv_heads, dk, dv, &need));
    if (work_bytes < (uint64_t)need) return fail(LUMI_E_INVALID, "%s: a work area of %lld bytes, %lld are needed", what, (long long)work_bytes, (long long)need);
    if (nseq == 0 || rows == 0 || max_new == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory(what, {q, kv, page_table, row_start, tokens, y, work, status}));
    AttendArgs a{};
    a.q = (const void*)q; a.y = (void*)y; a.kv = (const uint8_t*)kv;
    a.table = (const int32_t*)page_table; a.row_start = (const int32_t*)row_start; a.tokens = (const int32_t*)tokens; a.status = (int32_t*)status;
    a.ldq = ldq; a.ldy = ldy; a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.dk = dk; a.dv = dv;
    a.window = window; a.sink = sink != 0; a.nseq = nseq; a.rows = rows; a.max_new = max_new; a.n_pages = n_pages; a.width = pages_per_seq; a.scale = scale;
    a.wide_q = (q & 15) == 0 && dk % 8 == 0 && (long)ldq * (f32 ? 4 : 2) % 16 == 0;
    a.wide_y = (y & (f32 ? 15 : 7)) == 0 && dv % 4 == 0 && ldy % 4 == 0;
    a.wide_y16 = (y & 15) == 0 && dv % (f32 ? 4 : 8) == 0 && ldy % (f32 ? 4 : 8) == 0;
    a.few = kFewColumns; a.wait_ns = wait_ns; a.skip = skip;
    LUMI_TRY(f32 ? step<float>(a, work, st) : step<__nv_bfloat16>(a, work, st));
    return (long)max_new * a.group > a.few ? launch_kv4_prompt(a, f32, work, st) : LUMI_OK;
}

}  // namespace

extern "C" int32_t lumi_k_kv4_attention(uint64_t q, int32_t ldq, int32_t dtype, uint64_t kv, int32_t n_pages, uint64_t page_table, int32_t pages_per_seq, uint64_t row_start,
                                        uint64_t tokens, uint64_t y, int32_t ldy, int32_t heads, int32_t kv_heads, int32_t dk, int32_t dv, int32_t window, float scale, int32_t sink,
                                        int32_t nseq, int32_t rows, int32_t max_new, uint64_t work, uint64_t work_bytes, uint64_t status, uint64_t stream) {
    return check_and_run("lumi_k_kv4_attention", q, ldq, dtype, kv, n_pages, page_table, pages_per_seq, row_start, tokens, y, ldy, heads, kv_heads, dk, dv, window, scale, sink, nseq, rows,
                         max_new, work, work_bytes, status, kWaitLimitNs, -1, (cudaStream_t)stream);
}

extern "C" int32_t lumi_debug_kv4_attention_wait_timeout(uint64_t q, int32_t ldq, int32_t dtype, uint64_t kv, int32_t n_pages, uint64_t page_table, int32_t pages_per_seq,
                                                         uint64_t row_start, uint64_t tokens, uint64_t y, int32_t ldy, int32_t heads, int32_t kv_heads, int32_t dk, int32_t dv,
                                                         int32_t window, float scale, int32_t sink, int32_t nseq, int32_t rows, int32_t max_new, uint64_t work, uint64_t work_bytes,
                                                         uint64_t status, uint64_t wait_limit_ns, int32_t skip_page) {
    if (!status || !wait_limit_ns) return fail(LUMI_E_INVALID, "bad argument to lumi_debug_kv4_attention_wait_timeout");
    LUMI_TRY(check_and_run("lumi_debug_kv4_attention_wait_timeout", q, ldq, dtype, kv, n_pages, page_table, pages_per_seq, row_start, tokens, y, ldy, heads, kv_heads, dk, dv, window, scale,
                           sink, nseq, rows, max_new, work, work_bytes, status, wait_limit_ns, skip_page, nullptr));
    int32_t word = 0;
    LUMI_CUDA(cudaMemcpy(&word, (const void*)status, sizeof(word), cudaMemcpyDeviceToHost));
    return (word & STATUS_TIMEOUT) ? fail(LUMI_E_TIMEOUT, "a bounded wait of the attention ran out") : LUMI_OK;
}
