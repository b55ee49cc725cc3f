// Attention over a paged cache in 4 bits: y = softmax(scale q K^T) V for the rows of sequences of different lengths, with an optional sliding window and an optional sink (one more
// score, 0, without a value).  Row i of a sequence's n new rows stands at position tokens - n + i and sees the positions up to its own.
//
// kv4_step_kernel (few rows per sequence): the work is a line of pages, unit after unit; a unit is a sequence's head of the cache with up to 8 or 16 columns, a column being a row and a query
// head that reads that cache head.  CTAs, and within them warps, take equal runs of that line, whatever the lengths.  A page's block comes by one bulk copy into the warp's ring, and a warp
// needs no other one until its run ends: then the parts of a unit are joined, first within the CTA, then by the CTA that arrives last.
//
// Scores: columns are the rows of A (fp16, times a power of two per column), keys are B: codes n as subnormals n 2^-24 straight from the words (an AND each), those of a word's second
// pair as n 2^-20 against q / 16.  The accumulator starts at -8 sum q, so that it ends with sum q (n - 8); a fp32 multiply-add per score and group brings the scale in.  Nothing is
// rounded but q: as two fp16 terms of fp32 rows, whole of bf16 rows.
// Values: codes are A (numbers of a head in its rows, tokens along K, which the transposing matrix load gives), softmax weights times the group's scale are B.  These products are kept
// in fp16's range by 2^7 / (largest scale so far), and 8 sum p s is taken off at the end (one more MMA with a constant A).  fp32 rows: two fp16 terms of p s; bf16 rows: one (2^-12).
//
// Bound by memory on paper (18 bytes per 32 numbers), and close to the issue rate in fact: a page of 128 + 128 numbers is 9216 bytes and about 850 warp instructions.
#include "device_args.h"
#include "kv4.cuh"
#include "rows.cuh"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace lumi {
namespace {

constexpr int kMaxRows = 1 << 24;                          // numbers of parts of work are 32-bit numbers
constexpr int kBadPage = 1;                                // bit of the status word: a page or a length outside of what the cache holds
constexpr int kMaxCtas = 296;                              // of the step kernel: places for parts
constexpr float kLog2e = 1.4426950408889634f;

struct AttendArgs {
    const void* q; void* y;
    const uint8_t* kv;
    const int32_t *table, *row_start, *tokens;
    int32_t* status;
    int32_t* tickets;                                      // [kMaxCtas], zero between calls
    float* parts;                                          // [kMaxCtas][2] parts of units that CTAs share, then [kMaxCtas][warps] of units that end within a warp's run
    uint64_t wait_ns;
    long ldq, ldy;
    int heads, kv_heads, group, dk, dv, window, sink, nseq, rows, max_new, n_pages, width;
    int few;                                               // columns per head of the cache up to which a sequence is the step kernel's
    int slots, slot_bytes;                                 // of a warp's ring
    int skip;                                              // failure tests: the copy of this page of the line is not issued
    float scale;
};

__device__ __forceinline__ float number(const float* p) { return *p; }
__device__ __forceinline__ float number(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    mma16(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unhalves(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ float low_bf16(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_bf16(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127

// What a sequence is to the call.
struct Sequence { int first, n, total, page0, pages, units; };
__device__ __forceinline__ bool lengths_of(const AttendArgs& a, int s, Sequence& q) {      // false: they make no sense
    q.first = a.row_start[s];
    const int end = a.row_start[s + 1];
    q.total = a.tokens[s];
    q.n = end - q.first;
    return q.first >= 0 && end >= q.first && end <= a.rows && q.total >= q.n && q.total <= (long)a.width * kPage;
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
// MODE 0: up to 8 columns of bf16 rows; 1: up to 16; 2: up to 8 columns of fp32 rows, as two terms.
template <int NG, int MODE>
struct StepShape {
    static constexpr int kCols = MODE == 1 ? 16 : 8;
    // registers: accumulators of values 4 NG per eight columns and number block, of their offsets, scores, q
    static constexpr int kWarps = NG == 8 ? 6 : MODE == 1 ? (NG == 4 ? 8 : 12) : (NG == 4 ? 12 : 16);
    static constexpr int kStage = 1024;                    // of a warp: one group of its columns on their way into registers
};

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// One part of a unit: columns' largest score m (in units of log2), sum l and numbers o [column][dv], all relative to 2^m.  Where parts lie: m [cols], l [cols], o [cols][pad].
__host__ __device__ inline int part_floats(int cols, int dv) { return cols * (2 + kv4_groups(dv) * kGroup); }

struct Open { long long lo, hi; int s, unit; };

template <typename T, int NG, int MODE>
__global__ void __launch_bounds__(StepShape<NG, MODE>::kWarps * 32, 1) kv4_step_kernel(const AttendArgs a) {
    using Shape = StepShape<NG, MODE>;
    constexpr int W = Shape::kWarps, COLS = Shape::kCols, NT = W * 32, SETS = MODE == 1 ? 2 : 1;
    constexpr bool TWO = MODE == 2;                        // two terms of q and of the weights
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ long long before[NT + 1];                   // pages of the sequences ahead of each thread's
    __shared__ uint64_t full[W][4];
    __shared__ long long warp_pages[W];
    __shared__ Open heads_s[W], tails_s[W];                // units that began ahead of a warp's run and end in it; that its run ends with and that it does not hold whole
    __shared__ int last_s, lost_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i8 = lane >> 2, j4 = lane & 3;
    uint8_t* const ring = sm + (size_t)warp * a.slots * a.slot_bytes;
    uint8_t* const stage = sm + (size_t)W * a.slots * a.slot_bytes + warp * Shape::kStage;
    const int gk = kv4_groups(a.dk), gv = kv4_groups(a.dv), part = kv4_part(a.dk), block = kv4_block(a.dk, a.dv);
    const int rec = part_floats(COLS, a.dv), pad = gv * kGroup;

    if (lane < 4) mbar_init(&full[warp][lane], 1);
    if (lane == 0) heads_s[warp].lo = tails_s[warp].lo = -1;
    if (tid == 0) lost_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    pdl_release();
    pdl_sync();

    // ---- the line of pages: each thread sums up a run of sequences
    const int each = (a.nseq + NT - 1) / NT, s_lo = min(a.nseq, tid * each), s_hi = min(a.nseq, s_lo + each);
    long long mine = 0;
    bool any_bad = false;
    for (int s = s_lo; s < s_hi; ++s) {
        bool bad;
        const Sequence q = step_sequence(a, s, COLS, bad);
        any_bad |= bad;
        mine += (long long)q.pages * q.units;
    }
    if (any_bad && blockIdx.x == 0 && a.status != nullptr) atomicOr(a.status, kBadPage);
    long long run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += t; }
    if (lane == 31) warp_pages[warp] = run;
    __syncthreads();
    long long ahead = 0, total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) { const long long p = warp_pages[w]; if (w < warp) ahead += p; total += p; }
    before[tid] = ahead + run - mine;
    if (tid == NT - 1) before[NT] = total;
    __syncthreads();
    // CTAs that get work: a page per warp at least.  CTA c takes the pages from c total / ctas on.
    const int ctas = (int)min((long long)gridDim.x, (total + W - 1) / W), cta = blockIdx.x;
    if (cta >= ctas) return;
    const long long c_lo = total * cta / ctas, c_hi = total * (cta + 1) / ctas;
    auto warp_from = [&](int w) { return c_lo + (c_hi - c_lo) * w / W; };
    const long long x_lo = warp_from(warp), x_hi = warp_from(warp + 1);

    // where page x of the line lies: sequence, unit, page of the unit's
    struct Spot { int s, unit, p, page; };
    auto find = [&](long long x) {
        int lo = 0, hi = NT;
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
                r.unit = (int)(rel / q.pages);
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

    // ---- state of the unit at hand
    float O[SETS][2 * NG][4], OFF[SETS][NG][4], m[SETS], l[SETS];
    uint32_t Q[2 * NG][4];
    float qc[NG][2];                                       // what the scores' accumulators start at
    float cx[SETS];                                        // factor from accumulators to scores in units of log2
    int lo_pos[SETS], hi_pos[SETS];                        // positions that the column sees: lo .. hi
    int e_v = 0;                                           // scales of values are below 2^e_v so far
    int first_full = 0, last_full = 0;                     // pages whose every token is seen by every column, as positions: [first_full, last_full]
    bool dead = false;                                     // a wait gave up
    const float sign = a.scale < 0.f ? -1.f : 1.f;

    auto begin_unit = [&](const Sequence& q, int unit) {
        const int cols = q.n * a.group, head = unit % a.kv_heads, col0 = unit / a.kv_heads * COLS;
        float raw[COLS][NG];
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            const int col = col0 + c;
            const T* const p = (const T*)a.q + (long)(q.first + col / a.group) * a.ldq + (long)(head * a.group + col % a.group) * a.dk;
#pragma unroll
            for (int g = 0; g < NG; ++g) raw[c][g] = col < cols && g * kGroup + lane < a.dk ? number(p + g * kGroup + lane) : 0.f;
        }
        // times a power of two that brings the column's largest to 2^13 .. 2^14
        float by[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            uint32_t top = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) top = max(top, __float_as_uint(raw[c][g]) & 0x7fffffffu);
            top = __reduce_max_sync(0xffffffffu, top);
            const int k = top >= 0x7f800000u || top == 0 ? 0 : min(126, 13 + 127 - (int)(top >> 23));
            by[c] = power_of_two(k) * sign;
        }
        // number d of a group: word j, pair half, step; the second pair of a step meets codes that are 16 times as large
        const int step = lane % 8 / 4, half = lane % 4 / 2, k8 = lane / 8 * 2 + lane % 2;
        uint16_t* const to = reinterpret_cast<uint16_t*>(stage) + (step * 2 + half) * 128 + k8;
        const float sixteenth = half ? 0.0625f : 1.f;
        const uint32_t from = smem_u32(stage) + (lane / 16) * 256 + (lane % 16) * 16;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (g >= gk) break;
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const float v = raw[c][g] * by[c] * sixteenth;
                const __half h = __float2half_rn(v);
                to[c * 8] = __half_as_ushort(h);
                if (TWO) to[(c + 8) * 8] = __half_as_ushort(__float2half_rn(v - __half2float(h)));
                else if (COLS == 8) to[(c + 8) * 8] = 0;
            }
            __syncwarp();
            ldmatrix4(from, Q[2 * g]);
            ldmatrix4(from + 512, Q[2 * g + 1]);
            __syncwarp();
            float t[4];
            mma16(t, Q[2 * g][0], Q[2 * g][1], Q[2 * g][2], Q[2 * g][3], 0x80088008u, 0x80808080u, 0.f, 0.f, 0.f, 0.f);          // -8 2^-24 and -128 2^-24
            mma16(t, Q[2 * g + 1][0], Q[2 * g + 1][1], Q[2 * g + 1][2], Q[2 * g + 1][3], 0x80088008u, 0x80808080u);
            qc[g][0] = t[0]; qc[g][1] = t[2];
        }
        first_full = 0; last_full = 0x7fffffff;
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
            float b = 1.f;
#pragma unroll
            for (int c = 0; c < 8; ++c) if (c == i8) b = by[set * 8 + c] * sign;
            cx[set] = fminf(fmaxf(__fdiv_rn(fabsf(a.scale) * kLog2e, b) * 16777216.f, 1e-37f), 3.4e38f);      // (not 0: hidden scores are -inf)
            const int row = min(col0 + set * 8 + i8, cols - 1) / a.group, pos = q.total - q.n + row;
            hi_pos[set] = pos;
            lo_pos[set] = a.window > 0 ? max(0, pos - a.window + 1) : 0;
            m[set] = -INFINITY;
            l[set] = 0.f;
        }
        {
            const int row0 = col0 / a.group, row1 = min(col0 + COLS, cols) - 1;
            last_full = q.total - q.n + row0;
            const int far = q.total - q.n + row1 / a.group;
            first_full = a.window > 0 ? max(0, far - a.window + 1) : 0;
        }
        e_v = -90;
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
#pragma unroll
            for (int t = 0; t < 2 * NG; ++t) O[set][t][0] = O[set][t][1] = O[set][t][2] = O[set][t][3] = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) OFF[set][g][0] = OFF[set][g][1] = OFF[set][g][2] = OFF[set][g][3] = 0.f;
        }
    };
    auto scale_values = [&](int set, float f0, float f1) {     // of columns 2 j and 2 j + 1
#pragma unroll
        for (int t = 0; t < 2 * NG; ++t) { O[set][t][0] *= f0; O[set][t][1] *= f1; O[set][t][2] *= f0; O[set][t][3] *= f1; }
#pragma unroll
        for (int g = 0; g < NG; ++g) { OFF[set][g][0] *= f0; OFF[set][g][1] *= f1; OFF[set][g][2] *= f0; OFF[set][g][3] *= f1; }
    };

    // ---- one page of the unit
    auto work_page = [&](uint8_t* slot, int pos0) {
        const uint32_t base = smem_u32(slot);
        const bool edge = pos0 < first_full || pos0 + kPage - 1 > last_full;
        if (edge) {
            // scales of tokens that no column sees may be any bits: they become 0
            const int lo = __reduce_min_sync(0xffffffffu, SETS == 2 ? min(lo_pos[0], lo_pos[SETS - 1]) : lo_pos[0]);
            const int hi = __reduce_max_sync(0xffffffffu, SETS == 2 ? max(hi_pos[0], hi_pos[SETS - 1]) : hi_pos[0]);
            uint16_t* const sv = reinterpret_cast<uint16_t*>(slot + part + gv * kPlane);
            for (int k = lane; k < gv * kPage; k += 32) {
                const int pos = pos0 + k % kPage;
                if (pos < lo || pos > hi) sv[k] = 0;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        }
        float S[SETS][8][2];
#pragma unroll
        for (int set = 0; set < SETS; ++set)
#pragma unroll
            for (int t = 0; t < 8; ++t) S[set][t][0] = S[set][t][1] = 0.f;
        // scores
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (g >= gk) break;
            const uint32_t codes = base + g * kPlane + lane * 16, scales = base + gk * kPlane + g * kScales + (lane / 8) * 16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[4], sc[4];
                ldmatrix4(codes + h * 512, w);
                ldmatrix4(scales + h * 64, sc);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float d[4];
                    mma16(d, Q[2 * g][0], Q[2 * g][1], Q[2 * g][2], Q[2 * g][3], w[t] & 0x000f000fu, w[t] & 0x00f000f0u, qc[g][0], qc[g][0], qc[g][1], qc[g][1]);
                    const uint32_t u = w[t] >> 8;
                    mma16(d, Q[2 * g + 1][0], Q[2 * g + 1][1], Q[2 * g + 1][2], Q[2 * g + 1][3], u & 0x000f000fu, u & 0x00f000f0u);
                    const float s0 = low_bf16(sc[t]), s1 = high_bf16(sc[t]);
                    if (TWO) { d[0] += d[2]; d[1] += d[3]; }
                    S[0][h * 4 + t][0] = fmaf(d[0], s0, S[0][h * 4 + t][0]);
                    S[0][h * 4 + t][1] = fmaf(d[1], s1, S[0][h * 4 + t][1]);
                    if (SETS == 2) {
                        S[SETS - 1][h * 4 + t][0] = fmaf(d[2], s0, S[SETS - 1][h * 4 + t][0]);
                        S[SETS - 1][h * 4 + t][1] = fmaf(d[3], s1, S[SETS - 1][h * 4 + t][1]);
                    }
                }
            }
        }
        if (edge) {
#pragma unroll
            for (int set = 0; set < SETS; ++set)
#pragma unroll
                for (int t = 0; t < 8; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int pos = pos0 + t * 8 + 2 * j4 + e;
                        if (pos < lo_pos[set] || pos > hi_pos[set]) S[set][t][e] = -INFINITY;
                    }
        }
        // the largest scale of values: a lane looks at eight of them
        {
            uint32_t top = 0;
            const uint4* const sv = reinterpret_cast<const uint4*>(slot + part + gv * kPlane);
#pragma unroll
            for (int k = 0; k < (NG + 3) / 4; ++k) {
                const int at = k * 32 + lane;
                if (at < gv * 8) {
                    const uint4 u = sv[at];
                    const __nv_bfloat162* const b = reinterpret_cast<const __nv_bfloat162*>(&u);
                    const __nv_bfloat162 x = __hmax2(__hmax2(b[0], b[1]), __hmax2(b[2], b[3]));
                    const uint32_t bits = *reinterpret_cast<const uint32_t*>(&x);
                    const uint32_t b0 = bits & 0x7fffu, b1 = bits >> 16 & 0x7fffu;
                    top = max(top, max(b0 < 0x7f80u ? b0 : 0u, b1 < 0x7f80u ? b1 : 0u));      // what is no number has no size
                }
            }
            const int e = min(127, (int)(top >> 7) - 126);     // the largest is below 2^e
            if (__any_sync(0xffffffffu, e > e_v)) {
                const int to = __reduce_max_sync(0xffffffffu, e), by = max(e_v - to, -252);
                const float f = power_of_two(by / 2), f2 = power_of_two(by - by / 2);
#pragma unroll
                for (int set = 0; set < SETS; ++set) {
                    scale_values(set, f, f);
                    scale_values(set, f2, f2);
                    l[set] = l[set] * f * f2;
                }
                e_v = to;
            }
        }
        // weights relative to the running maximum, which moves where it would have to by more than 2^8
        const int up = 7 - e_v;
        bool moves = false;
        float top[SETS];
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
            float t = S[set][0][0];
#pragma unroll
            for (int k = 0; k < 8; ++k) t = fmaxf(t, fmaxf(S[set][k][0], S[set][k][1]));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            top[set] = t * cx[set];
            moves |= top[set] > m[set] + 8.f || (m[set] == -INFINITY && top[set] > -INFINITY);
        }
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int set = 0; set < SETS; ++set) {
                const float to = fmaxf(m[set], top[set]);
                const float f = m[set] == -INFINITY ? 0.f : exp2_fast(m[set] - to);      // nothing so far: the numbers are 0
                m[set] = to;
                l[set] *= f;
                scale_values(set, __shfl_sync(0xffffffffu, f, 8 * j4), __shfl_sync(0xffffffffu, f, 8 * j4 + 4));
            }
        }
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
            const float off = m[set] == -INFINITY ? 0.f : (float)up - m[set];
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                S[set][t][0] = exp2_fast(fmaf(S[set][t][0], cx[set], off));
                S[set][t][1] = exp2_fast(fmaf(S[set][t][1], cx[set], off));
                l[set] += S[set][t][0] + S[set][t][1];
            }
        }
        // values
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (g >= gv) break;
            const uint32_t codes = base + part + g * kPlane + lane * 16, scales = base + part + gv * kPlane + g * kScales + (lane / 8) * 16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[4], sc[4];
                ldmatrix4_trans(codes + h * 512, w);
                ldmatrix4(scales + h * 64, sc);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t r0 = w[2 * k], r1 = w[2 * k + 1], u0 = r0 >> 8, u1 = r1 >> 8;
                    const float s0 = low_bf16(sc[2 * k]), s1 = high_bf16(sc[2 * k]), s2 = low_bf16(sc[2 * k + 1]), s3 = high_bf16(sc[2 * k + 1]);
#pragma unroll
                    for (int set = 0; set < SETS; ++set) {
                        const float(&p)[2] = S[set][h * 4 + 2 * k];
                        const float(&q)[2] = S[set][h * 4 + 2 * k + 1];
                        const float v0 = p[0] * s0, v1 = p[1] * s1, v2 = q[0] * s2, v3 = q[1] * s3;
                        uint32_t b0 = halves(v0, v1), b1 = halves(v2, v3);
#pragma unroll
                        for (int term = 0; term < (TWO ? 2 : 1); ++term) {
                            mma16(O[set][2 * g], r0 & 0x000f000fu, r0 & 0x00f000f0u, r1 & 0x000f000fu, r1 & 0x00f000f0u, b0, b1);
                            mma16(O[set][2 * g + 1], u0 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x000f000fu, u1 & 0x00f000f0u, b0, b1);
                            mma16(OFF[set][g], 0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u, b0, b1);
                            if (TWO && term == 0) {
                                const float2 h0 = unhalves(b0), h1 = unhalves(b1);
                                b0 = halves(v0 - h0.x, v1 - h0.y);
                                b1 = halves(v2 - h1.x, v3 - h1.y);
                            }
                        }
                    }
                }
            }
        }
    };

    // ---- what a unit leaves: numbers 4 i .. 4 i + 3 of each group, of columns 2 j and 2 j + 1, before the division by the sum
    auto number_at = [&](int set, int g, int t, int col) { return (O[set][2 * g + (t >> 1)][(t & 1) * 2 + col] * ((t & 1) ? 0.0625f : 1.f) - OFF[set][g][col]); };
    auto finish_unit = [&](int s, int unit) {              // the whole unit was this warp's
        Sequence q;
        lengths_of(a, s, q);
        const int cols = q.n * a.group, head = unit % a.kv_heads, col0 = unit / a.kv_heads * COLS;
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
            float sum = l[set];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (a.sink && m[set] != -INFINITY) sum += exp2_fast((float)(7 - e_v) - m[set]);
            const float inv = dead ? __uint_as_float(0x7fc00000u) : m[set] == -INFINITY && sum == 0.f ? 0.f : __fdiv_rn(16777216.f, sum);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f = __shfl_sync(0xffffffffu, inv, 8 * j4 + 4 * e);
                const int col = col0 + set * 8 + 2 * j4 + e;
                if (col >= cols) continue;
                T* const y = (T*)a.y + (long)(q.first + col / a.group) * a.ldy + (long)(head * a.group + col % a.group) * a.dv;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (g >= gv) break;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const int d = g * kGroup + 4 * i8 + t;
                        if (d < a.dv) y[d] = (T)(number_at(set, g, t, e) * f);
                    }
                }
            }
        }
    };
    auto leave_part = [&](float* to) {
        const float by = power_of_two(e_v / 2), by2 = power_of_two(e_v - e_v / 2);          // back from 2^(7 - e_v)
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
            float sum = l[set];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (j4 == 0) {
                to[set * 8 + i8] = m[set];
                to[COLS + set * 8 + i8] = dead ? __uint_as_float(0x7fc00000u) : sum * 0.0078125f * by * by2;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (g >= gv) break;
                    float v[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) v[t] = number_at(set, g, t, e) * 131072.f * by * by2;
                    *reinterpret_cast<float4*>(to + 2 * COLS + (set * 8 + 2 * j4 + e) * pad + g * kGroup + 4 * i8) = make_float4(v[0], v[1], v[2], v[3]);
                }
        }
    };

    // ---- the warp's run
    float* const head_part = a.parts + (size_t)kMaxCtas * 2 * rec + ((size_t)cta * W + warp) * rec;
    uint32_t pending = 0, phases = 0;                      // bits of slots: a copy is on its way; parity of the next one's end
    Spot now{0, 0, 0, -1}, then{0, 0, 0, -1};              // of the 32 pages at hand, one per lane, and of the next 32
    auto issue = [&](long long x, int slot, int page, int unit) {      // (uniform)
        if (page < 0) return;
        pending |= 1u << slot;
        if (lane == 0) {
            mbar_expect_tx(&full[warp][slot], block);
            if (x != a.skip) bulk_copy(smem_u32(ring) + slot * a.slot_bytes, a.kv + ((size_t)page * a.kv_heads + unit % a.kv_heads) * block, block, &full[warp][slot]);
        }
    };
    int s = 0, unit = 0, pages = 0, page0 = 0;             // the unit at hand
    long long unit_lo = -1, unit_hi = -1;                  // its pages of the line
    if (x_lo < x_hi) {
        long long batch = x_lo, asked = x_lo;
        if (batch + lane < x_hi) now = find(batch + lane);
        for (; asked < min(x_hi, x_lo + a.slots); ++asked) {
            const int k = (int)(asked - batch);
            issue(asked, k, __shfl_sync(0xffffffffu, now.page, k), __shfl_sync(0xffffffffu, now.unit, k));
        }
        int slot = 0;
        for (long long x = x_lo; x < x_hi; ++x) {
            const int k = (int)(x - batch), p = __shfl_sync(0xffffffffu, now.p, k);
            if (x == x_lo || p == 0) {
                s = __shfl_sync(0xffffffffu, now.s, k);
                unit = __shfl_sync(0xffffffffu, now.unit, k);
                bool bad;
                const Sequence q = step_sequence(a, s, COLS, bad);
                pages = q.pages; page0 = q.page0;
                unit_lo = x - p; unit_hi = unit_lo + pages;
                begin_unit(q, unit);
            }
            if (k == 8 && batch + 32 < x_hi && batch + 32 + lane < x_hi) then = find(batch + 32 + lane);
            __syncwarp();
            if (pending >> slot & 1) {
                if (!dead) dead = __any_sync(0xffffffffu, !mbar_wait(&full[warp][slot], phases >> slot & 1, a.wait_ns));
                if (!dead) {
                    pending &= ~(1u << slot);
                    phases ^= 1u << slot;
                    work_page(ring + slot * a.slot_bytes, (page0 + p) * kPage);
                    __syncwarp();
                }
            }
            if (p == pages - 1) {
                if (unit_lo >= x_lo) finish_unit(s, unit);
                else if (x + 1 < x_hi) {
                    leave_part(head_part);
                    if (lane == 0) heads_s[warp] = Open{unit_lo, unit_hi, s, unit};
                }
            }
            // the slot is free for the page `slots` further on
            if (asked < x_hi && !dead) {
                const int kk = (int)(asked - batch);
                const int page = __shfl_sync(0xffffffffu, kk < 32 ? now.page : then.page, kk & 31), u = __shfl_sync(0xffffffffu, kk < 32 ? now.unit : then.unit, kk & 31);
                issue(asked, slot, page, u);
                ++asked;
            }
            if (k == 31) { now = then; batch += 32; }
            slot = slot + 1 == a.slots ? 0 : slot + 1;
        }
        for (int i = 0; i < a.slots; ++i)                  // (only after a wait gave up: copies in flight land before the CTA ends)
            if (pending >> i & 1) mbar_wait(&full[warp][i], phases >> i & 1, a.wait_ns);
        if (dead && lane == 0) {
            lost_s = 1;
            if (a.status != nullptr) atomicOr(a.status, STATUS_TIMEOUT);
        }
        const bool open = unit_hi > x_hi || unit_lo < x_lo;    // the last unit goes on, or began ahead and ends with the run
        if (open) {
            leave_part(reinterpret_cast<float*>(ring));
            if (lane == 0) tails_s[warp] = Open{unit_lo, unit_hi, s, unit};
        }
    }
    __syncthreads();

    // ---- parts of units, joined: numbers 4 at a time, a column's weights by each thread for itself
    auto put_numbers = [&](int s, int unit, int col, int d, float4 v, float m, float sum) {      // sums over all of the unit
        Sequence q;
        lengths_of(a, s, q);
        const int cols = q.n * a.group, head = unit % a.kv_heads;
        col += unit / a.kv_heads * COLS;
        if (col >= cols) return;
        if (a.sink && m != -INFINITY) sum += exp2_fast(-m);
        const float f = lost_s ? __uint_as_float(0x7fc00000u) : m == -INFINITY && sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
        T* const y = (T*)a.y + (long)(q.first + col / a.group) * a.ldy + (long)(head * a.group + col % a.group) * a.dv + d;
        const float t[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
#pragma unroll
        for (int i = 0; i < 4; ++i) if (d + i < a.dv) y[i] = (T)t[i];
    };
    // adds a part, given its largest score, to sums relative to m
    auto join = [](float& m, float& sum, float4& o, float pm, float ps, float4 po) {
        const float to = fmaxf(m, pm), f = m == -INFINITY ? 0.f : exp2_fast(m - to), g = pm == -INFINITY ? 0.f : exp2_fast(pm - to);
        m = to;
        sum = sum * f + (ps == ps ? ps * g : ps);
        o.x = o.x * f + po.x * g; o.y = o.y * f + po.y * g; o.z = o.z * f + po.z * g; o.w = o.w * f + po.w * g;
    };
    Open shared_units[2];
    shared_units[0].lo = shared_units[1].lo = -1;
    for (int w = 0; w < W; ++w)
        for (int kind = 0; kind < 2; ++kind) {             // a run's head lies ahead of its tail
            const Open u = kind == 0 ? heads_s[w] : tails_s[w];
            if (u.lo < 0) continue;
            bool first = true;
            for (int v = 0; v < w; ++v) first &= tails_s[v].lo != u.lo;
            if (!first) continue;
            const bool whole = u.lo >= c_lo && u.hi <= c_hi;
            const int place = u.lo < c_lo ? 0 : 1;
            float* const to = a.parts + ((size_t)cta * 2 + place) * rec;
            for (int i = tid; i < COLS * pad / 4; i += NT) {
                const int col = i * 4 / pad, d = i * 4 % pad;
                float m = -INFINITY, sum = 0.f;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int v = w; v < W; ++v)
                    for (int k2 = v == w ? kind : 0; k2 < 2; ++k2) {
                        if ((k2 == 0 ? heads_s[v].lo : tails_s[v].lo) != u.lo) continue;
                        const float* const p = k2 == 0 ? a.parts + (size_t)kMaxCtas * 2 * rec + ((size_t)cta * W + v) * rec : reinterpret_cast<const float*>(sm + (size_t)v * a.slots * a.slot_bytes);
                        join(m, sum, o, p[col], p[COLS + col], *reinterpret_cast<const float4*>(p + 2 * COLS + i * 4));
                    }
                if (whole) put_numbers(u.s, u.unit, col, d, o, m, sum);
                else {
                    *reinterpret_cast<float4*>(to + 2 * COLS + i * 4) = o;
                    if (d == 0) { to[col] = m; to[COLS + col] = lost_s ? __uint_as_float(0x7fc00000u) : sum; }
                }
            }
            if (!whole) shared_units[place] = u;
        }
    // ---- units that CTAs share: who arrives last joins them, in their order
    for (int place = 0; place < 2; ++place) {
        const Open u = shared_units[place];
        if (u.lo < 0) continue;                            // (the same for all threads)
        const int c0 = (int)(((u.lo + 1) * ctas - 1) / total), c1 = (int)((u.hi * ctas - 1) / total);
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            const int n = atomicAdd(a.tickets + c0, 1);
            last_s = n == c1 - c0;
            if (last_s) a.tickets[c0] = 0;
        }
        __syncthreads();
        if (!last_s) continue;
        __threadfence();
        for (int i = tid; i < COLS * pad / 4; i += NT) {
            const int col = i * 4 / pad, d = i * 4 % pad;
            float m = -INFINITY, sum = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int c = c0; c <= c1; ++c) {
                const float* const p = a.parts + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * rec;
                join(m, sum, o, __ldcg(p + col), __ldcg(p + COLS + col), __ldcg(reinterpret_cast<const float4*>(p + 2 * COLS + i * 4)));
            }
            put_numbers(u.s, u.unit, col, d, o, m, sum);
        }
        __syncthreads();
    }
}

template <typename T, int NG, int MODE>
int32_t launch_step(AttendArgs a, uint64_t work, cudaStream_t st) {
    using Shape = StepShape<NG, MODE>;
    constexpr int W = Shape::kWarps;
    const int rec = part_floats(Shape::kCols, a.dv) * 4;
    a.slot_bytes = (std::max(kv4_block(a.dk, a.dv), rec) + 127) / 128 * 128;
    // 232448 bytes of shared memory per CTA, less what is declared in the kernel
    a.slots = std::min(4, (int)((232448 - 1024 - W * (Shape::kStage + 360)) / (W * a.slot_bytes)));
    a.tickets = (int32_t*)work;
    a.parts = (float*)(work + 4096);
    const size_t smem = (size_t)W * (a.slots * a.slot_bytes + Shape::kStage);
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
        if (groups <= 2) return launch_step<T, 2, 2>(a, work, st);
        if (groups <= 4) return launch_step<T, 4, 2>(a, work, st);
        return launch_step<T, 8, 2>(a, work, st);
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
    *bytes = 64 << 20;
    return LUMI_OK;
}

extern "C" int32_t lumi_k_kv4_attention(uint64_t q, int32_t ldq, int32_t dtype, uint64_t kv, int32_t n_pages, uint64_t page_table, int32_t pages_per_seq, uint64_t row_start,
                                        uint64_t tokens, uint64_t y, int32_t ldy, int32_t heads, int32_t kv_heads, int32_t dk, int32_t dv, int32_t window, float scale, int32_t sink,
                                        int32_t nseq, int32_t rows, int32_t max_new, uint64_t work, uint64_t work_bytes, uint64_t status, uint64_t stream) {
    const bool f32 = dtype == LUMI_DTYPE_F32;
    if (!q || !kv || !page_table || !row_start || !tokens || !y || !work || (!f32 && dtype != LUMI_DTYPE_BF16) || n_pages <= 0 || pages_per_seq <= 0 || heads <= 0 || kv_heads <= 0 ||
        heads % kv_heads || dk <= 0 || dv <= 0 || window < 0 || !(scale >= -3.4e38f && scale <= 3.4e38f) || nseq < 0 || rows < 0 || max_new < 0 || ldq < (long)heads * dk ||
        ldy < (long)heads * dv)
        return fail(LUMI_E_INVALID, "bad argument to lumi_k_kv4_attention");
    if ((kv & 15) || (work & 15) || ((page_table | row_start | tokens | status) & 3) || ((q | y) & (f32 ? 3 : 1)))
        return fail(LUMI_E_INVALID, "lumi_k_kv4_attention: cache and work area have to begin on 16-byte boundaries, numbers on their own");
    if (dk > kMaxHead || dv > kMaxHead || n_pages > kMaxPages || pages_per_seq > kMaxPages || heads > 65535 || rows > kMaxRows)
        return fail(LUMI_E_UNSUPPORTED, "lumi_k_kv4_attention: heads of %d and %d numbers (at most %d), %d heads, %d pages (at most %d), %d rows (at most %d)", dk, dv, kMaxHead,
                    heads, n_pages, kMaxPages, rows, kMaxRows);
    int64_t need = 0;
    LUMI_TRY(lumi_k_kv4_attention_work_bytes(heads, kv_heads, dk, dv, &need));
    if (work_bytes < (uint64_t)need) return fail(LUMI_E_INVALID, "lumi_k_kv4_attention: a work area of %lld bytes, %lld are needed", (long long)work_bytes, (long long)need);
    if (nseq == 0 || rows == 0 || max_new == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory("lumi_k_kv4_attention", {q, kv, page_table, row_start, tokens, y, work, status}));
    AttendArgs a{};
    a.q = (const void*)q; a.y = (void*)y; a.kv = (const uint8_t*)kv;
    a.table = (const int32_t*)page_table; a.row_start = (const int32_t*)row_start; a.tokens = (const int32_t*)tokens; a.status = (int32_t*)status;
    a.ldq = ldq; a.ldy = ldy; a.heads = heads; a.kv_heads = kv_heads; a.group = heads / kv_heads; a.dk = dk; a.dv = dv;
    a.window = window; a.sink = sink != 0; a.nseq = nseq; a.rows = rows; a.max_new = max_new; a.n_pages = n_pages; a.width = pages_per_seq; a.scale = scale;
    a.few = 1 << 30; a.wait_ns = kWaitLimitNs; a.skip = -1;
    return f32 ? step<float>(a, work, (cudaStream_t)stream) : step<__nv_bfloat16>(a, work, (cudaStream_t)stream);
}
