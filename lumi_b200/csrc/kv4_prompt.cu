// Attention over the paged cache in 4 bits for many rows per sequence, on the tensor cores (tcgen05): prompts, and slices behind what a sequence holds already.
//
// A tile is 128 columns (a column: a row and a query head that reads the unit's cache head), two tiles of a unit at once for heads of up to 128 numbers.  CTAs take equal runs of the
// line of pages of all units, whatever the lengths; a unit that CTAs share is joined by the one that arrives last.  Per page of 64 tokens:
//
//   copy warp        the page's block into a ring, by one bulk copy
//   4 dequant warps  codes and scales to (n - 8) s as fp16 tiles of keys and values, times a power of two per page (keys) or per unit so far (values): exact, since a number has 3 + 8
//                    significant bits, down to 2^-8 of the largest scale, and to 2^-19 of it below
//   2 MMA warps      S = Q K^T (128 x 64 per tile), O += P V, P from tensor memory
//   softmax warps    8 per tile, two threads per column: S from tensor memory, running maximum and sum, P back as fp16; O is scaled in place where the maximum moves by more than 2^8
//
// fp32 rows: q and P as two fp16 terms each, their products into the same accumulators (2^-22).  Products and exponentials need about the same time (16 exponentials per SM and clock,
// 4096 multiply-adds): 1024 clocks each per page and two tiles at heads of 128.  Measured: 2500 clocks per page at heads of 64 and 2750 at 128, with instructions issued in 56 % of cycles,
// exponentials in 30 %, tensor cores busy in 25 %: no unit is the bound, the chain of a page is (scores, maximum over two warps, exponentials, weights to tensor memory, products).  Without
// the maximum it would be 19 % less, without exponentials 15 %, without the work on codes 7 %, without scores 3 %; the maximum of both halves by each of two threads was slower (288 us for 257).
// 8 prompts of 2048, 16 / 4 bf16 heads of 64: 255 us, 269 TFLOP/s of the products that count; heads of 128 336 us, 409; 2 x 512 rows behind 16000 tokens, 32 / 8 heads of 128: 378 us, 720.
#include "device_args.h"
#include "kv4.cuh"
#include "rows.cuh"

#include <algorithm>

namespace lumi {
namespace {

constexpr int kTile = 128;
constexpr int kPromptCtas = 160;                           // places for parts
constexpr int kTicketsAt = 320;                            // behind the step kernel's
constexpr int kUnitPages = 3;                              // what a unit costs beside its pages: queries, pipeline, results.  On the line it begins with as many places without a page
constexpr int kRunPages = 4;                               // a CTA's places, at least: a unit's beginning and a page (64 rows behind 400 tokens, eight heads of 128: 46 us; 8 places 58)
constexpr int kMaxRing = 4;
constexpr int kStatic = 10 * 1024;                         // bytes declared in the kernel, at most
constexpr int kInfos = 8;                                  // pages whose exponents are kept: the copies run up to kMaxRing ahead of the values' tiles, these two ahead of the softmax

template <int NG, bool TWO>
struct PromptShape {
    static constexpr int kTiles = NG <= 4 ? 2 : 1;
    static constexpr int kCols = kTile * kTiles;
    static constexpr int kTerms = TWO ? 2 : 1;
    static constexpr int kBlocks = NG / 2;                 // of 64 numbers: one 128-byte row each
    static constexpr int kBufs = NG == 8 && TWO ? 1 : 2;   // tiles of keys and of values
    static constexpr int kQ = kTiles * kTerms * kBlocks * kTile * 128, kKv = kBlocks * kPage * 128;
    static constexpr int kFixed = kQ + 2 * kBufs * kKv;
    static constexpr int kThreads = (kTiles * 8 + 4 + kTiles + 2) * 32;
    // tensor memory: O of each tile, S, P
    static constexpr int kO = NG * kGroup, kS = kTiles * kO, kP = kS + kTiles * kPage, kPCols = TWO ? 64 : 32;
};

__device__ __forceinline__ void tmem_ld32f(uint32_t taddr, float (&r)[32]) { tmem_ld32(taddr, reinterpret_cast<uint32_t(&)[32]>(r)); }
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// A from tensor memory
__device__ __forceinline__ void umma_tmem_a(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Values: 64 numbers of a token are a 128-byte row (the operand's N), tokens go along K: groups of eight 1024 bytes apart, blocks of 64 numbers kPage * 128.
__device__ __forceinline__ uint64_t values_desc(uint32_t addr) {
    uint64_t d = make_smem_desc(addr) & ~((uint64_t)0x3fff << 16);
    return d | (uint64_t)((kPage * 128) >> 4) << 16;
}
__device__ __forceinline__ void pair_barrier(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void tile_barrier(int id) { asm volatile("bar.sync %0, 256;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_any(int id, bool v) {      // of two warps
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"(id), "r"((uint32_t)v) : "memory");
    return any != 0;
}

// A wait that asks seldom: the hardware wakes the warp, and idle roles leave the issue slots to the others.
__device__ __noinline__ void patient_wait(uint64_t* bar, uint32_t parity, uint64_t limit_ns, volatile int* dead) {
    const uint64_t t0 = globaltimer_ns();
    while (!*dead) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(20000u) : "memory");
        if (ok) return;
        if (globaltimer_ns() - t0 > limit_ns) { *dead = 1; return; }
    }
}

// Eight numbers of a row that has n of them, as memory holds them; and as fp32.
__device__ __forceinline__ void eight_raw(const float* p, int n, bool wide, uint4 (&w)[2]) {
    w[0] = w[1] = make_uint4(0, 0, 0, 0);
    if (wide) {
        if (n > 0) { w[0] = reinterpret_cast<const uint4*>(p)[0]; w[1] = reinterpret_cast<const uint4*>(p)[1]; }
    } else {
        uint32_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = e < n ? __float_as_uint(p[e]) : 0u;
        w[0] = make_uint4(u[0], u[1], u[2], u[3]);
        w[1] = make_uint4(u[4], u[5], u[6], u[7]);
    }
}
__device__ __forceinline__ void eight_raw(const __nv_bfloat16* p, int n, bool wide, uint4 (&w)[1]) {
    w[0] = make_uint4(0, 0, 0, 0);
    if (wide) {
        if (n > 0) w[0] = *reinterpret_cast<const uint4*>(p);
    } else {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            u[e] = (2 * e < n ? (uint32_t)__bfloat16_as_ushort(p[2 * e]) : 0u) | (2 * e + 1 < n ? (uint32_t)__bfloat16_as_ushort(p[2 * e + 1]) << 16 : 0u);
        w[0] = make_uint4(u[0], u[1], u[2], u[3]);
    }
}
__device__ __forceinline__ void eight_of(const uint4 (&w)[2], float (&t)[8]) {
    t[0] = __uint_as_float(w[0].x); t[1] = __uint_as_float(w[0].y); t[2] = __uint_as_float(w[0].z); t[3] = __uint_as_float(w[0].w);
    t[4] = __uint_as_float(w[1].x); t[5] = __uint_as_float(w[1].y); t[6] = __uint_as_float(w[1].z); t[7] = __uint_as_float(w[1].w);
}
__device__ __forceinline__ void eight_of(const uint4 (&w)[1], float (&t)[8]) {
    const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { t[2 * i] = low_bf16(u[i]); t[2 * i + 1] = high_bf16(u[i]); }
}
// 16 bytes of a row of y that has n numbers from here on.
__device__ __forceinline__ void put_16(float* y, int n, bool wide, uint4 u) {
    if (wide) { if (n > 0) *reinterpret_cast<uint4*>(y) = u; return; }
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) if (i < n) y[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void put_16(__nv_bfloat16* y, int n, bool wide, uint4 u) {
    if (wide) { if (n > 0) *reinterpret_cast<uint4*>(y) = u; return; }
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < n) y[i] = __ushort_as_bfloat16((unsigned short)(w[i / 2] >> (i % 2 * 16)));
}

struct PageInfo { int e_k, e_v, absent; uint32_t no_number[2]; };      // exponents of keys and values; tokens with values that are no numbers

struct Cursor { int s, head, tile, skip; };                // a unit, and pages of it that are the CTA's ahead

template <typename T, int NG>
__global__ void __launch_bounds__(PromptShape<NG, sizeof(T) == 4>::kThreads, 1) kv4_prompt_kernel(const AttendArgs a, const int ring_n) {
    constexpr bool TWO = sizeof(T) == 4;
    using Shape = PromptShape<NG, TWO>;
    constexpr int TILES = Shape::kTiles, COLS = Shape::kCols, TERMS = Shape::kTerms, BLOCKS = Shape::kBlocks, BUFS = Shape::kBufs, THREADS = Shape::kThreads;
    extern __shared__ __align__(1024) uint8_t sm_raw[];
    uint8_t* const sm = sm_raw + ((1024 - (smem_u32(sm_raw) & 1023)) & 1023);
    uint8_t *const q_sm = sm, *const k_sm = q_sm + Shape::kQ, *const v_sm = k_sm + BUFS * Shape::kKv, *const ring = v_sm + BUFS * Shape::kKv;
    __shared__ uint64_t raw_full[kMaxRing], raw_empty[kMaxRing], k_full[2], k_empty[2], v_full[2], v_empty[2], q_full[2], s_full[2], s_empty[2], p_full[2], o_done[2], info_full[kInfos], all_done;
    __shared__ PageInfo info[kInfos];
    __shared__ int absent_s[kMaxRing];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_flag, last_s[2];
    __shared__ long long warp_pages[THREADS / 32];
    __shared__ Cursor start_s;
    __shared__ float tops_s[2][TILES][kTile], factors_s[TILES][kTile];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int* const dead_s = &dead_flag;
    const int gk = kv4_groups(a.dk), gv = kv4_groups(a.dv), part = kv4_part(a.dk), block = kv4_block(a.dk, a.dv), pad = gv * kGroup;

    if (tid == 0) {
        for (int i = 0; i < kMaxRing; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 5); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 4); mbar_init(&k_empty[i], TILES); mbar_init(&v_full[i], 4); mbar_init(&v_empty[i], TILES);
            mbar_init(&q_full[i], 8); mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 8); mbar_init(&p_full[i], 8); mbar_init(&o_done[i], 1);
        }
        for (int i = 0; i < kInfos; ++i) mbar_init(&info_full[i], 1);
        mbar_init(&all_done, TILES);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        dead_flag = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_release();
    pdl_sync();
    const uint32_t tmem = tmem_slot;

    // ---- the line of pages
    auto unit_pages = [&](const Sequence& q, int tile, int& lo, int& hi) {
        const int cols = q.n * a.group, row0 = tile * COLS / a.group, row1 = (min((tile + 1) * COLS, cols) - 1) / a.group;
        lo = a.window > 0 ? max(0, q.total - q.n + row0 - a.window + 1) / kPage : 0;
        hi = (q.total - q.n + row1) / kPage + 1;
    };
    auto tiles_of = [&](const Sequence& q) { return (q.n * a.group + COLS - 1) / COLS; };
    auto pages_of = [&](const Sequence& q, int tile) {
        int lo, hi;
        unit_pages(q, tile, lo, hi);
        return hi - lo + kUnitPages;
    };
    auto has_work = [&](int s, Sequence& q) { return lengths_of(a, s, q) && q.n > 0 && q.n <= a.max_new && (long)q.n * a.group > a.few; };
    auto warp_sum = [&](long long v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    // Places of one head of each lane's sequence (s < 0: none), 0 where there is nothing of this kernel's.  Sequences of many tiles are summed up by the whole warp.
    auto head_pages = [&](int s) {
        Sequence q;
        long long sum = 0;
        const bool work = s >= 0 && has_work(s, q);
        const int tiles = work ? tiles_of(q) : 0;
        for (int t = 0; t < tiles && tiles <= 8; ++t) sum += pages_of(q, t);
        for (uint32_t many = __ballot_sync(0xffffffffu, tiles > 8); many != 0; many &= many - 1) {
            const int lane_of = __ffs(many) - 1;
            Sequence w;
            lengths_of(a, __shfl_sync(0xffffffffu, s, lane_of), w);
            long long part_sum = 0;
            for (int t = lane, n = tiles_of(w); t < n; t += 32) part_sum += pages_of(w, t);
            part_sum = warp_sum(part_sum);
            if (lane == lane_of) sum = part_sum;
        }
        return sum;
    };
    const int each = (a.nseq + THREADS - 1) / THREADS, s_lo = tid * each;
    long long mine = 0;
    for (int k = 0; k < each; ++k) mine += head_pages(s_lo + k < a.nseq ? s_lo + k : -1) * a.kv_heads;
    long long run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += t; }
    if (lane == 31) warp_pages[warp] = run;
    __syncthreads();
    long long ahead = 0, total = 0;
    for (int w = 0; w < THREADS / 32; ++w) { const long long p = warp_pages[w]; if (w < warp) ahead += p; total += p; }
    const long long begins = ahead + run - mine;
    const int ctas = (int)min((long long)gridDim.x, quotient(total + kRunPages - 1, kRunPages)), cta = blockIdx.x;
    const bool works = cta < ctas;
    const long long c_lo = works ? quotient(total * cta, ctas) : 0, c_hi = works ? quotient(total * (cta + 1), ctas) : 0;
    // the warp whose sequences hold the CTA's first page looks for its place
    const uint32_t holds = __ballot_sync(0xffffffffu, works && mine > 0 && begins <= c_lo && c_lo < begins + mine);
    if (holds != 0) {
        const int lane_of = __ffs(holds) - 1;
        long long at = __shfl_sync(0xffffffffu, begins, lane_of);
        Cursor c{__shfl_sync(0xffffffffu, s_lo, lane_of), 0, 0, 0};
        for (int k = 0; k < each; ++k, ++c.s) {
            long long per = head_pages(lane == 0 && c.s < a.nseq ? c.s : -1);
            per = __shfl_sync(0xffffffffu, per, 0);
            if (c_lo >= at + per * a.kv_heads) { at += per * a.kv_heads; continue; }
            c.head = (int)quotient(c_lo - at, per);
            long long rel = c_lo - at - c.head * per;
            Sequence q;
            lengths_of(a, c.s, q);
            for (int t0 = 0, n = tiles_of(q); t0 < n; t0 += 32) {       // 32 tiles at a time
                const int here = t0 + lane < n ? pages_of(q, t0 + lane) : 0;
                long long upto = here;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += t; }
                const uint32_t in = __ballot_sync(0xffffffffu, rel < upto);
                if (in != 0) {
                    const int x = __ffs(in) - 1;
                    c.tile = t0 + x;
                    c.skip = (int)(rel - (__shfl_sync(0xffffffffu, upto, x) - __shfl_sync(0xffffffffu, here, x)));
                    break;
                }
                rel -= __shfl_sync(0xffffffffu, upto, 31);
            }
            break;
        }
        if (lane == 0) start_s = c;
    }
    __syncthreads();

    // ---- what all roles walk over: the CTA's share of one unit after another
    struct Segment { Sequence q; int s, head, tile, cols, lo, hi, p0, p1; };      // pages lo .. hi of the unit, p0 .. p1 of them here
    auto walk = [&](auto&& body) {
        if (!works) return;
        Cursor c = start_s;
        long long left = c_hi - c_lo, at = c_lo;
        while (left > 0) {
            Segment g;
            lengths_of(a, c.s, g.q);
            g.s = c.s; g.head = c.head; g.tile = c.tile;
            g.cols = g.q.n * a.group;
            unit_pages(g.q, c.tile, g.lo, g.hi);
            const int take = (int)min(left, (long long)(g.hi - g.lo + kUnitPages - c.skip));
            g.p0 = g.lo + max(0, c.skip - kUnitPages);
            g.p1 = g.lo + max(0, c.skip + take - kUnitPages);
            if (g.p1 > g.p0) body(g, at - c.skip + kUnitPages);
            left -= take;
            at += take;
            if (left <= 0) break;
            c.skip = 0;
            if (++c.tile * COLS >= g.cols) {
                c.tile = 0;
                if (++c.head == a.kv_heads) {
                    c.head = 0;
                    Sequence q;
                    do ++c.s; while (c.s + 1 < a.nseq && !has_work(c.s, q));      // (there is one more: pages are left)
                }
            }
        }
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!mbar_try_wait(bar, parity & 1)) patient_wait(bar, parity & 1, a.wait_ns, dead_s);
        __syncwarp();
    };
    auto arrive = [&](uint64_t* bar) {                     // one of four warps, all of its lanes
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    int copied = 0;                                        // (copy warp) copies issued

    if (warp < TILES * 8) {
        // ---- softmax: two threads per column, each 32 of a page's 64 tokens and half of the column's numbers
        const int tile = warp / 8, half = warp / 4 % 2, r = tid % kTile, pair = 1 + tile * 4 + warp % 4;
        const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
        const uint32_t t_o = tmem + tile * Shape::kO + lanes, t_s = tmem + Shape::kS + tile * kPage + half * 32 + lanes, t_p = tmem + Shape::kP + tile * Shape::kPCols + half * 16 + lanes;
        const int d_lo = half == 0 ? 0 : (gv + 1) / 2 * kGroup, d_hi = half == 0 ? (gv + 1) / 2 * kGroup : pad;      // numbers of values
        uint32_t pages = 0, done = 0;                      // of the CTA, of this tile
        walk([&](const Segment& g, long long unit_lo) {
            const int col0 = g.tile * COLS + tile * kTile, n_pages = g.p1 - g.p0;
            if (col0 >= g.cols) { pages += n_pages; return; }
            const int col = min(col0 + r, g.cols - 1), row = col / a.group, h = col - row * a.group;
            const bool valid = col0 + r < g.cols;
            const int pos = g.q.total - g.q.n + row, lo_pos = a.window > 0 ? max(0, pos - a.window + 1) : 0;
            const long out_row = g.q.first + row;
            const int out_head = g.head * a.group + h;
            // q, times a power of two that brings the column's largest to 2^13 .. 2^14: each warp 16 columns of the tile, eight numbers per lane
            {
                constexpr int PER = NG * 4, AT_ONCE = TWO ? 4 : NG * 2 < 8 ? NG * 2 : 8;      // lanes per column; loads under way
                const int c_lane = lane / PER, d = lane % PER * 8, c0 = warp % 8 * 16;
#pragma unroll 1
                for (int i0 = 0; i0 < PER / 2; i0 += AT_ONCE) {
                    uint4 raw[AT_ONCE][sizeof(T) / 2];
#pragma unroll
                    for (int i = 0; i < AT_ONCE; ++i) {
                        const int c = col0 + c0 + (i0 + i) * (32 / PER) + c_lane, c_row = min(c, g.cols - 1) / a.group, c_head = min(c, g.cols - 1) - c_row * a.group;
                        const T* const p = (const T*)a.q + (long)(g.q.first + c_row) * a.ldq + (long)(g.head * a.group + c_head) * a.dk + d;
                        eight_raw(p, c < g.cols ? a.dk - d : 0, a.wide_q, raw[i]);
                    }
#pragma unroll
                    for (int i = 0; i < AT_ONCE; ++i) {
                        const int c = c0 + (i0 + i) * (32 / PER) + c_lane;
                        float t[8];
                        eight_of(raw[i], t);
                        uint32_t top = 0;
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(t[e]) & 0x7fffffffu);
#pragma unroll
                        for (int o = 1; o < PER; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const float by = power_of_two(top >= 0x7f800000u || top == 0 ? 0 : min(126, 13 + 127 - (int)(top >> 23)));
                        if (lane % PER == 0) factors_s[tile][c] = fminf(fmaxf(__fdiv_rn(fabsf(a.scale) * kLog2e, by), 1e-37f), 3.4e38f);
                        const float f = a.scale < 0.f ? -by : by;
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = t[2 * e] * f, y = t[2 * e + 1] * f;
                            hi[e] = halves(x, y);
                            if (TWO) { const float2 b = unhalves(hi[e]); lo[e] = halves(x - b.x, y - b.y); }
                        }
                        uint8_t* const to = q_sm + ((tile * TERMS) * BLOCKS + d / 64) * (kTile * 128) + c * 128 + ((d / 8 % 8) ^ (c & 7)) * 16;
                        *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        if (TWO) *reinterpret_cast<uint4*>(to + BLOCKS * (kTile * 128)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(&q_full[tile]);
                tile_barrier(9 + tile);
            }
            const float cx = factors_s[tile][r];
            const int first_full = __reduce_max_sync(0xffffffffu, lo_pos), last_full = __reduce_min_sync(0xffffffffu, pos);      // positions that all of the warp's columns see
            float m = -INFINITY, l = 0.f;                  // (l: of this thread's tokens)
            int e_v = 0;
            for (int i = 0; i < n_pages; ++i, ++pages, ++done) {
                wait(&s_full[tile], done);
                wait(&info_full[pages % kInfos], pages / kInfos);
                const PageInfo& of = info[pages % kInfos];
                tc_fence_after();
                float s[32];
                tmem_ld32f(t_s, s);
                tc_fence_before();
                arrive(&s_empty[tile]);
                const int up = of.e_k + 9;
                const float c = fmaxf(cx * power_of_two(up / 2) * power_of_two(up - up / 2), 1e-37f);
                const int pos0 = (g.p0 + i) * kPage + half * 32, new_e = of.e_v;
                if (pos0 < first_full || pos0 + 31 > last_full || of.absent) {
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (pos0 + k < lo_pos || pos0 + k > pos || of.absent) s[k] = -INFINITY;
                }
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int k = 4; k < 32; ++k) top[k % 4] = fmaxf(top[k % 4], s[k]);
                float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
                const bool moves = t > m + 8.f || (m == -INFINITY && t > -INFINITY);
                bool waited = i == 0;
                if (pair_any(pair, moves || (i > 0 && new_e != e_v))) {      // of both halves of 32 columns
                    tops_s[half][tile][r] = t;
                    pair_barrier(pair);
                    t = fmaxf(t, tops_s[1 - half][tile][r]);
                    const bool both = t > m + 8.f || (m == -INFINITY && t > -INFINITY);
                    const float to = both ? t : m;
                    const float f = m == -INFINITY ? 0.f : exp2_fast(m - to);
                    const float fo = m == -INFINITY ? 0.f : exp2_fast(0.5f * (m - to + (float)(e_v - new_e)));
                    m = to;
                    l *= f;
                    if (i > 0) {
                        wait(&o_done[tile], done - 1);
                        waited = true;
                        tc_fence_after();
#pragma unroll 1
                        for (int d = d_lo; d < d_hi; d += 16) {
                            uint32_t o[16];
                            tmem_ld16(t_o + d, o);
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fo * fo);
                            tmem_st16(t_o + d, o);
                        }
                        tmem_st_wait();
                        tc_fence_before();
                    }
                    pair_barrier(pair);                    // tops_s has been read
                }
                e_v = new_e;
                const float off = m == -INFINITY ? 0.f : -m;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};       // (two chains of pairs)
                uint32_t p[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    float &x = s[2 * k], &y = s[2 * k + 1];
                    fma2(x, y, x, y, c, c, off, off);
                    x = exp2_fast(x);
                    y = exp2_fast(y);
                    add2(sum[k % 2 * 2], sum[k % 2 * 2 + 1], x, y);
                    p[k] = halves(x, y);
                    if (TWO) { const float2 b = unhalves(p[k]); x -= b.x; y -= b.y; }
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (!waited) wait(&o_done[tile], done - 1);
                tmem_st16(t_p, p);
                if constexpr (TWO) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) p[k] = halves(s[2 * k], s[2 * k + 1]);
                    tmem_st16(t_p + 32, p);
                }
                if (of.no_number[half])                    // (rare) a row that sees such a token is none
                    for (int k = 0; k < 32; ++k)
                        if ((of.no_number[half] >> k & 1) && pos0 + k >= lo_pos && pos0 + k <= pos) l = __uint_as_float(0x7fc00000u);
                tmem_st_wait();
                tc_fence_before();
                arrive(&p_full[tile]);
            }
            tops_s[half][tile][r] = l;
            pair_barrier(pair);
            l += tops_s[1 - half][tile][r];
            pair_barrier(pair);
            wait(&o_done[tile], done - 1);
            tc_fence_after();
            const int e = e_v + 9;                         // numbers are O 2^e / l
            const float back = power_of_two(e / 2), back2 = power_of_two(e - e / 2);
            auto inverse = [&](float mm, float ll) {
                if (a.sink && mm != -INFINITY) ll += exp2_fast(-mm);
                return *dead_s ? __uint_as_float(0x7fc00000u) : mm == -INFINITY && ll == 0.f ? 0.f : __fdiv_rn(1.f, ll);
            };
            const bool whole = g.p0 == g.lo && g.p1 == g.hi;
            const int places = COLS, at = tile * kTile + r;
            const int rec = places * (2 + pad);
            float* const to = a.parts + ((size_t)cta * 2 + (g.p0 == g.lo ? 1 : 0)) * rec;
            const float inv = whole ? inverse(m, l) : 1.f;
            // Rows of y by way of the queries' places that this warp alone fills (their products are done): 32 columns, CHUNKS x 16 bytes each
            constexpr int CHUNKS = NG / 2 * kGroup * (int)sizeof(T) / 16, PIECE = 16 * 128, E = 16 / (int)sizeof(T);
            auto stage = [&](int c, int chunk) {
                const int x = (c * CHUNKS + (CHUNKS >= 8 ? chunk ^ (c & 7) : chunk ^ (c >> 1 & 3))) * 16;
                return q_sm + (tile * TERMS * BLOCKS + x / PIECE) * (kTile * 128) + warp % 8 * PIECE + x % PIECE;
            };
#pragma unroll 1
            for (int d = d_lo; d < d_hi; d += 16) {
                uint32_t o[16];
                tmem_ld16(t_o + d, o);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(o[8 * k + j]) * back * back2;
                    if (whole) {                           // (numbers of a tile lie as 0 4 1 5 2 6 3 7)
                        const int chunk = (d - d_lo + 8 * k) / E;
                        if constexpr (TWO) {
                            *reinterpret_cast<float4*>(stage(lane, chunk)) = make_float4(v[0] * inv, v[2] * inv, v[4] * inv, v[6] * inv);
                            *reinterpret_cast<float4*>(stage(lane, chunk + 1)) = make_float4(v[1] * inv, v[3] * inv, v[5] * inv, v[7] * inv);
                        } else {
                            const __nv_bfloat162 x0 = __floats2bfloat162_rn(v[0] * inv, v[2] * inv), x1 = __floats2bfloat162_rn(v[4] * inv, v[6] * inv);
                            const __nv_bfloat162 x2 = __floats2bfloat162_rn(v[1] * inv, v[3] * inv), x3 = __floats2bfloat162_rn(v[5] * inv, v[7] * inv);
                            *reinterpret_cast<uint4*>(stage(lane, chunk)) = make_uint4(*reinterpret_cast<const uint32_t*>(&x0), *reinterpret_cast<const uint32_t*>(&x1),
                                                                                      *reinterpret_cast<const uint32_t*>(&x2), *reinterpret_cast<const uint32_t*>(&x3));
                        }
                    } else {
                        *reinterpret_cast<float4*>(to + 2 * places + ((d / 4 + 2 * k) * places + at) * 4) = make_float4(v[0], v[1], v[2], v[3]);
                        *reinterpret_cast<float4*>(to + 2 * places + ((d / 4 + 2 * k + 1) * places + at) * 4) = make_float4(v[4], v[5], v[6], v[7]);
                    }
                }
            }
            if (whole) {
                __syncwarp();
                const unsigned long long mine_at = (unsigned long long)((T*)a.y + out_row * a.ldy + (long)out_head * a.dv) | (valid ? 0 : 1ull << 63);
#pragma unroll 4
                for (int i = 0; i < CHUNKS; ++i) {
                    const int c = (i * 32 + lane) / CHUNKS, chunk = (i * 32 + lane) % CHUNKS, d = d_lo + chunk * E;
                    const unsigned long long y = __shfl_sync(0xffffffffu, mine_at, c);
                    const uint4 u = *reinterpret_cast<const uint4*>(stage(c, chunk));
                    if (y >> 63 == 0 && d < d_hi) put_16((T*)y + d, a.dv - d, a.wide_y16, u);
                }
            }
            tc_fence_before();
            if (whole) return;
            // ---- the unit is shared: who arrives last joins the parts, in the order of CTAs
            if (half == 0) {
                to[at] = m;
                to[places + at] = *dead_s ? __uint_as_float(0x7fc00000u) : l;
            }
            __threadfence();
            tile_barrier(9 + tile);
            const long long unit_hi = unit_lo + (g.hi - g.lo);
            const int c0 = (int)quotient((unit_lo + 1) * ctas - 1, total), c1 = (int)quotient(unit_hi * ctas - 1, total);
            if (r == 0 && half == 0) {
                int32_t* const ticket = a.tickets + kTicketsAt + c0 * 2 + tile;
                last_s[tile] = atomicAdd(ticket, 1) == c1 - c0;
                if (last_s[tile]) *ticket = 0;
            }
            tile_barrier(9 + tile);
            if (!last_s[tile]) return;
            __threadfence();
            auto place_of = [&](int k) { return a.parts + ((size_t)k * 2 + (k == c0 ? 1 : 0)) * rec; };
            // a thread per column, eight numbers at a time, or several where the tile has few columns
            const int here = min(kTile, g.cols - col0), ways = 2 * kTile / here, x = half * kTile + r, way = x / here, c = x - way * here, from = tile * kTile + c;
            if (way >= ways) return;
            float mm = -INFINITY, ll = 0.f;
#pragma unroll 8
            for (int k = c0; k <= c1; ++k) mm = fmaxf(mm, __ldcg(place_of(k) + from));
#pragma unroll 4
            for (int k = c0; k <= c1; ++k) {
                const float pm = __ldcg(place_of(k) + from), pl = __ldcg(place_of(k) + places + from);
                ll += pl == pl ? pl * (pm == -INFINITY ? 0.f : exp2_fast(pm - mm)) : pl;
            }
            const float f = inverse(mm, ll);
            const int c_row = (col0 + c) / a.group, c_head = col0 + c - c_row * a.group;
            T* const y = (T*)a.y + (long)(g.q.first + c_row) * a.ldy + (long)(g.head * a.group + c_head) * a.dv;
            for (int d = way * 8; d < pad; d += ways * 8) {
                float o[8] = {};
#pragma unroll 4
                for (int k = c0; k <= c1; ++k) {
                    const float* const p = place_of(k);
                    const float pm = __ldcg(p + from), w = pm == -INFINITY ? 0.f : exp2_fast(pm - mm);
                    const float4 u = __ldcg(reinterpret_cast<const float4*>(p + 2 * places + (d / 4 * places + from) * 4)), v = __ldcg(reinterpret_cast<const float4*>(p + 2 * places + ((d / 4 + 1) * places + from) * 4));
                    o[0] = fmaf(u.x, w, o[0]); o[1] = fmaf(u.y, w, o[1]); o[2] = fmaf(u.z, w, o[2]); o[3] = fmaf(u.w, w, o[3]);
                    o[4] = fmaf(v.x, w, o[4]); o[5] = fmaf(v.y, w, o[5]); o[6] = fmaf(v.z, w, o[6]); o[7] = fmaf(v.w, w, o[7]);
                }
                const float lo[4] = {o[0] * f, o[2] * f, o[4] * f, o[6] * f}, hi[4] = {o[1] * f, o[3] * f, o[5] * f, o[7] * f};      // as they lie in the tile
                put_four(y + d, a.dv - d, a.wide_y, lo);
                put_four(y + d + 4, a.dv - d - 4, a.wide_y, hi);
            }
        });
    } else if (warp < TILES * 8 + 4) {
        // ---- codes and scales to fp16 tiles
        const int dt = tid - TILES * 2 * kTile;
        uint32_t pages = 0;
        walk([&](const Segment& g, long long) {
            for (int p = g.p0; p < g.p1; ++p, ++pages) {
                const int slot = pages % ring_n, live = min(kPage, g.q.total - p * kPage);      // tokens that have been written
                const uint8_t* const raw = ring + slot * block;
                wait(&raw_full[slot], pages / ring_n);
                wait(&info_full[pages % kInfos], pages / kInfos);
                const PageInfo& of = info[pages % kInfos];
                const int e_k = of.e_k, e_v = of.e_v;
                const bool absent = of.absent != 0;
                const int buf = pages % BUFS;
                auto tile_of = [&](bool keys) {
                    const int groups = keys ? gk : gv;
                    const uint8_t* const codes = raw + (keys ? 0 : part);
                    uint8_t* const out = (keys ? k_sm : v_sm) + buf * Shape::kKv;
                    const float by = power_of_two(15 - (keys ? e_k : e_v));
                    uint4 u[NG / 2];                       // a token's group each
                    float sc[NG / 2];
#pragma unroll
                    for (int i = 0; i < NG / 2; ++i) {
                        const int x = i * 128 + dt, tok = x % kPage, grp = x / kPage;
                        u[i] = make_uint4(0, 0, 0, 0);
                        sc[i] = 0.f;
                        if (grp < groups && !absent && tok < live) {
                            u[i] = *reinterpret_cast<const uint4*>(codes + grp * kPlane + tok * 16);
                            const uint32_t bits = *reinterpret_cast<const uint16_t*>(codes + groups * kPlane + grp * kScales + tok * 2);
                            sc[i] = !keys && (bits & 0x7fffu) >= 0x7f80u ? 0.f : __uint_as_float(bits << 16);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < NG / 2; ++i) {
                        const int x = i * 128 + dt, tok = x % kPage, grp = x / kPage;
                        const float s = sc[i] * by;
                        const __half2 t = __float2half2_rn(s), t16 = __float2half2_rn(s * 0.0625f), t8 = __float2half2_rn(s * -4.76837158203125e-07f);      // -8 2^-24
                        uint8_t* const row = out + grp / 2 * (kPage * 128) + tok * 128;
                        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t c[4] = {w[j] & 0x000f000fu, w[j] & 0x00f000f0u, w[j] >> 8 & 0x000f000fu, w[j] >> 8 & 0x00f000f0u};
                            uint32_t o[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&c[k]), k % 2 ? t16 : t, t8);
                                o[k] = *reinterpret_cast<const uint32_t*>(&v);
                            }
                            if (grp < groups) *reinterpret_cast<uint4*>(row + ((grp % 2 * 4 + j) ^ (tok & 7)) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                };
                wait(&k_empty[buf], pages / BUFS + 1);
                tile_of(true);
                arrive(&k_full[buf]);
                wait(&v_empty[buf], pages / BUFS + 1);
                tile_of(false);
                arrive(&v_full[buf]);
                arrive(&raw_empty[slot]);
            }
        });
    } else if (warp < TILES * 9 + 4) {
        // ---- products: a warp per tile, so that neither waits for the other one's softmax
        const int t = warp - TILES * 8 - 4;
        const uint32_t id_s = (1u << 4) | ((uint32_t)(kPage >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
        const uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(pad >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);      // B: numbers contiguous
        // descriptors count in 16 bytes: a step of 16 numbers or tokens is an addition
        const uint64_t q_desc = make_smem_desc(smem_u32(q_sm) + t * TERMS * BLOCKS * (kTile * 128)), k_desc = make_smem_desc(smem_u32(k_sm)), v_desc = values_desc(smem_u32(v_sm));
        uint32_t pages = 0, done = 0, outs = 0, units = 0;
        walk([&](const Segment& g, long long) {
            if (g.tile * COLS + t * kTile >= g.cols) {     // not a column of this tile: the buffers are free of it
                for (int p = g.p0; p < g.p1; ++p, ++pages) {
                    wait(&k_full[pages % BUFS], pages / BUFS);
                    if (lane == 0) mbar_arrive(&k_empty[pages % BUFS]);
                    wait(&v_full[pages % BUFS], pages / BUFS);
                    if (lane == 0) mbar_arrive(&v_empty[pages % BUFS]);
                }
                return;
            }
            auto values = [&](uint32_t page, bool first) {
                const int buf = page % BUFS;
                wait(&v_full[buf], page / BUFS);
                wait(&p_full[t], outs);
                ++outs;
                tc_fence_after();
                if (lane == 0) {
                    const uint64_t v = v_desc + buf * (Shape::kKv >> 4);
#pragma unroll
                    for (int term = 0; term < TERMS; ++term)
#pragma unroll
                        for (int k = 0; k < kPage / 16; ++k)
                            umma_tmem_a(tmem + t * Shape::kO, tmem + Shape::kP + t * Shape::kPCols + term * 32 + k * 8, v + k * (2048 >> 4), id_o, !(first && term == 0 && k == 0));
                    umma_commit(&o_done[t]);
                    umma_commit(&v_empty[buf]);
                }
                __syncwarp();
            };
            wait(&q_full[t], units);
            ++units;
            for (int p = g.p0; p < g.p1; ++p, ++pages) {
                const int buf = pages % BUFS;
                wait(&k_full[buf], pages / BUFS);
                wait(&s_empty[t], done + 1);
                tc_fence_after();
                if (lane == 0) {
                    const uint64_t k = k_desc + buf * (Shape::kKv >> 4);
#pragma unroll 1
                    for (int term = TERMS - 1; term >= 0; --term)      // (second terms first: sums are cut off, not rounded, and less so while they are small)
#pragma unroll 1
                        for (int x = 0; x < 2 * gk; x += 2) {      // a group of 32 numbers
                            const uint64_t qd = q_desc + (((term * BLOCKS + x / 4) * (kTile * 128) + x % 4 * 32) >> 4), kd = k + ((x / 4 * (kPage * 128) + x % 4 * 32) >> 4);
                            umma_bf16(tmem + Shape::kS + t * kPage, qd, kd, id_s, term < TERMS - 1 || x > 0);
                            umma_bf16(tmem + Shape::kS + t * kPage, qd + 2, kd + 2, id_s, 1u);
                        }
                    umma_commit(&s_full[t]);
                    umma_commit(&k_empty[buf]);
                }
                __syncwarp();
                if (p > g.p0) values(pages - 1, p - 1 == g.p0);
                ++done;
            }
            values(pages - 1, g.p1 - 1 == g.p0);
        });
        if (lane == 0) umma_commit(&all_done);
        __syncwarp();
    } else if (warp == TILES * 9 + 4) {
        // ---- the largest scales of a page, a power of two each: keys' of the page, values' of the unit so far
        uint32_t pages = 0;
        walk([&](const Segment& g, long long) {
            int e_run = -90;
            for (int p = g.p0; p < g.p1; ++p, ++pages) {
                const int slot = pages % ring_n, live = min(kPage, g.q.total - p * kPage);      // tokens that have been written
                const uint8_t* const raw = ring + slot * block;
                wait(&raw_full[slot], pages / ring_n);
                const bool absent = absent_s[slot] != 0;
                uint32_t top[2] = {0, 0}, none[2] = {0, 0};
                if (!absent)
#pragma unroll
                    for (int i = 0; i < NG / 2; ++i) {     // eight tokens' scales of a group
                        const int x = i * 32 + lane, values = x >= gk * 8, tok = x % 8 * 8;
                        if (x >= (gk + gv) * 8) break;
                        const uint4 u = *reinterpret_cast<const uint4*>(raw + (values ? part + gv * kPlane + (x - gk * 8) * 16 : gk * kPlane + x * 16));
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            uint32_t b = (w[k / 2] >> (k % 2 * 16)) & 0x7fffu;
                            if (tok + k >= live) b = 0;
                            if (b >= 0x7f80u) { if (values) none[tok / 32] |= 1u << ((tok + k) % 32); b = 0; }
                            top[values] = max(top[values], b);
                        }
                    }
                top[0] = __reduce_max_sync(0xffffffffu, top[0]);
                top[1] = __reduce_max_sync(0xffffffffu, top[1]);
                none[0] = __reduce_or_sync(0xffffffffu, none[0]);
                none[1] = __reduce_or_sync(0xffffffffu, none[1]);
                // scales are below 2^e; they become fp16 numbers below 2^15
                e_run = max(e_run, max(-90, min(127, (int)(top[1] >> 7) - 126)));
                if (lane == 0) {
                    PageInfo& to = info[pages % kInfos];
                    to.e_k = max(-90, min(127, (int)(top[0] >> 7) - 126));
                    to.e_v = e_run;
                    to.absent = absent;
                    to.no_number[0] = none[0]; to.no_number[1] = none[1];
                    mbar_arrive(&info_full[pages % kInfos]);
                    mbar_arrive(&raw_empty[slot]);
                }
                __syncwarp();
            }
        });
    } else {
        // ---- copies
        uint32_t pages = 0;
        walk([&](const Segment& g, long long unit_lo) {
            // rows of the tile behind this one, on their way into L2
            if (a.wide_q && (g.tile + 1) * COLS < g.cols) {
                const int row0 = (g.tile + 1) * COLS / a.group, row1 = (min((g.tile + 2) * COLS, g.cols) - 1) / a.group;
                const uint32_t bytes = (uint32_t)(a.group * a.dk * sizeof(T));
                for (int x = row0 + lane; x <= row1; x += 32) l2_prefetch((const T*)a.q + (long)(g.q.first + x) * a.ldq + (long)g.head * a.group * a.dk, bytes);
            }
            for (int p = g.p0; p < g.p1; ++p, ++pages) {
                const int slot = pages % ring_n;
                int page = lane == 0 ? a.table[(size_t)g.s * a.width + p] : 0;
                wait(&raw_empty[slot], pages / ring_n + 1);
                if (lane == 0 && !*dead_s) {
                    const bool absent = page < 0 || page >= a.n_pages;
                    absent_s[slot] = absent;
                    if (absent) {
                        if (a.status != nullptr) atomicOr(a.status, kBadPage);
                        mbar_arrive(&raw_full[slot]);
                    } else {
                        mbar_expect_tx(&raw_full[slot], block);
                        if (a.skip < 0 || unit_lo + (p - g.lo) != a.skip) bulk_copy(smem_u32(ring) + slot * block, a.kv + ((size_t)page * a.kv_heads + g.head) * block, block, &raw_full[slot]);
                    }
                    ++copied;
                }
                __syncwarp();
            }
        });
    }
    // ---- nothing may be under way when the CTA ends: products have ended, and after a wait that gave up so have copies
    if (warp >= TILES * 8 + 4 && warp < TILES * 9 + 4) wait(&all_done, 0);
    __syncthreads();
    if (*dead_s && warp == TILES * 9 + 5 && lane == 0) {
        mbar_wait(&all_done, 0, a.wait_ns);
        for (int i = max(0, copied - ring_n); i < copied; ++i) mbar_wait(&raw_full[i % ring_n], (i / ring_n) & 1, a.wait_ns);
        if (a.status != nullptr) atomicOr(a.status, STATUS_TIMEOUT);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <typename T, int NG>
int32_t launch(AttendArgs a, uint64_t work, cudaStream_t st) {
    using Shape = PromptShape<NG, sizeof(T) == 4>;
    const int block = kv4_block(a.dk, a.dv);
    // 232448 bytes of shared memory per CTA, less what is declared in the kernel and what alignment to 1024 bytes may cost
    const int ring_n = std::min(kMaxRing, (232448 - 1024 - kStatic - Shape::kFixed) / block);
    a.tickets = (int32_t*)work;
    a.parts = (float*)(work + 4096);
    const size_t smem = 1024 + Shape::kFixed + (size_t)ring_n * block;
    LUMI_CUDA(cudaFuncSetAttribute(kv4_prompt_kernel<T, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)std::min(kPromptCtas, sm_count()));
    cfg.blockDim = dim3(Shape::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // the launch itself overlaps the kernel in front
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    LUMI_CUDA(cudaLaunchKernelEx(&cfg, kv4_prompt_kernel<T, NG>, a, ring_n));
    return LUMI_OK;
}

template <typename T>
int32_t of_type(const AttendArgs& a, uint64_t work, cudaStream_t st) {
    const int groups = std::max(kv4_groups(a.dk), kv4_groups(a.dv));
    if (groups <= 2) return launch<T, 2>(a, work, st);
    if (groups <= 4) return launch<T, 4>(a, work, st);
    return launch<T, 8>(a, work, st);
}

}  // namespace

int32_t launch_kv4_prompt(const AttendArgs& a, bool f32, uint64_t work, cudaStream_t st) { return f32 ? of_type<float>(a, work, st) : of_type<__nv_bfloat16>(a, work, st); }

}  // namespace lumi
