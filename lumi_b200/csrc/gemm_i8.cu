// Products in 8-bit integers: D[m][n] = (sum over k of A[m][k] W[n][k]) * a_scale[m] * w_scale[n] + bias[n] (+ D[m][n]).  The sums are 32-bit
// integers and therefore exact in any order: the kernels below, and any share of K, give the same bits.
//
// Three kernels: vector_kernel for up to eight rows (multiply-adds of four bytes on the CUDA cores, bound by the stream of W), tile_kernel for a batch of rows
// (tcgen05, one tile per CTA or, with K shared, per cluster), pair_kernel for many (tcgen05 by pairs of CTAs, persistent, two accumulators).  In both tensor-core kernels the
// weights are on the MMA's 128-row side and the rows of A are its columns: an accumulator lane is a column of D, so that a warp's 32 lanes write
// 32 neighbouring results of a row of D without any rearrangement, whatever D's alignment.
#include "device_args.h"
#include "rows.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <atomic>

namespace lumi {
namespace {

constexpr int kBlockK = 128;                 // bytes of K per pipeline stage: one row of the 128-byte swizzle
constexpr int kWRows = 128;                  // rows of W per CTA: the M of the MMA (a pair's: 256)
constexpr int kWBytes = kWRows * kBlockK;
constexpr int kMaxCols = 256;                // rows of A per tile: the N of the MMA
constexpr int kMaxStages = 8;

struct I8Args {
    const int8_t *a, *w;
    const float *a_scale, *w_scale, *bias;
    void* d;
    long lda, ldw, ldd;
    int M, N, K, accumulate;
    int32_t* status;
    uint64_t wait_ns;
    int skip_unit;                           // failure tests: operands of this tile never arrive
};

__device__ __forceinline__ float old_value(const float* p) { return *p; }
__device__ __forceinline__ float old_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void put_value(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
// the sum's way to a result, the same operations in every kernel
__device__ __forceinline__ float scaled(int sum, float sa, float sw, float bias) { return __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(sum), sa), sw), bias); }

// ---- up to eight rows: a warp takes R rows of W and a share of K --------------------------------
__device__ __forceinline__ int4 bytes16(const int8_t* p, int n) {       // the first n bytes, n < 16, zeros behind
    uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i) if (i < n) u[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
    return make_int4((int)u[0], (int)u[1], (int)u[2], (int)u[3]);
}
// of W: read once, and only behind the dependency wait
__device__ __forceinline__ int4 stream16(const int8_t* p) {
    int4 v;
    asm volatile("ld.global.cs.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ int dot16(const int4& a, const int4& b, int s) {
    return __dp4a(a.w, b.w, __dp4a(a.z, b.z, __dp4a(a.y, b.y, __dp4a(a.x, b.x, s))));
}

constexpr int kVecRows = 2;                  // rows of W per warp
constexpr int kVecDeep = 4;                  // pieces of 512 bytes of each that are under way

template <int MB, typename DT>
__global__ void __launch_bounds__(256) vector_kernel(I8Args g, int shares) {
    __shared__ int part[8][kVecRows * MB];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int share = warp % shares, n0 = (blockIdx.x * (8 / shares) + warp / shares) * kVecRows;
    pdl_release();
    pdl_sync();
    int sum[kVecRows][MB];
#pragma unroll
    for (int r = 0; r < kVecRows; ++r)
#pragma unroll
        for (int m = 0; m < MB; ++m) sum[r][m] = 0;
    const int8_t* w[kVecRows];
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) w[r] = g.w + (long)min(n0 + r, g.N - 1) * g.ldw;
    const int step = shares * 512, whole = g.K & ~15;
    for (int k0 = (share * 32 + lane) * 16; k0 < whole; k0 += kVecDeep * step) {
        int4 v[kVecDeep][kVecRows];
#pragma unroll
        for (int u = 0; u < kVecDeep; ++u)
#pragma unroll
            for (int r = 0; r < kVecRows; ++r)
                v[u][r] = k0 + u * step < whole ? stream16(w[r] + k0 + u * step) : make_int4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < kVecDeep; ++u) {
            if (k0 + u * step >= whole) break;
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                if (m >= g.M) break;
                const int4 a = *reinterpret_cast<const int4*>(g.a + m * g.lda + k0 + u * step);
#pragma unroll
                for (int r = 0; r < kVecRows; ++r) sum[r][m] = dot16(a, v[u][r], sum[r][m]);
            }
        }
    }
    if (whole < g.K && share == 0 && lane == 0) {         // the last bytes of a K that is no multiple of 16
#pragma unroll
        for (int r = 0; r < kVecRows; ++r) {
            const int4 v = bytes16(w[r] + whole, g.K - whole);
#pragma unroll
            for (int m = 0; m < MB; ++m)
                if (m < g.M) sum[r][m] = dot16(bytes16(g.a + m * g.lda + whole, g.K - whole), v, sum[r][m]);
        }
    }
#pragma unroll
    for (int r = 0; r < kVecRows; ++r)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int t = __reduce_add_sync(0xffffffffu, sum[r][m]);
            if (lane == 0) part[warp][r * MB + m] = t;
        }
    if (shares > 1) __syncthreads(); else __syncwarp();
    if (share != 0) return;
    for (int i = lane; i < kVecRows * MB; i += 32) {
        const int n = n0 + i / MB, m = i % MB;
        if (n >= g.N || m >= g.M) continue;
        int t = part[warp][i];
        for (int s = 1; s < shares; ++s) t += part[warp + s][i];
        float v = scaled(t, g.a_scale[m], g.w_scale[n], g.bias != nullptr ? g.bias[n] : 0.f);
        DT* d = (DT*)g.d + m * g.ldd + n;
        if (g.accumulate) v = __fadd_rn(v, old_value(d));
        put_value(d, v);
    }
}

// ---- tensor cores ---------------------------------------------------------------------------------
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// signed bytes by signed bytes into 32-bit integers, `rows` x `cols`
__device__ __forceinline__ uint32_t i8_idesc(int rows, int cols) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(rows >> 4) << 24); }
__device__ __forceinline__ void st_cluster_s32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

// Results of one row of W (this lane's) for 32 rows of A from m0 on, of which `live` exist.  buf: 32 floats of shared memory of this warp's own.
template <bool WHOLE, typename DT>
__device__ __forceinline__ void finish_columns(const I8Args& g, const uint32_t (&sum)[32], const float* buf, DT* d, int live, bool in, float sw, float bias) {
    constexpr int STEP = 16;                              // old values that are under way together
#pragma unroll
    for (int j0 = 0; j0 < 32; j0 += STEP) {
        float old[STEP];
        if (g.accumulate) {
            const DT* p = d;
#pragma unroll
            for (int j = 0; j < STEP; ++j, p += g.ldd) old[j] = in && (WHOLE || j0 + j < live) ? old_value(p) : 0.f;
        }
#pragma unroll
        for (int j4 = 0; j4 < STEP; j4 += 4) {
            const float4 sa = *reinterpret_cast<const float4*>(buf + j0 + j4);
            const float s[4] = {sa.x, sa.y, sa.z, sa.w};
#pragma unroll
            for (int e = 0; e < 4; ++e, d += g.ldd) {
                float v = scaled((int)sum[j0 + j4 + e], s[e], sw, bias);
                if (g.accumulate) v = __fadd_rn(v, old[j4 + e]);
                if (in && (WHOLE || j0 + j4 + e < live)) put_value(d, v);
            }
        }
    }
}
template <typename DT>
__device__ __forceinline__ void finish_strip(const I8Args& g, uint32_t acc, float* buf, int m0, int n, float sw, float bias, bool lost) {
    const int lane = threadIdx.x & 31, live = min(32, g.M - m0);
    const bool in = n < g.N;
    DT* d = (DT*)g.d + (long)m0 * g.ldd + n;
    if (lost) {
        for (int j = 0; j < live; ++j) if (in) put_value(d + j * g.ldd, __uint_as_float(0x7fffffffu));
        return;
    }
    __syncwarp();                                         // the last strip's scales have been read
    buf[lane] = lane < live ? g.a_scale[m0 + lane] : 0.f;
    uint32_t sum[32];
    tmem_ld32(acc, sum);
    __syncwarp();
    if (live == 32) finish_columns<true, DT>(g, sum, buf, d, live, in, sw, bias);
    else finish_columns<false, DT>(g, sum, buf, d, live, in, sw, bias);
}

struct TileTail {
    uint64_t full[kMaxStages], empty[kMaxStages], done, drain;
    uint32_t tmem_slot;
    int lost;                                // a wait of this CTA, or of one that shares K with it, ran out
    alignas(16) float scales[8][32];
};
constexpr int kTailBytes = 1280;
static_assert(sizeof(TileTail) <= kTailBytes, "tail of the shared memory");

struct TileShape { int cols, stages, splits; };

// A tile of 128 rows of W and `cols` rows of A per cluster of `splits` CTAs, which share K; each of them finishes cols / splits rows of A.
// Warp 0: copies.  Warp 1: TMEM and MMA.  All eight: accumulators (warp w reads the lanes of quarter w % 4, columns by halves).
template <typename DT>
__global__ void __launch_bounds__(256) tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, I8Args g, TileShape sh) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int S = sh.stages, cols = sh.cols, splits = sh.splits, stage = kWBytes + cols * kBlockK;
    int* part = reinterpret_cast<int*>(base + S * stage);               // splits > 1: [split][row of A][row of W]
    TileTail& tl = *reinterpret_cast<TileTail*>(base + S * stage + (splits > 1 ? cols * kWRows * 4 : 0));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % splits, n0 = (int)blockIdx.x / splits * kWRows, m0 = blockIdx.y * cols;
    const int num_kb = (g.K + kBlockK - 1) / kBlockK, kb0 = (int)((long)rank * num_kb / splits), nkb = (int)((long)(rank + 1) * num_kb / splits) - kb0;
    const uint32_t tmem_cols = cols <= 32 ? 32u : (cols <= 64 ? 64u : (cols <= 128 ? 128u : 256u));

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(&tl.full[s], 1); mbar_init(&tl.empty[s], 1); }
        mbar_init(&tl.done, 1);
        mbar_init(&tl.drain, 1);
        tl.lost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tl.tmem_slot)), "r"(tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // behind the allocation: a dependent that becomes resident beside this CTA may want TMEM too, and must not get it first
    pdl_release();
    if (splits > 1) cluster_arrive();                                   // "this CTA runs": sums may be sent to it
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tl.tmem_slot);
    bool timed_out = false;
    pdl_sync();

    if (warp == 0) {
        if (lane == 0 && (int)(blockIdx.y * gridDim.x + blockIdx.x) != g.skip_unit) {
            int s = 0, issued = 0;
            uint32_t ph = 0;
            for (int i = 0; i < nkb; ++i) {
                if (!mbar_wait(&tl.empty[s], ph ^ 1u, g.wait_ns)) { timed_out = true; break; }
                mbar_expect_tx(&tl.full[s], (uint32_t)stage);
                tma_load_2d(base + s * stage, &map_w, &tl.full[s], (kb0 + i) * kBlockK, n0);
                tma_load_2d(base + s * stage + kWBytes, &map_a, &tl.full[s], (kb0 + i) * kBlockK, m0);
                issued = i + 1;
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            if (timed_out)                                              // let the copies land (bounded) that nobody may consume
                for (int i = max(0, issued - S); i < issued; ++i) mbar_wait(&tl.full[i % S], (uint32_t)(i / S) & 1u, g.wait_ns);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = i8_idesc(kWRows, cols);
            int s = 0;
            uint32_t ph = 0;
            for (int i = 0; i < nkb; ++i) {
                if (!mbar_wait(&tl.full[s], ph, g.wait_ns)) { timed_out = true; break; }
                tc_fence_after();
                const uint32_t w = smem_u32(base + s * stage);
#pragma unroll
                for (int k = 0; k < kBlockK / 32; ++k)
                    umma_i8(tmem, make_smem_desc(w + k * 32), make_smem_desc(w + kWBytes + k * 32), idesc, (i > 0 || k > 0) ? 1u : 0u);
                umma_commit(&tl.empty[s]);
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            if (!timed_out) {
                umma_commit(&tl.done);
            } else {                                                    // let every MMA issued so far finish (bounded), then pass the word on
                umma_commit(&tl.drain);
                mbar_wait(&tl.drain, 0, g.wait_ns);
                *reinterpret_cast<volatile int*>(&tl.lost) = 1;
                mbar_arrive(&tl.done);
            }
        }
    }
    __syncwarp();
    const int q = warp & 3, half = warp >> 2;                           // TMEM lane quarter this warp may read; its share of the columns
    const int n = n0 + q * 32 + lane;
    const float sw = n < g.N ? g.w_scale[n] : 0.f, bias = n < g.N && g.bias != nullptr ? g.bias[n] : 0.f;
    if (splits > 1) cluster_wait();                                     // every CTA of the cluster runs
    if (!mbar_wait(&tl.done, 0, g.wait_ns)) timed_out = true;
    timed_out = __any_sync(0xffffffffu, timed_out);                     // tcgen05.ld below is warp-collective
    const bool lost = timed_out || *reinterpret_cast<volatile int*>(&tl.lost) != 0;
    tc_fence_after();
    const int RB = cols / splits;                                       // rows of A that each CTA of the cluster finishes
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    if (splits == 1) {
#pragma unroll 1
        for (int cb = half; cb < cols / 32; cb += 2) {
            if (m0 + cb * 32 >= g.M) break;
            finish_strip<DT>(g, lanes + (uint32_t)(cb * 32), tl.scales[warp], m0 + cb * 32, n, sw, bias, lost);
        }
    } else {
        if (lost) {
            if (lane == 0)
                for (int c = 0; c < splits; ++c) st_cluster_u32(map_to_rank(smem_u32(&tl.lost), (uint32_t)c), 1u);
        } else {
            const uint32_t slot = smem_u32(part) + (uint32_t)(rank * RB * kWRows + q * 32 + lane) * 4u;
#pragma unroll 1
            for (int cb = half; cb < cols / 32; cb += 2) {
                if (m0 + cb * 32 >= g.M) break;
                uint32_t r[32];
                tmem_ld32(lanes + (uint32_t)(cb * 32), r);
#pragma unroll
                for (int j4 = 0; j4 < 32; j4 += 4) {                    // RB is a multiple of four
                    const int b = cb * 32 + j4, to = b / RB;
                    const uint32_t at = map_to_rank(slot + (uint32_t)(b - to * RB) * (kWRows * 4u), (uint32_t)to);
#pragma unroll
                    for (int j = 0; j < 4; ++j) st_cluster_s32(at + (uint32_t)j * (kWRows * 4u), r[j4 + j]);
                }
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    if (splits > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    if (warp == 1) {                                                    // every accumulator has been read
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
    }
    if (timed_out && g.status != nullptr) atomicOr(g.status, STATUS_TIMEOUT);
    if (splits == 1) return;

    // ---- the rows of A that this CTA finishes: a warp's quarter of the rows of W, every second row of A
    const bool any_lost = *reinterpret_cast<volatile int*>(&tl.lost) != 0;
    if (n >= g.N) return;
    for (int r = half; r < RB; r += 2) {
        const int m = m0 + rank * RB + r;
        if (m >= g.M) break;
        int sum = 0;
        for (int c = 0; c < splits; ++c) sum += part[(c * RB + r) * kWRows + q * 32 + lane];
        DT* d = (DT*)g.d + (long)m * g.ldd + n;
        float v = scaled(sum, g.a_scale[m], sw, bias);
        if (g.accumulate) v = __fadd_rn(v, old_value(d));
        put_value(d, any_lost ? __uint_as_float(0x7fffffffu) : v);
    }
}

// ---- many rows: pairs of CTAs ------------------------------------------------------------------------
// Two CTAs of a cluster (two SMs) take tiles of 256 rows of W and `cols` rows of A (cta_group::2): each stages its 128 rows of W and half of the rows of A, the
// first one issues the MMAs for both, each finishes its own rows of W.  Persistent, with two accumulators: a tile is finished while the next is multiplied.
// Tiles go in blocks of 16 tiles of rows of A, rows of W by rows of W within a block, so that both operands come out of L2.
// Warp 0: copies.  Warp 1: TMEM and MMA.  Warps 2 to 9: accumulators, two warps per quarter of the lanes, columns in turn.
constexpr int kPairThreads = 320;
struct PairTail {
    uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
    uint32_t tmem_slot, gave_up, issued[2];
    alignas(16) float scales[8][32];
};
static_assert(sizeof(PairTail) <= kTailBytes, "tail of the shared memory");
constexpr int kBlockTiles = 16;

struct PairShape { int cols, stages, tiles_a, tiles; };

template <typename DT>
__global__ void __launch_bounds__(kPairThreads, 1) pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, I8Args g, PairShape sh) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int S = sh.stages, cols = sh.cols, stage = kWBytes + cols / 2 * kBlockK;
    PairTail& tl = *reinterpret_cast<PairTail*>(base + S * stage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x & 1), first = (int)(blockIdx.x >> 1), at_once = (int)(gridDim.x >> 1);
    const int num_kb = (g.K + kBlockK - 1) / kBlockK, tiles_w = sh.tiles / sh.tiles_a;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(&tl.full[s], 1); mbar_init(&tl.empty[s], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&tl.acc_full[i], 1); mbar_init(&tl.acc_empty[i], 16); }
        mbar_init(&tl.drain, 1);
        tl.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tl.tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncwarp();
    cluster_arrive();                                                   // the other CTA's barriers exist, its TMEM is allocated
    cluster_wait();
    tc_fence_after();
    pdl_release();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tl.tmem_slot);
    auto place = [&](int t, int& m0, int& n0) {                         // first row of A of a tile, first row of W of the pair's
        const int blk = t / (kBlockTiles * tiles_w), r = t - blk * kBlockTiles * tiles_w, rows = min(kBlockTiles, sh.tiles_a - blk * kBlockTiles);
        const int tw = r / rows;
        m0 = (blk * kBlockTiles + r - tw * rows) * cols;
        n0 = tw * 2 * kWRows;
    };
    bool timed_out = false;
    pdl_sync();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t kbg = 0;                                           // k-blocks issued so far, over all tiles
            int s = 0;
            uint32_t ph = 0;
            for (int t = first; t < sh.tiles && !timed_out; t += at_once) {
                if (t == g.skip_unit && rank == 1) break;
                int m0, n0;
                place(t, m0, n0);
                for (int kb = 0; kb < num_kb; ++kb, ++kbg) {
                    if (!mbar_wait(&tl.empty[s], ph ^ 1u, g.wait_ns)) { timed_out = true; break; }
                    const uint32_t bar = map_to_rank(smem_u32(&tl.full[s]), 0);      // both CTAs' copies complete on the first one's barrier
                    if (rank == 0) mbar_expect_tx(&tl.full[s], 2u * (uint32_t)stage);
                    tma_load_2d_pair(base + s * stage, &map_w, bar, kb * kBlockK, n0 + rank * kWRows);
                    tma_load_2d_pair(base + s * stage + kWBytes, &map_a, bar, kb * kBlockK, m0 + rank * (cols / 2));
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
            }
            st_cluster_u32(map_to_rank(smem_u32(&tl.issued[rank]), 0), kbg);
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = i8_idesc(2 * kWRows, cols);
            int s = 0;
            uint32_t ph = 0, it = 0;
            for (int t = first; t < sh.tiles && !timed_out; t += at_once, ++it) {
                const uint32_t as = it & 1u, aph = (it >> 1) & 1u, acc = tmem + as * kMaxCols;
                if (!mbar_wait(&tl.acc_empty[as], aph ^ 1u, g.wait_ns)) { timed_out = true; break; }      // this accumulator has been read
                tc_fence_after();
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(&tl.full[s], ph, g.wait_ns)) { timed_out = true; break; }
                    tc_fence_after();
                    const uint32_t w = smem_u32(base + s * stage);
#pragma unroll
                    for (int k = 0; k < kBlockK / 32; ++k)
                        umma_i8_pair(acc, make_smem_desc(w + k * 32), make_smem_desc(w + kWBytes + k * 32), idesc, (kb > 0 || k > 0) ? 1u : 0u);
                    umma_commit_pair(&tl.empty[s]);
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
                if (timed_out) break;
                umma_commit_pair(&tl.acc_full[as]);
            }
            if (timed_out) {                                            // let every MMA issued so far finish (bounded) before TMEM is freed
                umma_commit_pair(&tl.drain);
                mbar_wait(&tl.drain, 0, g.wait_ns);
            }
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;
        uint32_t it = 0;
        for (int t = first; t < sh.tiles; t += at_once, ++it) {
            const uint32_t as = it & 1u, aph = (it >> 1) & 1u;
            int m0, n0;
            place(t, m0, n0);
            const int n = n0 + rank * kWRows + q * 32 + lane;
            const float sw = n < g.N ? g.w_scale[n] : 0.f, bias = n < g.N && g.bias != nullptr ? g.bias[n] : 0.f;
            // after a wait that ran out, this tile and all that follow are left as NaN
            if (!timed_out && !mbar_wait(&tl.acc_full[as], aph, g.wait_ns)) timed_out = true;
            timed_out = __any_sync(0xffffffffu, timed_out);             // tcgen05.ld is warp-collective
            tc_fence_after();
            const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + as * kMaxCols;
#pragma unroll 1
            for (int cb = half; cb < cols / 32; cb += 2) {
                if (m0 + cb * 32 >= g.M) break;
                finish_strip<DT>(g, lanes + (uint32_t)(cb * 32), tl.scales[warp - 2], m0 + cb * 32, n, sw, bias, timed_out);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(map_to_rank(smem_u32(&tl.acc_empty[as]), 0));
        }
    }
    if (timed_out && g.status != nullptr) atomicOr(g.status, STATUS_TIMEOUT);
    tc_fence_before();
    // neither CTA's memory goes away under the other's MMAs and arrivals
    if (timed_out)
        for (uint32_t r = 0; r < 2; ++r) st_cluster_u32(map_to_rank(smem_u32(&tl.gave_up), r), 1u);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (*reinterpret_cast<volatile uint32_t*>(&tl.gave_up) != 0) {      // ... nor under a copy: the first CTA waits (bounded) for both CTAs' copies
        if (rank == 0 && threadIdx.x == 0) {
            volatile uint32_t* issued = tl.issued;
            const uint32_t i0 = issued[0], i1 = issued[1], lo = min(i0, i1), hi = max(i0, i1);      // at most S apart: neither gets past an unconsumed stage
            for (uint32_t k = lo; k < hi; ++k) {                        // only one CTA issued this block: the barrier expects both halves, or neither
                if (i0 > i1) mbar_complete_tx(&tl.full[k % S], (uint32_t)stage);
                else mbar_expect_tx(&tl.full[k % S], (uint32_t)stage);
            }
            for (uint32_t k = hi > (uint32_t)S ? hi - S : 0; k < hi; ++k) mbar_wait(&tl.full[k % S], (k / S) & 1u, g.wait_ns);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---- host ------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// [rows][K] bytes in rows of ld, box of 128 bytes by box_rows, 128-byte swizzle, zeros behind K and behind the last row
int32_t make_i8_map(CUtensorMap* map, const void* ptr, long ld, int rows, int K, int box_rows) {
    static std::atomic<EncodeTiledFn> encode{nullptr};
    EncodeTiledFn fn = encode.load(std::memory_order_acquire);
    if (fn == nullptr) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        LUMI_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
        if (p == nullptr || q != cudaDriverEntryPointSuccess) return fail(LUMI_E_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
        fn = reinterpret_cast<EncodeTiledFn>(p);
        encode.store(fn, std::memory_order_release);
    }
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {(cuuint32_t)kBlockK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LUMI_E_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (%d rows of %d bytes)", (int)r, rows, K);
    return LUMI_OK;
}

// Lets a kernel have as much shared memory as there is, once per device.
int32_t allow_smem(const void* kernel, std::atomic<uint64_t>& devices) {
    int dev = 0;
    LUMI_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (devices.load(std::memory_order_relaxed) & bit)) return LUMI_OK;
    LUMI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    devices.fetch_or(bit, std::memory_order_relaxed);
    return LUMI_OK;
}

struct Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    Launch(dim3 grid, int threads, int smem, int cluster, cudaStream_t st) {
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // the set-up overlaps the kernel in front
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = cluster > 1 ? 2 : 1;
    }
};

template <int MB, typename DT>
int32_t launch_vector(const I8Args& g, cudaStream_t st) {
    int shares = 1;                          // warps that share K: until the GPU has about 16 warps per SM, as long as each has 512 bytes of a row
    while (shares < 8 && (long)g.N / kVecRows * shares < 16l * sm_count() && g.K > 512 * shares) shares *= 2;
    const int rows = 8 / shares * kVecRows;
    Launch l(dim3((g.N + rows - 1) / rows), 256, 0, 1, st);
    LUMI_CUDA(cudaLaunchKernelEx(&l.cfg, vector_kernel<MB, DT>, g, shares));
    return LUMI_OK;
}

template <typename DT>
int32_t launch_tile(const I8Args& g, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    const int num_kb = (g.K + kBlockK - 1) / kBlockK;
    TileShape sh;
    sh.cols = g.M <= 32 ? 32 : (g.M <= 64 ? 64 : 128);
    const long tiles = (long)((g.N + kWRows - 1) / kWRows), whole = tiles * ((g.M + sh.cols - 1) / sh.cols);
    sh.splits = 1;
    while (sh.splits < 8 && num_kb >= 4 * sh.splits && whole * 2 * sh.splits <= sm_count()) sh.splits *= 2;
    const int stage = kWBytes + sh.cols * kBlockK, part = sh.splits > 1 ? sh.cols * kWRows * 4 : 0;
    const int budget = (whole * sh.splits > sm_count() ? 112 : 220) * 1024 - part - kTailBytes - 1024;
    sh.stages = std::max(2, std::min({kMaxStages, budget / stage, (num_kb + sh.splits - 1) / sh.splits}));
    CUtensorMap ma, mw;
    LUMI_TRY(make_i8_map(&ma, g.a, g.lda, g.M, g.K, sh.cols));
    LUMI_TRY(make_i8_map(&mw, g.w, g.ldw, g.N, g.K, kWRows));
    LUMI_TRY(allow_smem((const void*)tile_kernel<DT>, ready));
    Launch l(dim3((unsigned)(tiles * sh.splits), (g.M + sh.cols - 1) / sh.cols), 256, sh.stages * stage + part + kTailBytes + 1024, sh.splits, st);
    LUMI_CUDA(cudaLaunchKernelEx(&l.cfg, tile_kernel<DT>, ma, mw, g, sh));
    return LUMI_OK;
}

template <typename DT>
int32_t launch_pair(const I8Args& g, int cols, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    PairShape sh;
    sh.cols = cols;
    sh.tiles_a = (g.M + cols - 1) / cols;
    sh.tiles = sh.tiles_a * ((g.N + 2 * kWRows - 1) / (2 * kWRows));
    const int stage = kWBytes + cols / 2 * kBlockK;
    sh.stages = std::min(kMaxStages, (220 * 1024 - kTailBytes) / stage);
    CUtensorMap ma, mw;
    LUMI_TRY(make_i8_map(&ma, g.a, g.lda, g.M, g.K, cols / 2));
    LUMI_TRY(make_i8_map(&mw, g.w, g.ldw, g.N, g.K, kWRows));
    LUMI_TRY(allow_smem((const void*)pair_kernel<DT>, ready));
    Launch l(dim3(2 * std::min(sh.tiles, sm_count() / 2)), kPairThreads, sh.stages * stage + kTailBytes + 1024, 2, st);
    LUMI_CUDA(cudaLaunchKernelEx(&l.cfg, pair_kernel<DT>, ma, mw, g, sh));
    return LUMI_OK;
}

// Columns of the pairs' tiles: the GPU works in rounds of a tile per pair, a round costs about its tile's columns.
int pair_cols(const I8Args& g, long& cost) {
    const long pairs = sm_count() / 2, tiles_w = (g.N + 2 * kWRows - 1) / (2 * kWRows);
    int best = 0;
    cost = 0;
    for (int c = kMaxCols; c >= 64; c -= 32) {
        const long k = (tiles_w * ((g.M + c - 1) / c) + pairs - 1) / pairs * (c + 32);
        if (best == 0 || k < cost) { best = c; cost = k; }
    }
    return best;
}

template <typename DT>
int32_t launch_product(const I8Args& g, cudaStream_t st) {
    if (g.M <= 1) return launch_vector<1, DT>(g, st);
    if (g.M <= 2) return launch_vector<2, DT>(g, st);
    if (g.M <= 4) return launch_vector<4, DT>(g, st);
    if (g.M <= 8) return launch_vector<8, DT>(g, st);
    long cost;
    if (g.M > 1024) return launch_pair<DT>(g, pair_cols(g, cost), st);
    return launch_tile<DT>(g, st);
}

}  // namespace
}  // namespace lumi

using namespace lumi;

extern "C" int32_t lumi_k_gemm_i8(uint64_t a, int32_t lda, uint64_t a_scale, uint64_t w, int32_t ldw, uint64_t w_scale, uint64_t bias, uint64_t d,
                                  int32_t d_dtype, int32_t ldd, int32_t M, int32_t N, int32_t K, int32_t accumulate, uint64_t status, uint64_t stream) {
    if (!a || !a_scale || !w || !w_scale || !d || M < 0 || N < 0 || K <= 0 || lda < K || ldw < K || ldd < N ||
        (d_dtype != LUMI_DTYPE_F32 && d_dtype != LUMI_DTYPE_BF16))
        return fail(LUMI_E_INVALID, "bad argument to lumi_k_gemm_i8");
    if ((a & 15) || (w & 15) || lda % 16 || ldw % 16 || ((a_scale | w_scale | bias | status) & 3) || (d & (d_dtype == LUMI_DTYPE_F32 ? 3 : 1)))
        return fail(LUMI_E_INVALID, "lumi_k_gemm_i8: rows of A and W have to begin on 16-byte boundaries, numbers on their own");
    // 131071 products of -128 and -128 are the most that a 32-bit sum holds
    if (K > 131071) return fail(LUMI_E_UNSUPPORTED, "lumi_k_gemm_i8: K %d (at most 131071)", K);
    if (M == 0 || N == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory("lumi_k_gemm_i8", {a, a_scale, w, w_scale, bias, d, status}));
    const I8Args g{(const int8_t*)a, (const int8_t*)w, (const float*)a_scale, (const float*)w_scale, (const float*)bias, (void*)d, lda, ldw, ldd, M, N, K, accumulate,
                   (int32_t*)status, kWaitLimitNs, -1};
    return d_dtype == LUMI_DTYPE_F32 ? launch_product<float>(g, (cudaStream_t)stream) : launch_product<__nv_bfloat16>(g, (cudaStream_t)stream);
}
