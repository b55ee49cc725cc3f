// Products in 8-bit integers: D[m][n] = (sum over k of A[m][k] W[n][k]) * a_scale[m] * w_scale[n] + bias[n] (+ D[m][n]).  The sums are 32-bit
// integers and therefore exact in any order: the kernels below, and any share of K, give the same bits.
//
// Four kernels: vector_kernel for one or two rows (multiply-adds of four bytes on the CUDA cores), few_kernel for up to eight and a small W (warp-level MMA),
// tile_kernel for a batch of rows (tcgen05, one tile per CTA or, with K shared, per cluster) and pair_kernel for many (tcgen05 by pairs of CTAs, persistent, two
// accumulators).  In both tcgen05 kernels the weights are on the MMA's 128-row side and the rows of A are its columns: an accumulator lane is a column
// of D, so that a warp's 32 lanes write 32 neighbouring results of a row of D without any rearrangement, whatever D's alignment.
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
constexpr int kMaxRows = 1 << 30;            // of A and of W: places of tiles are 32-bit numbers
constexpr int kClusterCtas = 128;             // CTAs in clusters that run at once for certain

struct I8Args {
    const int8_t *a, *w;
    const float *a_scale, *w_scale, *bias;
    void* d;
    long lda, ldw, ldd;
    int M, N, K, accumulate;
    int32_t* status;
    uint64_t wait_ns;
    int skip_unit;                           // failure tests: operands of this tile never arrive
    int give_up;                             // failure tests: a wait of this tile runs out at once (tile_kernel: the MMA warp's first; pair_kernel: one finishing warp's for the sums)
};

__device__ __forceinline__ float old_value(const float* p) { return *p; }
__device__ __forceinline__ float old_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put_value(float* p, float v) { *p = v; }
__device__ __forceinline__ void put_value(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
// the sum's way to a result, the same operations in every kernel
__device__ __forceinline__ float scaled(int sum, float sa, float sw, float bias) { return __fmaf_rn(__fmul_rn(__int2float_rn(sum), sa), sw, bias); }

// ---- one or two rows: a warp takes two rows of W and a share of K --------------------------------
__device__ __forceinline__ int4 bytes16(const int8_t* p, int n) {       // the first n bytes, n < 16, zeros behind
    uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i) if (i < n) u[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
    return make_int4((int)u[0], (int)u[1], (int)u[2], (int)u[3]);
}
// of W: read once, and only behind the dependency wait
__device__ __forceinline__ int4 stream16(const int8_t* p) {
    int4 v;
    asm volatile("ld.global.L1::no_allocate.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ int dot16(const int4& a, const int4& b, int s) {
    return __dp4a(a.w, b.w, __dp4a(a.z, b.z, __dp4a(a.y, b.y, __dp4a(a.x, b.x, s))));
}

// Bound by the stream of W, for small products by its latency.  Device time, us, 1 x 7360 x 1024 / 1 x 1024 x 8448 / 1 x 16384 x 4096 (67 MB, DRAM's floor 10.2): two rows of W per
// warp and three pieces of each under way 3.0 / 3.5 / 12.4, four pieces 3.6 / 4.9 / 12.5, two 3.1 / 4.7 / 13.1; one row and four pieces 3.8 / 4.2 / 12.9.
constexpr int kVecRows = 2;                  // rows of W per warp
constexpr int kVecDeep = 3;                  // pieces of 512 bytes of each that are under way

// MB rows of A
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
            for (int m = 0; m < MB; ++m) sum[r][m] = dot16(bytes16(g.a + m * g.lda + whole, g.K - whole), v, sum[r][m]);
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
        if (n >= g.N) continue;
        int t = part[warp][i];
        for (int s = 1; s < shares; ++s) t += part[warp + s][i];
        float v = scaled(t, g.a_scale[m], g.w_scale[n], g.bias != nullptr ? g.bias[n] : 0.f);
        DT* d = (DT*)g.d + m * g.ldd + n;
        if (g.accumulate) v = __fadd_rn(v, old_value(d));
        put_value(d, v);
    }
}

// ---- three to eight rows: a warp takes 16 rows of W and a share of K ------------------------------
__device__ __forceinline__ void mma_i8(int (&c)[4], int a0, int a1, int a2, int a3, int b0, int b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A warp-level MMA needs neither TMEM nor tensor maps and no barrier to start, which is what a small product's time goes to; a large W streams better through the tiles
// below.  Device time, us, this kernel / tile_kernel, 8 rows: 1024 x 1024 2.4 / 3.6, 7360 x 1024 4.0 / 4.4, 1024 x 2048 3.2 / 3.9, 5632 x 2048 5.8 / 6.1, 16384 x 1024 6.0 / 5.9,
// 1024 x 2816 4.5 / 4.0, 1024 x 4096 7.1 / 4.3; with two such tiles for 16 rows 7360 x 1024 5.3 / 4.4.
constexpr int kFewW = 16;                    // rows of W per warp: the M of the MMA; rows of A are its columns
constexpr int kFewRows = 8, kFewK = 2048;
constexpr long kFewBytes = 12l << 20;        // of W
constexpr int kFewDeep = 3;                  // steps of 64 bytes of each that are under way

// Lane 4 g + t holds bytes 16 t to 16 t + 15 of a step of rows g and g + 8 of W and of row g of A.  An MMA wants bytes 4 t and 16 + 4 t of 32: which bytes of K
// these are does not matter as long as they are the same of both operands, so it is given words 0 and 1, the next one words 2 and 3.
template <typename DT>
__global__ void __launch_bounds__(256) few_kernel(I8Args g, int shares) {
    __shared__ int4 part[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, t = lane & 3;
    const int share = warp % shares, n0 = (blockIdx.x * (8 / shares) + warp / shares) * kFewW;
    pdl_release();
    pdl_sync();
    int sum[4] = {0, 0, 0, 0};
    const int8_t *w0 = g.w + (long)min(n0 + row, g.N - 1) * g.ldw, *w1 = g.w + (long)min(n0 + row + 8, g.N - 1) * g.ldw;
    const int whole = g.K & ~15, step = shares * 64;
    const int8_t* a = g.a + min(row, g.M - 1) * g.lda;
    auto multiply = [&](const int4& u, const int4& v, const int4& x) {
        mma_i8(sum, u.x, v.x, u.y, v.y, x.x, x.y);
        mma_i8(sum, u.z, v.z, u.w, v.w, x.z, x.w);
    };
    const int4 zero = make_int4(0, 0, 0, 0);
    for (int k0 = share * 64 + t * 16; k0 - t * 16 < whole; k0 += kFewDeep * step) {      // (the same for a whole warp)
        int4 u[kFewDeep], v[kFewDeep];
#pragma unroll
        for (int d = 0; d < kFewDeep; ++d) {
            const bool in = k0 + d * step < whole;
            u[d] = in ? stream16(w0 + k0 + d * step) : zero;
            v[d] = in ? stream16(w1 + k0 + d * step) : zero;
        }
#pragma unroll
        for (int d = 0; d < kFewDeep; ++d)
            multiply(u[d], v[d], k0 + d * step < whole && row < g.M ? *reinterpret_cast<const int4*>(a + k0 + d * step) : zero);
    }
    if (whole < g.K && share == shares - 1) {             // the last bytes of a K that is no multiple of 16
        const int n = t == 0 ? g.K - whole : 0;
        multiply(bytes16(w0 + whole, n), bytes16(w1 + whole, n), bytes16(a + whole, row < g.M ? n : 0));
    }
    if (shares > 1) {
        part[warp][lane] = make_int4(sum[0], sum[1], sum[2], sum[3]);
        __syncthreads();
        if (share != 0) return;
        for (int s = 1; s < shares; ++s) {
            const int4 p = part[warp + s][lane];
            sum[0] += p.x; sum[1] += p.y; sum[2] += p.z; sum[3] += p.w;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int n = n0 + row + (e >> 1) * 8, m = 2 * t + (e & 1);
        if (n >= g.N || m >= g.M) continue;
        float v = scaled(sum[e], g.a_scale[m], g.w_scale[n], g.bias != nullptr ? g.bias[n] : 0.f);
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
// Bounded wait, as mbar_wait, but the clock is only looked at every so many tries: reading it takes about as long as a stage of the pipeline.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
    uint64_t t0 = 0;
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63) == 0) {
            const uint64_t t = globaltimer_ns();
            if (t0 == 0) t0 = t;
            else if (t - t0 > limit_ns) return false;
        }
    }
}
// An arrival that orders nothing but itself: a release would wait for this thread's results to reach memory, while all that the barrier guards has been read.
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// An operand tile's descriptor changes in its low word alone, by 16 bytes per one: the issuing thread adds, since composing two of them per MMA takes it
// longer than a narrow MMA.
__device__ __forceinline__ uint64_t moved(uint64_t desc, uint32_t units) { return (desc & 0xffffffff00000000ull) | (uint32_t)((uint32_t)desc + units); }
// One lane of a warp that has not parted.  The warps that issue copies and MMAs run their loops whole, so that what these instructions want in uniform registers is computed there: by
// one lane in a branch of its own, each MMA took its issuing thread four moves more.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }
// signed bytes by signed bytes into 32-bit integers, `rows` x `cols`
__device__ __forceinline__ uint32_t i8_idesc(int rows, int cols) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(rows >> 4) << 24); }
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void shared_load4(uint32_t at, float (&v)[32], int i) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3]) : "r"(at + 4 * i) : "memory");
}
__device__ __forceinline__ float shared_value(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void shared_put(uint32_t at, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
// bf16 strips cross shared memory as 8 x 8 matrices, transposed on their way: a quarter of the accesses that results one by one take.  A strip holds rows of A, 64 bytes each, whose
// 16-byte pieces are XOR-ed with the row's place (the 64-byte swizzle of tensor maps), so that the eight rows of a matrix meet eight different banks.
// Lane 4 r + c of a warp has columns 2 c and 2 c + 1 (rows of A) of rows r and r + 8 (of W) of 16 x 8 accumulators.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&a)[16], uint32_t (&b)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]),
                   "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15]),
                   "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]), "+r"(b[5]), "+r"(b[6]), "+r"(b[7]),
                   "+r"(b[8]), "+r"(b[9]), "+r"(b[10]), "+r"(b[11]), "+r"(b[12]), "+r"(b[13]), "+r"(b[14]), "+r"(b[15])
                 :: "memory");
}
__device__ __forceinline__ uint32_t strip_piece(uint32_t strip, int b, int lane) {       // where lane points for the matrices of rows 8 b to 8 b + 7 of A
    const int row = 8 * b + (lane & 7);
    return strip + (uint32_t)(row * 64 + (((lane >> 3) ^ ((row >> 1) & 3)) << 4));
}
__device__ __forceinline__ void put_matrices(uint32_t at, const uint32_t (&m)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3]) : "memory");
}
__device__ __forceinline__ void get_matrices(uint32_t at, uint32_t (&m)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3]) : "r"(at) : "memory");
}
// sums[g]: rows 16 g to 16 g + 15 of W, 32 rows of A; sw, bias: of rows lane / 4 + 8 k of W.
__device__ __forceinline__ void finish_matrices(const uint32_t (&lo)[16], const uint32_t (&hi)[16], const float* a_scale, const float (&sw)[4], const float (&bias)[4], bool add,
                                                uint32_t strip, int lane) {
    float2 sa[4];
#pragma unroll
    for (int b = 0; b < 4; ++b)
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(sa[b].x), "=f"(sa[b].y) : "r"(smem_u32(a_scale) + (uint32_t)(8 * b + 2 * (lane & 3)) * 4u) : "memory");
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const uint32_t at = strip_piece(strip, b, lane);
        uint32_t old[4], out[4];
        if (add) get_matrices(at, old);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t s0 = k < 2 ? lo[4 * b + 2 * k] : hi[4 * b + 2 * (k - 2)], s1 = k < 2 ? lo[4 * b + 2 * k + 1] : hi[4 * b + 2 * (k - 2) + 1];
            float v0 = scaled((int)s0, sa[b].x, sw[k], bias[k]), v1 = scaled((int)s1, sa[b].y, sw[k], bias[k]);
            if (add) {
                v0 = __fadd_rn(v0, __uint_as_float(old[k] << 16));
                v1 = __fadd_rn(v1, __uint_as_float(old[k] & 0xffff0000u));
            }
            const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
            out[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
        put_matrices(at, out);
    }
}
// Results of one row of W (this lane's) for 32 rows of A, of which `live` exist; a_scale: in shared memory.
template <bool WHOLE, typename DT>
__device__ __forceinline__ void finish_columns(const I8Args& g, const uint32_t (&sum)[32], const float* a_scale, DT* d, int live, bool in, float sw, float bias) {
    // everything is read before anything is written: the compiler cannot tell results from scales, and would wait for each group of them
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; j += 4) shared_load4(smem_u32(a_scale), v, j);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = scaled((int)sum[j], v[j], sw, bias);
    constexpr int STEP = 16;                              // old values that are under way together
#pragma unroll
    for (int j0 = 0; j0 < 32; j0 += STEP) {
        if (g.accumulate) {
            float old[STEP];
            const DT* p = d;
#pragma unroll
            for (int j = 0; j < STEP; ++j, p += g.ldd) old[j] = in && (WHOLE || j0 + j < live) ? old_value(p) : 0.f;
#pragma unroll
            for (int j = 0; j < STEP; ++j) v[j0 + j] = __fadd_rn(v[j0 + j], old[j]);
        }
#pragma unroll
        for (int j = 0; j < STEP; ++j, d += g.ldd)
            if (in && (WHOLE || j0 + j < live)) put_value(d, v[j0 + j]);
    }
}
template <typename DT>
__device__ __forceinline__ void finish_strip(const I8Args& g, uint32_t acc, const float* a_scale, int m0, int n, float sw, float bias, bool lost) {
    const int live = min(32, g.M - m0);
    const bool in = n < g.N;
    DT* d = (DT*)g.d + (long)m0 * g.ldd + n;
    if (lost) {
        for (int j = 0; j < live; ++j) if (in) put_value(d + j * g.ldd, __uint_as_float(0x7fffffffu));
        return;
    }
    uint32_t sum[32];
    tmem_ld32(acc, sum);
    if (live == 32) finish_columns<true, DT>(g, sum, a_scale, d, live, in, sw, bias);
    else finish_columns<false, DT>(g, sum, a_scale, d, live, in, sw, bias);
}

// The same for a kernel that knows whether it adds, with old values that were asked for ahead: `old` has this strip's and then takes the next one's, from m_next on (-1: there is none).
template <typename DT>
__device__ __forceinline__ void load_old(const I8Args& g, int m0, int n, float (&old)[32]) {
    const int live = n < g.N ? g.M - m0 : 0;
    const DT* p = (const DT*)g.d + (long)m0 * g.ldd + n;
#pragma unroll
    for (int j = 0; j < 32; ++j, p += g.ldd) old[j] = j < live ? old_value(p) : 0.f;
}
template <bool ADD, typename DT>
__device__ __forceinline__ void tile_strip(const I8Args& g, uint32_t acc, const float* a_scale, int m0, int n, float sw, float bias, float (&old)[32], int m_next) {
    const int live = n < g.N ? g.M - m0 : 0;
    DT* d = (DT*)g.d + (long)m0 * g.ldd + n;
    uint32_t sum[32];
    tmem_ld32(acc, sum);
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; j += 4) shared_load4(smem_u32(a_scale), v, j);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = scaled((int)sum[j], v[j], sw, bias);
    if constexpr (ADD) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __fadd_rn(v[j], old[j]);
        if (m_next >= 0) load_old<DT>(g, m_next, n, old);
    }
    if (live >= 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j, d += g.ldd) put_value(d, v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j, d += g.ldd) if (j < live) put_value(d, v[j]);
    }
}
// Results that a lost wait cost.
template <typename DT>
__device__ __forceinline__ void lose_strip(const I8Args& g, int m0, int n) {
    if (n < g.N)
#pragma unroll 1
        for (int m = m0; m < min(m0 + 32, g.M); ++m) put_value((DT*)g.d + (long)m * g.ldd + n, __uint_as_float(0x7fffffffu));
}

struct TileTail {
    uint64_t full[kMaxStages], empty[kMaxStages], done, drain;
    uint32_t tmem_slot;
    int lost;                                // a wait of this CTA, or of one that shares K with it, ran out
    alignas(16) float a_scale[kMaxCols];     // of the tile's rows of A
};
constexpr int kTailBytes = 1536;
static_assert(sizeof(TileTail) <= kTailBytes, "tail of the shared memory");

struct TileShape { int cols, stages, splits; };

// A tile of 128 rows of W and `cols` rows of A per cluster of `splits` CTAs, which share K; each of them finishes cols / splits rows of A.
// Warp 0: copies.  Warp 1: TMEM and MMA.  All eight: accumulators (warp w reads the lanes of quarter w % 4, strips of 32 columns in turn).
// What bounds it is a chain: launch and barriers, the first copies, 0.19 us per k-block (a wait, four MMAs, a commit; issued by one lane in a branch of its own it took 0.25, with
// descriptors composed anew 0.29; copies by two threads or sums in turn in four accumulators changed nothing), the results.  203 x 2053 x 1111: 4.3 us, DRAM's floor 0.5.
template <typename DT, bool ADD>
__global__ void __launch_bounds__(256, 2) tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, I8Args g, TileShape sh) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int S = sh.stages, cols = sh.cols, splits = sh.splits, stage = kWBytes + cols * kBlockK;
    int* part = reinterpret_cast<int*>(base + S * stage);               // splits > 1: [split][four rows of A][row of W][4]
    TileTail& tl = *reinterpret_cast<TileTail*>(base + S * stage + (splits > 1 ? cols * kWRows * 4 : 0));
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
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
    int issued = 0;                                                     // (warp 0) k-blocks whose copies are on their way or have landed
    pdl_sync();

    if (warp == 0) {
        if ((int)(blockIdx.y * gridDim.x + blockIdx.x) != g.skip_unit) {
            int s = 0;
            uint32_t ph = 0;
            for (int i = 0; i < nkb; ++i) {
                if (!__all_sync(0xffffffffu, wait_for(&tl.empty[s], ph ^ 1u, g.wait_ns))) { timed_out = true; break; }
                if (elect_one()) {
                    mbar_expect_tx(&tl.full[s], (uint32_t)stage);
                    tma_load_2d(base + s * stage, &map_w, &tl.full[s], (kb0 + i) * kBlockK, n0);
                    tma_load_2d(base + s * stage + kWBytes, &map_a, &tl.full[s], (kb0 + i) * kBlockK, m0);
                }
                __syncwarp();
                issued = i + 1;
                if (++s == S) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        const uint32_t idesc = i8_idesc(kWRows, cols), units = (uint32_t)stage >> 4;
        const uint64_t w0 = make_smem_desc(smem_u32(base)), a0 = make_smem_desc(smem_u32(base) + kWBytes);
        int s = 0;
        uint32_t ph = 0;
        timed_out = (int)(blockIdx.y * gridDim.x + blockIdx.x) == g.give_up;
        const int steps = timed_out ? 0 : nkb;
        for (int i = 0; i < steps; ++i) {
            if (!__all_sync(0xffffffffu, wait_for(&tl.full[s], ph, g.wait_ns))) { timed_out = true; break; }
            tc_fence_after();
            if (elect_one()) {
                const uint64_t w = moved(w0, (uint32_t)s * units), a = moved(a0, (uint32_t)s * units);
#pragma unroll
                for (int k = 0; k < kBlockK / 32; ++k) umma_i8(tmem, moved(w, 2 * k), moved(a, 2 * k), idesc, (i > 0 || k > 0) ? 1u : 0u);
                umma_commit(&tl.empty[s]);
                if (i + 1 == nkb) umma_commit(&tl.done);
            }
            __syncwarp();
            if (++s == S) { s = 0; ph ^= 1u; }
        }
        if (timed_out && elect_one()) {                                 // let every MMA issued so far finish (bounded), then pass the word on
            umma_commit(&tl.drain);
            wait_for(&tl.drain, 0, kWaitLimitNs);
            *reinterpret_cast<volatile int*>(&tl.lost) = 1;
            mbar_arrive(&tl.done);
        }
    } else if (warp < 6) {
        for (int i = threadIdx.x - 64; i < cols; i += 128) tl.a_scale[i] = m0 + i < g.M ? g.a_scale[m0 + i] : 0.f;
    }
    __syncwarp();
    const int q = warp & 3, half = warp >> 2;                           // TMEM lane quarter this warp may read; its share of the columns
    const int n = n0 + q * 32 + lane;
    const float sw = n < g.N ? g.w_scale[n] : 0.f, bias = n < g.N && g.bias != nullptr ? g.bias[n] : 0.f;
    const int RB = cols / splits, mine = m0 + rank * RB;                // rows of A that each CTA of the cluster finishes, a multiple of four; this one's first
    // groups of four of them go to this warp and the one with the same quarter in turn; old values of the first group are asked for ahead of the wait
    DT* const d = (DT*)g.d + (long)mine * g.ldd + n;
    auto old_of = [&](int r, float (&o)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = ADD && n < g.N && r + e < RB && mine + r + e < g.M ? old_value(d + (r + e) * g.ldd) : 0.f;
    };
    float ahead[4] = {0.f, 0.f, 0.f, 0.f};
    float old[32];                                                      // K not shared: of this warp's next strip
    if (splits > 1) {
        old_of(4 * half, ahead);
        cluster_wait();                                                 // every CTA of the cluster runs
    } else if (ADD && half < cols / 32) {                               // (a tile of 32 rows of A has no strip for the second half: those rows are another CTA's)
        load_old<DT>(g, m0 + half * 32, n, old);
    }
    __syncthreads();                                                    // the rows' scales are there
    // (the warp that issued the MMAs frees their TMEM below: it does not go by a caller's shorter limit)
    if (!wait_for(&tl.done, 0, warp == 1 ? max(g.wait_ns, kWaitLimitNs) : g.wait_ns)) timed_out = true;
    timed_out = __any_sync(0xffffffffu, timed_out);                     // tcgen05.ld below is warp-collective
    const bool lost = timed_out || *reinterpret_cast<volatile int*>(&tl.lost) != 0;
    tc_fence_after();
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    if (splits == 1) {
#pragma unroll 1
        for (int cb = half; cb < cols / 32; cb += 2) {
            if (m0 + cb * 32 >= g.M) break;
            if (lost) lose_strip<DT>(g, m0 + cb * 32, n);
            else tile_strip<ADD, DT>(g, lanes + (uint32_t)(cb * 32), tl.a_scale + cb * 32, m0 + cb * 32, n, sw, bias, old, cb + 2 < cols / 32 ? m0 + (cb + 2) * 32 : -1);
        }
    } else {
        if (lost) {
            if (lane == 0)
                for (int c = 0; c < splits; ++c) st_cluster_u32(map_to_rank(smem_u32(&tl.lost), (uint32_t)c), 1u);
        } else {
            const uint32_t slot = smem_u32(part) + (uint32_t)(rank * RB * kWRows + (q * 32 + lane) * 4) * 4u;
#pragma unroll 1
            for (int cb = half; cb < cols / 32; cb += 2) {
                if (m0 + cb * 32 >= g.M) break;
                uint32_t r[32];
                tmem_ld32(lanes + (uint32_t)(cb * 32), r);
#pragma unroll
                for (int j4 = 0; j4 < 32; j4 += 4) {
                    const int b = cb * 32 + j4, to = b / RB;
                    st_cluster_v4(map_to_rank(slot + (uint32_t)(b - to * RB) * (kWRows * 4u), (uint32_t)to), r[j4], r[j4 + 1], r[j4 + 2], r[j4 + 3]);
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
    const bool any_lost = *reinterpret_cast<volatile int*>(&tl.lost) != 0;
    // copies that no MMA waited for land (bounded) before this CTA's memory goes away, whichever of its waits ran out
    if (any_lost && warp == 0)
        for (int i = max(0, issued - S); i < issued; ++i) wait_for(&tl.full[i % S], (uint32_t)(i / S) & 1u, kWaitLimitNs);
    if (splits == 1) return;

    // ---- the rows of A that this CTA finishes
    if (n >= g.N) return;
    for (int r = 4 * half; r < RB; r += 8) {
        if (mine + r >= g.M) break;
        float next[4];
        old_of(r + 8, next);
        const int4* from = reinterpret_cast<const int4*>(part) + (r / 4) * kWRows + q * 32 + lane;
        int4 sum = from[0];
        for (int c = 1; c < splits; ++c) {
            const int4 t = from[c * (RB / 4) * kWRows];
            sum.x += t.x; sum.y += t.y; sum.z += t.z; sum.w += t.w;
        }
        const float4 sa = *reinterpret_cast<const float4*>(tl.a_scale + rank * RB + r);
        const float v[4] = {scaled(sum.x, sa.x, sw, bias), scaled(sum.y, sa.y, sw, bias), scaled(sum.z, sa.z, sw, bias), scaled(sum.w, sa.w, sw, bias)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (mine + r + e < g.M) put_value(d + (r + e) * g.ldd, any_lost ? __uint_as_float(0x7fffffffu) : (ADD ? __fadd_rn(v[e], ahead[e]) : v[e]));
            ahead[e] = next[e];
        }
    }
}

// ---- many rows: pairs of CTAs ------------------------------------------------------------------------
// Two CTAs of a cluster (two SMs) take tiles of 256 rows of W and `cols` rows of A (cta_group::2): each stages its 128 rows of W and half of the rows of A, the
// first one issues the MMAs for both, each finishes its own rows of W.  Persistent, with two accumulators: a tile is finished while the next is multiplied.
// Tiles go in blocks of four tiles of rows of A, rows of W by rows of W within a block, so that both operands come out of L2 (back to back for a second, in blocks of 16 / 8 / 4 / 2:
// 8192 x 2048 x 8448 into an fp32 stream 117 / 114 / 112 / 113 us, 8192 x 8192 x 4096 189 / 192 / 190 / 189, of 64: 135 for the first).
// Warp 0: copies.  Warp 1: TMEM and MMA.  Warps 2 to 9: accumulators, two warps per quarter of the lanes, strips of 32 columns in turn.
//
// Results go through shared memory to tensor-map stores where D's rows allow it, old values of D come the same way, asked for a strip ahead (4096 x 7360 x 1024 into fp32: 51 us; by
// single loads 71).  The arrival that gives an accumulator back is relaxed: as a release it waited for the results to reach memory (4096 x 7360 x 1024 35 -> 29 us).  Copies and MMAs are issued
// by whole warps with one lane elected (29 -> 28 us; 8192 x 8192 x 8192 325 -> 316).
//
// What bounds it, 10^12 operations a second (twice the measured bf16 rate: 3342): 8192 x 8192 x 8192 3520, the tensor cores; 8192 x 2048 x 8448 into an fp32 stream 3020; at short K rounds
// of whole tiles and the results.  A round of 74 tiles of 256 x 256 takes 2.6 us in bf16 at K = 128, whose MMAs take 0.4 at that rate; 3.9 at K = 1024 (3.0); 6.2 at K = 2048 (5.9); in fp32
// 3.5, 4.9 and 7.6.  4096 x 7360 x 1024 is 6.27 such rounds and takes the time of seven: 26 to 27 us (28 with the results of a bf16 strip put one by one), 21 with the results left out,
// of which more than two are the last round, where 20 of 74 pairs have work.  Called back to back for a second, the power limit takes the clock from 1.97 to 1.55 GHz there (32 us) and to 1.3 GHz at long K (8192 x 2048 x 8448: 94 -> 111 us).
constexpr int kPairThreads = 320;
struct PairTail {
    uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
    uint64_t old[8][2];                      // old values of D have arrived in a warp's buffers
    uint32_t tmem_slot, gave_up, issued[2];
    alignas(16) float scales[8][32];
};
static_assert(sizeof(PairTail) <= kTailBytes, "tail of the shared memory");
constexpr int kBlockTiles = 4;

// staged: results (and old values) travel by tensor-map copies, which want D's rows to begin and end on 16-byte boundaries
struct PairShape { int cols, stages, tiles_a, tiles, staged; };
template <typename DT>
constexpr int kStripBytes = 32 * 32 * (int)sizeof(DT);                  // a warp's strip of results; it has two such buffers

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* smem, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(smem_u32(smem)), "r"(x), "r"(y) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// all but the last N stores of this thread have been read from shared memory
template <int N>
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }

template <typename DT>
__global__ void __launch_bounds__(kPairThreads, 1) pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                                                                   const __grid_constant__ CUtensorMap map_d, I8Args g, PairShape sh) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int S = sh.stages, cols = sh.cols, stage = kWBytes + cols / 2 * kBlockK;
    uint8_t* strips = base + S * stage;
    PairTail& tl = *reinterpret_cast<PairTail*>(strips + 16 * kStripBytes<DT>);
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x & 1), first = (int)(blockIdx.x >> 1), at_once = (int)(gridDim.x >> 1);
    const int num_kb = (g.K + kBlockK - 1) / kBlockK, tiles_w = sh.tiles / sh.tiles_a;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(&tl.full[s], 1); mbar_init(&tl.empty[s], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&tl.acc_full[i], 1); mbar_init(&tl.acc_empty[i], 16); }
        for (int i = 0; i < 16; ++i) mbar_init(&tl.old[i >> 1][i & 1], 1);
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
        uint32_t kbg = 0;                                               // k-blocks issued so far, over all tiles
        int s = 0;
        uint32_t ph = 0;
        for (int t = first; t < sh.tiles && !timed_out; t += at_once) {
            if (t == g.skip_unit && rank == 1) break;
            int m0, n0;
            place(t, m0, n0);
            for (int kb = 0; kb < num_kb; ++kb, ++kbg) {
                if (!__all_sync(0xffffffffu, wait_for(&tl.empty[s], ph ^ 1u, g.wait_ns))) { timed_out = true; break; }
                if (elect_one()) {
                    const uint32_t bar = map_to_rank(smem_u32(&tl.full[s]), 0);      // both CTAs' copies complete on the first one's barrier
                    if (rank == 0) mbar_expect_tx(&tl.full[s], 2u * (uint32_t)stage);
                    tma_load_2d_pair(base + s * stage, &map_w, bar, kb * kBlockK, n0 + rank * kWRows);
                    tma_load_2d_pair(base + s * stage + kWBytes, &map_a, bar, kb * kBlockK, m0 + rank * (cols / 2));
                }
                __syncwarp();
                if (++s == S) { s = 0; ph ^= 1u; }
            }
        }
        if (lane == 0) st_cluster_u32(map_to_rank(smem_u32(&tl.issued[rank]), 0), kbg);
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = i8_idesc(2 * kWRows, cols), units = (uint32_t)stage >> 4;
            const uint64_t w0 = make_smem_desc(smem_u32(base)), a0 = make_smem_desc(smem_u32(base) + kWBytes);
            int s = 0;
            uint32_t ph = 0, it = 0;
            for (int t = first; t < sh.tiles && !timed_out; t += at_once, ++it) {
                const uint32_t as = it & 1u, aph = (it >> 1) & 1u, acc = tmem + as * kMaxCols;
                if (!__all_sync(0xffffffffu, wait_for(&tl.acc_empty[as], aph ^ 1u, g.wait_ns))) { timed_out = true; break; }      // this accumulator has been read
                tc_fence_after();
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!__all_sync(0xffffffffu, wait_for(&tl.full[s], ph, g.wait_ns))) { timed_out = true; break; }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t w = moved(w0, (uint32_t)s * units), a = moved(a0, (uint32_t)s * units);
#pragma unroll
                        for (int k = 0; k < kBlockK / 32; ++k) umma_i8_pair(acc, moved(w, 2 * k), moved(a, 2 * k), idesc, (kb > 0 || k > 0) ? 1u : 0u);
                        umma_commit_pair(&tl.empty[s]);
                        if (kb + 1 == num_kb) umma_commit_pair(&tl.acc_full[as]);
                    }
                    __syncwarp();
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
            }
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2, strips_here = (cols / 32 - half + 1) >> 1;
        DT* const buf = reinterpret_cast<DT*>(strips + (warp - 2) * 2 * kStripBytes<DT>);
        uint64_t* const old = tl.old[warp - 2];
        float* const a_scale = tl.scales[warp - 2];
        const bool add = g.accumulate != 0;
        uint32_t it = 0, b = 0, arrivals = 0;                           // b: the buffer of the next strip; arrivals: parity of either buffer's old values
        int waited = 0;                                                 // buffers with old values under way (bits)
        // the old values of strip i of tile t into buffer `to`, which the strip before the last has left
        auto request = [&](int t, int i, uint32_t to) {
            if (t >= sh.tiles) return;
            int m0, n0;
            place(t, m0, n0);
            const int m = m0 + (half + 2 * i) * 32, nw = n0 + rank * kWRows + q * 32;
            if (m >= g.M || nw >= g.N) return;
            waited |= 1 << to;
            if (lane == 0) {
                stores_read<0>();
                mbar_expect_tx(&old[to], (uint32_t)kStripBytes<DT>);
                tma_load_2d(buf + to * 1024, &map_d, &old[to], nw, m);
            }
        };
        // scales and bias of a tile: this lane's row of W, and its rows of A in this warp's strips; asked for while the tile before is finished
        float next_w = 0.f, next_b = 0.f, next_a[kMaxCols / 64];
        auto ask = [&](int t) {
            if (t >= sh.tiles) return;
            int m0, n0;
            place(t, m0, n0);
            const int n = n0 + rank * kWRows + q * 32 + lane;
            next_w = n < g.N ? g.w_scale[n] : 0.f;
            next_b = n < g.N && g.bias != nullptr ? g.bias[n] : 0.f;
#pragma unroll
            for (int i = 0; i < kMaxCols / 64; ++i) {
                const int m = m0 + (half + 2 * i) * 32 + lane;
                next_a[i] = i < strips_here && m < g.M ? g.a_scale[m] : 0.f;
            }
        };
        ask(first);
        if (sh.staged && add) request(first, 0, 0);
        for (int t = first; t < sh.tiles; t += at_once, ++it) {
            const uint32_t as = it & 1u, aph = (it >> 1) & 1u;
            int m0, n0;
            place(t, m0, n0);
            const int nw = n0 + rank * kWRows + q * 32, n = nw + lane;
            const float sw = next_w, bias = next_b;
            float sa[kMaxCols / 64];
#pragma unroll
            for (int i = 0; i < kMaxCols / 64; ++i) sa[i] = next_a[i];
            // after a wait that ran out, this tile and all that follow are left as NaN
            if (!timed_out && ((t == g.give_up && warp == 2 && rank == 1) || !wait_for(&tl.acc_full[as], aph, g.wait_ns))) timed_out = true;
            timed_out = __any_sync(0xffffffffu, timed_out);             // tcgen05.ld is warp-collective
            tc_fence_after();
            const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + as * kMaxCols;
            ask(t + at_once);
            auto column = [&](int i) { return (uint32_t)(half + 2 * i) * 32u; };
            // This warp has read its share of the accumulator.  After a lost wait it stays silent: it runs ahead of the others, and its arrivals would stand in for theirs, so that an
            // accumulator were written that they still read.  The MMAs' wait for it then runs out too.
            auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && !timed_out) mbar_arrive_relaxed(map_to_rank(smem_u32(&tl.acc_empty[as]), 0));
            };
            auto set_scales = [&](int i) {
                __syncwarp();                                           // the last strip's have been read
                a_scale[lane] = i == 0 ? sa[0] : (i == 1 ? sa[1] : (i == 2 ? sa[2] : sa[3]));
                __syncwarp();
            };
            float sw4[4], bias4[4];                                     // bf16: of the rows of W that this lane has in matrices
            if constexpr (sizeof(DT) == 2)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    sw4[k] = __shfl_sync(0xffffffffu, sw, (lane >> 2) + 8 * k);
                    bias4[k] = __shfl_sync(0xffffffffu, bias, (lane >> 2) + 8 * k);
                }
            auto finish = [&](const auto& sum, const auto& high, int i) {
                const int m = m0 + (int)column(i);
                const bool some = m < g.M && nw < g.N;
                set_scales(i);
                if (!timed_out && add) request(i + 1 < strips_here ? t : t + at_once, i + 1 < strips_here ? i + 1 : 0, b ^ 1u);
                else if (lane == 0) stores_read<1>();
                if (some) {
                    if (add) {
                        if (!timed_out && !wait_for(&old[b], (arrivals >> b) & 1u, g.wait_ns)) timed_out = true;
                        timed_out = __any_sync(0xffffffffu, timed_out);
                        if (timed_out) {                                // results of which the old value is missing
                            finish_strip<DT>(g, 0, a_scale, m, n, sw, bias, true);
                            return;
                        }
                        arrivals ^= 1u << b;
                        waited &= ~(1 << b);
                    } else {
                        __syncwarp();                                   // the buffer's last store has been read
                    }
                    if constexpr (sizeof(DT) == 2) {
                        finish_matrices(sum, high, a_scale, sw4, bias4, add, smem_u32(buf + b * 1024), lane);
                    } else {
                        const uint32_t at = smem_u32(buf + b * 1024 + lane);
                        float v[32];
#pragma unroll
                        for (int j = 0; j < 32; j += 4) shared_load4(smem_u32(a_scale), v, j);
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = scaled((int)sum[j], v[j], sw, bias);
                        if (add) {
                            float o[32];
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = shared_value(at + j * 128u);
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = __fadd_rn(v[j], o[j]);
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) shared_put(at + j * 128u, v[j]);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tma_store_2d(&map_d, buf + b * 1024, nw, m);
                    b ^= 1u;
                } else if (add) {
                    b ^= 1u;                                            // its neighbour's old values are on their way into the other buffer
                }
            };
            if (!sh.staged || timed_out) {
                for (int i = 0; i < strips_here; ++i) {
                    const int m = m0 + (int)column(i);
                    set_scales(i);
                    if (m < g.M && nw < g.N) finish_strip<DT>(g, lanes + column(i), a_scale, m, n, sw, bias, timed_out);
                }
                release();
            } else {
#pragma unroll 1
                for (int i = 0; i < strips_here; ++i) {
                    if constexpr (sizeof(DT) == 2) {
                        uint32_t lo[16], hi[16];
                        tmem_ld_16x32(lanes + column(i), lo);
                        tmem_ld_16x32(lanes + (16u << 16) + column(i), hi);
                        tmem_arrived(lo, hi);
                        if (i + 1 == strips_here) release();
                        finish(lo, hi, i);
                    } else {
                        uint32_t sum[32];
                        tmem_ld32(lanes + column(i), sum);
                        if (i + 1 == strips_here) release();
                        finish(sum, sum, i);
                    }
                }
            }
        }
        if (lane == 0) {
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            for (int i = 0; i < 2; ++i) if (waited >> i & 1) wait_for(&old[i], (arrivals >> i) & 1u, kWaitLimitNs);      // (after a lost wait) copies under way
        }
        __syncwarp();
    }
    if (timed_out && g.status != nullptr) atomicOr(g.status, STATUS_TIMEOUT);
    tc_fence_before();
    // neither CTA's memory goes away under the other's MMAs and arrivals
    if (timed_out)
        for (uint32_t r = 0; r < 2; ++r) st_cluster_u32(map_to_rank(smem_u32(&tl.gave_up), r), 1u);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (*reinterpret_cast<volatile uint32_t*>(&tl.gave_up) != 0) {      // ... whoever's wait ran out: the first CTA waits (bounded) for both CTAs' MMAs and copies
        if (rank == 0 && warp == 1) {
            if (elect_one()) {                                          // (the lane that issued the MMAs)
                umma_commit_pair(&tl.drain);
                wait_for(&tl.drain, 0, kWaitLimitNs);
            }
            __syncwarp();
        }
        if (rank == 0 && threadIdx.x == 0) {
            volatile uint32_t* issued = tl.issued;
            const uint32_t i0 = issued[0], i1 = issued[1], lo = min(i0, i1), hi = max(i0, i1);      // at most S apart: neither gets past an unconsumed stage
            for (uint32_t k = lo; k < hi; ++k) {                        // only one CTA issued this block: the barrier expects both halves, or neither
                if (i0 > i1) mbar_complete_tx(&tl.full[k % S], (uint32_t)stage);
                else mbar_expect_tx(&tl.full[k % S], (uint32_t)stage);
            }
            for (uint32_t k = hi > (uint32_t)S ? hi - S : 0; k < hi; ++k) wait_for(&tl.full[k % S], (k / S) & 1u, kWaitLimitNs);
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

int32_t make_map(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, long row_bytes, int rows, int cols, int box_rows, int box_cols, CUtensorMapSwizzle swizzle) {
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
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)row_bytes};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    auto encode_map = [&] {
        return fn(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode_map();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {                // a host thread that has launched nothing yet: its device is chosen, but the driver does not know
        int dev = 0;
        LUMI_CUDA(cudaGetDevice(&dev));
        LUMI_CUDA(cudaSetDevice(dev));
        r = encode_map();
    }
    if (r != CUDA_SUCCESS) return fail(LUMI_E_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d (%d rows of %d)", (int)r, rows, cols);
    return LUMI_OK;
}
// [rows][K] bytes in rows of ld, box of 128 bytes by box_rows, 128-byte swizzle, zeros behind K and behind the last row
int32_t make_i8_map(CUtensorMap* map, const void* ptr, long ld, int rows, int K, int box_rows) {
    return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, ptr, ld, rows, K, box_rows, kBlockK, CU_TENSOR_MAP_SWIZZLE_128B);
}
// D by strips of 32 x 32
template <typename DT>
int32_t make_result_map(CUtensorMap* map, const I8Args& g) {
    return make_map(map, sizeof(DT) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, g.d, g.ldd * (long)sizeof(DT), g.M, g.N, 32, 32,
                    sizeof(DT) == 4 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_64B);
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

// Warps that share K: until the GPU has about 16 warps per SM, as long as each has a piece of a row.
int shares_of_k(long groups, int K, int piece) {
    int shares = 1;
    while (shares < 8 && groups * shares < 16l * sm_count() && K > piece * shares) shares *= 2;
    return shares;
}
template <typename DT>
int32_t launch_few(const I8Args& g, cudaStream_t st) {
    const bool one_or_two = g.M <= 2;
    const int per_warp = one_or_two ? kVecRows : kFewW, shares = shares_of_k(((long)g.N + per_warp - 1) / per_warp, g.K, one_or_two ? 512 : 64);
    const long rows = 8 / shares * per_warp;
    Launch l(dim3((unsigned)((g.N + rows - 1) / rows)), 256, 0, 1, st);
    if (g.M == 1) LUMI_CUDA(cudaLaunchKernelEx(&l.cfg, vector_kernel<1, DT>, g, shares));
    else if (one_or_two) LUMI_CUDA(cudaLaunchKernelEx(&l.cfg, vector_kernel<2, DT>, g, shares));
    else LUMI_CUDA(cudaLaunchKernelEx(&l.cfg, few_kernel<DT>, g, shares));
    return LUMI_OK;
}

// Tile and shares of K for a product whose tiles fit on the GPU at once (cols 0: they do not).  The estimate, in microseconds behind what every launch
// takes: 0.19 per k-block, and for the results, or for sums that cross the cluster's shared memory, by the tile's width and the number of CTAs.  Measured, columns /
// shares (CTAs): 16 x 7360 x 1024 32/1 (58) 4.6, 32/2 (116) 5.6; 64 x 1024 x 2816 32/2 (32) 5.4, 32/4 (64) 4.4, 32/8 (128) 4.8, 64/4 (32) 5.3; 512 x 1024 x 2816 32/1 (128) 7.1, 64/2 (128)
// 9.0; 512 x 259 x 8192 32/2 (96) 11.9, 64/4 (96) 9.9; 512 x 5632 x 2048 192/1 (132) 9.2, 256/1 (88) 10.9.  A second round of CTAs costs more than the first: 256 x 7360 x 1024 128/1
// (116) 6.3, 32/1 (464) 16.5, 128/2 (232) 18.3.
TileShape tile_shape(const I8Args& g) {
    const int num_kb = (g.K + kBlockK - 1) / kBlockK;
    const long tiles = ((long)g.N + kWRows - 1) / kWRows;
    TileShape best{0, 0, 1};
    double least = 0;
    for (int cols = 32; cols <= kMaxCols; cols += 32) {
        const long whole = tiles * ((g.M + cols - 1) / cols);
        if (whole > sm_count()) continue;
        for (int splits = 1; splits <= 8; splits *= 2) {
            if (splits > 1 && (cols > 128 || splits > num_kb || whole * splits > kClusterCtas)) break;
            const double cost = 0.19 * ((num_kb + splits - 1) / splits) + (splits > 1 ? 0.2 + 0.025 * cols + 0.012 * (double)(whole * splits) : 0.008 * cols);
            if (best.cols == 0 || cost < least) { best.cols = cols; best.splits = splits; least = cost; }
        }
    }
    if (best.cols == 0) return best;
    const long ctas = tiles * ((g.M + best.cols - 1) / best.cols) * best.splits;
    // clusters find room beside one another where a CTA leaves half an SM
    const int stage = kWBytes + best.cols * kBlockK, part = best.splits > 1 ? best.cols * kWRows * 4 : 0;
    const int budget = (best.splits > 1 && ctas > 64 ? 112 : 220) * 1024 - part - kTailBytes - 1024;
    best.stages = std::max(2, std::min({kMaxStages, budget / stage, (num_kb + best.splits - 1) / best.splits}));
    return best;
}

template <typename DT, bool ADD>
int32_t launch_tile(const I8Args& g, const TileShape& sh, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    CUtensorMap ma, mw;
    LUMI_TRY(make_i8_map(&ma, g.a, g.lda, g.M, g.K, sh.cols));
    LUMI_TRY(make_i8_map(&mw, g.w, g.ldw, g.N, g.K, kWRows));
    LUMI_TRY(allow_smem((const void*)tile_kernel<DT, ADD>, ready));
    const int part = sh.splits > 1 ? sh.cols * kWRows * 4 : 0;
    Launch l(dim3((unsigned)((g.N + kWRows - 1) / kWRows * sh.splits), (unsigned)((g.M + sh.cols - 1) / sh.cols)), 256,
             sh.stages * (kWBytes + sh.cols * kBlockK) + part + kTailBytes + 1024, sh.splits, st);
    LUMI_CUDA(cudaLaunchKernelEx(&l.cfg, tile_kernel<DT, ADD>, ma, mw, g, sh));
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
    sh.stages = std::min(kMaxStages, (227 * 1024 - 1024 - kTailBytes - 16 * kStripBytes<DT>) / stage);
    // (a store is cut at the end of a row by whole 16 bytes)
    sh.staged = ((uintptr_t)g.d & 15) == 0 && g.ldd * sizeof(DT) % 16 == 0 && g.N * sizeof(DT) % 16 == 0;
    CUtensorMap ma, mw, md{};
    if (sh.staged) LUMI_TRY(make_result_map<DT>(&md, g));
    LUMI_TRY(make_i8_map(&ma, g.a, g.lda, g.M, g.K, cols / 2));
    LUMI_TRY(make_i8_map(&mw, g.w, g.ldw, g.N, g.K, kWRows));
    LUMI_TRY(allow_smem((const void*)pair_kernel<DT>, ready));
    Launch l(dim3(2 * std::min(sh.tiles, sm_count() / 2)), kPairThreads, sh.stages * stage + 16 * kStripBytes<DT> + kTailBytes + 1024, 2, st);
    LUMI_CUDA(cudaLaunchKernelEx(&l.cfg, pair_kernel<DT>, ma, mw, md, g, sh));
    return LUMI_OK;
}

// Columns of the pairs' tiles: the GPU works in rounds of a tile per pair, a round costs about its tile's columns.
int pair_cols(const I8Args& g) {
    const long pairs = sm_count() / 2, tiles_w = (g.N + 2 * kWRows - 1) / (2 * kWRows);
    int best = 0;
    long cost = 0;
    for (int c = kMaxCols; c >= 64; c -= 32) {
        const long k = (tiles_w * ((g.M + c - 1) / c) + pairs - 1) / pairs * (c + 32);
        if (best == 0 || k < cost) { best = c; cost = k; }
    }
    return best;
}

template <typename DT>
int32_t launch_product(const I8Args& g, cudaStream_t st) {
    if (g.M <= 2 || (g.M <= kFewRows && g.K <= kFewK && (long)g.N * g.K <= kFewBytes)) return launch_few<DT>(g, st);
    const TileShape sh = tile_shape(g);
    if (sh.cols == 0) return launch_pair<DT>(g, pair_cols(g), st);
    return g.accumulate ? launch_tile<DT, true>(g, sh, st) : launch_tile<DT, false>(g, sh, st);
}

}  // namespace
}  // namespace lumi

using namespace lumi;

static int32_t check_and_run(const char* name, uint64_t a, int32_t lda, uint64_t a_scale, uint64_t w, int32_t ldw, uint64_t w_scale, uint64_t bias, uint64_t d,
                             int32_t d_dtype, int32_t ldd, int32_t M, int32_t N, int32_t K, int32_t accumulate, uint64_t status, uint64_t wait_ns, int skip_unit,
                             cudaStream_t st) {
    if (!a || !a_scale || !w || !w_scale || !d || M < 0 || N < 0 || K <= 0 || lda < K || ldw < K || ldd < N ||
        (d_dtype != LUMI_DTYPE_F32 && d_dtype != LUMI_DTYPE_BF16))
        return fail(LUMI_E_INVALID, "bad argument to %s", name);
    if ((a & 15) || (w & 15) || lda % 16 || ldw % 16 || ((a_scale | w_scale | bias | status) & 3) || (d & (d_dtype == LUMI_DTYPE_F32 ? 3 : 1)))
        return fail(LUMI_E_INVALID, "%s: rows of A and W have to begin on 16-byte boundaries, numbers on their own", name);
    // 131071 products of -128 and -128 are the most that a 32-bit sum holds
    if (K > 131071 || M > kMaxRows || N > kMaxRows) return fail(LUMI_E_UNSUPPORTED, "%s: M %d, N %d (at most %d), K %d (at most 131071)", name, M, N, kMaxRows, K);
    if (M == 0 || N == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory(name, {a, a_scale, w, w_scale, bias, d, status}));
    const I8Args g{(const int8_t*)a, (const int8_t*)w, (const float*)a_scale, (const float*)w_scale, (const float*)bias, (void*)d, lda, ldw, ldd, M, N, K, accumulate,
                   (int32_t*)status, wait_ns, skip_unit, skip_unit < -1 ? -2 - skip_unit : -1};
    return d_dtype == LUMI_DTYPE_F32 ? launch_product<float>(g, st) : launch_product<__nv_bfloat16>(g, st);
}

extern "C" int32_t lumi_k_gemm_i8(uint64_t a, int32_t lda, uint64_t a_scale, uint64_t w, int32_t ldw, uint64_t w_scale, uint64_t bias, uint64_t d,
                                  int32_t d_dtype, int32_t ldd, int32_t M, int32_t N, int32_t K, int32_t accumulate, uint64_t status, uint64_t stream) {
    return check_and_run("lumi_k_gemm_i8", a, lda, a_scale, w, ldw, w_scale, bias, d, d_dtype, ldd, M, N, K, accumulate, status, kWaitLimitNs, -1, (cudaStream_t)stream);
}

// Failure-path test hook: waits limited by the caller and a tile whose operands (a pair: the second CTA's) never arrive, or (skip_unit < -1) one wait that runs out at once.
extern "C" int32_t lumi_debug_gemm_i8_wait_timeout(uint64_t a, int32_t lda, uint64_t a_scale, uint64_t w, int32_t ldw, uint64_t w_scale, uint64_t d, int32_t d_dtype,
                                                   int32_t ldd, int32_t M, int32_t N, int32_t K, int32_t accumulate, uint64_t wait_limit_ns, int32_t skip_unit,
                                                   uint64_t status) {
    if (!status || !wait_limit_ns) return fail(LUMI_E_INVALID, "bad argument to lumi_debug_gemm_i8_wait_timeout");
    LUMI_TRY(check_and_run("lumi_debug_gemm_i8_wait_timeout", a, lda, a_scale, w, ldw, w_scale, 0, d, d_dtype, ldd, M, N, K, accumulate, status, wait_limit_ns,
                           skip_unit, nullptr));
    int32_t word = 0;
    LUMI_CUDA(cudaMemcpy(&word, (const void*)status, sizeof(word), cudaMemcpyDeviceToHost));
    return (word & STATUS_TIMEOUT) ? fail(LUMI_E_TIMEOUT, "a bounded wait of the 8-bit product ran out") : LUMI_OK;
}
