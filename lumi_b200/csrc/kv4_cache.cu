// A paged cache of keys and values in 4 bits: page tables and slots from the lengths of requests, rows into the cache, rows back.
//
// A group of up to 32 numbers t of a token and head has the scale s = m (1 / 7) (an fp32 product with 1 / 7 in fp32) rounded up to bf16, m = max(max |t|, 2^-100), and codes
// n = 8 + rint(t / s) in 1 .. 15.  Rounding the scale up keeps |t / s| <= 7 but for a rounding, so nothing is cut off and t is off by s / 2 at most.  (n - 8) s has 3 + 8 significant bits: exact in fp32 and, scaled, in fp16.  A group that holds an infinity
// or a NaN gets codes 8 and s = NaN.
#include "device_args.h"
#include "kv4.cuh"
#include "rows.cuh"

#include <algorithm>

namespace lumi {
namespace {

constexpr float kLeast = 7.888609052210118e-31f;           // 2^-100
constexpr int kMaxSeqs = 8192;                             // of a plan: its prefix sums lie in shared memory
constexpr int kPlanThreads = 1024, kPlanCtas = 8;

void dependent(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, dim3 grid, int threads, size_t smem, cudaStream_t st) {
    cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // the launch itself overlaps the kernel in front
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
}

// ---- plan ------------------------------------------------------------------------------------------------------
// Every CTA takes the prefix sums over all sequences itself (they are few numbers), so that nothing has to pass between CTAs: as many run as there are rows for.  Where results lie where
// inputs lie they are a cluster of eight at most, and a barrier keeps them from being written before all have read.  Then each row finds its sequence by bisection in shared memory.
// Bound by latency (chains of loads, sums and barriers): 256 sequences of a token each 4.7 us; 2048 sequences and 57000 rows 7.6 us, in place 19 us; the launch alone is about 2.
//
// Free pages are a stack; the pages of requests that end lie on top of it, in the order of sequences, and new pages are taken from the top.  Taken are either pages that came back
// in this call and all of those, then older ones, or some of those that came back: entries that are read lie below the old count, and entries that are written above.
struct PlanArgs {
    const int32_t *tokens, *len, *pool;
    int32_t *table, *free, *pool_after, *tokens_after, *row_start, *pos, *slot;
    int nseq, width, n_pages, rows;
};
struct PlanSums { long long rows, taken, given; };

__device__ __forceinline__ int last_at_most(const int* a, int n, int v) {      // of ascending a[0 .. n), a[0] <= v: the last place with a[i] <= v
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid; else hi = mid;
    }
    return lo;
}

// TOGETHER: results lie where inputs lie; the CTAs are a cluster.
template <bool TOGETHER>
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PlanArgs a) {
    extern __shared__ int sm[];
    int* const held = sm;                                  // tokens before
    int* const row_at = held + a.nseq;                     // prefix sums: rows, pages taken, pages given back
    int* const take_at = row_at + a.nseq + 1;
    int* const give_at = take_at + a.nseq + 1;
    __shared__ PlanSums warp_sums[kPlanThreads / 32];
    __shared__ int bad_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_release();
    if (tid == 0) bad_s = 0;
    pdl_sync();
    __syncthreads();
    const int n_free = a.pool[0], status = a.pool[1];
    const int each = (a.nseq + kPlanThreads - 1) / kPlanThreads, s0 = min(a.nseq, tid * each), s1 = min(a.nseq, s0 + each);
    PlanSums sum = {0, 0, 0};
    int bad = 0;
    auto of = [&](int h, int n, PlanSums& p) {             // one sequence's part of the sums
        const int before = (int)(((long long)h + kPage - 1) / kPage);
        if (n < 0) { p = {0, 0, before}; return; }
        p = {n, ((long long)h + n + kPage - 1) / kPage - before, 0};
    };
    for (int s = s0; s < s1; ++s) {
        const int h = a.tokens[s], n = a.len[s];
        held[s] = h;
        if (h < 0 || (long long)h + max(n, 0) > (long long)a.width * kPage) { bad |= 2; continue; }
        PlanSums p;
        of(h, n, p);
        sum.rows += p.rows; sum.taken += p.taken; sum.given += p.given;
    }
    PlanSums run = sum;                                    // inclusive over the warp, then over warps
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long r = __shfl_up_sync(0xffffffffu, run.rows, o), t = __shfl_up_sync(0xffffffffu, run.taken, o), g = __shfl_up_sync(0xffffffffu, run.given, o);
        if (lane >= o) { run.rows += r; run.taken += t; run.given += g; }
    }
    if (lane == 31) warp_sums[warp] = run;
    if (bad) atomicOr(&bad_s, bad);
    __syncthreads();
    PlanSums total = {0, 0, 0}, at = {run.rows - sum.rows, run.taken - sum.taken, run.given - sum.given};
#pragma unroll 4
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        const PlanSums p = warp_sums[w];
        if (w < warp) { at.rows += p.rows; at.taken += p.taken; at.given += p.given; }
        total.rows += p.rows; total.taken += p.taken; total.given += p.given;
    }
    bad = bad_s;
    if (n_free < 0 || n_free > a.n_pages || total.taken > n_free + total.given || n_free + total.given - total.taken > a.n_pages) bad |= 1;
    if (total.rows > a.rows) bad |= 4;
    for (int s = s0; s < s1; ++s) {
        const int n = a.len[s];
        row_at[s] = (int)at.rows; take_at[s] = (int)at.taken; give_at[s] = (int)at.given;
        PlanSums p = {0, 0, 0};
        if (bad == 0) of(held[s], n, p);
        at.rows += p.rows; at.taken += p.taken; at.given += p.given;
        if (blockIdx.x == 0) a.row_start[s] = bad ? 0 : row_at[s];
    }
    if (tid == 0) {
        row_at[a.nseq] = (int)total.rows; take_at[a.nseq] = (int)total.taken; give_at[a.nseq] = (int)total.given;
        if (blockIdx.x == 0) a.row_start[a.nseq] = bad ? 0 : (int)total.rows;
    }
    __syncthreads();
    if constexpr (TOGETHER) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (blockIdx.x == 0) {
        for (int s = s0; s < s1; ++s) {
            const bool gone = give_at[s + 1] > give_at[s];
            a.tokens_after[s] = bad ? held[s] : gone ? 0 : held[s] + row_at[s + 1] - row_at[s];
        }
        if (tid == 0) {
            a.pool_after[0] = bad ? n_free : (int)(n_free + total.given - total.taken);
            a.pool_after[1] = status | bad;
        }
    }
    const int n_rows = bad ? 0 : (int)total.rows, given = (int)total.given, taken = (int)total.taken, step = gridDim.x * kPlanThreads;
    auto given_page = [&](int i) {                         // the i-th page that comes back
        const int s = last_at_most(give_at, a.nseq, i);
        return a.table[(size_t)s * a.width + (i - give_at[s])];
    };
    for (int r = blockIdx.x * kPlanThreads + tid; r < a.rows; r += step) {
        int pos = -1, slot = -1;
        if (r < n_rows) {
            const int s = last_at_most(row_at, a.nseq, r), h = held[s];
            pos = h + r - row_at[s];
            const int i = pos / kPage, before = (h + kPage - 1) / kPage;
            int32_t* const entry = a.table + (size_t)s * a.width + i;
            int page;
            if (i < before) page = *entry;
            else {
                const int v = n_free + given - 1 - (take_at[s] + i - before);
                page = v < n_free ? a.free[v] : given_page(v - n_free);
                if (pos % kPage == 0) *entry = page;
            }
            slot = page >= 0 && page < a.n_pages ? page * kPage + pos % kPage : -1;
        }
        a.pos[r] = pos;
        a.slot[r] = slot;
    }
    if (bad == 0)
        for (int i = blockIdx.x * kPlanThreads + tid; i < given - taken; i += step) a.free[n_free + i] = given_page(i);
}

// ---- rows into the cache, and back ---------------------------------------------------------------------------------
// A warp takes one group of a head, of eight rows at a time, four lanes a row: eight numbers each, one word of codes.  Rows of a prompt are neighbouring tokens of a page, so that a
// warp's words are 128 bytes in a row and its scales 16.  kDeep eights of rows per warp where there are many: their loads are under way together, and what a group's place costs in
// arithmetic is shared.  Bound by memory where rows are many: 65536 rows of 4 fp32 heads of 64 + 64 both ways 61 us, 309 MB at 5.1 TB/s (one eight of rows per warp: 90 us); 64 rows of 8 bf16
// heads of 128 + 128 both ways 3.1 us, two launches.
constexpr float kSeventh = 0.14285715f;                    // 1 / 7 rounded to fp32, which is above it: numbers of a group are at most 7 steps
constexpr int kDeep = 4;
constexpr int kManyRows = 4096;                            // rows from which on warps take kDeep eights
struct RowsArgs {
    const void *k, *v;
    void *k_out, *v_out;
    const int32_t* slot;
    uint8_t* kv;
    long ldk, ldv;
    int n_slots, heads, dk, dv, rows;
    int split;                                             // log2 of the groups that a block of eight warps takes; its warps share rows by the rest
};
// One group of a head: where it lies in a page and in a row.
struct Place { size_t page_bytes; int codes, scale, d, column; bool keys, any; };
__device__ __forceinline__ Place place_of(const RowsArgs& a, int quarter) {
    const int gk = kv4_groups(a.dk), gv = kv4_groups(a.dv), block = kv4_block(a.dk, a.dv);
    const int item = (blockIdx.y << a.split) + ((threadIdx.x >> 5) & ((1 << a.split) - 1));      // [head][groups of keys, then of values]
    const int head = item / (gk + gv), i = item - head * (gk + gv);
    Place p;
    p.any = head < a.heads;
    p.keys = i < gk;
    const int g = p.keys ? i : i - gk, part = head * block + (p.keys ? 0 : kv4_part(a.dk)), first = g * kGroup + quarter * 8;
    p.page_bytes = (size_t)a.heads * block;
    p.codes = part + g * kPlane + quarter * 4;
    p.scale = part + (p.keys ? gk : gv) * kPlane + g * kScales;
    p.d = (p.keys ? a.dk : a.dv) - first;                  // numbers that the head has from here on
    p.column = head * (p.keys ? a.dk : a.dv) + first;
    return p;
}
template <int DEEP>
__device__ __forceinline__ long first_row(const RowsArgs& a) {
    return (((long)blockIdx.x << (3 - a.split)) + (threadIdx.x >> (5 + a.split))) * (8 * DEEP) + ((threadIdx.x & 31) >> 2);
}
// Where number e of a lane's eight lies in its word, as a shift.
__device__ __forceinline__ int nibble_shift(bool keys, int e) { return 4 * (keys ? (e >> 1) + 4 * (e & 1) : e); }

// WHOLE: eight numbers lie on a 16-byte boundary and end with the head at the earliest
template <typename T, bool WHOLE>
__device__ __forceinline__ void load8(const T* p, int n, float (&t)[8]) {
    if constexpr (WHOLE) {
        if (n > 0) {
            if constexpr (sizeof(T) == 4) {
                const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
                t[0] = x.x; t[1] = x.y; t[2] = x.z; t[3] = x.w; t[4] = y.x; t[5] = y.y; t[6] = y.z; t[7] = y.w;
            } else {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) { t[2 * i] = __uint_as_float(u[i] << 16); t[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = !WHOLE && i < n ? (float)p[i] : 0.f;
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void store8(T* p, int n, const float (&t)[8]) {
    if constexpr (WHOLE) {
        if (n <= 0) return;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(t[0], t[1], t[2], t[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(t[4], t[5], t[6], t[7]);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(t[2 * i], t[2 * i + 1]);
                u[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < n) p[i] = (T)t[i];
    }
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

template <typename T, bool WHOLE, int DEEP>
__global__ void __launch_bounds__(256) kv4_append_kernel(RowsArgs a) {
    const int lane = threadIdx.x & 31;
    const Place p = place_of(a, lane & 3);
    const long row0 = first_row<DEEP>(a);
    pdl_release();
    pdl_sync();
    if (!p.any) return;                                    // (the whole warp)
    const T* const from = p.keys ? (const T*)a.k : (const T*)a.v;
    const long ld = p.keys ? a.ldk : a.ldv;
    int slot[DEEP];
    float t[DEEP][8];
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
        const long row = row0 + 8 * k;
        slot[k] = row < a.rows ? a.slot[row] : -1;
        if (slot[k] >= a.n_slots) slot[k] = -1;
    }
#pragma unroll
    for (int k = 0; k < DEEP; ++k) load8<T, WHOLE>(from + (row0 + 8 * k) * ld + p.column, slot[k] >= 0 ? p.d : 0, t[k]);
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
        float m = fabsf(t[k][0]);                          // the largest; infinities and NaN stay
#pragma unroll
        for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(t[k][i]));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const bool numbers = m < INFINITY;
        const uint32_t up = numbers ? (__float_as_uint(__fmul_rn(fmaxf(m, kLeast), kSeventh)) + 0xffffu) & 0xffff0000u : 0x7fc00000u;
        const float s = __uint_as_float(up), inv = __frcp_rn(s);
        // 8 + rint(t / s) by way of t (1 / s), which is the quotient to 2^-20: the low half of a sum at 1.5 2^23.  Beside a half, where that might round the other way, the quotient itself.
        float x[8], off = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = fmaf(t[k][i], inv, 12582920.f);
            off = fmaxf(off, fabsf(fmaf(t[k][i], inv, 12582920.f - x[i])));
        }
        if (numbers && off > 0.49999f) {
            if constexpr (sizeof(T) == 2) {
                // bf16 numbers are often exactly half a step off, and else further from it than a quotient rounds: what is left of t decides, which is exact
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float left = fmaf(12582920.f - x[i], s, t[k][i]), over = fabsf(left) - 0.5f * s;
                    if (over > 0.f || (over == 0.f && (__float_as_uint(x[i]) & 1u))) x[i] += copysignf(1.f, left);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = 12582920.f + rintf(__fdiv_rn(t[k][i], s));
            }
        }
        // two codes side by side in halves, four such pairs four bits apart: numbers 2 i and 2 i + 1 of keys, i and i + 4 of values
        uint32_t word = 0;
#pragma unroll
        for (int i = 3; i >= 0; --i)
            word = word * 16 + (p.keys ? __byte_perm(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]), 0x5410) : __byte_perm(__float_as_uint(x[i]), __float_as_uint(x[i + 4]), 0x5410));
        if (!numbers) word = 0x88888888u;
        if (slot[k] < 0) continue;
        uint8_t* const page = a.kv + (size_t)(slot[k] / kPage) * p.page_bytes;
        *reinterpret_cast<uint32_t*>(page + p.codes + slot[k] % kPage * 16) = word;
        if ((lane & 3) == 0) *reinterpret_cast<uint16_t*>(page + p.scale + slot[k] % kPage * 2) = (uint16_t)(up >> 16);
    }
}

// The low nibble's code under the exponent of 2^23, less 2^23 + 8, times s.
__device__ __forceinline__ float code_times(uint32_t w, float s) { return (__uint_as_float((w & 15u) | 0x4b000000u) - 8388616.f) * s; }

template <typename T, bool WHOLE, int DEEP>
__global__ void __launch_bounds__(256) kv4_read_kernel(RowsArgs a) {
    const int lane = threadIdx.x & 31;
    const Place p = place_of(a, lane & 3);
    const long row0 = first_row<DEEP>(a);
    pdl_release();
    pdl_sync();
    if (!p.any) return;
    T* const to = p.keys ? (T*)a.k_out : (T*)a.v_out;
    const long ld = p.keys ? a.ldk : a.ldv;
    int slot[DEEP];
    uint32_t word[DEEP], scale[DEEP];
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
        const long row = row0 + 8 * k;
        slot[k] = row < a.rows ? a.slot[row] : -1;
        if (slot[k] >= a.n_slots) slot[k] = -1;
    }
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
        word[k] = scale[k] = 0;
        if (slot[k] < 0) continue;
        const uint8_t* const page = a.kv + (size_t)(slot[k] / kPage) * p.page_bytes;
        word[k] = *reinterpret_cast<const uint32_t*>(page + p.codes + slot[k] % kPage * 16);
        scale[k] = *reinterpret_cast<const uint16_t*>(page + p.scale + slot[k] % kPage * 2);
    }
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
        const float s = __uint_as_float(scale[k] << 16);
        if constexpr (WHOLE && sizeof(T) == 4) {
            // 32 numbers are 128 bytes: each store takes 16 of them per lane side by side, numbers 4 q .. and 16 + 4 q .., whose words neighbours hold
            const int q = lane & 3, back = (q & 1) * (p.keys ? 8 : 16);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t w = __shfl_sync(0xffffffffu, word[k], (lane & 28) + 2 * h + (q >> 1)) >> back;
                float t[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] = code_times(w >> nibble_shift(p.keys, i), s);
                const int at = 16 * h + 4 * q - 8 * q;     // from the lane's own first number
                if (slot[k] >= 0 && at < p.d) *reinterpret_cast<float4*>(to + (row0 + 8 * k) * ld + p.column + at) = make_float4(t[0], t[1], t[2], t[3]);
            }
        } else {
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = code_times(word[k] >> nibble_shift(p.keys, i), s);
            if (slot[k] >= 0) store8<T, WHOLE>(to + (row0 + 8 * k) * ld + p.column, p.d, t);
        }
    }
}

bool whole(uint64_t p, int ld, int d, int dtype) { const int e = dtype == LUMI_DTYPE_F32 ? 4 : 2; return (p & 15) == 0 && (long)ld * e % 16 == 0 && d % 8 == 0; }

int32_t check_cache(const char* name, uint64_t kv, int n_pages, int kv_heads, int dk, int dv) {
    if (!kv || n_pages <= 0 || kv_heads <= 0 || dk <= 0 || dv <= 0) return fail(LUMI_E_INVALID, "bad argument to %s", name);
    if (kv & 15) return fail(LUMI_E_INVALID, "%s: the cache has to begin on a 16-byte boundary", name);
    if (dk > kMaxHead || dv > kMaxHead || n_pages > kMaxPages || kv_heads > 65535)
        return fail(LUMI_E_UNSUPPORTED, "%s: heads of %d and %d numbers (at most %d), %d heads, %d pages (at most %d)", name, dk, dv, kMaxHead, kv_heads, n_pages, kMaxPages);
    return LUMI_OK;
}
bool known(int dtype) { return dtype == LUMI_DTYPE_F32 || dtype == LUMI_DTYPE_BF16; }

template <bool READ>
int32_t rows_call(const char* name, RowsArgs a, int dtype, bool fits, cudaStream_t st) {
    const int items = a.heads * (kv4_groups(a.dk) + kv4_groups(a.dv)), deep = a.rows >= kManyRows ? kDeep : 1;
    a.split = items >= 8 ? 3 : items >= 4 ? 2 : 1;         // (there are two groups at least)
    const long rows_per_block = 8l * deep << (3 - a.split), blocks = ((long)a.rows + rows_per_block - 1) / rows_per_block, across = ((long)items + (1 << a.split) - 1) >> a.split;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[1];
    dependent(cfg, attr, dim3((unsigned)blocks, (unsigned)across), 256, 0, st);
    auto of_depth = [&](auto t, auto w, auto d) {
        using T = decltype(t);
        if constexpr (READ) return cudaLaunchKernelEx(&cfg, kv4_read_kernel<T, decltype(w)::value, decltype(d)::value>, a);
        else return cudaLaunchKernelEx(&cfg, kv4_append_kernel<T, decltype(w)::value, decltype(d)::value>, a);
    };
    auto go = [&](auto t, auto w) { return deep == 1 ? of_depth(t, w, std::integral_constant<int, 1>()) : of_depth(t, w, std::integral_constant<int, kDeep>()); };
    using Yes = std::integral_constant<bool, true>;
    using No = std::integral_constant<bool, false>;
    if (dtype == LUMI_DTYPE_F32) LUMI_CUDA(fits ? go(float(), Yes()) : go(float(), No()));
    else LUMI_CUDA(fits ? go(__nv_bfloat16(), Yes()) : go(__nv_bfloat16(), No()));
    return LUMI_OK;
}

int32_t check_rows(const char* name, uint64_t k, int ldk, uint64_t v, int ldv, int dtype, uint64_t slot, uint64_t kv, int n_pages, int kv_heads, int dk, int dv, int rows) {
    if (!k || !v || !slot || !known(dtype) || rows < 0) return fail(LUMI_E_INVALID, "bad argument to %s", name);
    LUMI_TRY(check_cache(name, kv, n_pages, kv_heads, dk, dv));
    if ((long)kv_heads * (kv4_groups(dk) + kv4_groups(dv)) > 8 * 65535) return fail(LUMI_E_UNSUPPORTED, "%s: %d heads of %d and %d numbers", name, kv_heads, dk, dv);      // a launch's second axis
    if (ldk < (long)kv_heads * dk || ldv < (long)kv_heads * dv) return fail(LUMI_E_INVALID, "%s: rows hold %d heads of %d and %d numbers", name, kv_heads, dk, dv);
    if (((k | v) & (dtype == LUMI_DTYPE_F32 ? 3 : 1)) || (slot & 3)) return fail(LUMI_E_INVALID, "%s: numbers have to lie on their own boundaries", name);
    return LUMI_OK;
}

}  // namespace
}  // namespace lumi

using namespace lumi;

extern "C" int32_t lumi_k_kv4_page_bytes(int32_t kv_heads, int32_t dk, int32_t dv, int64_t* bytes) {
    if (!bytes || kv_heads <= 0 || dk <= 0 || dv <= 0) return fail(LUMI_E_INVALID, "bad argument to lumi_k_kv4_page_bytes");
    if (dk > kMaxHead || dv > kMaxHead || kv_heads > 65535)
        return fail(LUMI_E_UNSUPPORTED, "lumi_k_kv4_page_bytes: %d heads of %d and %d numbers (at most %d)", kv_heads, dk, dv, kMaxHead);
    *bytes = (int64_t)kv_heads * kv4_block(dk, dv);
    return LUMI_OK;
}

extern "C" int32_t lumi_k_page_plan(uint64_t tokens, uint64_t len, int32_t nseq, uint64_t page_table, int32_t pages_per_seq, uint64_t free_pages, int32_t n_pages, uint64_t pool,
                                    uint64_t pool_after, uint64_t tokens_after, uint64_t row_start, uint64_t pos, uint64_t slot, int32_t rows, uint64_t stream) {
    if (!tokens || !len || !page_table || !free_pages || !pool || !pool_after || !tokens_after || !row_start || !pos || !slot || nseq < 0 || pages_per_seq <= 0 ||
        n_pages <= 0 || rows < 0)
        return fail(LUMI_E_INVALID, "bad argument to lumi_k_page_plan");
    if ((tokens | len | page_table | free_pages | pool | pool_after | tokens_after | row_start | pos | slot) & 3)
        return fail(LUMI_E_INVALID, "lumi_k_page_plan: arrays of 32-bit numbers have to lie on 4-byte boundaries");
    if (nseq > kMaxSeqs || n_pages > kMaxPages || pages_per_seq > kMaxPages)
        return fail(LUMI_E_UNSUPPORTED, "lumi_k_page_plan: %d sequences (at most %d), %d pages (at most %d)", nseq, kMaxSeqs, n_pages, kMaxPages);
    LUMI_TRY(check_device_memory("lumi_k_page_plan", {tokens, len, page_table, free_pages, pool, pool_after, tokens_after, row_start, pos, slot}));
    const PlanArgs a{(const int32_t*)tokens, (const int32_t*)len, (const int32_t*)pool, (int32_t*)page_table, (int32_t*)free_pages, (int32_t*)pool_after, (int32_t*)tokens_after,
                     (int32_t*)row_start, (int32_t*)pos, (int32_t*)slot, nseq, pages_per_seq, n_pages, rows};
    const size_t smem = sizeof(int) * (4 * (size_t)nseq + 3);
    const bool together = pool == pool_after || tokens == tokens_after;
    const auto kernel = together ? page_plan_kernel<true> : page_plan_kernel<false>;
    if (smem > 48 * 1024) LUMI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    const int wanted = std::max(1, (rows + kPlanThreads - 1) / kPlanThreads);
    const int ctas = together ? (wanted > 2 ? kPlanCtas : 1) : std::min(wanted, sm_count());
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    dependent(cfg, attr, dim3(ctas), kPlanThreads, smem, (cudaStream_t)stream);
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)(together ? ctas : 1);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
    LUMI_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
    return LUMI_OK;
}

extern "C" int32_t lumi_k_kv4_append(uint64_t k, int32_t ldk, uint64_t v, int32_t ldv, int32_t dtype, uint64_t slot, uint64_t kv, int32_t n_pages, int32_t kv_heads, int32_t dk,
                                     int32_t dv, int32_t rows, uint64_t stream) {
    LUMI_TRY(check_rows("lumi_k_kv4_append", k, ldk, v, ldv, dtype, slot, kv, n_pages, kv_heads, dk, dv, rows));
    if (rows == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory("lumi_k_kv4_append", {k, v, slot, kv}));
    const RowsArgs a{(const void*)k, (const void*)v, nullptr, nullptr, (const int32_t*)slot, (uint8_t*)kv, ldk, ldv, n_pages * kPage, kv_heads, dk, dv, rows, 0};
    return rows_call<false>("lumi_k_kv4_append", a, dtype, whole(k, ldk, dk, dtype) && whole(v, ldv, dv, dtype), (cudaStream_t)stream);
}

extern "C" int32_t lumi_k_kv4_read(uint64_t kv, int32_t n_pages, uint64_t slot, uint64_t k, int32_t ldk, uint64_t v, int32_t ldv, int32_t dtype, int32_t kv_heads, int32_t dk,
                                   int32_t dv, int32_t rows, uint64_t stream) {
    LUMI_TRY(check_rows("lumi_k_kv4_read", k, ldk, v, ldv, dtype, slot, kv, n_pages, kv_heads, dk, dv, rows));
    if (rows == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory("lumi_k_kv4_read", {k, v, slot, kv}));
    const RowsArgs a{nullptr, nullptr, (void*)k, (void*)v, (const int32_t*)slot, (uint8_t*)kv, ldk, ldv, n_pages * kPage, kv_heads, dk, dv, rows, 0};
    return rows_call<true>("lumi_k_kv4_read", a, dtype, whole(k, ldk, dk, dtype) && whole(v, ldv, dv, dtype), (cudaStream_t)stream);
}
