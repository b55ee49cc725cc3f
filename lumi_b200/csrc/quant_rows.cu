// Rows of numbers as 8-bit integers with a scale per row, for products in 8-bit integers: the norm in front of a projection (with the
// residual's addition), weights on their way into 8 bits, the gate between a feed-forward's products; and such rows back as numbers.
//
// A row t is held as q = rint(t * (127 / m)) and s = m / 127, m = max(max |t|, 2^-100).  The norm's factor r = 1 / sqrt(mean x^2 + eps) is the same for the
// whole row and cancels out of q: t = x w without it, and s = m / 127 * r.  So the sum of squares and the maximum are reduced side by side, in one
// pass over registers.  The maximum keeps infinities and NaN: such a row gets q = 0 and s = NaN.  Sums, maxima and scales are fp32.
//
// What bounds them is memory: each number is read once and written once.  Arithmetic comes close where rows are bf16: the norm of 8192 x 4096 rows without a residual
// (3 bytes per number, about 10 instructions) takes 21 us where DRAM takes 15.  Against rates that a plain copy reaches (6.55 TB/s): norm of 32768 x 1024 fp32 rows with a
// residual 66 us, 101 %; gate of 32768 x 2816 bf16 rows 72 us, 97 %; these back as bf16 45 us, 93 %.  One row takes 1.8 us, which is its launch.
#include "device_args.h"
#include "rows.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace lumi {
namespace {

constexpr float kLeast = 7.888609052210118e-31f;           // 2^-100: keeps 127 / m finite
constexpr int kMaxWidth = 1 << 30;                         // places within a row are 32-bit numbers
constexpr uint32_t kInfBits = 0x7f800000u;

struct QuantOut {
    int8_t* q;
    float* scale;
    int ldq;
};

// 1 / (1 + e^-v).  Of fp32 gates: expf (one ulp), then the hardware's reciprocal (one ulp) of an eighth of the sum, which stays in its range where the sigmoid no longer is a normal
// number: under 2^-21 of it for all v above -88.7, below which expf leaves fp32's range and the gate is closed.  Their bytes take longer than that: 32768 x 2816 116 us, with both
// approximations of the bf16 form too, with a rounded division 136.
// Of bf16 gates: hardware exponential and reciprocal, a relative error of 2^-21 and, below zero, of |v| 2^-23 (the rounding of the exponent), closed below -87.3.  These are few
// instructions, which such rows are close to being bound by: 32768 x 2816 72 us, with expf 86, with a rounded division too 115.  Half a step of an 8-bit integer is 2^-8.
__device__ __forceinline__ float gate_sigmoid(float v, const float*) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(expf(-v), 0.125f, 0.125f)));
    return r * 0.125f;
}
__device__ __forceinline__ float gate_sigmoid(float v, const __nv_bfloat16*) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
}

// ---- E numbers of a row as memory holds them, four or eight
template <typename T, int E>
struct Words { uint32_t u[E * sizeof(T) / 4]; };
template <int E>
__device__ __forceinline__ void unpack(const Words<float, E>& w, float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = __uint_as_float(w.u[i]);
}
template <int E>
__device__ __forceinline__ void unpack(const Words<__nv_bfloat16, E>& w, float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
        v[2 * i] = __uint_as_float(w.u[i] << 16);
        v[2 * i + 1] = __uint_as_float(w.u[i] & 0xffff0000u);
    }
}
// Of the norm's weights, which no store of the kernel changes: loads that may pass the stores of x, but not the dependency wait.
__device__ __forceinline__ void load_weights(const float* p, float& a, float& b, float& c, float& d) {
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a), "=f"(b), "=f"(c), "=f"(d) : "l"(p));
}
// The row ends n numbers from here.  Numbers are taken E at a time where a row has that many; those behind the last whole E (`tail`s, up to seven) go to the first
// threads of the row, one each.  What is behind a row is neither read nor written.
template <typename T, int E>
__device__ __forceinline__ void load_whole(const T* p, int n, Words<T, E>& w) {
    constexpr int N = E * (int)sizeof(T) / 4;
#pragma unroll
    for (int i = 0; i < N; ++i) w.u[i] = 0;
    if (n < E) return;
    if constexpr (N == 2) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        w.u[0] = t.x; w.u[1] = t.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 t = reinterpret_cast<const uint4*>(p)[i];
            w.u[4 * i] = t.x; w.u[4 * i + 1] = t.y; w.u[4 * i + 2] = t.z; w.u[4 * i + 3] = t.w;
        }
    }
}
__device__ __forceinline__ float number(const float* p) { return *p; }
__device__ __forceinline__ float number(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void put_one(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float stored(float v, const float*) { return v; }
__device__ __forceinline__ float stored(float v, const __nv_bfloat16*) { return __bfloat162float(__float2bfloat16_rn(v)); }
template <int E>
__device__ __forceinline__ void store_whole(float* p, const float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) *reinterpret_cast<float4*>(p + 4 * i) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
}
template <int E>
__device__ __forceinline__ void store_whole(__nv_bfloat16* p, const float (&v)[E]) {
    static_assert(E == 8, "");
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

// ---- sources of rows: load(): what memory holds of E numbers; values(): the numbers to be held in 8 bits, with the sum of squares
//
// How a row is laid over threads goes by what a source reads (device time, us; DRAM's floor in brackets):
// kWarp: up to this many numbers a row is a warp's, four warps per block.  fp32 without a residual 32768 x 1024: 26 (26), by blocks of 64 threads 35; with one, 74
//   (65), by blocks of 128 threads 66: twice the bytes want more threads.
// kEights: eights of numbers that each thread of a block holds, at least.  Gate of 32768 x 2816 bf16 rows: four 71 (70), two 81, one 117; norm of 16384 x 2048 fp32 rows with a
//   residual: one 66 (66), four 68; of 8192 x 4096 bf16 rows with a residual: two 39 (36), one 42, four 60; without: four 21 (15), two 25.
// kStay: as many blocks as run at once stay for row after row, the next one's loads ahead of this one's reduction.  It wins where a row is few bytes and has a residual's
//   sum to write (bf16, 16384 x 2048: 41 against 59), and loses elsewhere: the registers cost more blocks (gate of 32768 x 2816 bf16 rows: 94 against 75).
// Norm, or rows as they are.  ADD: x += o first, rounded to x's type, so that the norm sees what later readers of x see.
// TAIL: widths are no multiples of E.
template <typename XT, typename OT, bool ADD, bool NORM, bool TAIL>
struct NormSource {
    static constexpr bool kTail = TAIL;
    static constexpr int E = sizeof(XT) == 4 ? 4 : 8;
    static constexpr bool kNorm = NORM, kStay = E == 8 && ADD;
    static constexpr int kEights = ADD ? 1 : (E == 8 ? 4 : 2), kWarp = E == 8 || !ADD ? 1024 : 512;
    XT* x; const OT* o; const float* w;
    long ldx, ldo;
    int width;
    float eps;
    struct None {};
    struct Raw { Words<XT, E> x; std::conditional_t<ADD, Words<OT, E>, None> o; };
    template <bool AGAIN>
    __device__ __forceinline__ void load(long row, int c, Raw& r) const {
        load_whole(x + row * ldx + c, width - c, r.x);
        if constexpr (ADD && !AGAIN) load_whole(o + row * ldo + c, width - c, r.o);
    }
    // AGAIN: x has been added to already
    template <bool AGAIN>
    __device__ __forceinline__ void values(long row, int c, const Raw& r, float (&t)[E], float& sum) const {
        unpack(r.x, t);
        if constexpr (ADD && !AGAIN) {
            float add[E];
            unpack(r.o, add);
#pragma unroll
            for (int i = 0; i < E; ++i) t[i] = stored(t[i] + add[i], x);
            if (width - c >= E) store_whole<E>(x + row * ldx + c, t);
        }
        if constexpr (NORM) {
            float f[E];
            if (width - c >= E) {
#pragma unroll
                for (int i = 0; i < E; i += 4) load_weights(w + c + i, f[i], f[i + 1], f[i + 2], f[i + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < E; ++i) {
                sum = fmaf(t[i], t[i], sum);
                t[i] *= f[i];
            }
        }
    }
    // the same of one number
    static constexpr bool kTailFree = false;
    struct Tail { float x, o; };
    template <bool AGAIN>
    __device__ __forceinline__ void load_tail(long row, int c, Tail& r) const {
        r.x = number(x + row * ldx + c);
        if constexpr (ADD && !AGAIN) r.o = number(o + row * ldo + c);
    }
    template <bool AGAIN>
    __device__ __forceinline__ float tail(long row, int c, const Tail& r, float& sum) const {
        float v = r.x;
        if constexpr (ADD && !AGAIN) {
            v = stored(v + r.o, x);
            put_one(x + row * ldx + c, v);
        }
        if constexpr (!NORM) return v;
        sum = fmaf(v, v, sum);
        return v * number(w + c);
    }
    // sums of squares of numbers times k, from memory
    __device__ __forceinline__ float squares(long row, int c, float k) const {
        Raw r;
        float v[E], part = 0.f;
        load<true>(row, c, r);
        unpack(r.x, v);
#pragma unroll
        for (int i = 0; i < E; ++i) part = fmaf(v[i] * k, v[i] * k, part);
        return part;
    }
    __device__ __forceinline__ float squares_tail(long row, int c, float k) const {
        const float v = number(x + row * ldx + c) * k;
        return v * v;
    }
};

// Gate: rows hold gates, and from column `up` on as many ups.
template <typename XT, bool SILU, bool TAIL>
struct GateSource {
    static constexpr bool kTail = TAIL;
    static constexpr int E = sizeof(XT) == 4 ? 4 : 8;
    static constexpr bool kNorm = false, kStay = false;
    static constexpr int kEights = E == 8 ? 4 : 1, kWarp = E == 8 ? 1024 : 512;
    const XT* gu;
    long ld;
    int up, width;
    struct Raw { Words<XT, E> g, u; };
    template <bool AGAIN>
    __device__ __forceinline__ void load(long row, int c, Raw& r) const {
        load_whole(gu + row * ld + c, width - c, r.g);
        load_whole(gu + row * ld + up + c, width - c, r.u);
    }
    template <bool AGAIN>
    __device__ __forceinline__ void values(long, int, const Raw& r, float (&t)[E], float&) const {
        float u[E];
        unpack(r.g, t);
        unpack(r.u, u);
#pragma unroll
        for (int i = 0; i < E; ++i) t[i] = gated(t[i], u[i]);
    }
    // A tail of zeros is zero: taken by all threads without a branch, it runs beside the other numbers (fp32, 45248 x 1111 80 -> 73 us; bf16 no gain).
    static constexpr bool kTailFree = E == 4;
    struct Tail { float g, u; };
    template <bool AGAIN>
    __device__ __forceinline__ void load_tail(long row, int c, Tail& r) const {
        r.g = number(gu + row * ld + c);
        r.u = number(gu + row * ld + up + c);
    }
    template <bool AGAIN>
    __device__ __forceinline__ float tail(long, int, const Tail& r, float&) const { return gated(r.g, r.u); }
    static __device__ __forceinline__ float gated(float gate, float v) {
        const float z = gate_sigmoid(gate, (const XT*)nullptr);
        return (SILU ? gate * z : z) * v;
    }
};

// m: the largest |t| so far, or NaN once there was one.
template <int E>
__device__ __forceinline__ void largest(const float (&t)[E], float& m) {
#pragma unroll
    for (int i = 0; i < E; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(t[i])));
}
__device__ __forceinline__ void largest(float t, float& m) { asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(t))); }

// t * inv, rounded to fp32, to the nearest integer, ties to even: added to 1.5 * 2^23, the integer is the sum's low byte.  (Without the first rounding a quotient that lies on a half
// falls to the side that the reciprocal's error points to.)  Zeros where the row is not all numbers.
__device__ __forceinline__ uint32_t rounded(float t, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(t, inv), 12582912.f)); }
template <int E>
__device__ __forceinline__ void put(int8_t* q, int n, const float (&t)[E], float inv, bool numbers) {
    uint32_t b[E];
    if (numbers) {
#pragma unroll
        for (int i = 0; i < E; ++i) b[i] = rounded(t[i], inv);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) b[i] = 0;
    }
    if (n < E) return;
    uint32_t u[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
        u[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    if constexpr (E == 8) *reinterpret_cast<uint2*>(q) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint32_t*>(q) = u[0];
}

// Sum (SUM) and maximum over the threads of a row: a warp's, or the block's.  turn counts a block's reductions.
template <bool WARP, bool SUM>
__device__ __forceinline__ void reduce_row(float& sum, float& largest, uint32_t& turn) {
    if constexpr (SUM) sum = warp_total(sum);
    // as bits, numbers from zero on are in order, infinity above them and NaN above that
    uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));
    if constexpr (!WARP) {
        __shared__ float ss[2][32];                   // in turn: nobody is two reductions ahead of anybody
        __shared__ uint32_t sm[2][32];
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, b = turn++ & 1;
        if (lane == 0) {
            if constexpr (SUM) ss[b][warp] = sum;
            sm[b][warp] = m;
        }
        __syncthreads();
        if constexpr (SUM) sum = warp_total(lane < warps ? ss[b][lane] : 0.f);
        m = __reduce_max_sync(0xffffffffu, lane < warps ? sm[b][lane] : 0u);
    }
    largest = __uint_as_float(m);
}

// The norm's factor k / sqrt(sum / width + eps k^2), sum: of the squares of numbers times k.  k is 1, but a sum that has overflowed, or vanished beside a small
// eps, is taken again with another; again(k) gives it, to every thread alike.
struct Factor { float sum, k; };
template <typename AGAIN>
__device__ __forceinline__ Factor norm_sum(float sum, float eps, AGAIN again) {
    Factor f{sum, 1.f};
    if (!(sum < __uint_as_float(kInfBits))) f.k = 8.271806125530277e-25f;                        // 2^-80
    else if (sum < kLeast && eps < 8.470329472543003e-22f) f.k = 1.152921504606847e18f;          // 2^-70; 2^60
    if (f.k != 1.f) f.sum = again(f.k);
    return f;
}
__device__ __forceinline__ float norm_factor(const Factor& f, int width, float eps) {
    return __fmul_rn(f.k, __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(f.sum, (float)width), __fmul_rn(__fmul_rn(eps, f.k), f.k)))));
}

template <typename SRC>
__device__ __forceinline__ float row_scale(const SRC& src, const Factor& f, bool numbers, float top) {
    if (!numbers) return __uint_as_float(0x7fffffffu);
    float s = __fdiv_rn(top, 127.f);
    if constexpr (SRC::kNorm) s = __fmul_rn(s, norm_factor(f, src.width, src.eps));
    return s;
}

// Row per block of NT threads, the numbers read twice (the second time from L2): any width.  LONG: a thread's pieces are so many that their sums of squares are added up in 64 bits.  In one
// fp32 chain a norm's scale was off by up to 6e-6 at 2^20 equal numbers, 2.2e-5 at 2^22 and 3e-4 at 2^26; by 8e-8 so.  Up to kChain numbers per thread a chain is as good as the
// tree behind it, and faster (1024 x 32768 bf16 rows with a residual 51 us, in 64 bits 61).
constexpr int kChain = 64;
template <typename SRC, int NT, bool LONG>
__global__ void __launch_bounds__(NT) quant_wide_kernel(SRC src, QuantOut out) {
    constexpr int E = SRC::E;
    const long row = blockIdx.x;
    pdl_release();
    pdl_sync();
    const int whole = src.width / E * E, tail_at = whole + threadIdx.x;
    const bool has_tail = SRC::kTail && tail_at < src.width;
    float sum = 0.f, m = 0.f;
    double total = 0.0;
    uint32_t turn = 0;
    for (int c = threadIdx.x * E; c < whole; c += NT * E) {
        typename SRC::Raw r;
        float t[E];
        src.template load<false>(row, c, r);
        src.template values<false>(row, c, r, t, sum);
        if constexpr (LONG) {
            total += sum;
            sum = 0.f;
        }
        largest<E>(t, m);
    }
    if constexpr (LONG) sum = (float)total;
    typename SRC::Tail r1{};
    if (has_tail) {
        src.template load_tail<false>(row, tail_at, r1);
        largest(src.template tail<false>(row, tail_at, r1, sum), m);
    }
    reduce_row<false, SRC::kNorm>(sum, m, turn);
    const bool numbers = m < __uint_as_float(kInfBits);
    Factor f{0.f, 1.f};
    if constexpr (SRC::kNorm)
        f = norm_sum(sum, src.eps, [&](float k) {
            std::conditional_t<LONG, double, float> squares = has_tail ? src.squares_tail(row, tail_at, k) : 0.f;
            for (int c = threadIdx.x * E; c < whole; c += NT * E) squares += src.squares(row, c, k);
            float part = (float)squares, unused = 0.f;
            reduce_row<false, true>(part, unused, turn);
            return part;
        });
    const float top = fmaxf(m, kLeast), inv = __fdiv_rn(127.f, top);
    if (threadIdx.x == 0) out.scale[row] = row_scale(src, f, numbers, top);
    int8_t* const q = out.q + row * out.ldq;
    float unused = 0.f;
    for (int c = threadIdx.x * E; c < whole; c += NT * E) {
        typename SRC::Raw r;
        float t[E];
        src.template load<true>(row, c, r);
        src.template values<true>(row, c, r, t, unused);
        put<E>(q + c, E, t, inv, numbers);
    }
    if (has_tail) {
        src.template load_tail<true>(row, tail_at, r1);
        q[tail_at] = numbers ? (int8_t)rounded(src.template tail<true>(row, tail_at, r1, unused), inv) : 0;
    }
}

// The numbers of a row in the registers of a warp (WARP) or a block, NC times E for each thread: memory is read once, all of it asked for before the first is
// used, and the next row's while this one is reduced and written.
// Blocks of 512 that have room on an SM, whatever the compiler would like: with fewer, an fp32 silu gate of 8192 x 8192 took 117 us (now 86), of 32768 x 1536 69 (65).
template <typename SRC, bool WARP, int NC>
constexpr int kRoom = WARP ? 1 : (SRC::E == 8 ? 2 : (SRC::kNorm ? 1 : (NC == 2 ? 3 : 2)));
template <typename SRC, bool WARP, int NC>
__global__ void __launch_bounds__(WARP ? 128 : 512, kRoom<SRC, WARP, NC>) quant_rows_kernel(SRC src, QuantOut out, int rows) {
    constexpr int E = SRC::E;
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, NT = WARP ? 32 : blockDim.x;
    const long step = WARP ? 4l * gridDim.x : (long)gridDim.x;
    long row = WARP ? (long)blockIdx.x * 4 + (threadIdx.x >> 5) : (long)blockIdx.x;
    uint32_t turn = 0;
    pdl_release();
    pdl_sync();
    if (row >= rows) return;                              // whole warps, and only where a row is a warp's
    const int tail_at = src.width / E * E + tid;
    const bool has_tail = SRC::kTail && tail_at < src.width;
    typename SRC::Raw r[NC];
    typename SRC::Tail r1{};
#pragma unroll
    for (int i = 0; i < NC; ++i) src.template load<false>(row, (i * NT + tid) * E, r[i]);
    if (has_tail) src.template load_tail<false>(row, tail_at, r1);
    for (; row < rows; row += step) {
        float sum = 0.f, t[NC][E], m = 0.f, t1 = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            src.template values<false>(row, (i * NT + tid) * E, r[i], t[i], sum);
            largest<E>(t[i], m);
        }
        if (SRC::kTail && (has_tail || SRC::kTailFree)) {
            t1 = src.template tail<false>(row, tail_at, r1, sum);
            largest(t1, m);
        }
        if (SRC::kStay && row + step < rows) {
#pragma unroll
            for (int i = 0; i < NC; ++i) src.template load<false>(row + step, (i * NT + tid) * E, r[i]);
            if (has_tail) src.template load_tail<false>(row + step, tail_at, r1);
        }
        reduce_row<WARP, SRC::kNorm>(sum, m, turn);
        const bool numbers = m < __uint_as_float(kInfBits);
        Factor f{0.f, 1.f};
        if constexpr (SRC::kNorm)
            f = norm_sum(sum, src.eps, [&](float k) {
                float part = has_tail ? src.squares_tail(row, tail_at, k) : 0.f, unused = 0.f;
                for (int i = 0; i < NC; ++i) part += src.squares(row, (i * NT + tid) * E, k);
                reduce_row<WARP, true>(part, unused, turn);
                return part;
            });
        const float top = fmaxf(m, kLeast), inv = __fdiv_rn(127.f, top);
        int8_t* const q = out.q + row * out.ldq;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (i * NT + tid) * E;
            put<E>(q + c, src.width - c, t[i], inv, numbers);
        }
        if (has_tail) q[tail_at] = numbers ? (int8_t)rounded(t1, inv) : 0;
        if (tid == 0) out.scale[row] = row_scale(src, f, numbers, top);      // by one thread: its divisions and root take longer than a row's numbers
        if constexpr (!SRC::kStay) break;
    }
}

// the launch itself overlaps the kernel in front
cudaLaunchConfig_t dependent_launch(dim3 grid, int threads, cudaLaunchAttribute* attr, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

template <typename SRC, bool WARP, int NC>
int32_t launch_rows_of(const SRC& src, const QuantOut& out, int rows, cudaStream_t st) {
    static std::atomic<int> registers{0};
    int regs = registers.load(std::memory_order_relaxed);
    if (regs == 0) {
        cudaFuncAttributes at;
        LUMI_CUDA(cudaFuncGetAttributes(&at, quant_rows_kernel<SRC, WARP, NC>));
        regs = at.numRegs;
        registers.store(regs, std::memory_order_relaxed);
    }
    const int chunks = std::max(1, src.width / SRC::E), threads = WARP ? 128 : ((chunks + NC - 1) / NC + 31) / 32 * 32;
    // as many blocks as run at once; registers are given out by eights per thread
    const int per_sm = std::max(1, std::min({32, 2048 / threads, 65536 / ((regs + 7) / 8 * 8 * threads)}));
    const long blocks = WARP ? ((long)rows + 3) / 4 : rows;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = dependent_launch(dim3((unsigned)(SRC::kStay ? std::min(blocks, (long)per_sm * sm_count()) : blocks)), threads, attr, st);
    LUMI_CUDA(cudaLaunchKernelEx(&cfg, quant_rows_kernel<SRC, WARP, NC>, src, out, rows));
    return LUMI_OK;
}

// Two eights of numbers per thread instead of four, where whole warps then leave fewer threads without numbers: 1536 columns are 192 eights, 64 threads of four or 96 of
// two.  Gate of 32768 x 1536 bf16 rows 42 -> 37 us, 16384 x 2400 35 -> 31.
inline bool two_eights(int width) {
    const int n = width / 8;
    auto slots = [&](int per) { return ((n + per - 1) / per + 31) / 32 * 32 * per; };
    return 10 * slots(2) < 9 * slots(4);
}

// The shape goes by the width alone, so that a row has the same bits alone and among others.
template <typename SRC>
int32_t launch(const SRC& src, const QuantOut& out, int rows, cudaStream_t st) {
    constexpr int L = 8 / SRC::E;                         // loads for eight numbers
    const int width = src.width;
    if (width <= 32 * 8) return launch_rows_of<SRC, true, L>(src, out, rows, st);
    if (width <= 32 * 16) return launch_rows_of<SRC, true, 2 * L>(src, out, rows, st);
    if constexpr (SRC::kWarp == 1024) {
        if (width <= 32 * 24) return launch_rows_of<SRC, true, 3 * L>(src, out, rows, st);
        if (width <= 32 * 32) return launch_rows_of<SRC, true, 4 * L>(src, out, rows, st);
    }
    if constexpr (SRC::kEights == 1) {
        if (width <= 256 * 8) return launch_rows_of<SRC, false, L>(src, out, rows, st);
    }
    if (width <= 512 * 16 && (SRC::kEights <= 2 || two_eights(width))) return launch_rows_of<SRC, false, 2 * L>(src, out, rows, st);
    if (width <= 512 * 32) return launch_rows_of<SRC, false, 4 * L>(src, out, rows, st);
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = dependent_launch(dim3((unsigned)rows), 1024, attr, st);
    if (SRC::kNorm && width > 1024 * kChain) LUMI_CUDA(cudaLaunchKernelEx(&cfg, quant_wide_kernel<SRC, 1024, SRC::kNorm>, src, out));
    else LUMI_CUDA(cudaLaunchKernelEx(&cfg, quant_wide_kernel<SRC, 1024, false>, src, out));
    return LUMI_OK;
}

template <typename XT, typename OT>
int32_t launch_norm(uint64_t x, int ldx, uint64_t o, int ldo, uint64_t w, const QuantOut& out, int rows, int width, float eps, cudaStream_t st) {
    auto go = [&](auto src) {
        src.x = (XT*)x; src.o = (decltype(src.o))o; src.w = (const float*)w;
        src.ldx = ldx; src.ldo = ldo; src.width = width; src.eps = eps;
        return launch(src, out, rows, st);
    };
    auto with_tail = [&](auto tail) {
        constexpr bool T = decltype(tail)::value;
        if (o) return w ? go(NormSource<XT, OT, true, true, T>{}) : go(NormSource<XT, OT, true, false, T>{});
        return w ? go(NormSource<XT, XT, false, true, T>{}) : go(NormSource<XT, XT, false, false, T>{});
    };
    return width % NormSource<XT, OT, true, true, true>::E != 0 ? with_tail(std::true_type{}) : with_tail(std::false_type{});
}

// ---- rows back as numbers: y = q s.  A warp takes up to 1024 numbers of a row, 16 bytes of y per lane at a time.  ANY: rows of y begin anywhere, or end within
// 16 bytes: the 16-byte pieces that lie whole within a row are written as such, from bytes of q that lie across its words, and the numbers in
// front of them and behind one by one.  (Written one by one throughout, 20000 x 1111 into bf16 took 33 us.)
__device__ __forceinline__ float byte_value(uint32_t word, int b, float s) {
    // a byte q + 128 under the exponent of 2^23 is the float 2^23 + 128 + q
    return __fmul_rn(__uint_as_float(__byte_perm(word ^ 0x80808080u, 0x4b000000u, 0x7540u | (uint32_t)b)) - 8388736.f, s);
}
template <typename YT, bool ANY>
__global__ void __launch_bounds__(256) dequant_kernel(const int8_t* q, long ldq, const float* scale, YT* y, long ldy, int rows, int width) {
    constexpr int E = 16 / (int)sizeof(YT), DEEP = 1024 / 32 / E;       // numbers in 16 bytes, pieces per lane
    const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    pdl_release();
    pdl_sync();
    if (row >= rows) return;
    const float s = scale[row];
    q += row * ldq;
    y += row * ldy;
    const int head = ANY ? min(width, (int)((E - (reinterpret_cast<uintptr_t>(y) / sizeof(YT)) % E) % E)) : 0, pieces = (width - head) / E;
    if (ANY && blockIdx.y == 0) {
        const int c = lane < 8 ? lane : head + pieces * E + lane - 8;       // lanes 0 to 7: the head; 8 to 15: what the pieces leave
        if (lane < 8 ? c < head : lane < 16 && c < width) put_one(y + c, __fmul_rn((float)q[c], s));
    }
    for (long j0 = (long)blockIdx.y * (1024 / E); j0 < pieces; j0 += (long)gridDim.y * (1024 / E)) {
        uint32_t u[DEEP][E / 4];
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            const long j = j0 + i * 32 + lane, a = head + j * E;
#pragma unroll
            for (int e = 0; e < E / 4; ++e) u[i][e] = 0;
            if (j >= pieces) continue;
            if constexpr (!ANY) {
                if constexpr (E == 8) asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(u[i][0]), "=r"(u[i][1]) : "l"(q + a));
                else asm volatile("ld.global.u32 %0, [%1];" : "=r"(u[i][0]) : "l"(q + a));
            } else if (((a + E - 1) | 3) < width) {                     // all words that it lies across are the row's
                const uint32_t* w = reinterpret_cast<const uint32_t*>(q + (a & ~3l));
                const uint32_t shift = 8 * (uint32_t)(a & 3);
                uint32_t last = w[0];
#pragma unroll
                for (int e = 0; e < E / 4; ++e) {
                    const uint32_t next = shift != 0 || e + 1 < E / 4 ? w[e + 1] : 0u;
                    u[i][e] = __funnelshift_r(last, next, shift);
                    last = next;
                }
            } else {
                for (int e = 0; e < E; ++e) u[i][e / 4] |= (uint32_t)(uint8_t)q[a + e] << (8 * (e % 4));
            }
        }
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            const long j = j0 + i * 32 + lane;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = byte_value(u[i][e / 4], e & 3, s);
            if (j < pieces) store_whole<E>(y + head + j * E, v);
        }
    }
}

bool aligned_rows(uint64_t p, int dtype, int ld) { return (p & 15) == 0 && ld % (dtype == LUMI_DTYPE_F32 ? 4 : 8) == 0; }
bool known(int dtype) { return dtype == LUMI_DTYPE_F32 || dtype == LUMI_DTYPE_BF16; }

}  // namespace
}  // namespace lumi

using namespace lumi;

extern "C" int32_t lumi_k_norm_quant(uint64_t x, int32_t x_dtype, int32_t ldx, uint64_t o, int32_t o_dtype, int32_t ldo, uint64_t w, uint64_t q, int32_t ldq,
                                     uint64_t scale, int32_t rows, int32_t width, float eps, uint64_t stream) {
    if (!x || !q || !scale || !known(x_dtype) || (o && !known(o_dtype)) || rows < 0 || width <= 0 || ldx < width || (o && ldo < width) || ldq < width ||
        (w && !(eps > 0.f && eps <= 3.4e38f)))
        return fail(LUMI_E_INVALID, "bad argument to lumi_k_norm_quant");
    if (!aligned_rows(x, x_dtype, ldx) || (o && !aligned_rows(o, o_dtype, ldo)) || (w & 15) || (q & 15) || ldq % 16 || (scale & 3))
        return fail(LUMI_E_INVALID, "lumi_k_norm_quant: rows have to begin on 16-byte boundaries");
    if (width > kMaxWidth) return fail(LUMI_E_UNSUPPORTED, "lumi_k_norm_quant: width %d (at most %d)", width, kMaxWidth);
    if (rows == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory("lumi_k_norm_quant", {x, o, w, q, scale}));
    const QuantOut out{(int8_t*)q, (float*)scale, ldq};
    const cudaStream_t st = (cudaStream_t)stream;
    if (x_dtype == LUMI_DTYPE_F32)
        return o && o_dtype == LUMI_DTYPE_BF16 ? launch_norm<float, __nv_bfloat16>(x, ldx, o, ldo, w, out, rows, width, eps, st)
                                               : launch_norm<float, float>(x, ldx, o, ldo, w, out, rows, width, eps, st);
    return o && o_dtype == LUMI_DTYPE_F32 ? launch_norm<__nv_bfloat16, float>(x, ldx, o, ldo, w, out, rows, width, eps, st)
                                          : launch_norm<__nv_bfloat16, __nv_bfloat16>(x, ldx, o, ldo, w, out, rows, width, eps, st);
}

extern "C" int32_t lumi_k_gate_quant(uint64_t gu, int32_t dtype, int32_t ld, int32_t up, int32_t act, uint64_t q, int32_t ldq, uint64_t scale,
                                     int32_t rows, int32_t width, uint64_t stream) {
    if (!gu || !q || !scale || !known(dtype) || act < 0 || act > 1 || rows < 0 || width <= 0 || up < width || ld < width || up > ld - width || ldq < width)
        return fail(LUMI_E_INVALID, "bad argument to lumi_k_gate_quant");
    if (!aligned_rows(gu, dtype, ld) || up % (dtype == LUMI_DTYPE_F32 ? 4 : 8) || (q & 15) || ldq % 16 || (scale & 3))
        return fail(LUMI_E_INVALID, "lumi_k_gate_quant: rows, gates and ups have to begin on 16-byte boundaries");
    if (rows == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory("lumi_k_gate_quant", {gu, q, scale}));
    const QuantOut out{(int8_t*)q, (float*)scale, ldq};
    const cudaStream_t st = (cudaStream_t)stream;
    auto go = [&](auto src) {
        using SRC = decltype(src);
        src.gu = (decltype(src.gu))gu;
        src.ld = ld; src.up = up; src.width = width;
        return launch<SRC>(src, out, rows, st);
    };
    auto with_tail = [&](auto tail) {
        constexpr bool T = decltype(tail)::value;
        if (dtype == LUMI_DTYPE_F32) return act ? go(GateSource<float, true, T>{}) : go(GateSource<float, false, T>{});
        return act ? go(GateSource<__nv_bfloat16, true, T>{}) : go(GateSource<__nv_bfloat16, false, T>{});
    };
    return width % (dtype == LUMI_DTYPE_F32 ? 4 : 8) != 0 ? with_tail(std::true_type{}) : with_tail(std::false_type{});
}

extern "C" int32_t lumi_k_dequant_rows(uint64_t q, int32_t ldq, uint64_t scale, uint64_t y, int32_t y_dtype, int32_t ldy, int32_t rows, int32_t width,
                                       uint64_t stream) {
    if (!q || !scale || !y || !known(y_dtype) || rows < 0 || width <= 0 || ldq < width || ldy < width) return fail(LUMI_E_INVALID, "bad argument to lumi_k_dequant_rows");
    if ((q & 15) || ldq % 16 || (scale & 3) || (y & (y_dtype == LUMI_DTYPE_F32 ? 3 : 1)))
        return fail(LUMI_E_INVALID, "lumi_k_dequant_rows: rows of q have to begin on 16-byte boundaries, numbers on their own");
    if (rows == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory("lumi_k_dequant_rows", {q, scale, y}));
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = dependent_launch(dim3((unsigned)(((long)rows + 7) / 8), (unsigned)std::min(65535l, ((long)width + 1023) / 1024)), 256, attr, (cudaStream_t)stream);
    auto go = [&](auto* to, auto any) {
        using YT = std::remove_pointer_t<decltype(to)>;
        return cudaLaunchKernelEx(&cfg, dequant_kernel<YT, decltype(any)::value>, (const int8_t*)q, (long)ldq, (const float*)scale, to, (long)ldy, rows, width);
    };
    const bool any = width % 8 != 0 || !aligned_rows(y, y_dtype, ldy);
    if (y_dtype == LUMI_DTYPE_F32) LUMI_CUDA(any ? go((float*)y, std::true_type{}) : go((float*)y, std::false_type{}));
    else LUMI_CUDA(any ? go((__nv_bfloat16*)y, std::true_type{}) : go((__nv_bfloat16*)y, std::false_type{}));
    return LUMI_OK;
}
