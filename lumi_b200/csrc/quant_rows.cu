// Rows of numbers as 8-bit integers with a scale per row, for products in 8-bit integers: the norm in front of a projection (with the
// residual's addition), weights on their way into 8 bits, the gate between a feed-forward's products; and such rows back as numbers.
//
// A row t is held as q = rint(t * 127 / m) and s = m / 127, m = max(max |t|, 2^-100).  The norm's factor r = 1 / sqrt(mean x^2 + eps) is the same for the
// whole row and cancels out of q: t = x w without it, and s = m / 127 * r.  So the sum of squares and the maximum are reduced side by side, in one
// pass over registers.  The maximum is taken over the bits of |t|, where infinities and NaN are largest: such a row gets q = 0 and s = NaN.
#include "device_args.h"
#include "rows.cuh"

#include <algorithm>
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

// ---- loads of four or eight numbers, as fp32
// fast forms of the gate: relative error 2^-21 times the size of a negative gate
__device__ __forceinline__ float fast_sigmoid(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

template <int E>
__device__ __forceinline__ void load_whole(const float* p, float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(p + 4 * i);
        v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
}
template <int E>
__device__ __forceinline__ void load_whole(const __nv_bfloat16* p, float (&v)[E]) {
    uint32_t u[E / 2];
    if constexpr (E == 8) {
        const uint4 t = *reinterpret_cast<const uint4*>(p);
        u[0] = t.x; u[1] = t.y; u[2] = t.z; u[3] = t.w;
    } else {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        u[0] = t.x; u[1] = t.y;
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
// Of the norm's weights, which no store of the kernel changes: loads that may pass the stores of x, but not the dependency wait.
template <bool RAGGED>
__device__ __forceinline__ void load_weights(const float* p, int n, float& a, float& b, float& c, float& d) {
    a = b = c = d = 0.f;
    if (RAGGED ? n >= 4 : n > 0) {
        asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a), "=f"(b), "=f"(c), "=f"(d) : "l"(p));
    } else if (RAGGED) {
        if (n > 0) a = p[0];
        if (n > 1) b = p[1];
        if (n > 2) c = p[2];
    }
}
__device__ __forceinline__ float one(const float* p) { return *p; }
__device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
// The row ends n numbers from here (n <= 0: before); what is behind it is neither read nor counted.  RAGGED: it may end within these E.
template <bool RAGGED, int E, typename T>
__device__ __forceinline__ void load_some(const T* p, int n, float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = 0.f;
    if (RAGGED ? n >= E : n > 0) {
        load_whole<E>(p, v);
    } else if (RAGGED) {
#pragma unroll
        for (int i = 0; i < E; ++i) if (i < n) v[i] = one(p + i);
    }
}
__device__ __forceinline__ void put_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void put_one(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float stored(float v, const float*) { return v; }
__device__ __forceinline__ float stored(float v, const __nv_bfloat16*) { return __bfloat162float(__float2bfloat16_rn(v)); }
template <bool RAGGED, int E>
__device__ __forceinline__ void store_some(float* p, int n, const float (&v)[E]) {
    if (RAGGED ? n >= E : n > 0) {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) *reinterpret_cast<float4*>(p + 4 * i) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        return;
    }
    if (RAGGED)
#pragma unroll
        for (int i = 0; i < E; ++i) if (i < n) p[i] = v[i];
}
template <bool RAGGED, int E>
__device__ __forceinline__ void store_some(__nv_bfloat16* p, int n, const float (&v)[E]) {
    static_assert(E == 8, "");
    if (RAGGED ? n >= E : n > 0) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
        return;
    }
    if (RAGGED)
#pragma unroll
        for (int i = 0; i < E; ++i) if (i < n) p[i] = __float2bfloat16_rn(v[i]);
}

// ---- sources of rows: load(): what memory holds of E numbers; values(): the numbers to be held in 8 bits, with the sum of squares
// Norm, or rows as they are.  ADD: x += o first, rounded to x's type, so that the norm sees what later readers of x see.
template <typename XT, typename OT, bool ADD, bool NORM, bool RAGGED>
struct NormSource {
    static constexpr bool kRagged = RAGGED;
    static constexpr int E = sizeof(XT) == 4 ? 4 : 8;
    static constexpr bool kNorm = NORM;
    XT* x; const OT* o; const float* w;
    long ldx, ldo;
    int width;
    float eps;
    struct Raw { float x[E], o[ADD ? E : 1]; };
    template <bool AGAIN>
    __device__ __forceinline__ void load(long row, int c, Raw& r) const {
        load_some<RAGGED, E>(x + row * ldx + c, width - c, r.x);
        if constexpr (ADD && !AGAIN) load_some<RAGGED, E>(o + row * ldo + c, width - c, r.o);
    }
    // AGAIN: x has been added to already
    template <bool AGAIN>
    __device__ __forceinline__ void values(long row, int c, Raw& r, float (&t)[E], float& sum) const {
        if constexpr (ADD && !AGAIN) {
#pragma unroll
            for (int i = 0; i < E; ++i) r.x[i] = stored(r.x[i] + r.o[i], x);
            store_some<RAGGED, E>(x + row * ldx + c, width - c, r.x);
        }
        float f[E];
        if constexpr (NORM)
#pragma unroll
            for (int i = 0; i < E; i += 4) load_weights<RAGGED>(w + c + i, width - c - i, f[i], f[i + 1], f[i + 2], f[i + 3]);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if constexpr (NORM) {
                sum = fmaf(r.x[i], r.x[i], sum);
                t[i] = r.x[i] * f[i];
            } else {
                t[i] = r.x[i];
            }
        }
    }
};

// Gate: rows hold gates, and from column `up` on as many ups.
template <typename XT, bool SILU, bool RAGGED>
struct GateSource {
    static constexpr bool kRagged = RAGGED;
    static constexpr int E = sizeof(XT) == 4 ? 4 : 8;
    static constexpr bool kNorm = false;
    const XT* gu;
    long ld;
    int up, width;
    struct Raw { float g[E], u[E]; };
    template <bool AGAIN>
    __device__ __forceinline__ void load(long row, int c, Raw& r) const {
        load_some<RAGGED, E>(gu + row * ld + c, width - c, r.g);
        load_some<RAGGED, E>(gu + row * ld + up + c, width - c, r.u);
    }
    template <bool AGAIN>
    __device__ __forceinline__ void values(long, int, Raw& r, float (&t)[E], float&) const {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float z = fast_sigmoid(r.g[i]);
            t[i] = (SILU ? r.g[i] * z : z) * r.u[i];
        }
    }
};

template <int E>
__device__ __forceinline__ void largest(const float (&t)[E], uint32_t& m) {
#pragma unroll
    for (int i = 0; i < E; ++i) m = max(m, __float_as_uint(t[i]) & 0x7fffffffu);
}

// t * inv to the nearest integer, ties to even: added to 1.5 * 2^23, the integer is the sum's low byte.
template <bool RAGGED, int E>
__device__ __forceinline__ void put(int8_t* q, int n, const float (&t)[E], float inv) {
    uint32_t b[E];
#pragma unroll
    for (int i = 0; i < E; ++i) b[i] = __float_as_uint(fmaf(t[i], inv, 12582912.f));
    if (RAGGED ? n >= E : n > 0) {
        uint32_t u[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; ++i)
            u[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
        if constexpr (E == 8) *reinterpret_cast<uint2*>(q) = make_uint2(u[0], u[1]);
        else *reinterpret_cast<uint32_t*>(q) = u[0];
        return;
    }
    if (RAGGED)
#pragma unroll
        for (int i = 0; i < E; ++i) if (i < n) q[i] = (int8_t)b[i];
}

// Sum and maximum over the NT threads of a row (a whole warp, or the block).
template <int NT>
__device__ __forceinline__ void reduce_row(float& sum, uint32_t& m) {
    sum = warp_total(sum);
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (NT > 32) {
        __shared__ float ss[NT / 32];
        __shared__ uint32_t sm[NT / 32];
        const int warp = threadIdx.x >> 5;
        __syncthreads();                              // an earlier reduction's values have been read
        if ((threadIdx.x & 31) == 0) { ss[warp] = sum; sm[warp] = m; }
        __syncthreads();
        sum = 0.f; m = 0;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) { sum += ss[i]; m = max(m, sm[i]); }
    }
}

// 1 / sqrt(sum / width + eps).  A sum of squares that has overflowed or vanished beside a small eps is taken again of numbers times k; again(k) gives it.
template <typename AGAIN>
__device__ __forceinline__ float norm_factor(float sum, int width, float eps, AGAIN again) {
    float k = 1.f;
    if (!(sum < __uint_as_float(kInfBits))) k = 8.271806125530277e-25f;                          // 2^-80
    else if (sum < kLeast && eps < 8.470329472543003e-22f) k = 1.152921504606847e18f;            // 2^-70; 2^60
    if (k != 1.f) sum = again(k);
    return __fmul_rn(k, __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)width), __fmul_rn(__fmul_rn(eps, k), k)))));
}

// Row per block of NT threads, the numbers read twice (the second time from L2): any width.
template <typename SRC, int NT>
__global__ void __launch_bounds__(NT) quant_wide_kernel(SRC src, QuantOut out) {
    constexpr int E = SRC::E;
    const long row = blockIdx.x;
    pdl_release();
    pdl_sync();
    float sum = 0.f;
    uint32_t m = 0;
    for (int c = threadIdx.x * E; c < src.width; c += NT * E) {
        typename SRC::Raw r;
        float t[E];
        src.template load<false>(row, c, r);
        src.template values<false>(row, c, r, t, sum);
        largest<E>(t, m);
    }
    reduce_row<NT>(sum, m);
    const bool numbers = m < kInfBits;
    float factor = 1.f;
    if constexpr (SRC::kNorm)
        factor = norm_factor(sum, src.width, src.eps, [&](float k) {
            float part = 0.f;
            uint32_t unused = 0;
            for (int c = threadIdx.x * E; c < src.width; c += NT * E) {
                typename SRC::Raw r;
                src.template load<true>(row, c, r);
#pragma unroll
                for (int i = 0; i < E; ++i) part = fmaf(r.x[i] * k, r.x[i] * k, part);
            }
            reduce_row<NT>(part, unused);
            return part;
        });
    const float top = fmaxf(__uint_as_float(m), kLeast), inv = numbers ? __fdiv_rn(127.f, top) : 0.f;
    if (threadIdx.x == 0) out.scale[row] = numbers ? __fdiv_rn(top, 127.f) * factor : __uint_as_float(0x7fffffffu);
    for (int c = threadIdx.x * E; c < src.width; c += NT * E) {
        typename SRC::Raw r;
        float t[E], unused = 0.f;
        src.template load<true>(row, c, r);
        src.template values<true>(row, c, r, t, unused);
        if (!numbers)
#pragma unroll
            for (int i = 0; i < E; ++i) t[i] = 0.f;
        put<SRC::kRagged, E>(out.q + row * out.ldq + c, src.width - c, t, inv);
    }
}

// The numbers of a row in the registers of NT threads (a warp, or the block), NC times E each: memory is read once, all of it asked for before the
// first is used.
template <typename SRC, int NT, int NC>
__global__ void __launch_bounds__(NT == 32 ? 128 : NT) quant_rows_kernel(SRC src, QuantOut out, int rows) {
    constexpr int E = SRC::E;
    const long row = NT == 32 ? (long)blockIdx.x * 4 + (threadIdx.x >> 5) : (long)blockIdx.x;
    const int tid = NT == 32 ? threadIdx.x & 31 : threadIdx.x;
    pdl_release();
    pdl_sync();
    if (row >= rows) return;                              // whole warps, and only where a row is a warp's
    typename SRC::Raw r[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) src.template load<false>(row, (i * NT + tid) * E, r[i]);
    float sum = 0.f, t[NC][E];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        src.template values<false>(row, (i * NT + tid) * E, r[i], t[i], sum);
        largest<E>(t[i], m);
    }
    reduce_row<NT>(sum, m);
    const bool numbers = m < kInfBits;
    float factor = 1.f;
    if constexpr (SRC::kNorm)
        factor = norm_factor(sum, src.width, src.eps, [&](float k) {
            float part = 0.f;
            uint32_t unused = 0;
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) part = fmaf(r[i].x[e] * k, r[i].x[e] * k, part);
            reduce_row<NT>(part, unused);
            return part;
        });
    const float top = fmaxf(__uint_as_float(m), kLeast), inv = numbers ? __fdiv_rn(127.f, top) : 0.f;
    if (tid == 0) out.scale[row] = numbers ? __fdiv_rn(top, 127.f) * factor : __uint_as_float(0x7fffffffu);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = (i * NT + tid) * E;
        if (!numbers)
#pragma unroll
            for (int e = 0; e < E; ++e) t[i][e] = 0.f;
        put<SRC::kRagged, E>(out.q + row * out.ldq + c, src.width - c, t[i], inv);
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

template <typename SRC, int NT, int NC>
int32_t launch_rows_of(const SRC& src, const QuantOut& out, int rows, cudaStream_t st) {
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = dependent_launch(dim3(NT == 32 ? (unsigned)(((long)rows + 3) / 4) : (unsigned)rows), NT == 32 ? 128 : NT, attr, st);
    if constexpr (NC > 0) LUMI_CUDA(cudaLaunchKernelEx(&cfg, quant_rows_kernel<SRC, NT, NC>, src, out, rows));
    else LUMI_CUDA(cudaLaunchKernelEx(&cfg, quant_wide_kernel<SRC, NT>, src, out));
    return LUMI_OK;
}

// The shape goes by the width alone, so that a row has the same bits alone and among others.
template <typename SRC>
int32_t launch(const SRC& src, const QuantOut& out, int rows, cudaStream_t st) {
    constexpr int E = SRC::E, L = 8 / E;                  // L: a row's numbers are 2 L (4 L, 8 L) loads of a thread
    if (src.width <= 32 * 8) return launch_rows_of<SRC, 32, L>(src, out, rows, st);
    if (src.width <= 32 * 32) return launch_rows_of<SRC, 32, 4 * L>(src, out, rows, st);
    if (src.width <= 256 * 8) return launch_rows_of<SRC, 256, L>(src, out, rows, st);
    if (src.width <= 256 * 16) return launch_rows_of<SRC, 256, 2 * L>(src, out, rows, st);
    if (src.width <= 256 * 32) return launch_rows_of<SRC, 256, 4 * L>(src, out, rows, st);
    if (src.width <= 512 * 32) return launch_rows_of<SRC, 512, 4 * L>(src, out, rows, st);
    return launch_rows_of<SRC, 1024, 0>(src, out, rows, st);
}

template <typename XT, typename OT>
int32_t launch_norm(uint64_t x, int ldx, uint64_t o, int ldo, uint64_t w, const QuantOut& out, int rows, int width, float eps, cudaStream_t st) {
    auto go = [&](auto src) {
        src.x = (XT*)x; src.o = (decltype(src.o))o; src.w = (const float*)w;
        src.ldx = ldx; src.ldo = ldo; src.width = width; src.eps = eps;
        return launch(src, out, rows, st);
    };
    auto ragged = [&](auto r) {
        constexpr bool R = decltype(r)::value;
        if (o) return w ? go(NormSource<XT, OT, true, true, R>{}) : go(NormSource<XT, OT, true, false, R>{});
        return w ? go(NormSource<XT, XT, false, true, R>{}) : go(NormSource<XT, XT, false, false, R>{});
    };
    return width % NormSource<XT, OT, true, true, true>::E != 0 ? ragged(std::true_type{}) : ragged(std::false_type{});
}

// ---- rows back as numbers: y = q s.  A warp takes up to 1024 numbers of a row: eight per lane at a time, or (ONE) one, for rows of y that begin
// anywhere and widths that are no multiples of eight.
template <typename YT, bool ONE>
__global__ void __launch_bounds__(256) dequant_kernel(const int8_t* q, long ldq, const float* scale, YT* y, long ldy, int rows, int width) {
    const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    pdl_release();
    pdl_sync();
    if (row >= rows) return;
    const float s = scale[row];
    q += row * ldq;
    y += row * ldy;
    for (long c0 = (long)blockIdx.y * 1024; c0 < width; c0 += (long)gridDim.y * 1024) {
        if constexpr (ONE) {
            const long end = min(c0 + 1024, (long)width);
#pragma unroll 8
            for (long c = c0 + lane; c < end; c += 32) put_one(y + c, __fmul_rn((float)q[c], s));
            continue;
        }
        uint2 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long c = c0 + (i * 32 + lane) * 8;
            u[i] = make_uint2(0, 0);
            if (c < width) asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(u[i].x), "=r"(u[i].y) : "l"(q + c));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long c = c0 + (i * 32 + lane) * 8;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // a byte b + 128 under the exponent of 2^23 is the float 2^23 + 128 + b
                const uint32_t w = (e < 4 ? u[i].x : u[i].y) ^ 0x80808080u;
                v[e] = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540u | (uint32_t)(e & 3))) - 8388736.f, s);
            }
            if (c < width) store_some<false, 8>(y + c, 8, v);
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
    auto ragged = [&](auto r) {
        constexpr bool R = decltype(r)::value;
        if (dtype == LUMI_DTYPE_F32) return act ? go(GateSource<float, true, R>{}) : go(GateSource<float, false, R>{});
        return act ? go(GateSource<__nv_bfloat16, true, R>{}) : go(GateSource<__nv_bfloat16, false, R>{});
    };
    return width % (dtype == LUMI_DTYPE_F32 ? 4 : 8) != 0 ? ragged(std::true_type{}) : ragged(std::false_type{});
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
    auto go = [&](auto* to, auto one) {
        using YT = std::remove_pointer_t<decltype(to)>;
        return cudaLaunchKernelEx(&cfg, dequant_kernel<YT, decltype(one)::value>, (const int8_t*)q, (long)ldq, (const float*)scale, to, (long)ldy, rows, width);
    };
    const bool one = width % 8 != 0 || !aligned_rows(y, y_dtype, ldy);
    if (y_dtype == LUMI_DTYPE_F32) LUMI_CUDA(one ? go((float*)y, std::true_type{}) : go((float*)y, std::false_type{}));
    else LUMI_CUDA(one ? go((__nv_bfloat16*)y, std::true_type{}) : go((__nv_bfloat16*)y, std::false_type{}));
    return LUMI_OK;
}
