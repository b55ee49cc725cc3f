// The norms around a block in one pass over its rows: x += scale * g * (o / rms(o)) * w_post, y = x / rms(x) * w_pre, rms(t) = sqrt(mean t^2 + eps).
//
// A row lies in registers from its loads to its stores: o, x and the gates are read once, x and y written once.  Two reductions in turn (the second norm needs the sum of the first), both of
// fp32 numbers.  Memory bounds it.
#include "device_args.h"
#include "rows.cuh"

#include <algorithm>
#include <type_traits>

namespace lumi {
namespace {

constexpr int kMaxWidth = 32768;                           // 1024 threads of four eights

struct BlockNormArgs {
    void* x; const void *o, *gate; void* y;
    const float *post, *pre;
    long ldx, ldo, ldg, ldy;
    int rows, width;
    float scale, eps;
};

template <typename T>
struct Eight { uint4 u[sizeof(T) / 2]; };

// Eight numbers, of which the row has n; none behind it are touched.
template <typename T>
__device__ __forceinline__ void fetch(const T* p, int n, Eight<T>& w) {
    constexpr int N = sizeof(T) / 2;
#pragma unroll
    for (int i = 0; i < N; ++i) w.u[i] = make_uint4(0, 0, 0, 0);
    if (n >= 8) {
#pragma unroll
        for (int i = 0; i < N; ++i) w.u[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if (n > 0) {
        uint32_t* const u = reinterpret_cast<uint32_t*>(w.u);
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < n) {
                if constexpr (N == 2) u[i] = __float_as_uint(p[i]);
                else u[i / 2] |= (uint32_t)__bfloat16_as_ushort(p[i]) << (16 * (i % 2));
            }
    }
}
__device__ __forceinline__ void numbers(const Eight<float>& w, float (&t)[8]) {
    const uint32_t* const u = reinterpret_cast<const uint32_t*>(w.u);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void numbers(const Eight<__nv_bfloat16>& w, float (&t)[8]) {
    const uint32_t* const u = reinterpret_cast<const uint32_t*>(w.u);
#pragma unroll
    for (int i = 0; i < 4; ++i) { t[2 * i] = __uint_as_float(u[i] << 16); t[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}
__device__ __forceinline__ float stored(float v, const float*) { return v; }
__device__ __forceinline__ float stored(float v, const __nv_bfloat16*) { return __bfloat162float(__float2bfloat16_rn(v)); }
__device__ __forceinline__ void put(float* p, int n, const float (&t)[8]) {
    if (n >= 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(t[0], t[1], t[2], t[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(t[4], t[5], t[6], t[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i) if (i < n) p[i] = t[i];
    }
}
__device__ __forceinline__ void put(__nv_bfloat16* p, int n, const float (&t)[8]) {
    if (n >= 8) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(t[2 * i], t[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i) if (i < n) p[i] = __float2bfloat16_rn(t[i]);
    }
}

// Sums or maxima over the threads of a row: a warp, or the block.
template <bool WARP, bool MAX>
__device__ __forceinline__ float over_row(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? fmaxf(v, w) : v + w;
    }
    if constexpr (!WARP) {
        const int warps = blockDim.x >> 5;
        __syncthreads();                                   // the last reduction's numbers have been read
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = red[0];
        for (int w = 1; w < warps; ++w) v = MAX ? fmaxf(v, red[w]) : v + red[w];
    }
    return v;
}

// 1 / sqrt(mean t^2 + eps).  Squares that leave fp32's range, or that vanish beside a tiny eps, are taken of the numbers times a power of two.
template <bool WARP, int NC>
__device__ __forceinline__ float inverse_rms(const float (&t)[NC][8], int width, float eps, float* red) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(t[c][i], t[c][i], s);
    s = over_row<WARP, false>(s, red);
    if (s < 3.4e38f && (s > 8.3e-25f || eps > 8.5e-22f)) return __frcp_rn(__fsqrt_rn(__fdiv_rn(s, (float)width) + eps));     // (uniform)
    float m = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(t[c][i]));
    m = over_row<WARP, true>(m, red);
    if (!(s == s) || !(m <= 3.4028235e38f) || m == 0.f) return __frcp_rn(__fsqrt_rn(__fdiv_rn(s, (float)width) + eps));
    const float k = ldexpf(1.f, max(-126, min(60, -ilogbf(m))));
    s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) { const float v = t[c][i] * k; s = fmaf(v, v, s); }
    s = over_row<WARP, false>(s, red);
    return __fmul_rn(k, __frcp_rn(__fsqrt_rn(__fdiv_rn(s, (float)width) + eps * k * k)));
}

template <typename XT, typename OT, typename YT, bool WARP, int NC>
__global__ void __launch_bounds__(WARP ? 128 : 1024) block_norm_kernel(BlockNormArgs a) {
    __shared__ float red[32];
    const int lane = WARP ? threadIdx.x & 31 : threadIdx.x, step = WARP ? 32 : blockDim.x;
    const long row = WARP ? (long)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    pdl_release();
    pdl_sync();
    if (WARP && row >= a.rows) return;
    XT* const x = (XT*)a.x + row * a.ldx;
    const OT* const o = (const OT*)a.o + row * a.ldo;
    const OT* const g = (const OT*)a.gate + row * a.ldg;
    Eight<OT> ow[NC], gw[NC];
    Eight<XT> xw[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int at = (c * step + lane) * 8, n = a.width - at;
        fetch(o + at, n, ow[c]);
        fetch(x + at, n, xw[c]);
        if (a.gate != nullptr) fetch(g + at, n, gw[c]);
    }
    float t[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) numbers(ow[c], t[c]);
    const float by = a.post != nullptr ? inverse_rms<WARP, NC>(t, a.width, a.eps, red) : 1.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int at = (c * step + lane) * 8, n = a.width - at;
        Eight<float> w;
        float f[8], v[8];
        if (a.post != nullptr) {
            fetch(a.post + at, n, w);
            numbers(w, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[c][i] = t[c][i] * by * f[i];
        }
        if (a.gate != nullptr) {
            numbers(gw[c], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[c][i] *= f[i];
        }
        numbers(xw[c], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) t[c][i] = stored(fmaf(a.scale, t[c][i], v[i]), x);
        put(x + at, n, t[c]);
        if (n < 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (i >= n) t[c][i] = 0.f;      // (behind the row: a scale that is no number would leave one here)
        }
    }
    if (a.y == nullptr) return;
    const float norm = inverse_rms<WARP, NC>(t, a.width, a.eps, red);
    YT* const y = (YT*)a.y + row * a.ldy;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int at = (c * step + lane) * 8, n = a.width - at;
        Eight<float> w;
        float f[8];
        fetch(a.pre + at, n, w);
        numbers(w, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = t[c][i] * norm * f[i];
        put(y + at, n, f);
    }
}

template <typename XT, typename OT, typename YT>
cudaError_t launch(const BlockNormArgs& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // the launch itself overlaps the kernel in front
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.stream = st;
    const int eights = (a.width + 7) / 8;
    auto warps = [&](auto kernel) {
        cfg.gridDim = dim3((unsigned)(((long)a.rows + 3) / 4));
        cfg.blockDim = dim3(128);
        return cudaLaunchKernelEx(&cfg, kernel, a);
    };
    auto blocks = [&](auto kernel, int nc) {
        cfg.gridDim = dim3((unsigned)a.rows);
        cfg.blockDim = dim3((unsigned)(((eights + nc - 1) / nc + 31) / 32 * 32));
        return cudaLaunchKernelEx(&cfg, kernel, a);
    };
    if (eights <= 32) return warps(block_norm_kernel<XT, OT, YT, true, 1>);
    if (eights <= 64) return warps(block_norm_kernel<XT, OT, YT, true, 2>);
    // two eights per thread from 1024 numbers on: 16384 x 2048 bf16 rows with gates 57 us, with one 71, with four 71; 3000 x 700 fp32 rows 12 us, with one 9.7
    if (eights < 128) return blocks(block_norm_kernel<XT, OT, YT, false, 1>, 1);
    if (eights <= 2048) return blocks(block_norm_kernel<XT, OT, YT, false, 2>, 2);
    return blocks(block_norm_kernel<XT, OT, YT, false, 4>, 4);
}

bool known(int dtype) { return dtype == LUMI_DTYPE_F32 || dtype == LUMI_DTYPE_BF16; }
bool aligned_rows(uint64_t p, int dtype, int ld) { return (p & 15) == 0 && ld % (dtype == LUMI_DTYPE_F32 ? 4 : 8) == 0; }

}  // namespace
}  // namespace lumi

using namespace lumi;

extern "C" int32_t lumi_k_block_norm(uint64_t x, int32_t x_dtype, int32_t ldx, uint64_t o, int32_t o_dtype, int32_t ldo, uint64_t w_post, uint64_t gate, int32_t ldg, float scale,
                                     uint64_t w_pre, uint64_t y, int32_t y_dtype, int32_t ldy, int32_t rows, int32_t width, float eps, uint64_t stream) {
    if (!x || !o || !known(x_dtype) || !known(o_dtype) || (y && (!known(y_dtype) || !w_pre)) || rows < 0 || width <= 0 || ldx < width || ldo < width ||
        (gate && ldg != 0 && ldg < width) || (y && ldy < width) || ((w_post || y) && !(eps > 0.f && eps <= 3.4e38f)))
        return fail(LUMI_E_INVALID, "bad argument to lumi_k_block_norm");
    if (!aligned_rows(x, x_dtype, ldx) || !aligned_rows(o, o_dtype, ldo) || (gate && !aligned_rows(gate, o_dtype, ldg)) || (y && !aligned_rows(y, y_dtype, ldy)) || (w_post & 15) ||
        (w_pre & 15))
        return fail(LUMI_E_INVALID, "lumi_k_block_norm: rows have to begin on 16-byte boundaries");
    if (width > kMaxWidth) return fail(LUMI_E_UNSUPPORTED, "lumi_k_block_norm: width %d (at most %d)", width, kMaxWidth);
    if (rows == 0) return LUMI_OK;
    LUMI_TRY(check_device_memory("lumi_k_block_norm", {x, o, w_post, gate, y ? w_pre : 0, y}));
    const BlockNormArgs a{(void*)x, (const void*)o, (const void*)gate, (void*)y, (const float*)w_post, (const float*)w_pre, ldx, ldo, gate ? ldg : 0, ldy, rows, width, scale, eps};
    const cudaStream_t st = (cudaStream_t)stream;
    auto types = [&](auto xt, auto ot) {
        using XT = decltype(xt);
        using OT = decltype(ot);
        return y && y_dtype == LUMI_DTYPE_BF16 ? launch<XT, OT, __nv_bfloat16>(a, st) : launch<XT, OT, float>(a, st);
    };
    const bool xb = x_dtype == LUMI_DTYPE_BF16, ob = o_dtype == LUMI_DTYPE_BF16;
    LUMI_CUDA(xb ? (ob ? types(__nv_bfloat16(), __nv_bfloat16()) : types(__nv_bfloat16(), float())) : (ob ? types(float(), __nv_bfloat16()) : types(float(), float())));
    return LUMI_OK;
}
