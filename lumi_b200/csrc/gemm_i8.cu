// Products in 8-bit integers: D[m][n] = (sum over k of A[m][k] W[n][k]) * a_scale[m] * w_scale[n] + bias[n] (+ D[m][n]).  The sums are 32-bit
// integers and therefore exact in any order.
#include "device_args.h"

namespace lumi {
namespace {

struct I8Args {
    const int8_t *a, *w;
    const float *a_scale, *w_scale, *bias;
    void* d;
    long lda, ldw, ldd;
    int M, N, K, accumulate;
};

// A thread per result.
template <typename DT>
__global__ void __launch_bounds__(256) gemm_i8_kernel(I8Args g) {
    const int n = blockIdx.x * 32 + (threadIdx.x & 31), m = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (n >= g.N || m >= g.M) return;
    const int8_t *a = g.a + m * g.lda, *w = g.w + n * g.ldw;
    int sum = 0, k = 0;
    for (; k + 16 <= g.K; k += 16) {
        const int4 u = *reinterpret_cast<const int4*>(a + k), v = *reinterpret_cast<const int4*>(w + k);
        sum = __dp4a(u.x, v.x, sum); sum = __dp4a(u.y, v.y, sum); sum = __dp4a(u.z, v.z, sum); sum = __dp4a(u.w, v.w, sum);
    }
    for (; k < g.K; ++k) sum += (int)a[k] * (int)w[k];
    float r = (float)sum * g.a_scale[m] * g.w_scale[n];
    if (g.bias != nullptr) r += g.bias[n];
    DT* d = (DT*)g.d + m * g.ldd + n;
    if (g.accumulate) r += (float)*d;
    *d = (DT)r;
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
    const I8Args g{(const int8_t*)a, (const int8_t*)w, (const float*)a_scale, (const float*)w_scale, (const float*)bias, (void*)d, lda, ldw, ldd, M, N, K, accumulate};
    const dim3 grid((N + 31) / 32, (M + 7) / 8);
    if (d_dtype == LUMI_DTYPE_F32) gemm_i8_kernel<float><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
    else gemm_i8_kernel<__nv_bfloat16><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
    LUMI_CUDA(cudaGetLastError());
    return LUMI_OK;
}
