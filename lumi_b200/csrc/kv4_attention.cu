// Attention over a paged cache in 4 bits: y = softmax(scale q K^T) V for the rows of sequences of different lengths, with an optional sliding window and an optional sink (one more
// score, 0, without a value).  Row i of a sequence's n new rows stands at position tokens - n + i and sees the positions up to its own.
#include "device_args.h"
#include "kv4.cuh"
#include "rows.cuh"

#include <algorithm>

namespace lumi {
namespace {

struct AttendArgs {
    const void* q; void* y;
    const uint8_t* kv;
    const int32_t *table, *row_start, *tokens;
    int32_t* status;
    long ldq, ldy;
    int heads, kv_heads, dk, dv, window, sink, nseq, rows, max_new, n_pages, width;
    float scale;
};

constexpr int kMaxRows = 1 << 24;                          // numbers of parts of work are 32-bit numbers
constexpr int kBadPage = 1;                                // bit of the status word: a page or a length outside of what the cache holds

__device__ __forceinline__ float number(const float* p) { return *p; }
__device__ __forceinline__ float number(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float code_value(const uint8_t* part, int groups, int token, int d, bool keys) {
    const int g = d / kGroup, i = d % kGroup, nibble = keys ? i / 8 * 8 + (i % 8) / 2 + 4 * (i & 1) : i;
    const int n = part[g * kPlane + token * 16 + nibble / 2] >> (4 * (nibble & 1)) & 15;
    const uint32_t s = *reinterpret_cast<const uint16_t*>(part + groups * kPlane + g * kScales + token * 2);
    return (float)(n - 8) * __uint_as_float(s << 16);
}

// One block per row and head: a page at a time, a thread per token for the scores, a thread per number for the values.
template <typename T>
__global__ void __launch_bounds__(128) kv4_simple_kernel(AttendArgs a) {
    __shared__ float q[kMaxHead], p[kPage], red[2];
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    pdl_release();
    pdl_sync();
    int lo = 0, hi = a.nseq;                               // the sequence: the last one that starts at or before the row
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.row_start[mid] <= row) lo = mid; else hi = mid; }
    const int first = a.row_start[lo], n = a.row_start[lo + 1] - first, total = a.tokens[lo];
    if (row < first || row >= first + n) return;
    const int pos = total - n + row - first;
    if (first < 0 || first + n > a.rows || total > (long)a.width * kPage || total < n) {
        if (tid == 0 && a.status != nullptr) atomicOr(a.status, kBadPage);
        return;
    }
    if (n > a.max_new) return;
    for (int i = tid; i < a.dk; i += 128) q[i] = number((const T*)a.q + row * a.ldq + head * a.dk + i);
    __syncthreads();
    const int group = a.heads / a.kv_heads, from = a.window > 0 ? max(0, pos - a.window + 1) : 0, gk = kv4_groups(a.dk), gv = kv4_groups(a.dv);
    float m = a.sink ? 0.f : -INFINITY, sum = a.sink ? 1.f : 0.f, acc[2] = {0.f, 0.f};
    for (int page0 = from / kPage; page0 * kPage <= pos; ++page0) {
        const int page = a.table[(size_t)lo * a.width + page0];
        if (page < 0 || page >= a.n_pages) {
            if (tid == 0 && a.status != nullptr) atomicOr(a.status, kBadPage);
            continue;
        }
        const uint8_t* const block = a.kv + ((size_t)page * a.kv_heads + head / group) * kv4_block(a.dk, a.dv);
        const int at = page0 * kPage + tid;
        float x = -INFINITY;
        if (tid < kPage && at >= from && at <= pos) {
            float s = 0.f;
            for (int d = 0; d < a.dk; ++d) s = fmaf(q[d], code_value(block, gk, tid, d, true), s);
            x = s * a.scale;
        }
        if (tid < kPage) {
            float t = x;
            for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
            if (isnan(x)) t = x;
            if ((tid & 31) == 0) red[tid >> 5] = t;
        }
        __syncthreads();
        const float top = fmaxf(m, fmaxf(red[0], red[1])), by = top == -INFINITY ? 1.f : expf(m - top);
        if (tid < kPage) p[tid] = x == -INFINITY ? 0.f : expf(x - top);
        __syncthreads();
        float part = 0.f;
        for (int i = 0; i < kPage; ++i) part += p[i];
        sum = sum * by + part;
        for (int e = 0; e < 2; ++e) {
            const int d = tid + 128 * e;
            if (d >= a.dv) continue;
            float s = acc[e] * by;
            for (int i = 0; i < kPage; ++i)
                if (page0 * kPage + i >= from && page0 * kPage + i <= pos) s = fmaf(p[i], code_value(block + kv4_part(a.dk), gv, i, d, false), s);
            acc[e] = s;
        }
        m = top;
        __syncthreads();
    }
    for (int e = 0; e < 2; ++e) {
        const int d = tid + 128 * e;
        if (d < a.dv) put((T*)a.y + row * a.ldy + head * a.dv + d, sum == 0.f ? 0.f : acc[e] / sum);
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
    const AttendArgs a{(const void*)q, (void*)y, (const uint8_t*)kv, (const int32_t*)page_table, (const int32_t*)row_start, (const int32_t*)tokens, (int32_t*)status, ldq, ldy,
                       heads, kv_heads, dk, dv, window, sink != 0, nseq, rows, max_new, n_pages, pages_per_seq, scale};
    const cudaStream_t st = (cudaStream_t)stream;
    if (f32) LUMI_CUDA(launch_rows(kv4_simple_kernel<float>, dim3((unsigned)rows, (unsigned)heads), 128, 0, st, a));
    else LUMI_CUDA(launch_rows(kv4_simple_kernel<__nv_bfloat16>, dim3((unsigned)rows, (unsigned)heads), 128, 0, st, a));
    return LUMI_OK;
}
