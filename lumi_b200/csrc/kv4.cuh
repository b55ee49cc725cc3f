// Layout of a cache in 4 bits, shared by the kernels that write, read and attend to it.
//
// A page holds 64 tokens and has one block per head of keys and values.  A token's numbers go in groups of 32 (the last one may be shorter): codes n = 8 + rint(t / s), scale s (bf16).
// Block: keys' codes [group][token][16 bytes], keys' scales [group][token], values' codes, values' scales.
//
// Codes of values lie in their order, two in a byte.  A group of keys is four words of eight; number e of a word is nibble e / 2 + 4 (e % 2).  So (word >> 4 p) & 0x000f000f
// holds numbers 2 p and 2 p + 1 as two halves: codes as the smallest subnormals of fp16, which the tensor cores take as they are (n 2^-24, no conversion).  Of values the
// matrix load that transposes pairs two tokens' words instead.  A group's 16 bytes are one row of such a load in both cases.
#pragma once
#include "internal.h"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

namespace lumi {

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
    int wide_q, wide_y, wide_y16;                          // rows and heads of q lie on boundaries of 16 bytes; of y on those of four numbers, of 16 bytes
    int slots, slot_bytes;                                 // of a warp's ring
    int skip;                                              // failure tests: the copy of this page of the line is not issued
    float scale;
};
int32_t launch_kv4_prompt(const AttendArgs& a, bool f32, uint64_t work, cudaStream_t st);      // kv4_prompt.cu: sequences of more than a.few columns

namespace {

constexpr int kPage = 64;                                  // tokens
constexpr int kGroup = 32;                                 // numbers that share a scale
constexpr int kPlane = kPage * 16;                         // bytes of a group's codes
constexpr int kScales = kPage * 2;                         // bytes of a group's scales
constexpr int kMaxHead = 256;                              // numbers of a head
constexpr int kMaxPages = (1 << 25) - 1;                   // slots are 32-bit numbers

__host__ __device__ inline int kv4_groups(int d) { return (d + kGroup - 1) / kGroup; }
__host__ __device__ inline int kv4_part(int d) { return kv4_groups(d) * (kPlane + kScales); }
__host__ __device__ inline int kv4_block(int dk, int dv) { return kv4_part(dk) + kv4_part(dv); }

constexpr int kMaxRows = 1 << 24;                          // numbers of parts of work are 32-bit numbers
constexpr int kBadPage = 1;                                // bit of the status word: a page or a length outside of what the cache holds
constexpr float kLog2e = 1.4426950408889634f;

// ---- shared by the attention kernels
__device__ __forceinline__ float number(const float* p) { return *p; }
__device__ __forceinline__ float number(const __nv_bfloat16* p) { return __bfloat162float(*p); }
// Eight numbers on a 16-byte boundary, or none.
__device__ __forceinline__ void eight_numbers(const float* p, int n, float (&t)[8]) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    if (n > 0) { x = reinterpret_cast<const float4*>(p)[0]; y = reinterpret_cast<const float4*>(p)[1]; }
    t[0] = x.x; t[1] = x.y; t[2] = x.z; t[3] = x.w; t[4] = y.x; t[5] = y.y; t[6] = y.z; t[7] = y.w;
}
__device__ __forceinline__ void eight_numbers(const __nv_bfloat16* p, int n, float (&t)[8]) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (n > 0) x = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { t[2 * i] = __uint_as_float(u[i] << 16); t[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}
// Four results of a row, of which it has n.
__device__ __forceinline__ void put_four(float* p, int n, bool wide, const float (&t)[4]) {
    if (wide && n >= 4) *reinterpret_cast<float4*>(p) = make_float4(t[0], t[1], t[2], t[3]);
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < n) p[i] = t[i];
    }
}
__device__ __forceinline__ void put_four(__nv_bfloat16* p, int n, bool wide, const float (&t)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(t[0], t[1]), b = __floats2bfloat162_rn(t[2], t[3]);
    if (wide && n >= 4) *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    else {
        if (n > 0) p[0] = a.x;
        if (n > 1) p[1] = a.y;
        if (n > 2) p[2] = b.x;
        if (n > 3) p[3] = b.y;
    }
}
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unhalves(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ float low_bf16(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_bf16(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ long long quotient(long long n, long long d) {       // of numbers that are nearly always small
    return ((n | d) >> 32) == 0 ? (long long)((uint32_t)n / (uint32_t)d) : n / d;
}

// two fp32 operations in one
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void add2(float& d0, float& d1, float a0, float a1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%0, %1};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(d0), "+f"(d1) : "f"(a0), "f"(a1));
}

// What a sequence is to the call.
struct Sequence { int first, n, total, page0, pages, units; };
__device__ __forceinline__ bool lengths_of(const AttendArgs& a, int s, Sequence& q) {      // false: they make no sense
    q.first = a.row_start[s];
    const int end = a.row_start[s + 1];
    q.total = a.tokens[s];
    q.n = end - q.first;
    return q.first >= 0 && end >= q.first && end <= a.rows && q.total >= q.n && q.total <= (long)a.width * kPage;
}

}  // namespace
}  // namespace lumi
