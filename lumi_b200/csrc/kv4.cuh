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

namespace lumi {
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

}  // namespace
}  // namespace lumi
