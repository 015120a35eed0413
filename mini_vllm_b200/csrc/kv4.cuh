// A layer's paged cache of keys and values in 4 bits.
//
// A row is one token's key (or value) of one KV head: D channels in groups of 64.  With m and M a group's least and greatest value,
//     minimum m,   scale s = bf16((M - m) * fp32(1/15)),   code c = round((x - m) / s) held to 0..15,   the row stands for m + s c.
// A value that is not finite makes m or s so: no channel of its group is read as a number that could pass for one.
// Codes lie in [blocks, kv heads, block_size, D / 2] bytes, (s, m) as a bf16 pair in [blocks, kv heads, block_size, D / 64, 2]: a head's
// tokens are contiguous inside a block, so 32 tokens of a head are one piece of memory.  4.5 bits a value, against 16.
//
// A 32-bit word holds eight neighbouring channels 8 L .. 8 L + 7: the even ones in its low half, the odd ones in its high half, four bits
// each, so that one AND leaves channels (2 i, 2 i + 1) in the two halves of a register.  Such a masked half is, read as fp16, the
// subnormal c * 2^-24 (bits 0-3) or c * 2^-20 (bits 4-7): exact, without any conversion, and what the tensor core takes.
// The words of a row are ordered for the fragments of mma.m16n8k16:
//     keys    word (D / 32) c + j holds L = 4 j + c:  lane c of a quad reads its D / 32 words in one piece, word j of the four lanes makes
//             up two K steps, and a group of 64 channels is two consecutive j
//     values  word (D / 64) g + j holds L = 8 j + g:  lane g of eight reads its D / 64 words in one piece, word j is of group j
#pragma once
#include <stdint.h>

#include "common.cuh"
#include "mini_vllm_b200.h"

namespace mvb {

constexpr int kKv4Group = 64;         // channels that share a scale and a minimum
constexpr int kKv4Span = 64;          // tokens that share a pair of bounds (and the grain of the lists of spans)

// the word of a row that holds channels 8 L .. 8 L + 7
template <int D>
__host__ __device__ __forceinline__ int kv4_word(int L, bool keys) {
  return keys ? (D / 32) * (L & 3) + (L >> 2) : (D / 64) * (L & 7) + (L >> 3);
}

// the 4-bit place of channel e (0..7) inside its word
__host__ __device__ __forceinline__ constexpr int kv4_shift(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

// row of (block, head, token of the block)
__host__ __device__ __forceinline__ int64_t kv4_row(int64_t block, int hkv, int head, int block_size, int token) {
  return (block * hkv + head) * block_size + token;
}

__device__ __forceinline__ float kv4_scale(uint32_t affine) { return __uint_as_float(affine << 16); }
__device__ __forceinline__ float kv4_min(uint32_t affine) { return __uint_as_float(affine & 0xffff0000u); }

// What the eight codes of a word stand for; the product is exact in fp32 and the sum is rounded once.  A code becomes a float as the last
// bits of 2^23 + 16^i c, less 2^23 and over 16^i in one exact step: one integer instruction a code, the rest on the multipliers.
__device__ __forceinline__ void kv4_values(uint32_t word, uint32_t affine, float (&v)[8]) {
  const float2 s = make_float2(kv4_scale(affine), kv4_scale(affine)), m = make_float2(kv4_min(affine), kv4_min(affine));
  const uint32_t upper = word >> 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {                              // channels 2 i and 2 i + 1
    const uint32_t mask = 15u << (4 * i);
    const float unit = 1.f / static_cast<float>(1u << (4 * i)), less = -8388608.f * unit;
    const float2 x = make_float2(__uint_as_float((word & mask) | 0x4b000000u), __uint_as_float((upper & mask) | 0x4b000000u));
    const float2 y = fma_f32x2(s, fma_f32x2(x, make_float2(unit, unit), make_float2(less, less)), m);
    v[2 * i] = y.x; v[2 * i + 1] = y.y;
  }
}

inline bool kv4_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// what every entry point asks of a cache
inline int kv4_check(const mvb_kv4_cache* c) {
  if (c == nullptr || !c->k_codes || !c->k_affine || !c->v_codes || !c->v_affine || c->num_blocks <= 0 || c->block_size <= 0 ||
      c->num_kv_heads <= 0)
    return kInvalidArgument;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return kUnsupportedShape;
  if (c->block_size % kKv4Span != 0 || c->num_blocks > 0x7fffffffLL / c->block_size) return kUnsupportedShape;
  if (!kv4_aligned(c->k_codes, 16) || !kv4_aligned(c->v_codes, 16) || !kv4_aligned(c->k_affine, 16) || !kv4_aligned(c->v_affine, 16))
    return kMisaligned;
  return kOk;
}

// x / n by a multiplication (Granlund and Montgomery, 1994), for x < 2^31 and 1 <= n < 2^31
struct FastDiv {
  uint32_t n, mul, shift;
  FastDiv() = default;
  explicit FastDiv(uint32_t d) : n(d) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __host__ __device__ __forceinline__ uint32_t div(uint32_t x) const {
#ifdef __CUDA_ARCH__
    const uint32_t hi = __umulhi(x, mul);
#else
    const uint32_t hi = static_cast<uint32_t>((static_cast<uint64_t>(x) * mul) >> 32);
#endif
    return (hi + x) >> shift;                                // no overflow: both are below 2^31
  }
};

}  // namespace mvb
