// The layout of the paged cache in 4 bits, shared by the kernels that fill it
// and that read it.
//
// Codes of a head lie in the order of the attention's operand registers, so
// that its lanes load their part of a row in one piece.  With the head's
// values padded to W = 64, 96, 128 or 256 and blocks of 32 of them:
//   keys: a word holds the 8 values 32j + 8t ... + 7 (from the lowest nibble
//     up), for lane t of four and block j; a lane's words of an even number of
//     blocks lie together, those of a last odd block (W = 96) behind;
//   values: 16 bits hold the 4 values 32j + 4g ... + 3, for lane g of eight
//     and block j; again a lane's even number of blocks lie together.  Two
//     tokens of a page next to each other share words, the even one's 16 bits
//     in the low halves: the operand's registers pair keys.
// A head's scales are a word for each group: step's bfloat16 bits in the high
// half, low's in the low half; their number is rounded up to a power of two.
// Token o of page p of head h is record (p * heads + h) * page_size + o of the
// keys and of both scales, and in pair (p * heads + h) * pairs + o / 2 of the
// values, pairs = (page_size + 1) / 2: a head's tokens of a page lie together.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../common.hpp"
#include "decode.cuh"

namespace pfb {

inline int cache4_width(int64_t head_dim) {
  return head_dim <= 64 ? 64 : head_dim <= 96 ? 96 : head_dim <= 128 ? 128 : 256;
}

inline int cache4_groups(int64_t head_dim, int64_t group) {  // words of a record's scales
  int n = 1;
  while (n * group < cache4_width(head_dim)) n *= 2;
  return n;
}

// Word of a key row that holds values 8 * chunk ... + 7.
__host__ __device__ __forceinline__ int cache4_key_word(int chunk, int blocks) {
  const int j = chunk >> 2, t = chunk & 3, even = blocks & ~1;
  return j < even ? t * even + j : 4 * even + t;
}

// 16-bit place in a value row of values 4 * part ... + 3.
__host__ __device__ __forceinline__ int cache4_value_half(int part, int blocks) {
  const int j = part >> 3, g = part & 7, even = blocks & ~1;
  return j < even ? g * even + j : 8 * even + g;
}

inline void check_cache4(const pfk_cache4& c) {
  PFB_CHECK_ARG(c.num_pages >= 1 && c.page_size >= 1 && c.heads >= 1, "4-bit cache: sizes must be positive");
  PFB_CHECK_ARG(c.head_dim >= 8 && c.head_dim % 8 == 0 && c.head_dim <= 256, "4-bit cache: head_dim must be a multiple of 8, at most 256");
  PFB_CHECK_ARG(c.group == 32 || c.group == 64 || c.group == 128, "4-bit cache: group must be 32, 64 or 128");
  PFB_CHECK_ARG(c.num_pages <= INT32_MAX && c.page_size <= INT32_MAX && c.num_pages * c.page_size <= INT32_MAX,
                "4-bit cache: 2^31 tokens or more");
  PFB_CHECK_ARG(c.heads <= 65536 && c.num_pages * c.page_size * c.heads < 0xffffffffll, "4-bit cache: 2^32 - 1 or more heads of tokens");
  PFB_CHECK_ARG(c.k && c.v && c.k_scales && c.v_scales, "4-bit cache: null pointer");
  PFB_CHECK_ARG((uintptr_t)c.k % 16 == 0 && (uintptr_t)c.v % 16 == 0 && (uintptr_t)c.k_scales % 16 == 0 && (uintptr_t)c.v_scales % 16 == 0,
                "4-bit cache: pointers must be 16-byte aligned");
}

}  // namespace pfb
