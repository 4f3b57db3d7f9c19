// The 4-bit paged key/value cache: layout and bounds shared by its operators.
//
// A page holds `page` tokens (16, 32, 64, 128 or 256) of every kv head; a head's tokens come in blocks of 16, 640 contiguous bytes per
// group of 32 features.  A value is m + n s with n in 0..15 and a half-precision s and m per token and group:
//   keys    [group][key % 8][d % 8 / 2][d / 16 % 2] words; byte 2 (d % 2) + key / 8 of a word, low half d % 16 < 8, high half the rest
//   values  [group][d % 8][key % 8 / 2][d / 16 % 2] words; byte 2 (key % 2) + key / 8 of a word, low half d % 16 < 8, high half the rest
//   key scales, key minima      [group][key % 8][key / 8] halves
//   value scales, value minima  [group][key % 8 / 2][key / 8][key % 2] halves
// A word is what one lane of an m16n8k16 MMA holds of a 16 x 16 tile (keys: rows = keys, columns = features; values: rows = features,
// columns = keys), and the scales stand in the order in which a lane needs them.  A byte belongs to one token, so tokens of a block can be
// written apart from one another.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace lmb {
namespace kv4 {

constexpr int kGroup = 32;                 // features that share a scale and a minimum
constexpr int kMostTokens = 1 << 30;       // of a sequence, and rows of a call: sums of two stay below 2^31
constexpr int kErrPage = 1;                // Ctx::dev_arg: a slot or a block table names a place outside the cache, or the rows do not fit together
constexpr int kErrFree = 2;                // the free list, the lengths and the tables do not fit together

__host__ __device__ inline int groups(int D) { return D / kGroup; }
__host__ __device__ inline int block_bytes(int D) { return 20 * D; }
__host__ __device__ inline int key_word(int key, int d) { return (d >> 5) * 64 + ((key & 7) * 4 + ((d & 7) >> 1)) * 2 + ((d >> 4) & 1); }
__host__ __device__ inline int key_byte(int key, int d) { return key_word(key, d) * 4 + 2 * (d & 1) + (key >> 3); }
__host__ __device__ inline int value_word(int key, int d) { return (d >> 5) * 64 + ((d & 7) * 4 + ((key & 7) >> 1)) * 2 + ((d >> 4) & 1); }
__host__ __device__ inline int value_byte(int key, int d) { return value_word(key, d) * 4 + 2 * (key & 1) + (key >> 3); }
__host__ __device__ inline int key_meta(int key, int g) { return g * 16 + (key & 7) * 2 + (key >> 3); }
__host__ __device__ inline int value_meta(int key, int g) { return g * 16 + ((key & 7) >> 1) * 4 + (key >> 3) * 2 + (key & 1); }

// page sizes the operators take, as a shift; -1 for any other
inline int page_shift(int page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

// The shape of a cache, checked the same way by every operator that takes one.
inline int32_t check_cache(const char* who, int n_kv_heads, int D, int n_pages, int page) {
  LMB_REQUIRE(page_shift(page) >= 0, "%s: page size %d (16, 32, 64, 128 or 256)", who, page);
  LMB_REQUIRE(D >= kGroup && D <= 256 && D % kGroup == 0, "%s: head_dim %d (a multiple of 32 up to 256)", who, D);
  LMB_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 65535, "%s: %d kv heads", who, n_kv_heads);
  LMB_REQUIRE(n_pages >= 1 && (int64_t)n_pages * page <= INT32_MAX, "%s: %d pages of %d tokens (at most 2^31 - 1 tokens)", who, n_pages, page);
  return LMB200_OK;
}

// Whether rows of `width` bytes, a_stride and b_stride bytes apart from a and b on, share no byte: arrays apart, or interleaved in the rows of one.
inline bool apart(const void* a, int64_t a_stride, const void* b, int64_t b_stride, int rows, int64_t width) {
  const int64_t off = (int64_t)((uintptr_t)b - (uintptr_t)a);
  if (off >= (rows - 1) * a_stride + width || -off >= (rows - 1) * b_stride + width) return true;
  if (rows == 1 || a_stride != b_stride) return false;
  const int64_t in = (off % a_stride + a_stride) % a_stride;
  return in >= width && in + width <= a_stride;
}

}  // namespace kv4
}  // namespace lmb
