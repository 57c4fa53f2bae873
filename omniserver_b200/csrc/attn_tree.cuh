// What the kernels of the attention over drafted trees share: where a long request's keys are cut.
#pragma once

#include "common.cuh"

namespace attn_tree {
constexpr int MAX_SPLITS = 32;
constexpr int MIN_SPLIT_KEYS = 256;
constexpr int MAX_KEYS = 1 << 30;     // of one request: places and their sums stay in 32 bits
enum : int { ERR_PAGE = 4, ERR_BOUNDS = 7 };

// Keys per range of a request of kv_len keys in the 32-bit kernel: a function of the request's own length alone.
__host__ __device__ __forceinline__ int split_keys(int kv_len) {
  const int per = kv_len <= 0 ? 1 : (kv_len - 1) / MAX_SPLITS + 1;
  return (per + MIN_SPLIT_KEYS - 1) / MIN_SPLIT_KEYS * MIN_SPLIT_KEYS;
}
__host__ __device__ __forceinline__ int num_ranges(int kv_len) {
  return kv_len <= 0 ? 1 : (kv_len - 1) / split_keys(kv_len) + 1;
}
}  // namespace attn_tree
