// What the kernels of the attention over drafted trees share.
#pragma once

#include "common.cuh"

namespace attn_tree {
constexpr int MAX_KEYS = 1 << 30;     // of one request: places and their sums stay in 32 bits
enum : int { ERR_PAGE = 4, ERR_BOUNDS = 7 };

// What a producer put into a place of a ring of copies last (-1: nothing). Tile i is put into place i % STAGES when the tile STAGES before
// it has been used up: so a place has one tile under way at most, the last one that any producer put there, and phase i / STAGES of the
// place's barrier ends when it has landed.
template <int STAGES> struct LastPut {
  int tile = -1;
  __host__ __device__ __forceinline__ void put(int place, int i) {
    if (place == (int)((unsigned)i % STAGES)) tile = i;
  }
};
}  // namespace attn_tree
