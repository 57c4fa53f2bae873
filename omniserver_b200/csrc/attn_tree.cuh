// What the kernels of the attention over drafted trees share.
#pragma once

#include "common.cuh"

namespace attn_tree {
constexpr int MAX_KEYS = 1 << 30;     // of one request: places and their sums stay in 32 bits
enum : int { ERR_PAGE = 4, ERR_BOUNDS = 7 };

// What a CTA has under way that writes to or reads from its memory by itself: it must not go before that is done, in whatever place its
// warps gave up. Tile i of a ring of copies is put into place i % STAGES, when the tile STAGES before it has been used up: so a
// place has one tile on its way at most, the one put there last, and its barrier's phase i / STAGES ends when it has landed.
template <int STAGES> struct UnderWay {
  int tile[STAGES];     // put into each place last, -1: none
  int q, s, pv;         // loads of Q and products of both kinds that were issued; they complete in this order
  __host__ __device__ void clear() {
    for (int k = 0; k < STAGES; ++k) tile[k] = -1;
    q = s = pv = 0;
  }
  __host__ __device__ void put(int i) { tile[i % STAGES] = i; }
  // the phase of place k's barrier that has to end, -1: none
  __host__ __device__ int phase(int k) const { return tile[k] < 0 ? -1 : tile[k] / STAGES; }
};
}  // namespace attn_tree
