// What the kernels of the attention over drafted trees share.
#pragma once

#include "common.cuh"

namespace attn_tree {
constexpr int MAX_KEYS = 1 << 30;     // of one request: places and their sums stay in 32 bits
enum : int { ERR_PAGE = 4, ERR_BOUNDS = 7 };
}  // namespace attn_tree
