// Attention of a tree of drafted tokens over the paged cache on the fifth-generation tensor cores (bf16, head sizes 64 and 128).
//
// What a node sees, and its formula: attn_tree.cu. The query rows of a request and kv head are its nodes times the group's heads
// (row = node x group + head), so that one pass over the keys serves the whole group: a unit of work is one (request, kv head, tile
// of up to 128 rows, range of keys), a tile being whole nodes. Q comes with one 3-D TMA box (64 dims, the group's heads, nodes) per
// half of the head; keys and values as in attn_prefill_tc.cu, from which the rest of the pipeline is taken too: K and V tiles of
// 128 keys gathered page by page into a ring of three stages, S = Q K^T and O += P V as tcgen05.mma issued by one thread each, S, P
// (bf16) and O in tensor memory, two groups of four softmax warps that take key tiles in turn and pass a row's exponent offset on,
// an offset that moves only when the maximum has grown by more than 2^8.
// What bounds it: up to one tile of rows per kv head the keys and values (a tile of 128 keys is 64 KB, 1.5 us at a
// 148th of the memory's rate, against some 0.5 us for its products and softmax); with more rows the two products
// (about 1,000 cycles for 128 x 128 x 128 each way, the softmax of one group just beside it).
//
// Keys are cut into as many ranges per request as fill the SMs (osb_attn_tree_tc_splits); a range leaves its unnormalised fp32
// output, maximum and sum in scratch, laid out [4 dims][row] so that neighbouring threads (rows) write neighbouring 16 bytes straight
// from tensor memory, and a second kernel joins them in order. The CTAs of one launch never wait for one another.
//
// Masks. A tile of keys that are all committed and inside every row's window needs none. Otherwise a row's 128 bits come from its
// mask words (places before the tree count as ones). P is 0 where a row does not see a key, but 0 times a NaN or an infinity in V
// would still reach the row through the tensor core: in such tiles the values that are not finite are replaced by zeros in shared
// memory, and if there were any, the rows that do see them get them added at the end, from the cache.
#include "attn_tree.cuh"
#include "tc_utils.cuh"

namespace {
using namespace tc;
using namespace attn_tree;

constexpr int BLOCK_M = 128, TILE_N = 128;
constexpr int NUM_THREADS = 384;
constexpr int SOFTMAX_REGS = 216, OTHER_REGS = 64;   // 256 x 216 + 128 x 64 registers of the 64 K
constexpr int STAGES = 3;  // K and V tiles in flight
constexpr int ATOM_BYTES = 128 * 128;  // 128 rows of 128 bytes
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_THRESHOLD = 8.0f;  // in log2 units
constexpr int MAX_TC_SPLITS = 64;

// The step and how it is cut, the same for every item.
struct Plan {
  const int* block_table;
  const int* cu_q;
  const int* seq_lens;
  const unsigned* mask;
  const int* depth;
  int* err;
  int bt_stride, mask_words, S, nh, nkv, grp, log2ps, num_pages, window, max_q_len, kv_cap;
  int nodes_per_tile, m_tiles, splits, chunk_tiles, n_items;
};

// Key tiles that a request's rows look at: the first, how many, and into how many ranges of how many tiles they are cut.
struct Cut {
  int first, count, ranges, per;
};
__device__ __forceinline__ Cut cut_of(const Plan& p, int kv_len, int base) {
  const int lo = p.window > 0 && base - p.window + 1 > 0 ? min(base - p.window + 1, kv_len - 1) : 0;
  Cut c;
  c.first = lo / TILE_N;
  c.count = (kv_len - 1) / TILE_N - c.first + 1;
  c.ranges = min(p.splits, (c.count + p.chunk_tiles - 1) / p.chunk_tiles);
  c.per = (c.count + c.ranges - 1) / c.ranges;
  c.ranges = (c.count + c.per - 1) / c.per;
  return c;
}

// One unit of work.
struct Item {
  int s, kvh, node0, q0, n, rows, kv_len, base, tile_begin, n_tiles, ranges;
  const int* bt;
};

// idx = ((request x kv heads + head) x ranges + range) x row tiles + tile: the tiles of one range run side by side, and the second to
// read its keys finds them in the L2
__device__ __forceinline__ bool item_of(int idx, Item& it, const Plan& p) {
  const int m = idx % p.m_tiles;
  idx /= p.m_tiles;
  const int range = idx % p.splits;
  idx /= p.splits;
  it.kvh = idx % p.nkv;
  it.s = idx / p.nkv;
  it.q0 = p.cu_q[it.s];
  it.n = p.cu_q[it.s + 1] - it.q0;
  it.node0 = m * p.nodes_per_tile;
  if (it.node0 >= it.n) return false;
  const int kv_all = p.seq_lens[it.s];
  it.kv_len = min(kv_all, p.kv_cap);
  it.base = kv_all - it.n;
  if (it.kv_len <= 0) {
    atomicExch(p.err, ERR_BOUNDS);
    return false;
  }
  const Cut c = cut_of(p, it.kv_len, it.base);
  if (range >= c.ranges) return false;
  it.ranges = c.ranges;
  it.tile_begin = c.first + range * c.per;
  it.n_tiles = min(c.per, c.count - range * c.per);
  it.rows = min(p.nodes_per_tile, it.n - it.node0) * p.grp;
  it.bt = p.block_table + (size_t)it.s * p.bt_stride;
  return true;
}

// Whether some row does not see some key of the tile from key0 on (depths are below the number of nodes).
__device__ __forceinline__ bool tile_masked(const Item& it, const Plan& p, int key0) {
  return key0 + TILE_N > min(it.base, it.kv_len) || (p.window > 0 && key0 < it.base + it.n - p.window);
}

// Which of the keys key0 .. key0 + 31 row `t` of the step sees; lo: the first place inside its window.
__device__ __forceinline__ unsigned sees32(const Item& it, const Plan& p, int t, int lo, int key0) {
  const int off = key0 - it.base;                       // of the tree's node numbers
  const unsigned* row = p.mask + (size_t)t * p.mask_words;
  auto word = [&](int i) -> unsigned { return i < 0 ? 0xffffffffu : i < p.mask_words ? row[i] : 0u; };
  unsigned v = __funnelshift_r(word(off >> 5), word((off >> 5) + 1), off & 31);
  const int left = it.kv_len - key0;
  v = left >= 32 ? v : left > 0 ? v & ((1u << left) - 1u) : 0u;
  if (p.window > 0) {
    const int hidden = min(lo, it.base) - key0;         // committed keys in front of the window
    v = hidden >= 32 ? 0u : hidden > 0 ? v & (0xffffffffu << hidden) : v;
    if (lo > it.base) {                                 // a window shorter than the path: ancestors by their depth
      for (unsigned w = v; w != 0; w &= w - 1) {
        const int j = off + __ffs(w) - 1;
        if (j >= 0 && it.base + p.depth[it.q0 + j] < lo) v &= ~(w & (0u - w));
      }
    }
  }
  return v;
}

// Bits 15 and 31 say which of two bf16 are not finite.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ uint32_t without_not_finite(uint32_t w) {
  const uint32_t b = not_finite(w);
  return w & ~((b & 0x8000u ? 0xffffu : 0u) | (b & 0x80000000u ? 0xffff0000u : 0u));
}

// Adds to a row's 32 outputs from column c0 on what was taken out of the V tiles: the values that are not finite of the keys that it
// sees, from the cache. Only reached when a masked tile held such values.
__device__ __noinline__ void add_not_finite(uint32_t (&o)[32], const Item& it, const Plan& p, int tok, int lo, const bf16* v_cache,
                                            int hd, int c0) {
  for (int t = 0; t < it.n_tiles; ++t) {
    const int tile0 = (it.tile_begin + t) * TILE_N;
    if (!tile_masked(it, p, tile0)) continue;
    for (int k0 = tile0; k0 < tile0 + TILE_N; k0 += 32)
      for (unsigned w = sees32(it, p, tok, lo, k0); w != 0; w &= w - 1) {
        const int key = k0 + __ffs(w) - 1, page = it.bt[key >> p.log2ps];
        if (page < 0 || page >= p.num_pages) continue;
        const int off = key & ((1 << p.log2ps) - 1);
        const bf16* v = v_cache + ((((size_t)page * p.nkv + it.kvh) << p.log2ps) + off) * hd + c0;
        for (int j = 0; j < 32; ++j) {
          const float f = __bfloat162float(v[j]);
          if (!(fabsf(f) < INFINITY)) o[j] = __float_as_uint(__uint_as_float(o[j]) + f);
        }
      }
  }
}

// Barrier of the eight softmax warps that also tells every one of them whether any saw `v`.
__device__ __forceinline__ bool softmax_bar_or(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 2, 256, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v)
      : "memory");
  return r != 0;
}

template <int HD>
__global__ void __launch_bounds__(NUM_THREADS, 1) attn_tree_tc_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
    const __grid_constant__ CUtensorMap map_v, bf16* __restrict__ out, float4* __restrict__ part_o,
    float2* __restrict__ part_ml, const bf16* __restrict__ v_cache, const __grid_constant__ Plan plan, float scale_log2,
    int* __restrict__ err) {
  constexpr int NA = HD / 64;                 // 64-element atoms along the head dimension
  constexpr int Q_BYTES = NA * ATOM_BYTES;    // [atom][128 rows][128 B]
  constexpr int KV_BYTES = NA * ATOM_BYTES;   // one K or V tile: [atom][128 keys][128 B]
  constexpr uint32_t TMEM_COLS = 512;
  // two S buffers of 128 columns (fp32), two P buffers of 64 columns (two bf16 per column), then O
  constexpr uint32_t S_COL0 = 0, P_COL0 = 2 * TILE_N, O_COL = 3 * TILE_N;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* q_smem = base;
  unsigned char* k_smem = q_smem + Q_BYTES;                  // STAGES tiles
  unsigned char* v_smem = k_smem + STAGES * KV_BYTES;     // STAGES tiles
  // The tiles a CTA works through are counted across its items: tile u uses K/V stage u % STAGES and S/P buffer u % 2.
  // k_free / s_full: Q K^T of a tile complete (the K tile may be overwritten / S may be read);
  // s_free: the softmax warps hold the tile's S in registers (the S buffer may be overwritten);
  // p_full: P of a tile is in tensor memory; v_free / p_free: P V of a tile complete (the V tile / the P buffer
  // may be overwritten, O may be read); epi_done: an item's output has left tensor and shared memory (the next
  // item's Q may be loaded; its first P V, which overwrites O, follows from that)
  __shared__ uint64_t q_full, epi_done, k_full[STAGES], v_full[STAGES], k_free[STAGES], v_free[STAGES];
  __shared__ uint64_t s_full[2], s_free[2], p_full[2], p_free[2];
  // max_done[u % 2]: the rows' exponent offsets after tile u are in row_offset (the group of tile u + 1 may go on)
  __shared__ uint64_t max_done[2];
  __shared__ float row_offset[BLOCK_M];   // per query row: the exponent offset in use (log2 units), -inf before the first key
  __shared__ float row_sum[2][BLOCK_M];   // per group and row: its sum of P at the final offset
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int found_bad[2];            // by the parity of the CTA's items: values that are not finite were taken out of a V tile

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ps = 1 << plan.log2ps, log2ps = plan.log2ps;
  const int box_rows = ps < TILE_N ? ps : TILE_N;  // keys per TMA box: a page, or a tile's worth of a larger page
  const int n_boxes = TILE_N / box_rows;

  if (lane == 0 && warp < 3) prefetch_tensormap(warp == 0 ? &map_k : warp == 1 ? &map_q : &map_v);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    found_bad[0] = found_bad[1] = 0;
    mbar_init(&q_full, 1);
    mbar_init(&epi_done, 8);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&k_free[i], 1);
      mbar_init(&v_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_free[i], 1);
    }
    mbar_init(&max_done[0], BLOCK_M);
    mbar_init(&max_done[1], BLOCK_M);
    mbar_init_fence();
  }
  if (threadIdx.x < BLOCK_M) row_offset[threadIdx.x] = -INFINITY;
  if (warp == 1) tmem_alloc(&tmem_slot, TMEM_COLS);
  // until here nothing was read that the kernel before this one in the stream may still be writing (q, the pages)
  pdl_wait();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* vabort = &abort_flag;
  Item it;
  int idx = 0;
  auto next_item = [&](int& pass) -> bool {   // the same sequence of items in every warp
    for (;;) {
      idx = (int)blockIdx.x + (int)gridDim.x * pass++;
      if (idx >= plan.n_items) return false;
      if (item_of(idx, it, plan)) return true;
    }
  };

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------ TMA producers: warp 0 keys, warp 2 values
    const int which = warp == 0 ? 0 : 1;
    unsigned char* tiles = which ? v_smem : k_smem;
    const CUtensorMap* map = which ? &map_v : &map_k;
    // lane = (box b, atom a) of a tile: boxes * NA <= 32, a box being at least 8 keys
    const int b = lane / NA, a = lane - b * NA;
    int u0 = 0;   // tiles of the items before this one
    int issued = 0;
    for (int pass = 0; next_item(pass) && !*vabort; u0 += it.n_tiles) {
      const int p_last = it.kv_len - 1;
      if (which == 0 && lane == 0 && (it.kv_len < it.base + it.n || it.n > plan.max_q_len || it.base < 0)) atomicExch(err, ERR_BOUNDS);
      // a page outside the pool reads as zeros; it is reported unless every row's window has passed it (then it was given back)
      auto page_of = [&](int t) -> int {
        const int key = (it.tile_begin + t) * TILE_N + b * box_rows;
        if (t >= it.n_tiles || b >= n_boxes || key > p_last) return -1;
        const int page = it.bt[key >> log2ps];
        if (page >= 0 && page < plan.num_pages) return page;
        if (plan.window <= 0 || key + box_rows > it.base - plan.window + 1) atomicExch(err, ERR_PAGE);
        return -1;
      };
      int page = page_of(0);
      for (int t = 0; t < it.n_tiles; ++t) {
        const int u = u0 + t, st = u % STAGES;
        const uint32_t ph = (uint32_t)(u / STAGES) & 1u;
        const int key0 = (it.tile_begin + t) * TILE_N;
        const int next_page = page_of(t + 1);  // in flight while this tile's copies are issued
        // whole boxes (pages) up to the last key this item may look at; a box that starts beyond it is skipped
        const int boxes = min(n_boxes, (p_last - key0) / box_rows + 1);
        uint64_t* empty = which ? &v_free[st] : &k_free[st];
        uint64_t* full = which ? &v_full[st] : &k_full[st];
        if (lane == 0) {
          if (!mbar_wait(empty, ph ^ 1u, vabort)) {
            if (!*vabort) atomicExch(err, 111);
            *vabort = 1;
          } else {
            mbar_expect_tx(full, (uint32_t)(boxes * NA * box_rows * 128));
          }
        }
        __syncwarp();
        if (*vabort) break;
        if (lane < boxes * NA)
          tma_load_4d(tiles + st * KV_BYTES + a * ATOM_BYTES + b * box_rows * 128, map, full, a * 64,
                      (key0 + b * box_rows) & (ps - 1), it.kvh, page);
        page = next_page;
        issued = u + 1;
      }
    }
    // after a failure: every copy that was issued lands before the CTA goes (a tile's barrier completes with it)
    if (*vabort && lane == 0) {
      for (int u = max(0, issued - STAGES); u < issued; ++u) {
        uint64_t* full = which ? &v_full[u % STAGES] : &k_full[u % STAGES];
        for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(full, (uint32_t)(u / STAGES) & 1u); ++w) {
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ issuer of S = Q K^T, up to two tiles ahead
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc(BLOCK_M, TILE_N, 0, 0);
      bool ok = true;
      int u0 = 0, n_done = 0;
      for (int pass = 0; ok && next_item(pass); u0 += it.n_tiles, ++n_done) {
        ok = mbar_wait(&q_full, (uint32_t)n_done & 1u, vabort);
        for (int t = 0; t < it.n_tiles && ok; ++t) {
          const int u = u0 + t, st = u % STAGES;
          // the keys have landed, and the softmax warps have taken tile u - 2 out of this S buffer
          if (!mbar_wait(&k_full[st], (uint32_t)(u / STAGES) & 1u, vabort) ||
              !mbar_wait(&s_free[u & 1], ((uint32_t)(u >> 1) & 1u) ^ 1u, vabort)) {
            ok = false;
            break;
          }
          fence_after();
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint64_t ad = desc_kmajor(q_smem + (ks >> 2) * ATOM_BYTES) + (uint64_t)((ks & 3) * 2);
            const uint64_t bd = desc_kmajor(k_smem + st * KV_BYTES + (ks >> 2) * ATOM_BYTES) + (uint64_t)((ks & 3) * 2);
            umma_bf16(tmem + S_COL0 + (uint32_t)((u & 1) * TILE_N), ad, bd, idesc_s, ks > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[u & 1]);
          umma_commit(&k_free[st]);
        }
      }
      if (!ok) {
        if (!*vabort) atomicExch(err, 112);
        *vabort = 1;
      }
    }
  } else {
    // ------------------------------------------------------------------ warp 3: loads Q, issues O += P V
    if (lane == 0) {
      constexpr uint32_t idesc_o = make_idesc(BLOCK_M, HD, 0, 1);  // B = V: N (head dim) contiguous
      bool ok = true;
      int u0 = 0, n_done = 0, q_issued = 0;
      for (int pass = 0; ok && next_item(pass); u0 += it.n_tiles, ++n_done) {
        // Q goes where the item before staged its output: wait until that has left
        if (n_done > 0 && !mbar_wait(&epi_done, (uint32_t)(n_done - 1) & 1u, vabort)) {
          ok = false;
          break;
        }
        mbar_expect_tx(&q_full, (uint32_t)(NA * plan.nodes_per_tile * plan.grp * 128));
        for (int a = 0; a < NA; ++a)
          tma_load_3d(q_smem + a * ATOM_BYTES, &map_q, &q_full, a * 64, it.kvh * plan.grp, it.q0 + it.node0);
        q_issued = n_done + 1;
        for (int t = 0; t < it.n_tiles && ok; ++t) {
          const int u = u0 + t, st = u % STAGES;
          if (!mbar_wait(&p_full[u & 1], (uint32_t)(u >> 1) & 1u, vabort) ||
              !mbar_wait(&v_full[st], (uint32_t)(u / STAGES) & 1u, vabort)) {
            ok = false;
            break;
          }
          fence_after();
          const uint32_t p_tmem = tmem + P_COL0 + (uint32_t)((u & 1) * (TILE_N / 2));
#pragma unroll
          for (int ks = 0; ks < TILE_N / 16; ++ks) {
            const uint64_t bd = desc_mnmajor(v_smem + st * KV_BYTES, ATOM_BYTES) + (uint64_t)(ks * (16 * 128 / 16));
            umma_bf16_ts(tmem + O_COL, p_tmem + (uint32_t)(ks * 8), bd, idesc_o, (t > 0 || ks > 0) ? 1u : 0u);
          }
          umma_commit(&p_free[u & 1]);
          umma_commit(&v_free[st]);
        }
      }
      if (!ok) {
        if (!*vabort) atomicExch(err, 112);
        *vabort = 1;
        for (uint32_t w = 0; q_issued > 0 && w < WAIT_LIMIT && !mbar_try_wait(&q_full, (uint32_t)(q_issued - 1) & 1u); ++w) {
        }
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    // ------------------------------------------------------------------ softmax and epilogue: two groups of four warps
    const int grp = (warp - 4) >> 2;     // group 0 takes the even tiles of the CTA's count, group 1 the odd ones
    const int qd = warp & 3;             // TMEM lane quarter of this warp
    const int r = qd * 32 + lane;        // query row of this thread
    const uint32_t lane_addr = (uint32_t)(qd * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + S_COL0 + (uint32_t)(grp * TILE_N);
    const uint32_t p_addr = tmem + lane_addr + P_COL0 + (uint32_t)(grp * (TILE_N / 2));
    int u0 = 0, n_done = 0;
    bool stop = false;
    for (int pass = 0; !stop && next_item(pass); u0 += it.n_tiles, ++n_done) {
      const int tok = r < it.rows ? it.q0 + it.node0 + r / plan.grp : -1;   // this row's token, or none
      int lo_row = 0;
      if (plan.window > 0 && tok >= 0) lo_row = it.base + min(max(plan.depth[tok], 0), it.n - 1) - plan.window + 1;
      const int u_last = u0 + it.n_tiles - 1;
      // my_off: the offset this thread's sum l_run is expressed at (what it last saw or set)
      float my_off = -INFINITY, l_run = 0.0f;
      bool ok = true;
      for (int t = (u0 & 1) == grp ? 0 : 1; t < it.n_tiles; t += 2) {
        const int u = u0 + t;                             // u % 2 == grp
        const uint32_t ph2 = (uint32_t)(u >> 1) & 1u;     // phase of this group's S/P barriers
        const int key0 = (it.tile_begin + t) * TILE_N;
        const bool masked = tile_masked(it, plan, key0);
        unsigned sees[4] = {0u, 0u, 0u, 0u};
        if (masked && tok >= 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c) sees[c] = sees32(it, plan, tok, lo_row, key0 + c * 32);
        }
        if (!mbar_wait(&s_full[grp], ph2, vabort)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        fence_after();
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + (uint32_t)(c * 32), v[c]);
        tmem_ld_wait();
        // the row is in registers: the S buffer is free for the tile after the next
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[grp]);
        if (masked) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!((sees[c] >> j) & 1u)) v[c][j] = 0xff800000u;  // -inf
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          mx0 = fmaxf(mx0, __uint_as_float(v[0][j]));
          mx1 = fmaxf(mx1, __uint_as_float(v[1][j]));
          mx2 = fmaxf(mx2, __uint_as_float(v[2][j]));
          mx3 = fmaxf(mx3, __uint_as_float(v[3][j]));
        }
        const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * scale_log2;  // the scale is positive
        // the row's offset after the tile before, which the other group's thread of this row has set
        if (t > 0) {
          if (!mbar_wait(&max_done[(u - 1) & 1], (uint32_t)((u - 1) >> 1) & 1u, vabort)) ok = false;
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
        }
        const float m_used = row_offset[r];   // -inf at an item's first tile
        // the exponent offset in use moves only when the maximum has grown enough (or at the first keys)
        const bool grow = mx > m_used + RESCALE_THRESHOLD || (m_used == -INFINITY && mx > -INFINITY);
        const float m_new = grow ? mx : m_used;
        row_offset[r] = m_new;
        mbar_arrive(&max_done[grp]);    // releases the write above to the thread that waits for this tile's offsets
        // this thread's sum at the new offset: first to what the other group left, then to what this tile sets
        if (my_off != m_new) l_run = my_off == -INFINITY ? 0.0f : l_run * ex2_approx(my_off - m_new);
        my_off = m_new;
        const float alpha = (grow && m_used != -INFINITY) ? ex2_approx(m_used - m_new) : 1.0f;
        if (t > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
          // O belongs to the tensor cores until the product of the tile before has completed; the product of this
          // tile waits for this thread's P, the products after it for this one: nothing else touches O meanwhile
          if (!mbar_wait(&p_free[(u - 1) & 1], (uint32_t)((u - 1) >> 1) & 1u, vabort)) ok = false;
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          fence_after();
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += 32) {
            uint32_t o[32];
            tmem_ld32(tmem + lane_addr + O_COL + (uint32_t)c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            tmem_st32(tmem + lane_addr + O_COL + (uint32_t)c0, o);
          }
        }
        // the product that read this P buffer last (tile u - 2) has completed
        if (u >= 2) {
          if (!mbar_wait(&p_free[grp], ph2 ^ 1u, vabort)) ok = false;
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          fence_after();
        }
        // P = exp2(S * scale - offset), two bf16 per column of this group's P buffer;
        // rows that have seen no key yet (offset -inf) are all masked here: exp2(-inf) = 0 with any finite offset
        const float offset = m_new == -INFINITY ? 0.0f : m_new;
        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float p0 = ex2_approx(fmaf(__uint_as_float(v[c][j]), scale_log2, -offset));
            const float p1 = ex2_approx(fmaf(__uint_as_float(v[c][j + 1]), scale_log2, -offset));
            sum0 += p0;
            sum1 += p1;
            __nv_bfloat162 b = __floats2bfloat162_rn(p0, p1);
            v[c >> 1][(c & 1) * 16 + (j >> 1)] = *reinterpret_cast<uint32_t*>(&b);
          }
          if (c == 1) tmem_st32(p_addr, v[0]);
        }
        tmem_st32(p_addr + 32u, v[1]);
        l_run += sum0 + sum1;
        // V of a masked tile: rows from the first key that was not loaded (shared memory never written, or an older tile) or that
        // lies at or beyond the request's length (whatever the page held before) are cleared, and so is every value that is
        // not finite: P = 0 must hide it
        if (masked) {
          const int loaded = min(n_boxes, (it.kv_len - 1 - key0) / box_rows + 1) * box_rows;
          const int first_bad = min(it.kv_len - key0, loaded);
          const int st = u % STAGES;
          if (!mbar_wait(&v_full[st], (uint32_t)(u / STAGES) & 1u, vabort)) ok = false;
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          unsigned char* vrow = v_smem + st * KV_BYTES + r * 128;
          if (r >= first_bad) {
            for (int a = 0; a < NA; ++a)
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(vrow + a * ATOM_BYTES + c * 16) = make_uint4(0, 0, 0, 0);
          } else {
            uint32_t any = 0u;
#pragma unroll
            for (int c = 0; c < 8 * NA; ++c) {
              const uint4 w = *reinterpret_cast<const uint4*>(vrow + (c >> 3) * ATOM_BYTES + (((c ^ r) & 7) << 4));
              any |= not_finite(w.x) | not_finite(w.y) | not_finite(w.z) | not_finite(w.w);
            }
            if (any) {
              for (int c = 0; c < 8 * NA; ++c) {
                uint4* at = reinterpret_cast<uint4*>(vrow + (c >> 3) * ATOM_BYTES + ((c & 7) << 4));
                uint4 w = *at;
                w.x = without_not_finite(w.x);
                w.y = without_not_finite(w.y);
                w.z = without_not_finite(w.z);
                w.w = without_not_finite(w.w);
                *at = w;
              }
              found_bad[n_done & 1] = 1;
            }
          }
          fence_async_smem();
        }
        tmem_st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[grp]);
      }
      // both groups bring their sums to the offset after the last tile and exchange them
      if (ok && (u_last & 1) != grp) {   // the other group had the last tile
        if (!mbar_wait(&max_done[u_last & 1], (uint32_t)(u_last >> 1) & 1u, vabort)) ok = false;
      }
      const float m_final = row_offset[r];
      {
        const float m_fin = m_final;
        if (my_off != m_fin) l_run = my_off == -INFINITY ? 0.0f : l_run * ex2_approx(my_off - m_fin);
        row_sum[grp][r] = l_run;
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");   // the eight softmax warps
      if (grp == 0) row_offset[r] = -INFINITY;          // for the next item; its first tile is read after the barrier below
      if (threadIdx.x == 128) found_bad[(n_done + 1) & 1] = 0;   // last read before the barrier that ended the item before
      if ((int)blockIdx.x + (int)gridDim.x * pass >= plan.n_items) pdl_trigger();   // the last item of this CTA
      // epilogue. One range: O / l as bf16 through the shared memory that held Q (every product that read it has completed),
      // each group half of the head's columns, so that the rows go out in whole 16-byte pieces side by side. Several: O as
      // fp32 into this item's scratch.
      constexpr int CPR = HD / 8;          // 16-byte pieces per row; piece c of row r lies at slot c ^ (r % CPR)
      ok = __all_sync(0xffffffffu, ok);
      if (ok && !mbar_wait(&p_free[u_last & 1], (uint32_t)(u_last >> 1) & 1u, vabort)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        fence_after();
        const float l = row_sum[0][r] + row_sum[1][r];
        const float inv = it.ranges > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        const bool bad = found_bad[n_done & 1] != 0;
#pragma unroll
        for (int c0 = grp * (HD / 2); c0 < (grp + 1) * (HD / 2); c0 += 32) {
          uint32_t o[32];
          tmem_ld32(tmem + lane_addr + O_COL + (uint32_t)c0, o);
          tmem_ld_wait();
          if (bad && tok >= 0) add_not_finite(o, it, plan, tok, lo_row, v_cache, HD, c0);
          if (it.ranges > 1) {
            float4* po = part_o + ((size_t)idx * (HD / 4) + c0 / 4) * BLOCK_M + r;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              po[(j / 4) * BLOCK_M] = make_float4(__uint_as_float(o[j]), __uint_as_float(o[j + 1]), __uint_as_float(o[j + 2]),
                                                  __uint_as_float(o[j + 3]));
            continue;
          }
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 w;
            __nv_bfloat162* hh = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              hh[e] = __floats2bfloat162_rn(__uint_as_float(o[j + 2 * e]) * inv, __uint_as_float(o[j + 2 * e + 1]) * inv);
            const int c = (c0 + j) >> 3;
            *reinterpret_cast<uint4*>(q_smem + r * (HD * 2) + ((c ^ (r & (CPR - 1))) << 4)) = w;
          }
        }
        if (it.ranges > 1 && grp == 0) part_ml[(size_t)idx * BLOCK_M + r] = make_float2(m_final, l);
        fence_before();
      } else if (lane == 0) {
        if (!*vabort) atomicExch(err, 113);
        *vabort = 1;
      }
      stop = softmax_bar_or(!ok || *vabort != 0);
      if (!stop) {
        const int ts = (int)threadIdx.x - 128;
        const int c = ts % CPR;
        if (it.ranges == 1) {
          for (int row = ts / CPR; row < it.rows; row += 256 / CPR) {
            const int node = row / plan.grp, g = row - node * plan.grp;
            *reinterpret_cast<uint4*>(out + ((size_t)(it.q0 + it.node0 + node) * plan.nh + it.kvh * plan.grp + g) * HD + c * 8) =
                *reinterpret_cast<const uint4*>(q_smem + row * (HD * 2) + ((c ^ (row & (CPR - 1))) << 4));
          }
        }
        // what this warp read of O (tensor memory) and of the staged rows is in its registers or on its way out
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&epi_done);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Joins the ranges of a row in order. A thread has one row and eight dims; rows are the fast index, as in the scratch.
template <int HD>
__global__ void __launch_bounds__(BLOCK_M) attn_tree_tc_join_kernel(bf16* __restrict__ out, const float4* __restrict__ part_o,
                                                                    const float2* __restrict__ part_ml,
                                                                    const __grid_constant__ Plan plan) {
  pdl_wait();
  const int r = threadIdx.x, d8 = blockIdx.y;
  const int m = blockIdx.x % plan.m_tiles, sh = blockIdx.x / plan.m_tiles;
  const int kvh = sh % plan.nkv, s = sh / plan.nkv;
  const int q0 = plan.cu_q[s], n = plan.cu_q[s + 1] - q0, node0 = m * plan.nodes_per_tile;
  if (node0 >= n || r >= min(plan.nodes_per_tile, n - node0) * plan.grp) return;
  const int kv_all = plan.seq_lens[s], kv_len = min(kv_all, plan.kv_cap);
  if (kv_len <= 0) return;
  const int ranges = cut_of(plan, kv_len, kv_all - n).ranges;
  if (ranges == 1) return;
  const size_t slot0 = (size_t)sh * plan.splits * plan.m_tiles + m;
  float M = -INFINITY, L = 0.0f, acc[8] = {};
  constexpr int U = 4;     // ranges in flight
  for (int k0 = 0; k0 < ranges; k0 += U) {
    float2 ml[U];
    float4 a[U], b[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const size_t slot = slot0 + (size_t)min(k0 + k, ranges - 1) * plan.m_tiles;
      const float4* po = part_o + (slot * (HD / 4) + d8 * 2) * BLOCK_M + r;
      ml[k] = part_ml[slot * BLOCK_M + r];
      a[k] = po[0];
      b[k] = po[BLOCK_M];
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      // a range of which the row sees nothing has neither weight nor maximum (but NaN scores have a sum without a maximum)
      if (k0 + k >= ranges || (ml[k].x == -INFINITY && ml[k].y == 0.0f)) continue;
      const float mk = ml[k].x;
      const float m_new = fmaxf(M, mk);
      const float keep = M == m_new ? 1.0f : M == -INFINITY ? 0.0f : ex2_approx(M - m_new);
      const float f = mk == m_new ? 1.0f : ex2_approx(mk - m_new);
      M = m_new;
      L = L * keep + ml[k].y * f;
      const float v[8] = {a[k].x, a[k].y, a[k].z, a[k].w, b[k].x, b[k].y, b[k].z, b[k].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = keep == 1.0f ? fmaf(v[e], f, acc[e]) : fmaf(v[e], f, acc[e] * keep);
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  uint4 w;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  const int node = r / plan.grp, g = r - node * plan.grp;
  *reinterpret_cast<uint4*>(out + ((size_t)(q0 + node0 + node) * plan.nh + kvh * plan.grp + g) * HD + d8 * 8) = w;
}

// Key tiles that a request of the batch looks at, at most.
int most_tiles(int max_q_len, int max_kv_len, int window) {
  long long t = ((long long)max_kv_len + TILE_N - 1) / TILE_N;
  if (window > 0) {
    const long long w = ((long long)window + max_q_len + TILE_N - 1) / TILE_N + 1;
    if (w < t) t = w;
  }
  return (int)(t < 1 ? 1 : t);
}

template <int HD>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, bf16* out, float* part_o, float* part_ml,
           const bf16* v_cache, const Plan& plan, float scale_log2, int* err, cudaStream_t stream) {
  // at least 120 KB so that one CTA is resident per SM: each takes all 512 tensor-memory columns
  constexpr size_t need = (size_t)(HD / 64) * ATOM_BYTES * (1 + 2 * STAGES) + 1024;
  constexpr size_t smem = need > 120 * 1024 ? need : 120 * 1024;
  int sms = 0;
  int rc = osb_allow_smem<attn_tree_tc_kernel<HD>>(smem);
  if (rc == 0) rc = osb_num_sms(&sms);
  if (rc) return rc;
  rc = osb_launch(attn_tree_tc_kernel<HD>, dim3((unsigned)(plan.n_items < sms ? plan.n_items : sms)), dim3(NUM_THREADS), smem, stream, mq, mk, mv, out,
                      (float4*)part_o, (float2*)part_ml, v_cache, plan, scale_log2, err);
  if (rc == 0 && plan.splits > 1)
    rc = osb_launch(attn_tree_tc_join_kernel<HD>, dim3((unsigned)(plan.S * plan.nkv * plan.m_tiles), HD / 8), dim3(BLOCK_M), 0, stream,
                    out, (const float4*)part_o, (const float2*)part_ml, plan);
  return rc ? rc : osb_last_error();
}
}  // namespace

// Into how many ranges (at most) a request's keys are cut, 0 if the kernel does not take the shapes. The cost of a cut in units of
// one key tile: the waves of items over the SMs, each a range plus some 2 tiles for starting and ending it, and some 2 for the second
// kernel; the smallest cut of the least cost.
OSB_API int osb_attn_tree_tc_splits(int S, int nh, int nkv, int hd, int page_size, int q_row_stride, float scale, int window,
                                    int max_q_len, int max_kv_len) {
  if ((hd != 64 && hd != 128) || nkv <= 0 || nh <= 0 || nh % nkv != 0 || nh / nkv > BLOCK_M || !(scale > 0.0f)) return 0;
  if (page_size < 8 || (page_size & (page_size - 1)) || (q_row_stride & 7) || S <= 0 || max_q_len <= 0 || max_kv_len <= 0) return 0;
  if (max_kv_len > MAX_KEYS || window < 0) return 0;
  const int nodes = BLOCK_M / (nh / nkv);
  const long long units = (long long)S * nkv * ((max_q_len + nodes - 1) / nodes);
  if (units * MAX_TC_SPLITS > 2147483647LL) return 0;
  const int tiles = most_tiles(max_q_len, max_kv_len, window);
  int sms = 1;
  osb_num_sms(&sms);
  int best = 1;
  long long best_cost = 0;
  for (int s = 1; s <= MAX_TC_SPLITS && s <= tiles; ++s) {
    const long long waves = (units * s + sms - 1) / sms;
    const long long cost = waves * ((tiles + s - 1) / s + 2) + (s > 1 ? 2 : 0);
    if (s == 1 || cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

// As osb_attn_tree for bf16 operands. splits: what osb_attn_tree_tc_splits gave for the same arguments (0 there: refused here with
// OSB_ERR_UNSUPPORTED). With splits > 1: items = S x nkv x row tiles x splits, part_o items x 128 x hd and part_ml items x 256
// floats, row tiles = ceil(max_q_len / (128 / (nh / nkv))).
OSB_API int osb_attn_tree_tc(void* out, const void* q, int q_row_stride, int T, const void* k_cache, const void* v_cache,
                             const int* block_table, int bt_stride, const int* cu_q, const int* seq_lens, const unsigned* mask,
                             int mask_words, const int* depth, int S, int nh, int nkv, int hd, int page_size, int num_pages,
                             float scale, int window, int max_q_len, int max_kv_len, int splits, float* part_o, float* part_ml,
                             int* err, cudaStream_t stream) {
  if (S <= 0 || T <= 0 || max_q_len <= 0) return OSB_OK;
  if (splits <= 0 || splits > MAX_TC_SPLITS || num_pages <= 0 ||
      osb_attn_tree_tc_splits(S, nh, nkv, hd, page_size, q_row_stride, scale, window, max_q_len, max_kv_len) == 0)
    return OSB_ERR_UNSUPPORTED;
  if (((uintptr_t)q & 15) || ((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15) || ((uintptr_t)out & 15))
    return OSB_ERR_UNSUPPORTED;
  if ((window > 0 && depth == nullptr) || (splits > 1 && (part_o == nullptr || part_ml == nullptr))) return OSB_ERR_BAD_SHAPE;
  Plan p = {};
  p.block_table = block_table;
  p.cu_q = cu_q;
  p.seq_lens = seq_lens;
  p.mask = mask;
  p.depth = depth;
  p.err = err;
  p.bt_stride = bt_stride;
  p.mask_words = mask_words;
  p.S = S;
  p.nh = nh;
  p.nkv = nkv;
  p.grp = nh / nkv;
  while ((1 << p.log2ps) < page_size) ++p.log2ps;
  p.num_pages = num_pages;
  p.window = window;
  p.max_q_len = max_q_len;
  const long long table = (long long)bt_stride * page_size;     // keys behind the block table cannot be read
  p.kv_cap = table < max_kv_len ? (int)table : max_kv_len;
  p.nodes_per_tile = BLOCK_M / p.grp;
  p.m_tiles = (max_q_len + p.nodes_per_tile - 1) / p.nodes_per_tile;
  p.splits = splits;
  p.chunk_tiles = (most_tiles(max_q_len, max_kv_len, window) + splits - 1) / splits;
  p.n_items = S * nkv * p.m_tiles * splits;
  CUtensorMap mq, mk, mv;
  {
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)nh, (cuuint64_t)T};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)q_row_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)p.grp, (cuuint32_t)p.nodes_per_tile};
    const int rc = make_map_bf16(&mq, q, 3, dims, strides, box);
    if (rc) return rc;
  }
  {
    const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)page_size, (cuuint64_t)nkv, (cuuint64_t)num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)hd * 2, (cuuint64_t)page_size * hd * 2,
                                   (cuuint64_t)nkv * page_size * hd * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(page_size < 128 ? page_size : 128), 1, 1};
    int rc = make_map_bf16(&mk, k_cache, 4, dims, strides, box);
    if (rc) return rc;
    rc = make_map_bf16(&mv, v_cache, 4, dims, strides, box);
    if (rc) return rc;
  }
  const float scale_log2 = scale * LOG2E;
  if (hd == 64)
    return launch<64>(mq, mk, mv, (bf16*)out, part_o, part_ml, (const bf16*)v_cache, p, scale_log2, err, stream);
  return launch<128>(mq, mk, mv, (bf16*)out, part_o, part_ml, (const bf16*)v_cache, p, scale_log2, err, stream);
}
