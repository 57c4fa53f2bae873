// Attention of a tree of drafted tokens over the paged cache on the fifth-generation tensor cores (bf16, head sizes 64 and 128).
//
// What a node sees, and its formula: attn_tree.cu. The query rows of a request and kv head are its nodes times the group's heads
// (row = node x group + head), in tiles of up to 128 rows that are whole nodes, so that one pass over the keys serves the whole
// group. Q comes with one 3-D TMA box (64 dims, the group's heads, nodes) per half of the head; keys and values come in tiles of
// 64 keys, gathered page by page with 4-D boxes (128-byte swizzle) into one ring of tiles. S = Q K^T and O += P V are tcgen05.mma,
// each kind issued by one thread; P goes to tensor memory as bf16, over the S that it was made from, and is the A operand of the
// second product. Eight softmax warps, two threads per row with half of a tile's keys each, have two S/P buffers, so that the next
// tile's scores are there when a tile's weights are done. A row's exponent offset moves only when its maximum has grown by more
// than 2^8, and only then do its two threads tell each other their maxima.
// What bounds it: a tile of keys and values is 32 KB, 0.74 us at a 148th of the memory's rate. Its 64 exponentials a row take 512
// cycles on a unit that makes 16 a cycle, its two products 512 on the tensor cores, but the way from tensor memory and back, the
// instructions around the exponentials and the waits between the stages take longer (one CTA with four softmax warps: 2,090 cycles a
// tile). So two CTAs share an SM, each with half of its tensor memory and shared memory: while one begins or ends a unit or waits for
// a product, the other one works. Each then takes some 1,800 cycles for a tile, the SM half of that, with half of its issue slots taken.
// Measured (us, with the second kernel): one request of 16 nodes and 2,048 keys, 12 heads on 2, 11.0 (latency: 3 us until the first keys
// arrive, one or two tiles, 2.5 for the second kernel); 64 requests of 8 nodes and up to 2,100 keys, 28 heads on 4 (206 MB), 50, 4.1
// TB/s; one of 64 nodes and 32,768 keys, 64 heads on 8 (69 GFLOP), 95 in a row of calls, under the power cap: 720 TFLOP/s (by itself 79).
//
// The work is cut evenly: all key tiles of all units (request, kv head, row tile) stand in one line, and every CTA takes an equal
// piece of it: the end of one unit, some whole ones, the beginning of another. (Where units are few and short, whole ones; see
// WHOLE_EXTRA.) Every CTA finds its piece itself from the
// requests' lengths. A unit that was cut leaves its unnormalised fp32 output, maximum and sum in scratch, two places per
// CTA, laid out [4 dims][row] so that neighbouring threads (rows) write neighbouring 16 bytes straight from tensor memory; a second
// kernel joins them in order. CTAs of one launch never wait for one another. A single request with several row tiles is the
// exception in the order: its row tiles go to neighbouring CTAs that take the same keys at the same time, so that the keys of a long
// context, more than the L2 holds, are fetched from memory once.
//
// Masks. A tile of keys that are all committed and inside every row's window needs none. Otherwise a row's 128 bits come from its
// mask words (places before the tree count as ones). P is 0 where a row does not see a key, but 0 times a NaN or an infinity in V
// would still reach the row through the tensor core: in such tiles the values that are not finite are replaced by zeros in shared
// memory, and if there were any, the rows that do see them get them added at the end, from the cache.
//
// All mbarrier waits are bounded; on a time-out the CTA records a code in *err, frees its tensor memory and returns. Each warp that issues
// copies or products waits (bounded too) until they are done before it leaves, whoever gave up, and before the tensor memory goes.
#include "attn_tree.cuh"
#include "tc_utils.cuh"

namespace {
using namespace tc;
using namespace attn_tree;

constexpr int BLOCK_M = 128, TILE_N = 64;
constexpr int NUM_THREADS = 384, CTAS_PER_SM = 2;
constexpr int Q_ATOM = BLOCK_M * 128, KV_ATOM = TILE_N * 128;   // rows of 128 bytes
// Key tiles that a CTA takes beyond an even piece to have a unit whole, where there are no more units than CTAs: cutting costs the second
// kernel and the way through scratch. Whole or cut, us: 3 requests of 87 keys and 4 kv heads (2 tiles) 8.7, 12.7; 8 of 320 and 2 heads
// (5 tiles) 11.7, 13.9; with 10 instead of 6, 22 of 740 and 2 heads (12 tiles) 19.4, 14.0.
constexpr int WHOLE_EXTRA = 6;
constexpr int OTHER_REGS = 64, SOFTMAX_REGS = 88;    // of a thread
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_THRESHOLD = 8.0f;            // in log2 units

// A unit (request, kv head, row tile): the CTA in whose piece it begins, and into how many pieces it was cut.
struct Cut {
  int cta, pieces;
};

// The step, the same for every CTA.
struct Plan {
  const int* block_table;
  const int* cu_q;
  const int* seq_lens;
  const unsigned* mask;
  const int* depth;
  int* err;
  Cut* cuts;           // scratch, by unit: (request x kv heads + head) x row tiles + tile
  int T, bt_stride, mask_words, S, nh, nkv, grp, log2ps, num_pages, window, max_q_len, kv_cap;
  int nodes_per_tile, m_tiles, ctas;
  int whole_tiles;                  // key tiles of a unit at most, if there are no more units than CTAs (if there are: a huge number)
  int abreast;                      // row tiles that neighbouring CTAs take at the same time (1: row tiles are units like others)
  unsigned inv_nodes, inv_grp;      // 2^32 / nodes_per_tile and / grp, rounded up
};
// x / d for x below 2^25 and d up to 128, inv = ceil(2^32 / d) (d = 1: 0)
__device__ __forceinline__ int div_by(int x, unsigned inv) { return inv == 0 ? x : (int)__umulhi((unsigned)x, inv); }
// x / d where the quotient is below 2^20: a division in fp32, put right by one at most
__device__ __forceinline__ int small_quotient(int x, int d) {
  int q = (int)__fdividef((float)x, (float)d);
  const int r = x - q * d;
  if (r < 0) --q;
  else if (r >= d) ++q;
  return q;
}

// What a request brings: its key tiles and its row tiles.
struct Req {
  int q0, n, kv_len, base, first_tile, tiles, m_tiles;
};
__device__ __forceinline__ Req req_of(const Plan& p, int s) {
  Req r;
  r.q0 = p.cu_q[s];
  const int q1 = p.cu_q[s + 1], kv_all = p.seq_lens[s];
  r.n = r.q0 >= 0 && q1 <= p.T ? q1 - r.q0 : -1;       // (tokens that are not there: reported, and nothing is done)
  r.kv_len = min(kv_all, p.kv_cap);
  r.base = kv_all - r.n;
  const int lo = p.window > 0 && r.base - p.window + 1 > 0 ? min(r.base - p.window + 1, r.kv_len - 1) : 0;
  r.first_tile = lo / TILE_N;
  r.tiles = r.n > 0 && r.kv_len > 0 ? (r.kv_len - 1) / TILE_N - r.first_tile + 1 : 0;
  r.m_tiles = min(div_by(max(min(r.n, p.max_q_len), 0) + p.nodes_per_tile - 1, p.inv_nodes), p.m_tiles);
  return r;
}
__device__ __forceinline__ int units_of(const Plan& p, const Req& r) { return p.abreast > 1 ? 1 : r.m_tiles; }   // per kv head
__device__ __forceinline__ int tiles_of(const Plan& p, const Req& r) { return r.tiles > 0 ? p.nkv * units_of(p, r) * r.tiles : 0; }

// One stretch of a CTA's piece: key tiles of one unit.
struct Seg {
  Req r;
  int kvh, node0, rows;         // the row tile: its first node, its number of rows
  int tile_begin, n_tiles;
  bool whole, began;            // whole: all the unit's tiles; began: the unit began in an earlier piece
  int unit, pieces;             // the unit's number; into how many pieces it is cut, if it begins here
  const int* bt;
};

// Walks over the stretches of the piece [g, hi) of the line; `s`, `p_s`: a request and where its units begin, at or before g.
struct Walk {
  int g, hi, s, p_s;
  int m, piece;                 // this CTA's row tile where row tiles go abreast; the tiles of a piece
  Req r;                        // of request s
  __device__ __forceinline__ bool next(const Plan& p, Seg& seg) {
    if (g >= hi) return false;
    for (;;) {
      const int mine = tiles_of(p, r);
      if (g < p_s + mine) break;
      p_s += mine;
      if (++s >= p.S) return false;
      r = req_of(p, s);
    }
    const int unit = small_quotient(g - p_s, r.tiles), t0 = g - p_s - unit * r.tiles, units = units_of(p, r);
    seg.r = r;
    seg.kvh = units == 1 ? unit : small_quotient(unit, units);
    seg.node0 = (p.abreast > 1 ? m : unit - seg.kvh * units) * p.nodes_per_tile;
    seg.rows = min(p.nodes_per_tile, r.n - seg.node0) * p.grp;
    seg.n_tiles = min(r.tiles - t0, hi - g);
    seg.tile_begin = r.first_tile + t0;
    seg.whole = seg.n_tiles == r.tiles;
    seg.began = t0 > 0;
    seg.unit = (s * p.nkv + seg.kvh) * p.m_tiles + (p.abreast > 1 ? m : unit - seg.kvh * units);
    seg.pieces = 1 + (seg.whole ? 0 : (r.tiles - seg.n_tiles + piece - 1) / piece);
    seg.bt = p.block_table + (size_t)s * p.bt_stride;
    g += seg.n_tiles;
    return true;
  }
};

// Whether some row does not see some key of the tile from key0 on (depths are below the number of nodes).
__device__ __forceinline__ bool tile_masked(const Req& r, const Plan& p, int key0) {
  return key0 + TILE_N > min(r.base, r.kv_len) || (p.window > 0 && key0 < r.base + r.n - p.window);
}

// Which of the keys key0 .. key0 + 31 row `t` of the step sees; lo: the first place inside its window.
__device__ __forceinline__ unsigned sees32(const Req& r, const Plan& p, int t, int lo, int key0) {
  const int off = key0 - r.base;                        // of the tree's node numbers
  const unsigned* row = p.mask + (size_t)t * p.mask_words;
  auto word = [&](int i) -> unsigned { return i < 0 ? 0xffffffffu : i < p.mask_words ? row[i] : 0u; };
  unsigned v = __funnelshift_r(word(off >> 5), word((off >> 5) + 1), off & 31);
  const int left = r.kv_len - key0;
  v = left >= 32 ? v : left > 0 ? v & ((1u << left) - 1u) : 0u;
  if (p.window > 0) {
    const int hidden = min(lo, r.base) - key0;          // committed keys in front of the window
    v = hidden >= 32 ? 0u : hidden > 0 ? v & (0xffffffffu << hidden) : v;
    if (lo > r.base) {                                  // a window shorter than the path: ancestors by their depth
      for (unsigned w = v; w != 0; w &= w - 1) {
        const int j = off + __ffs(w) - 1;
        if (j >= 0 && r.base + p.depth[r.q0 + j] < lo) v &= ~(w & (0u - w));
      }
    }
  }
  return v;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  return (uint64_t)__float_as_uint(lo) | ((uint64_t)__float_as_uint(hi) << 32);
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  lo = __uint_as_float((uint32_t)v);
  hi = __uint_as_float((uint32_t)(v >> 32));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Bits 15 and 31 say which of two bf16 are not finite.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ uint32_t without_not_finite(uint32_t w) {
  const uint32_t b = not_finite(w);
  return w & ~((b & 0x8000u ? 0xffffu : 0u) | (b & 0x80000000u ? 0xffff0000u : 0u));
}

// What was taken out of the V tile from key0 on for 8 dims of a row: the values that are not finite among the keys that the row
// sees, from the cache. Only reached when a masked tile held such values.
__device__ __forceinline__ void add_taken_out(float (&x)[8], unsigned sees, int key0, const int* bt, const Plan& p, int kvh,
                                              const bf16* v_cache, int hd, int d) {
  for (; sees != 0; sees &= sees - 1) {
    const int key = key0 + __ffs(sees) - 1, page = bt[key >> p.log2ps];
    if (page < 0 || page >= p.num_pages) continue;
    const int off = key & ((1 << p.log2ps) - 1);
    const bf16* v = v_cache + ((((size_t)page * p.nkv + kvh) << p.log2ps) + off) * hd + d;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const float f = __bfloat162float(v[e]);
      if (!(fabsf(f) < INFINITY)) x[e] += f;
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
// The same for the two warps that share 32 rows.
__device__ __forceinline__ bool pair_bar_or(int quarter, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, %2, 64, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(3 + quarter)
      : "memory");
  return r != 0;
}

// Barrier of the two warps that fill the ring.
__device__ __forceinline__ void producers_bar() { asm volatile("bar.sync 7, 64;" ::: "memory"); }

template <int HD>
struct Layout {
  static constexpr int NA = HD / 64;                  // 64-element atoms along the head dimension
  static constexpr int Q_BYTES = NA * Q_ATOM;         // [atom][128 rows][128 B]
  static constexpr int KV_BYTES = NA * KV_ATOM;       // a K or V tile: [atom][64 rows][128 B]
  static constexpr int STAGES = HD == 128 ? 4 : 8;    // key and value tiles in flight: 64 KB in each of the SM's two CTAs
  static constexpr size_t SMEM = (size_t)Q_BYTES + STAGES * KV_BYTES + 1024;
};

// Barriers (u: the CTA's key tiles, counted on across stretches; S / P buffer u % 2):
//  full / empty: a place of the ring has its tile / the products that read it have completed. Tiles pass through the ring in the
//    order K0, K1, V0, K2, V1, .. of a stretch, numbered on across stretches: tile i is in place i % STAGES.
//  s_full: Q K^T of key tile u is in S. p_full: its P is there (and V may be read). pv_done: P V complete, so S / P may be overwritten,
//    and, of a stretch's last tile, O read. q_full / staged_out: a stretch's Q has landed / a staged output has left Q's place.
template <int HD>
__global__ void __launch_bounds__(NUM_THREADS, CTAS_PER_SM) attn_tree_tc_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
    const __grid_constant__ CUtensorMap map_v, bf16* __restrict__ out, float4* __restrict__ part_o,
    float2* __restrict__ part_ml, const bf16* __restrict__ v_cache, const __grid_constant__ Plan plan, float scale_log2) {
  constexpr int NA = Layout<HD>::NA, Q_BYTES = Layout<HD>::Q_BYTES, KV_BYTES = Layout<HD>::KV_BYTES, STAGES = Layout<HD>::STAGES;
  constexpr uint32_t TMEM_COLS = 256, O_COL = 2 * TILE_N;    // S and over it P of buffer b in columns 64 b on, O in 128 on
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char* q_smem = base;
  unsigned char* ring = base + Q_BYTES;               // STAGES tiles of keys or values
  __shared__ uint64_t q_full, staged_out, full[STAGES], empty[STAGES], s_full[2], p_full[2], pv_done[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int ring_end[2][STAGES];     // the tile that each producer put into a place of the ring last
  __shared__ int found_bad[3];            // by the number of the CTA's stretch modulo 3: values that are not finite were taken out of a V tile
  __shared__ int scan[NUM_THREADS / 32];
  __shared__ int start_s, start_p;        // the request in which this CTA's piece begins, where its units begin
  __shared__ Req start_r;
  __shared__ float row_max[2][2][BLOCK_M];   // by the parity of the key tile, half of the keys, row
  __shared__ float row_sum[2][BLOCK_M];      // by half, row

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int log2ps = plan.log2ps, ps = 1 << log2ps;
  const int box_rows = ps < TILE_N ? ps : TILE_N;  // keys per TMA box: a page, or a tile's worth of a larger page
  const int n_boxes = TILE_N / box_rows;
  int* err = plan.err;

  if (lane == 0 && warp < 3) prefetch_tensormap(warp == 0 ? &map_k : warp == 1 ? &map_q : &map_v);
  if (tid == 0) {
    abort_flag = 0;
    found_bad[0] = found_bad[1] = found_bad[2] = 0;
    start_s = 0;
    mbar_init(&q_full, 1);
    mbar_init(&staged_out, 8);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(&tmem_slot, TMEM_COLS);
  // until here nothing was read that the kernel before this one in the stream may still be writing (lengths, q, the pages)
  pdl_wait();

  // ---- this CTA's piece of the line of tiles, or its unit
  const int own = (int)blockIdx.x;
  Req own_r = {};
  if (plan.whole_tiles < MAX_KEYS) own_r = req_of(plan, min(own / (plan.nkv * plan.m_tiles), plan.S - 1));
  Req mine = {};                                // of request `tid`
  int my_tiles = 0;
  long long all = 0;
  for (int s = tid; s < plan.S; s += NUM_THREADS) {
    const Req r = req_of(plan, s);
    const int t = tiles_of(plan, r);
    if (s == tid) {
      mine = r;
      my_tiles = t;
    }
    all += t;
    if (blockIdx.x == 0 && r.n != 0 && (r.n < 0 || r.kv_len < r.base + r.n || r.n > plan.max_q_len || r.base < 0)) atomicExch(err, ERR_BOUNDS);
  }
  auto block_scan = [&](int v, int& total) -> int {      // exclusive
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NUM_THREADS / 32; ++w) {
      before += w < warp ? scan[w] : 0;
      total += scan[w];
    }
    return before + inc - v;
  };
  int total;
  const int first = block_scan((int)all, total);
  // (row tiles abreast: a group of CTAs has one piece)
  const int groups = plan.abreast > 1 ? (int)gridDim.x / plan.abreast : (int)gridDim.x;
  const int group = plan.abreast > 1 ? (int)blockIdx.x / plan.abreast : (int)blockIdx.x;
  const int piece = max(1, (total + groups - 1) / groups);
  const bool whole = plan.whole_tiles <= piece + WHOLE_EXTRA;
  const int g0 = (int)min((long long)total, (long long)group * piece), g1 = group < groups ? min(total, g0 + piece) : g0;
  if (plan.S <= NUM_THREADS) {
    if (my_tiles > 0 && g0 >= first && g0 < first + my_tiles) {
      start_s = tid;
      start_p = first;
      start_r = mine;
    }
  } else {
    int run = 0;
    for (int s0 = 0; s0 < plan.S; s0 += NUM_THREADS) {
      const int s = s0 + tid;
      const int t = s < plan.S ? tiles_of(plan, req_of(plan, s)) : 0;
      int chunk;
      __syncthreads();                          // everyone has read the scan's words
      const int at = run + block_scan(t, chunk);
      if (t > 0 && g0 >= at && g0 < at + t) {
        start_s = s;
        start_p = at;
        start_r = req_of(plan, s);
      }
      run += chunk;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* vabort = &abort_flag;
  Walk walk;
  walk.g = g0;
  walk.hi = g1;
  walk.s = start_s;
  walk.p_s = start_p;
  walk.r = start_r;
  walk.piece = piece;
  walk.m = plan.abreast > 1 ? (int)blockIdx.x - group * plan.abreast : 0;
  if (whole) {
    // this CTA's unit, or none
    walk.s = own / (plan.nkv * plan.m_tiles);
    walk.r = own_r;
    const int unit = own - walk.s * plan.nkv * plan.m_tiles, kvh = unit / plan.m_tiles, m = unit - kvh * plan.m_tiles;
    walk.p_s = 0;
    walk.g = (kvh * own_r.m_tiles + m) * own_r.tiles;
    walk.hi = own < plan.S * plan.nkv * plan.m_tiles && m < own_r.m_tiles ? walk.g + own_r.tiles : walk.g;
  }
  if (plan.abreast > 1 && walk.m >= start_r.m_tiles) walk.hi = walk.g;     // the request has fewer row tiles than it might
  Seg seg;
  // The softmax warps take registers over from the others: 128 x 64 + 256 x 88 = the 384 x 80 of the launch. (Without, and with 48 and
  // 96, something is kept in local memory, whose first use alone costs a microsecond: one request 13.8 us instead of 12.7.)
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------ TMA producers: warp 0 keys, warp 2 values
    // Lane b looks up the page of box b; one thread issues all copies of a tile one after the other (a copy per lane would be
    // a loop over the lanes, some 190 cycles each).
    const bool keys = warp == 0;
    const CUtensorMap* map = keys ? &map_k : &map_v;
    int i0 = 0;             // tiles that were put into the ring before this stretch, by both
    LastPut<STAGES> last_put;               // of this warp's tiles; lane k has the ring's place k
    for (; !*vabort && walk.next(plan, seg); i0 += 2 * seg.n_tiles) {
      const int p_last = seg.r.kv_len - 1;
      auto page_of = [&](int t) -> int {      // of this lane's box of tile t
        const int key = (seg.tile_begin + t) * TILE_N + lane * box_rows;
        return t >= seg.n_tiles || lane >= n_boxes || key > p_last ? -1 : seg.bt[key >> log2ps];
      };
      int page = page_of(0), next_page = page_of(1);
      for (int t = 0; t < seg.n_tiles && !*vabort; ++t) {
        const int after_next = page_of(t + 2);  // in flight while these tiles' copies are issued (nothing looks at it yet)
        const int i = i0 + (keys ? (t == 0 ? 0 : 2 * t - 1) : (t + 1 < seg.n_tiles ? 2 * t + 2 : 2 * t + 1)), st = i % STAGES;
        const int key0 = (seg.tile_begin + t) * TILE_N;
        // whole boxes (pages) up to the request's last key; a box that starts beyond it is skipped
        const int boxes = min(n_boxes, (p_last - key0) / box_rows + 1);
        if (lane == 0) {
          if (!mbar_wait(&empty[st], ((uint32_t)(i / STAGES) & 1u) ^ 1u, vabort)) {
            if (!*vabort) atomicExch(err, 111);
            *vabort = 1;
          } else {
            mbar_expect_tx(&full[st], (uint32_t)(boxes * NA * box_rows * 128));
          }
        }
        // a page outside the pool reads as zeros; it is reported unless every row's window has passed it (then it was given back)
        if ((unsigned)page >= (unsigned)plan.num_pages) {
          page = -1;
          const int key = key0 + lane * box_rows;
          if (lane < n_boxes && key <= p_last && (plan.window <= 0 || key + box_rows > seg.r.base - plan.window + 1))
            atomicExch(err, ERR_PAGE);
        }
        __syncwarp();
        if (*vabort) break;
        unsigned char* to = ring + st * KV_BYTES;
        const int row0 = key0 & (ps - 1);       // of the first box in its page (the others begin a page)
#pragma unroll 2
        for (int b = 0; b < boxes; ++b) {
          const int pg = __shfl_sync(0xffffffffu, page, b);
          if (lane == 0) {
#pragma unroll
            for (int a = 0; a < NA; ++a)
              tma_load_4d(to + a * KV_ATOM + b * box_rows * 128, map, &full[st], a * 64, (row0 + b * box_rows) & (ps - 1), seg.kvh, pg);
          }
        }
        last_put.put(lane, i);
        page = next_page;
        next_page = after_next;
      }
    }
    // when neither puts anything more, they wait until what was put into each place last has landed
    if (lane < STAGES) ring_end[keys ? 0 : 1][lane] = last_put.tile;
    __syncwarp();
    producers_bar();
    const int i = lane < STAGES ? max(ring_end[0][lane], ring_end[1][lane]) : -1;
    for (uint32_t w = 0; i >= 0 && w < WAIT_LIMIT && !mbar_try_wait(&full[lane], (uint32_t)(i / STAGES) & 1u); ++w) {
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ loads Q, issues S = Q K^T
    // (the whole warp goes through the loops, one thread issues: the descriptors then stay in uniform registers)
    constexpr uint32_t idesc_s = make_idesc(BLOCK_M, TILE_N, 0, 0);
    const uint64_t q_desc = desc_kmajor(q_smem), k_desc = desc_kmajor(ring);
    bool ok = true, staged = false;      // staged: the stretch before stages its output where Q lies
    int i0 = 0, n_done = 0, u = 0, q_issued = 0, n_staged = 0;
    for (; ok && walk.next(plan, seg); i0 += 2 * seg.n_tiles, ++n_done) {
      // Q goes where the stretch before had its own: until its last scores are complete, or, if it stages its output there, until
      // that has left. (staged_out has a phase for each stretch of that kind, and this warp sees every one of them.)
      if (staged) ok = mbar_wait(&staged_out, (uint32_t)(n_staged - 1) & 1u, vabort);
      else if (n_done > 0) ok = mbar_wait(&s_full[(u - 1) & 1], (uint32_t)((u - 1) >> 1) & 1u, vabort);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (elect_one()) {
        mbar_expect_tx(&q_full, (uint32_t)(NA * plan.nodes_per_tile * plan.grp * 128));
#pragma unroll
        for (int a = 0; a < NA; ++a)
          tma_load_3d(q_smem + a * Q_ATOM, &map_q, &q_full, a * 64, seg.kvh * plan.grp, seg.r.q0 + seg.node0);
      }
      __syncwarp();
      q_issued = n_done + 1;
      staged = seg.whole;
      n_staged += staged ? 1 : 0;
      ok = mbar_wait(&q_full, (uint32_t)n_done & 1u, vabort);
      for (int t = 0; t < seg.n_tiles; ++t, ++u) {
        const int i = i0 + (t == 0 ? 0 : 2 * t - 1), st = i % STAGES, b = u & 1;
        // the keys have landed, and P V of the tile before the last has completed: its S / P may be overwritten
        ok = ok && mbar_wait(&full[st], (uint32_t)(i / STAGES) & 1u, vabort) &&
             (u < 2 || mbar_wait(&pv_done[b], (uint32_t)((u >> 1) - 1) & 1u, vabort));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        const uint64_t bd = k_desc + (uint64_t)((st * KV_BYTES) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks)
            umma_bf16(tmem + (uint32_t)(b * TILE_N), q_desc + (uint64_t)((ks >> 2) * (Q_ATOM >> 4) + (ks & 3) * 2),
                      bd + (uint64_t)((ks >> 2) * (KV_ATOM >> 4) + (ks & 3) * 2), idesc_s, ks > 0 ? 1u : 0u);
          umma_commit(&s_full[b]);
          umma_commit(&empty[st]);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      if (lane == 0) {
        if (!*vabort) atomicExch(err, 112);
        *vabort = 1;
      }
      for (uint32_t w = 0; q_issued > 0 && w < WAIT_LIMIT && !mbar_try_wait(&q_full, (uint32_t)(q_issued - 1) & 1u); ++w) {
      }
    }
    // the last product completes, and so have those before it
    for (uint32_t w = 0; u > 0 && w < WAIT_LIMIT && !mbar_try_wait(&s_full[(u - 1) & 1], (uint32_t)((u - 1) >> 1) & 1u); ++w) {
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ issuer of O += P V
    constexpr uint32_t idesc_o = make_idesc(BLOCK_M, HD, 0, 1);  // B = V: N (head dim) contiguous
    const uint64_t v_desc = desc_mnmajor(ring, KV_ATOM);
    bool ok = true;
    int i0 = 0, u = 0;
    for (; ok && walk.next(plan, seg); i0 += 2 * seg.n_tiles) {
      for (int t = 0; t < seg.n_tiles; ++t, ++u) {
        const int i = i0 + (t + 1 < seg.n_tiles ? 2 * t + 2 : 2 * t + 1), st = i % STAGES, b = u & 1;
        ok = mbar_wait(&p_full[b], (uint32_t)(u >> 1) & 1u, vabort) && mbar_wait(&full[st], (uint32_t)(i / STAGES) & 1u, vabort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        const uint64_t bd = v_desc + (uint64_t)((st * KV_BYTES) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < TILE_N / 16; ++ks)
            umma_bf16_ts(tmem + O_COL, tmem + (uint32_t)(b * TILE_N + (ks >> 1) * 32 + (ks & 1) * 8), bd + (uint64_t)(ks * (16 * 128 / 16)), idesc_o,
                         (t > 0 || ks > 0) ? 1u : 0u);
          umma_commit(&pv_done[b]);
          umma_commit(&empty[st]);
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) {
      if (!*vabort) atomicExch(err, 112);
      *vabort = 1;
    }
    for (uint32_t w = 0; u > 0 && w < WAIT_LIMIT && !mbar_try_wait(&pv_done[(u - 1) & 1], (uint32_t)((u - 1) >> 1) & 1u); ++w) {
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    // ------------------------------------------------------------------ softmax and epilogue: eight warps
    const int qd = warp & 3;             // TMEM lane quarter of this warp
    const int half = (warp - 4) >> 2;    // of a tile's keys, and of the output's columns
    const int r = qd * 32 + lane;        // query row of this thread
    const int ts = tid - 128;
    const uint32_t s_addr = tmem + ((uint32_t)(qd * 32) << 16), o_addr = s_addr + O_COL + (uint32_t)(half * (HD / 2));
    int i0 = 0, u = 0, bad_slot = 0;
    bool stop = false;
    auto gave_up = [&] {
      if (lane == 0) {
        if (!*vabort) atomicExch(err, 113);
        *vabort = 1;
      }
      __syncwarp();
    };
    for (; !stop && walk.next(plan, seg); i0 += 2 * seg.n_tiles, bad_slot = bad_slot == 2 ? 0 : bad_slot + 1) {
      const int tok = r < seg.rows ? seg.r.q0 + seg.node0 + div_by(r, plan.inv_grp) : -1;   // this row's token, or none
      int lo_row = 0;
      if (plan.window > 0 && tok >= 0) lo_row = seg.r.base + min(max(plan.depth[tok], 0), seg.r.n - 1) - plan.window + 1;
      // the row's exponent offset in use (none yet; what is no row has one that nothing exceeds) and the sum at it over this half's keys
      float m_run = tok >= 0 ? -INFINITY : INFINITY, l_run = 0.0f;
      bool ok = true;
      // tiles plain0 .. plain1 - 1 are seen whole by every row (tile_masked)
      const int plain1 = min(seg.r.base, seg.r.kv_len) / TILE_N - seg.tile_begin;
      const int plain0 = plan.window > 0 ? (max(seg.r.base + seg.r.n - plan.window, 0) + TILE_N - 1) / TILE_N - seg.tile_begin : 0;
      for (int t = 0; t < seg.n_tiles; ++t, ++u) {
        const int key0 = (seg.tile_begin + t) * TILE_N, b = u & 1;
        const bool masked = t < plain0 || t >= plain1;
        unsigned sees = 0u;
        if (masked && tok >= 0) sees = sees32(seg.r, plan, tok, lo_row, key0 + half * 32);
        const uint32_t phase = (uint32_t)(u >> 1) & 1u;
        if (!__all_sync(0xffffffffu, mbar_try_wait(&s_full[b], phase)))
          ok = __all_sync(0xffffffffu, ok && mbar_wait(&s_full[b], phase, vabort));
        if (!ok) {
          // the other warp of these rows may still have got its scores: it must find this one at the barriers of every tile
          gave_up();
          if (pair_bar_or(qd, false)) pair_bar_or(qd, false);
          continue;
        }
        fence_after();
        uint32_t v[32];                            // the scores of this half's keys
        tmem_ld32(s_addr + (uint32_t)(b * TILE_N + half * 32), v);
        tmem_ld_wait();
        if (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (!((sees >> j) & 1u)) v[j] = 0xff800000u;  // -inf
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 32; j += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mx4[e] = fmaxf(fmaxf(mx4[e], __uint_as_float(v[j + e])), __uint_as_float(v[j + 4 + e]));
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;  // the scale is positive
        // the exponent offset in use moves only when the maximum has grown enough, or at the first keys
        bool grow = mx > m_run + RESCALE_THRESHOLD;
        if (pair_bar_or(qd, grow)) {
          row_max[b][half][r] = mx;
          pair_bar_or(qd, false);
          mx = fmaxf(mx, row_max[b][half ^ 1][r]);
          grow = mx > m_run + RESCALE_THRESHOLD;
          const float alpha = (grow && m_run != -INFINITY) ? ex2_approx(m_run - mx) : 1.0f;
          if (grow) m_run = mx;
          if (t > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
            // once the tile before has left the tensor cores nothing else touches O until all P of this one is there
            if (!mbar_wait(&pv_done[b ^ 1], (uint32_t)((u - 1) >> 1) & 1u, vabort)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
              fence_after();
              l_run *= alpha;
#pragma unroll 1
              for (int c0 = 0; c0 < HD / 2; c0 += 16) {
                uint32_t o[16];
                tmem_ld16(o_addr + (uint32_t)c0, o);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                tmem_st16(o_addr + (uint32_t)c0, o);
              }
            }
          }
        }
        // P = exp2(S * scale - offset), two bf16 per column, over the S that was read;
        // rows that have seen no key yet (offset -inf) are all masked here: exp2(-inf) = 0 with any finite offset
        const float offset = m_run == -INFINITY ? 0.0f : m_run;
        const uint64_t scale2 = pack2(scale_log2, scale_log2), offset2 = pack2(-offset, -offset);
        uint64_t sum_a = 0ull, sum_b = 0ull;
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float x, y;
          unpack2(fma2((uint64_t)v[j] | ((uint64_t)v[j + 1] << 32), scale2, offset2), x, y);
          const float p0 = ex2_approx(x), p1 = ex2_approx(y);
          if (j & 2) sum_b = add2(sum_b, pack2(p0, p1));
          else sum_a = add2(sum_a, pack2(p0, p1));
          __nv_bfloat162 w = __floats2bfloat162_rn(p0, p1);
          pk[j >> 1] = *reinterpret_cast<uint32_t*>(&w);
        }
        tmem_st16(s_addr + (uint32_t)(b * TILE_N + half * 32), pk);
        float s0, s1;
        unpack2(add2(sum_a, sum_b), s0, s1);
        l_run += s0 + s1;
        // V of a masked tile: rows from the first key that was not loaded (shared memory never written, or an older tile) or that
        // lies at or beyond the request's length (whatever the page held before) are cleared, and so is every value that is
        // not finite: P = 0 must hide it. A thread has a quarter of one key's row.
        if (masked) {
          const int i = i0 + (t + 1 < seg.n_tiles ? 2 * t + 2 : 2 * t + 1), st = i % STAGES;
          const int loaded = min(n_boxes, (seg.r.kv_len - 1 - key0) / box_rows + 1) * box_rows;
          const int first_bad = min(seg.r.kv_len - key0, loaded);
          if (ok && !mbar_wait(&full[st], (uint32_t)(i / STAGES) & 1u, vabort)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (ok) {
            const int row = ts & (TILE_N - 1), c0 = (ts / TILE_N) * (2 * NA);     // 16-byte pieces c0 .. c0 + 2 NA - 1 of 8 NA
            unsigned char* vrow = ring + st * KV_BYTES + row * 128;
            auto piece_at = [&](int c) { return reinterpret_cast<uint4*>(vrow + (c >> 3) * KV_ATOM + (((c ^ row) & 7) << 4)); };
            if (row >= first_bad) {
#pragma unroll
              for (int c = 0; c < 2 * NA; ++c) *piece_at(c0 + c) = make_uint4(0, 0, 0, 0);
            } else {
              uint32_t any = 0u;
#pragma unroll
              for (int c = 0; c < 2 * NA; ++c) {
                const uint4 w = *piece_at(c0 + c);
                any |= not_finite(w.x) | not_finite(w.y) | not_finite(w.z) | not_finite(w.w);
              }
              if (any) {
                found_bad[bad_slot] = 1;
#pragma unroll 1
                for (int c = 0; c < 2 * NA; ++c) {
                  uint4 w = *piece_at(c0 + c);
                  w.x = without_not_finite(w.x);
                  w.y = without_not_finite(w.y);
                  w.z = without_not_finite(w.z);
                  w.w = without_not_finite(w.w);
                  *piece_at(c0 + c) = w;
                }
              }
            }
            fence_async_smem();
          }
        }
        tmem_st_wait();
        if (!ok) {
          gave_up();
          continue;
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
      }
      // ---- epilogue, when the last product has completed
      row_sum[half][r] = l_run;
      if (ok && !mbar_wait(&pv_done[(u - 1) & 1], (uint32_t)((u - 1) >> 1) & 1u, vabort)) ok = false;
      if (walk.g >= walk.hi) pdl_trigger();        // the last stretch of this CTA
      stop = softmax_bar_or(!ok || *vabort != 0);
      if (stop) {
        gave_up();
        break;
      }
      const bool cut = !seg.whole, bad = found_bad[bad_slot] != 0;
      const int slot = 2 * (int)blockIdx.x + (seg.began ? 0 : 1);
      float4* po = part_o + (size_t)slot * (HD / 4) * BLOCK_M + r;
      // One range of keys: O / l as bf16 through the shared memory that held Q (every product that read it has completed), so that
      // the rows go out in whole lines: 16-byte piece c of row r lies at slot c ^ (r % CPR) of its row. Cut: O as fp32 to scratch.
      constexpr int CPR = HD / 8;
      const float l_all = row_sum[0][r] + row_sum[1][r];
      const float inv = cut ? 1.0f : l_all == 0.0f ? 0.0f : 1.0f / l_all;
      fence_after();
#pragma unroll
      for (int c0 = 0; c0 < HD / 2; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(o_addr + (uint32_t)c0, o);
        tmem_ld_wait();
        const int col = half * (HD / 2) + c0;
        if (cut) {
          if (tok >= 0)
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              po[((col + j) / 4) * BLOCK_M] = make_float4(__uint_as_float(o[j]), __uint_as_float(o[j + 1]),
                                                          __uint_as_float(o[j + 2]), __uint_as_float(o[j + 3]));
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 w;
            __nv_bfloat162* hh = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              hh[e] = __floats2bfloat162_rn(__uint_as_float(o[j + 2 * e]) * inv, __uint_as_float(o[j + 2 * e + 1]) * inv);
            const int c = (col + j) >> 3;
            *reinterpret_cast<uint4*>(q_smem + r * (HD * 2) + ((c ^ (r & (CPR - 1))) << 4)) = w;
          }
        }
      }
      if (cut && tok >= 0 && half == 0) part_ml[(size_t)slot * BLOCK_M + r] = make_float2(m_run, l_all);
      fence_before();
      if (bad && tok >= 0) {
        // the values that were taken out of V, to the rows that see them (every thread finishes what it wrote)
#pragma unroll 1
        for (int d = half * (HD / 2); d < (half + 1) * (HD / 2); d += 8) {
          float x[8] = {};
#pragma unroll 1
          for (int k = 0; k < TILE_N / 32 * seg.n_tiles; ++k) {
            const int key0 = seg.tile_begin * TILE_N + 32 * k;
            if (tile_masked(seg.r, plan, key0 & ~(TILE_N - 1)))
              add_taken_out(x, sees32(seg.r, plan, tok, lo_row, key0), key0, seg.bt, plan, seg.kvh, v_cache, HD, d);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (x[e] == 0.0f) continue;
            if (cut) {
              float* at = reinterpret_cast<float*>(po + ((d + e) / 4) * BLOCK_M) + (e & 3);
              *at += x[e];
            } else {
              bf16* at = reinterpret_cast<bf16*>(q_smem + r * (HD * 2) + (((d >> 3) ^ (r & (CPR - 1))) << 4)) + e;
              *at = __float2bfloat16_rn(__bfloat162float(*at) + x[e]);
            }
          }
        }
      }
      if (!cut) {
        softmax_bar_or(false);
        const int c = ts % CPR;
        for (int row = ts / CPR; row < seg.rows; row += 256 / CPR) {
          const int node = div_by(row, plan.inv_grp), h = row - node * plan.grp;
          *reinterpret_cast<uint4*>(out + ((size_t)(seg.r.q0 + seg.node0 + node) * plan.nh + seg.kvh * plan.grp + h) * HD + c * 8) =
              *reinterpret_cast<const uint4*>(q_smem + row * (HD * 2) + ((c ^ (row & (CPR - 1))) << 4));
        }
      }
      if (plan.cuts != nullptr && !seg.began && ts == 0) plan.cuts[seg.unit] = Cut{(int)blockIdx.x, seg.pieces};     // for the second kernel
      // the slot of the stretch before, and of the one after the next: everyone read it before this stretch's barrier, and no one
      // writes it before the next one's
      if (ts == 0) found_bad[bad_slot == 0 ? 2 : bad_slot - 1] = 0;
      // what this warp read of O (tensor memory) and of the staged rows is in its registers or on its way out
      fence_async_smem();
      __syncwarp();
      if (!cut && lane == 0) mbar_arrive(&staged_out);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Joins the pieces of the units that were cut. A warp has 32 rows (the fast index, as in the scratch), DIMS dims and every WARPS-th
// piece, all its loads in flight at once where they fit; the WARPS warps of the same rows then join what they have, in order. What it
// takes is three round trips to the L2, if all warps are on the SMs at once: few units in many pieces take many warps with few
// dims each, many units in two or three pieces one warp per 32 rows and 32 dims.
template <int HD, int DIMS, int WARPS>
__global__ void __launch_bounds__(256, DIMS == 32 ? 2 : 3) attn_tree_tc_join_kernel(bf16* __restrict__ out, const float4* __restrict__ part_o,
                                                                   const float2* __restrict__ part_ml,
                                                                   const __grid_constant__ Plan plan) {
  constexpr int Q = DIMS / 4, U = DIMS == 8 ? 4 : 2;     // U: pieces of a warp in flight
  __shared__ float2 sh_ml[8][32];
  __shared__ float4 sh_o[8][Q][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % WARPS;
  const int group = (int)blockIdx.y * (8 / WARPS) + warp / WARPS, block = group / (HD / DIMS);
  const int unit = blockIdx.x, sh = unit / plan.m_tiles, m = unit - sh * plan.m_tiles;
  const int s = sh / plan.nkv, kvh = sh - s * plan.nkv;
  const Cut cut = plan.cuts[unit];                       // (not written where there is no such unit)
  const Req q = req_of(plan, s);
  const int node0 = m * plan.nodes_per_tile, step = plan.abreast;
  if (q.tiles <= 0 || m >= q.m_tiles || cut.pieces < 2) return;
  // (a CTA that gave up in a wait wrote no cut: what stands there instead must not lead out of the scratch)
  if (cut.cta < 0 || cut.cta >= plan.ctas || cut.pieces > (plan.ctas - cut.cta + step - 1) / step) return;
  const int rows = min(plan.nodes_per_tile, q.n - node0) * plan.grp;
  const int r = block * 32 + lane, d0 = (group - block * (HD / DIMS)) * DIMS;
  float M = -INFINITY, L = 0.0f, acc[DIMS] = {};
  // a piece of which the row sees nothing has neither weight nor maximum (but NaN scores have a sum without a maximum)
  auto take = [&](float2 ml, const float4 (&o)[Q]) {
    if (ml.x == -INFINITY && ml.y == 0.0f) return;
    const float m_new = fmaxf(M, ml.x);
    const float keep = M == m_new ? 1.0f : M == -INFINITY ? 0.0f : ex2_approx(M - m_new);
    const float f = ml.x == m_new ? 1.0f : ex2_approx(ml.x - m_new);
    M = m_new;
    L = L * keep + ml.y * f;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      const float v[4] = {o[k].x, o[k].y, o[k].z, o[k].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[4 * k + e] = fmaf(v[e], f, keep == 1.0f ? acc[4 * k + e] : acc[4 * k + e] * keep);
    }
  };
  if (r < rows)
    for (int k0 = mine; k0 < cut.pieces; k0 += WARPS * U) {
      float2 ml[U];
      float4 o[U][Q];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int piece = k0 + WARPS * k;
        ml[k] = make_float2(-INFINITY, 0.0f);
        if (piece < cut.pieces) {
          const size_t at = (size_t)(2 * (cut.cta + piece * step) + (piece == 0 ? 1 : 0)) * BLOCK_M;
          const float4* po = part_o + at * (HD / 4) + (d0 / 4) * BLOCK_M + r;
          ml[k] = part_ml[at + r];
#pragma unroll
          for (int e = 0; e < Q; ++e) o[k][e] = po[e * BLOCK_M];
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (k0 + WARPS * k < cut.pieces) take(ml[k], o[k]);
    }
  if (mine > 0) {
    sh_ml[warp][lane] = make_float2(M, L);
#pragma unroll
    for (int e = 0; e < Q; ++e) sh_o[warp][e][lane] = make_float4(acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]);
  }
  __syncthreads();
  if (mine > 0 || r >= rows) return;
#pragma unroll
  for (int w = 1; w < WARPS; ++w) {
    float4 o[Q];
#pragma unroll
    for (int e = 0; e < Q; ++e) o[e] = sh_o[warp + w][e][lane];
    take(sh_ml[warp + w][lane], o);
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  const int node = div_by(r, plan.inv_grp), g = r - node * plan.grp;
  bf16* to = out + ((size_t)(q.q0 + node0 + node) * plan.nh + kvh * plan.grp + g) * HD + d0;
#pragma unroll
  for (int d = 0; d < DIMS; d += 8) {
    uint4 w;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(acc[d + 2 * e] * inv, acc[d + 2 * e + 1] * inv);
    *reinterpret_cast<uint4*>(to + d) = w;
  }
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

struct Sizes {
  int grp, nodes, m_tiles, row_blocks, tiles, ctas, abreast, whole_tiles;
  bool cuts;                             // whether a unit may be cut: then there is a second kernel
  long long cut_bytes, part_floats;      // the scratch: the cuts, then the pieces
};
// 0 if the kernel does not take these shapes
bool sizes_of(Sizes& z, int S, int nh, int nkv, int hd, int page_size, int q_row_stride, float scale, int window, int max_q_len,
              int max_kv_len) {
  if ((hd != 64 && hd != 128) || nkv <= 0 || nh <= 0 || nh % nkv != 0 || nh / nkv > BLOCK_M || !(scale > 0.0f)) return false;
  if (page_size < 8 || (page_size & (page_size - 1)) || (q_row_stride & 7) || S <= 0 || max_q_len <= 0 || max_kv_len <= 0) return false;
  if (max_kv_len > MAX_KEYS || max_q_len > (1 << 24) || window < 0) return false;
  z.grp = nh / nkv;
  z.nodes = BLOCK_M / z.grp;
  z.m_tiles = (max_q_len + z.nodes - 1) / z.nodes;
  z.row_blocks = ((max_q_len < z.nodes ? max_q_len : z.nodes) * z.grp + 31) / 32;
  z.tiles = most_tiles(max_q_len, max_kv_len, window);
  const double line = (double)S * nkv * z.m_tiles * z.tiles;
  if (line > 1e9 || (double)S * nkv * z.m_tiles > 1e9) return false;
  int sms = 1;
  osb_num_sms(&sms);
  const int most = CTAS_PER_SM * sms;
  z.ctas = line < most ? (int)line : most;
  z.abreast = S == 1 && z.m_tiles > 1 && z.m_tiles <= z.ctas ? z.m_tiles : 1;
  z.whole_tiles = z.abreast == 1 && (long long)S * nkv * z.m_tiles <= z.ctas ? z.tiles : MAX_KEYS;
  z.cuts = z.tiles > 1 && z.whole_tiles > 1 + WHOLE_EXTRA;
  z.cut_bytes = z.cuts ? ((long long)S * nkv * z.m_tiles * (long long)sizeof(Cut) + 15) / 16 * 16 : 0;
  z.part_floats = z.cuts ? (long long)2 * z.ctas * BLOCK_M * (hd + 2) : 0;
  return true;
}

template <int HD>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, bf16* out, float* part, const bf16* v_cache,
           const Plan& plan, const Sizes& z, float scale_log2, cudaStream_t stream) {
  int rc = osb_allow_smem<attn_tree_tc_kernel<HD>>(Layout<HD>::SMEM);
  if (rc) return rc;
  float4* po = (float4*)part;
  float2* ml = (float2*)(part + (long long)2 * z.ctas * BLOCK_M * HD);
  rc = osb_launch(attn_tree_tc_kernel<HD>, dim3((unsigned)z.ctas), dim3(NUM_THREADS), Layout<HD>::SMEM, stream, mq, mk, mv, out, po, ml,
                  v_cache, plan, scale_log2);
  if (rc == 0 && z.cuts) {
    const int units = plan.S * plan.nkv * plan.m_tiles;
    // warps for so many dims each and so many sharing the pieces of a row: as many as make about one wave. Both kernels with each
    // of the four, in this order, us: one request of 2,048 keys on 2 kv heads 10.9, 12.2, 14.4, 22.7; 8 ragged ones of up to 4,096
    // on 4 kv heads 40.9, 30.3, 28.7, 30.3; 64 of 2,100 78.2, 55.2, 51.0, 49.6
    const long long groups = (long long)units * z.row_blocks, wave = 12LL * z.ctas;
    auto join = [&](auto k, int dims, int warps) {
      const int per_unit = z.row_blocks * (HD / dims), per_cta = 8 / warps;
      return osb_launch(k, dim3((unsigned)units, (unsigned)((per_unit + per_cta - 1) / per_cta)), dim3(256), 0, stream, out,
                        (const float4*)po, (const float2*)ml, plan);
    };
    if (groups * (HD / 8) * 8 <= wave) rc = join(attn_tree_tc_join_kernel<HD, 8, 8>, 8, 8);
    else if (groups * (HD / 16) * 4 <= wave) rc = join(attn_tree_tc_join_kernel<HD, 16, 4>, 16, 4);
    else if (groups * (HD / 16) * 2 <= wave / 3 * 4) rc = join(attn_tree_tc_join_kernel<HD, 16, 2>, 16, 2);
    else rc = join(attn_tree_tc_join_kernel<HD, 32, 1>, 32, 1);
  }
  return rc ? rc : osb_last_error();
}
}  // namespace

// Bytes of scratch that osb_attn_tree_tc needs for these arguments: 0 if it does not take them, 1 if it takes them and needs none.
OSB_API long long osb_attn_tree_tc_scratch(int S, int nh, int nkv, int hd, int page_size, int q_row_stride, float scale, int window,
                                           int max_q_len, int max_kv_len) {
  Sizes z;
  if (!sizes_of(z, S, nh, nkv, hd, page_size, q_row_stride, scale, window, max_q_len, max_kv_len)) return 0;
  return z.cuts ? z.cut_bytes + z.part_floats * 4 : 1;
}

// As osb_attn_tree for bf16 operands; scratch: osb_attn_tree_tc_scratch bytes for the same arguments, on a 16-byte boundary. Shapes
// for which that is 0 are refused with OSB_ERR_UNSUPPORTED.
OSB_API int osb_attn_tree_tc(void* out, const void* q, int q_row_stride, int T, const void* k_cache, const void* v_cache,
                             const int* block_table, int bt_stride, const int* cu_q, const int* seq_lens, const unsigned* mask,
                             int mask_words, const int* depth, int S, int nh, int nkv, int hd, int page_size, int num_pages,
                             float scale, int window, int max_q_len, int max_kv_len, void* scratch, int* err,
                             cudaStream_t stream) {
  if (S <= 0 || T <= 0 || max_q_len <= 0) return OSB_OK;
  Sizes z;
  if (num_pages <= 0 || !sizes_of(z, S, nh, nkv, hd, page_size, q_row_stride, scale, window, max_q_len, max_kv_len))
    return OSB_ERR_UNSUPPORTED;
  if ((max_q_len - 1) / 32 >= mask_words) return OSB_ERR_BAD_SHAPE;
  if (((uintptr_t)q & 15) || ((uintptr_t)k_cache & 15) || ((uintptr_t)v_cache & 15) || ((uintptr_t)out & 15))
    return OSB_ERR_UNSUPPORTED;
  if ((window > 0 && depth == nullptr) || (z.cuts && (scratch == nullptr || ((uintptr_t)scratch & 15)))) return OSB_ERR_BAD_SHAPE;
  Plan p = {};
  p.block_table = block_table;
  p.cu_q = cu_q;
  p.seq_lens = seq_lens;
  p.mask = mask;
  p.depth = depth;
  p.err = err;
  p.cuts = z.cuts ? (Cut*)scratch : nullptr;
  p.bt_stride = bt_stride;
  p.mask_words = mask_words;
  p.T = T;
  p.S = S;
  p.nh = nh;
  p.nkv = nkv;
  p.grp = z.grp;
  while ((1 << p.log2ps) < page_size) ++p.log2ps;
  p.num_pages = num_pages;
  p.window = window;
  p.max_q_len = max_q_len;
  const long long table = (long long)bt_stride * page_size;     // keys behind the block table cannot be read
  p.kv_cap = table < max_kv_len ? (int)table : max_kv_len;
  p.nodes_per_tile = z.nodes;
  p.m_tiles = z.m_tiles;
  p.ctas = z.ctas;
  p.abreast = z.abreast;
  p.whole_tiles = z.whole_tiles;
  p.inv_nodes = z.nodes == 1 ? 0u : (unsigned)((0x100000000ull + z.nodes - 1) / z.nodes);
  p.inv_grp = z.grp == 1 ? 0u : (unsigned)((0x100000000ull + z.grp - 1) / z.grp);
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
    const cuuint32_t box[4] = {64, (cuuint32_t)(page_size < TILE_N ? page_size : TILE_N), 1, 1};
    int rc = make_map_bf16(&mk, k_cache, 4, dims, strides, box);
    if (rc) return rc;
    rc = make_map_bf16(&mv, v_cache, 4, dims, strides, box);
    if (rc) return rc;
  }
  float* part = (float*)((unsigned char*)scratch + z.cut_bytes);
  const float scale_log2 = scale * LOG2E;
  if (hd == 64) return launch<64>(mq, mk, mv, (bf16*)out, part, (const bf16*)v_cache, p, z, scale_log2, stream);
  return launch<128>(mq, mk, mv, (bf16*)out, part, (const bf16*)v_cache, p, z, scale_log2, stream);
}
OSB_PACKED(osb_attn_tree_tc)
OSB_PACKED(osb_attn_tree_tc_scratch)
