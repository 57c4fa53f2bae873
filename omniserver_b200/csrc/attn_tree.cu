// Attention of a tree of drafted tokens over the paged cache: any types, head sizes and page sizes, in 32 bits.
//
// A request's drafted tokens (nodes) lie in the cache behind its committed ones, node j at place base + j. Node i sees every
// committed key and the nodes whose bit is set in its row of mask words (its ancestors and itself); with a window w only places
// above base + depth[i] - w, a node's own place counting as base + depth. o = sum softmax(q k scale) v over those; a node that
// sees nothing gets zeros. Query head h reads kv head h / (nh / nkv).
//
// The query rows of a request and kv head are its nodes times the group's heads (row = node x group + head). A CTA takes 32 rows
// and one range of keys in tiles of 32: keys and values pass through shared memory as fp32 once for all rows, scores and outputs
// are register tiles (4 rows x 2 keys, 4 rows x HD / 16 dims a thread) with an online softmax.
// What bounds it at the sizes of a step of drafted tokens is latency: a CTA has a few tiles, loads one, meets three barriers and sums, with
// nothing of the next tile under way, and three CTAs share an SM (134 registers a thread at 128 dims; the 64-dim forms keep 12 to 20 bytes in
// local memory). 4 requests of 24 nodes and 1,000 keys, 12 heads on 2, by counters: 16 % of an SM's warps, the fp32 pipe 25 % and the
// load pipe 16 % busy, a third of a warp's time between instructions spent on loads from memory.
// A request's keys are cut into ranges of 64 and more that are joined by a second kernel in order: as many as make, with its row
// tiles, up to 128 CTAs per kv head (a CTA by itself keeps few loads and sums going: 4 requests of 24 nodes and 1,000 keys, 12 heads
// on 2, took 83 us in ranges of 256 keys; they take 34 to 38, 9 to 10 TFLOP/s; with up to 64 CTAs 40 to 47). The cut
// depends on the request's own nodes and keys alone, so a node's result does not depend on the batch it was in. Sums run in
// key order within a row's lane and in a fixed tree across the lanes.
// A key that a row does not see is left out, not multiplied by zero: what a masked place holds (NaN, infinities) does not matter.
#include "attn_tree.cuh"

namespace {
using namespace attn_tree;
constexpr int RT = 32, KT = 32, NT = 128;   // query rows, keys per tile, threads
constexpr int ROWS = 4, KEYS = 2;           // a thread's piece of the scores
constexpr int MIN_RANGE = 64, MAX_CTAS = 128; // keys of a range at least; row tiles x ranges of a request and kv head at most

// Keys per range of a request with `rows` query rows per kv head, and how many ranges that makes.
__host__ __device__ __forceinline__ int range_keys(int kv_len, int rows) {
  const int tiles = rows <= 0 ? 1 : (rows - 1) / RT + 1, most = tiles >= MAX_CTAS ? 1 : MAX_CTAS / tiles;
  const int per = kv_len <= 0 ? 1 : (kv_len - 1) / most + 1;
  return (per + MIN_RANGE - 1) / MIN_RANGE * MIN_RANGE;
}
__host__ __device__ __forceinline__ int num_ranges(int kv_len, int rows) {
  return kv_len <= 0 ? 1 : (kv_len - 1) / range_keys(kv_len, rows) + 1;
}
// Rows of scratch per request and kv head: row x its ranges, for requests of up to these sizes.
__host__ __device__ __forceinline__ int scratch_rows(int max_kv_len, long long max_rows) {
  const long long all = max_rows * ((max_kv_len - 1) / MIN_RANGE + 1), most = (long long)RT * MAX_CTAS;
  return (int)(all < most ? all : most);
}

template <typename T> __device__ __forceinline__ void load4(const T* p, bool vec, int left, float (&v)[4]);
template <> __device__ __forceinline__ void load4<float>(const float* p, bool vec, int left, float (&v)[4]) {
  if (vec) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? p[e] : 0.0f;
  }
}
template <> __device__ __forceinline__ void load4<bf16>(const bf16* p, bool vec, int left, float (&v)[4]) {
  if (vec) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const float2 a = __bfloat1622float2(h[0]), b = __bfloat1622float2(h[1]);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? to_f32(p[e]) : 0.0f;
  }
}

// HDP: the head size rounded up to 64, 128 or 256
template <typename QT, typename KVT, typename OT, int HDP>
__global__ void __launch_bounds__(NT) attn_tree_kernel(
    OT* __restrict__ out, float* __restrict__ part_o, float* __restrict__ part_ml, const QT* __restrict__ q,
    int q_row_stride, const KVT* __restrict__ k_cache, const KVT* __restrict__ v_cache, const int* __restrict__ block_table,
    int bt_stride, const int* __restrict__ cu_q, const int* __restrict__ seq_lens, const unsigned* __restrict__ mask,
    int mask_words, const int* __restrict__ depth, int nh, int nkv, int hd, int page_size, int num_pages, float scale,
    int window, int max_ranges, int cap_rows, int max_q_len, int kv_cap, int T, int* __restrict__ err) {
  constexpr int LD = HDP + 4;
  constexpr int ND = HDP / 64;       // 4-dim pieces of an output row per thread
  extern __shared__ __align__(16) float sm[];
  float* qs = sm;                    // [RT][LD]
  float* ks = qs + RT * LD;          // [KT][LD]
  float* vs = ks + KT * LD;          // [KT][LD]
  float* ps = vs + KT * LD;          // [RT][KT + 4]: weights, -1 where the row does not see the key
  __shared__ long long s_at[KT];     // where a key's row of this kv head begins in the caches, or -1: no key, or no page
  pdl_wait();
  const int split = blockIdx.x % max_ranges, tile = blockIdx.x / max_ranges;
  const int kvh = blockIdx.y, s = blockIdx.z;
  const int q0 = cu_q[s], n = cu_q[s + 1] - q0;
  if (q0 < 0 || n < 0 || q0 + n > T) {        // tokens that are not there
    if (tile == 0 && split == 0 && threadIdx.x == 0) atomicExch(err, ERR_BOUNDS);
    return;
  }
  const int grp = nh / nkv, rows = min(n, max_q_len) * grp, r0 = tile * RT;
  if (r0 >= rows) return;
  const int kv_all = seq_lens[s], kv_len = min(kv_all, kv_cap);
  const int base = kv_all - n;
  const int chunk = range_keys(kv_len, rows), n_splits = num_ranges(kv_len, rows);
  if (split >= n_splits) return;
  const int k_begin = split * chunk, k_end = min(kv_len, k_begin + chunk);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  if ((kv_all > kv_len || n > max_q_len || base < 0) && split == 0 && tid == 0) atomicExch(err, ERR_BOUNDS);

  const bool vec = (hd & 3) == 0 && ((q_row_stride & 3) == 0) &&
                   (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0;
  for (int i = tid; i < RT * (HDP / 4); i += NT) {
    const int r = i / (HDP / 4), d = (i - r * (HDP / 4)) * 4;
    float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (r0 + r < rows && d < hd) {
      const int node = (r0 + r) / grp, h = kvh * grp + (r0 + r) % grp;
      load4(q + (size_t)(q0 + node) * q_row_stride + (size_t)h * hd + d, vec, hd - d, f);
    }
    *reinterpret_cast<float4*>(qs + r * LD + d) = make_float4(f[0], f[1], f[2], f[3]);
  }
  float acc[ROWS][ND][4], m[ROWS], l[ROWS];
  int node_of[ROWS], lo_of[ROWS];    // a row's node (-1: no row) and the first place that it sees
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = r0 + ty * ROWS + i;
    node_of[i] = r < rows ? r / grp : -1;
    lo_of[i] = 0;
    if (window > 0 && node_of[i] >= 0) lo_of[i] = base + min(max(depth[q0 + node_of[i]], 0), n - 1) - window + 1;
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[i][d][0] = acc[i][d][1] = acc[i][d][2] = acc[i][d][3] = 0.0f;
  }

  for (int k0 = k_begin; k0 < k_end; k0 += KT) {
    if (window > 0 && k0 + KT <= base - window + 1) continue;    // behind every row's window
    __syncthreads();
    if (tid < KT) {
      const int key = k0 + tid;
      int page = -1;
      if (key < k_end) {
        page = block_table[(size_t)s * bt_stride + key / page_size];
        if (page < 0 || page >= num_pages) {
          // a page that a window has passed was given back: no row sees it, and nobody is told
          if (window <= 0 || key > base - window) atomicExch(err, ERR_PAGE);
          page = -1;
        }
      }
      s_at[tid] = page < 0 ? -1 : (((long long)page * nkv + kvh) * page_size + key % page_size) * hd;
    }
    __syncthreads();
#pragma unroll 8      // (a tile's loads at once: 34.5 us for those requests, 36.9 with four)
    for (int i = tid; i < KT * (HDP / 4); i += NT) {
      const int r = i / (HDP / 4), d = (i - r * (HDP / 4)) * 4;
      float a[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      const long long at = s_at[r];
      if (at >= 0 && d < hd) {
        load4(k_cache + at + d, vec, hd - d, a);
        load4(v_cache + at + d, vec, hd - d, b);
      }
      *reinterpret_cast<float4*>(ks + r * LD + d) = make_float4(a[0], a[1], a[2], a[3]);
      *reinterpret_cast<float4*>(vs + r * LD + d) = make_float4(b[0], b[1], b[2], b[3]);
    }
    __syncthreads();
    float sc[ROWS][KEYS] = {};
#pragma unroll 4
    for (int d = 0; d < HDP; d += 4) {
      float4 a[ROWS], b[KEYS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) a[i] = *reinterpret_cast<const float4*>(qs + (ty * ROWS + i) * LD + d);
#pragma unroll
      for (int j = 0; j < KEYS; ++j) b[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * LD + d);
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int j = 0; j < KEYS; ++j)
          sc[i][j] = fmaf(a[i].w, b[j].w, fmaf(a[i].z, b[j].z, fmaf(a[i].y, b[j].y, fmaf(a[i].x, b[j].x, sc[i][j]))));
    }
    // all keys of the tile are committed, present and inside every row's window: no mask
    const bool plain = k0 + KT <= min(base, k_end) && window <= 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      bool sees[KEYS];
#pragma unroll
      for (int j = 0; j < KEYS; ++j) {
        const int key = k0 + tx + 16 * j;
        sees[j] = node_of[i] >= 0 && s_at[tx + 16 * j] >= 0;
        if (!plain && sees[j]) {
          const int dj = key - base;
          if (dj >= 0) {
            sees[j] = dj < n && (dj >> 5) < mask_words &&
                      ((mask[(size_t)(q0 + node_of[i]) * mask_words + (dj >> 5)] >> (dj & 31)) & 1u);
            if (sees[j] && window > 0) sees[j] = base + depth[q0 + dj] >= lo_of[i];
          } else {
            sees[j] = key >= lo_of[i];
          }
        }
        sc[i][j] = sees[j] ? sc[i][j] * scale : -INFINITY;
      }
      // NaN scores stay: fmaxf leaves them out of the maximum, exp keeps them
      float mx = fmaxf(sc[i][0], sc[i][1]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float m_new = fmaxf(m[i], mx);
      const float ref = m_new == -INFINITY ? 0.0f : m_new;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < KEYS; ++j) {
        const float p = sees[j] ? expf(sc[i][j] - ref) : 0.0f;
        sum += p;
        ps[(ty * ROWS + i) * (KT + 4) + tx + 16 * j] = sees[j] ? p : -1.0f;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float alpha = m[i] == -INFINITY ? 0.0f : expf(m[i] - m_new);
      l[i] = m[i] == m_new ? l[i] + sum : l[i] * alpha + sum;
      if (m[i] != m_new)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][d][e] *= alpha;
      m[i] = m_new;
    }
    __syncwarp();     // a warp's 8 rows of weights are read by itself alone
#pragma unroll 2
    for (int j0 = 0; j0 < KT; j0 += 4) {
      float p4[ROWS][4];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(ps + (ty * ROWS + i) * (KT + 4) + j0);
        p4[i][0] = f.x; p4[i][1] = f.y; p4[i][2] = f.z; p4[i][3] = f.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float4 v[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) v[d] = *reinterpret_cast<const float4*>(vs + (j0 + j) * LD + (tx + 16 * d) * 4);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const float p = p4[i][j];
          if (!plain && p == -1.0f) continue;     // not seen (a weight that is NaN is not)
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            acc[i][d][0] = fmaf(p, v[d].x, acc[i][d][0]);
            acc[i][d][1] = fmaf(p, v[d].y, acc[i][d][1]);
            acc[i][d][2] = fmaf(p, v[d].z, acc[i][d][2]);
            acc[i][d][3] = fmaf(p, v[d].w, acc[i][d][3]);
          }
        }
      }
    }
  }
  const size_t prow0 = ((size_t)s * nkv + kvh) * cap_rows;      // this request's and kv head's rows of scratch
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (node_of[i] < 0) continue;
    const int h = kvh * grp + (r0 + ty * ROWS + i) % grp;
    const size_t row = (size_t)(q0 + node_of[i]) * nh + h;
    const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int dim = (tx + 16 * d) * 4;
      if (n_splits == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (dim + e < hd) out[row * hd + dim + e] = from_f32<OT>(acc[i][d][e] * inv);
      } else {
        float* po = part_o + (prow0 + (size_t)(r0 + ty * ROWS + i) * n_splits + split) * hd + dim;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (dim + e < hd) po[e] = acc[i][d][e];
      }
    }
    if (n_splits > 1 && tx == 0) {
      part_ml[(prow0 + (size_t)(r0 + ty * ROWS + i) * n_splits + split) * 2] = m[i];
      part_ml[(prow0 + (size_t)(r0 + ty * ROWS + i) * n_splits + split) * 2 + 1] = l[i];
    }
  }
}

// Joins the ranges of a row in order: a warp per (node, head).
template <typename OT>
__global__ void __launch_bounds__(128) attn_tree_join_kernel(OT* __restrict__ out, const float* __restrict__ part_o,
                                                             const float* __restrict__ part_ml, const int* __restrict__ cu_q,
                                                             const int* __restrict__ seq_lens, int nh, int nkv, int hd,
                                                             int max_q_len, int kv_cap, int cap_rows, int T) {
  constexpr int HELD = MAX_CTAS / 32;       // ranges whose weights a lane has: k, k + 32, ..
  pdl_wait();
  const int s = blockIdx.z, kvh = blockIdx.y, q0 = cu_q[s], q1 = cu_q[s + 1], n = min(q1 - q0, max_q_len);
  if (q0 < 0 || q1 > T) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = nh / nkv, rows = n * grp, r = blockIdx.x * 4 + warp;
  if (r >= rows) return;
  const int ranges = num_ranges(min(seq_lens[s], kv_cap), rows);
  if (ranges == 1) return;
  const size_t prow = ((size_t)s * nkv + kvh) * cap_rows + (size_t)r * ranges;
  const int node = r / grp, h = kvh * grp + r - node * grp;
  const size_t row = (size_t)(q0 + node) * nh + h;
  float m[HELD], f[HELD], top = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    const int k = lane + 32 * e;
    const float2 ml = k < ranges ? reinterpret_cast<const float2*>(part_ml)[prow + k] : make_float2(-INFINITY, 0.0f);
    m[e] = ml.x;
    f[e] = ml.y;
    top = fmaxf(top, m[e]);
  }
  const float M = warp_max(top);
#pragma unroll
  for (int e = 0; e < HELD; ++e) {
    // a range of which the row sees nothing counts for nothing; NaN scores leave a sum without a maximum
    const bool empty = m[e] == -INFINITY && f[e] == 0.0f;
    const float w = empty ? 0.0f : m[e] == -INFINITY ? 1.0f : expf(m[e] - M);
    l += empty ? 0.0f : f[e] * w;
    f[e] = empty ? -1.0f : w;
  }
  const float L = warp_sum(l), inv = L == 0.0f ? 0.0f : 1.0f / L;
  // a lane has four dims (heads of no multiple of 4: one by one, further ones in further rounds)
  const bool vec = (hd & 3) == 0;
  const int width = vec ? 4 : 1;
  for (int d0 = 0; d0 < hd; d0 += 32 * width) {
    const int d = d0 + lane * width;
    float a[4] = {};
#pragma unroll
    for (int e = 0; e < HELD; ++e) {
#pragma unroll 8
      for (int k = 0; k < min(32, ranges - 32 * e); ++k) {
        const float w = __shfl_sync(0xffffffffu, f[e], k);
        const float* po = part_o + (prow + 32 * e + k) * hd + d;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (d < hd) {
          if (vec) x = *reinterpret_cast<const float4*>(po);
          else x.x = *po;
        }
        if (w < 0.0f) continue;
        a[0] = fmaf(x.x, w, a[0]);
        a[1] = fmaf(x.y, w, a[1]);
        a[2] = fmaf(x.z, w, a[2]);
        a[3] = fmaf(x.w, w, a[3]);
      }
    }
    if (d < hd)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < width) out[row * hd + d + e] = from_f32<OT>(a[e] * inv);
  }
}
}  // namespace

// Floats of scratch that osb_attn_tree needs for these arguments (0: none).
OSB_API long long osb_attn_tree_scratch(int S, int nh, int nkv, int hd, int max_q_len, int max_kv_len) {
  if (S <= 0 || nkv <= 0 || nh < nkv || hd <= 0 || max_q_len <= 0 || max_kv_len <= MIN_RANGE) return 0;
  return (long long)S * nkv * scratch_rows(max_kv_len, (long long)max_q_len * (nh / nkv)) * (hd + 2) + 1;
}

// out [T, nh*hd]; q rows of q_row_stride elements, caches [num_pages, nkv, page_size, hd], mask [T, mask_words] words, depth [T]
// (needed with a window; below the request's number of nodes), scratch: osb_attn_tree_scratch floats for the same arguments.
// max_q_len / max_kv_len: at least the largest of the batch; a request beyond them is reported in *err, and what lies beyond is
// not computed.
OSB_API int osb_attn_tree(void* out, int out_dtype, const void* q, int q_dtype, int q_row_stride, int T, const void* k_cache,
                          const void* v_cache, int cache_dtype, const int* block_table, int bt_stride, const int* cu_q,
                          const int* seq_lens, const unsigned* mask, int mask_words, const int* depth, int S, int nh, int nkv,
                          int hd, int page_size, int num_pages, float scale, int window, int max_q_len, int max_kv_len,
                          float* scratch, int* err, cudaStream_t stream) {
  if (S <= 0 || T <= 0 || max_q_len <= 0) return OSB_OK;
  if (hd <= 0 || nkv <= 0 || nh % nkv != 0 || page_size <= 0 || (window > 0 && depth == nullptr) ||
      (max_q_len - 1) / 32 >= mask_words)
    return OSB_ERR_BAD_SHAPE;
  if (hd > 256) return OSB_ERR_UNSUPPORTED;
  if (S > 65535 || nkv > 65535 || max_kv_len > MAX_KEYS) return OSB_ERR_TOO_LARGE;
  const long long need = osb_attn_tree_scratch(S, nh, nkv, hd, max_q_len, max_kv_len);
  if (need > 0 && (scratch == nullptr || ((uintptr_t)scratch & 15))) return OSB_ERR_BAD_SHAPE;
  const long long table = (long long)bt_stride * page_size;     // keys behind the block table cannot be read
  const int kv_cap = table < max_kv_len ? (int)table : max_kv_len;
  const long long max_rows = (long long)max_q_len * (nh / nkv), tiles = (max_rows + RT - 1) / RT;
  if (max_rows > MAX_KEYS) return OSB_ERR_TOO_LARGE;
  // the most ranges of a request in the batch: one with a single row tile is cut most
  const int ranges = max_kv_len <= 0 ? 1 : num_ranges(max_kv_len < MIN_RANGE * MAX_CTAS ? max_kv_len : MIN_RANGE * MAX_CTAS, 1);
  if (tiles * ranges > 2147483647LL) return OSB_ERR_TOO_LARGE;
  const int cap_rows = need > 0 ? scratch_rows(max_kv_len, max_rows) : 0;
  float* part_o = scratch;                             // rows of hd floats, then (maximum, sum)
  float2* part_ml = (float2*)(scratch + (((long long)S * nkv * cap_rows * hd + 1) & ~1LL));
  return osb_dispatch(q_dtype, [&](auto qt) {
    return osb_dispatch(cache_dtype, [&](auto kt) {
      return osb_dispatch(out_dtype, [&](auto ot) {
        typedef OSB_T(qt) QT;
        typedef OSB_T(kt) KVT;
        typedef OSB_T(ot) OT;
        const int hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
        const size_t smem = sizeof(float) * ((size_t)(RT + 2 * KT) * (hdp + 4) + RT * (KT + 4));
        auto go = [&](auto k, int rc) -> int {
          if (rc) return rc;
          return osb_launch(k, dim3((unsigned)(tiles * ranges), (unsigned)nkv, (unsigned)S), dim3(NT), smem, stream, (OT*)out,
                            part_o, (float*)part_ml, (const QT*)q, q_row_stride, (const KVT*)k_cache, (const KVT*)v_cache, block_table,
                            bt_stride, cu_q, seq_lens, mask, mask_words, depth, nh, nkv, hd, page_size, num_pages, scale,
                            window, ranges, cap_rows, max_q_len, kv_cap, T, err);
        };
        int rc = hdp == 64    ? go(attn_tree_kernel<QT, KVT, OT, 64>, osb_allow_smem<attn_tree_kernel<QT, KVT, OT, 64>>(smem))
                 : hdp == 128 ? go(attn_tree_kernel<QT, KVT, OT, 128>, osb_allow_smem<attn_tree_kernel<QT, KVT, OT, 128>>(smem))
                              : go(attn_tree_kernel<QT, KVT, OT, 256>, osb_allow_smem<attn_tree_kernel<QT, KVT, OT, 256>>(smem));
        if (rc == 0 && need > 0)
          rc = osb_launch(attn_tree_join_kernel<OT>, dim3((unsigned)((max_rows + 3) / 4), (unsigned)nkv, (unsigned)S), dim3(128), 0,
                          stream, (OT*)out, (const float*)part_o, (const float*)part_ml, cu_q, seq_lens, nh, nkv, hd, max_q_len,
                          kv_cap, cap_rows, T);
        return rc ? rc : osb_last_error();
      });
    });
  });
}
OSB_PACKED(osb_attn_tree)
OSB_PACKED(osb_attn_tree_scratch)
