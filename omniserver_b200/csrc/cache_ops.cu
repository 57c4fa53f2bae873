// Moving tokens and pages of the paged cache [layers, 2, pages, kv heads, page size, head size].
//
// `compact_kernel`: after a tree of drafted tokens has been verified, the tokens of the accepted path lie at places base + path[i]
// of their request (base: the request's committed tokens) and have to lie at base + i, in every layer, for keys, values and
// every head. A path ascends, so path[i] >= i and a token never moves onto one that has yet to move if they move in order:
// a thread owns one piece of 16 bytes of one head's row and takes it along the whole path, up to eight tokens in flight, so no
// order between threads is needed. Bound: four loads in a chain (counts and offsets, the path, page numbers, tokens; a few of 4 to 16 KB a
// layer): 3.1 us for one request in 28 layers of 2 heads, 5.6 for 64 requests in 28 of 4 (10.9 MB).
//
// `copy_pages_kernel`: whole pages, e.g. the last, partly filled page of a request that is forked. A page of one layer's keys or
// values is contiguous; a CTA copies 16 KB of it with 16-byte loads, four in flight per thread. Bound: the copy rate of the
// memory: 64 pages of 32 tokens in 28 layers of 4 heads (235 MB read and written) 37 us, 6.3 TB/s; one page 1.7 us. The pairs of pages
// come as kernel arguments (the host owns the block tables), so a call needs no copy to the device.
#include "common.cuh"

namespace {
constexpr int THREADS = 256;
constexpr int BATCH = 8;            // tokens in flight per thread
constexpr int PATH_TILE = 256;      // entries of a path whose places are worked out at once
enum : int { ERR_SLOT = 3, ERR_PATH = 6 };

template <typename U>
__global__ void __launch_bounds__(THREADS) compact_kernel(U* __restrict__ cache, const int* __restrict__ block_table,
                                                          int bt_stride, const int* __restrict__ cu_q,
                                                          const int* __restrict__ seq_lens, const int* __restrict__ path,
                                                          int path_stride, const int* __restrict__ counts, int planes,
                                                          int num_pages, int nkv, int page_size, int row_units,
                                                          int* __restrict__ err) {
  __shared__ long long from[PATH_TILE], to[PATH_TILE];   // row of (page, offset) within a plane's head 0, or -1: stays
  pdl_wait();
  const int s = blockIdx.y, tid = threadIdx.x;
  const int n = counts[s];
  const int q_len = cu_q[s + 1] - cu_q[s];
  const int base = seq_lens[s] - q_len;
  const int* p = path + (size_t)s * path_stride;
  if (n <= 0) return;
  // a path that leaves its tree or does not ascend moves nothing
  bool ok = n <= path_stride && n <= q_len && base >= 0;
  bool moves = false;
  if (ok)
    for (int i = tid; i < n; i += THREADS) {
      const int a = p[i];
      ok = ok && a >= 0 && a < q_len && (i == 0 || p[i - 1] < a);
      moves = moves || a != i;
    }
  if (!__syncthreads_and(ok)) {
    if (blockIdx.x == 0 && tid == 0) atomicExch(err, ERR_PATH);
    return;
  }
  if (!__syncthreads_or(moves)) return;      // the accepted tokens lie where they belong
  // this thread's piece: unit u of the row of head h in plane (layer, keys or values)
  const long long item = (long long)blockIdx.x * THREADS + tid;
  const int u = (int)(item % row_units);
  const long long hp = item / row_units;
  const int h = (int)(hp % nkv);
  const long long plane = hp / nkv;
  const bool mine = plane < planes;
  U* own = cache + ((size_t)plane * num_pages * nkv + h) * page_size * row_units + u;
  const int* bt = block_table + (size_t)s * bt_stride;
  for (int t0 = 0; t0 < n; t0 += PATH_TILE) {
    const int m = min(PATH_TILE, n - t0);
    __syncthreads();
    if (tid < m) {
      const int i = t0 + tid, a = p[i];
      long long f = -1, d = -1;
      if (a != i) {
        const int sf = (base + a) / page_size, sd = (base + i) / page_size;
        const int pf = sf < bt_stride ? bt[sf] : -1, pd = sd < bt_stride ? bt[sd] : -1;
        if (pf < 0 || pf >= num_pages || pd < 0 || pd >= num_pages) {
          atomicExch(err, ERR_SLOT);
        } else {
          f = (long long)pf * nkv * page_size + (base + a) % page_size;
          d = (long long)pd * nkv * page_size + (base + i) % page_size;
        }
      }
      from[tid] = f;
      to[tid] = d;
    }
    __syncthreads();
    if (mine)
      for (int i0 = 0; i0 < m; i0 += BATCH) {
        U v[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
          if (i0 + k < m && from[i0 + k] >= 0) v[k] = own[(size_t)from[i0 + k] * row_units];
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
          if (i0 + k < m && from[i0 + k] >= 0) own[(size_t)to[i0 + k] * row_units] = v[k];
      }
  }
}

constexpr int MAX_PAIRS = 256;
struct PagePairs {
  int src[MAX_PAIRS], dst[MAX_PAIRS];
};
constexpr int COPY_LOADS = 4;

template <typename U>
__global__ void __launch_bounds__(THREADS) copy_pages_kernel(U* __restrict__ cache, const __grid_constant__ PagePairs pairs,
                                                             long long page_units, long long plane_units, int blocks_per_page) {
  pdl_wait();
  const int pair = blockIdx.x / blocks_per_page, part = blockIdx.x - pair * blocks_per_page;
  const size_t plane = (size_t)blockIdx.y * plane_units;
  const U* src = cache + plane + (size_t)pairs.src[pair] * page_units;
  U* dst = cache + plane + (size_t)pairs.dst[pair] * page_units;
  const long long i0 = (long long)part * (THREADS * COPY_LOADS) + threadIdx.x;
  U v[COPY_LOADS];
#pragma unroll
  for (int k = 0; k < COPY_LOADS; ++k)
    if (i0 + k * THREADS < page_units) v[k] = src[i0 + k * THREADS];
#pragma unroll
  for (int k = 0; k < COPY_LOADS; ++k)
    if (i0 + k * THREADS < page_units) dst[i0 + k * THREADS] = v[k];
}

// f(Tag<unit>) with the largest unit of 16, 4 or 2 bytes that divides `bytes` and that the address is a multiple of
template <typename F> int with_unit(long long bytes, const void* at, F&& f) {
  if (bytes % 16 == 0 && ((uintptr_t)at & 15) == 0) return f(Tag<uint4>{});
  if (bytes % 4 == 0 && ((uintptr_t)at & 3) == 0) return f(Tag<unsigned>{});
  return f(Tag<unsigned short>{});
}
}  // namespace

// cache: `planes` = layers x 2 planes [num_pages, nkv, page_size, hd] of elements of elem_size bytes (2 or 4), one behind the
// other. path [S, path_stride], counts [S]: the first counts[s] entries of row s ascend and lie below the request's number of nodes.
OSB_API int osb_compact_cache(void* cache, int elem_size, int planes, int num_pages, int nkv, int page_size, int hd,
                              const int* block_table, int bt_stride, const int* cu_q, const int* seq_lens, const int* path,
                              int path_stride, const int* counts, int S, int* err, cudaStream_t stream) {
  if (S <= 0 || planes <= 0 || path_stride <= 0) return OSB_OK;
  if ((elem_size != 2 && elem_size != 4) || num_pages <= 0 || nkv <= 0 || page_size <= 0 || hd <= 0) return OSB_ERR_BAD_SHAPE;
  if (S > 65535) return OSB_ERR_TOO_LARGE;
  const long long row_bytes = (long long)hd * elem_size;
  return with_unit(row_bytes, cache, [&](auto tag) {
    typedef OSB_T(tag) U;
    const int row_units = (int)(row_bytes / (long long)sizeof(U));
    const long long blocks = ((long long)planes * nkv * row_units + THREADS - 1) / THREADS;
    if (blocks > 2147483647LL) return (int)OSB_ERR_TOO_LARGE;
    const int rc = osb_launch(compact_kernel<U>, dim3((unsigned)blocks, (unsigned)S), dim3(THREADS), 0, stream, (U*)cache,
                              block_table, bt_stride, cu_q, seq_lens, path, path_stride, counts, planes, num_pages, nkv,
                              page_size, row_units, err);
    return rc ? rc : osb_last_error();
  });
}

// cache as above; src, dst: n page numbers on the host, every dst once and none of them a src (the caller has checked).
OSB_API int osb_copy_pages(void* cache, long long page_bytes, int planes, int num_pages, const int* src, const int* dst, int n,
                           cudaStream_t stream) {
  if (n <= 0 || planes <= 0) return OSB_OK;
  if (page_bytes <= 0 || page_bytes % 2 || num_pages <= 0) return OSB_ERR_BAD_SHAPE;
  if (planes > 65535) return OSB_ERR_TOO_LARGE;
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages) return OSB_ERR_BAD_SHAPE;
  return with_unit(page_bytes, cache, [&](auto tag) {
    typedef OSB_T(tag) U;
    const long long units = page_bytes / (long long)sizeof(U);
    const long long per_page = (units + THREADS * COPY_LOADS - 1) / (THREADS * COPY_LOADS);
    if (per_page * MAX_PAIRS > 2147483647LL) return (int)OSB_ERR_TOO_LARGE;
    for (int i0 = 0; i0 < n; i0 += MAX_PAIRS) {
      const int m = n - i0 < MAX_PAIRS ? n - i0 : MAX_PAIRS;
      PagePairs pairs;
      for (int i = 0; i < m; ++i) {
        pairs.src[i] = src[i0 + i];
        pairs.dst[i] = dst[i0 + i];
      }
      for (int i = m; i < MAX_PAIRS; ++i) pairs.src[i] = pairs.dst[i] = 0;
      const int rc = osb_launch(copy_pages_kernel<U>, dim3((unsigned)(per_page * m), (unsigned)planes), dim3(THREADS), 0, stream,
                                (U*)cache, pairs, units, units * num_pages, (int)per_page);
      if (rc) return rc;
    }
    return osb_last_error();
  });
}
OSB_PACKED(osb_compact_cache)
OSB_PACKED(osb_copy_pages)
