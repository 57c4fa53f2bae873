// Verification of drafted tokens against the target's probabilities from given random numbers.
//
// A request brings a tree of nodes (node 0: the last token it has, the others: drafted tokens, parents before children)
// and one fp32 row of logits per node. At node i with p = softmax(l_i / T) the children are tested in index order with
// r = p at first: child c with token x and random number u_c in [0, 1) is accepted if u_c q(x) < r(x), where q is the
// draft's distribution behind node i (a point mass at x if there is none: u_c < r(x)). A rejection leaves
// r <- max(r - q, 0) / sum (without q: r(x) <- 0, renormalised; r stays as it was if nothing is left). The walk ends where no
// child is accepted, and the next token is drawn there from r: the smallest index whose running sum passes u times the total,
// u being the root's random number (the root itself is never tested). Emitted tokens then follow the target's distribution:
// without q whatever the drafts are; with q if siblings were drawn from it independently of one another, the same word twice at times
// (drawn without putting words back, each would need a q of its own, less the words before it and renormalised). Rows with T <= 0 are
// greedy: p is one at the first largest logit. A row of which no logit is above -inf accepts nothing, and its next token is 0.
//
// Two kernels. `verify_stats_kernel` reads every logit once (what bounds the operator: T x V x 4 bytes): a warp takes 1,024 words of
// one row in registers, the next 1,024 on their way meanwhile, and leaves their maximum, its first place, and the sum of
// exp((l - maximum) / T); no two warps wait for each other. `verify_walk_kernel` then needs a few numbers per node to walk the tree;
// the draw scans one slice of 1,024 words. Only a rejection against a draft's distribution needs its whole row, and the row of
// logits, once more: then a cluster of CTAs walks the request together, each CTA summing its part of the row.
// Measured, both kernels: 256 rows of 152,064 words (156 MB) in 8 trees 39.8 us, some 27 of them (5.8 TB/s) the first one, the walk the
// rest; 32 chains of 6 drafts with draft probabilities (224 of those rows, and some rows of both kinds once more) 47; one chain of 6
// rows 10.3, of which the walk's chain of loads is 6.
//
// Numbers. A word's weight is one fp32 value W = 2^(l c - m c), c = log2(e) / T and m the maximum of its slice, as one fused
// multiply-add and one exponential (the first kernel has no time for more: at the memory's rate an SM has 22 cycles for 32 words);
// m c is rounded, and the slice's factor 2^(m c - m_row c) takes the same rounded numbers, so that all words of
// a row are off by one common factor and each by some 2^-22 of its own, at random. Sums and comparisons are in 64 bits: what
// is left of a row behind a random number near 1, or when its largest words were rejected, would not survive 32. A rejected word's
// weight is the same number that went into its slice's sum; it is subtracted where that leaves enough of the sum for its digits, and where
// it does not, what is left is summed again without the rejected words (KEPT). A weight of 2^-126 of the row's largest or less may be 0: 32
// bits end there, and a random number of 24 bits is no finer than 0 for it (of 11,000 random walks those that differed from 64 bits all drew
// with 0 and a word lighter than that).
#include <cooperative_groups.h>

#include "mma_utils.cuh"

namespace cg = cooperative_groups;

namespace {
constexpr int SLICE = 1024;            // words of a row that a warp of the first kernel takes at a time
constexpr int STAT_THREADS = 128;
constexpr int STAT_WARPS = STAT_THREADS / 32;
constexpr int STAT_STAGES = 2;         // slices of a warp in shared memory: the one in hand and the next
// Of the first kernel on an SM: 20 warps of 8 KB and 96 registers a thread. (Six leave 80 registers, and fewer loads from shared memory
// ahead of the arithmetic: 256 rows of 152,064 words 42.5 us with the walk instead of 39.3; four 41.4.)
constexpr int STAT_CTAS = 5;
constexpr int PER_LANE = SLICE / 32;
constexpr int MAX_CLUSTER = 8;
constexpr float MIN_TEMP = 1e-30f, MAX_TEMP = 1e38f;   // others are taken as these: log2(e) / T is finite and has all its bits
enum : int { ERR_TOKEN = 5, ERR_BOUNDS = 7 };

struct SliceStat {
  double sum;    // of the weights against the slice's own maximum
  float mx;      // the slice's largest logit (NaN counts as -inf)
  int arg;       // greedy rows: its first place in the row
};

// log2(e) / T, right to the last place: a division in 32 bits and its remainder (a division in 64 takes some 500 cycles)
__device__ __forceinline__ float log2e_over(float t) {
  constexpr float HI = 1.44269502f, LO = (float)(1.4426950408889634074 - (double)HI);
  t = fminf(fmaxf(t, MIN_TEMP), MAX_TEMP);
  const float q = HI / t;
  return fmaf(fmaf(-q, t, HI) + LO, q * 0.69314718f, q);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A slice whose maximum is infinite, or so large that the rounding of m c is no small number any more (half a unit of 2^22 is 1/4; at
// a temperature of 1e-8 it would be 128, and the weights out of range): the weights are then those of the differences l - m.
__device__ __forceinline__ bool odd_slice(float m, float c) { return !(fabsf(m * c) < 4194304.0f); }
// The weight of a word of an ordinary slice, mc = m * c; 0 for -inf and NaN (the maximum of a number and NaN is the number).
__device__ __forceinline__ float weight(float l, float c, float mc) { return ex2(fmaxf(fmaf(l, c, -mc), -200.0f)); }
__device__ __forceinline__ float weight_any(float l, float m, float c) {
  if (!odd_slice(m, c)) return weight(l, c, m * c);
  if (m == -INFINITY) return 0.0f;
  return l == m ? 1.0f : ex2(fmaxf((l - m) * c, -200.0f));
}
// A slice's factor against its row's maximum, from the numbers that the weights of both were taken against (m c rounded, or exactly m c
// in an odd slice): exact to some 2^-22 like a weight, and then used in 64 bits.
__device__ __forceinline__ double factor(float m, float m_row, float c) {
  if (m == -INFINITY) return 0.0;
  if (m == m_row) return 1.0;
  if (m_row == INFINITY) return 0.0;
  const float mc = m * c, rc = m_row * c;
  float x;
  if (!odd_slice(m, c)) x = odd_slice(m_row, c) ? fmaf(-m_row, c, mc) : __fsub_rn(mc, rc);
  else x = odd_slice(m_row, c) ? (m - m_row) * c : fmaf(m, c, -rc);
  return (double)ex2(fmaxf(x, -200.0f));
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_scan_d(double v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Words i .. i + 3 of a row, `fill` from `end` on; `wide`: rows and i are multiples of 16 bytes.
__device__ __forceinline__ void load4(const float* row, int i, int end, bool wide, float fill, float (&v)[4]) {
  if (wide && i + 4 <= end) {
    const float4 f = *reinterpret_cast<const float4*>(row + i);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < end ? row[i + e] : fill;
  }
}

__device__ __forceinline__ void max_combine(float& bv, int& bi, float v, int i) {
  if (v > bv || (v == bv && i < bi)) {
    bv = v;
    bi = i;
  }
}

// A warp: `per_warp` slices one after the other, the next one's words on their way into shared memory meanwhile. Rows behind the
// last request are skipped.
__global__ void __launch_bounds__(STAT_THREADS, STAT_CTAS) verify_stats_kernel(SliceStat* __restrict__ stats,
                                                                               const float* __restrict__ logits,
                                                                               const int* __restrict__ cu_q,
                                                                               const float* __restrict__ temperature, int S,
                                                                               int V, int n_slices, int n_items, int per_warp) {
  extern __shared__ __align__(16) float ring[];      // [warp][stage][SLICE]
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long first = ((long long)blockIdx.x * STAT_WARPS + warp) * per_warp;
  pdl_trigger();
  if (first >= n_items) return;
  const int item1 = (int)min((long long)n_items, first + per_warp);
  float* mine = ring + warp * (STAT_STAGES * SLICE);
  const bool vec = ((V & 3) == 0) && (((uintptr_t)logits & 15) == 0);
  // asks for the words of slice s of row r; those behind the row's end are zeros
  auto ask = [&](int r, int s, int stage) {
    const float* x = logits + (size_t)r * V + s * SLICE;
    float* to = mine + stage * SLICE;
    const int left = V - s * SLICE;
    if (vec) {
#pragma unroll
      for (int k = 0; k < PER_LANE / 4; ++k) {
        const int i = 4 * (lane + 32 * k);
        cp_async16(to + i, i < left ? x + i : x, i < left);
      }
    } else {
#pragma unroll
      for (int k = 0; k < PER_LANE; ++k) {
        const int i = lane + 32 * k;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(smem_u32(to + i)), "l"(i < left ? x + i : x),
                     "r"(i < left ? 4 : 0));
      }
    }
  };
  int row = (int)first / n_slices, sl = (int)first - row * n_slices;      // of the slice in hand
  int ask_row = row, ask_sl = sl;                                         // of the slice to ask for next
  int known_row = -1, req = 0;
  float c = 0.0f;
  bool sums = false;
  for (int k = 0; k < STAT_STAGES - 1; ++k) {
    if ((int)first + k < item1) ask(ask_row, ask_sl, k);
    cp_async_commit();
    if (++ask_sl == n_slices) ask_sl = 0, ++ask_row;
  }
  int stage = 0;
  for (int item = (int)first; item < item1; ++item) {
    if (item + STAT_STAGES - 1 < item1) ask(ask_row, ask_sl, stage == 0 ? STAT_STAGES - 1 : stage - 1);
    cp_async_commit();
    if (++ask_sl == n_slices) ask_sl = 0, ++ask_row;
    if (row != known_row) {
      // the row's request, as many as end at or before it: 32 ends at a time
      req = 0;
      for (int end = S; end > req;) {
        const int step = (end - req + 31) / 32, at = req + lane * step;
        const int cnt = __popc(__ballot_sync(0xffffffffu, at < end && cu_q[min(at, S - 1) + 1] <= row));
        if (cnt == 0) break;
        end = min(end, req + cnt * step);
        req += (cnt - 1) * step + 1;
      }
      const float temp = req < S && temperature != nullptr ? temperature[req] : 0.0f;
      sums = temp > 0.0f;
      c = log2e_over(sums ? temp : 1.0f);
      known_row = row;
    }
    cp_async_wait<STAT_STAGES - 1>();
    __syncwarp();
    if (req >= S) break;       // and all rows behind it
    // lane t has words 4 (t + 32 k) .. + 3 of the slice
    float v[PER_LANE];
    const float* from = mine + stage * SLICE;
#pragma unroll
    for (int k = 0; k < PER_LANE / 4; ++k) {
      const float4 f = *reinterpret_cast<const float4*>(from + 4 * (lane + 32 * k));
      v[4 * k] = f.x;
      v[4 * k + 1] = f.y;
      v[4 * k + 2] = f.z;
      v[4 * k + 3] = f.w;
    }
    __syncwarp();              // the stage may be filled again
    const int left = V - sl * SLICE;
    if (left < SLICE) {
#pragma unroll
      for (int k = 0; k < PER_LANE; ++k)
        if (4 * (lane + 32 * (k >> 2)) + (k & 3) >= left) v[k] = -INFINITY;
    }
    float most[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int k = 4; k < PER_LANE; ++k) most[k & 3] = fmaxf(most[k & 3], v[k]);      // leaves NaN out
    const float bv = warp_max(fmaxf(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), -INFINITY));
    int bi = 0;
    double sum = 0.0;
    if (sums) {
      double part[4] = {0.0, 0.0, 0.0, 0.0};
      if (!odd_slice(bv, c)) {
        const float mc = bv * c;
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) part[k & 3] += (double)ex2(fmaf(v[k], c, -mc));
        sum = (part[0] + part[1]) + (part[2] + part[3]);
        if (sum != sum) {                        // a NaN among the words: once more, with care
          sum = 0.0;
#pragma unroll
          for (int k = 0; k < PER_LANE; ++k) sum += (double)weight(v[k], c, mc);
        }
      } else {
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) sum += (double)weight_any(v[k], bv, c);
      }
      sum = warp_sum_d(sum);
    } else {
      // greedy: the maximum's first place (places ascend within a lane)
      bi = 0x7fffffff;
      if (bv > -INFINITY) {
#pragma unroll
        for (int k = PER_LANE - 1; k >= 0; --k)
          if (v[k] == bv) bi = 4 * (lane + 32 * (k >> 2)) + (k & 3);
      }
      bi = __reduce_min_sync(0xffffffffu, bi);
      if (bi == 0x7fffffff) bi = 0;
    }
    if (lane == 0) stats[item] = SliceStat{sum, bv, sl * SLICE + bi};
    stage = stage + 1 == STAT_STAGES ? 0 : stage + 1;
    if (++sl == n_slices) sl = 0, ++row;
  }
  cp_async_wait<0>();          // nothing of this warp is on its way when its shared memory goes
}

// A difference of sums is used as long as it is at least this part of the sum that it started from: a sum is right to some 2^-50, so what
// is left of it to some 2^-26, a sixteenth of what a word's weight is off by.
constexpr double KEPT = 1.0 / (1 << 24);

constexpr int WALK_THREADS = 512;
constexpr int WALK_WARPS = WALK_THREADS / 32;
constexpr int HELD = 5;               // slices a lane keeps in registers (a vocabulary of 163,840 words); more are read again
struct WalkSmem {                     // the fixed part; per-node and per-slice arrays follow
  double part[2][WALK_WARPS];         // the CTA's sums of its parts of a row, warp by warp: after the last rejection, and the one in hand
  double scan[WALK_WARPS];
  double before;                      // the draw: the running sum in front of `slice`
  int slice, pick, last_pos;
};

// One request: one CTA, or (DENSE: with draft_probs) one cluster, every CTA of which walks alike; see the top of the file. What it
// takes is a chain of round trips to memory (the request's place, its nodes and slices, its tokens' logits, the slice drawn
// from), so loads that do not depend on one another are issued together, and numbers that the walk needs are made for all nodes
// at once.
template <bool DENSE>
__global__ void __launch_bounds__(WALK_THREADS, 1) verify_walk_kernel(
    int* __restrict__ out_tokens, int* __restrict__ out_path, int* __restrict__ out_count,
    const SliceStat* __restrict__ stats, const float* __restrict__ logits, const int* __restrict__ tokens,
    const int* __restrict__ parents, const int* __restrict__ cu_q, const float* __restrict__ uniform,
    const float* __restrict__ temperature, const float* __restrict__ draft_probs, int T, int V, int n_slices, int max_nodes,
    int max_depth, int* __restrict__ err) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  WalkSmem& sh = *reinterpret_cast<WalkSmem*>(smem_raw);
  double* ztot = reinterpret_cast<double*>(smem_raw + ((sizeof(WalkSmem) + 15) & ~(size_t)15));   // [max_nodes] a node's total weight
  double* ptok = ztot + max_nodes;                 // [max_nodes] a node's token's weight (DENSE: probability) behind its parent
  double* psl = ptok + max_nodes;                  // [max_nodes] without q: the weight of the slice that the word is in
  double* rej_left = psl + max_nodes;              // [max_nodes] without q: what a rejected word left of its slice
  float* fac = reinterpret_cast<float*>(rej_left + max_nodes);   // DENSE: [n_slices] probability of a weight of 1, of the node in hand
  float* smx = fac + n_slices;                     // DENSE: [n_slices]
  float* rmx = smx + n_slices;                     // [max_nodes] a node's largest logit
  float* qtok = rmx + max_nodes;                   // [max_nodes] q of a node's token
  float* unif = qtok + max_nodes;                  // [max_nodes]
  float* rej_inv = unif + max_nodes;               // [max_nodes] with q: 1 / what a rejection left
  int* amax = reinterpret_cast<int*>(rej_inv + max_nodes);
  int* tok = amax + max_nodes;
  int* par = tok + max_nodes;
  int* rej = par + max_nodes;                      // [max_nodes] rejected tokens at the node in hand
  int* path = rej + max_nodes;                     // [max_nodes] the nodes of the walk

  cg::cluster_group cluster = cg::this_cluster();
  const int csize = DENSE ? (int)cluster.num_blocks() : 1, crank = DENSE ? (int)cluster.block_rank() : 0;
  const int s = blockIdx.x / csize;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto everyone = [&]() {
    if (DENSE && csize > 1) cluster.sync(); else __syncthreads();
  };
  pdl_wait();
  const int q0 = cu_q[s], q1 = cu_q[s + 1];
  const float tempf = temperature != nullptr ? temperature[s] : 0.0f;
  const int n = q0 >= 0 && q1 <= T ? min(q1 - q0, max_nodes) : -1;     // (tokens that are not there: none)
  if ((n < 0 || n != q1 - q0) && crank == 0 && tid == 0) atomicExch(err, ERR_BOUNDS);
  const int width = max_depth + 1;
  int* my_tokens = out_tokens + (size_t)s * width;
  int* my_path = out_path + (size_t)s * width;
  if (n <= 0) {            // a request without nodes (the whole cluster leaves)
    if (crank == 0) {
      for (int i = tid; i < width; i += WALK_THREADS) my_tokens[i] = my_path[i] = -1;
      if (tid == 0) out_count[s] = 0;
    }
    return;
  }
  const bool greedy = !(tempf > 0.0f);
  const float c = log2e_over(greedy ? 1.0f : tempf);
  const SliceStat* my_stats = stats + (size_t)q0 * n_slices;
  const float* my_logits = logits + (size_t)q0 * V;
  const float* my_q = DENSE ? draft_probs + (size_t)q0 * V : nullptr;

  // A thread's node (further ones below), and the first node of which this warp adds up the slices.
  int t = -1, p = -1;
  float u = 0.0f;
  if (tid < n) {
    t = tokens[q0 + tid];
    p = parents[q0 + tid];
    u = uniform[q0 + tid];
  }
  SliceStat h[HELD];
  auto load_slices = [&](int i) {
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      h[k] = i < n && lane + 32 * k < n_slices ? my_stats[(size_t)i * n_slices + lane + 32 * k] : SliceStat{0.0, -INFINITY, 0x7fffffff};
  };
  load_slices(warp);
  auto is_child = [&](int i, int ti, int pi) { return !greedy && pi >= 0 && pi < i && ti >= 0 && ti < V; };
  float tok_l = 0.0f, tok_m = -INFINITY, tok_q = 1.0f;    // of this thread's node: its token's logit, that slice's maximum, q
  double tok_s = 0.0;                                     // and, without q, its sum
  auto load_token = [&](int i, int ti, int pi) {
    if (!is_child(i, ti, pi)) return;
    tok_l = my_logits[(size_t)pi * V + ti];
    const SliceStat& st = my_stats[(size_t)pi * n_slices + ti / SLICE];
    tok_m = st.mx;
    if (!DENSE) tok_s = st.sum;
    if (DENSE) tok_q = my_q[(size_t)pi * V + ti];
  };
  load_token(tid, t, p);
  for (int i = tid; i < n; i += WALK_THREADS) {
    if (i != tid) {
      t = tokens[q0 + i];
      p = parents[q0 + i];
      u = uniform[q0 + i];
    }
    tok[i] = t;
    par[i] = p;
    unif[i] = u;
    if (i > 0 && (t < 0 || t >= V) && crank == 0) atomicExch(err, ERR_TOKEN);
  }
  // a node's maximum, its first place, and its total weight
  for (int i = warp; i < n; i += WALK_WARPS) {
    if (i != warp) load_slices(i);
    const SliceStat* st = my_stats + (size_t)i * n_slices;
    float bv = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < HELD; ++k) max_combine(bv, bi, h[k].mx, h[k].arg);
    for (int k = lane + 32 * HELD; k < n_slices; k += 32) max_combine(bv, bi, st[k].mx, st[k].arg);
    const float row_mx = warp_max(bv);
    bi = __reduce_min_sync(0xffffffffu, bv == row_mx ? bi : 0x7fffffff);
    double z = 0.0;
    if (!greedy) {
#pragma unroll
      for (int k = 0; k < HELD; ++k) z += h[k].sum * factor(h[k].mx, row_mx, c);
      for (int k = lane + 32 * HELD; k < n_slices; k += 32) z += st[k].sum * factor(st[k].mx, row_mx, c);
      z = warp_sum_d(z);
    }
    if (lane == 0) {
      rmx[i] = row_mx;
      amax[i] = bi == 0x7fffffff ? 0 : bi;
      ztot[i] = z;
    }
  }
  if (tid == 0) {
    path[0] = 0;
    sh.pick = 0x7fffffff;
    sh.last_pos = -1;
  }
  __syncthreads();
  for (int i = tid; i < n; i += WALK_THREADS) {
    const int ti = tok[i], pi = par[i];
    double x = 0.0, in_slice = 0.0;
    if (i != tid) load_token(i, ti, pi);
    if (is_child(i, ti, pi) && ztot[pi] > 0.0) {
      const double f = factor(tok_m, rmx[pi], c) * (DENSE ? 1.0 / ztot[pi] : 1.0);
      x = (double)weight_any(tok_l, tok_m, c) * f;
      if (!DENSE) in_slice = tok_s * f;
    }
    ptok[i] = x;
    if (!DENSE) psl[i] = in_slice;
    qtok[i] = is_child(i, ti, pi) ? fmaxf(tok_q, 0.0f) : 1.0f;      // 0 for NaN
  }
  __syncthreads();

  int cur = 0, count = 1, n_rej = 0, last = 0;
  double rest = ztot[0], row_total = 0.0;               // without q: weight left at the node in hand / with q: what the last pass summed
  bool have_parts = false, have_fac = false;
  // the parts of a row that this CTA's warps take in a pass: contiguous, in order of (CTA, warp)
  const int span = ((V + csize * WALK_WARPS - 1) / (csize * WALK_WARPS) + 3) & ~3;
  const bool wide = (V & 3) == 0 && (((uintptr_t)logits | (uintptr_t)draft_probs) & 15) == 0;
  // with q: the probability of a word after `k` rejections at the node in hand, x before them and q its draft probability. Products
  // and differences are rounded one by one wherever a word is looked at (no fused multiply-add): the sum of a row and the running
  // sum of the draw have to be of the same numbers.
  auto take_out = [](float x, float q) -> float { return fmaxf(__fsub_rn(x, q), 0.0f); };
  auto after = [&](float x, float q, int k) -> float {
    for (int i = 0; i < k; ++i) x = __fmul_rn(take_out(x, q), rej_inv[i]);
    return x;
  };
  // Without q, where differences are not enough: what the first k words of the list leave of slice `sl` of the node in hand, and of its
  // row. (The whole CTA; the numbers are the same in every thread.)
  auto cta_sum = [&](double v) -> double {
    v = warp_sum_d(v);
    __syncthreads();
    if (lane == 0) sh.scan[warp] = v;
    __syncthreads();
    return warp_sum_d(lane < WALK_WARPS ? sh.scan[lane] : 0.0);
  };
  auto sum_slice = [&](int sl, int k) -> double {
    const float m = my_stats[(size_t)cur * n_slices + sl].mx;
    const double f = factor(m, rmx[cur], c);
    double v = 0.0;
    for (int i = sl * SLICE + tid; i < min(V, (sl + 1) * SLICE); i += WALK_THREADS) {
      double w = (double)weight_any(my_logits[(size_t)cur * V + i], m, c) * f;
      for (int r = 0; r < k; ++r)
        if (rej[r] == i) w = 0.0;
      v += w;
    }
    return cta_sum(v);
  };
  // slice sl, whose sum is x
  auto slice_left = [&](int sl, const SliceStat& x, int k) -> double {
    for (int r = k - 1; r >= 0; --r)
      if (rej[r] / SLICE == sl) return rej_left[r];
    return x.sum * factor(x.mx, rmx[cur], c);
  };
  auto sum_row = [&](int k) -> double {
    const SliceStat* st = my_stats + (size_t)cur * n_slices;
    double v = 0.0;
    for (int sl = tid; sl < n_slices; sl += WALK_THREADS) v += slice_left(sl, st[sl], k);
    return cta_sum(v);
  };
  while (count <= max_depth) {
    // the next child of cur behind the one tested last
    int j = n;
    for (int b = (last + 1) & ~31; b < n; b += 32) {
      const unsigned hit = __ballot_sync(0xffffffffu, b + lane > last && b + lane < n && par[b + lane] == cur);
      if (hit) {
        j = b + __ffs(hit) - 1;
        break;
      }
    }
    if (j >= n) break;
    last = j;
    const int word = tok[j];
    if (word < 0 || word >= V) continue;         // no word: it cannot be accepted, and takes nothing away
    bool yes;
    if (greedy) {
      yes = rmx[cur] > -INFINITY && word == amax[cur];      // (a row without logits has no best word)
    } else if (!DENSE) {
      double x = ptok[j], in_slice = psl[j];
      for (int k = 0; k < n_rej; ++k) {
        if (rej[k] == word) x = 0.0;             // rejected before: nothing of it is left
        if (rej[k] / SLICE == word / SLICE) in_slice = rej_left[k];
      }
      yes = (double)unif[j] * rest < x;
      if (!yes && x > 0.0) {
        in_slice -= x;
        __syncthreads();                          // everyone has read the list
        if (tid == 0) {
          rej[n_rej] = word;
          rej_left[n_rej] = in_slice;
        }
        __syncthreads();
        if (in_slice < psl[j] * KEPT) {
          in_slice = sum_slice(word / SLICE, n_rej + 1);
          if (tid == 0) rej_left[n_rej] = in_slice;
          __syncthreads();
        }
        double left = rest - x;
        if (left < ztot[cur] * KEPT) left = sum_row(n_rej + 1);
        // (where nothing would be left the word stays)
        if (left > 0.0) {
          ++n_rej;
          rest = left;
        }
      }
    } else {
      const float q = qtok[j];
      yes = (double)unif[j] * (double)q < (n_rej == 0 ? ptok[j] : (double)after((float)ptok[j], q, n_rej));
      if (!yes && ztot[cur] > 0.0) {
        // what is left of the row: its sum, warp by warp over contiguous parts
        if (!have_fac) {                          // maxima and factors of the node's slices
          const SliceStat* st = my_stats + (size_t)cur * n_slices;
          const double inv = 1.0 / ztot[cur];
          for (int k = tid; k < n_slices; k += WALK_THREADS) {
            const float m = st[k].mx;
            smx[k] = m;
            fac[k] = (float)(factor(m, rmx[cur], c) * inv);
          }
          have_fac = true;
          __syncthreads();
        }
        const float* x = my_logits + (size_t)cur * V;
        const float* dq = my_q + (size_t)cur * V;
        const int a = min((crank * WALK_WARPS + warp) * span, V), e = min(a + span, V);
        constexpr int UNROLL = 5;       // 4 words of both rows each, in flight
        double part[4] = {0.0, 0.0, 0.0, 0.0};
        for (int i0 = a; i0 < e; i0 += 128 * UNROLL) {
          float xl[UNROLL][4], ql[UNROLL][4];
          if (wide && i0 + 128 * UNROLL <= e) {        // no test between the loads: all of them in flight at once
#pragma unroll
            for (int k = 0; k < UNROLL; ++k) {
              const float4 fx = *reinterpret_cast<const float4*>(x + i0 + 128 * k + 4 * lane);
              const float4 fq = *reinterpret_cast<const float4*>(dq + i0 + 128 * k + 4 * lane);
              xl[k][0] = fx.x; xl[k][1] = fx.y; xl[k][2] = fx.z; xl[k][3] = fx.w;
              ql[k][0] = fq.x; ql[k][1] = fq.y; ql[k][2] = fq.z; ql[k][3] = fq.w;
            }
          } else {
#pragma unroll
            for (int k = 0; k < UNROLL; ++k) {
              const int i = i0 + 128 * k + 4 * lane;
              load4(x, i, e, wide, -INFINITY, xl[k]);
              load4(dq, i, e, wide, 0.0f, ql[k]);
            }
          }
#pragma unroll
          for (int k = 0; k < UNROLL; ++k) {
            const int sl = min(i0 + 128 * k + 4 * lane, V - 1) / SLICE;     // four words lie in one slice
            const float m = smx[sl], f = fac[sl];
            if (n_rej == 0 && !odd_slice(m, c)) {
              const float mc = m * c;
#pragma unroll
              for (int w = 0; w < 4; ++w) part[w] += (double)take_out(__fmul_rn(weight(xl[k][w], c, mc), f), fmaxf(ql[k][w], 0.0f));
            } else {
              for (int w = 0; w < 4; ++w) {
                const float qq = fmaxf(ql[k][w], 0.0f);
                part[w] += (double)take_out(after(__fmul_rn(weight_any(xl[k][w], m, c), f), qq, n_rej), qq);
              }
            }
          }
        }
        const double sum = warp_sum_d((part[0] + part[1]) + (part[2] + part[3]));
        everyone();                     // nobody still reads the parts of an earlier pass
        double* mine = sh.part[n_rej & 1];
        if (lane == 0) mine[warp] = sum;
        everyone();
        double total = 0.0;             // the same in every warp: the CTAs in order, a CTA's warps in a fixed tree
        for (int r = 0; r < csize; ++r) {
          const double* from = csize > 1 ? cluster.map_shared_rank(mine, r) : mine;
          total += warp_sum_d(lane < WALK_WARPS ? from[lane] : 0.0);
        }
        if (total > 0.0) {
          if (tid == 0) rej_inv[n_rej] = (float)(1.0 / total);
          ++n_rej;
          row_total = total;
          have_parts = true;
        }
        __syncthreads();
      }
    }
    if (yes) {
      cur = j;
      if (tid == 0) path[count] = j;
      ++count;
      n_rej = 0;
      rest = ztot[j];
      have_parts = have_fac = false;
    }
  }

  // the draw at node cur: a range [a, e) of words, the running sum in front of it and the target
  double target = 0.0, before = 0.0, one_fac = 0.0;
  float one_mx = 0.0f;
  int a = 0, e = 0;
  const bool search = !greedy && ztot[cur] > 0.0;
  const bool parts = DENSE && have_parts;
  if (search && !parts && crank == 0) {
    // slice by slice, less what was rejected; a lane of the first warp has consecutive slices
    const SliceStat* st = my_stats + (size_t)cur * n_slices;
    target = (double)unif[0] * rest;
    if (warp == 0) {
      auto left = [&](int k, const SliceStat& x) -> double { return slice_left(k, x, n_rej); };
      const int per = (n_slices + 31) / 32, k0 = min(lane * per, n_slices), k1 = min(k0 + per, n_slices);
      double held[HELD], v = 0.0;
#pragma unroll
      for (int k = 0; k < HELD; ++k) h[k] = k0 + k < k1 ? st[k0 + k] : SliceStat{0.0, -INFINITY, 0};
#pragma unroll
      for (int k = 0; k < HELD; ++k) v += held[k] = k0 + k < k1 ? left(k0 + k, h[k]) : 0.0;
#pragma unroll 1
      for (int k = k0 + HELD; k < k1; ++k) v += left(k, st[k]);
      const double inc = warp_scan_d(v, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, v > 0.0 && inc > target), pos = __ballot_sync(0xffffffffu, v > 0.0);
      // the lane in whose slices the target is passed; if it rounded up to the total, the last one that has weight
      const int src = hit ? __ffs(hit) - 1 : pos ? 31 - __clz(pos) : 0;
      if (lane == src) {
        int found = k0;
        double run = inc - v, in_front = run;
        bool passed = false;
#pragma unroll
        for (int k = 0; k < HELD; ++k)
          if (!passed && held[k] > 0.0) {
            found = k0 + k;
            in_front = run;
            run += held[k];
            passed = run > target;
          }
#pragma unroll 1
        for (int k = k0 + HELD; k < k1 && !passed; ++k) {
          const double w = left(k, st[k]);
          if (w > 0.0) {
            found = k;
            in_front = run;
            run += w;
            passed = run > target;
          }
        }
        sh.slice = found;
        sh.before = in_front;
      }
    }
    __syncthreads();
    before = sh.before;
    one_mx = st[sh.slice].mx;
    one_fac = factor(one_mx, rmx[cur], c);
    a = sh.slice * SLICE;
    e = min(V, a + SLICE);
  } else if (search && parts) {
    // the (CTA, warp) part of the row in which the running sum passes the target; its CTA searches it
    target = (double)unif[0] * row_total;
    int part = -1, last_pos = 0;
    double run = 0.0, last_before = 0.0;
    double* mine = sh.part[(n_rej - 1) & 1];
    for (int r = 0; r < csize && part < 0; ++r) {
      const double* from = csize > 1 ? cluster.map_shared_rank(mine, r) : mine;
      const double v = lane < WALK_WARPS ? from[lane] : 0.0, inc = warp_scan_d(v, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, v > 0.0 && run + inc > target), pos = __ballot_sync(0xffffffffu, v > 0.0);
      const int src = hit ? __ffs(hit) - 1 : pos ? 31 - __clz(pos) : -1;
      const double prev = run + __shfl_sync(0xffffffffu, inc - v, src < 0 ? 0 : src);
      if (src >= 0) {
        last_pos = r * WALK_WARPS + src;
        last_before = prev;
      }
      if (hit) part = last_pos;
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (part < 0) part = last_pos;
    before = last_before;
    if (part / WALK_WARPS == crank) {
      a = min(part * span, V);
      e = min(a + span, V);
    }
  }
  int next = greedy ? amax[cur] : 0;      // a row without weight: word 0
  if (a < e) {
    // four words per thread in index order, one round for a slice
    const float* x = my_logits + (size_t)cur * V;
    const float* dq = parts ? my_q + (size_t)cur * V : nullptr;
    double run = before;
    for (int a0 = a; a0 < e; a0 += 4 * WALK_THREADS) {
      const int i0 = a0 + 4 * tid;
      float xl[4], ql[4] = {};
      load4(x, i0, e, wide, -INFINITY, xl);
      if (parts) load4(dq, i0, e, wide, 0.0f, ql);
      double left[4], sum = 0.0;
      const int k = min(i0, V - 1) / SLICE;
      const float m = parts ? smx[k] : one_mx, f = parts ? fac[k] : 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float wt = weight_any(xl[w], m, c);
        double v;
        if (parts) {
          const float qq = fmaxf(ql[w], 0.0f);
          v = (double)take_out(after(__fmul_rn(wt, f), qq, n_rej - 1), qq);     // as summed in the pass behind the last rejection
        } else {
          v = (double)wt * one_fac;
          for (int r = 0; r < n_rej; ++r)
            if (rej[r] == i0 + w) v = 0.0;
        }
        left[w] = v;
        sum += v;
      }
      const double inc = warp_scan_d(sum, lane);
      if (lane == 31) sh.scan[warp] = inc;
      __syncthreads();
      const double wsum = lane < WALK_WARPS ? sh.scan[lane] : 0.0, winc = warp_scan_d(wsum, lane);
      double at = run + __shfl_sync(0xffffffffu, winc - wsum, warp) + (inc - sum);
      run += __shfl_sync(0xffffffffu, winc, 31);
      int pick = 0x7fffffff, my_last = -1;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        at += left[w];
        if (left[w] > 0.0) {
          my_last = i0 + w;
          if (at > target) pick = min(pick, i0 + w);
        }
      }
      if (pick != 0x7fffffff) atomicMin(&sh.pick, pick);
      if (my_last >= 0) atomicMax(&sh.last_pos, my_last);
      __syncthreads();
      if (sh.pick != 0x7fffffff) break;
    }
    if (sh.pick != 0x7fffffff) next = sh.pick;
    else if (sh.last_pos >= 0) next = sh.last_pos;
  }
  __syncthreads();
  if (search ? a < e : crank == 0) {
    for (int i = tid; i < width; i += WALK_THREADS) {
      my_path[i] = i < count ? path[i] : -1;
      my_tokens[i] = i < count - 1 ? tok[path[i + 1]] : i == count - 1 ? next : -1;
    }
    if (tid == 0) out_count[s] = count;
  }
  if (DENSE && csize > 1) cluster.sync();     // nobody's shared memory goes away while another CTA still reads it
}
}  // namespace

static size_t walk_smem_bytes(int max_nodes, int n_slices) {
  return ((sizeof(WalkSmem) + 15) & ~(size_t)15) + (size_t)n_slices * 8 + (size_t)max_nodes * (4 * 8 + 9 * 4) + 16;
}

// logits [T, V] fp32; tokens, parents [T] int32 (parents within the request, < 0 for its node 0); cu_q [S + 1]; uniform [T];
// temperature [S] or null (all greedy); draft_probs [T, V] fp32 or null. Out: tokens and path [S, max_depth + 1] (-1 behind the
// end), count [S]. stats: scratch of T x ceil(V / 1024) x 16 bytes. max_nodes: the most nodes of one request (at most 1,024);
// further nodes of a request are not looked at.
OSB_API int osb_verify_drafts(int* out_tokens, int* out_path, int* out_count, void* stats, const float* logits,
                              const int* tokens, const int* parents, const int* cu_q, const float* uniform,
                              const float* temperature, const float* draft_probs, int S, int T, int V, int max_nodes,
                              int max_depth, int* err, cudaStream_t stream) {
  if (S <= 0) return OSB_OK;
  if (V <= 0 || T < 0 || max_nodes < 0 || max_depth < 0) return OSB_ERR_BAD_SHAPE;
  const int n_slices = (V + SLICE - 1) / SLICE;
  if (max_nodes > 1024 || max_depth >= 1 << 30 || n_slices > 8192 || (long long)T * n_slices > 2147483647LL || (long long)S * MAX_CLUSTER > 2147483647LL)
    return OSB_ERR_TOO_LARGE;
  int sms = 0;
  int rc = osb_num_sms(&sms);
  if (rc) return rc;
  constexpr size_t ring = sizeof(float) * STAT_WARPS * STAT_STAGES * SLICE;
  static_assert(ring <= 48 * 1024, "no leave to ask for");
  if (T > 0) {
    const int items = T * n_slices, warps = STAT_WARPS * STAT_CTAS * sms, per = (items - 1) / warps + 1;
    const int used = (items - 1) / per + 1;
    rc = osb_launch(verify_stats_kernel, dim3((unsigned)((used + STAT_WARPS - 1) / STAT_WARPS)), dim3(STAT_THREADS), ring, stream, (SliceStat*)stats,
                    logits, cu_q, temperature, S, V, n_slices, items, per);
    if (rc) return rc;
  }
  const size_t smem = walk_smem_bytes(max_nodes, n_slices);
  auto walk = [&](auto k, int ready, int csize) -> int {
    if (ready) return ready;
    return osb_launch_cluster(k, dim3((unsigned)(S * csize)), dim3(WALK_THREADS), smem, stream, csize, out_tokens, out_path,
                              out_count, (const SliceStat*)stats, logits, tokens, parents, cu_q, uniform, temperature,
                              draft_probs, T, V, n_slices, max_nodes, max_depth, err);
  };
  if (draft_probs != nullptr && temperature != nullptr) {
    // a row of draft probabilities is summed by a cluster: a CTA per 16,384 words, and as many as let every request have its own at
    // once, one per SM. Both kernels with 1, 2, 4 and 8 CTAs, us: 8 requests of 7 nodes, 16,384 words 13.5, 14.1, 15.1, 16.7 (the
    // cluster costs more than the row), 50,000 words 19.1, 18.1, 18.4, 19.2, 152,064 words 42.6, 32.6, 28.0, 26.6
    int csize = 1;
    while (csize < MAX_CLUSTER && V >= 2 * csize * 16384 && (long long)S * 2 * csize <= sms) csize <<= 1;
    rc = walk(verify_walk_kernel<true>, osb_allow_smem<verify_walk_kernel<true>>(smem), csize);
  } else {
    rc = walk(verify_walk_kernel<false>, osb_allow_smem<verify_walk_kernel<false>>(smem), 1);
  }
  return rc ? rc : osb_last_error();
}
OSB_PACKED(osb_verify_drafts)
