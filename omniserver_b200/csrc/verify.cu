// Verification of drafted tokens against the target's probabilities from given random numbers.
//
// A request brings a tree of nodes (node 0: the last token it has, the others: drafted tokens, parents before children)
// and one fp32 row of logits per node. At node i with p = softmax(l_i / T) the children are tested in index order with
// r = p at first: child c with token x and random number u_c in [0, 1) is accepted if u_c q(x) < r(x), where q is the
// draft's distribution behind node i (a point mass at x if there is none: u_c < r(x)). A rejection leaves
// r <- max(r - q, 0) / sum (without q: r(x) <- 0, renormalised; r stays as it was if nothing is left). The walk ends where no
// child is accepted, and the next token is drawn there from r: the smallest index whose running sum passes u times the total,
// u being the root's random number (the root itself is never tested). Emitted tokens then follow the target's distribution
// whatever the draft was. Rows with T <= 0 are greedy: p is one at the first largest logit.
//
// Two kernels. `verify_stats_kernel` reads every logit once (what bounds the operator: T x V x 4 bytes): a CTA takes 4,096 words of
// one row in registers and leaves their maximum, its first place, and the sum of exp((l - maximum) / T). `verify_walk_kernel` then
// needs a few numbers per node to walk the tree; the draw scans one slice of 4,096 words. Only a rejection against a draft's
// distribution needs its whole row, and the row of logits, once more: then a cluster of CTAs walks the request together, each CTA
// summing its part of the row.
//
// Numbers. A word's weight is one fp32 value W = exp((l - m) / T), m the maximum of its slice: the difference and the product with
// log2(e) / T carry their rounding errors along, so that W is right to about 2 units in the last place. Sums, products with a
// slice's factor exp((m - m_row) / T), and comparisons are in 64 bits: with 150,000 words the place where a running sum passes a
// random number, and what is left of a row whose largest words were rejected, would not survive 32. A rejected word's weight is
// the same number that went into its slice's sum, so taking it out leaves the rest exactly.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {
constexpr int SLICE = 4096;            // words of a row that one CTA of the first kernel takes
constexpr int STAT_THREADS = 256;
constexpr int PER_THREAD = SLICE / STAT_THREADS;
constexpr int WALK_THREADS = 512;
constexpr int WALK_WARPS = WALK_THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr float MIN_TEMP = 1e-30f;     // smaller ones are taken as this: log2(e) / T has to stay finite
enum : int { ERR_TOKEN = 5 };

struct SliceStat {
  double sum;    // of the weights against the slice's own maximum
  float mx;      // the slice's largest logit (NaN counts as -inf)
  int arg;       // its first place in the row
};

// log2(e) / T as two floats
struct InvTemp {
  float hi, lo;
};
__device__ __forceinline__ InvTemp inv_temp(float t) {
  const double c = 1.4426950408889634074 / (double)fmaxf(t, MIN_TEMP);
  InvTemp r;
  r.hi = (float)c;
  r.lo = (float)(c - (double)r.hi);
  return r;
}

// exp((l - m) / T) for l <= m; 1 where they are equal, 0 for NaN and where m is -inf
__device__ __forceinline__ float weight(float l, float m, InvTemp c) {
  const float d = l - m;
  const float bb = d - l;                                  // the rounding error of the difference (two-sum)
  const float e = (l - (d - bb)) + (-m - bb);
  const float t = d * c.hi;
  if (!(t > -160.0f)) return 0.0f;                         // also NaN, and -inf anywhere
  const float lo = fmaf(d, c.hi, -t) + fmaf(d, c.lo, e * c.hi);
  const float w = exp2f(t);
  return fmaf(w, lo * 0.69314718f, w);
}
// the same with the cases the arithmetic above does not cover (an infinite maximum)
__device__ __forceinline__ float weight_any(float l, float m, InvTemp c) {
  if (m == INFINITY) return l == m ? 1.0f : 0.0f;
  return m == -INFINITY ? 0.0f : weight(l, m, c);
}
// a slice's factor exp((m - m_row) / T) in 64 bits
__device__ __forceinline__ double factor(float m, float m_row, double t) {
  if (m == m_row) return m == -INFINITY ? 0.0 : 1.0;
  if (m == -INFINITY || m_row == INFINITY) return 0.0;
  return exp(((double)m - (double)m_row) / t);
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

__device__ __forceinline__ void max_combine(float& bv, int& bi, float v, int i) {
  if (v > bv || (v == bv && i < bi)) {
    bv = v;
    bi = i;
  }
}

// One CTA: one slice of one row. Rows behind the last request are skipped.
__global__ void __launch_bounds__(STAT_THREADS) verify_stats_kernel(SliceStat* __restrict__ stats,
                                                                    const float* __restrict__ logits,
                                                                    const int* __restrict__ cu_q,
                                                                    const float* __restrict__ temperature, int S, int V,
                                                                    int n_slices) {
  __shared__ float smx[STAT_THREADS / 32];
  __shared__ int sarg[STAT_THREADS / 32];
  __shared__ double ssum[STAT_THREADS / 32];
  pdl_wait();
  const int row = blockIdx.x / n_slices, sl = blockIdx.x - row * n_slices;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* x = logits + (size_t)row * V;
  const int lo = sl * SLICE, hi = min(V, lo + SLICE);
  // thread t holds words lo + 4 (t + 256 k) .. + 3 (16-byte loads) or lo + t + 256 k
  float v[PER_THREAD];
  const bool vec = ((V & 3) == 0) && (((uintptr_t)logits & 15) == 0);
  if (vec) {
#pragma unroll
    for (int k = 0; k < PER_THREAD / 4; ++k) {
      const int i = lo + 4 * (tid + STAT_THREADS * k);
      float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (i < hi) f = __ldcs(reinterpret_cast<const float4*>(x + i));
      v[4 * k] = f.x;
      v[4 * k + 1] = f.y;
      v[4 * k + 2] = f.z;
      v[4 * k + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < PER_THREAD; ++k) {
      const int i = lo + tid + STAT_THREADS * k;
      v[k] = i < hi ? __ldcs(x + i) : -INFINITY;
    }
  }
  // the row's request: as many as end at or before it
  int req = 0;
  for (int b = 0; b < S; b += STAT_THREADS) req += __syncthreads_count(b + tid < S && cu_q[b + tid + 1] <= row);
  if (req >= S) return;
  const float temp = temperature != nullptr ? temperature[req] : 0.0f;

  float bv = -INFINITY;
  int bi = 0x7fffffff;
#pragma unroll
  for (int k = 0; k < PER_THREAD; ++k) {
    const int i = vec ? lo + 4 * (tid + STAT_THREADS * (k >> 2)) + (k & 3) : lo + tid + STAT_THREADS * k;
    if (v[k] != v[k]) v[k] = -INFINITY;
    if (v[k] > bv) {     // places ascend within a thread
      bv = v[k];
      bi = i;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    max_combine(bv, bi, ov, oi);
  }
  if (lane == 0) {
    smx[warp] = bv;
    sarg[warp] = bi;
  }
  __syncthreads();
  bv = smx[0];
  bi = sarg[0];
#pragma unroll
  for (int w = 1; w < STAT_THREADS / 32; ++w) max_combine(bv, bi, smx[w], sarg[w]);
  double sum = 0.0;
  if (temp > 0.0f) {
    const InvTemp c = inv_temp(temp);
    if (bv > -INFINITY && bv < INFINITY) {
#pragma unroll
      for (int k = 0; k < PER_THREAD; ++k) sum += (double)weight(v[k], bv, c);
    } else {
#pragma unroll
      for (int k = 0; k < PER_THREAD; ++k) sum += (double)weight_any(v[k], bv, c);
    }
    sum = warp_sum_d(sum);
    if (lane == 0) ssum[warp] = sum;
    __syncthreads();
    sum = ssum[0];
#pragma unroll
    for (int w = 1; w < STAT_THREADS / 32; ++w) sum += ssum[w];
  }
  if (tid == 0) stats[blockIdx.x] = SliceStat{sum, bv, bi == 0x7fffffff ? lo : bi};
}

struct WalkSmem {             // the fixed part; per-node and per-slice arrays follow
  double part[2][WALK_WARPS]; // the CTA's sums of its parts of a row, warp by warp: after the last rejection, and the one in hand
  double scan[WALK_WARPS];
  int pick;
  int last_pos;
};

// One request: one CTA, or (draft_probs) one cluster, every CTA of which walks alike; see the top of the file.
__global__ void __launch_bounds__(WALK_THREADS) verify_walk_kernel(
    int* __restrict__ out_tokens, int* __restrict__ out_path, int* __restrict__ out_count,
    const SliceStat* __restrict__ stats, const float* __restrict__ logits, const int* __restrict__ tokens,
    const int* __restrict__ parents, const int* __restrict__ cu_q, const float* __restrict__ uniform,
    const float* __restrict__ temperature, const float* __restrict__ draft_probs, int V, int n_slices, int max_nodes,
    int max_depth, int* __restrict__ err) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  WalkSmem& sh = *reinterpret_cast<WalkSmem*>(smem_raw);
  double* fac = reinterpret_cast<double*>(smem_raw + ((sizeof(WalkSmem) + 15) & ~(size_t)15));   // [n_slices] of the node in hand
  double* ztot = fac + n_slices;                   // [max_nodes] a node's total weight
  double* wtok = ztot + max_nodes;                 // [max_nodes] a node's token's weight behind its parent; < 0: no such word
  double* rej_w = wtok + max_nodes;                // [max_nodes] what rejections at the node in hand took (or 1 / sum, with q)
  float* smx = reinterpret_cast<float*>(rej_w + max_nodes);   // [n_slices]
  float* rmx = smx + n_slices;                     // [max_nodes] a node's largest logit
  float* qtok = rmx + max_nodes;                   // [max_nodes] q of a node's token
  int* amax = reinterpret_cast<int*>(qtok + max_nodes);
  int* tok = amax + max_nodes;
  int* par = tok + max_nodes;
  int* rej = par + max_nodes;                      // [max_nodes] rejected tokens at the node in hand
  int* path = rej + max_nodes;                     // [max_nodes] the nodes of the walk

  cg::cluster_group cluster = cg::this_cluster();
  const int csize = (int)cluster.num_blocks(), crank = (int)cluster.block_rank();
  const int s = blockIdx.x / csize;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int q0 = cu_q[s];
  const int n = min(cu_q[s + 1] - q0, max_nodes);
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
  const float tempf = temperature != nullptr ? temperature[s] : 0.0f;
  const bool greedy = !(tempf > 0.0f);
  const double temp = (double)fmaxf(tempf, MIN_TEMP);
  const InvTemp c = inv_temp(greedy ? 1.0f : tempf);
  for (int i = tid; i < n; i += WALK_THREADS) {
    const int t = tokens[q0 + i];
    tok[i] = t;
    par[i] = parents[q0 + i];
    if (i > 0 && (t < 0 || t >= V) && crank == 0) atomicExch(err, ERR_TOKEN);
  }
  // a node's maximum, its first place, and its total weight
  for (int i = warp; i < n; i += WALK_WARPS) {
    const SliceStat* st = stats + (size_t)(q0 + i) * n_slices;
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    for (int k = lane; k < n_slices; k += 32) max_combine(bv, bi, st[k].mx, st[k].arg);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      max_combine(bv, bi, ov, oi);
    }
    double z = 0.0;
    if (!greedy)
      for (int k = lane; k < n_slices; k += 32) z += st[k].sum * factor(st[k].mx, bv, temp);
    z = warp_sum_d(z);
    if (lane == 0) {
      rmx[i] = bv;
      amax[i] = bi == 0x7fffffff ? 0 : bi;
      ztot[i] = z;
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += WALK_THREADS) {
    const int p = par[i], t = tok[i];
    double w = -1.0;
    float q = 1.0f;
    if (p >= 0 && p < i && t >= 0 && t < V && !greedy) {
      const size_t row = (size_t)(q0 + p);
      const float m = stats[row * n_slices + t / SLICE].mx;
      w = (double)weight_any(logits[row * V + t], m, c) * factor(m, rmx[p], temp);
      if (draft_probs != nullptr) q = draft_probs[row * V + t];
    }
    wtok[i] = w;
    qtok[i] = q;
  }
  __syncthreads();

  int cur = 0, count = 1, n_rej = 0, last = 0;
  double removed = 0.0, row_total = 0.0;     // weight rejected without q / what the last pass over a row summed
  bool have_parts = false;
  if (tid == 0) path[0] = 0;
  // the parts of a row that this CTA's warps take in a pass: contiguous, in order of (CTA, warp)
  const int span = ((V + csize * WALK_WARPS - 1) / (csize * WALK_WARPS) + 3) & ~3;
  auto residual = [&](double w, double q) -> double {   // the weight of a word after this node's rejections, q its draft probability
    double r = w / ztot[cur];
    for (int k = 0; k < n_rej; ++k) r = fmax(r - q, 0.0) * rej_w[k];
    return r;
  };
  auto slice_numbers = [&]() {                          // maxima and factors of the slices of the node in hand
    const SliceStat* st = stats + (size_t)(q0 + cur) * n_slices;
    for (int k = tid; k < n_slices; k += WALK_THREADS) {
      smx[k] = st[k].mx;
      fac[k] = factor(st[k].mx, rmx[cur], temp);
    }
    __syncthreads();
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
    bool yes;
    if (tok[j] < 0 || tok[j] >= V) continue;     // no word: it cannot be accepted, and takes nothing away
    if (greedy) {
      yes = tok[j] == amax[cur];
      if (!yes) continue;
    } else if (draft_probs == nullptr) {
      double w = wtok[j];
      for (int k = 0; k < n_rej; ++k)
        if (rej[k] == tok[j]) w = 0.0;           // rejected before: nothing of it is left
      yes = (double)uniform[q0 + j] * (ztot[cur] - removed) < w;
      if (!yes && w > 0.0 && ztot[cur] - removed - w > 0.0) {
        __syncthreads();                          // everyone has read the list
        if (tid == 0) {
          rej[n_rej] = tok[j];
          rej_w[n_rej] = w;
        }
        ++n_rej;
        removed += w;
        __syncthreads();
      }
    } else {
      const double q = fmax((double)qtok[j], 0.0);
      yes = ztot[cur] > 0.0 && (double)uniform[q0 + j] * q < residual(wtok[j], q);
      if (!yes && ztot[cur] > 0.0) {
        // what is left of the row: its sum, warp by warp over contiguous parts
        slice_numbers();
        const float* x = logits + (size_t)(q0 + cur) * V;
        const float* dq = draft_probs + (size_t)(q0 + cur) * V;
        const int a = min((crank * WALK_WARPS + warp) * span, V), e = min(a + span, V);
        double sum = 0.0;
        for (int i0 = a; i0 < e; i0 += 128) {
          float xl[4], ql[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int i = i0 + 32 * u + lane;
            xl[u] = i < e ? x[i] : -INFINITY;
            ql[u] = i < e ? dq[i] : 0.0f;
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int i = min(i0 + 32 * u + lane, V - 1);
            const int k = i / SLICE;
            const double qq = fmax((double)ql[u], 0.0);
            sum += fmax(residual((double)weight_any(xl[u], smx[k], c) * fac[k], qq) - qq, 0.0);
          }
        }
        sum = warp_sum_d(sum);
        if (csize > 1) cluster.sync(); else __syncthreads();    // nobody still reads the parts of an earlier pass
        if (lane == 0) sh.part[n_rej & 1][warp] = sum;
        if (csize > 1) cluster.sync(); else __syncthreads();
        double total = 0.0;
        for (int r = 0; r < csize; ++r) {
          const double* p = csize > 1 ? cluster.map_shared_rank(sh.part[n_rej & 1], r) : sh.part[n_rej & 1];
          for (int w = 0; w < WALK_WARPS; ++w) total += p[w];
        }
        if (total > 0.0) {
          if (tid == 0) rej_w[n_rej] = 1.0 / total;
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
      removed = 0.0;
      have_parts = false;
    }
  }

  // the draw at node cur: a range [a, e) of words, the running sum in front of it and the target
  double target, before = 0.0;
  int a = 0, e = 0, next = amax[cur];
  if (tid == 0) {
    sh.pick = 0x7fffffff;
    sh.last_pos = -1;
  }
  bool search = false;
  if (!greedy && ztot[cur] > 0.0) {
    search = true;
    if (!have_parts) {
      // one CTA; slice by slice, less what was rejected
      if (crank == 0) {
        slice_numbers();
        target = (double)uniform[q0] * (ztot[cur] - removed);
        const SliceStat* st = stats + (size_t)(q0 + cur) * n_slices;
        int found = -1, last_pos = -1;
        double last_before = 0.0;
        for (int b = 0; b < n_slices && found < 0; b += 32) {
          const int k = b + lane;
          double v = 0.0;
          if (k < n_slices) {
            v = st[k].sum * fac[k];
            for (int r = 0; r < n_rej; ++r)
              if (rej[r] / SLICE == k) v -= rej_w[r];
            v = fmax(v, 0.0);
          }
          const double inc = warp_scan_d(v, lane);
          const unsigned hit = __ballot_sync(0xffffffffu, v > 0.0 && before + inc > target);
          const unsigned pos = __ballot_sync(0xffffffffu, v > 0.0);
          const int src = hit ? __ffs(hit) - 1 : (pos ? 31 - __clz(pos) : 0);
          const double prev = before + __shfl_sync(0xffffffffu, inc - v, src);
          if (hit) {
            found = b + src;
            last_before = prev;
          } else if (pos) {
            last_pos = b + src;
            last_before = prev;
          }
          before += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (found < 0) found = last_pos;       // the target rounded up to the total: the last slice that has weight
        if (found < 0) found = 0;
        before = last_before;
        a = found * SLICE;
        e = min(V, a + SLICE);
      }
    } else {
      // the (CTA, warp) part of the row in which the running sum passes the target; its CTA searches it
      target = (double)uniform[q0] * row_total;
      int part = -1, last_pos = 0;
      double run = 0.0, last_before = 0.0;
      for (int r = 0; r < csize && part < 0; ++r) {
        const double* p = csize > 1 ? cluster.map_shared_rank(sh.part[(n_rej - 1) & 1], r) : sh.part[(n_rej - 1) & 1];
        for (int w = 0; w < WALK_WARPS; ++w) {
          const double v = p[w];
          if (v > 0.0) {
            last_pos = r * WALK_WARPS + w;
            last_before = run;
            if (run + v > target) {
              part = last_pos;
              break;
            }
          }
          run += v;
        }
      }
      if (part < 0) part = last_pos;
      before = last_before;
      if (part / WALK_WARPS == crank) {
        a = min(part * span, V);
        e = min(a + span, V);
        slice_numbers();
        --n_rej;       // below, as in the pass: the last rejection's subtraction without its 1 / sum
      }
    }
  }
  __syncthreads();
  if (search && a < e) {
    // contiguous words per thread, so that the running sum goes in index order
    const float* x = logits + (size_t)(q0 + cur) * V;
    const float* dq = have_parts ? draft_probs + (size_t)(q0 + cur) * V : nullptr;
    const int per = (e - a + WALK_THREADS - 1) / WALK_THREADS;
    const int b0 = min(a + tid * per, e), b1 = min(b0 + per, e);
    auto left = [&](int i) -> double {
      const int k = i / SLICE;
      const double w = (double)weight_any(x[i], smx[k], c) * fac[k];
      if (have_parts) {
        const double qq = fmax((double)dq[i], 0.0);
        return fmax(residual(w, qq) - qq, 0.0);
      }
      for (int r = 0; r < n_rej; ++r)
        if (rej[r] == i) return 0.0;
      return w;
    };
    double sum = 0.0;
    for (int i = b0; i < b1; ++i) sum += left(i);
    const double inc = warp_scan_d(sum, lane);
    if (lane == 31) sh.scan[warp] = inc;
    __syncthreads();
    double run = before;
    for (int w = 0; w < warp; ++w) run += sh.scan[w];
    run += inc - sum;
    int mine = 0x7fffffff, my_last = -1;
    for (int i = b0; i < b1; ++i) {
      const double v = left(i);
      run += v;
      if (v > 0.0) {
        my_last = i;
        if (run > target) {
          mine = i;
          break;
        }
      }
    }
    if (mine != 0x7fffffff) atomicMin(&sh.pick, mine);
    if (my_last >= 0) atomicMax(&sh.last_pos, my_last);
    __syncthreads();
    next = sh.pick != 0x7fffffff ? sh.pick : (sh.last_pos >= 0 ? sh.last_pos : amax[cur]);
  }
  const bool writer = search ? a < e : crank == 0;
  if (writer) {
    for (int i = tid; i < width; i += WALK_THREADS) {
      my_path[i] = i < count ? path[i] : -1;
      my_tokens[i] = i < count - 1 ? tok[path[i + 1]] : i == count - 1 ? next : -1;
    }
    if (tid == 0) out_count[s] = count;
  }
  if (csize > 1) cluster.sync();     // nobody's shared memory goes away while another CTA still reads it
}
}  // namespace

static size_t walk_smem_bytes(int max_nodes, int n_slices) {
  return ((sizeof(WalkSmem) + 15) & ~(size_t)15) + (size_t)n_slices * 12 + (size_t)max_nodes * (3 * 8 + 7 * 4) + 16;
}

// logits [T, V] fp32; tokens, parents [T] int32 (parents within the request, < 0 for its node 0); cu_q [S + 1]; uniform [T];
// temperature [S] or null (all greedy); draft_probs [T, V] fp32 or null. Out: tokens and path [S, max_depth + 1] (-1 behind the
// end), count [S]. stats: scratch of T x ceil(V / 4096) x 16 bytes. max_nodes: the most nodes of one request (at most 1,024);
// further nodes of a request are not looked at.
OSB_API int osb_verify_drafts(int* out_tokens, int* out_path, int* out_count, void* stats, const float* logits,
                              const int* tokens, const int* parents, const int* cu_q, const float* uniform,
                              const float* temperature, const float* draft_probs, int S, int T, int V, int max_nodes,
                              int max_depth, int* err, cudaStream_t stream) {
  if (S <= 0) return OSB_OK;
  if (V <= 0 || T < 0 || max_nodes < 0 || max_depth < 0) return OSB_ERR_BAD_SHAPE;
  const int n_slices = (V + SLICE - 1) / SLICE;
  if (max_nodes > 1024 || n_slices > 4096 || (long long)T * n_slices > 2147483647LL || (long long)S * MAX_CLUSTER > 2147483647LL)
    return OSB_ERR_TOO_LARGE;
  if (T > 0) {
    const int rc = osb_launch(verify_stats_kernel, dim3((unsigned)(T * n_slices)), dim3(STAT_THREADS), 0, stream,
                              (SliceStat*)stats, logits, cu_q, temperature, S, V, n_slices);
    if (rc) return rc;
  }
  const size_t smem = walk_smem_bytes(max_nodes, n_slices);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(verify_walk_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
  }
  // a row of draft probabilities is summed by a cluster: 8 CTAs, or one where a row is short
  const int csize = draft_probs != nullptr && temperature != nullptr && V > 8192 ? MAX_CLUSTER : 1;
  const int rc = osb_launch_cluster(verify_walk_kernel, dim3((unsigned)(S * csize)), dim3(WALK_THREADS), smem, stream, csize,
                                    out_tokens, out_path, out_count, (const SliceStat*)stats, logits, tokens, parents, cu_q,
                                    uniform, temperature, draft_probs, V, n_slices, max_nodes, max_depth, err);
  return rc ? rc : osb_last_error();
}
