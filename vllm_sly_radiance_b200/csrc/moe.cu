// Mixture of experts around the experts' products (linear_fused.cu): router, sorting plan, rows by expert, weighted sum.
//
//   route    s = softmax(l) or sigmoid(l);  c = s + bias;  group value = the two best c of a group added up (bias), or its
//            best c;  the best `top_groups` groups;  in them the best k of c;  w = s (/ their sum) * scale
//   plan     rows = the (token, slot) pairs of this rank's experts, those of one expert side by side, in the pairs' order
//   gather   row r = the activations of its token
//   combine  out[t] = sum_j w[t, j] rows[pos[t, j]] (+ sigmoid(gate[t]) shared[t])
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "refuse.h"

namespace rad {
namespace moe {

constexpr int MAX_E = 1024;
constexpr unsigned FULL = 0xffffffffu;

DEVI float to_f(float x) { return x; }
DEVI float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
DEVI float to_f(__half x) { return __half2float(x); }

// ---------------------------------------------------------------------------------------------
// route: one warp a token.  The lanes of a group hold its experts in order, V neighbours each, so that a lane's own best two
// and log2(lanes) exchanges give every group's value at once, and the lowest lane among equals has the lowest index.
// Values become whole numbers of the same order (0: no candidate, 1: NaN, then -inf and up), whose warp maximum is one
// instruction.  Without a bias the logits themselves are ranked, which is the scores' order.  With a bias the scores enter the
// order: they are computed in 32 bits, and once more in 64 for the few tokens (about one in 500) where two candidates, or two
// groups, lie so near that the rounding could have turned them.
// ---------------------------------------------------------------------------------------------
// Bound by one warp's chain of instructions (device times, graphs of 10 calls): 3.2 us for one token, 11 us for 8192 of 256 experts,
// 22 us with sigmoid scores, groups and a bias (their bytes take 1.4 us).
struct RouteArgs {
  const void* logits;
  const float* bias;
  int64_t* ids;
  float* w;
  int64_t ld;
  int T, E, k, groups, top_groups, gsize, lanes;           // lanes of a group
  bool sigmoid, renorm, vec;
  float scale;
};

DEVI uint32_t key_of(float c) {
  if (c != c) return 1u;
  const uint32_t b = __float_as_uint(c + 0.f);             // -0 as +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
DEVI uint64_t key_of(double c) {
  if (c != c) return 1ull;
  const uint64_t b = (uint64_t)__double_as_longlong(c + 0.0);
  return b >> 63 ? ~b : b | (1ull << 63);
}
DEVI uint32_t warp_max_key(uint32_t v) { return __reduce_max_sync(FULL, v); }
DEVI uint64_t warp_max_key(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(FULL, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(FULL, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (uint64_t)hi << 32 | lo;
}
DEVI float value_of(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }       // of a key above 1

DEVI float exp_of(float x) { return expf(x); }
DEVI double exp_of(double x) { return exp(x); }

// A score
template <typename F> DEVI F score_of(const RouteArgs& p, float x, float top, F total) {
  if (p.sigmoid) return F(1) / (F(1) + exp_of(-(F)x));
  const F s = exp_of((F)x - (F)top);
  return total > 0 ? s / total : total;
}

// Lanes' chosen logits (-inf without one) -> their scores but for a common factor, of which no weight is left once they are divided by
// their sum: relative to the largest where the scores themselves may be below what 32 bits hold
DEVI float ratio_of(bool sigmoid, float x) {
  if (sigmoid && !__any_sync(FULL, x < -80.f && x > -INFINITY)) return 1.f / (1.f + expf(-x));
  const float a = sigmoid ? fminf(x, 0.f) : x;             // sigmoid(x) = e^min(x, 0) / (1 + e^-|x|)
  float m = warp_max(a);
  if (m == -INFINITY) m = 0.f;                             // masked throughout: scores of zero
  const float d = a - m, e = expf(d);
  if (!sigmoid) return e;
  // what the difference rounded off, up to 2^-18 of e^d where the logits lie far apart
  const float t = d - a, r = d > -128.f ? (a - (d - t)) - (m + t) : 0.f;
  return fmaf(e, r, e) / (1.f + expf(-fabsf(x)));
}

// Best two of a lane's candidates -> of its group's
template <typename F> DEVI void best_two(F& b1, F& b2, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    const F o1 = __shfl_xor_sync(FULL, b1, o), o2 = __shfl_xor_sync(FULL, b2, o);
    const F lo = min(o1, b1);
    b1 = max(o1, b1);
    b2 = max(lo, max(o2, b2));
  }
}

// The choice in 64 bits, with a bias -> the expert of lane j < k.  A call of its own, so that its registers do not cost the ordinary
// path its warps.
template <typename L, int V>
__device__ __noinline__ int choose_wide(const RouteArgs& p, const L* row, int e0, int n, float top, int lane) {
  double c[V], total = 1.0;
  if (!p.sigmoid) {
    total = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) total += exp((double)to_f(row[e0 + i]) - (double)top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
  }
  double b1 = -INFINITY, b2 = -INFINITY;
  // in step for all lanes: eight independent chains of double operations, where a loop waited for one after the other
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = score_of<double>(p, i < n ? to_f(row[e0 + i]) : 0.f, top, total);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) {
      c[i] += (double)p.bias[e0 + i];
      const double x = fmax(c[i], -INFINITY), lo = fmin(x, b1);      // a NaN adds nothing to the group's value
      b1 = fmax(x, b1);
      b2 = fmax(lo, b2);
    }
  if (p.groups > 1) {
    best_two(b1, b2, p.lanes);
    const double value = b1 + b2;
    const uint64_t key = key_of(value);
    const int mine = lane / p.lanes;
    int rank = 0;
#pragma unroll 1
    for (int g = 0; g < p.groups; ++g) {
      const uint64_t o = key_of(__shfl_sync(FULL, value, g * p.lanes));
      rank += o > key || (o == key && g < mine);
    }
    if (rank >= p.top_groups) n = 0;
  }
  uint64_t keys[V];
#pragma unroll
  for (int i = 0; i < V; ++i) keys[i] = i < n ? key_of(c[i]) : 0;
  int expert = 0;
#pragma unroll 1
  for (int j = 0; j < p.k; ++j) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (keys[i] > best) best = keys[i], at = i;
    const uint64_t m = warp_max_key(best);
    const int w = __ffs(__ballot_sync(FULL, best == m)) - 1, ew = __shfl_sync(FULL, e0 + at, w);
    if (lane == j) expert = ew;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane == w && i == at) keys[i] = 0;
  }
  return expert;
}

// Lane j < k ends with the j-th expert.  False: 32 bits could not tell the order.  total: of the softmax, where it is needed
template <int V, bool BIAS>
DEVI bool choose(const RouteArgs& p, const float (&l)[V], int e0, int n, float top, int lane, int& expert, float& total) {
  // How far rounding can move two candidates' difference, u = 2^-24, relative to 1 + |c|.  A sigmoid is off by at most 2 u (exp 2 u
  // of e, sum, quotient), two by 4 u.  A softmax's two are off by at most (V + 17) u of their sum, which is at most 1: exp 2 u and
  // its argument 0.4 u each; the total V + 4 additions in a row, its terms' exp 2 u and their arguments ln E < 7 u; the quotient u.
  // The bias adds u of each c.  Either with a margin.
  const float tol = p.sigmoid ? 8.f / (1 << 24) : (V + 24.f) / (1 << 24);
  total = 0.f;
  if (!p.sigmoid && (BIAS || !p.renorm)) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) total += expf(l[i] - top);
    total = warp_sum(total);
  }
  bool clear = true;
  float c[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    c[i] = 0.f;
    if (i < n) c[i] = BIAS ? score_of<float>(p, l[i], top, total) + p.bias[e0 + i] : l[i];
  }
  if (p.groups > 1) {
    float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) {
        const float x = fmaxf(c[i], -INFINITY), lo = fminf(x, b1);   // a NaN adds nothing to the group's value
        b1 = fmaxf(x, b1);
        b2 = fmaxf(lo, b2);
      }
    best_two(b1, b2, p.lanes);
    const float value = BIAS ? b1 + b2 : b1;
    const uint32_t key = key_of(value);
    const int mine = lane / p.lanes;
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const float other = __shfl_sync(FULL, value, g * p.lanes);
      const uint32_t ko = key_of(other);
      rank += ko > key || (ko == key && g < mine);
      // two scores more, and the rounding of each expert's c, which may cancel in the value; the other group asks this by its own
      if (BIAS && g != mine && mine < p.groups) clear &= fabsf(value - other) > tol * (2.f + fabsf(b1) + fabsf(b2));
    }
    if (rank >= p.top_groups) n = 0;
  }
  uint32_t key[V], best = 0;
  int at = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    key[i] = i < n ? key_of(c[i]) : 0u;
    if (key[i] > best) best = key[i], at = i;
  }
  float before = 0.f;
  for (int j = 0; j < p.k + (BIAS ? 1 : 0); ++j) {
    const uint32_t m = warp_max_key(best);
    if (m == 0) break;                                     // the candidate behind the last one does not exist
    const int w = __ffs(__ballot_sync(FULL, best == m)) - 1, ew = __shfl_sync(FULL, e0 + at, w);
    if (BIAS) {
      const float cw = m > 1 ? value_of(m) : NAN;
      if (j > 0) clear &= before - cw > tol * (1.f + fabsf(cw));
      before = cw;
    }
    if (lane == j && j < p.k) expert = ew;
    if (lane == w) {
      best = 0;
      const int gone = at;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (i == gone) key[i] = 0;
        if (key[i] > best) best = key[i], at = i;
      }
    }
  }
  return __all_sync(FULL, clear);
}

template <typename L, int V, bool BIAS>
__global__ void __launch_bounds__(256, V <= 8 ? 4 : V <= 32 ? 2 : 1) route_kernel(const __grid_constant__ RouteArgs p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x % 32, t = blockIdx.x * 8 + threadIdx.x / 32;
  if (t >= p.T) return;
  const L* row = static_cast<const L*>(p.logits) + (int64_t)t * p.ld;
  const int v = (p.gsize + p.lanes - 1) / p.lanes, group = lane / p.lanes, first = lane % p.lanes * v;
  const int n = group < p.groups ? max(0, min(v, p.gsize - first)) : 0, e0 = group * p.gsize + first;
  float l[V];
  if (p.vec && V * sizeof(L) >= 16) {                      // a lane's experts are V and start on 16 bytes
    if constexpr (V * sizeof(L) >= 16) {
      constexpr int Q = 16 / sizeof(L);
#pragma unroll
      for (int i = 0; i < V; i += Q) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (i < n) q = *reinterpret_cast<const uint4*>(row + e0 + i);
        const L* x = reinterpret_cast<const L*>(&q);
#pragma unroll
        for (int j = 0; j < Q; ++j) l[i + j] = to_f(x[j]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = i < n ? to_f(row[e0 + i]) : 0.f;
  }
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) top = fmaxf(top, l[i]), nan |= l[i] != l[i];
  top = warp_max(top);
  nan = __any_sync(FULL, nan || (!p.sigmoid && top == INFINITY));
  if (top == -INFINITY) top = 0.f;                         // every expert masked: scores of zero
  int expert = 0;
  float total, s = 0.f;
  const bool clear = choose<V, BIAS>(p, l, e0, n, top, lane, expert, total);
  if (BIAS && !clear) expert = choose_wide<L, V>(p, row, e0, n, top, lane);
  if (p.renorm) {
    s = ratio_of(p.sigmoid, lane < p.k ? to_f(row[expert]) : -INFINITY);
    const float sum = warp_sum(s);
    s = sum > 0.f ? s / sum : 0.f;
  } else if (lane < p.k) {
    s = score_of<float>(p, to_f(row[expert]), top, total);
  }
  if (lane < p.k) {
    p.ids[(int64_t)t * p.k + lane] = expert;
    p.w[(int64_t)t * p.k + lane] = nan ? NAN : s * p.scale;
  }
}

// ---------------------------------------------------------------------------------------------
// plan: one cluster.  Every warp owns neighbouring pairs; it counts them by expert, the counts are added up over warps and
// CTAs (distributed shared memory), and a second pass over the pairs hands out the rows.  Equal experts of 32 pairs find one
// another by a vote per bit of their number (a warp match instead took 12.2 us for 4096 pairs, this 8.7), so nothing is atomic
// and the rows come in the pairs' order.
// ---------------------------------------------------------------------------------------------
// Bound by the same kind of chain: 3.5 us for 512 pairs (one CTA), 18 us for 131072 (16 CTAs, votes and shared memory; 16 where half
// of the experts are another rank's).
struct PlanArgs {
  const void* ids;
  int R, k, E, first, seg, warps, bits;                    // pairs, experts of this rank, pairs of a warp, warps that have some
  bool wide;                                               // ids of 64 bits
  int* order;
  int* pos;
  int* counts;
  int* starts;
  int* items;                                              // (expert, first row, rows) per tile of `tile` rows
  int tile, max_items;
};
constexpr int PLAN_WARPS = 32, PLAN_CTAS = 16, PLAN_AHEAD = 8;

DEVI int plan_expert(const PlanArgs& p, int f, int end) {
  if (f >= end) return -1;
  const int64_t e = (p.wide ? static_cast<const int64_t*>(p.ids)[f] : (int64_t) static_cast<const int*>(p.ids)[f]) - p.first;
  return e >= 0 && e < p.E ? (int)e : -1;
}

// lanes with the same expert; those without one (-1) are in nobody's set but their own
DEVI unsigned same_expert(int e, int bits) {
  unsigned same = __ballot_sync(FULL, e >= 0);
  for (int b = 0; b < bits; ++b) {
    const unsigned set = __ballot_sync(FULL, e >> b & 1);
    same &= e >> b & 1 ? set : ~set;
  }
  return same;
}

// exclusive sums of v over the block's threads (1024); total: of all
DEVI int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(FULL, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int s = warp_sums[lane], before = lane < warp ? s : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(FULL, s, o);
    before += __shfl_xor_sync(FULL, before, o);
  }
  total = s;
  __syncthreads();
  return x - v + before;
}

__global__ void __launch_bounds__(1024) plan_kernel(const __grid_constant__ PlanArgs p) {
  extern __shared__ int smem[];
  int* cnt = smem;                                         // [warps][E]
  int* tot = cnt + p.warps * p.E;                          // [E] of this CTA
  int* base = tot + p.E;                                   // [E] first row of this CTA's pairs
  __shared__ int warp_sums[32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t rank = cluster_ctarank();
  const int ctas = gridDim.x;
  pdl_trigger();
  for (int i = threadIdx.x; i < p.warps * p.E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  pdl_wait();
  int* mine = cnt + warp * p.E;
  const int64_t f0 = ((int64_t)rank * p.warps + warp) * p.seg;
  const int lo = warp < p.warps ? (int)min(f0, (int64_t)p.R) : p.R, hi = warp < p.warps ? (int)min(f0 + p.seg, (int64_t)p.R) : p.R;
  for (int f = lo; f < hi; f += 32 * PLAN_AHEAD) {
    int x[PLAN_AHEAD];
#pragma unroll
    for (int u = 0; u < PLAN_AHEAD; ++u) x[u] = plan_expert(p, f + 32 * u + lane, hi);
#pragma unroll
    for (int u = 0; u < PLAN_AHEAD; ++u) {
      if (f + 32 * u >= hi) break;
      const unsigned same = same_expert(x[u], p.bits);
      if (x[u] >= 0 && lane == __ffs(same) - 1) mine[x[u]] += __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
  const int e = threadIdx.x;
  int sum = 0;
  if (e < p.E) {
#pragma unroll 8
    for (int w = 0; w < p.warps; ++w) {
      const int n = cnt[w * p.E + e];
      cnt[w * p.E + e] = sum;
      sum += n;
    }
    tot[e] = sum;
  }
  int all = sum, before = 0;
  if (ctas > 1) {
    cluster_sync();
    if (e < p.E) {
      all = 0;
      const uint32_t at = smem_u32(tot + e);
      for (int c = 0; c < ctas; ++c) {
        int n;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(n) : "r"(mapa_shared(at, c)));
        if (c < (int)rank) before += n;
        all += n;
      }
    }
    cluster_arrive();                                      // the others may leave once this CTA has read their counts
  }
  int rows;
  const int start = block_scan(all, warp_sums, rows);
  if (e < p.E) {
    base[e] = start + before;
    if (rank == 0) p.counts[e] = all, p.starts[e] = start;
  }
  if (rank == 0 && threadIdx.x == 0) p.starts[p.E] = rows;
  if (p.items && rank == 0) {
    int tiles;
    const int n = e < p.E ? (all + p.tile - 1) / p.tile : 0, i0 = block_scan(n, warp_sums, tiles);
    for (int i = 0; i < n && i0 + i < p.max_items; ++i) {
      int* q = p.items + 3 * (int64_t)(i0 + i);
      q[0] = e;
      q[1] = start + i * p.tile;
      q[2] = min(p.tile, all - i * p.tile);
    }
    for (int i = tiles + threadIdx.x; i < p.max_items; i += blockDim.x)
      p.items[3 * (int64_t)i] = p.items[3 * (int64_t)i + 1] = p.items[3 * (int64_t)i + 2] = 0;
  }
  __syncthreads();
  for (int f = lo; f < hi; f += 32 * PLAN_AHEAD) {
    int x[PLAN_AHEAD];
#pragma unroll
    for (int u = 0; u < PLAN_AHEAD; ++u) x[u] = plan_expert(p, f + 32 * u + lane, hi);
#pragma unroll
    for (int u = 0; u < PLAN_AHEAD; ++u) {
      if (f + 32 * u >= hi) break;
      const unsigned same = same_expert(x[u], p.bits);
      int row = -1;
      if (x[u] >= 0) row = base[x[u]] + mine[x[u]] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (x[u] >= 0 && lane == __ffs(same) - 1) mine[x[u]] += __popc(same);
      __syncwarp();
      const int at = f + 32 * u + lane;
      if (at < hi) {
        p.pos[at] = row;
        if (row >= 0) p.order[row] = at;
      }
    }
  }
  for (int r = rows + rank * blockDim.x + threadIdx.x; r < p.R; r += ctas * blockDim.x) p.order[r] = -1;
  if (ctas > 1) cluster_wait();
}

// ---------------------------------------------------------------------------------------------
// gather, combine: bound by memory, 16 bytes a thread.  combine reads rows of a few KB in as many places as a token has experts:
// 8192 x 8 rows of 2048 take 53 us (5.7 TB/s), with the shared rows 66 (5.1 TB/s; 74 while the gate's
// sigmoid was taken before the rows were asked for).  gather: the same rows in e4m3 43 us (their bytes take 23).
// ---------------------------------------------------------------------------------------------
// rows of `vecs` 16-byte pieces; x [T] -> out [R], a pair's row is its token's.  scale: fp32 beside each row, or null
__global__ void __launch_bounds__(256) gather_kernel(const uint4* x, int64_t ld, const float* xs, const int* order, uint4* out,
                                                     float* os, int R, int T, int k, unsigned vecs, int* status) {
  pdl_trigger();
  pdl_wait();
  const unsigned i = blockIdx.x * 256 + threadIdx.x;
  const int r = i / vecs, v = i % vecs;
  if (r >= R) return;
  const int f = order[r];
  if (f < 0) return;
  const int t = f / k;
  if (t >= T) {
    atomicExch(status, (int)kErrBounds);
    return;
  }
  out[(int64_t)r * vecs + v] = x[t * ld + v];
  if (os && v == 0) os[r] = xs[t];
}

struct CombineArgs {
  const __nv_bfloat16* rows;
  const int* pos;
  const float* w;
  const __nv_bfloat16* shared;
  const float* gate;
  __nv_bfloat16* out;
  int64_t ld_rows, ld_shared, ld_gate, ld_out;
  int T, k, H, R;
  int* status;
};

// rows are read once: past the L1
DEVI uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
DEVI uint16_t load_once(const uint16_t* p) { return *p; }

// One thread: W neighbouring columns of a token at a time.  The rows of K slots are asked for before the first is added, and where
// the next token's rows are before this one's have come.
template <int W>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ CombineArgs p) {
  pdl_trigger();
  pdl_wait();
  constexpr int K = 8;
  const unsigned vecs = (p.H + W - 1) / W, total = vecs * (unsigned)p.T, step = gridDim.x * 256u;
  using Vec = typename std::conditional<W == 8, uint4, uint16_t>::type;
  int r[K];
  float w[K];
  auto places = [&](int t, int j0) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      r[j] = -1;
      w[j] = 0.f;
      if (j0 + j < p.k) {
        r[j] = p.pos[(int64_t)t * p.k + j0 + j];
        w[j] = p.w[(int64_t)t * p.k + j0 + j];
      }
    }
  };
  unsigned i = blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  places(i / vecs, 0);
  while (true) {
    const int t = i / vecs, c = i % vecs * W;
    float acc[W];
#pragma unroll
    for (int q = 0; q < W; ++q) acc[q] = 0.f;
    auto add = [&](const Vec& v, float a) {
      const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(&v);
#pragma unroll
      for (int q = 0; q < W; ++q) acc[q] = fmaf(a, __bfloat162float(x[q]), acc[q]);
    };
    Vec sh;
    float g = INFINITY;                                    // what its sigmoid is taken of, once the rows are asked for
    if (p.shared) {
      sh = load_once(reinterpret_cast<const Vec*>(p.shared + t * p.ld_shared + c));
      if (p.gate) g = p.gate[t * p.ld_gate];
    }
    const unsigned next = i + step;
    for (int j0 = 0; j0 < p.k; j0 += K) {
      if (j0) places(t, j0);
      Vec v[K];
      float a[K];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (r[j] >= p.R) {
          atomicExch(p.status, (int)kErrBounds);
          r[j] = -1;
        }
        v[j] = Vec{};
        a[j] = r[j] >= 0 ? w[j] : 0.f;                     // another rank's expert, or none
        if (r[j] >= 0) v[j] = load_once(reinterpret_cast<const Vec*>(p.rows + r[j] * p.ld_rows + c));
      }
      if (j0 + K >= p.k && next < total) places(next / vecs, 0);
#pragma unroll
      for (int j = 0; j < K; ++j) add(v[j], a[j]);
    }
    if (p.shared) add(sh, 1.f / (1.f + __expf(-g)));
    Vec o;
    __nv_bfloat16* x = reinterpret_cast<__nv_bfloat16*>(&o);
#pragma unroll
    for (int q = 0; q < W; ++q) x[q] = __float2bfloat16_rn(acc[q]);
    *reinterpret_cast<Vec*>(p.out + t * p.ld_out + c) = o;
    if (next >= total || next < i) break;
    i = next;
  }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
torch::Tensor empty(at::IntArrayRef size, at::ScalarType type, const torch::Tensor& beside) {
  return at::detail::empty_cuda(size, type, beside.device(), c10::nullopt);
}

template <typename L, int V>
void launch_route(const RouteArgs& p, cudaStream_t stream) {
  const dim3 grid((p.T + 7) / 8);
  if (p.bias) C10_CUDA_CHECK(launch_pdl(route_kernel<L, V, true>, grid, dim3(256), 0, stream, p));
  else C10_CUDA_CHECK(launch_pdl(route_kernel<L, V, false>, grid, dim3(256), 0, stream, p));
}
template <typename L>
void launch_route(RouteArgs& p, cudaStream_t stream) {
  const int v = (p.gsize + p.lanes - 1) / p.lanes;
  const int V = v <= 2 ? 2 : v <= 4 ? 4 : v <= 8 ? 8 : v <= 16 ? 16 : v <= 32 ? 32 : 64;
  // 16-byte loads where every lane's experts are whole pieces of 16 bytes
  p.vec = v == V && p.gsize % v == 0 && V * sizeof(L) >= 16 && (uintptr_t)p.logits % 16 == 0 && p.ld * sizeof(L) % 16 == 0;
  switch (V) {
    case 2: launch_route<L, 2>(p, stream); break;
    case 4: launch_route<L, 4>(p, stream); break;
    case 8: launch_route<L, 8>(p, stream); break;
    case 16: launch_route<L, 16>(p, stream); break;
    case 32: launch_route<L, 32>(p, stream); break;
    // numbers of groups just above a power of two, at most 60 experts a lane (8192 tokens, 17 groups of 40: 74 us, 187 with a bias;
    // 4 groups of 256, 32 a lane: 39 and 95)
    default: launch_route<L, 64>(p, stream);
  }
}

}  // namespace moe

std::tuple<torch::Tensor, torch::Tensor> moe_route(const torch::Tensor& logits, int64_t k, bool sigmoid,
                                     const c10::optional<torch::Tensor>& bias, int64_t groups, int64_t top_groups, bool renorm,
                                     double scale) {
  const auto type = logits.scalar_type();
  RAD_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && (logits.size(0) <= 1 || logits.stride(0) >= logits.size(1)) &&
                        (logits.size(1) <= 1 || logits.stride(1) == 1),
                    "moe_route: logits [T, E], rows contiguous");
  RAD_CHECK_VALUE(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, "moe_route: logits fp32, bf16 or fp16");
  const int64_t T = logits.size(0), E = logits.size(1);
  RAD_CHECK_VALUE(E >= 1 && E <= moe::MAX_E, "moe_route: 1 to ", moe::MAX_E, " experts, got ", E);
  RAD_CHECK_VALUE(k >= 1 && k <= 32 && k <= E, "moe_route: top_k ", k, " of ", E, " experts (at most 32)");
  RAD_CHECK_VALUE(groups >= 1 && groups <= 32 && E % groups == 0, "moe_route: ", groups, " groups of ", E, " experts");
  RAD_CHECK_VALUE(top_groups >= 1 && top_groups <= groups && top_groups * (E / groups) >= k, "moe_route: ", k, " experts in ",
                    top_groups, " of ", groups, " groups");
  RAD_CHECK_VALUE(T < (1ll << 31) - 8, "moe_route: rows");
  if (bias.has_value()) {
    RAD_CHECK_VALUE(bias->device() == logits.device() && bias->scalar_type() == at::kFloat && bias->dim() == 1 &&
                          bias->size(0) == E && bias->is_contiguous(),
                      "moe_route: bias fp32 [E] on the logits' device");
    RAD_CHECK_VALUE(groups == 1 || E / groups >= 2, "moe_route: a group's value is that of two experts");
  }
  moe::RouteArgs p = {};
  int lanes = 32;
  while (lanes * groups > 32) lanes /= 2;
  const at::cuda::CUDAGuard guard(logits.device());
  torch::Tensor ids = moe::empty({T, k}, at::kLong, logits), w = moe::empty({T, k}, at::kFloat, logits);
  if (T == 0) return {ids, w};
  p.logits = logits.data_ptr();
  p.bias = bias.has_value() ? bias->data_ptr<float>() : nullptr;
  p.ids = ids.data_ptr<int64_t>();
  p.w = w.data_ptr<float>();
  p.ld = T == 1 ? (E + 15) / 16 * 16 : logits.stride(0);
  p.T = T; p.E = E; p.k = k; p.groups = groups; p.top_groups = top_groups; p.gsize = E / groups; p.lanes = lanes;
  p.sigmoid = sigmoid; p.renorm = renorm; p.scale = (float)scale;
  auto stream = at::cuda::getCurrentCUDAStream();
  if (type == at::kFloat) moe::launch_route<float>(p, stream);
  else if (type == at::kBFloat16) moe::launch_route<__nv_bfloat16>(p, stream);
  else moe::launch_route<__half>(p, stream);
  return {ids, w};
}

// -> order [T k], pos [T, k], counts [E], starts [E + 1], items [max_items, 3] (empty without a tile height)
std::vector<torch::Tensor> moe_plan(const torch::Tensor& ids_, int64_t E, int64_t first, int64_t tile) {
  const auto type = ids_.scalar_type();
  RAD_CHECK_VALUE(ids_.is_cuda() && ids_.dim() == 2 && (type == at::kLong || type == at::kInt),
                    "moe_plan: ids [T, k], int64 or int32");
  RAD_CHECK_VALUE(E >= 1 && E <= moe::MAX_E, "moe_plan: 1 to ", moe::MAX_E, " experts, got ", E);
  RAD_CHECK_VALUE(first >= 0 && first < (1ll << 30) && tile >= 0 && tile <= (1 << 20), "moe_plan: first expert, tile height");
  const int64_t T = ids_.size(0), k = ids_.size(1), R = T * k;
  RAD_CHECK_VALUE(k >= 1 && R < (1ll << 30), "moe_plan: 1 to 2^30 pairs");
  const at::cuda::CUDAGuard guard(ids_.device());
  const torch::Tensor ids = ids_.contiguous();
  torch::Tensor order = moe::empty({R}, at::kInt, ids), pos = moe::empty({T, k}, at::kInt, ids),
                counts = moe::empty({E}, at::kInt, ids), starts = moe::empty({E + 1}, at::kInt, ids);
  const int64_t max_items = tile ? (R + tile - 1) / tile + E : 0;
  torch::Tensor items = tile ? moe::empty({max_items, 3}, at::kInt, ids) : counts;
  moe::PlanArgs p = {};
  p.ids = ids.data_ptr(); p.R = R; p.k = k; p.E = E; p.first = first; p.wide = type == at::kLong;
  while (1ll << p.bits < E) ++p.bits;
  p.order = order.data_ptr<int>(); p.pos = pos.data_ptr<int>();
  p.counts = counts.data_ptr<int>(); p.starts = starts.data_ptr<int>();
  p.items = tile ? items.data_ptr<int>() : nullptr; p.tile = tile; p.max_items = max_items;
  int ctas = 1;
  while (ctas < moe::PLAN_CTAS && R > 4096ll * ctas) ctas *= 2;
  p.seg = std::max<int64_t>(32, ((R + 32 * ctas - 1) / (32 * ctas) + 31) / 32 * 32);
  p.warps = std::max<int64_t>(1, std::min<int64_t>(moe::PLAN_WARPS, (R + (int64_t)p.seg * ctas - 1) / ((int64_t)p.seg * ctas)));
  const size_t smem = (moe::PLAN_WARPS + 2) * E * sizeof(int);
  static std::atomic<uint64_t> set{0};                     // devices whose kernel may take clusters of 16 and the shared memory of MAX_E experts
  const int dev = ids.get_device();
  if (dev >= 64 || !(set.load() >> dev & 1)) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(moe::plan_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    C10_CUDA_CHECK(cudaFuncSetAttribute(moe::plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)((moe::PLAN_WARPS + 2) * moe::MAX_E * sizeof(int))));
    if (dev < 64) set.fetch_or(1ull << dev);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(1024);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = at::cuda::getCurrentCUDAStream();
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)ctas, 1, 1};
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, moe::plan_kernel, p));
  return {order, pos, counts, starts, items};
}

void moe_gather(const torch::Tensor& x, const c10::optional<torch::Tensor>& xs, const torch::Tensor& order, int64_t k,
                const torch::Tensor& out, const c10::optional<torch::Tensor>& out_s, const torch::Tensor& status) {
  const int64_t T = x.size(0), R = order.size(0), bytes = x.size(1) * x.element_size();
  RAD_CHECK_VALUE(x.is_cuda() && x.dim() == 2 && x.stride(1) == 1 && bytes % 16 == 0 && (uintptr_t)x.data_ptr() % 16 == 0 &&
                        (T <= 1 || x.stride(0) * x.element_size() % 16 == 0) && order.device() == x.device(),
                    "moe_gather: rows of whole 16 bytes");
  RAD_CHECK_VALUE(R == T * k && out.is_contiguous() && out.size(0) == R && out.size(1) == x.size(1), "moe_gather: rows");
  RAD_CHECK_VALUE(!xs.has_value() || (xs->device() == x.device() && xs->scalar_type() == at::kFloat && xs->is_contiguous() &&
                                        xs->numel() == T && out_s->numel() == R),
                    "moe_gather: scales fp32 [T]");
  if (R == 0 || bytes == 0) return;
  const at::cuda::CUDAGuard guard(x.device());
  const unsigned vecs = bytes / 16;
  RAD_CHECK_VALUE(R * vecs < (1ll << 31), "moe_gather: rows");
  C10_CUDA_CHECK(launch_pdl(moe::gather_kernel, dim3((R * vecs + 255) / 256), dim3(256), 0, at::cuda::getCurrentCUDAStream(),
                            (const uint4*)x.data_ptr(), (int64_t)(x.stride(0) * x.element_size() / 16),
                            xs.has_value() ? (const float*)xs->data_ptr<float>() : nullptr, (const int*)order.data_ptr<int>(),
                            (uint4*)out.data_ptr(), xs.has_value() ? out_s->data_ptr<float>() : nullptr, (int)R, (int)T, (int)k,
                            vecs, status.data_ptr<int>()));
}

torch::Tensor moe_combine(const torch::Tensor& rows, const torch::Tensor& pos, const torch::Tensor& w,
                          const c10::optional<torch::Tensor>& shared, const c10::optional<torch::Tensor>& gate,
                          const torch::Tensor& status) {
  RAD_CHECK_VALUE(rows.is_cuda() && rows.dim() == 2, "moe_combine: rows bf16 [T k, H]");
  const int64_t T = pos.size(0), k = pos.size(1), H = rows.size(1), R = rows.size(0);
  const auto bf16_rows = [&](const torch::Tensor& t, int64_t n) {
    return t.dim() == 2 && t.size(0) == n && t.size(1) == H && (H <= 1 || t.stride(1) == 1) && t.scalar_type() == at::kBFloat16 &&
           t.device() == rows.device();
  };
  RAD_CHECK_VALUE(rows.is_cuda() && bf16_rows(rows, R) && R == T * k, "moe_combine: rows bf16 [T k, H]");
  RAD_CHECK_VALUE(w.device() == rows.device() && w.scalar_type() == at::kFloat && w.is_contiguous() && w.dim() == 2 &&
                        w.size(0) == T && w.size(1) == k,
                    "moe_combine: weights fp32 [T, k]");
  RAD_CHECK_VALUE(pos.device() == rows.device(), "moe_combine: operands on one device");
  RAD_CHECK_VALUE(!shared.has_value() || bf16_rows(*shared, T), "moe_combine: shared bf16 [T, H]");
  RAD_CHECK_VALUE(!gate.has_value() || (shared.has_value() && gate->device() == rows.device() &&
                                          gate->scalar_type() == at::kFloat && gate->dim() == 1 && gate->size(0) == T),
                    "moe_combine: gate fp32 [T], beside shared");
  const at::cuda::CUDAGuard guard(rows.device());
  torch::Tensor out = moe::empty({T, H}, at::kBFloat16, rows);
  if (T == 0 || H == 0) return out;
  moe::CombineArgs p = {};
  p.rows = (const __nv_bfloat16*)rows.data_ptr();
  p.pos = pos.data_ptr<int>();
  p.w = w.data_ptr<float>();
  p.shared = shared.has_value() ? (const __nv_bfloat16*)shared->data_ptr() : nullptr;
  p.gate = gate.has_value() ? gate->data_ptr<float>() : nullptr;
  p.out = (__nv_bfloat16*)out.data_ptr();
  p.ld_rows = rows.stride(0); p.ld_shared = shared.has_value() ? shared->stride(0) : 0;
  p.ld_gate = gate.has_value() ? gate->stride(0) : 0; p.ld_out = out.stride(0);
  p.T = T; p.k = k; p.H = H; p.R = R;
  p.status = status.data_ptr<int>();
  const bool vec = H % 8 == 0 && (p.ld_rows | p.ld_shared | p.ld_out) % 8 == 0 &&
                   ((uintptr_t)p.rows | (uintptr_t)p.shared | (uintptr_t)p.out) % 16 == 0;
  const int64_t blocks = (T * (vec ? H / 8 : H) + 255) / 256;
  RAD_CHECK_VALUE(blocks < (1ll << 23), "moe_combine: rows");
  auto stream = at::cuda::getCurrentCUDAStream();
  // four blocks an SM, of which two run at once (116 registers), each over several tokens (8192 x 8 rows of 2048 and shared ones:
  // 66 us, 83 with three, which leave half of the places empty at the end, 76 with a block for every 256 pieces)
  const unsigned grid = (unsigned)std::min<int64_t>(blocks, 4ll * at::cuda::getDeviceProperties(rows.get_device())->multiProcessorCount);
  if (vec) C10_CUDA_CHECK(launch_pdl(moe::combine_kernel<8>, dim3(grid), dim3(256), 0, stream, p));
  else C10_CUDA_CHECK(launch_pdl(moe::combine_kernel<1>, dim3(grid), dim3(256), 0, stream, p));
  return out;
}

}  // namespace rad
