// bf16 product with an epilogue, of one weight or of one weight per expert (rows sorted by expert, moe.cu's plan):
//
//   y[r]   = x[row(r)] W[e(r)]^T + b[e(r)]          K products of bf16 numbers, exact and summed in 32 bits
//   out[r] = res[r] + scale[r] * act(y[r])          act: y, or SwiGLU of y = [g | u]: g / (1 + exp(-g)) * u
//
// rounded once.  An output tile is 128 weight rows (the MMA's M) of one expert x up to BN of its rows (N).  With SwiGLU the
// weight rows of a tile are 64 pairs of a gate row and its up row, which a TMA box over [.., 2, N / 2, ..] brings in this
// order, so that both factors of an output meet in one tile.  Warp 0 fills the ring of 64-k stages by TMA, warp 1 issues the MMAs
// into one of two accumulators in tensor memory, eight warps carry the other one out, straight from registers.  Rows that are
// picked by token come by asynchronous 16-byte copies of four more warps: TMA takes four rows by number a load and some 65 cycles
// for each, which a tile of more than 32 rows waits for (512 tokens, 256 experts: 264 us, this 166).
//
// Up to 32 rows an expert it is bound by memory, the weights (256 experts, top-8, 2048 -> 512 SwiGLU and 512 -> 2048, B200, best of
// 7 graphs of 10 calls): 64 tokens, which use 197 of the experts, 126 and 65 us (6.5 and 6.4 TB/s), 1024 tokens 172 and 94 us (6.3
// and 6.1 TB/s), one token 10 us, of which 5 are the bytes and the rest one chain of latencies (plan, first tiles, the cluster's sum).
// With more rows tiles wait for what L2 hands out, weights and rows together some 10 TB/s: 4096 tokens 228 and 124 us, 8192 tokens
// 342 and 192 us (call after call for longer, when clocks fall, 400).  One weight, 5120 -> 8704 SwiGLU, 4096 rows: 451 us, 1619
// TFLOP/s, MMAs.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <map>
#include <mutex>

#include "common.cuh"
#include "refuse.h"
#include "tma_host.h"

namespace rad {
namespace lf {

constexpr int BM = 128, BK = 64;
constexpr int A_BYTES = BM * BK * 2;
constexpr int SUM_LD = 144;                                // floats of a staged row (SPLIT); the up half starts 16 banks behind the gate half
constexpr int SMEM_MAX = 227 * 1024;
constexpr int MAX_E = 1024;
// warps: 0 loads weights (and rows in order), 1 issues MMAs, 8 carry sums out, 4 pick rows by token; on a pair one more, which tells the
// first CTA that the second one's sums are out
constexpr int EPI0 = 2, EPI_WARPS = 8, GATHER0 = EPI0 + EPI_WARPS, GATHER_WARPS = 4, RELAY = GATHER0 + GATHER_WARPS;
constexpr int threads(bool pair) { return 32 * (RELAY + (pair ? 1 : 0)); }

struct Args {
  const int* starts;                                       // [E + 1] rows of the experts; null: one expert, R rows
  const int* order;                                        // [R] pair of a row, pair / k is its token; null: rows of x in order
  const __nv_bfloat16* x;
  const __nv_bfloat16* bias;                               // [E, N]
  const __nv_bfloat16* res;
  const float* scale;
  __nv_bfloat16* out;
  int64_t x_ld, res_ld, out_ld;
  int R, T, k, E, N, W, K;                                 // W: width of out (N, or N / 2 with SwiGLU)
  int tile;                                                // rows of a tile, at most the kernel's BN
  bool vec;
  int* status;
};

// BN rows of a tile, of which a CTA of a pair stages half
template <int BN, bool PAIR, bool SPLIT> struct Cfg {
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
  static constexpr int STAGE = A_BYTES + B_ROWS * BK * 2;
  static constexpr int SUMS = SPLIT ? BN * SUM_LD * 4 : 0;
  static constexpr int META = 1024 + 2 * (MAX_E + 1) * 4;
  static constexpr int STAGES = (SMEM_MAX - 1024 - SUMS - META) / STAGE < 12 ? (SMEM_MAX - 1024 - SUMS - META) / STAGE : 12;
  static constexpr int SMEM = 1024 + STAGES * STAGE + SUMS + META;
  static constexpr int TMEM = 2 * BN < 32 ? 32 : 2 * BN;
};

struct Bars {
  uint4 token;                                             // what send_token copies
  uint64_t full[12], picked[12], empty[12], acc_full[2], acc_empty[2], drained[2];
  uint32_t tmem;
  int abort;
};

// x in boxes of 16, 32, 64 and 128 rows: a load instruction costs some 65 cycles whatever it brings, so that a stage of 128 rows
// in boxes of 16 took 600 cycles of loads for 512 of MMAs (8192 rows, 5120 -> 17408: 1111 TFLOP/s)
struct RowMaps {
  CUtensorMap box[4];
};

struct Item {
  int e, n0, row0, rows;                                   // weight block (out's first feature), rows of out
};

DEVI uint32_t idesc_bf16(int m, int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
DEVI void tma_2d(uint32_t dst, const void* map, uint32_t bar, int c, int r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c), "r"(r)
      : "memory");
}
DEVI void tma_4d(uint32_t dst, const void* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// the same on a CTA pair: into this CTA's memory, counted by the barrier at a cluster address
DEVI void tma_2d_pair(uint32_t dst, const void* map, uint32_t bar, int c, int r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c), "r"(r)
      : "memory");
}
DEVI void tma_4d_pair(uint32_t dst, const void* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
DEVI void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrive on the barrier at a cluster address once the pair's MMAs so far are done
DEVI void commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Arrive on the other CTA's barrier, after all that this thread has seen: a release of cluster scope.  It takes some 0.8 us, so that a
// thread does it which nobody waits for (the warp RELAY, once an item; 512 -> 2048, 4096 tokens of 256 experts: 124 us, 123 with no release)
DEVI void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Tell the other CTA's barrier of what this thread has seen, for the tensor cores to read: a copy of 16 bytes in the proxy of
// the MMAs, whose arrival counts there as bytes of the stage do.  The thread does not wait, as it would for a release of cluster scope at
// some 0.8 us a stage (4096 tokens of 256 experts, 2048 -> 512 SwiGLU: 559 us, this 228, and 226 with an arrival that orders nothing)
DEVI void send_token(uint32_t dst, uint32_t src, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], 16, [%2];" ::"r"(dst), "r"(src),
               "r"(bar)
               : "memory");
}
// mbar_wait for arrivals of the other CTA
DEVI bool wait_cluster(uint64_t* bar, uint32_t phase, int* err) {
  const auto done = [&]() {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(phase)
        : "memory");
    return ok != 0;
  };
  if (done()) return true;
  const uint64_t t0 = globaltimer_ns(), limit = wait_limit_ns(err, 2, kWaitNs);
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (done()) return true;
    if (globaltimer_ns() - t0 > limit) break;
  }
  if (err) atomicExch(err, (int)kErrMbarTimeout);
  return false;
}
DEVI void tmem_ld_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// 16 bytes global -> shared; none of them (zeros) unless `in`
DEVI void cp_async16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
// arrive on this CTA's barrier once the thread's copies so far have landed
DEVI void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Tiles before each expert -> tiles[0 .. E] from starts[0 .. E], by one warp: a lane adds up neighbours.
DEVI void count_tiles(const Args& p, int bn, int* tiles, const int* starts, int lane) {
  const int each = (p.E + 31) / 32, e0 = min(p.E, lane * each), e1 = min(p.E, e0 + each);
  int sum = 0;
  for (int e = e0; e < e1; ++e) {
    tiles[e] = sum;
    sum += (max(0, starts[e + 1] - starts[e]) + bn - 1) / bn;
  }
  int before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += y;
  }
  before -= sum;
  for (int e = e0; e < e1; ++e) tiles[e] += before;
  if (lane == 31) tiles[p.E] = before + sum;
}

// Item i: the row tiles of one weight block are neighbours, so that the CTAs which need the block ask for it together.
DEVI Item item_of(const Args& p, int i, int blocks, int bn, int span, const int* tiles, const int* starts) {
  const int t = i / blocks;
  int lo = 0, hi = p.E;
  while (hi - lo > 1) {                                    // the last expert whose first tile is not behind t
    const int mid = (lo + hi) / 2;
    if (tiles[mid] <= t) lo = mid; else hi = mid;
  }
  const int n = tiles[lo + 1] - tiles[lo], local = i - tiles[lo] * blocks;
  Item q;
  q.e = lo;
  q.n0 = local / n * span;
  q.row0 = starts[lo] + local % n * bn;
  q.rows = min(bn, starts[lo + 1] - q.row0);
  return q;
}

DEVI float silu(float g) { return __fdividef(g, 1.f + __expf(-g)); }
DEVI uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What four neighbouring features f .. f + 3 of a row need from memory
struct Rest {
  float scale;
  uint2 res;
};
// column of a lane's j-th four features, and the first of them
template <bool SWIGLU> DEVI int column_of(int j, int lane) { return SWIGLU ? 8 * j + (lane & 7) : 4 * j + (lane & 3); }
template <bool SWIGLU> DEVI int feature_of(int lane) { return SWIGLU ? (lane >> 1) & ~3 : lane & ~3; }

template <bool WHOLE, bool FULL> DEVI Rest load_rest(const Args& p, int64_t row, int f, bool in) {
  Rest q = {1.f, make_uint2(0, 0)};
  if (p.scale && (FULL || in)) q.scale = p.scale[row];
  if (p.res && (FULL || in)) {
    const __nv_bfloat16* r = p.res + row * p.res_ld + f;
    if (WHOLE || (p.vec && f + 4 <= p.W)) {
      q.res = *reinterpret_cast<const uint2*>(r);
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(r);
      if (f < p.W) q.res.x = h[0];
      if (f + 1 < p.W) q.res.x |= (uint32_t)h[1] << 16;
      if (f + 2 < p.W) q.res.y = h[2];
      if (f + 3 < p.W) q.res.y |= (uint32_t)h[3] << 16;
    }
  }
  return q;
}
template <bool REST, bool WHOLE, bool FULL>
DEVI void store4(const Args& p, __nv_bfloat16* out, int f, bool in, const Rest& q, float y0, float y1, float y2, float y3) {
  if (REST) {
    y0 *= q.scale, y1 *= q.scale, y2 *= q.scale, y3 *= q.scale;
    if (p.res) {                                           // without one, -0 stays -0
      y0 += __uint_as_float(q.res.x << 16), y1 += __uint_as_float(q.res.x & 0xffff0000u);
      y2 += __uint_as_float(q.res.y << 16), y3 += __uint_as_float(q.res.y & 0xffff0000u);
    }
  }
  const uint32_t a = pack(y0, y1), b = pack(y2, y3);
  if (FULL || in) {
    if (WHOLE || (p.vec && f + 4 <= p.W)) {
      *reinterpret_cast<uint2*>(out) = make_uint2(a, b);
    } else {
      uint16_t* o = reinterpret_cast<uint16_t*>(out);
      if (f < p.W) o[0] = (uint16_t)a;
      if (f + 1 < p.W) o[1] = (uint16_t)(a >> 16);
      if (f + 2 < p.W) o[2] = (uint16_t)b;
      if (f + 3 < p.W) o[3] = (uint16_t)(b >> 16);
    }
  }
}

// 32 columns (rows of out from row0 on, n of them in use) of a warp's 32 weight rows -> out.  A lane holds one weight row; lanes
// trade columns until each has four neighbouring features of one row, so that a store covers whole 32-byte sectors.
// WHOLE: the features are all in use and on 8 bytes; FULL: so are all columns, and nothing branches, so that the trades of all of
// them overlap: 8192 tokens of 256 experts, 512 -> 2048, took half as long again (257 us) with a test at every store.
template <bool SWIGLU, bool REST, bool WHOLE, bool FULL>
DEVI void store_columns(const Args& p, const float (&v)[32], int64_t row0, int n, int f0, int lane) {
  constexpr int J = SWIGLU ? 4 : 8, STEP = 32 / J;
  const bool l0 = lane & 1, l1 = lane & 2, l2 = lane & 4;
  const int f = f0 + feature_of<SWIGLU>(lane), c0 = column_of<SWIGLU>(0, lane);
  // each pair of lanes trades one of two columns
  auto trade = [&](float mine, float other, bool second, int lanes) {
    return __shfl_xor_sync(0xffffffffu, second ? mine : other, lanes);
  };
  Rest rest[J];
  if (REST)
#pragma unroll
    for (int j = 0; j < J; ++j)
      rest[j] = load_rest<WHOLE, FULL>(p, row0 + c0 + j * STEP, f, c0 + j * STEP < n && f < p.W);
  __nv_bfloat16* out = p.out + (row0 + c0) * p.out_ld + f;
  const int64_t step = STEP * p.out_ld;
#pragma unroll
  for (int j = 0; j < J; ++j, out += step) {
    if (!FULL && j * STEP >= n) break;
    float y[2][2];
    if constexpr (SWIGLU) {
      // lane 2 i holds the gate and lane 2 i + 1 the up row of feature f0 + i
      float h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = v[8 * j + 2 * i], b = v[8 * j + 2 * i + 1], o = trade(a, b, l0, 1);
        h[i] = silu(l0 ? o : a) * (l0 ? b : o);            // column 8 j + 2 i + l0
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float o = trade(h[2 * i], h[2 * i + 1], l1, 2);
        y[i][0] = l1 ? o : h[2 * i];
        y[i][1] = l1 ? h[2 * i + 1] : o;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float a = v[4 * j + 2 * i], b = v[4 * j + 2 * i + 1], o = trade(a, b, l0, 1);
        y[i][0] = l0 ? o : a;
        y[i][1] = l0 ? b : o;
      }
    }
    const bool last = SWIGLU ? l2 : l1;
    constexpr int LANES = SWIGLU ? 4 : 2;
    const float o0 = trade(y[0][0], y[1][0], last, LANES), o1 = trade(y[0][1], y[1][1], last, LANES);
    store4<REST, WHOLE, FULL>(p, out, f, c0 + j * STEP < n && f < p.W, rest[j], last ? o0 : y[0][0], last ? o1 : y[0][1],
                        last ? y[1][0] : o0, last ? y[1][1] : o1);
  }
}

// Staged sums of one row (position of a weight row: sum_pos) -> out, by 128 threads
DEVI int sum_pos(bool swiglu, int row) { return swiglu ? (row & 1) * 80 + row / 2 : row; }

template <bool SWIGLU>
DEVI void store_row(const Args& p, const Item& q, const float* st, int c, int tid) {
  const int f = q.n0 + tid;
  if (tid >= (SWIGLU ? BM / 2 : BM) || f >= p.W) return;
  const __nv_bfloat16* b = p.bias + (int64_t)q.e * p.N;
  float y = st[tid];
  if (p.bias) y += __bfloat162float(b[f]);
  if (SWIGLU) {
    float u = st[80 + tid];
    if (p.bias) u += __bfloat162float(b[p.W + f]);
    y = silu(y) * u;
  }
  const int64_t row = q.row0 + c;
  if (p.scale) y *= p.scale[row];
  if (p.res) y += __bfloat162float(p.res[row * p.res_ld + f]);
  p.out[row * p.out_ld + f] = __float2bfloat16_rn(y);
}

// PAIR: two CTAs share a tile of 256 weight rows; each stages its 128 and its half of the tile's rows, and the first one issues
// the MMAs of both.  SPLIT: a cluster shares one item's K; its CTAs' sums meet through distributed shared memory, each CTA adds
// up and stores some of the rows.  Otherwise a CTA (or pair) an SM (or two) runs every n-th item.
template <int BN, bool SWIGLU, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(threads(PAIR), 1) kernel(const __grid_constant__ Args p, const __grid_constant__ CUtensorMap wm,
                                                     const __grid_constant__ RowMaps xm) {
  using C = Cfg<BN, PAIR, SPLIT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* st = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE);
  Bars* bars = reinterpret_cast<Bars*>(smem + C::STAGES * C::STAGE + C::SUMS);
  int* tiles = reinterpret_cast<int*>(smem + C::STAGES * C::STAGE + C::SUMS + 1024);
  int* starts = tiles + MAX_E + 1;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int splits = SPLIT ? gridDim.y : 1, share = SPLIT ? blockIdx.y : 0;
  const int rank = PAIR ? cluster_ctarank() : 0;           // 0 issues the MMAs
  const int unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, units = PAIR ? gridDim.x >> 1 : gridDim.x;
  constexpr int HALF = SWIGLU ? BM / 2 : BM;               // features of a CTA
  constexpr int SPAN = PAIR ? 2 * HALF : HALF;
  const int blocks = (p.W + SPAN - 1) / SPAN;
  const int all_k = (p.K + BK - 1) / BK;
  const int k0 = (int)((int64_t)all_k * share / splits), k1 = (int)((int64_t)all_k * (share + 1) / splits);
  const bool gather = p.order != nullptr;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->picked[s], 32 * GATHER_WARPS);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], EPI_WARPS + (PAIR ? 1 : 0));
      mbar_init(&bars->drained[b], EPI_WARPS);
    }
    bars->abort = 0;
    bars->token = make_uint4(0, 0, 0, 0);
    fence_mbar_init();
    tma_prefetch_desc(&wm);
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem)), "r"(C::TMEM)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(&bars->tmem, C::TMEM);
      tmem_relinquish();
    }
  }
  pdl_wait();
  for (int e = threadIdx.x; e <= p.E; e += threads(PAIR)) starts[e] = p.starts ? p.starts[e] : e ? p.R : 0;
  __syncthreads();
  if (warp == 2) count_tiles(p, p.tile, tiles, starts, lane);
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (PAIR) cluster_sync();                                // both CTAs' barriers and tensor memory are there
  tc_fence_after();
  pdl_trigger();                                           // this block holds its tensor memory
  const uint32_t tmem = bars->tmem;
  const int items = tiles[p.E] * blocks;
  volatile int* abort = &bars->abort;
  const uint32_t abort_peer = PAIR ? mapa_shared(smem_u32(&bars->abort), rank ^ 1) : 0;
  // a failed wait stops the CTA, and its partner
  auto give_up = [&]() {
    *abort = 1;
    if (PAIR) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(abort_peer), "r"(1) : "memory");
  };
  auto in_order = [&](const Item& q) { return q.row0 >= 0 && q.rows > 0 && q.row0 + q.rows <= p.R; };
  // rows of the MMA, and of them those that this CTA stages: [b0, b0 + bn)
  auto mma_rows = [&](const Item& q) { return PAIR ? (q.rows + 31) / 32 * 32 : (q.rows + 15) / 16 * 16; };

  if (warp == 0) {
    uint32_t it = 0;
    for (int i = unit; i < items; i += units) {
      if (__any_sync(0xffffffffu, *abort)) break;          // the same answer in all lanes
      const Item q = item_of(p, i, blocks, p.tile, SPAN, tiles, starts);
      if (!in_order(q)) {
        if (lane == 0) atomicExch(p.status, (int)kErrBounds);
        give_up();
        break;
      }
      // rows of the tile: the boxes that make up their number, one a lane, the largest first
      const int bn = mma_rows(q) / (PAIR ? 2 : 1), box = min(lane, 3), above = bn >> (box + 5) << (box + 5);
      const bool loads = !gather && lane < 4 && (bn >> (box + 4) & 1);
      const uint32_t bbytes = gather ? 0 : bn * BK * 2;
      const int row = q.row0 + rank * bn + above;
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&bars->empty[s], ((it / C::STAGES) & 1) ^ 1, p.status)) give_up();
        if (__any_sync(0xffffffffu, *abort)) break;
        const uint32_t a = smem_u32(smem + s * C::STAGE), b = a + A_BYTES;
        uint32_t full = smem_u32(&bars->full[s]);
        if (PAIR) full = mapa_shared(full, 0);
        if (lane == 0) {
          if (rank == 0)
            mbar_arrive_expect_tx(&bars->full[s], (PAIR ? 2 : 1) * (A_BYTES + bbytes) + (PAIR && gather ? sizeof(bars->token) : 0));
          const int f = q.n0 + rank * HALF;
          if (PAIR && SWIGLU) tma_4d_pair(a, &wm, full, kb * BK, 0, f, q.e);
          else if (PAIR) tma_4d_pair(a, &wm, full, kb * BK, f, 0, q.e);
          else if (SWIGLU) tma_4d(a, &wm, full, kb * BK, 0, f, q.e);
          else tma_4d(a, &wm, full, kb * BK, f, 0, q.e);
        }
        __syncwarp();
        if (loads) {
          if (PAIR) tma_2d_pair(b + above * 128, &xm.box[box], full, kb * BK, row);
          else tma_2d(b + above * 128, &xm.box[box], full, kb * BK, row);
        }
      }
    }
    // given up: the loads in flight land before the block leaves
    if (*abort && rank == 0)
      for (uint32_t j = it > C::STAGES ? it - C::STAGES : 0; j < it; ++j)
        mbar_wait(&bars->full[j % C::STAGES], (j / C::STAGES) & 1, p.status);
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t empty1 = PAIR ? mapa_shared(smem_u32(&bars->empty[0]), 1) : 0;
      const uint32_t acc_full1 = PAIR ? mapa_shared(smem_u32(&bars->acc_full[0]), 1) : 0;
      uint32_t it = 0, n = 0;
      for (int i = unit; i < items && !*abort; i += units, ++n) {
        const Item q = item_of(p, i, blocks, p.tile, SPAN, tiles, starts);
        const int ab = n & 1;
        const uint32_t aph = ((n >> 1) & 1) ^ 1;
        if (!(PAIR ? wait_cluster(&bars->acc_empty[ab], aph, p.status) : mbar_wait(&bars->acc_empty[ab], aph, p.status))) {
          give_up();
          break;
        }
        tc_fence_after();
        const uint32_t idesc = idesc_bf16(PAIR ? 2 * BM : BM, mma_rows(q));
        bool ok = true;
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int s = it % C::STAGES;
          const uint32_t ph = (it / C::STAGES) & 1;
          if (!mbar_wait(&bars->full[s], ph, p.status)) { ok = false; break; }
          if (gather) {
            if (!mbar_wait(&bars->picked[s], ph, p.status)) { ok = false; break; }
            fence_proxy_async();                           // the copies were ordinary writes
          }
          tc_fence_after();
          const uint32_t a = smem_u32(smem + s * C::STAGE), b = a + A_BYTES;
#pragma unroll
          for (int j = 0; j < BK / 16; ++j) {
            if (PAIR) mma_pair(tmem + ab * BN, sdesc_sw128(a + j * 32), sdesc_sw128(b + j * 32), idesc, kb > k0 || j > 0);
            else mma_f16(tmem + ab * BN, sdesc_sw128(a + j * 32), sdesc_sw128(b + j * 32), idesc, kb > k0 || j > 0);
          }
          if (PAIR) {
            commit_pair(smem_u32(&bars->empty[s]));
            commit_pair(empty1 + s * 8);
          } else {
            mma_commit(&bars->empty[s]);
          }
        }
        if (!ok) { give_up(); break; }
        if (PAIR) {
          commit_pair(smem_u32(&bars->acc_full[ab]));
          commit_pair(acc_full1 + ab * 8);
        } else {
          mma_commit(&bars->acc_full[ab]);
        }
      }
    }
    if (PAIR && gather && rank == 1 && elect_one()) {
      // this CTA's picked rows, for the one that issues the MMAs
      const uint32_t full0 = mapa_shared(smem_u32(&bars->full[0]), 0), token0 = mapa_shared(smem_u32(&bars->token), 0);
      uint32_t it = 0;
      for (int i = unit; i < items && !*abort; i += units)
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&bars->picked[s], (it / C::STAGES) & 1, p.status)) { give_up(); break; }
          fence_proxy_async();
          send_token(token0, smem_u32(&bars->token), full0 + s * 8);
        }
    }
    __syncwarp();
  } else if (warp < GATHER0) {
    const int quad = warp & 3, part = (warp - EPI0) / 4;   // 32 weight rows; columns 64 j + 32 part
    const bool rest = p.scale || p.res;
    uint64_t* out_of = PAIR && rank ? bars->drained : bars->acc_empty;
    uint32_t n = 0;
    for (int i = unit; i < items; i += units, ++n) {
      const Item q = item_of(p, i, blocks, p.tile, SPAN, tiles, starts);
      const int ab = n & 1;
      const int f0 = q.n0 + rank * HALF + quad * (HALF / 4);          // the warp's first feature
      float bias = 0.f;
      if (!SPLIT && p.bias) {
        const int f = f0 + (SWIGLU ? lane >> 1 : lane);
        if (f < p.W) bias = __bfloat162float(p.bias[(int64_t)q.e * p.N + f + (SWIGLU && (lane & 1) ? p.W : 0)]);
      }
      if (!mbar_wait(&bars->acc_full[ab], (n >> 1) & 1, p.status)) give_up();
      if (__any_sync(0xffffffffu, *abort)) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + ab * BN;
      if constexpr (SPLIT) {
        if (part == 0) {
#pragma unroll
          for (int c = 0; c < BN; c += 16) {
            uint32_t r[16];
            tmem_ld_32x32b_x16(acc + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) st[(c + j) * SUM_LD + sum_pos(SWIGLU, quad * 32 + lane)] = __uint_as_float(r[j]);
          }
        }
      } else {
        for (int c0 = 32 * part; c0 < q.rows; c0 += 64) {
          uint32_t r[32];
          if constexpr (BN == 16) {
            uint32_t h[16];
            tmem_ld_32x32b_x16(acc, h);
#pragma unroll
            for (int j = 0; j < 16; ++j) r[j] = h[j], r[16 + j] = 0;
          } else {
            tmem_ld_x32(acc + c0, r);
          }
          tmem_ld_wait();
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]) + bias;
          if (c0 + 64 >= q.rows) {                         // this warp has read all that it needs
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&out_of[ab]);
          }
          const int cols = min(32, q.rows - c0);
          const bool whole = p.vec && f0 + HALF / 4 <= p.W;
          if (whole && cols == 32) {
            if (rest) store_columns<SWIGLU, true, true, true>(p, v, q.row0 + c0, cols, f0, lane);
            else store_columns<SWIGLU, false, true, true>(p, v, q.row0 + c0, cols, f0, lane);
          } else if (whole) {
            if (rest) store_columns<SWIGLU, true, true, false>(p, v, q.row0 + c0, cols, f0, lane);
            else store_columns<SWIGLU, false, true, false>(p, v, q.row0 + c0, cols, f0, lane);
          } else {
            store_columns<SWIGLU, true, false, false>(p, v, q.row0 + c0, cols, f0, lane);
          }
        }
        if (32 * part >= q.rows && lane == 0) mbar_arrive(&out_of[ab]);
      }
    }
  } else if (PAIR && warp == RELAY) {
    if (rank == 1 && elect_one()) {
      const uint32_t acc_empty0 = mapa_shared(smem_u32(&bars->acc_empty[0]), 0);
      uint32_t n = 0;
      for (int i = unit; i < items && !*abort; i += units, ++n) {
        if (!mbar_wait(&bars->drained[n & 1], (n >> 1) & 1, p.status)) { give_up(); break; }
        tc_fence_after();
        tc_fence_before();
        arrive_at(acc_empty0 + (n & 1) * 8);
      }
    }
    __syncwarp();
  } else if (gather) {
    // rows by token: thread t brings 16-byte piece t % 8 of rows t / 8, t / 8 + 16, ... of every stage
    const int tid = threadIdx.x - 32 * GATHER0, piece = tid % 8, r0 = tid / 8;
    constexpr int EACH = C::B_ROWS / 16;
    uint32_t it = 0;
    for (int i = unit; i < items; i += units) {
      if (__any_sync(0xffffffffu, *abort)) break;
      const Item q = item_of(p, i, blocks, p.tile, SPAN, tiles, starts);
      if (!in_order(q)) break;                             // warp 0 says so
      const int bn = mma_rows(q) / (PAIR ? 2 : 1), first = rank * bn, mine = min(bn, q.rows - first);
      const __nv_bfloat16* src[EACH];
#pragma unroll
      for (int h = 0; h < EACH; ++h) {
        const int c = r0 + 16 * h;
        src[h] = nullptr;
        if (c < mine) {
          int t = p.order[q.row0 + first + c];
          if (t < 0 || t >= (int64_t)p.T * p.k) {
            atomicExch(p.status, (int)kErrBounds);
            t = 0;
          }
          src[h] = p.x + (int64_t)(t / p.k) * p.x_ld + piece * 8;
        }
      }
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&bars->empty[s], ((it / C::STAGES) & 1) ^ 1, p.status)) give_up();
        if (__any_sync(0xffffffffu, *abort)) break;
        const uint32_t b = smem_u32(smem + s * C::STAGE) + A_BYTES + r0 * 128 + ((piece ^ (r0 & 7)) << 4);
        const bool in = kb * BK + piece * 8 < p.K;
#pragma unroll
        for (int h = 0; h < EACH; ++h)
          if (src[h]) cp_async16(b + h * 2048, in ? src[h] + kb * BK : src[h], in);
        cp_async_arrive(&bars->picked[s]);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if (PAIR) cluster_sync();                                // the pair's MMAs and arrivals are done
  if (warp == 1) {
    tc_fence_after();
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM) : "memory");
    else
      tmem_dealloc(tmem, C::TMEM);
  }
  if constexpr (SPLIT) {
    cluster_sync();                                        // every CTA's sums are staged
    if (unit < items && warp >= EPI0 && warp < EPI0 + 4 && !*abort) {
      const Item q = item_of(p, unit, blocks, p.tile, SPAN, tiles, starts);
      const int tid = threadIdx.x - 32 * EPI0;
      float* sums = reinterpret_cast<float*>(smem);        // stage memory, which no load uses any more
      // rows share, share + splits, ... of the tile: the CTAs' sums in their order
      for (int c = share; c < q.rows; c += splits) {
        const int at = c * SUM_LD + sum_pos(SWIGLU, tid);
        float sum = 0.f;
        for (int r = 0; r < splits; ++r) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(st + at), r)));
          sum += v;
        }
        sums[at] = sum;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int c = share; c < q.rows; c += splits) store_row<SWIGLU>(p, q, sums + c * SUM_LD, c, tid);
    }
    cluster_sync();                                        // the other CTAs have read this one's sums
  }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
template <typename... A>
void launch(void (*kern)(A...), dim3 grid, int threads, dim3 cluster, size_t smem, cudaStream_t stream, A... args) {
  static std::mutex m;
  static std::map<std::pair<const void*, int>, bool> set;
  int dev;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  {
    const std::lock_guard<std::mutex> lock(m);
    bool& have = set[{(const void*)kern, dev}];
    if (!have) C10_CUDA_CHECK(cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    have = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster.x * cluster.y > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n++].val.clusterDim = {cluster.x, cluster.y, 1};
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args...));
}

int sm_count(int dev) {
  static std::mutex m;
  static std::map<int, int> have;
  const std::lock_guard<std::mutex> lock(m);
  int& n = have[dev];
  if (!n) C10_CUDA_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
  return n;
}

[[noreturn]] void refuse(const char* what) { refuse_value("linear_fused: ", what); }

// memory from a tensor's first to its last element
std::pair<uintptr_t, uintptr_t> extent(const torch::Tensor& t) {
  const uintptr_t a = (uintptr_t)t.data_ptr();
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {a, a + (last + 1) * t.element_size()};
}
bool overlap(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto x = extent(a), y = extent(b);
  return x.first < y.second && y.first < x.second;
}

template <int BN, bool PAIR, bool SPLIT>
void run(const Args& p, bool swiglu, const CUtensorMap& wm, const RowMaps& xm, dim3 grid, dim3 cluster, cudaStream_t stream) {
  launch(swiglu ? kernel<BN, true, PAIR, SPLIT> : kernel<BN, false, PAIR, SPLIT>, grid, threads(PAIR), cluster,
         Cfg<BN, PAIR, SPLIT>::SMEM, stream, p, wm, xm);
}

// How a product of R rows is cut: rows of a tile, CTA pairs or single CTAs, CTAs that share an item's K, items at most
struct Tiles {
  int tile;
  bool pair;
  unsigned splits;
  int64_t items;
};

Tiles tiles_of(int64_t R, int64_t E, int64_t W, int64_t K, bool swiglu, int sms) {
  const int64_t kb = (K + 63) / 64, half = swiglu ? 64 : 128;
  const auto blocks_of = [&](bool pair) { return (W + half * (pair ? 2 : 1) - 1) / (half * (pair ? 2 : 1)); };
  const auto items_of = [&](bool pair, int64_t tile) { return (std::min<int64_t>(E, R) + R / tile) * blocks_of(pair); };   // at most
  Tiles q = {16, false, 1, 0};
  // the height up to `most` that takes the fewest cycles: waves of items x (k blocks x the longer of loads, at some 60 bytes a
  // cycle and SM, and MMAs, 2 a row; start and end some 3000)
  const auto choose = [&](int most) {
    int64_t best = INT64_MAX;
    for (int t = 16; t <= most; t = t < 64 ? 2 * t : t + 32)
      for (int two = t >= 64 && R > 32; two >= (t > 64); --two) {
        const int64_t items = E == 1 ? (R + t - 1) / t * blocks_of(two) : items_of(two, t), units = two ? sms / 2 : sms;
        const int64_t rows = std::min<int64_t>(t, R), stage = std::max<int64_t>((16384 + rows * 128 / (two ? 2 : 1)) / 60, 2 * rows);
        const int64_t cost = (items + units - 1) / units * (kb * stage + 3000);
        if (cost < best) best = cost, q.tile = t, q.pair = two;
      }
  };
  if (E > 1) {
    // about twice the rows that an expert has on average, so that few experts need a second pass over their weights; above 64
    // rows CTA pairs, whose MMAs are cut to 32 rows.  Where that leaves SMs without an item, lower tiles by their cost (500 tokens,
    // 2 of 4 experts, 640 -> 700: 10.5 us, 15.8 on pairs)
    const int64_t want = 2 * ((R + E - 1) / E);
    q.tile = want <= 16 ? 16 : want <= 32 ? 32 : want <= 64 ? 64 : 256;
    q.pair = q.tile == 256;
    if (q.tile > 16 && items_of(q.pair, q.tile) < (q.pair ? sms / 2 : sms)) choose(q.tile);
  } else {
    choose(256);
  }
  q.items = items_of(q.pair, q.tile);
  // too few items for the SMs: clusters share the items' K, each CTA at least four 64-blocks
  if (q.tile == 16)
    while (q.splits < 8 && q.items * q.splits * 2 <= sms && kb / (q.splits * 2) >= 4) q.splits *= 2;
  return q;
}

}  // namespace lf

// The weights of a product [E, N, K] (models/layers.LinearBank checks them), with their tensor map
struct LinearBank {
  torch::Tensor w;
  c10::optional<torch::Tensor> bias;
  bool swiglu;
  torch::Tensor status;
  CUtensorMap wm;
  LinearBank(torch::Tensor w_, c10::optional<torch::Tensor> bias_, bool swiglu_, torch::Tensor status_)
      : w(w_), bias(bias_), swiglu(swiglu_), status(status_) {
    RAD_CHECK_VALUE(w.is_cuda() && w.dim() == 3 && w.is_contiguous() && w.scalar_type() == at::kBFloat16 && w.numel() > 0 &&
                          w.size(0) <= lf::MAX_E && w.size(2) % 8 == 0 && (!swiglu || w.size(1) % 2 == 0) &&
                          (uintptr_t)w.data_ptr() % 16 == 0,
                      "LinearBank: bf16 [E, N, K], contiguous, at most ", lf::MAX_E, " experts, K a multiple of 8");
    RAD_CHECK_VALUE(!bias.has_value() || (bias->device() == w.device() && bias->scalar_type() == at::kBFloat16 &&
                                            bias->is_contiguous() && bias->numel() == w.size(0) * w.size(1)),
                      "LinearBank: bias bf16 [E, N]");
    const cuuint64_t E = w.size(0), N = w.size(1), K = w.size(2), row = K * 2, half = N / 2;
    // (k, gate or up, feature, expert), or (k, feature, -, expert)
    const cuuint64_t dims[4] = {K, swiglu ? 2 : N, swiglu ? half : 1, E};
    const cuuint64_t strides[3] = {swiglu ? half * row : row, swiglu ? row : N * row, N * row};
    const cuuint32_t box[4] = {lf::BK, swiglu ? 2u : (cuuint32_t)lf::BM, swiglu ? (cuuint32_t)lf::BM / 2 : 1u, 1};
    const cuuint32_t each[4] = {1, 1, 1, 1};
    TORCH_CHECK(get_encode_tiled()(&wm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, w.data_ptr(), dims, strides, box, each,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
                "LinearBank: tensor map");
  }
};

// order / starts: the plan's, or none (one expert, x's rows in order); by_token: x [T, K] is picked by the plan's order
torch::Tensor linear_fused(const torch::Tensor& x, const LinearBank& bank, const c10::optional<torch::Tensor>& order,
                           const c10::optional<torch::Tensor>& starts, int64_t k, bool by_token,
                           const c10::optional<torch::Tensor>& scale, const c10::optional<torch::Tensor>& res,
                           const c10::optional<torch::Tensor>& out_) {
  using lf::refuse;
  const int64_t E = bank.w.size(0), N = bank.w.size(1), K = bank.w.size(2), W = bank.swiglu ? N / 2 : N;
  if (x.dim() != 2 || x.size(1) != K || x.scalar_type() != at::kBFloat16) refuse("x bf16 [rows, K]");
  if (x.device() != bank.w.device()) refuse("operands on one device");
  if (!starts.has_value() && (E != 1 || by_token)) refuse("the weights of several experts, or rows by token, need a plan");
  int64_t R = x.size(0);
  if (starts.has_value()) {
    if (starts->device() != x.device() || order->device() != x.device()) refuse("operands on one device");
    if (starts->numel() != E + 1) refuse("a plan of as many experts as weights");
    R = order->numel();
    if (k < 1 || R % k) refuse("a plan of whole tokens");
    if (x.size(0) != (by_token ? R / k : R)) refuse(by_token ? "one row of x per token of the plan" : "one row of x per row of the plan");
  }
  if (x.size(0) > 0 && ((K > 1 && x.stride(1) != 1) || (x.size(0) > 1 && (x.stride(0) < K || x.stride(0) % 8)) ||
                        (uintptr_t)x.data_ptr() % 16))
    refuse("rows of x contiguous and on 16 bytes");
  if (R >= (1ll << 31) - 256) refuse("rows");
  if (scale.has_value() && (scale->device() != x.device() || scale->scalar_type() != at::kFloat || scale->dim() != 1 ||
                            scale->size(0) != R || !scale->is_contiguous()))
    refuse("scale fp32 [rows]");
  const auto rows_of = [&](const torch::Tensor& t) {
    return t.dim() == 2 && t.size(0) == R && t.size(1) == W && t.scalar_type() == at::kBFloat16 && t.device() == x.device() &&
           (W <= 1 || t.stride(1) == 1);
  };
  if (res.has_value() && !rows_of(*res)) refuse("residual bf16, of the output's shape");
  if (out_.has_value() && (!rows_of(*out_) || (R > 1 && out_->stride(0) < W))) refuse("out bf16, of the output's shape");
  const at::cuda::CUDAGuard guard(x.device());
  torch::Tensor out = out_.has_value() ? *out_ : (torch::Tensor)at::detail::empty_cuda({R, W}, at::kBFloat16, x.device(), c10::nullopt);
  if (R == 0) return out;
  if (out_.has_value()) {
    const bool same = res.has_value() && res->data_ptr() == out.data_ptr() && res->stride(0) == out.stride(0);
    if (lf::overlap(out, x) || (res.has_value() && !same && lf::overlap(out, *res)))
      refuse("out overlaps x, or the residual other than being it");
  }
  lf::Args p = {};
  p.starts = starts.has_value() ? starts->data_ptr<int>() : nullptr;
  p.order = by_token ? order->data_ptr<int>() : nullptr;
  p.bias = bank.bias.has_value() ? (const __nv_bfloat16*)bank.bias->data_ptr() : nullptr;
  p.res = res.has_value() ? (const __nv_bfloat16*)res->data_ptr() : nullptr;
  p.scale = scale.has_value() ? scale->data_ptr<float>() : nullptr;
  p.out = (__nv_bfloat16*)out.data_ptr();
  p.res_ld = res.has_value() ? res->stride(0) : 0;
  p.out_ld = out.stride(0);
  p.x = (const __nv_bfloat16*)x.data_ptr();
  p.x_ld = x.stride(0);
  p.R = R; p.T = x.size(0); p.k = k; p.E = E; p.N = N; p.W = W; p.K = K;
  p.vec = ((uintptr_t)p.out | (uintptr_t)p.res) % 8 == 0 && (R == 1 || (p.out_ld | p.res_ld) % 4 == 0);   // one row's stride says nothing
  p.status = bank.status.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  const int sms = lf::sm_count(x.get_device());
  const lf::Tiles how = lf::tiles_of(R, E, W, K, bank.swiglu, sms);
  const bool pair = how.pair;
  const int64_t items = how.items;
  p.tile = how.tile;
  if (items >= (1ll << 30)) refuse("rows");
  const unsigned n = (unsigned)std::min<int64_t>(items, pair ? sms / 2 : sms);
  lf::RowMaps xm = {};
  if (!by_token)                                           // the boxes that a CTA's rows may take
    for (int i = 0; i < 4 && 16 << i <= (pair ? p.tile / 2 : p.tile); ++i)
      xm.box[i] = make_tma_2d(x.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, K, x.size(0), (x.size(0) == 1 ? K : x.stride(0)) * 2ll,
                              lf::BK, 16 << i, CU_TENSOR_MAP_SWIZZLE_128B);
  if (p.tile == 16) {
    if (how.splits > 1)
      lf::run<16, false, true>(p, bank.swiglu, bank.wm, xm, dim3((unsigned)items, how.splits), dim3(1, how.splits), stream);
    else lf::run<16, false, false>(p, bank.swiglu, bank.wm, xm, dim3(n), dim3(1), stream);
  } else if (pair) {
    lf::run<256, true, false>(p, bank.swiglu, bank.wm, xm, dim3(2 * n), dim3(2), stream);
  } else if (p.tile == 32) {
    lf::run<32, false, false>(p, bank.swiglu, bank.wm, xm, dim3(n), dim3(1), stream);
  } else {
    lf::run<64, false, false>(p, bank.swiglu, bank.wm, xm, dim3(n), dim3(1), stream);
  }
  return out;
}

void linear_fused_bind(pybind11::module_& m) {
  pybind11::class_<LinearBank>(m, "LinearBank")
      .def(pybind11::init<torch::Tensor, c10::optional<torch::Tensor>, bool, torch::Tensor>());
  m.def("linear_fused_tiles", [](int64_t R, int64_t E, int64_t W, int64_t K, bool swiglu, int sms) {
    RAD_CHECK_VALUE(R > 0 && E > 0 && W > 0 && K > 0 && sms > 1, "linear_fused_tiles: sizes above 0");
    const lf::Tiles q = lf::tiles_of(R, E, W, K, swiglu, sms);
    return std::make_tuple(q.tile, q.pair, q.splits);
  }, "(rows of a tile, CTA pairs, CTAs that share K) of a product of R rows on `sms` SMs");
  m.def("linear_fused", &linear_fused, "bf16 product (one weight, or one per expert) with bias, SwiGLU, row scale and residual");
}

}  // namespace rad
