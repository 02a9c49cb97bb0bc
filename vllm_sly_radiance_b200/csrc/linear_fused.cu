// bf16 product with an epilogue, of one weight or of one weight per expert (rows sorted by expert, moe.cu's plan):
//
//   y[r]   = x[row(r)] W[e(r)]^T + b[e(r)]          K products of bf16 numbers, exact and summed in 32 bits
//   out[r] = res[r] + scale[r] * act(y[r])          act: y, or SwiGLU of y = [g | u]: g / (1 + exp(-g)) * u
//
// rounded once.  An output tile is 128 weight rows (the MMA's M) of one expert x up to BN of its rows (N).  With SwiGLU the
// weight rows of a tile are 64 pairs of a gate row and its up row, which a TMA box over [.., 2, N / 2, ..] brings in this
// order, so that both factors of an output meet in one tile.  Rows that are picked by token come by TMA gather, four a load.
// Warp 0 fills the ring of 64-k stages, warp 1 issues the MMAs into one of two accumulators in tensor memory, four warps carry
// the other one out through shared memory, so that rows leave in 16-byte pieces.
#include <ATen/cuda/CUDAContext.h>
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

constexpr int BM = 128, BK = 64, THREADS = 192;
constexpr int A_BYTES = BM * BK * 2;
constexpr int OUT_COLS = 32;                               // rows of out that are staged at a time
constexpr int OUT_LD = 144;                                // floats; the up half starts 16 banks behind the gate half
constexpr int SMEM_MAX = 227 * 1024;
constexpr int MAX_E = 1024;

struct Args {
  const int* starts;                                       // [E + 1] rows of the experts; null: one expert, R rows
  const int* order;                                        // [R] pair of a row, pair / k is its token; null: rows of x in order
  const __nv_bfloat16* bias;                               // [E, N]
  const __nv_bfloat16* res;
  const float* scale;
  __nv_bfloat16* out;
  int64_t res_ld, out_ld;
  int R, T, k, E, N, W, K;                                 // W: width of out (N, or N / 2 with SwiGLU)
  bool swiglu, vec;
  int* status;
};

template <int BN> struct Cfg {
  static constexpr int B_BYTES = BN * BK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int OUT = (BN < OUT_COLS ? BN : OUT_COLS) * OUT_LD * 4;
  static constexpr int META = 2048 + 2 * (MAX_E + 1) * 4;
  static constexpr int STAGES = (SMEM_MAX - 1024 - OUT - META) / STAGE;
  static constexpr int SMEM = 1024 + STAGES * STAGE + OUT + META;
  static constexpr int TMEM = 2 * BN < 32 ? 32 : 2 * BN;
};

struct Bars {
  uint64_t full[16], empty[16], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int abort;
};

struct Item {
  int e, n0, row0, rows;                                   // weight block (out's first feature), rows of out
};

DEVI uint32_t idesc_bf16(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
DEVI void tma_2d(uint32_t dst, const void* map, uint64_t* bar, int c, int r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c), "r"(r)
      : "memory");
}
DEVI void tma_4d(uint32_t dst, const void* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// four rows of a 2-D map by number, one after another
DEVI void tma_gather4(uint32_t dst, const void* map, uint64_t* bar, int c, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w)
      : "memory");
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

// Staged sums st [columns][OUT_LD] (raw, position of a weight row in a column: out_pos) of `n` staged columns -> rows of out
DEVI int out_pos(bool swiglu, int row) { return swiglu ? (row & 1) * 80 + row / 2 : row; }

DEVI void store_rows(const Args& p, const Item& q, const float* st, int c0, int n, int tid) {
  const int span = p.swiglu ? BM / 2 : BM, vecs = span / 8;
  const int v = tid % vecs, f = q.n0 + v * 8;
  if (f >= p.W) return;
  const bool whole = p.vec && f + 8 <= p.W;
  float b[8], bu[8];
  if (p.bias) {
    const __nv_bfloat16* bp = p.bias + (int64_t)q.e * p.N;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      b[i] = f + i < p.W ? __bfloat162float(bp[f + i]) : 0.f;
      if (p.swiglu) bu[i] = f + i < p.W ? __bfloat162float(bp[p.W + f + i]) : 0.f;
    }
  }
  for (int c = tid / vecs; c < n; c += 128 / vecs) {
    const int64_t r = q.row0 + c0 + c;
    const float4* s = reinterpret_cast<const float4*>(st + c * OUT_LD + v * 8);
    float y[8];
    *reinterpret_cast<float4*>(y) = s[0];
    *reinterpret_cast<float4*>(y + 4) = s[1];
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += b[i];
    }
    if (p.swiglu) {
      float u[8];
      *reinterpret_cast<float4*>(u) = s[20];
      *reinterpret_cast<float4*>(u + 4) = s[21];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (p.bias) u[i] += bu[i];
        y[i] = __fdividef(y[i], 1.f + __expf(-y[i])) * u[i];
      }
    }
    if (p.scale) {
      const float a = p.scale[r];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= a;
    }
    __nv_bfloat16* out = p.out + r * p.out_ld + f;
    const __nv_bfloat16* res = p.res + r * p.res_ld + f;
    if (whole) {
      uint4 o;
      __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(&o);
      if (p.res) {
        const uint4 a = *reinterpret_cast<const uint4*>(res);
        const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] += __bfloat162float(x[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = __float2bfloat16_rn(y[i]);
      *reinterpret_cast<uint4*>(out) = o;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (f + i < p.W) out[i] = __float2bfloat16_rn(p.res ? y[i] + __bfloat162float(res[i]) : y[i]);
    }
  }
}

// SPLIT: a cluster shares one item's K; its CTAs' sums meet through distributed shared memory, each CTA adds up and stores some
// of the rows.  Otherwise one CTA an SM runs every gridDim.x-th item.
template <int BN, bool SPLIT>
__global__ void __launch_bounds__(THREADS) kernel(const __grid_constant__ Args p, const __grid_constant__ CUtensorMap wm,
                                                  const __grid_constant__ CUtensorMap xm) {
  using C = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* st = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE);
  Bars* bars = reinterpret_cast<Bars*>(smem + C::STAGES * C::STAGE + C::OUT);
  int* tiles = reinterpret_cast<int*>(smem + C::STAGES * C::STAGE + C::OUT + 2048);
  int* starts = tiles + MAX_E + 1;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int splits = SPLIT ? gridDim.y : 1;
  const int rank = SPLIT ? blockIdx.y : 0;
  const int span = p.swiglu ? BM / 2 : BM, blocks = (p.W + span - 1) / span;
  const int all_k = (p.K + BK - 1) / BK;
  const int k0 = (int)((int64_t)all_k * rank / splits), k1 = (int)((int64_t)all_k * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 1);
    }
    bars->abort = 0;
    fence_mbar_init();
    tma_prefetch_desc(&wm);
    tma_prefetch_desc(&xm);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem, C::TMEM);
    tmem_relinquish();
  }
  pdl_wait();
  for (int e = threadIdx.x; e <= p.E; e += THREADS) starts[e] = p.starts ? p.starts[e] : e ? p.R : 0;
  __syncthreads();
  if (warp == 2) count_tiles(p, BN, tiles, starts, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();                                           // this block holds its tensor memory
  const uint32_t tmem = bars->tmem;
  const int items = tiles[p.E] * blocks;
  volatile int* abort = &bars->abort;
  bool mine = (int)blockIdx.x < items;                     // SPLIT: this cluster has an item

  if (warp == 0) {
    uint32_t it = 0;
    for (int i = blockIdx.x; i < items; i += gridDim.x) {
      if (__any_sync(0xffffffffu, *abort)) break;          // the same answer in all lanes
      const Item q = item_of(p, i, blocks, BN, span, tiles, starts);
      const bool ok = q.row0 >= 0 && q.rows > 0 && q.row0 + q.rows <= p.R;
      // loads of the rows: four by number, or boxes of 16
      const int each = p.order ? 4 : 16, loads = ok ? (q.rows + each - 1) / each : 0;
      int4 rows[2];
      if (p.order) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int r[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = (lane + 32 * h) * 4 + j;
            r[j] = ok && c < q.rows ? p.order[q.row0 + c] : 0;
            if (r[j] < 0 || r[j] >= (int64_t)p.T * p.k) {
              atomicExch(p.status, (int)kErrBounds);
              r[j] = 0;
            }
            r[j] /= p.k;
          }
          rows[h] = make_int4(r[0], r[1], r[2], r[3]);
        }
      }
      if (!ok) {
        if (lane == 0) atomicExch(p.status, (int)kErrBounds);
        *abort = 1;
        break;
      }
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int s = it % C::STAGES;
        if (!mbar_wait(&bars->empty[s], ((it / C::STAGES) & 1) ^ 1, p.status)) *abort = 1;
        if (__any_sync(0xffffffffu, *abort)) break;
        const uint32_t a = smem_u32(smem + s * C::STAGE), b = a + A_BYTES;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->full[s], A_BYTES + loads * each * BK * 2);
          if (p.swiglu) tma_4d(a, &wm, &bars->full[s], kb * BK, 0, q.n0, q.e);
          else tma_4d(a, &wm, &bars->full[s], kb * BK, q.n0, 0, q.e);
        }
        __syncwarp();
        if (p.order) {
          if (lane < loads) tma_gather4(b + lane * 512, &xm, &bars->full[s], kb * BK, rows[0]);
          if (lane + 32 < loads) tma_gather4(b + (lane + 32) * 512, &xm, &bars->full[s], kb * BK, rows[1]);
        } else if (lane < loads) {
          tma_2d(b + lane * 2048, &xm, &bars->full[s], kb * BK, q.row0 + lane * 16);
        }
      }
    }
    // given up: the loads in flight land before the block leaves
    if (*abort)
      for (uint32_t j = it > C::STAGES ? it - C::STAGES : 0; j < it; ++j)
        mbar_wait(&bars->full[j % C::STAGES], (j / C::STAGES) & 1, p.status);
  } else if (warp == 1) {
    if (elect_one()) {
      uint32_t it = 0, n = 0;
      for (int i = blockIdx.x; i < items && !*abort; i += gridDim.x, ++n) {
        const Item q = item_of(p, i, blocks, BN, span, tiles, starts);
        const int ab = n & 1;
        if (!mbar_wait(&bars->acc_empty[ab], ((n >> 1) & 1) ^ 1, p.status)) { *abort = 1; break; }
        tc_fence_after();
        const uint32_t idesc = idesc_bf16((q.rows + 15) / 16 * 16);
        bool ok = true;
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int s = it % C::STAGES;
          if (!mbar_wait(&bars->full[s], (it / C::STAGES) & 1, p.status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a = smem_u32(smem + s * C::STAGE), b = a + A_BYTES;
#pragma unroll
          for (int j = 0; j < BK / 16; ++j)
            mma_f16(tmem + ab * BN, sdesc_sw128(a + j * 32), sdesc_sw128(b + j * 32), idesc, kb > k0 || j > 0);
          mma_commit(&bars->empty[s]);
        }
        if (!ok) { *abort = 1; break; }
        mma_commit(&bars->acc_full[ab]);
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3, tid = threadIdx.x - 64, pos = out_pos(p.swiglu, quad * 32 + lane);
    uint32_t n = 0;
    for (int i = blockIdx.x; i < items; i += gridDim.x, ++n) {
      const Item q = item_of(p, i, blocks, BN, span, tiles, starts);
      const int ab = n & 1;
      const bool got = mbar_wait(&bars->acc_full[ab], (n >> 1) & 1, p.status);
      if (!got) *abort = 1;
      if (bar_sync_or(1, 128, *abort != 0)) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + ab * BN;
      for (int c0 = 0; c0 < q.rows; c0 += OUT_COLS) {
        const int cols = min(OUT_COLS, q.rows - c0);
        for (int c = 0; c < cols; c += 16) {
          uint32_t r[16];
          tmem_ld_32x32b_x16(acc + c0 + c, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) st[(c + j) * OUT_LD + pos] = __uint_as_float(r[j]);
        }
        if (c0 + OUT_COLS >= q.rows) tc_fence_before();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (c0 + OUT_COLS >= q.rows && tid == 0) mbar_arrive(&bars->acc_empty[ab]);
        if (!SPLIT) {
          store_rows(p, q, st, c0, cols, tid);
          asm volatile("bar.sync 1, 128;" ::: "memory");
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
  if constexpr (SPLIT) {
    cluster_sync();                                        // every CTA's sums are staged
    if (mine && warp >= 2 && !*abort) {
      const Item q = item_of(p, blockIdx.x, blocks, BN, span, tiles, starts);
      const int tid = threadIdx.x - 64;
      // rows rank, rank + splits, ... of the tile: add up the other CTAs' sums in their order
      for (int c = rank; c < q.rows; c += splits) {
        const uint32_t at = smem_u32(st + c * OUT_LD + out_pos(p.swiglu, tid));
        float sum = 0.f;
        for (int r = 0; r < splits; ++r) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(at, r)));
          sum += v;
        }
        // into the stage memory, which no load uses any more
        reinterpret_cast<float*>(smem)[c * OUT_LD + out_pos(p.swiglu, tid)] = sum;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int c = rank; c < q.rows; c += splits) store_rows(p, q, reinterpret_cast<float*>(smem) + c * OUT_LD, c, 1, tid);
    }
    cluster_sync();                                        // the other CTAs have read this one's sums
  }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
template <typename... A>
void launch(void (*kern)(A...), dim3 grid, int cluster_y, size_t smem, cudaStream_t stream, A... args) {
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
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster_y > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n++].val.clusterDim = {1, (unsigned)cluster_y, 1};
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

template <int BN>
void run(const Args& p, const CUtensorMap& wm, const CUtensorMap& xm, int64_t items, int sms, cudaStream_t stream) {
  launch(kernel<BN, false>, dim3((unsigned)std::min<int64_t>(items, sms)), 1, Cfg<BN>::SMEM, stream, p, wm, xm);
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
  torch::Tensor out = out_.has_value() ? *out_ : torch::empty({R, W}, x.options());
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
  p.R = R; p.T = x.size(0); p.k = k; p.E = E; p.N = N; p.W = W; p.K = K;
  p.swiglu = bank.swiglu;
  // one row's stride says nothing
  p.vec = ((uintptr_t)p.out | (uintptr_t)p.res) % 16 == 0 && (R == 1 || (p.out_ld | p.res_ld) % 8 == 0);
  p.status = bank.status.data_ptr<int>();
  const CUtensorMap xm = make_tma_2d(x.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, K, x.size(0),
                                     (x.size(0) == 1 ? K : x.stride(0)) * 2ll, lf::BK, by_token ? 1 : 16,
                                     CU_TENSOR_MAP_SWIZZLE_128B);
  auto stream = at::cuda::getCurrentCUDAStream();
  const int sms = lf::sm_count(x.get_device());
  // Tile height: about twice the rows that an expert has on average, so that few experts need a second pass over their weights
  const int64_t avg = (R + E - 1) / E, want = E == 1 ? R : 2 * avg;
  const int bn = want <= 16 ? 16 : want <= 32 ? 32 : want <= 64 ? 64 : want <= 128 ? 128 : 256;
  const int span = bank.swiglu ? 64 : 128;
  const int64_t blocks = (W + span - 1) / span, items = (std::min<int64_t>(E, R) + R / bn) * blocks;   // at most
  if (items >= (1ll << 31)) refuse("rows");
  if (bn == 16) {
    // too few items for the SMs: clusters share the items' K, each CTA at least four 64-blocks
    int splits = 1;
    const int64_t kb = (K + 63) / 64;
    while (splits < 8 && items * splits * 2 <= sms && kb / (splits * 2) >= 4) splits *= 2;
    if (splits > 1) {
      lf::launch(lf::kernel<16, true>, dim3((unsigned)items, splits), splits, lf::Cfg<16>::SMEM, stream, p, bank.wm, xm);
      return out;
    }
  }
  switch (bn) {
    case 16: lf::run<16>(p, bank.wm, xm, items, sms, stream); break;
    case 32: lf::run<32>(p, bank.wm, xm, items, sms, stream); break;
    case 64: lf::run<64>(p, bank.wm, xm, items, sms, stream); break;
    case 128: lf::run<128>(p, bank.wm, xm, items, sms, stream); break;
    default: lf::run<256>(p, bank.wm, xm, items, sms, stream);
  }
  return out;
}

void linear_fused_bind(pybind11::module_& m) {
  pybind11::class_<LinearBank>(m, "LinearBank")
      .def(pybind11::init<torch::Tensor, c10::optional<torch::Tensor>, bool, torch::Tensor>());
  m.def("linear_fused", &linear_fused, "bf16 product (one weight, or one per expert) with bias, SwiGLU, row scale and residual");
}

}  // namespace rad
