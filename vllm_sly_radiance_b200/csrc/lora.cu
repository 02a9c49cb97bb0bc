// Low-rank adapters of many requests beside a shared projection.
//
//   v[t, s, j] = x[t, :] . A[l, s, j, :]                                  j < rank[l]
//   out[t, n]  = y[t, n] + scale[l] * sum_j v[t, s(n), j] * B[l, n, j]    l = slot of row t, or y[t, n] for none
//
// x: bf16 rows, or e4m3 rows with one fp32 scale each (the pair a W4A8 linear takes).  A [L, S, R, K], B [L, N, R]
// bf16; s(n) is the part of a merged projection that output feature n belongs to.  The rows come sorted by adapter in
// tiles of one adapter each (the plan); a tile of rows without an adapter only carries y over when out is not y.
//
// plan (int32): [0] tiles in use, [4 ...] (slot, first position, rows, 0) per tile, then the row of each position.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"

namespace rad {
namespace lora {

constexpr int MAX_S = 8;

struct Args {
  const void* x;            // bf16 or e4m3 [T, K]
  const float* xs;          // e4m3: row scales
  int64_t x_ld;
  const __nv_bfloat16* a;   // [L, S, R, K]
  const __nv_bfloat16* b;   // [L, N, R]
  const float* scale;       // [L]
  const int* rank;          // [L]
  const __nv_bfloat16* y;
  int64_t y_ld;
  __nv_bfloat16* out;
  int64_t out_ld;
  const int* plan;
  float* v;                 // [T, S, R], by position
  int* status;
  int T, K, N, L, S, R, max_tiles;
  int off[MAX_S + 1];       // slice s = output features [off[s], off[s + 1])
};

struct Tile { int slot, first, rows, rank; };

DEVI bool load_tile(const Args& p, int i, Tile& t) {
  const int4 q = reinterpret_cast<const int4*>(p.plan + 4)[i];
  t.slot = q.x; t.first = q.y; t.rows = q.z; t.rank = 0;
  if (q.x >= p.L || q.y < 0 || q.z < 0 || q.y > p.T - q.z) {      // a plan of other rows or adapters: refused
    if (threadIdx.x == 0) atomicExch(p.status, (int)kErrBounds);
    return false;
  }
  if (q.x >= 0) t.rank = min(max(p.rank[q.x], 0), p.R);
  return true;
}
DEVI const int* perm(const Args& p) { return p.plan + 4 + 4 * p.max_tiles; }
DEVI int row_of(const Args& p, int pos) {
  const int r = perm(p)[pos];
  if (r < 0 || r >= p.T) { atomicExch(p.status, (int)kErrBounds); return -1; }
  return r;
}

template <bool FP8>
DEVI float load_x(const Args& p, int64_t row, int k) {
  if (FP8) return e4m3_to_f32(static_cast<const uint8_t*>(p.x)[row * p.x_ld + k]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p.x)[row * p.x_ld + k]);
}

// one warp per (row, slice, rank index) of a tile
template <bool FP8>
__global__ void __launch_bounds__(256) shrink_kernel(const __grid_constant__ Args p) {
  pdl_wait();
  pdl_trigger();
  const int nt = min(p.plan[0], p.max_tiles), lane = threadIdx.x & 31;
  for (int i = blockIdx.x; i < nt; i += gridDim.x) {
    Tile t;
    if (!load_tile(p, i, t) || t.slot < 0) continue;
    for (int w = blockIdx.y * 8 + threadIdx.x / 32; w < t.rows * p.S * p.R; w += gridDim.y * 8) {
      const int pos = t.first + w / (p.S * p.R), sj = w % (p.S * p.R);
      const int row = row_of(p, pos);
      if (row < 0 || sj % p.R >= t.rank) continue;
      const __nv_bfloat16* a = p.a + ((int64_t)t.slot * p.S * p.R + sj) * p.K;
      float acc = 0.f;
      for (int k = lane; k < p.K; k += 32) acc += load_x<FP8>(p, row, k) * __bfloat162float(a[k]);
      acc = warp_sum(acc);
      if (lane == 0)
        p.v[(int64_t)pos * p.S * p.R + sj] = acc * p.scale[t.slot] * (FP8 ? p.xs[row] : 1.f);
    }
  }
}

// one thread per output feature, the rows of the tile in turn
__global__ void __launch_bounds__(256) expand_kernel(const __grid_constant__ Args p) {
  pdl_wait();
  pdl_trigger();
  const int nt = min(p.plan[0], p.max_tiles), n = blockIdx.y * 256 + threadIdx.x;
  for (int i = blockIdx.x; i < nt; i += gridDim.x) {
    Tile t;
    if (!load_tile(p, i, t) || (t.slot < 0 && p.out == p.y)) continue;
    if (n >= p.N) continue;
    int s = 0;
    while (s + 1 < p.S && n >= p.off[s + 1]) ++s;
    const __nv_bfloat16* b = p.b + ((int64_t)max(t.slot, 0) * p.N + n) * p.R;
    for (int r = 0; r < t.rows; ++r) {
      const int row = row_of(p, t.first + r);
      if (row < 0) continue;
      const float* v = p.v + ((int64_t)(t.first + r) * p.S + s) * p.R;
      float acc = 0.f;
      for (int j = 0; j < t.rank; ++j) acc += v[j] * __bfloat162float(b[j]);
      p.out[row * p.out_ld + n] = __float2bfloat16_rn(__bfloat162float(p.y[row * p.y_ld + n]) + acc);
    }
  }
}

}  // namespace lora

// x [T, K] bf16, or e4m3 with xs fp32 [T]; slices: S + 1 offsets from 0 to N; plan as described above with max_tiles
// tile entries; out may be y.
void lora_add(torch::Tensor y, torch::Tensor x, torch::Tensor xs, torch::Tensor a, torch::Tensor b,
              torch::Tensor scale, torch::Tensor ranks, std::vector<int64_t> slices,
              torch::Tensor plan, int64_t max_tiles, int64_t tile_rows, torch::Tensor out,
              torch::Tensor status) {
  const bool fp8 = x.scalar_type() == at::kFloat8_e4m3fn;
  const int64_t T = x.size(0), K = x.size(1), L = a.size(0), S = a.size(1), R = a.size(2), N = b.size(1);
  const at::cuda::CUDAGuard guard(x.device());
  // from the allocator, not a shared workspace: calls on several streams must not meet in it
  torch::Tensor ws = torch::empty({T, S, R}, scale.options());
  lora::Args p;
  p.x = x.data_ptr(); p.xs = fp8 ? xs.data_ptr<float>() : nullptr; p.x_ld = x.stride(0);
  p.a = (const __nv_bfloat16*)a.data_ptr(); p.b = (const __nv_bfloat16*)b.data_ptr();
  p.scale = scale.data_ptr<float>(); p.rank = ranks.data_ptr<int>();
  p.y = (const __nv_bfloat16*)y.data_ptr(); p.y_ld = y.stride(0);
  p.out = (__nv_bfloat16*)out.data_ptr(); p.out_ld = out.stride(0);
  p.plan = plan.data_ptr<int>(); p.v = ws.data_ptr<float>(); p.status = status.data_ptr<int>();
  p.T = T; p.K = K; p.N = N; p.L = L; p.S = S; p.R = R; p.max_tiles = max_tiles;
  for (int s = 0; s <= S; ++s) p.off[s] = slices[s];
  auto stream = at::cuda::getCurrentCUDAStream();
  const unsigned tiles = std::min<int64_t>(max_tiles, 4096);
  const dim3 gs(tiles, std::max<int64_t>(1, std::min<int64_t>(64, (tile_rows * S * R + 7) / 8)));
  C10_CUDA_CHECK(launch_pdl(fp8 ? lora::shrink_kernel<true> : lora::shrink_kernel<false>, gs, dim3(256), 0, stream, p));
  C10_CUDA_CHECK(launch_pdl(lora::expand_kernel, dim3(tiles, (N + 255) / 256), dim3(256), 0, stream, p));
}

}  // namespace rad
