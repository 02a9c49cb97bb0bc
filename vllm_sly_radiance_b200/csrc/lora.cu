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
  float* v;                 // [splits, T, S, Rp], by position
  int* status;
  int T, K, N, L, S, R, max_tiles;
  int Rp;                   // R rounded up to 16: row of v
  int splits;               // shares of K, one partial v each
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

// D[16 x 8] += A[16 x 16] B[16 x 8], bf16 with 32-bit sums
DEVI void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
DEVI uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// four e4m3 -> four bf16 (exact)
DEVI uint2 e4m3x4_to_bf16(uint32_t q) {
  const __half2_raw u = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q & 0xffff), __NV_E4M3);
  const __half2_raw w = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q >> 16), __NV_E4M3);
  const float2 f = __half22float2(__half2(u)), h = __half22float2(__half2(w));
  return make_uint2(pack2(f.x, f.y), pack2(h.x, h.y));
}

// elements k .. k + 7 of a row of K, as bf16, zero beyond K
template <bool FP8, bool VEC>
DEVI uint4 load8(const void* row, int k, int K) {
  if (VEC) {
    if (k >= K) return make_uint4(0, 0, 0, 0);
    if (FP8) {
      const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(row) + k);
      const uint2 u = e4m3x4_to_bf16(q.x), w = e4m3x4_to_bf16(q.y);
      return make_uint4(u.x, u.y, w.x, w.y);
    }
    return *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(row) + k);
  }
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int kk = k + 2 * i + e;
      f[e] = kk >= K ? 0.f
             : FP8   ? e4m3_to_f32(static_cast<const uint8_t*>(row)[kk])
                     : __bfloat162float(static_cast<const __nv_bfloat16*>(row)[kk]);
    }
    r[i] = pack2(f[0], f[1]);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// v, small tiles.  One CTA per (16 rank rows of a slice, share of K) and 16 rows at a time; its warps split the share.
// The adapter's rank rows are the 16-row operand of the MMA and the tokens its 8 columns.  Both operands go from global
// memory straight to registers: the sum over k has no order, so the four threads that share a rank row or a token each
// take 8 neighbouring k of a 32-block (16 bytes) and hand them to two MMAs in the same, permuted, order on both sides.
// The shares of K leave one partial v each; the expanding kernel adds them up in their order.
template <bool FP8, bool VEC>
__global__ void __launch_bounds__(256) shrink_kernel(const __grid_constant__ Args p) {
  __shared__ float red[8][16][20];                       // [warp][token][rank]
  pdl_wait();
  pdl_trigger();
  const int nt = min(p.plan[0], p.max_tiles), warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int groups = p.Rp / 16, s = blockIdx.y / groups, j0 = blockIdx.y % groups * 16;
  const int g = lane >> 2, k8 = (lane & 3) * 8;
  const int per = ((p.K + 31) / 32 + gridDim.z * 8 - 1) / (gridDim.z * 8) * 32;
  const int kb = (blockIdx.z * 8 + warp) * per, ke = min(kb + per, p.K);
  for (int i = blockIdx.x; i < nt; i += gridDim.x) {
    Tile t;
    if (!load_tile(p, i, t) || j0 >= t.rank) continue;   // uniform over the CTA
    const __nv_bfloat16* a = p.a + ((int64_t)(t.slot * p.S + s) * p.R + j0) * p.K;
    const bool u0 = j0 + g < t.rank, u1 = j0 + g + 8 < t.rank;
    for (int m0 = 0; m0 < t.rows; m0 += 16) {
      const uint8_t* x[2] = {nullptr, nullptr};
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (m0 + 8 * h + g < t.rows) {
          const int r = row_of(p, t.first + m0 + 8 * h + g);
          if (r >= 0) x[h] = static_cast<const uint8_t*>(p.x) + r * p.x_ld * (FP8 ? 1 : 2);
        }
      const bool two = m0 + 8 < t.rows;
      float c[2][4] = {};
#pragma unroll 4
      for (int k = kb; k < ke; k += 32) {
        const uint4 z = make_uint4(0, 0, 0, 0);
        const uint4 a0 = u0 ? load8<false, VEC>(a + (int64_t)g * p.K, k + k8, p.K) : z;
        const uint4 a1 = u1 ? load8<false, VEC>(a + (int64_t)(g + 8) * p.K, k + k8, p.K) : z;
        const uint4 x0 = x[0] ? load8<FP8, VEC>(x[0], k + k8, p.K) : z;
        mma_16816(c[0], a0.x, a1.x, a0.y, a1.y, x0.x, x0.y);
        mma_16816(c[0], a0.z, a1.z, a0.w, a1.w, x0.z, x0.w);
        if (two) {
          const uint4 x1 = x[1] ? load8<FP8, VEC>(x[1], k + k8, p.K) : z;
          mma_16816(c[1], a0.x, a1.x, a0.y, a1.y, x1.x, x1.y);
          mma_16816(c[1], a0.z, a1.z, a0.w, a1.w, x1.z, x1.w);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[warp][8 * h + 2 * (lane & 3) + (e & 1)][g + 8 * (e >> 1)] = c[h][e];
      __syncthreads();
      const int m = threadIdx.x / 16, j = threadIdx.x % 16;
      if (m0 + m < t.rows) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += red[w][m][j];
        const int pos = t.first + m0 + m;
        float f = p.scale[t.slot];
        if (FP8) {
          const int r = row_of(p, pos);
          f *= r >= 0 ? p.xs[r] : 0.f;
        }
        p.v[(((int64_t)blockIdx.z * p.T + pos) * p.S + s) * p.Rp + j0 + j] = v * f;
      }
      __syncthreads();
    }
  }
}

// 8 neighbouring features of a row from `at` on, those below ne
template <bool VEC>
DEVI uint4 load_y(const __nv_bfloat16* row, int at, int ne) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (row == nullptr || at >= ne) return v;
  if (VEC && at + 8 <= ne) return *reinterpret_cast<const uint4*>(row + at);
  for (int e = 0; e < 8; ++e)
    if (at + e < ne) reinterpret_cast<__nv_bfloat16*>(&v)[e] = row[at + e];
  return v;
}

// out = y + v B.  A warp takes 16 rows and steps over the features by 64.  The 8 columns of MMA m of a 32-feature block
// are the features 8 (c / 2) + 2 m + c % 2, so that each thread ends with 8 neighbouring features of two rows: y and out
// move in 16-byte vectors and nothing is staged; y of the next step is on its way during the MMAs of this one.  v is
// held as the sum of two bf16 numbers (its error is then 2^-16, not 2^-8), which doubles MMAs that wait on memory
// anyway.  MB: 16-row blocks of a tile, one per warp; with MB = 1 the warps take neighbouring features instead.  KBC:
// rank blocks of 16 whose v stays in registers; NS: steps of a warp.
template <int KBC, int MB, bool VEC>
__global__ void __launch_bounds__(256, 2) expand_kernel(const __grid_constant__ Args p) {
  constexpr int WN = 8 / MB, NS = MB == 1 ? 1 : 4, CH = 64 * NS * WN;      // CH: features of a CTA
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  int s = 0, ch = blockIdx.x;
  while (ch >= (p.off[s + 1] - p.off[s] + CH - 1) / CH) ch -= (p.off[s + 1] - p.off[s] + CH - 1) / CH, ++s;
  const int nb = p.off[s] + ch * CH + warp % WN * 64 * NS, ne = p.off[s + 1];
  const int nt = min(p.plan[0], p.max_tiles), mb = warp / WN * 16;
  bool first = true;
  for (int i = blockIdx.y; i < nt; i += gridDim.y) {
    Tile t;
    const bool ok = load_tile(p, i, t) && !(t.slot < 0 && p.out == p.y);
    for (int m0 = mb; ok && m0 < t.rows && nb < ne; m0 += 16 * MB) {
      const __nv_bfloat16* yr[2];
      __nv_bfloat16* to[2];
      uint4 y[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = m0 + 8 * h + g < t.rows ? row_of(p, t.first + m0 + 8 * h + g) : -1;
        yr[h] = r >= 0 ? p.y + r * p.y_ld : nullptr;
        to[h] = p.out + r * p.out_ld;
        // y was complete before the shrinking kernel started: it is read ahead of the wait for that kernel
#pragma unroll
        for (int n = 0; n < 2; ++n) y[n][h] = load_y<VEC>(yr[h], nb + 32 * n + 8 * q4, ne);
      }
      if (first) pdl_wait();
      first = false;
      uint32_t vh[KBC][4], vl[KBC][4];
#pragma unroll 1
      for (int st = 0; st < NS; ++st) {
        const int n0 = nb + 64 * st;
        if (n0 >= ne) break;
        uint4 yn[2][2];
        if (NS > 1 && st + 1 < NS) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) yn[n][h] = load_y<VEC>(yr[h], n0 + 64 + 32 * n + 8 * q4, ne);
        }
        float c[2][4][4] = {};
#pragma unroll 1
        for (int k0 = 0; k0 < t.rank; k0 += 16 * KBC) {
          if (st == 0 || t.rank > 16 * KBC) {
#pragma unroll
            for (int k = 0; k < KBC; ++k)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                if (m0 + 8 * h + g < t.rows && k0 + 16 * k < t.rank)
#pragma unroll 1
                  for (int z = 0; z < p.splits; ++z) {
                    const float4 w = *reinterpret_cast<const float4*>(
                        p.v + (((int64_t)z * p.T + t.first + m0 + 8 * h + g) * p.S + s) * p.Rp + k0 + 16 * k + 4 * q4);
                    f.x += w.x; f.y += w.y; f.z += w.z; f.w += w.w;
                  }
                const float u[4] = {f.x, f.y, f.z, f.w};
                float d[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  d[e] = u[e] - bf16_round(u[e]);
                  if (!(fabsf(d[e]) <= 3.4e38f)) d[e] = 0.f;   // infinities and NaN stay in the first number
                }
                vh[k][h] = pack2(u[0], u[1]); vh[k][h + 2] = pack2(u[2], u[3]);
                vl[k][h] = pack2(d[0], d[1]); vl[k][h + 2] = pack2(d[2], d[3]);
              }
          }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const int nn = n0 + 32 * n + 8 * (g >> 1) + 2 * m + (g & 1);
              const __nv_bfloat16* b = p.b + ((int64_t)t.slot * p.N + nn) * p.R + k0 + 4 * q4;
#pragma unroll
              for (int k = 0; k < KBC; ++k) {
                uint2 w = make_uint2(0, 0);
                const int left = t.rank - (k0 + 16 * k + 4 * q4);    // ranks beyond the adapter's own are not read
                if (nn < ne && left > 0) {
                  if (VEC) {                                         // R is a multiple of 4
                    w = *reinterpret_cast<const uint2*>(b + 16 * k);
                    if (left < 4) {
                      w.x &= left == 1 ? 0xffffu : ~0u;
                      w.y &= left == 3 ? 0xffffu : 0u;
                    }
                  } else {
#pragma unroll 1
                    for (int e = 0; e < min(left, 4); ++e)
                      (e < 2 ? w.x : w.y) |= (uint32_t)__bfloat16_as_ushort(b[16 * k + e]) << 16 * (e & 1);
                  }
                }
                mma_16816(c[n][m], vl[k][0], vl[k][1], vl[k][2], vl[k][3], w.x, w.y);
                mma_16816(c[n][m], vh[k][0], vh[k][1], vh[k][2], vh[k][3], w.x, w.y);
              }
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = n0 + 32 * n + 8 * q4;
            if (yr[h] == nullptr || at >= ne) continue;
            uint4 o = y[n][h];
            if (t.slot >= 0) {
              uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const __nv_bfloat162 f = *reinterpret_cast<const __nv_bfloat162*>(&w[m]);
                w[m] = pack2(__low2float(f) + c[n][m][2 * h], __high2float(f) + c[n][m][2 * h + 1]);
              }
            }
            if (VEC && at + 8 <= ne) *reinterpret_cast<uint4*>(to[h] + at) = o;
            else
              for (int e = 0; e < 8; ++e)
                if (at + e < ne) to[h][at + e] = reinterpret_cast<const __nv_bfloat16*>(&o)[e];
          }
        if (NS > 1) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) y[n][h] = yn[n][h];
        }
      }
    }
  }
  if (first) pdl_wait();
  pdl_trigger();
}

template <int KBC>
void launch_expand(const Args& p, bool tall, bool vec, unsigned tiles, cudaStream_t stream) {
  const int ch = tall ? 256 : 512;
  unsigned chunks = 0;
  for (int s = 0; s < p.S; ++s) chunks += (p.off[s + 1] - p.off[s] + ch - 1) / ch;
  auto k = tall ? (vec ? expand_kernel<KBC, 8, true> : expand_kernel<KBC, 8, false>)
                : (vec ? expand_kernel<KBC, 1, true> : expand_kernel<KBC, 1, false>);
  C10_CUDA_CHECK(launch_pdl(k, dim3(chunks, tiles), dim3(256), 0, stream, p));
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
  lora::Args p;
  p.x = x.data_ptr(); p.xs = fp8 ? xs.data_ptr<float>() : nullptr; p.x_ld = x.stride(0);
  p.a = (const __nv_bfloat16*)a.data_ptr(); p.b = (const __nv_bfloat16*)b.data_ptr();
  p.scale = scale.data_ptr<float>(); p.rank = ranks.data_ptr<int>();
  p.y = (const __nv_bfloat16*)y.data_ptr(); p.y_ld = y.stride(0);
  p.out = (__nv_bfloat16*)out.data_ptr(); p.out_ld = out.stride(0);
  p.plan = plan.data_ptr<int>(); p.status = status.data_ptr<int>();
  p.T = T; p.K = K; p.N = N; p.L = L; p.S = S; p.R = R; p.max_tiles = max_tiles;
  p.Rp = (R + 15) / 16 * 16;
  for (int s = 0; s <= S; ++s) p.off[s] = slices[s];
  auto stream = at::cuda::getCurrentCUDAStream();
  const unsigned tiles = std::min<int64_t>(max_tiles, 4096);
  // few tiles: shares of K over several CTAs, at least two 32-blocks a warp
  const int64_t ctas = tiles * S * (p.Rp / 16);
  p.splits = std::max<int64_t>(1, std::min<int64_t>({8, 148 / ctas, K / 512}));
  // v from the allocator, not a shared workspace: calls on several streams must not meet in it
  torch::Tensor ws = torch::empty({(int64_t)p.splits * T * S * p.Rp}, scale.options());
  p.v = ws.data_ptr<float>();
  const bool vec_k = K % 8 == 0 && p.x_ld % 8 == 0 && (uintptr_t)p.x % 16 == 0 && (uintptr_t)p.a % 16 == 0;
  bool vec_n = R % 4 == 0 && p.y_ld % 8 == 0 && p.out_ld % 8 == 0 &&
               ((uintptr_t)p.y | (uintptr_t)p.out | (uintptr_t)p.b) % 16 == 0;
  for (int s = 0; s < S; ++s) vec_n = vec_n && slices[s] % 8 == 0;
  auto shrink = fp8 ? (vec_k ? lora::shrink_kernel<true, true> : lora::shrink_kernel<true, false>)
                    : (vec_k ? lora::shrink_kernel<false, true> : lora::shrink_kernel<false, false>);
  C10_CUDA_CHECK(launch_pdl(shrink, dim3(tiles, S * p.Rp / 16, p.splits), dim3(256), 0, stream, p));
  const bool tall = tile_rows > 16;
  if (p.Rp <= 16) lora::launch_expand<1>(p, tall, vec_n, tiles, stream);
  else if (p.Rp <= 32) lora::launch_expand<2>(p, tall, vec_n, tiles, stream);
  else lora::launch_expand<4>(p, tall, vec_n, tiles, stream);
}

}  // namespace rad
