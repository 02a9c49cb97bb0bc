// Low-rank adapters of many requests beside a shared projection.
//
//   v[t, s, j] = scale[l] * x[t, :] . A[l, s, j, :]                  j < rank[l], l = slot of row t
//   out[t, n]  = y[t, n] + sum_j v[t, s(n), j] * B[l, n, j]          or y[t, n] for a row without an adapter
//
// x: bf16 rows, or e4m3 rows with one fp32 scale each (the pair a W4A8 linear takes).  A [L, S, R, K], B [L, N, R]
// bf16; s(n) is the part of a merged projection that output feature n belongs to.  The rows come sorted by adapter in
// tiles of one adapter each (the plan): 16 rows a tile for decode batches, 128 for prompts.
//
// plan (int32), one list of 16-row and one of 128-row tiles: [0] tiles in use, [1] those of rows without an adapter, which come
// first; from word 4 (slot, rows, 1 if the rows are consecutive, 0) per tile; then the row numbers, 16 or 128 per tile.
//
// Three forms (times: 5120 -> 17408 features in two slices, B200):
//   decode_kernel           16-row tiles whose clusters all run at once: one launch.  Bound by its chain of latencies (plan,
//                           x and A, cluster, B): 6.2 us for one row of rank 16, 8.5 us for 8 rows of 8 adapters, where the
//                           two launches below took 10.9 and 11.4 us.
//   shrink16 + expand16     more 16-row tiles: two launches that overlap.  Bound by the same chain and, beyond some
//                           30 adapters, by instructions: 25 us for 64 rows of 24 adapters up to rank 32 (one launch in
//                           two waves: 43 us).
//   shrink128 + expand128   128-row tiles: tcgen05.  Bound by memory: 8192 rows, rank 64, shrink 30 us (x at 4.7 TB/s), expand
//                           115 us (y and out at 5.0 TB/s; a plain copy of tiles 64 features wide reaches 5.3 TB/s at best,
//                           since its 128-byte rows open a DRAM page each, against 6.4 TB/s in address order).
//                           On mma.sync the same products took 307 and 787 us.
//
// Rounding: products of bf16 (or e4m3) numbers are exact in the MMA and summed in 32 bits.  v enters the second product
// as the sum of two bf16 numbers, so that its error is 2^-16 and not 2^-8: the second half doubles MMAs that wait on
// memory anyway.  The result is rounded once.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <map>
#include <mutex>

#include "common.cuh"
#include "tma_host.h"

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
  float* v;                 // 16-row tiles: fp32 [splits, tile rows, S, Rp]; 128: bf16 [tile rows, S, 2, Rp]
  int* status;
  int T, K, N, L, S, R, max_tiles, tile_rows;
  int Rp;                   // R rounded up to 16: row of v
  int splits;               // shares of K
  int steps;                // feature steps of a CTA
  int off[MAX_S + 1];       // slice s = output features [off[s], off[s + 1])
};

struct Tile { int slot, rows, rank, seq; };

// Tile i < max_tiles.  False: not in use, or a plan of other rows or adapters (refused, status word).  The count and
// the record are read together.
DEVI bool load_tile(const Args& p, int i, Tile& t) {
  const int n = p.plan[0];
  const int4 q = *reinterpret_cast<const int4*>(p.plan + 4 + 4 * (int64_t)i);
  t.slot = q.x; t.rows = q.y; t.rank = 0; t.seq = q.z;
  if (i >= n) return false;
  if (q.x >= p.L || q.y < 0 || q.y > p.tile_rows || n > p.max_tiles) {
    if (threadIdx.x == 0) atomicExch(p.status, (int)kErrBounds);
    return false;
  }
  if (q.x >= 0) t.rank = min(max(p.rank[q.x], 0), p.R);
  return true;
}
// row number of row r of tile i (-1: beyond the tile, or refused); row_word: as stored, to be read ahead of the record
DEVI int row_word(const Args& p, int i, int r) {
  return p.plan[4 + 4 * (int64_t)p.max_tiles + (int64_t)i * p.tile_rows + r];
}
DEVI int check_row(const Args& p, int r, int rows, int v) {
  if (r >= rows) return -1;
  if (v < 0 || v >= p.T) {
    atomicExch(p.status, (int)kErrBounds);
    return -1;
  }
  return v;
}
DEVI int row_of(const Args& p, int i, int r, int rows) { return check_row(p, r, rows, row_word(p, i, r)); }
// slice of the CTA's `span` output features: -> first feature, end of the slice
DEVI int slice_of(const Args& p, int ch, int span, int& s, int& ne) {
  s = 0;
  while (ch >= (p.off[s + 1] - p.off[s] + span - 1) / span) ch -= (p.off[s + 1] - p.off[s] + span - 1) / span, ++s;
  ne = p.off[s + 1];
  return p.off[s] + ch * span;
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

// four 32-bit values of v as two bf16 numbers each: the second holds what the first rounds off (error 2^-16)
DEVI void split_v(float4 f, bool use, uint32_t& h0, uint32_t& h1, uint32_t& l0, uint32_t& l1) {
  const float u[4] = {use ? f.x : 0.f, use ? f.y : 0.f, use ? f.z : 0.f, use ? f.w : 0.f};
  float d[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    d[e] = u[e] - bf16_round(u[e]);
    if (!(fabsf(d[e]) <= 3.4e38f)) d[e] = 0.f;             // infinities and NaN stay in the first number
  }
  h0 = pack2(u[0], u[1]); h1 = pack2(u[2], u[3]);
  l0 = pack2(d[0], d[1]); l1 = pack2(d[2], d[3]);
}

// out = y + c for the 16 rows x 32 NB features of second_product (add: false, out = y)
template <int NB, bool VEC>
DEVI void store_step(__nv_bfloat16* const (&to)[2], const __nv_bfloat16* const (&yr)[2], const uint4 (&y)[NB][2],
                     const float (&c)[NB][4][4], int n0, int ne, bool add) {
  const int q4 = threadIdx.x & 3;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = n0 + 32 * n + 8 * q4;
      if (yr[h] == nullptr || at >= ne) continue;
      uint4 o = y[n][h];
      if (add) {
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
}

// ---------------------------------------------------------------------------------------------
// 16-row tiles
// ---------------------------------------------------------------------------------------------
// First product of one warp's share of k: the adapter's rank rows are the 16-row operand of the MMA and the tokens its 8
// columns.  Both operands go from global memory straight to registers: the sum over k has no order, so the four threads
// that share a rank row or a token each take 8 neighbouring k of a 32-block (16 bytes) and hand them to two MMAs in the
// same, permuted, order on both sides.  The warp's sums go to red[warp][token][rank].  JG: 16-row rank groups.
template <int JG> constexpr int RS = 16 * JG + 4;          // row of red: the fragment writes meet no bank twice

template <int JG, bool FP8, bool VEC>
DEVI void first_product(const Args& p, const __nv_bfloat16* a, const uint8_t* const (&x)[2], bool two, int ranks, int kb,
                        int ke, float* red) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  float c[JG][2][4] = {};
  // Up to rank 16 four blocks of k in flight and not two: 1 row 5.95 / 6.13 us and the mixed step of 4096 rows 104.4 / 105.6
  // with A from DRAM; with A in L2 61 single rows take 25.3 / 24.6.
#pragma unroll (JG == 1 ? 4 : 2)
  for (int k = kb; k < ke; k += 32) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    uint4 xa[2], aa[JG][2];
    xa[0] = x[0] ? load8<FP8, VEC>(x[0], k + 8 * q4, p.K) : z;
    xa[1] = two && x[1] ? load8<FP8, VEC>(x[1], k + 8 * q4, p.K) : z;
#pragma unroll
    for (int j = 0; j < JG; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int jr = 16 * j + 8 * h + g;
        aa[j][h] = jr < ranks ? load8<false, VEC>(a + (int64_t)jr * p.K, k + 8 * q4, p.K) : z;
      }
#pragma unroll
    for (int j = 0; j < JG; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (h == 0 || two) {
          mma_16816(c[j][h], aa[j][0].x, aa[j][1].x, aa[j][0].y, aa[j][1].y, xa[h].x, xa[h].y);
          mma_16816(c[j][h], aa[j][0].z, aa[j][1].z, aa[j][0].w, aa[j][1].w, xa[h].z, xa[h].w);
        }
  }
#pragma unroll
  for (int j = 0; j < JG; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(warp * 16 + 8 * h + 2 * q4 + (e & 1)) * RS<JG> + 16 * j + g + 8 * (e >> 1)] = c[j][h][e];
}
template <int JG>
DEVI float red_sum(const float* red, int o) {
  float f = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) f += red[(w * 16 + o / (16 * JG)) * RS<JG> + o % (16 * JG)];
  return f;
}

// B of NB 32-feature blocks and JG rank groups from rank k0 on, in the fragments' order: the 8 columns of MMA m of a block
// are the features 8 (c / 2) + 2 m + c % 2, so that each thread ends with 8 neighbouring features of two rows.  Ranks
// beyond the adapter's own count as zero.
template <int JG, int NB, bool VEC>
DEVI void load_b(const __nv_bfloat16* bt, int R, int n0, int ne, int k0, int rank, uint2 (&w)[NB][4][JG]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int nf = n0 + 8 * (g >> 1) + (g & 1), left0 = rank - k0 - 4 * q4;
  const __nv_bfloat16* b = bt + (int64_t)nf * R + k0 + 4 * q4;
  if (VEC && n0 + 32 * NB <= ne && rank - k0 >= 16 * JG) {               // nothing to leave out
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int k = 0; k < JG; ++k)
          w[n][m][k] = *reinterpret_cast<const uint2*>(b + (uint32_t)((32 * n + 2 * m) * R) + 16 * k);
    return;
  }
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int k = 0; k < JG; ++k) {
        const __nv_bfloat16* bk = b + (uint32_t)((32 * n + 2 * m) * R) + 16 * k;
        const int left = left0 - 16 * k;
        uint2 u = make_uint2(0, 0);
        if (nf + 32 * n + 2 * m < ne && left > 0) {
          if (VEC) {                                       // R is a multiple of 4
            u = *reinterpret_cast<const uint2*>(bk);
          } else {
#pragma unroll 1
            for (int e = 0; e < min(left, 4); ++e)
              (e < 2 ? u.x : u.y) |= (uint32_t)__bfloat16_as_ushort(bk[e]) << 16 * (e & 1);
          }
        }
        if (VEC && left < 4) {
          u.x &= left == 1 ? 0xffffu : ~0u;
          u.y &= left == 3 ? 0xffffu : 0u;
        }
        w[n][m][k] = u;
      }
}
// v [16][vs] in shared memory, JG rank groups from k0 on, as the two bf16 operands of the MMA
template <int JG>
DEVI void load_v(const float* v, int vs, int k0, int rank, int rows, uint32_t (&vh)[JG][4], uint32_t (&vl)[JG][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
#pragma unroll
  for (int k = 0; k < JG; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool use = 8 * h + g < rows && k0 + 16 * k < rank;
      const float4 f = use ? *reinterpret_cast<const float4*>(v + (8 * h + g) * vs + k0 + 16 * k + 4 * q4) : make_float4(0.f, 0.f, 0.f, 0.f);
      split_v(f, use, vh[k][h], vh[k][h + 2], vl[k][h], vl[k][h + 2]);
    }
}
// the MMAs of load_b's and load_v's operands
template <int JG, int NB>
DEVI void second_product(const uint32_t (&vh)[JG][4], const uint32_t (&vl)[JG][4], const uint2 (&w)[NB][4][JG], float (&c)[NB][4][4]) {
#pragma unroll
  for (int k = 0; k < JG; ++k)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        mma_16816(c[n][m], vl[k][0], vl[k][1], vl[k][2], vl[k][3], w[n][m][k].x, w[n][m][k].y);
        mma_16816(c[n][m], vh[k][0], vh[k][1], vh[k][2], vh[k][3], w[n][m][k].x, w[n][m][k].y);
      }
}

// features of a CTA's step: B of one step takes 16 registers, so that the next step's fits beside it (64 ranks at once spilled
// and took 31 us where 32 at a time take 26: 8 tiles of rank 64)
template <int JG> constexpr int NBS = JG == 1 ? 2 : 1;
template <int JG> constexpr int STEPF = 8 * 32 * NBS<JG>;

// all steps of a warp's features from n0 on (STEPF apart); y and w hold the first step's
template <int JG, bool VEC>
DEVI void expand_steps(const Args& p, const Tile& t, const __nv_bfloat16* bt, const float* v, int vs, int n0, int ne, int steps,
                       const __nv_bfloat16* const (&yr)[2], __nv_bfloat16* const (&to)[2], uint4 (&y)[NBS<JG>][2],
                       uint2 (&w)[NBS<JG>][4][JG]) {
  constexpr int NB = NBS<JG>;
  const int q4 = threadIdx.x & 3;
  uint32_t vh[JG][4], vl[JG][4];
  load_v<JG>(v, vs, 0, t.rank, t.rows, vh, vl);
#pragma unroll 1
  for (int st = 0; st < steps && n0 < ne; ++st, n0 += STEPF<JG>) {
    uint4 yn[NB][2];
    uint2 wn[NB][4][JG];
    const bool more = st + 1 < steps;
    if (more) {
      load_b<JG, NB, VEC>(bt, p.R, n0 + STEPF<JG>, ne, 0, t.rank, wn);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) yn[n][h] = load_y<VEC>(yr[h], n0 + STEPF<JG> + 32 * n + 8 * q4, ne);
    }
    float c[NB][4][4] = {};
    second_product<JG, NB>(vh, vl, w, c);
    if (t.rank > 16 * JG) {
#pragma unroll 1
      for (int k0 = 16 * JG; k0 < t.rank; k0 += 16 * JG) {
        uint32_t uh[JG][4], ul[JG][4];
        load_b<JG, NB, VEC>(bt, p.R, n0, ne, k0, t.rank, w);
        load_v<JG>(v, vs, k0, t.rank, t.rows, uh, ul);
        second_product<JG, NB>(uh, ul, w, c);
      }
    }
    store_step<NB, VEC>(to, yr, y, c, n0, ne, t.slot >= 0);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) y[n][h] = yn[n][h];
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int k = 0; k < JG; ++k) w[n][m][k] = wn[n][m][k];
    }
  }
}

// Both products in one launch.  A cluster of 8 CTAs owns (16 rows of one adapter, up to 8 x STEPF x steps features of one
// slice): its CTAs and their warps share K, add up v through distributed shared memory in a fixed order, and each CTA
// then expands its own features.  A's rows are read once per cluster (again from L2 where a slice takes several), B once.
constexpr int CL = 8;

template <int JG, bool FP8, bool VEC>
__global__ void __launch_bounds__(256, 2) decode_kernel(const __grid_constant__ Args p) {
  constexpr int NB = NBS<JG>, STEP = STEPF<JG>;
  extern __shared__ float sm[];
  float* red = sm;                                         // [8 warps][16 tokens][RS]
  float* part = red + 8 * 16 * RS<JG>;                     // [16][16 JG] this CTA's share of v
  float* v = part + 16 * 16 * JG;                          // [16][Rp + 4]
  const int vs = p.Rp + 4, i = blockIdx.y;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int cr = cluster_ctarank();
  int s, ne;
  const int nb = slice_of(p, blockIdx.x / CL, CL * STEP * p.steps, s, ne) + cr * STEP * p.steps + warp * 32 * NB;
  const int per = ((p.K + 31) / 32 + CL * 8 - 1) / (CL * 8) * 32;
  const int kb = (cr * 8 + warp) * per, ke = min(kb + per, p.K);
  pdl_wait();
  pdl_trigger();
  const int rw[2] = {row_word(p, i, g), row_word(p, i, 8 + g)};
  Tile t;
  if (!load_tile(p, i, t) || (t.slot < 0 && p.out == p.y)) return;         // uniform over the cluster
  const __nv_bfloat16* yr[2];
  __nv_bfloat16* to[2];
  const uint8_t* x[2];
  uint4 y[NB][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = check_row(p, 8 * h + g, t.rows, rw[h]);
    x[h] = r >= 0 ? static_cast<const uint8_t*>(p.x) + r * p.x_ld * (FP8 ? 1 : 2) : nullptr;
    yr[h] = r >= 0 ? p.y + r * p.y_ld : nullptr;
    to[h] = p.out + r * p.out_ld;
#pragma unroll
    for (int n = 0; n < NB; ++n) y[n][h] = load_y<VEC>(yr[h], nb + 32 * n + 8 * q4, ne);
  }
  const __nv_bfloat16* bt = p.b + (int64_t)max(t.slot, 0) * p.N * p.R;
  uint2 w[NB][4][JG];                                      // B of the first step, on its way during the first product
  load_b<JG, NB, VEC>(bt, p.R, nb, ne, 0, t.rank, w);
  for (int j0 = 0; j0 < t.rank; j0 += 16 * JG) {
    const __nv_bfloat16* a = p.a + ((int64_t)(t.slot * p.S + s) * p.R + j0) * p.K;
    first_product<JG, FP8, VEC>(p, a, x, t.rows > 8, t.rank - j0, kb, ke, red);
    if (j0) cluster_wait();                                // every share of the ranks before read
    __syncthreads();
#pragma unroll
    for (int o = threadIdx.x; o < 256 * JG; o += 256) part[o] = red_sum<JG>(red, o);
    cluster_sync();
#pragma unroll
    for (int o = threadIdx.x; o < 256 * JG; o += 256) {
      float f[CL], sum = 0.f;
#pragma unroll
      for (int c = 0; c < CL; ++c)
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[c]) : "r"(mapa_shared(smem_u32(part + o), c)));
#pragma unroll
      for (int c = 0; c < CL; ++c) sum += f[c];
      const int m = o / (16 * JG);
      sum *= p.scale[t.slot];
      if (FP8) {
        const int r = row_of(p, i, m, t.rows);
        sum *= r >= 0 ? p.xs[r] : 0.f;
      }
      // beyond the rank A counts as zero, and zero times an infinity of x is NaN
      const int j = j0 + o % (16 * JG);
      if (j < p.Rp) v[m * vs + j] = j < t.rank ? sum : 0.f;
    }
    cluster_arrive();
  }
  __syncthreads();
  expand_steps<JG, VEC>(p, t, bt, v, vs, nb, ne, p.steps, yr, to, y, w);
  if (t.rank > 0) cluster_wait();                          // the other CTAs have read this one's share
}

// v of 16-row tiles: one CTA per (tile, 16 JG rank rows of a slice, share of K).  The shares leave one partial v each, which
// the expanding kernel adds up in order.
template <int JG, bool FP8, bool VEC>
__global__ void __launch_bounds__(256) shrink16_kernel(const __grid_constant__ Args p) {
  __shared__ float red[8 * 16 * RS<JG>];
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x, groups = (p.Rp + 16 * JG - 1) / (16 * JG);
  const int s = blockIdx.y / groups, j0 = blockIdx.y % groups * 16 * JG;
  const int warp = threadIdx.x / 32, g = (threadIdx.x & 31) >> 2;
  const int rw[2] = {row_word(p, i, g), row_word(p, i, 8 + g)};
  Tile t;
  if (!load_tile(p, i, t) || j0 >= t.rank) return;         // uniform over the CTA
  const uint8_t* x[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = check_row(p, 8 * h + g, t.rows, rw[h]);
    x[h] = r >= 0 ? static_cast<const uint8_t*>(p.x) + r * p.x_ld * (FP8 ? 1 : 2) : nullptr;
  }
  const int per = ((p.K + 31) / 32 + p.splits * 8 - 1) / (p.splits * 8) * 32;
  const int kb = (blockIdx.z * 8 + warp) * per;
  first_product<JG, FP8, VEC>(p, p.a + ((int64_t)(t.slot * p.S + s) * p.R + j0) * p.K, x, t.rows > 8, t.rank - j0, kb,
                              min(kb + per, p.K), red);
  __syncthreads();
#pragma unroll
  for (int o = threadIdx.x; o < 256 * JG; o += 256) {
    const int m = o / (16 * JG), j = j0 + o % (16 * JG);
    if (m >= t.rows || j >= p.Rp) continue;
    float f = p.scale[t.slot];
    if (FP8) {
      const int r = row_of(p, i, m, t.rows);
      f *= r >= 0 ? p.xs[r] : 0.f;
    }
    p.v[(((int64_t)blockIdx.z * p.max_tiles + i) * 16 + m) * p.S * p.Rp + s * p.Rp + j] =
        j < t.rank ? red_sum<JG>(red, o) * f : 0.f;         // (zero times an infinity of x is NaN)
  }
}

// out of 16-row tiles.  B and y, which do not depend on v, are read ahead of the wait for the shrinking kernel: that kernel
// itself waited for whatever wrote them.
template <int JG, bool VEC>
__global__ void __launch_bounds__(256, 2) expand16_kernel(const __grid_constant__ Args p) {
  constexpr int NB = NBS<JG>;
  extern __shared__ float v[];                             // [16][Rp + 4]
  const int vs = p.Rp + 4, i = blockIdx.y;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  int s, ne;
  const int nb = slice_of(p, blockIdx.x, STEPF<JG> * p.steps, s, ne) + warp * 32 * NB;
  const int rw[2] = {row_word(p, i, g), row_word(p, i, 8 + g)};
  Tile t;
  if (!load_tile(p, i, t) || (t.slot < 0 && p.out == p.y)) {
    pdl_wait();
    return;
  }
  const __nv_bfloat16* yr[2];
  __nv_bfloat16* to[2];
  uint4 y[NB][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = check_row(p, 8 * h + g, t.rows, rw[h]);
    yr[h] = r >= 0 ? p.y + r * p.y_ld : nullptr;
    to[h] = p.out + r * p.out_ld;
#pragma unroll
    for (int n = 0; n < NB; ++n) y[n][h] = load_y<VEC>(yr[h], nb + 32 * n + 8 * q4, ne);
  }
  const __nv_bfloat16* bt = p.b + (int64_t)max(t.slot, 0) * p.N * p.R;
  uint2 w[NB][4][JG];
  load_b<JG, NB, VEC>(bt, p.R, nb, ne, 0, t.rank, w);
  pdl_wait();
  pdl_trigger();
  const int rk = (t.rank + 15) / 16 * 16;
  for (int o = threadIdx.x; o < t.rows * rk; o += 256) {
    const int m = o / rk, j = o % rk;
    const float* q = p.v + (((int64_t)i * 16 + m) * p.S + s) * p.Rp + j;
    float f[8], sum = 0.f;
#pragma unroll
    for (int z = 0; z < 8; ++z) f[z] = z < p.splits ? q[(int64_t)z * p.max_tiles * 16 * p.S * p.Rp] : 0.f;
#pragma unroll
    for (int z = 0; z < 8; ++z) sum += f[z];
    v[m * vs + j] = sum;
  }
  __syncthreads();
  expand_steps<JG, VEC>(p, t, bt, v, vs, nb, ne, p.steps, yr, to, y, w);
}

// ---------------------------------------------------------------------------------------------
// 128-row tiles
// ---------------------------------------------------------------------------------------------
DEVI void st_shared16(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
DEVI uint4 ld_shared16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}
// 16-byte chunk `c` of row `r` in an operand tile of 128-byte rows, 128-byte swizzle (tiles 1024-byte aligned)
DEVI uint32_t sw128(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }
// kind::f16 instruction descriptor: bf16 x bf16 -> fp32, both K-major, M = 128
DEVI uint32_t idesc_bf16(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// TMEM -> registers: 16 lanes x 32 columns; a thread gets columns 8 m + 2 (lane % 4) + {0, 1} of rows lane / 4 (r[4 m],
// r[4 m + 1]) and lane / 4 + 8 (r[4 m + 2], r[4 m + 3]), the order of the mma.sync accumulators
DEVI void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// TMA, four rows of a 2-D map by number: 4 x box width, rows one after another
DEVI void tma_gather4(uint32_t dst, const void* map, uint64_t* bar, int c, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w)
      : "memory");
}
DEVI void tma_2d(uint32_t dst, const void* map, uint64_t* bar, int c, int r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c), "r"(r)
      : "memory");
}
DEVI void tma_5d(uint32_t dst, const void* map, uint64_t* bar, int c, int r) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %4, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c), "r"(0), "r"(r)
      : "memory");
}
// K-major operand tile with rows of `rb` = 32, 64 or 128 bytes, swizzled over its rows' width
DEVI uint64_t sdesc_rows(uint32_t saddr, int rb) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;                                  // LBO, not used by swizzled K-major tiles
  d |= (uint64_t)((8 * rb) >> 4) << 32;                    // SBO: 8 rows
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)(rb == 128 ? 2 : rb == 64 ? 4 : 6) << 61;
  return d;
}
// byte offset of 16-byte chunk `c` of row `r` in such a tile
DEVI uint32_t sw_rows(int r, int c, int rb) {
  return (uint32_t)(r * rb + ((c ^ (rb == 128 ? r & 7 : rb == 64 ? r >> 1 & 3 : r >> 2 & 1)) << 4));
}
// Rows of a tile for TMA: consecutive rows in boxes of 16 (the last may reach into rows that nothing reads the results of),
// others four by number (those beyond the tile repeat the first).  `lane` has one load of a 64-column tile; n: loads in use.
struct TmaRows {
  int n, each;                                             // loads, and rows of one
  bool seq;
  int4 r;
};
DEVI TmaRows tma_rows(const Args& p, int i, const Tile& t, int lane) {
  TmaRows q;
  const int* rows = p.plan + 4 + 4 * (int64_t)p.max_tiles + (int64_t)i * 128;
  const int first = rows[0];
  q.seq = t.seq && first >= 0 && first <= p.T - t.rows;
  q.n = q.seq ? (t.rows + 15) / 16 : (t.rows + 3) / 4;
  q.each = q.seq ? 16 : 4;
  q.r = make_int4(first + 16 * lane, 0, 0, 0);
  if (q.seq || lane >= q.n) return q;
  q.r = *reinterpret_cast<const int4*>(rows + 4 * lane);
  if (4 * lane + 1 >= t.rows) q.r.y = q.r.x;
  if (4 * lane + 2 >= t.rows) q.r.z = q.r.x;
  if (4 * lane + 3 >= t.rows) q.r.w = q.r.x;
  if ((unsigned)q.r.x >= (unsigned)p.T || (unsigned)q.r.y >= (unsigned)p.T || (unsigned)q.r.z >= (unsigned)p.T ||
      (unsigned)q.r.w >= (unsigned)p.T) {
    atomicExch(p.status, (int)kErrBounds);
    q.r = make_int4(0, 0, 0, 0);
  }
  return q;
}
DEVI void tma_load_rows(const TmaRows& q, uint32_t dst, const void* box, const void* gather, uint64_t* bar, int c, int lane,
                        int row_bytes) {
  if (lane >= q.n) return;
  if (q.seq) tma_2d(dst + lane * 16 * row_bytes, box, bar, c, q.r.x);
  else tma_gather4(dst + lane * 4 * row_bytes, gather, bar, c, q.r);
}

// The sums of the cluster's CTAs (part [128][ld], column ss * R + j) -> v, as two bf16 numbers each.  Thread `tid` of 256.
template <bool FP8>
DEVI void write_v(const Args& p, int i, const Tile& t, const float* part, int ld, int sr0, int nsr, int tid) {
  const int ns = nsr / p.R, rk = p.Rp / 4, total = t.rows * ns * rk;
  __nv_bfloat16* v = reinterpret_cast<__nv_bfloat16*>(p.v);
  const float sc = p.scale[t.slot];
  // the CTAs take the rows in turn; a thread four neighbouring values of a row
  for (int o = tid + 256 * (p.splits > 1 ? blockIdx.z : 0); o < total; o += 256 * p.splits) {
    const int m = o / (ns * rk), ss = o / rk % ns, j = o % rk * 4;
    float f = sc;
    if (FP8) {
      const int r = row_of(p, i, m, t.rows);
      f *= r >= 0 ? p.xs[r] : 0.f;
    }
    const float* at = part + m * ld + ss * p.R + j;
    float q[4] = {};
    if (p.R % 4 == 0) {                                    // (then j + 3 < R too)
      float4 w[8];
#pragma unroll
      for (int z = 0; z < 8; ++z)                          // all CTAs' sums on their way together, added in order
        if (z < p.splits && j < p.R)
          w[z] = p.splits > 1 ? ld_dsmem_f4(mapa_shared(smem_u32(at), z)) : *reinterpret_cast<const float4*>(at);
#pragma unroll
      for (int z = 0; z < 8; ++z)
        if (z < p.splits && j < p.R) q[0] += w[z].x, q[1] += w[z].y, q[2] += w[z].z, q[3] += w[z].w;
    } else {
      for (int z = 0; z < p.splits; ++z)
        for (int e = 0; e < min(4, p.R - j); ++e) {
          float w = at[e];
          if (p.splits > 1)
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w) : "r"(mapa_shared(smem_u32(at + e), z)));
          q[e] += w;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = j + e < t.rank ? q[e] * f : 0.f;
    uint2 hi, lo;
    split_v(make_float4(q[0], q[1], q[2], q[3]), true, hi.x, hi.y, lo.x, lo.y);
    __nv_bfloat16* to = v + (((int64_t)i * 128 + m) * p.S + sr0 / p.R + ss) * 2 * p.Rp + j;
    *reinterpret_cast<uint2*>(to) = hi;
    *reinterpret_cast<uint2*>(to + p.Rp) = lo;
  }
}

// TMEM sums [128 x nc] -> part, by warp quadrant `wq` (32 rows) and column half `wh`
DEVI void sums_to_smem(uint32_t tmem, bool have, int nc, float* part, int ld, int wq, int wh) {
  const int row = wq * 32 + (threadIdx.x & 31);
  for (int c = wh * 16; c < nc; c += 32) {
    uint32_t r[16] = {};
    if (have) {
      tmem_ld_32x32b_x16(tmem + ((uint32_t)(wq * 32) << 16) + c, r);
      tmem_ld_wait();
    }
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<float4*>(part + row * ld + c + e) =
          make_float4(__uint_as_float(r[e]), __uint_as_float(r[e + 1]), __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
  }
}
DEVI uint32_t tmem_cols(int nc) { return nc <= 32 ? 32 : nc <= 64 ? 64 : nc <= 128 ? 128 : 256; }

// v of 128-row tiles: D[128 x NC] = X[128 x K] A[NC x K]^T on tcgen05, NC <= 256 rank rows of all slices together, so that x
// is read once.  Warp 0 fills a ring of 64-k stages by TMA, x row by row number; warp 1 issues the MMAs; e4m3 rows are
// widened to bf16 in shared memory by the other eight warps, which also carry the sums out.  A cluster of `splits` CTAs
// shares K and adds up through distributed shared memory in a fixed order.
constexpr int TH = 320;

template <bool FP8>
__global__ void __launch_bounds__(TH) shrink128_kernel(const __grid_constant__ Args p, const __grid_constant__ CUtensorMap xm,
                                                       const __grid_constant__ CUtensorMap xg, const __grid_constant__ CUtensorMap am,
                                                       int nc_max, int stages) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[8], empty[8], cfull[2], cempty[2], done;
  __shared__ uint32_t tmem_at;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, i = blockIdx.x;
  const int sr0 = blockIdx.y * nc_max, nsr = min(nc_max, p.S * p.R - sr0), nc = (nsr + 15) / 16 * 16;
  const uint32_t abytes = (uint32_t)((nc_max + 15) / 16) * 2048, xbytes = FP8 ? 8192 : 16384;
  // e4m3: two widened x tiles first, then stages of (e4m3 x, A); bf16: stages of (x, A)
  const uint32_t ring = base + (FP8 ? 2 * 16384 : 0), sbytes = abytes + xbytes;      // A first: 1024-byte aligned
  const uint32_t cols = tmem_cols(nc);
  pdl_wait();
  Tile t;
  if (!load_tile(p, i, t) || t.rank == 0) return;          // uniform over the cluster
  if (warp == 1) {
    tmem_alloc(&tmem_at, cols);
    tmem_relinquish();                                   // until then the SM starts no other CTA that allocates
  }
  if (tid == 0) {
    for (int q = 0; q < stages; ++q) {
      mbar_init(&full[q], 1);
      mbar_init(&empty[q], FP8 ? 9 : 1);
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(&cfull[q], 8);
      mbar_init(&cempty[q], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  // Only now may the expanding kernel start: its CTAs allocate TMEM at once and keep it until this kernel has finished, so
  // that a CTA here that had yet to allocate could wait for one that waits for it.
  pdl_trigger();
  const int nk = (p.K + 63) / 64, per = (nk + p.splits - 1) / p.splits;
  const int k0 = blockIdx.z * per, n = max(0, min(per, nk - k0));
  bool ok = true;
  if (warp == 0) {                                         // loads
    constexpr int RBYTES = FP8 ? 64 : 128;
    const TmaRows rows = tma_rows(p, i, t, lane);
    int j = 0;
    for (; j < n; ++j) {
      const int st = j % stages;
      ok = __all_sync(~0u, j < stages || mbar_wait(&empty[st], (j / stages - 1) & 1, p.status));
      if (!ok) break;
      const uint32_t as = ring + st * sbytes, xs = as + abytes;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[st], abytes + rows.n * rows.each * RBYTES);
        tma_2d(as, &am, &full[st], (k0 + j) * 64, t.slot * p.S * p.R + sr0);
      }
      __syncwarp();
      tma_load_rows(rows, xs, &xm, &xg, &full[st], (k0 + j) * 64, lane, RBYTES);
    }
    for (int q = max(0, j - stages); q < j; ++q) mbar_wait(&full[q % stages], q / stages & 1, p.status);   // no copy in flight
  } else if (warp == 1) {                                  // MMAs
    for (int j = 0; j < n; ++j) {
      const int st = j % stages;
      ok = mbar_wait(&full[st], j / stages & 1, p.status) && (!FP8 || mbar_wait(&cfull[j & 1], j / 2 & 1, p.status));
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      if (lane == 0) {
        tc_fence_after();
        const uint32_t as = ring + st * sbytes, xs = FP8 ? base + (j & 1) * 16384 : as + abytes;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_f16(tmem, sdesc_sw128(xs + kk * 32), sdesc_sw128(as + kk * 32), idesc_bf16(nc), j > 0 || kk > 0);
        mma_commit(&empty[st]);
        if (FP8) mma_commit(&cempty[j & 1]);
        if (j == n - 1) mma_commit(&done);
      }
      __syncwarp();
    }
  } else if (FP8) {                                        // e4m3 -> bf16
    const int id = tid - 64, c = id % 4;
    for (int j = 0; j < n; ++j) {
      const int st = j % stages;
      ok = mbar_wait(&full[st], j / stages & 1, p.status) && (j < 2 || mbar_wait(&cempty[j & 1], (j / 2 - 1) & 1, p.status));
      if (!__all_sync(~0u, ok)) { ok = false; break; }
      const uint32_t from = ring + st * sbytes + abytes, to = base + (j & 1) * 16384;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = id / 4 + 64 * q;
        if (r >= t.rows) continue;
        const uint4 f = ld_shared16(from + r * 64 + c * 16);
        const uint2 e0 = e4m3x4_to_bf16(f.x), e1 = e4m3x4_to_bf16(f.y), e2 = e4m3x4_to_bf16(f.z), e3 = e4m3x4_to_bf16(f.w);
        st_shared16(to + sw128(r, 2 * c), make_uint4(e0.x, e0.y, e1.x, e1.y));
        st_shared16(to + sw128(r, 2 * c + 1), make_uint4(e2.x, e2.y, e3.x, e3.y));
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&cfull[j & 1]);
        mbar_arrive(&empty[st]);
      }
    }
  }
  if (warp != 0 && n > 0 && ok) ok = mbar_wait(&done, 0, p.status);
  ok = !__syncthreads_or(!ok);
  tc_fence_after();
  const int ld = nc + 4;
  float* part = reinterpret_cast<float*>(raw + (base - smem_u32(raw)));    // where the stages were
  if (warp >= 2) sums_to_smem(tmem, n > 0 && ok, nc, part, ld, warp % 4, (warp - 2) / 4);
  tc_fence_before();
  if (p.splits > 1) cluster_sync(); else __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, cols);
  if (warp >= 2) write_v<FP8>(p, i, t, part, ld, sr0, nsr, tid - 64);
  if (p.splits > 1) cluster_sync();                        // nobody leaves while its sums are being read
}

// out of 128-row tiles: D[128 x 64] = V[128 x 2 r] [B; B][64 x 2 r]^T on tcgen05, feature tile by feature tile.  Warp 0 loads B
// and y by TMA (rings of two and three tiles), warp 1 issues the MMAs into two TMEM buffers, eight warps add and store; two
// CTAs an SM, since a store warp's own chain of loads, adds and stores leaves an SM idle.  B's rows are gathered in the
// order that gives each thread of the epilogue 8 neighbouring features of a row (the 16x256b TMEM load hands out column
// pairs), so that out moves from registers in 16-byte vectors.  The CTAs divide the feature tiles of all row tiles evenly
// and run them as segments of one row tile and slice each; the rings go on across segments.
constexpr int FT = 64, YST = 4, BST = 4;
// stages of y and B: two CTAs an SM up to rank 64 (113 KB each)
__host__ __device__ inline int y_stages(int kc, int rb) { return kc == 1 ? (rb == 128 ? 3 : YST) : kc <= 3 ? YST : 2; }
__host__ __device__ inline int b_stages(int kc, int rb) { return kc == 1 ? (rb == 128 ? 3 : BST) : 2; }

struct Segment { int i, s, n0, ne, tiles; };               // row tile, slice, first feature, end of the slice, feature tiles
// the segment that starts at unit u (row tile x feature tile), ending before u1
DEVI Segment segment_at(const Args& p, int64_t u, int64_t u1, int per_row) {
  Segment g;
  g.i = (int)(u / per_row);
  int f = (int)(u % per_row), n = 0;
  for (g.s = 0;; ++g.s, f -= n) {
    n = (p.off[g.s + 1] - p.off[g.s] + FT - 1) / FT;
    if (f < n) break;
  }
  g.n0 = p.off[g.s] + FT * f;
  g.ne = p.off[g.s + 1];
  g.tiles = (int)min((int64_t)(n - f), u1 - u);
  return g;
}

__global__ void __launch_bounds__(TH, 2) expand128_kernel(const __grid_constant__ Args p, const __grid_constant__ CUtensorMap ym,
                                                          const __grid_constant__ CUtensorMap yg, const __grid_constant__ CUtensorMap vm,
                                                          const __grid_constant__ CUtensorMap bm, const __grid_constant__ CUtensorMap bg,
                                                          int per_row) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bfull[BST], bempty[BST], yfull[YST], yempty[YST], dfull[BST], dempty[BST], vfull, vempty;
  __shared__ uint32_t tmem_at;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const int rb = min(p.Rp, 64) <= 16 ? 32 : min(p.Rp, 64) <= 32 ? 64 : 128;    // bytes of an operand row
  const int kc = (p.Rp + 63) / 64, ot = 128 * rb;          // operand tiles over the ranks, and v's size of one
  const int yst = y_stages(kc, rb), bst = b_stages(kc, rb);
  const uint32_t yb = base, vb = yb + yst * 16384, bb = vb + 2 * kc * ot;
  if (warp == 1) {
    tmem_alloc(&tmem_at, BST * FT);
    tmem_relinquish();                                   // until then the SM starts no other CTA that allocates
  }
  if (tid == 0) {
    for (int q = 0; q < YST; ++q) {
      mbar_init(&yfull[q], 1);
      mbar_init(&yempty[q], 8);
    }
    for (int q = 0; q < BST; ++q) {
      mbar_init(&bfull[q], 1);
      mbar_init(&bempty[q], 1);
      mbar_init(&dfull[q], 1);
      mbar_init(&dempty[q], 8);
    }
    mbar_init(&vfull, 1);
    mbar_init(&vempty, 1);
    fence_mbar_init();
  }
  // rows without an adapter come first in the plan: nothing to do for them where out is y
  const int nt = min(p.plan[0], p.max_tiles), skip = p.out == p.y ? min(max(p.plan[1], 0), nt) : 0;
  const int64_t units = (int64_t)(nt - skip) * per_row;
  const int64_t u0 = (int64_t)skip * per_row + units * blockIdx.x / gridDim.x;
  const int64_t u1 = (int64_t)skip * per_row + units * (blockIdx.x + 1) / gridDim.x;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  bool ok = true;
  int yc = 0, bc = 0, vc = 0;                              // y tiles, B (and D) tiles, segments with an adapter so far
  Tile t;
  if (warp == 0) {                                         // loads
    bool waited = false;
    for (int64_t u = u0; ok && u < u1;) {
      const Segment g = segment_at(p, u, u1, per_row);
      u += g.tiles;
      if (!load_tile(p, g.i, t)) continue;
      const int ks = ((t.rank + 15) / 16 + 3) / 4;
      const TmaRows rows = tma_rows(p, g.i, t, lane);
      // 32 features in the epilogue's order: one box of a map that sees feature 8 a + 2 m + b as (b, a, m); at the end of the
      // last adapter, where that box would leave the tensor, four rows at a time by number.  Lanes 0 .. 7 and 8 .. 15 have
      // a block each.
      const int64_t l0 = (int64_t)t.slot * p.N;
      const int fb = 32 * (lane >> 3), fg = fb + (lane & 1) * 16 + (lane >> 1 & 3) * 2;   // rows 4 lane .. + 3 of the tile
      for (int j = 0; j < g.tiles; ++j, ++yc) {
        const int n0 = g.n0 + FT * j, ys = yc % yst, st = bc % bst;
        ok = __all_sync(~0u, yc < yst || mbar_wait(&yempty[ys], (yc / yst - 1) & 1, p.status));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&yfull[ys], rows.n * rows.each * 128);
        __syncwarp();
        tma_load_rows(rows, yb + ys * 16384, &ym, &yg, &yfull[ys], n0, lane, 128);
        if (t.rank == 0) continue;
        ok = __all_sync(~0u, bc < bst || mbar_wait(&bempty[st], (bc / bst - 1) & 1, p.status));
        if (!ok) { ++yc; break; }
        if (lane == 0) mbar_arrive_expect_tx(&bfull[st], ks * FT * rb);
        __syncwarp();
        const int64_t f = l0 + n0 + fb;
        const bool box = f + 32 <= (int64_t)p.L * p.N && f % 8 == 0;
        for (int k = 0; k < ks && lane < 16; ++k) {
          const uint32_t dst = bb + (st * kc + k) * FT * rb;
          if (box) {
            if (lane % 8 == 0) tma_5d(dst + fb * rb, &bm, &bfull[st], 64 * k, (int)(f / 8));
          } else {
            const int f4 = n0 + fg, last = g.ne - 1;
            tma_gather4(dst + lane * 4 * rb, &bg, &bfull[st], 64 * k,
                        make_int4((int)(l0 + min(f4, last)), (int)(l0 + min(f4 + 1, last)), (int)(l0 + min(f4 + 8, last)),
                                  (int)(l0 + min(f4 + 9, last))));
          }
        }
        ++bc;
        if (j > 0) continue;
        // y and B do not depend on v: the first tile is on its way before the wait for the shrinking kernel, which itself
        // waited for whatever wrote them
        if (!waited) pdl_wait();
        waited = true;
        ok = __all_sync(~0u, vc == 0 || mbar_wait(&vempty, (vc - 1) & 1, p.status));
        if (!ok) { ++yc; break; }
        if (lane == 0) {
          mbar_arrive_expect_tx(&vfull, 2 * ks * ot);
          for (int q = 0; q < 2 * ks; ++q)
            tma_2d(vb + (q / ks * kc + q % ks) * ot, &vm, &vfull, (g.s * 2 + q / ks) * p.Rp + 64 * (q % ks), g.i * 128);
        }
        __syncwarp();
        ++vc;
      }
    }
    if (!waited) pdl_wait();
    for (int q = max(0, yc - yst); q < yc; ++q) mbar_wait(&yfull[q % yst], q / yst & 1, p.status);   // no copy stays in flight
    for (int q = max(0, bc - bst); q < bc; ++q) mbar_wait(&bfull[q % bst], q / bst & 1, p.status);
    if (vc > 0) mbar_wait(&vfull, (vc - 1) & 1, p.status);
  } else if (warp == 1) {                                  // MMAs
    pdl_wait();                                            // a bounded wait covers no other kernel's time
    for (int64_t u = u0; ok && u < u1;) {
      const Segment g = segment_at(p, u, u1, per_row);
      u += g.tiles;
      if (!load_tile(p, g.i, t) || t.rank == 0) continue;
      const int rk16 = (t.rank + 15) / 16;                 // MMA steps
      for (int j = 0; j < g.tiles; ++j, ++bc) {
        const int st = bc % bst, dt = bc % BST;
        ok = (j > 0 || mbar_wait(&vfull, vc & 1, p.status)) && mbar_wait(&bfull[st], bc / bst & 1, p.status) &&
             (bc < BST || mbar_wait(&dempty[dt], (bc / BST - 1) & 1, p.status));
        if (!__all_sync(~0u, ok)) { ok = false; break; }
        const uint32_t bs = bb + st * kc * FT * rb;
        if (t.rank & 15) {                                 // what the slot holds beyond the adapter's rank counts as zero
          for (int r = lane; r < FT; r += 32)
            for (int k = t.rank; k < rk16 * 16; ++k)
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(bs + k / 64 * FT * rb + sw_rows(r, k % 64 / 8, rb) + k % 8 * 2),
                           "h"((uint16_t)0) : "memory");
          fence_proxy_async();
          __syncwarp();
        }
        if (lane == 0) {
          tc_fence_after();
          for (int hl = 1; hl >= 0; --hl)
            for (int kk = 0; kk < rk16; ++kk) {
              const uint32_t o = (kk % 4) * 32;
              mma_f16(tmem + dt * FT, sdesc_rows(vb + (hl * kc + kk / 4) * ot + o, rb), sdesc_rows(bs + kk / 4 * FT * rb + o, rb),
                      idesc_bf16(FT), hl == 0 || kk > 0);
            }
          mma_commit(&bempty[st]);
          mma_commit(&dfull[dt]);
          if (j == g.tiles - 1) mma_commit(&vempty);
        }
        __syncwarp();
      }
      ++vc;
    }
  } else {                                                 // out = y + D
    const int wq = warp % 4, wh = (warp - 2) / 4, g8 = lane >> 2, q4 = lane & 3;
    const uint32_t yat = yb + sw128(wq * 32 + g8, 4 * wh + q4);          // + 8 rows: the same swizzle
    pdl_wait();
    pdl_trigger();
    for (int64_t u = u0; ok && u < u1;) {
      const Segment g = segment_at(p, u, u1, per_row);
      u += g.tiles;
      if (!load_tile(p, g.i, t)) continue;
      const bool rows_here = wq * 32 < t.rows;
      __nv_bfloat16* to[2][2];
#pragma unroll
      for (int rh = 0; rh < 2; ++rh)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = row_of(p, g.i, wq * 32 + 16 * rh + 8 * h + g8, t.rows);
          to[rh][h] = r >= 0 ? p.out + r * p.out_ld + g.n0 + wh * 32 + 8 * q4 : nullptr;
        }
      for (int j = 0; j < g.tiles; ++j, ++yc) {
        const int ys = yc % yst, st = bc % BST;
        ok = mbar_wait(&yfull[ys], yc / yst & 1, p.status) && (t.rank == 0 || mbar_wait(&dfull[st], bc / BST & 1, p.status));
        if (!__all_sync(~0u, ok)) { ok = false; break; }
        tc_fence_after();
        const int left = g.ne - g.n0 - FT * j - wh * 32 - 8 * q4;        // features from this thread's first on
        if (rows_here) {
          uint32_t r[2][16];
          if (t.rank > 0) {
#pragma unroll
            for (int rh = 0; rh < 2; ++rh)
              tmem_ld_16x256b_x4(tmem + ((uint32_t)(wq * 32 + 16 * rh) << 16) + st * FT + wh * 32, r[rh]);
          }
          uint4 o[2][2];
#pragma unroll
          for (int rh = 0; rh < 2; ++rh)
#pragma unroll
            for (int h = 0; h < 2; ++h) o[rh][h] = ld_shared16(yat + ys * 16384 + (16 * rh + 8 * h) * 128);
          if (t.rank > 0) {
            tmem_ld_wait();
#pragma unroll
            for (int rh = 0; rh < 2; ++rh)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t* w = reinterpret_cast<uint32_t*>(&o[rh][h]);
#pragma unroll
                for (int m = 0; m < 4; ++m)
                  w[m] = pack2(__uint_as_float(w[m] << 16) + __uint_as_float(r[rh][4 * m + 2 * h]),
                               __uint_as_float(w[m] & 0xffff0000u) + __uint_as_float(r[rh][4 * m + 2 * h + 1]));
              }
          }
#pragma unroll
          for (int rh = 0; rh < 2; ++rh)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (to[rh][h] == nullptr || left <= 0) continue;
              __nv_bfloat16* at = to[rh][h] + FT * j;
              if (left >= 8) *reinterpret_cast<uint4*>(at) = o[rh][h];
              else {
                const uint32_t w[4] = {o[rh][h].x, o[rh][h].y, o[rh][h].z, o[rh][h].w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (e < left) at[e] = __ushort_as_bfloat16((uint16_t)(w[e / 2] >> 16 * (e % 2)));
              }
            }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&yempty[ys]);
          if (t.rank > 0) mbar_arrive(&dempty[st]);
        }
        if (t.rank > 0) ++bc;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, BST * FT);
}

// 128-row tiles whose rows TMA cannot take (an odd K, N or row stride): the same products, operands moved by ordinary loads.
// Eight warps fill the stage, one thread multiplies.
template <bool FP8>
__global__ void __launch_bounds__(256) shrink128_any_kernel(const __grid_constant__ Args p, int nc_max) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bar[2];
  __shared__ uint32_t tmem_at;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid / 32, i = blockIdx.x;
  const int sr0 = blockIdx.y * nc_max, nsr = min(nc_max, p.S * p.R - sr0), nc = (nsr + 15) / 16 * 16;
  const uint32_t sbytes = 16384 + (uint32_t)((nc_max + 15) / 16) * 2048, cols = tmem_cols(nc);
  pdl_wait();
  Tile t;
  if (!load_tile(p, i, t) || t.rank == 0) return;          // uniform over the cluster
  if (warp == 0) {
    tmem_alloc(&tmem_at, cols);
    tmem_relinquish();                                   // until then the SM starts no other CTA that allocates
  }
  if (tid < 2) mbar_init(&bar[tid], 1);
  fence_mbar_init();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  pdl_trigger();                                           // as in shrink128_kernel
  const int nk = (p.K + 63) / 64, per = (nk + p.splits - 1) / p.splits;
  const int k0 = blockIdx.z * per, n = max(0, min(per, nk - k0));
  const uint8_t* x[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int row = row_of(p, i, tid / 8 + 32 * q, t.rows);
    x[q] = row >= 0 ? static_cast<const uint8_t*>(p.x) + row * p.x_ld * (FP8 ? 1 : 2) : nullptr;
  }
  const __nv_bfloat16* a = p.a + ((int64_t)t.slot * p.S * p.R + sr0) * p.K;
  bool ok = true;
  for (int j = 0; j < n; ++j) {
    if (j >= 2) ok = mbar_wait(&bar[j & 1], (j / 2 - 1) & 1, p.status);     // its stage is free
    const uint32_t xs = base + (j & 1) * sbytes, as = xs + 16384;
    const int k = (k0 + j) * 64 + tid % 8 * 8;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (x[q]) st_shared16(xs + sw128(tid / 8 + 32 * q, tid % 8), load8<FP8, false>(x[q], k, p.K));
    for (int r = tid / 8; r < nsr; r += 32)
      st_shared16(as + sw128(r, tid % 8), load8<false, false>(a + (int64_t)r * p.K, k, p.K));
    fence_proxy_async();
    if (__syncthreads_or(!ok)) { ok = false; break; }
    if (tid == 0) {
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        mma_f16(tmem, sdesc_sw128(xs + kk * 32), sdesc_sw128(as + kk * 32), idesc_bf16(nc), j > 0 || kk > 0);
      mma_commit(&bar[j & 1]);
    }
  }
  if (n > 0 && ok) ok = mbar_wait(&bar[(n - 1) & 1], (n - 1) / 2 & 1, p.status);
  ok = !__syncthreads_or(!ok);
  tc_fence_after();
  const int ld = nc + 4;
  float* part = reinterpret_cast<float*>(raw + (base - smem_u32(raw)));    // where the stages were
  sums_to_smem(tmem, n > 0 && ok, nc, part, ld, warp % 4, warp / 4);
  tc_fence_before();
  if (p.splits > 1) cluster_sync(); else __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, cols);
  write_v<FP8>(p, i, t, part, ld, sr0, nsr, tid);
  if (p.splits > 1) cluster_sync();                        // nobody leaves while its sums are being read
}

template <bool VECN>
__global__ void __launch_bounds__(256, 2) expand128_any_kernel(const __grid_constant__ Args p) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bar;
  __shared__ uint32_t tmem_at;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, g = lane >> 2, q4 = lane & 3, i = blockIdx.y;
  const int kc = (p.Rp + 63) / 64;                         // 64-rank operand tiles
  const bool two = kc <= 3;                                // two stages of B, as far as shared memory goes
  const uint32_t vb = base, bb = base + 2 * kc * 16384, bstage = two ? kc * 16384 : 0;
  int s, ne;
  const int nb = slice_of(p, blockIdx.x, 128 * p.steps, s, ne), nt = min(p.steps, (ne - nb + 127) / 128);
  Tile t;
  if (!load_tile(p, i, t) || (t.slot < 0 && p.out == p.y)) {
    pdl_wait();
    return;
  }
  if (warp == 0) {
    tmem_alloc(&tmem_at, 128);
    tmem_relinquish();                                   // until then the SM starts no other CTA that allocates
  }
  if (tid == 0) mbar_init(&bar, 1);
  fence_mbar_init();
  // rows of this thread: 32 (warp % 4) + 16 rh + 8 h + g; features 64 (warp / 4) + 32 cb + 8 q4 of a tile
  int64_t yo[2][2], oo[2][2];
#pragma unroll
  for (int rh = 0; rh < 2; ++rh)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row_of(p, i, warp % 4 * 32 + 16 * rh + 8 * h + g, t.rows);
      yo[rh][h] = r >= 0 ? r * p.y_ld : -1;
      oo[rh][h] = r * p.out_ld;
    }
  const bool rows_here = warp % 4 * 32 < t.rows;
  const __nv_bfloat16* bt = p.b + (int64_t)max(t.slot, 0) * p.N * p.R;
  const int rk16 = (t.rank + 15) / 16, chunks = rk16 * 2;  // MMA steps; 16-byte chunks of a rank row in use
  auto load_b = [&](int j) {
    const int n0 = nb + 128 * j;
    for (int o = tid; o < 128 * chunks; o += 256) {
      const int r = o / chunks, c = o % chunks;
      const int nn = n0 + (r & ~31) + 8 * ((r & 7) >> 1) + 2 * (r >> 3 & 3) + (r & 1);
      if (nn >= ne) continue;
      uint32_t w[4] = {};
      for (int e = 0; e < min(t.rank - 8 * c, 8); ++e)     // ranks beyond the adapter's own count as zero
        w[e / 2] |= (uint32_t)__bfloat16_as_ushort(bt[(int64_t)nn * p.R + 8 * c + e]) << 16 * (e % 2);
      st_shared16(bb + (j & 1) * bstage + (c / 8) * 16384 + sw128(r, c % 8), make_uint4(w[0], w[1], w[2], w[3]));
    }
  };
  if (t.rank > 0) load_b(0);
  pdl_wait();
  if (t.rank > 0) {
    const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(p.v);
    for (int o = tid; o < t.rows * 2 * chunks; o += 256) {
      const int r = o / (2 * chunks), hl = o / chunks % 2, c = o % chunks;
      st_shared16(vb + (hl * kc + c / 8) * 16384 + sw128(r, c % 8),
                  *reinterpret_cast<const uint4*>(v + ((((int64_t)i * 128 + r) * p.S + s) * 2 + hl) * p.Rp + 8 * c));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  pdl_trigger();                                           // TMEM first: the next kernel's CTAs may allocate before they wait
  bool ok = true;
  for (int j = 0; j < nt; ++j) {
    const int n0 = nb + 128 * j;
    uint4 y[2][2][2];
#pragma unroll
    for (int rh = 0; rh < 2; ++rh)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
          y[rh][h][cb] = load_y<VECN>(yo[rh][h] >= 0 ? p.y + yo[rh][h] : nullptr, n0 + warp / 4 * 64 + 32 * cb + 8 * q4, ne);
    if (t.rank > 0) {
      fence_proxy_async();
      tc_fence_before();
      if (__syncthreads_or(!ok)) { ok = false; break; }
      if (tid == 0) {
        tc_fence_after();
        const uint32_t bs = bb + (j & 1) * bstage;
        for (int hl = 1; hl >= 0; --hl)
          for (int kk = 0; kk < rk16; ++kk) {
            const uint32_t o = (kk / 4) * 16384 + (kk % 4) * 32;
            mma_f16(tmem, sdesc_sw128(vb + hl * kc * 16384 + o), sdesc_sw128(bs + o), idesc_bf16(128), hl == 0 || kk > 0);
          }
        mma_commit(&bar);
      }
      if (two && j + 1 < nt) load_b(j + 1);
      ok = __all_sync(0xffffffffu, mbar_wait(&bar, j & 1, p.status));
      tc_fence_after();
      if (!two && j + 1 < nt) load_b(j + 1);
    }
    if (!rows_here || !ok) continue;
#pragma unroll
    for (int rh = 0; rh < 2; ++rh)
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) {
        uint32_t r[16];
        if (t.rank > 0) {
          tmem_ld_16x256b_x4(tmem + ((uint32_t)(warp % 4 * 32 + 16 * rh) << 16) + warp / 4 * 64 + 32 * cb, r);
          tmem_ld_wait();
        }
        const int at = n0 + warp / 4 * 64 + 32 * cb + 8 * q4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (yo[rh][h] < 0 || at >= ne) continue;
          uint4 o = y[rh][h][cb];
          if (t.rank > 0) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const __nv_bfloat162 f = *reinterpret_cast<const __nv_bfloat162*>(&w[m]);
              w[m] = pack2(__low2float(f) + __uint_as_float(r[4 * m + 2 * h]),
                           __high2float(f) + __uint_as_float(r[4 * m + 2 * h + 1]));
            }
          }
          __nv_bfloat16* to = p.out + oo[rh][h] + at;
          if (VECN && at + 8 <= ne) *reinterpret_cast<uint4*>(to) = o;
          else
            for (int e = 0; e < 8; ++e)
              if (at + e < ne) to[e] = reinterpret_cast<const __nv_bfloat16*>(&o)[e];
        }
      }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 128);
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
// Kernels with large stages: the size, and all of the SM's shared memory rather than what one CTA needs (without it the SM
// runs one CTA where two fit).  Once per kernel, device and larger size.
void allow_smem(const void* kern, size_t smem) {
  if (smem <= 16 * 1024) return;
  static std::mutex m;
  static std::map<std::pair<const void*, int>, size_t> set;
  int dev;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  const std::lock_guard<std::mutex> lock(m);
  size_t& have = set[{kern, dev}];
  if (smem <= have) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)std::max<size_t>(smem, 48 * 1024)));
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  have = smem;
}

template <typename... A>
void launch(void (*kern)(A...), dim3 grid, int threads, int cx, int cz, size_t smem, cudaStream_t stream, A... args) {
  allow_smem((const void*)kern, smem);
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
  if (cx * cz > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cx;
    at[n].val.clusterDim.y = 1;
    at[n++].val.clusterDim.z = cz;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args...));
}

unsigned chunks(const Args& p, int span) {
  unsigned n = 0;
  for (int s = 0; s < p.S; ++s) n += (p.off[s + 1] - p.off[s] + span - 1) / span;
  return n;
}

// 16-row tiles
template <int JG>
void launch16(Args& p, bool fp8, bool vec, const at::TensorOptions& opts, cudaStream_t st) {
  constexpr int STEP = STEPF<JG>;
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // one launch while all its clusters run at once (two CTAs an SM); beyond, its chain of latencies counts once per wave:
  // 64 rows of 24 adapters took 43 us so, and 20 to 25 us in two launches.  Only the plan's room for tiles is known here: a
  // decode graph's has room for a tile a row, and 64 rows of 4 adapters take 13.0 us so (rank 16, 5120 -> 17408), with a
  // plan of their size 7.7
  for (p.steps = 1; p.steps < 4 && (int64_t)chunks(p, CL * STEP * p.steps) * CL * p.max_tiles > 2 * sms;) p.steps *= 2;
  const unsigned ch = chunks(p, CL * STEP * p.steps);
  if ((int64_t)ch * CL * p.max_tiles <= 2 * sms) {
    const size_t smem = (8 * 16 * RS<JG> + 256 * JG + 16 * (p.Rp + 4)) * sizeof(float);
    auto k = fp8 ? (vec ? decode_kernel<JG, true, true> : decode_kernel<JG, true, false>)
                 : (vec ? decode_kernel<JG, false, true> : decode_kernel<JG, false, false>);
    launch(k, dim3(ch * CL, p.max_tiles), 256, CL, 1, smem, st, p);
    return;
  }
  const int groups = (p.Rp + 16 * JG - 1) / (16 * JG);
  // shares of K of at least two 32-blocks a warp, as many as run at once (three CTAs an SM)
  p.splits = std::max<int64_t>(1, std::min<int64_t>({8, 3 * sms / ((int64_t)p.max_tiles * p.S * groups), p.K / 512}));
  // v from the allocator, not a shared workspace: calls on several streams must not meet in it
  torch::Tensor ws = torch::empty({(int64_t)p.splits * p.max_tiles * 16 * p.S * p.Rp}, opts);
  p.v = ws.data_ptr<float>();
  auto k = fp8 ? (vec ? shrink16_kernel<JG, true, true> : shrink16_kernel<JG, true, false>)
               : (vec ? shrink16_kernel<JG, false, true> : shrink16_kernel<JG, false, false>);
  launch(k, dim3(p.max_tiles, p.S * groups, p.splits), 256, 1, 1, 0, st, p);
  // steps of a CTA: as many as leave four CTAs for every SM
  for (p.steps = 1; p.steps < 16 && (int64_t)chunks(p, STEP * (p.steps + 1)) * p.max_tiles >= 4 * sms;) ++p.steps;
  launch(vec ? expand16_kernel<JG, true> : expand16_kernel<JG, false>, dim3(chunks(p, STEP * p.steps), p.max_tiles), 256, 1, 1,
         16 * (p.Rp + 4) * sizeof(float), st, p);
}

// 128-row tiles
int rank_rows(const Args& p) { return std::max(1, std::min(p.S, 256 / p.R)) * p.R; }   // of whole slices: the MMA's N

void launch128(Args& p, const CUtensorMap& am, const CUtensorMap& bm, const CUtensorMap& bg, bool fp8, bool tma_k, bool tma_n, bool vec_n,
               const at::TensorOptions& opts, cudaStream_t st) {
  torch::Tensor ws = torch::empty({(int64_t)p.max_tiles * 128 * p.S * p.Rp}, opts);
  p.v = ws.data_ptr<float>();
  const int nc = rank_rows(p), groups = (p.S * p.R + nc - 1) / nc, nc16 = (nc + 15) / 16 * 16;
  const int64_t ctas = (int64_t)p.max_tiles * groups, sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // Shares of K: as many as give every SM two CTAs, each with four 64-k steps or more.  Both launches with 1, 2, 4, 8 shares:
  // 5 tiles (rank 16, 5120 -> 16480) 71, 45, 32, 27 us; 12 (rank 64, 8704 -> 5120) 93, 55, 37, 28; 33 (rank 16, as the
  // first) 113, 87, 75, 72; 64 (rank 64, 5120 -> 17408), where four fill the machine, 182, 162, 155, 165.
  for (p.splits = 1; p.splits < 8 && ctas * p.splits * 2 <= 2 * sms && p.K >= 256 * p.splits * 2;) p.splits *= 2;
  const size_t sums = 128 * (nc16 + 4) * sizeof(float) + 1024;
  const dim3 grid(p.max_tiles, groups, p.splits);
  if (tma_k) {
    const size_t fixed = 1024 + (fp8 ? 2 * 16384 : 0), stage = nc16 * 128 + (fp8 ? 8192 : 16384);
    const int stages = std::min<size_t>(8, (113 * 1024 - fixed) / stage >= 3 ? (113 * 1024 - fixed) / stage : (225 * 1024 - fixed) / stage);
    const auto map = [&](int box) {
      return make_tma_2d(const_cast<void*>(p.x), fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.K, p.T,
                         p.x_ld * (fp8 ? 1 : 2), 64, box, fp8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B);
    };
    launch(fp8 ? shrink128_kernel<true> : shrink128_kernel<false>, grid, TH, 1, p.splits, std::max(fixed + stages * stage, sums),
           st, p, map(16), map(1), am, nc, stages);
  } else {
    launch(fp8 ? shrink128_any_kernel<true> : shrink128_any_kernel<false>, grid, 256, 1, p.splits,
           std::max((size_t)1024 + 2 * (16384 + nc16 * 128), sums), st, p, nc);
  }
  const int kc = (p.Rp + 63) / 64, rb = p.Rp <= 16 ? 32 : p.Rp <= 32 ? 64 : 128;
  if (tma_n) {
    const auto map = [&](int box) {
      return make_tma_2d((void*)p.y, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.N, p.T, p.y_ld * 2, 64, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    const CUtensorMap vm = make_tma_2d(p.v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (uint64_t)p.S * 2 * p.Rp, (uint64_t)p.max_tiles * 128,
                                       (uint64_t)p.S * 4 * p.Rp, rb / 2, 128,
                                       rb == 32 ? CU_TENSOR_MAP_SWIZZLE_32B : rb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    const size_t smem = 1024 + y_stages(kc, rb) * 16384 + (size_t)kc * rb * (2 * 128 + b_stages(kc, rb) * FT);
    const int per_row = chunks(p, FT);
    const unsigned grid = std::min<int64_t>((int64_t)p.max_tiles * per_row, sms * (smem <= 113 * 1024 ? 2 : 1));
    launch(expand128_kernel, dim3(grid), TH, 1, 1, smem, st, p, map(16), map(1), vm, bm, bg, per_row);
  } else {
    // feature tiles of a CTA: v is staged once for all of them, as long as every SM has a few CTAs
    for (p.steps = 1; p.steps < 16 && (int64_t)chunks(p, 128 * p.steps * 2) * p.max_tiles >= 4 * sms;) p.steps *= 2;
    launch(vec_n ? expand128_any_kernel<true> : expand128_any_kernel<false>, dim3(chunks(p, 128 * p.steps), p.max_tiles), 256, 1, 1,
           (size_t)(kc <= 3 ? 4 : 3) * kc * 16384 + 1024, st, p);
  }
}

[[noreturn]] void refuse(const std::string& why) { throw pybind11::value_error("lora_add: " + why); }

bool overlap(const torch::Tensor& a, const torch::Tensor& b) {
  const auto span = [](const torch::Tensor& t) {
    return (t.size(0) - 1) * t.stride(0) * t.element_size() + t.size(1) * t.element_size();
  };
  const uint8_t *pa = (const uint8_t*)a.data_ptr(), *pb = (const uint8_t*)b.data_ptr();
  return pa < pb + span(b) && pb < pa + span(a);
}

}  // namespace lora

// The stacked adapters of one projection; the tensors are checked by the caller (models/lora.AdapterBank).
struct LoraBank {
  torch::Tensor a, b, scale, ranks, status;
  lora::Args args;
  bool tma_k = false, tma_n = false;                       // rows of a / b that TMA can take
  CUtensorMap am, bm, bg;
  LoraBank(torch::Tensor a_, torch::Tensor b_, torch::Tensor scale_, torch::Tensor ranks_, std::vector<int64_t> slices,
           torch::Tensor status_)
      : a(a_), b(b_), scale(scale_), ranks(ranks_), status(status_) {
    TORCH_CHECK(a.is_cuda() && (int64_t)slices.size() == a.size(1) + 1 && a.size(1) <= lora::MAX_S, "LoraBank");
    args = {};
    args.a = (const __nv_bfloat16*)a.data_ptr(); args.b = (const __nv_bfloat16*)b.data_ptr();
    args.scale = scale.data_ptr<float>(); args.rank = ranks.data_ptr<int>(); args.status = status.data_ptr<int>();
    args.L = a.size(0); args.S = a.size(1); args.R = a.size(2); args.K = a.size(3); args.N = b.size(1);
    args.Rp = (args.R + 15) / 16 * 16;
    for (size_t s = 0; s < slices.size(); ++s) args.off[s] = slices[s];
    const int64_t rows = (int64_t)args.L * args.S * args.R, brows = (int64_t)args.L * args.N;
    if ((tma_k = args.K % 8 == 0 && (uintptr_t)args.a % 16 == 0 && rows < (1ll << 31)))
      am = make_tma_2d(a.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, args.K, rows, args.K * 2ll, 64,
                       (lora::rank_rows(args) + 15) / 16 * 16, CU_TENSOR_MAP_SWIZZLE_128B);
    if ((tma_n = args.R % 8 == 0 && (uintptr_t)args.b % 16 == 0 && brows < (1ll << 31))) {
      const int rb = args.Rp <= 16 ? 32 : args.Rp <= 32 ? 64 : 128;
      const auto swz = rb == 32 ? CU_TENSOR_MAP_SWIZZLE_32B : rb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
      bg = make_tma_2d(b.data_ptr(), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, args.R, brows, args.R * 2ll, rb / 2, 1, swz);
      // (rank, b, a, m, u): feature 8 (u + a) + 2 m + b; the last three u would reach beyond the tensor
      const cuuint64_t row = args.R * 2ll, dims[5] = {(cuuint64_t)args.R, 2, 4, 4, (cuuint64_t)std::max<int64_t>(1, brows / 8 - 3)};
      const cuuint64_t strides[4] = {row, 8 * row, 2 * row, 8 * row};
      const cuuint32_t box[5] = {(cuuint32_t)rb / 2, 2, 4, 4, 1}, each[5] = {1, 1, 1, 1, 1};
      tma_n = brows >= 32;
      if (tma_n)
        TORCH_CHECK(get_encode_tiled()(&bm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, b.data_ptr(), dims, strides, box, each,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS, "LoraBank: tensor map of b");
    }
  }
};
// The rows of a step: words of the 16-row list, then of the 128-row list (models/lora.AdapterPlan).
struct LoraPlan {
  torch::Tensor buf;
  int64_t rows, tiles16, tiles128, slots;
  LoraPlan(torch::Tensor buf_, int64_t rows_, int64_t tiles16_, int64_t tiles128_, int64_t slots_)
      : buf(buf_), rows(rows_), tiles16(tiles16_), tiles128(tiles128_), slots(slots_) {
    TORCH_CHECK(buf.is_cuda() && buf.scalar_type() == at::kInt && buf.is_contiguous() && tiles16 >= 0 && tiles16 <= 65535 &&
                    tiles128 >= 0 && tiles128 <= 65535 && buf.numel() >= words16() + 4 + 132 * tiles128 &&
                    (uintptr_t)buf.data_ptr() % 16 == 0,
                "LoraPlan: int32 words on the device, 16-byte aligned");
  }
  int64_t words16() const { return 4 + 20 * tiles16; }
};

torch::Tensor lora_add(const torch::Tensor& y, const torch::Tensor& x, const c10::optional<torch::Tensor>& xs,
                       const LoraBank& bank, const LoraPlan& plan, const c10::optional<torch::Tensor>& out_) {
  using lora::refuse;
  lora::Args p = bank.args;
  const bool fp8 = xs.has_value();
  if (y.dim() != 2 || x.dim() != 2 || x.size(0) != y.size(0) || plan.rows != y.size(0)) refuse("rows of y, x and the plan");
  if (x.size(1) != p.K || y.size(1) != p.N || plan.slots > p.L) refuse("features or slots of the adapters");
  if (y.scalar_type() != at::kBFloat16 || x.scalar_type() != (fp8 ? at::kFloat8_e4m3fn : at::kBFloat16))
    refuse("y bf16, x bf16 or (e4m3, scale)");
  if (y.device() != bank.a.device() || x.device() != y.device() || plan.buf.device() != y.device())
    refuse("operands on one device");
  if (fp8 && (xs->device() != y.device() || xs->scalar_type() != at::kFloat || xs->dim() != 1 || xs->size(0) != x.size(0) ||
              !xs->is_contiguous()))
    refuse("x scales fp32 [T]");
  const at::cuda::CUDAGuard guard(y.device());
  const int64_t T = y.size(0);
  if (out_.has_value() && (out_->sizes() != y.sizes() || out_->scalar_type() != y.scalar_type() || out_->device() != y.device()))
    refuse("out as y");
  torch::Tensor out = out_.has_value() ? *out_ : torch::empty({T, (int64_t)p.N}, y.options());
  if (T == 0) return out;
  if (T > (1 << 30)) refuse("rows");
  if (x.stride(1) != 1 || y.stride(1) != 1 || out.stride(1) != 1) refuse("rows must be contiguous");
  const bool same = out.data_ptr() == y.data_ptr() && out.stride(0) == y.stride(0);
  if (out_.has_value() && ((!same && lora::overlap(out, y)) || lora::overlap(out, x) || (T > 1 && out.stride(0) < p.N)))
    refuse("out overlaps y or x other than being y");
  // one row's stride says nothing: any that fits the widest loads
  const auto ld = [T](const torch::Tensor& t) { return T == 1 ? (t.size(1) + 15) / 16 * 16 : t.stride(0); };
  p.x = x.data_ptr(); p.xs = fp8 ? xs->data_ptr<float>() : nullptr; p.x_ld = ld(x);
  p.y = (const __nv_bfloat16*)y.data_ptr(); p.y_ld = ld(y);
  p.out = (__nv_bfloat16*)out.data_ptr(); p.out_ld = ld(out);
  p.T = T;
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool vec_k = p.K % 8 == 0 && p.x_ld % 8 == 0 && (uintptr_t)p.x % 16 == 0 && (uintptr_t)p.a % 16 == 0;
  bool vec_n = p.y_ld % 8 == 0 && p.out_ld % 8 == 0 && ((uintptr_t)p.y | (uintptr_t)p.out) % 16 == 0 &&
               (uintptr_t)p.b % 16 == 0;
  for (int s = 0; s < p.S; ++s) vec_n = vec_n && p.off[s] % 8 == 0;
  const auto opts = bank.scale.options();
  if (plan.tiles128) {
    p.plan = plan.buf.data_ptr<int>() + plan.words16(); p.max_tiles = plan.tiles128; p.tile_rows = 128;
    // TMA takes no rows on top of one another (a broadcast x or y)
    lora::launch128(p, bank.am, bank.bm, bank.bg, fp8, bank.tma_k && vec_k && p.x_ld >= p.K && (!fp8 || p.x_ld % 16 == 0),
                    bank.tma_n && vec_n && p.y_ld >= p.N, vec_n, opts, stream);
  }
  if (plan.tiles16) {
    p.plan = plan.buf.data_ptr<int>(); p.max_tiles = plan.tiles16; p.tile_rows = 16;
    const bool vec = vec_k && vec_n && p.R % 4 == 0;
    if (p.Rp <= 16) lora::launch16<1>(p, fp8, vec, opts, stream);
    else lora::launch16<2>(p, fp8, vec, opts, stream);
  }
  return out;
}

void lora_bind(pybind11::module_& m) {
  pybind11::class_<LoraBank>(m, "LoraBank")
      .def(pybind11::init<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, std::vector<int64_t>, torch::Tensor>());
  pybind11::class_<LoraPlan>(m, "LoraPlan").def(pybind11::init<torch::Tensor, int64_t, int64_t, int64_t, int64_t>());
  m.def("lora_add", &lora_add, "projection output + the low-rank deltas of each row's adapter");
}

}  // namespace rad
