// Cache items copied onto other items of the same caches: pages of forked or compacted sequences, recurrent state slots.
//
// An item is one KV page (its rows in every attention layer's K and V cache) or one state slot (conv and SSM state of
// every GDN layer): tens of segments in as many tensors.  One launch copies a list of items in all of them; a source
// with several destinations is read once, and of a page only its first `tokens` rows of each kv head are moved.
//
// table int64 [n, 6] on the device, one row per cache tensor: base address, bytes from item to item, planes (kv heads),
// bytes of a plane, bytes of a token's row in a plane (0: items have no tokens), rows of a plane.
// pieces int32 [m, 2]: (tensor, index) of each 16 KB piece of an item.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"

namespace rad {
namespace cmv {

constexpr int PIECE = 16384;

// the list travels as a kernel argument: no copy to the device, nothing to keep alive
template <int G, int D>
struct List {
  int n;
  int src[G];
  int tokens[G];
  int first[G + 1];     // destinations of source i: dst[first[i] .. first[i + 1])
  int dst[D];
};
using Small = List<64, 128>;
using Large = List<1600, 3100>;

template <typename LIST>
__global__ void __launch_bounds__(256) move_kernel(const int64_t* __restrict__ table, const int2* __restrict__ pieces,
                                                   int* status, int num_items, const __grid_constant__ LIST q) {
  pdl_wait();
  pdl_trigger();
  const int g = blockIdx.y;
  const int2 pc = pieces[blockIdx.x];
  const int64_t* tb = table + 6 * (int64_t)pc.x;
  const int64_t base = tb[0], stride = tb[1], plane = tb[3], row = tb[4];
  int64_t used = plane;                                  // bytes of a plane that are copied
  if (row) used = min((int64_t)q.tokens[g], tb[5]) * row;
  const int64_t end = min(used * tb[2], (int64_t)(pc.y + 1) * PIECE);
  const int s = q.src[g];
  const bool wide = ((base | stride | plane | used) & 15) == 0;
  for (int d = q.first[g]; d < q.first[g + 1]; ++d) {
    if ((unsigned)s >= (unsigned)num_items || (unsigned)q.dst[d] >= (unsigned)num_items) {
      if (threadIdx.x == 0) atomicExch(status, (int)kErrBounds);
      continue;
    }
    const uint8_t* from = reinterpret_cast<const uint8_t*>(base + s * stride);
    uint8_t* to = reinterpret_cast<uint8_t*>(base + q.dst[d] * stride);
    const int step = wide ? 16 : 1;
    for (int64_t o = (int64_t)pc.y * PIECE + threadIdx.x * step; o < end; o += 256 * step) {
      const int64_t at = o / used * plane + o % used;
      if (wide) *reinterpret_cast<uint4*>(to + at) = *reinterpret_cast<const uint4*>(from + at);
      else to[at] = from[at];
    }
  }
}

template <typename LIST>
cudaError_t launch(const torch::Tensor& table, const torch::Tensor& pieces, int* status, int num_items,
                   const int* groups, int ng, const int* dst, cudaStream_t stream) {
  LIST q;
  q.n = ng;
  const int d0 = groups[1];
  for (int i = 0; i < ng; ++i) {
    q.src[i] = groups[4 * i];
    q.first[i] = groups[4 * i + 1] - d0;
    q.first[i + 1] = q.first[i] + groups[4 * i + 2];
    q.tokens[i] = groups[4 * i + 3];
  }
  for (int i = 0; i < q.first[ng]; ++i) q.dst[i] = dst[d0 + i];
  return launch_pdl(move_kernel<LIST>, dim3(pieces.size(0), ng), dim3(256), 0, stream,
                    (const int64_t*)table.data_ptr(), (const int2*)pieces.data_ptr(), status, num_items, q);
}

}  // namespace cmv

// groups int32 [G, 4] on the host: (source, first destination, destinations, tokens), destinations of a group side by
// side in dst (int32, on the host) and groups in their order.  No item may be both a source and a destination, or a
// destination twice (checked by the caller).
void cache_move(torch::Tensor table, torch::Tensor pieces, torch::Tensor status, int64_t num_items,
                torch::Tensor groups, torch::Tensor dst) {
  TORCH_CHECK(table.is_cuda() && table.scalar_type() == at::kLong && table.dim() == 2 && table.size(1) == 6 &&
                  table.is_contiguous(), "cache_move: table int64 [n, 6] on the device");
  TORCH_CHECK(pieces.is_cuda() && pieces.scalar_type() == at::kInt && pieces.dim() == 2 && pieces.size(1) == 2 &&
                  pieces.is_contiguous(), "cache_move: pieces int32 [m, 2] on the device");
  TORCH_CHECK(!groups.is_cuda() && groups.scalar_type() == at::kInt && groups.dim() == 2 && groups.size(1) == 4 &&
                  groups.is_contiguous() && !dst.is_cuda() && dst.scalar_type() == at::kInt && dst.is_contiguous(),
              "cache_move: groups int32 [G, 4] and dst int32 on the host");
  const int G = groups.size(0), D = dst.numel();
  const int *g = groups.data_ptr<int>(), *d = dst.data_ptr<int>();
  for (int i = 0, at = 0; i < G; ++i) {
    TORCH_CHECK(g[4 * i + 1] == at && g[4 * i + 2] > 0 && g[4 * i + 2] <= 128, "cache_move: group ", i);
    at += g[4 * i + 2];
    TORCH_CHECK(at <= D, "cache_move: destinations");
  }
  if (G == 0 || pieces.size(0) == 0) return;
  const at::cuda::CUDAGuard guard(table.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  int* st = status.data_ptr<int>();
  for (int i = 0; i < G;) {
    const bool small = G - i <= 64 && D - g[4 * i + 1] <= 128;
    const int gmax = small ? 64 : 1600, dmax = small ? 128 : 3100;
    int n = 0, nd = 0;
    while (i + n < G && n < gmax && nd + g[4 * (i + n) + 2] <= dmax) nd += g[4 * (i + n++) + 2];
    C10_CUDA_CHECK(small ? cmv::launch<cmv::Small>(table, pieces, st, num_items, g + 4 * i, n, d, stream)
                         : cmv::launch<cmv::Large>(table, pieces, st, num_items, g + 4 * i, n, d, stream));
    i += n;
  }
}

}  // namespace rad
