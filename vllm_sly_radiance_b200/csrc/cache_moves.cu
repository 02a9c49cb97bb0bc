// Cache items copied onto other items of the same caches: pages of forked or compacted sequences, recurrent state slots.
//
// An item is one KV page (its rows in every attention layer's K and V cache) or one state slot (conv and SSM state of
// every GDN layer): tens of segments in as many tensors.  One launch copies a list of pages and slots in all of them; a
// source with several destinations is read once, and of a page only its first `tokens` rows of each kv head are moved.
// Nothing is computed: the floor is one read of each source and one write of each destination.
//
// table int64 [n, 6] on the device, one row per cache tensor: base address, bytes from item to item, planes (kv heads),
// bytes of a plane, bytes of a token's row in a plane (0: items have no tokens), rows of a plane.
// pieces int32 [m, 2]: (tensor, index) of each 16 KB piece of an item.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/numpy.h>
#include <torch/extension.h>

#include <algorithm>
#include <numeric>

#include "common.cuh"

namespace rad {
namespace cmv {

constexpr int PIECE = 16384, THREADS = 256, VEC = PIECE / (16 * THREADS);

struct Kind {
  const int64_t* table;
  const int2* pieces;
  int num_pieces, num_items, groups;
};

// The list travels as a kernel argument (at most 32 KB): no copy to the device, nothing to keep alive.  The groups of
// pages come first.  Destinations of source g: dst[first[g] .. first[g + 1]).
template <int G, int D>
struct List {
  static constexpr int MAX_G = G, MAX_D = D;
  int src[G];
  int tokens[G];
  int first[G + 1];
  int dst[D];
};
using Small = List<64, 128>;
using Large = List<1600, 3100>;

// One CTA per (source, piece): a thread has its four 16-byte vectors in flight together, then stores them once per
// destination.  Bound by memory: 6.2 to 6.4 TB/s of the bytes that have to move (8 samples of a 151 MB state 223 us, 1500
// pages of 384 KB 190 us; one load and store at a time in twice the launches: 245 and 213 us).  Small lists are bound by
// the host's call, 5 us.
template <typename LIST>
__global__ void __launch_bounds__(THREADS) move_kernel(const Kind blocks, const Kind slots, int* status,
                                                       const __grid_constant__ LIST q) {
  pdl_wait();
  pdl_trigger();
  int64_t at = blockIdx.x;
  const int64_t nb = (int64_t)blocks.groups * blocks.num_pieces;
  const bool page = at < nb;
  const Kind& k = page ? blocks : slots;
  if (!page) at -= nb;
  const int g = (page ? 0 : blocks.groups) + (int)(at / k.num_pieces);
  const int2 pc = k.pieces[at % k.num_pieces];
  const int64_t* tb = k.table + 6 * (int64_t)pc.x;
  const int64_t base = tb[0], stride = tb[1], plane = tb[3], row = tb[4];
  const int64_t used = row ? min((int64_t)q.tokens[g], tb[5]) * row : plane;    // bytes of a plane that are copied
  const int64_t o0 = (int64_t)pc.y * PIECE, end = min(used * tb[2], o0 + PIECE);
  const int s = q.src[g];
  if ((unsigned)s >= (unsigned)k.num_items) {
    if (threadIdx.x == 0) atomicExch(status, (int)kErrBounds);
    return;
  }
  const uint8_t* from = reinterpret_cast<const uint8_t*>(base + s * stride);
  if (((base | stride | plane | used) & 15) == 0) {
    uint4 v[VEC];
    int64_t to_off[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int64_t o = o0 + (int64_t)(i * THREADS + threadIdx.x) * 16;
      // whole planes lie side by side; the used parts of partly filled ones do not
      to_off[i] = o >= end ? -1 : used == plane ? o : o / used * plane + o % used;
      if (to_off[i] >= 0) v[i] = __ldcs(reinterpret_cast<const uint4*>(from + to_off[i]));
    }
    for (int d = q.first[g]; d < q.first[g + 1]; ++d) {
      if ((unsigned)q.dst[d] >= (unsigned)k.num_items) {
        if (threadIdx.x == 0) atomicExch(status, (int)kErrBounds);
        continue;
      }
      uint8_t* to = reinterpret_cast<uint8_t*>(base + q.dst[d] * stride);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (to_off[i] >= 0) __stcs(reinterpret_cast<uint4*>(to + to_off[i]), v[i]);
    }
    return;
  }
  for (int64_t o = o0 + threadIdx.x; o < end; o += THREADS) {       // sizes that 16 bytes do not divide
    const int64_t a = o / used * plane + o % used;
    const uint8_t v = from[a];
    for (int d = q.first[g]; d < q.first[g + 1]; ++d)
      if ((unsigned)q.dst[d] < (unsigned)k.num_items) *(reinterpret_cast<uint8_t*>(base + q.dst[d] * stride) + a) = v;
  }
}

[[noreturn]] void refuse(const std::string& why) { throw pybind11::value_error("cache moves: " + why); }

struct Group { int src, tokens, first, count; };           // destinations dst[first .. first + count)

}  // namespace cmv

// One kind of item over its cache tensors, which the caller keeps where they are.
struct CacheItems {
  torch::Tensor table, pieces, status;
  int64_t num, rows;                                       // items; tokens of a page (0: items have no tokens)
  std::string name;
  CacheItems(std::string name_, torch::Tensor table_, torch::Tensor pieces_, torch::Tensor status_, int64_t num_, int64_t rows_)
      : table(table_), pieces(pieces_), status(status_), num(num_), rows(rows_), name(name_) {
    TORCH_CHECK(table.is_cuda() && table.scalar_type() == at::kLong && table.dim() == 2 && table.size(1) == 6 &&
                    table.is_contiguous() && pieces.is_cuda() && pieces.scalar_type() == at::kInt && pieces.dim() == 2 &&
                    pieces.size(1) == 2 && pieces.is_contiguous() && num < (1ll << 31) && pieces.size(0) < (1 << 24),
                "CacheItems: table int64 [n, 6] and pieces int32 [m, 2] on the device");
  }

  // m int64 [n, 2 or 3]: (src, dst[, tokens]).  Destinations of one (source, tokens) end up side by side.
  void group(const int64_t* m, int64_t n, int64_t cols, std::vector<cmv::Group>& groups, std::vector<int>& dst) const {
    if (cols != 2 && !(rows && cols == 3)) cmv::refuse(name + (rows ? " as (src, dst[, tokens])" : " as (src, dst)") + " rows");
    const auto tok = [&](int64_t i) { return cols == 3 ? m[i * cols + 2] : rows; };
    std::vector<uint8_t> seen(num, 0);
    bool sorted = true;
    for (int64_t i = 0; i < n; ++i) {
      const int64_t s = m[i * cols], d = m[i * cols + 1];
      if (s < 0 || s >= num || d < 0 || d >= num) cmv::refuse(name + " outside 0 .. " + std::to_string(num - 1));
      if (rows && (tok(i) < 0 || tok(i) > rows)) cmv::refuse("0 .. " + std::to_string(rows) + " tokens of a page");
      if (seen[d] & 2) cmv::refuse(name + ": a destination twice");
      seen[s] |= 1;
      seen[d] |= 2;
      if (i && (s < m[(i - 1) * cols] || (s == m[(i - 1) * cols] && tok(i) < tok(i - 1)))) sorted = false;
    }
    for (int64_t i = 0; i < n; ++i)
      if (seen[m[i * cols]] == 3) cmv::refuse(name + ": both source and destination");
    std::vector<int64_t> order(n);
    std::iota(order.begin(), order.end(), 0);
    if (!sorted)
      std::stable_sort(order.begin(), order.end(), [&](int64_t a, int64_t b) {
        return m[a * cols] != m[b * cols] ? m[a * cols] < m[b * cols] : tok(a) < tok(b);
      });
    for (const int64_t i : order) {
      const int s = m[i * cols], t = tok(i);
      if (groups.empty() || groups.back().src != s || groups.back().tokens != t || groups.back().count == 128)
        groups.push_back({s, t, (int)dst.size(), 0});
      ++groups.back().count;
      dst.push_back(m[i * cols + 1]);
    }
  }
};

namespace cmv {

template <typename LIST>
cudaError_t launch(const CacheItems* const (&kinds)[2], const Group* groups, const int* dst, const int (&count)[2],
                   cudaStream_t stream) {
  LIST q;
  Kind k[2] = {};
  int64_t ctas = 0;
  for (int i = 0; i < 2; ++i)
    if (count[i]) {
      k[i] = {(const int64_t*)kinds[i]->table.data_ptr(), (const int2*)kinds[i]->pieces.data_ptr(),
              (int)kinds[i]->pieces.size(0), (int)kinds[i]->num, count[i]};
      ctas += (int64_t)count[i] * k[i].num_pieces;
    }
  const int n = count[0] + count[1], d0 = groups[0].first;
  for (int i = 0; i < n; ++i) {
    q.src[i] = groups[i].src;
    q.tokens[i] = groups[i].tokens;
    q.first[i] = groups[i].first - d0;
  }
  q.first[n] = groups[n - 1].first + groups[n - 1].count - d0;
  std::copy(dst + d0, dst + d0 + q.first[n], q.dst);
  if (ctas == 0) return cudaSuccess;
  const CacheItems* any = count[0] ? kinds[0] : kinds[1];
  return launch_pdl(move_kernel<LIST>, dim3(ctas), dim3(THREADS), 0, stream, k[0], k[1], any->status.data_ptr<int>(), q);
}

void run(const CacheItems* const (&kinds)[2], std::vector<Group> (&g)[2], std::vector<int>& dst) {
  const CacheItems* any = g[0].empty() ? kinds[1] : kinds[0];
  const at::cuda::CUDAGuard guard(any->table.device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const size_t nb = g[0].size();
  std::vector<Group>& all = g[0];
  all.insert(all.end(), g[1].begin(), g[1].end());
  for (size_t i = 0; i < all.size();) {                    // one launch, unless the list is longer than an argument may be
    const bool small = all.size() - i <= Small::MAX_G && dst.size() - all[i].first <= Small::MAX_D;
    const int gmax = small ? Small::MAX_G : Large::MAX_G, dmax = small ? Small::MAX_D : Large::MAX_D;
    int n = 0, nd = 0, count[2] = {0, 0};
    while (i + n < all.size() && n < gmax && nd + all[i + n].count <= dmax) {
      nd += all[i + n].count;
      ++count[i + n < nb ? 0 : 1];
      ++n;
    }
    C10_CUDA_CHECK(small ? launch<Small>(kinds, &all[i], dst.data(), count, stream)
                         : launch<Large>(kinds, &all[i], dst.data(), count, stream));
    i += n;
  }
}

using Moves = pybind11::array_t<int64_t, pybind11::array::c_style | pybind11::array::forcecast>;

bool none(const pybind11::handle& rows) {
  const Py_ssize_t n = PySequence_Check(rows.ptr()) ? PySequence_Size(rows.ptr()) : -1;
  if (n < 0) PyErr_Clear();
  return n == 0;
}
// whole numbers only: a cast would cut 1.5 to the item 1
Moves whole(const pybind11::handle& rows) {
  const pybind11::array a = pybind11::array::ensure(rows);
  if (!a || (a.size() && a.dtype().kind() != 'i' && a.dtype().kind() != 'u')) refuse("moves as rows of whole numbers");
  return Moves(a);
}

// both kinds in one launch; everything is checked before anything moves
void copy(const CacheItems* blocks, const pybind11::handle& block_moves, const CacheItems* slots, const pybind11::handle& slot_moves) {
  const CacheItems* const kinds[2] = {blocks, slots};
  const pybind11::handle rows[2] = {block_moves, slot_moves};
  std::vector<Group> g[2];
  std::vector<int> dst;
  for (int i = 0; i < 2; ++i) {
    if (none(rows[i])) continue;
    const Moves m = whole(rows[i]);
    if (m.size() == 0) continue;
    if (m.ndim() != 2) refuse("moves as rows");
    if (!kinds[i]) refuse("the caches have no such items");
    kinds[i]->group(m.data(), m.shape(0), m.shape(1), g[i], dst);
  }
  if (!g[0].empty() || !g[1].empty()) run(kinds, g, dst);
}

// tables int [sequences, pages]: block ids, <= 0 for none.  The pages they name move to blocks 1 .. n: those behind the
// first n, ascending, into the free ones among them, ascending.  -> (new tables, n)
template <typename T>
pybind11::tuple compact(const CacheItems& blocks, const pybind11::array_t<T, pybind11::array::c_style>& tables) {
  const int64_t total = tables.size();
  const T* t = tables.data();
  std::vector<T> to(blocks.num, 0);
  int64_t n = 0;
  for (int64_t i = 0; i < total; ++i) {
    if (t[i] <= 0) continue;
    if (t[i] >= blocks.num) refuse("blocks outside 0 .. " + std::to_string(blocks.num - 1));
    n += to[t[i]] == 0;
    to[t[i]] = t[i];
  }
  std::vector<Group> g[2];
  std::vector<int> dst;
  int64_t hole = 1;
  for (int64_t b = n + 1; b < blocks.num; ++b) {
    if (!to[b]) continue;
    while (to[hole]) ++hole;
    g[0].push_back({(int)b, (int)blocks.rows, (int)dst.size(), 1});
    dst.push_back(hole);
    to[b] = hole++;                                        // of a page that moved; to[hole] itself is not looked up
  }
  pybind11::array_t<T> out(std::vector<pybind11::ssize_t>(tables.shape(), tables.shape() + tables.ndim()));
  T* o = out.mutable_data();
  for (int64_t i = 0; i < total; ++i) o[i] = t[i] > 0 ? to[t[i]] : t[i];
  const CacheItems* const kinds[2] = {&blocks, nullptr};
  if (!g[0].empty()) run(kinds, g, dst);
  return pybind11::make_tuple(out, n);
}

}  // namespace cmv

void cache_moves_bind(pybind11::module_& m) {
  pybind11::class_<CacheItems>(m, "CacheItems")
      .def(pybind11::init<std::string, torch::Tensor, torch::Tensor, torch::Tensor, int64_t, int64_t>());
  m.def("cache_copy", &cmv::copy, "cache items (pages, states) -> other items of the same caches");
  m.def("cache_compact", &cmv::compact<int>, pybind11::arg(), pybind11::arg().noconvert(),
        "pages in use -> the front of the pool, and their new tables");
  m.def("cache_compact", &cmv::compact<int64_t>, pybind11::arg(), pybind11::arg().noconvert());
}

}  // namespace rad
