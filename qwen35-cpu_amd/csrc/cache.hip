// Copies inside the paged FP16 cache: whole or partly filled pages (forks,
// copies before a shared page is written), and the rows of accepted tree nodes
// moved up behind their request's context. Each copied byte is read once and
// written once; what bounds the large ones is HBM, the small ones the launch.
#include <algorithm>

#include "q35_device.h"
#include "q35_internal.h"

namespace q35 {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyPieces = 4;  // pieces in flight per thread

// One workgroup per (1024 pieces of a page, pool and layer, pair). The pairs
// travel in the kernel's arguments, so a call stages nothing on the device. T
// is the widest piece that the rows and the pools allow.
template <typename T>
__global__ __launch_bounds__(kCopyThreads) void page_copy_kernel(PageCopyArgs a, PagePairs pairs) {
  const int i = static_cast<int>(blockIdx.x), z = static_cast<int>(blockIdx.z);
  const size_t row = static_cast<size_t>(a.row_elems) * 2 / sizeof(T);  // pieces
  const size_t n = row * pairs.tokens[i], page = row * a.page_tokens;
  T *pool = reinterpret_cast<T *>((z & 1) ? a.v_pool : a.k_pool) + static_cast<size_t>(z >> 1) * (a.layer_stride * 2 / sizeof(T));
  const T *src = pool + page * pairs.src[i];
  T *dst = pool + page * pairs.dst[i];
  const size_t at = static_cast<size_t>(blockIdx.y) * (kCopyThreads * kCopyPieces) + threadIdx.x;
  T v[kCopyPieces];
#pragma unroll
  for (int u = 0; u < kCopyPieces; ++u)
    if (at + u * kCopyThreads < n) v[u] = src[at + u * kCopyThreads];
#pragma unroll
  for (int u = 0; u < kCopyPieces; ++u)
    if (at + u * kCopyThreads < n) dst[at + u * kCopyThreads] = v[u];
}

// Row context + path[j] of a request to row context + j, in every layer, for
// j in order. A thread owns one piece of the row in one pool and layer, so it
// reads every source before it overwrites it: path[j] >= j, and a row that is
// both is read at the step j' <= j that needs it, in the same batch of loads
// or an earlier one. A request whose path or pages are out of bounds is left
// as it is.
constexpr int kMoveBatch = 8;

template <typename T>
__global__ __launch_bounds__(kCopyThreads) void row_compact_kernel(CompactArgs a) {
  __shared__ int refuse;
  const int b = static_cast<int>(blockIdx.y), tid = threadIdx.x;
  const int shift = a.page_shift, pmask = (1 << shift) - 1;
  const int capacity = a.max_pages << shift;
  const int32_t *table = a.page_table + static_cast<size_t>(b) * a.max_pages;
  const int32_t *path = a.path + static_cast<size_t>(b) * a.path_stride;
  const int context = a.context_lens[b], count = a.path_count[b];
  if (context < 0 || context > capacity || count <= 0 || count > a.path_stride) return;  // whole workgroup
  if (tid == 0) refuse = 0;
  __syncthreads();
  auto page_ok = [&](int t) { return static_cast<unsigned>(table[t >> shift]) < static_cast<unsigned>(a.total_pages); };
  for (int j = tid; j < count; j += kCopyThreads) {
    const int p = path[j];
    if (p < j || p >= capacity - context || !page_ok(context + j) || !page_ok(context + p)) refuse = 1;
  }
  __syncthreads();
  if (refuse != 0) return;
  const size_t row = static_cast<size_t>(a.row_elems) * 2 / sizeof(T);
  const size_t e = static_cast<size_t>(blockIdx.x) * kCopyThreads + tid;
  const size_t z = e / row;
  if (z >= static_cast<size_t>(2 * a.layers)) return;
  T *pool = reinterpret_cast<T *>((z & 1) ? a.v_pool : a.k_pool) + (z >> 1) * (a.layer_stride * 2 / sizeof(T)) + (e - z * row);
  auto cache_row = [&](int t) { return static_cast<size_t>((table[t >> shift] << shift) + (t & pmask)) * row; };
  for (int j0 = 0; j0 < count; j0 += kMoveBatch) {
    T v[kMoveBatch];
    int from[kMoveBatch];
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u) {
      const int j = j0 + u;
      from[u] = j < count ? path[j] : j;
      if (from[u] != j) v[u] = pool[cache_row(context + from[u])];
    }
#pragma unroll
    for (int u = 0; u < kMoveBatch; ++u)
      if (from[u] != j0 + u) pool[cache_row(context + j0 + u)] = v[u];
  }
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The widest piece (bytes) that divides the rows, the layer distance and the
// pools' addresses.
int piece_bytes(const void *k, const void *v, size_t row_elems, size_t layer_stride) {
  for (int n : {16, 4})
    if (aligned(k, n) && aligned(v, n) && row_elems * 2 % n == 0 && layer_stride * 2 % n == 0) return n;
  return 2;
}

}  // namespace

hipError_t launch_page_copy(const PageCopyArgs &a, const PagePairs &pairs, int count, hipStream_t stream) {
  const int piece = piece_bytes(a.k_pool, a.v_pool, a.row_elems, a.layer_stride);
  int most = 0;  // rows of the fullest page
  for (int i = 0; i < count; ++i) most = std::max(most, pairs.tokens[i]);
  if (most == 0) return hipSuccess;
  const size_t pieces = static_cast<size_t>(a.row_elems) * 2 / piece * most, per = kCopyThreads * kCopyPieces;
  const dim3 grid(count, static_cast<unsigned>((pieces + per - 1) / per), 2 * a.layers);
  switch (piece) {
    case 16: Q35_LAUNCH((page_copy_kernel<q35_u32x4>), grid, dim3(kCopyThreads), 0, stream, a, pairs); break;
    case 4: Q35_LAUNCH((page_copy_kernel<uint32_t>), grid, dim3(kCopyThreads), 0, stream, a, pairs); break;
    default: Q35_LAUNCH((page_copy_kernel<uint16_t>), grid, dim3(kCopyThreads), 0, stream, a, pairs); break;
  }
  return hipGetLastError();
}

hipError_t launch_row_compact(const CompactArgs &a, hipStream_t stream) {
  const int piece = piece_bytes(a.k_pool, a.v_pool, a.row_elems, a.layer_stride);
  const size_t pieces = static_cast<size_t>(a.row_elems) * 2 / piece * 2 * a.layers;
  const dim3 grid(static_cast<unsigned>((pieces + kCopyThreads - 1) / kCopyThreads), a.batch);
  switch (piece) {
    case 16: Q35_LAUNCH((row_compact_kernel<q35_u32x4>), grid, dim3(kCopyThreads), 0, stream, a); break;
    case 4: Q35_LAUNCH((row_compact_kernel<uint32_t>), grid, dim3(kCopyThreads), 0, stream, a); break;
    default: Q35_LAUNCH((row_compact_kernel<uint16_t>), grid, dim3(kCopyThreads), 0, stream, a); break;
  }
  return hipGetLastError();
}

}  // namespace q35
