// Copies inside the paged FP16 cache: whole or partly filled pages (forks,
// copies before a shared page is written), and the rows of accepted tree nodes
// moved up behind their request's context. Each copied byte is read once and
// written once; what bounds the large ones is HBM, the small ones the launch:
// 2047 pages in 8 layers of 4 KV heads of 256 take 460 us (2.1 GB, 4.7 TB/s read
// and written; a plain copy of 2 GiB reaches 4.9), 8 partly filled pages in 6
// layers of 2 KV heads 5.2 to 6.1 us by the host (the kernel 2.7), the accepted
// rows of 64 requests in 6 such layers 5.3 us.
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
template <typename T, int N>
__global__ __launch_bounds__(kCopyThreads) void page_copy_kernel(PageCopyArgs a, PagePairsOf<N> pairs) {
  const int i = static_cast<int>(blockIdx.x), z = static_cast<int>(blockIdx.z);
  const size_t row = static_cast<size_t>(a.row_elems) * 2 / sizeof(T);  // pieces
  const size_t n = row * pairs.tokens[i], page = row * a.page_tokens;
  T *pool = reinterpret_cast<T *>((z & 1) ? a.v_pool : a.k_pool) + static_cast<size_t>(z >> 1) * (a.layer_stride * 2 / sizeof(T));
  const T *src = pool + page * pairs.src[i];
  T *dst = pool + page * pairs.dst[i];
  for (size_t at = static_cast<size_t>(blockIdx.y) * (kCopyThreads * kCopyPieces) + threadIdx.x; at < n;
       at += static_cast<size_t>(gridDim.y) * (kCopyThreads * kCopyPieces)) {
    T v[kCopyPieces];
#pragma unroll
    for (int u = 0; u < kCopyPieces; ++u)
      if (at + u * kCopyThreads < n) v[u] = src[at + u * kCopyThreads];
#pragma unroll
    for (int u = 0; u < kCopyPieces; ++u)
      if (at + u * kCopyThreads < n) dst[at + u * kCopyThreads] = v[u];
  }
}

// Row context + path[j] of a request to row context + j, in every layer, for
// j in order. A thread owns one piece of the row in one pool and layer, so it
// reads every source before it overwrites it: path[j] >= j, and a row that is
// both is read at the step j' <= j that needs it, in the same batch of loads
// or an earlier one. A request whose path or pages are out of bounds is left
// as it is.
// The first 256 rows' places in the cache are kept in LDS by the check that
// comes before any write, so that the moves wait for three loads in all: the
// request's path, its pages, the rows.
constexpr int kMoveBatch = 8;

template <typename T>
__global__ __launch_bounds__(kCopyThreads) void row_compact_kernel(CompactArgs a) {
  __shared__ int refuse, from[kCopyThreads], to[kCopyThreads];  // rows of the pool
  const int b = static_cast<int>(blockIdx.y), tid = threadIdx.x;
  const int shift = a.page_shift, pmask = (1 << shift) - 1;
  const int capacity = a.max_pages << shift;
  const int32_t *table = a.page_table + static_cast<size_t>(b) * a.max_pages;
  const int32_t *path = a.path + static_cast<size_t>(b) * a.path_stride;
  const int context = a.context_lens[b], count = a.path_count[b];
  int p = path[min(tid, a.path_stride - 1)];
  if (tid == 0) refuse = 0;
  if (context < 0 || context > capacity || count <= 0 || count > a.path_stride) return;  // whole workgroup
  __syncthreads();
  auto place = [&](int j) {  // the rows of step j, where they are in bounds
    const bool ok = p >= j && p < capacity - context;
    const int t = context + j, f = context + (ok ? p : 0);
    const int dst = ok ? table[t >> shift] : -1, src = ok ? table[f >> shift] : -1;
    to[j & (kCopyThreads - 1)] = static_cast<int>(static_cast<unsigned>(dst) << shift) + (t & pmask);
    from[j & (kCopyThreads - 1)] = static_cast<int>(static_cast<unsigned>(src) << shift) + (f & pmask);
    return ok && static_cast<unsigned>(dst) < static_cast<unsigned>(a.total_pages) &&
           static_cast<unsigned>(src) < static_cast<unsigned>(a.total_pages);
  };
  for (int j = (count - 1) / kCopyThreads * kCopyThreads + tid; j >= 0; j -= kCopyThreads) {  // the first 256 last
    if (j >= count) continue;
    if (j >= kCopyThreads || count > kCopyThreads) p = path[j];
    if (!place(j)) refuse = 1;
  }
  __syncthreads();
  if (refuse != 0) return;
  const size_t row = static_cast<size_t>(a.row_elems) * 2 / sizeof(T);
  const size_t e = static_cast<size_t>(blockIdx.x) * kCopyThreads + tid;
  const size_t z = e / row;
  const bool mine = z < static_cast<size_t>(2 * a.layers);
  T *pool = reinterpret_cast<T *>((z & 1) ? a.v_pool : a.k_pool) + (z >> 1) * (a.layer_stride * 2 / sizeof(T)) + (e - z * row);
  for (int c = 0; c < count; c += kCopyThreads) {
    if (c > 0) {
      __syncthreads();
      if (c + tid < count) {
        p = path[c + tid];
        place(c + tid);
      }
      __syncthreads();
    }
    const int n = min(count - c, kCopyThreads);
    for (int j0 = 0; mine && j0 < n; j0 += kMoveBatch) {
      T v[kMoveBatch];
#pragma unroll
      for (int u = 0; u < kMoveBatch; ++u) {
        const int j = min(j0 + u, n - 1);
        v[u] = pool[static_cast<size_t>(from[j]) * row];
      }
#pragma unroll
      for (int u = 0; u < kMoveBatch; ++u)
        if (j0 + u < n && from[j0 + u] != to[j0 + u]) pool[static_cast<size_t>(to[j0 + u]) * row] = v[u];
    }
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

namespace {
template <int N>
void launch_pairs(const PageCopyArgs &a, const PagePairsOf<N> &pairs, int piece, dim3 grid, hipStream_t stream) {
  switch (piece) {
    case 16: Q35_LAUNCH((page_copy_kernel<q35_u32x4, N>), grid, dim3(kCopyThreads), 0, stream, a, pairs); break;
    case 4: Q35_LAUNCH((page_copy_kernel<uint32_t, N>), grid, dim3(kCopyThreads), 0, stream, a, pairs); break;
    default: Q35_LAUNCH((page_copy_kernel<uint16_t, N>), grid, dim3(kCopyThreads), 0, stream, a, pairs); break;
  }
}
}  // namespace

hipError_t launch_page_copy(const PageCopyArgs &a, const PagePairs &pairs, int count, hipStream_t stream) {
  const int piece = piece_bytes(a.k_pool, a.v_pool, a.row_elems, a.layer_stride);
  int most = 0;  // rows of the fullest page
  for (int i = 0; i < count; ++i) most = std::max(most, pairs.tokens[i]);
  if (most == 0) return hipSuccess;
  const size_t pieces = static_cast<size_t>(a.row_elems) * 2 / piece * most, per = kCopyThreads * kCopyPieces;
  const dim3 grid(count, static_cast<unsigned>(std::min<size_t>((pieces + per - 1) / per, 65535)), 2 * a.layers);
  if (count > kFewCopyPairs) {
    launch_pairs(a, pairs, piece, grid, stream);
  } else {
    PagePairsOf<kFewCopyPairs> few = {};
    std::copy_n(pairs.src, count, few.src);
    std::copy_n(pairs.dst, count, few.dst);
    std::copy_n(pairs.tokens, count, few.tokens);
    launch_pairs(a, few, piece, grid, stream);
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
