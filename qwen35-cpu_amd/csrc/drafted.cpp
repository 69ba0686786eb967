// Entry points of a drafted step (include/q35_hip.h): attention of drafted
// trees, sampling, acceptance, and the copies inside the paged cache. None of
// them waits for the device or reads device memory on the host, so each can be
// captured into a graph; what the host cannot check (lengths, page ids, tree
// indices on the device) the kernels check before they use it.
#include "runtime.h"

#include <algorithm>
#include <cmath>
#include <limits>
#include <new>
#include <vector>

namespace q35 {
namespace {

// The context's device for the length of a call, whatever the thread's current
// device is.
struct DeviceScope {
  int before = -1;
  bool moved = false;
  explicit DeviceScope(int device) {
    if (hipGetDevice(&before) == hipSuccess && before != device) moved = hipSetDevice(device) == hipSuccess;
  }
  ~DeviceScope() {
    if (moved) (void)hipSetDevice(before);
  }
};

// Runs the body of an entry point: nothing thrown leaves it.
template <typename F>
int guarded(q35_context *ctx, F body) {
  if (ctx == nullptr) return Q35_ERR_INVALID;
  try {
    DeviceScope scope(ctx->device);
    return body();
  } catch (const std::bad_alloc &) {
    return Q35_ERR_OOM;
  } catch (...) {
    return Q35_ERR_INVALID;
  }
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

constexpr size_t kMaxInt = static_cast<size_t>(std::numeric_limits<int32_t>::max());
// Up to 32 page pairs are compared with each other (0.8 us); a byte for every page
// takes 0.1 us for 4096 pages and 25 us for a million.
constexpr size_t kComparedPairs = 32;

// The caller's workspace, or the context's own (grown as needed). A call under
// capture needs its own: the context's may be freed by a later call that grows
// it, and graphs that share it could not run side by side.
int workspace_get(q35_context *ctx, void *given, size_t given_bytes, size_t need, void **out) {
  *out = nullptr;
  if (need == 0) return Q35_OK;
  if (given != nullptr) {
    if (given_bytes < need) return set_error(ctx, Q35_ERR_INVALID, "workspace too small");
    if (!aligned(given, 256)) return set_error(ctx, Q35_ERR_INVALID, "workspace not aligned to 256 bytes");
    *out = given;
    return Q35_OK;
  }
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  Q35_HIP_TRY(ctx, hipStreamIsCapturing(ctx->stream, &capture));
  if (capture != hipStreamCaptureStatusNone)
    return set_error(ctx, Q35_ERR_STATE, "a captured call needs a workspace of its own");
  if (ctx->work_bytes < need) {
    Q35_HIP_TRY(ctx, hipStreamSynchronize(ctx->stream));
    if (ctx->work != nullptr) (void)hipFree(ctx->work);
    ctx->work = nullptr;
    ctx->work_bytes = 0;
    Q35_HIP_TRY(ctx, hipMalloc(&ctx->work, need));
    ctx->work_bytes = need;
  }
  *out = ctx->work;
  return Q35_OK;
}

// The shape checks of the tree attention and its plan; 0 or an error status.
int tree_check(q35_context *ctx, size_t batch, size_t rows, size_t max_nodes, size_t max_len, int heads, int kv_heads,
               int head_dim, TreeArgs *a) {
  if (batch == 0 || max_nodes == 0 || max_len == 0 || kv_heads <= 0 || heads <= 0)
    return set_error(ctx, Q35_ERR_INVALID, "tree attention: an empty shape");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(ctx, Q35_ERR_UNSUPPORTED, "tree attention needs head_dim 64, 128 or 256");
  if (heads % kv_heads != 0) return set_error(ctx, Q35_ERR_UNSUPPORTED, "tree attention needs heads % kv_heads == 0");
  if (max_nodes > static_cast<size_t>(kMaxTreeNodes) || batch > 65535 || heads > 1024 || rows > kMaxInt / 1024 ||
      max_len > kMaxInt - 1024)
    return set_error(ctx, Q35_ERR_UNSUPPORTED, "tree attention: at most 256 nodes a request, 65535 requests, 1024 heads");
  a->batch = static_cast<int>(batch);
  a->rows = static_cast<int>(rows);
  a->max_nodes = static_cast<int>(max_nodes);
  a->max_len = static_cast<int>(max_len);
  a->heads = heads;
  a->kv_heads = kv_heads;
  a->head_dim = head_dim;
  const long long units = tree_request_units(a->max_nodes, a->max_len, heads, kv_heads);
  if (units > static_cast<long long>(kMaxInt) || units * a->batch > kMaxTreeUnits)
    return set_error(ctx, Q35_ERR_UNSUPPORTED, "tree attention: max_len times the KV heads and requests is too large");
  a->groups = tree_groups(a->batch, a->max_nodes, a->max_len, heads, kv_heads, ctx->cu_count);
  return Q35_OK;
}

int draw_check(q35_context *ctx, size_t rows, size_t vocab) {
  if (rows == 0 || vocab == 0) return set_error(ctx, Q35_ERR_INVALID, "sampling: no rows or no tokens");
  if (rows > 65535 || vocab > static_cast<size_t>(kDrawMaxVocab))
    return set_error(ctx, Q35_ERR_UNSUPPORTED, "sampling: at most 65535 rows of 1048576 tokens");
  return Q35_OK;
}

// Whether a layer of one pool shares memory with a layer of the other: their
// distance less a whole number of layer strides is below a layer's size.
bool pools_overlap(const void *k, const void *v, size_t layers, size_t layer_stride, size_t layer_elems) {
  const __int128 distance = static_cast<__int128>(reinterpret_cast<uintptr_t>(v)) - reinterpret_cast<uintptr_t>(k);
  const __int128 size = 2 * static_cast<__int128>(layer_elems), stride = layers > 1 ? 2 * static_cast<__int128>(layer_stride) : size;
  const __int128 most = static_cast<__int128>(layers) - 1;
  for (__int128 m = distance / stride - 1; m <= distance / stride + 1; ++m) {
    const __int128 rest = distance - std::clamp(m, -most, most) * stride;
    if (rest < size && -rest < size) return true;
  }
  return false;
}

// Pools of the cache copies: addresses and sizes. One pool for K and V is `same`
// (copies write the same bytes twice then, but moves would be made twice).
int pool_check(q35_context *ctx, const void *k, const void *v, size_t layers, size_t layer_stride, size_t total_pages,
               size_t page_tokens, size_t row_elems, bool same) {
  if (k == nullptr || v == nullptr || layers == 0 || total_pages == 0 || page_tokens == 0 || row_elems == 0 ||
      !aligned(k, 2) || !aligned(v, 2))
    return set_error(ctx, Q35_ERR_INVALID, "cache copy: a missing pool or an empty shape");
  if (layers > 32767 || page_tokens > (1u << 20) || row_elems > (1u << 20) || total_pages > kMaxInt / page_tokens)
    return set_error(ctx, Q35_ERR_UNSUPPORTED, "cache copy: at most 2^31 - 1 cache rows of 2^20 values");
  if (layers > 1 && layer_stride / row_elems / page_tokens < total_pages)
    return set_error(ctx, Q35_ERR_INVALID, "cache copy: layers overlap");
  if (!(same && k == v) && pools_overlap(k, v, layers, layer_stride, total_pages * page_tokens * row_elems))
    return set_error(ctx, Q35_ERR_INVALID, "cache copy: the K and V pools overlap");
  return Q35_OK;
}

}  // namespace

int copy_pages(q35_context *ctx, const PageCopyArgs &a, const int32_t *src, const int32_t *dst, const int32_t *tokens,
               size_t count) {
  DeviceScope scope(ctx->device);
  PagePairs pairs;
  for (size_t i = 0; i < count;) {
    int n = 0;
    for (; n < kCopyPairs && i < count; ++n, ++i) {
      pairs.src[n] = src[i];
      pairs.dst[n] = dst[i];
      pairs.tokens[n] = tokens != nullptr ? tokens[i] : a.page_tokens;
    }
    const hipError_t e = launch_page_copy(a, pairs, n, ctx->stream);
    if (e != hipSuccess) return hip_error(ctx, e, "page copy");
  }
  return Q35_OK;
}

}  // namespace q35

using namespace q35;

extern "C" int q35_attention_tree_workspace(q35_context *ctx, size_t batch, size_t rows, size_t max_nodes,
                                            size_t max_len, int heads, int kv_heads, int head_dim, size_t *bytes) {
  return guarded(ctx, [&]() -> int {
    if (bytes == nullptr) return set_error(ctx, Q35_ERR_INVALID, "tree attention: no place for the size");
    TreeArgs a;
    const int st = tree_check(ctx, batch, rows, max_nodes, max_len, heads, kv_heads, head_dim, &a);
    size_t part_o = 0, part_ml = 0;
    if (st == Q35_OK) *bytes = tree_workspace_bytes(a, &part_o, &part_ml);
    return st;
  });
}

extern "C" int q35_attention_tree_paged(q35_context *ctx, const float *q, const float *gates, const uint16_t *k_pool,
                                        const uint16_t *v_pool, size_t total_pages, const int32_t *page_table,
                                        size_t max_pages, size_t page_tokens, const int32_t *context_lens,
                                        const int32_t *node_start, const uint64_t *node_masks, float *output,
                                        size_t batch, size_t rows, size_t max_nodes, size_t max_len, int heads,
                                        int kv_heads, int head_dim, float scale, void *workspace,
                                        size_t workspace_bytes) {
  return guarded(ctx, [&]() -> int {
    if (q == nullptr || k_pool == nullptr || v_pool == nullptr || page_table == nullptr || context_lens == nullptr ||
        node_start == nullptr || node_masks == nullptr || output == nullptr)
      return set_error(ctx, Q35_ERR_INVALID, "tree attention: a missing buffer");
    if (!aligned(q, 16) || !aligned(gates, 16) || !aligned(output, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) ||
        !aligned(node_masks, 8))
      return set_error(ctx, Q35_ERR_INVALID, "tree attention: buffers need 16-byte alignment (masks 8)");
    TreeArgs a;
    int st = tree_check(ctx, batch, rows, max_nodes, max_len, heads, kv_heads, head_dim, &a);
    if (st != Q35_OK) return st;
    if (page_tokens == 0 || (page_tokens & (page_tokens - 1)) != 0 || page_tokens > (1u << 20))
      return set_error(ctx, Q35_ERR_UNSUPPORTED, "tree attention needs a power-of-two page size");
    if (total_pages == 0 || total_pages > kMaxInt / page_tokens || max_pages > kMaxInt ||
        max_len > max_pages * page_tokens)
      return set_error(ctx, Q35_ERR_INVALID, "tree attention: max_len beyond the page table, or an empty pool");
    if (!std::isfinite(scale)) return set_error(ctx, Q35_ERR_INVALID, "tree attention: scale is not finite");
    if (rows == 0) return Q35_OK;
    void *work = nullptr;
    size_t part_o = 0, part_ml = 0;
    st = workspace_get(ctx, workspace, workspace_bytes, tree_workspace_bytes(a, &part_o, &part_ml), &work);
    if (st != Q35_OK) return st;
    a.q = q;
    a.gates = gates;
    a.k_pool = k_pool;
    a.v_pool = v_pool;
    a.page_table = page_table;
    a.total_pages = static_cast<int>(total_pages);
    a.max_pages = static_cast<int>(max_pages);
    a.page_shift = __builtin_ctzll(page_tokens);
    a.context_lens = context_lens;
    a.node_start = node_start;
    a.masks = node_masks;
    a.mask_words = (a.max_nodes + 63) / 64;
    a.out = output;
    a.scale = scale;
    a.first_units = static_cast<long long *>(work);
    a.part_o = reinterpret_cast<float *>(static_cast<char *>(work) + part_o);
    a.part_ml = reinterpret_cast<float *>(static_cast<char *>(work) + part_ml);
    const hipError_t e = launch_tree_attention(a, ctx->stream);
    return e == hipSuccess ? Q35_OK : hip_error(ctx, e, "tree attention");
  });
}

extern "C" int q35_tree_accept(q35_context *ctx, const int32_t *node_start, const int32_t *parents,
                               const int32_t *draft_tokens, const int32_t *sampled_tokens, int32_t *path,
                               size_t path_stride, int32_t *path_count, int32_t *next_token, size_t batch, size_t rows,
                               size_t max_nodes) {
  return guarded(ctx, [&]() -> int {
    if (node_start == nullptr || parents == nullptr || draft_tokens == nullptr || sampled_tokens == nullptr ||
        path == nullptr || path_count == nullptr || next_token == nullptr || batch == 0 || max_nodes == 0 ||
        path_stride < max_nodes)
      return set_error(ctx, Q35_ERR_INVALID, "tree acceptance: a missing buffer, or a path row shorter than the tree");
    if (max_nodes > static_cast<size_t>(kMaxTreeNodes) || batch > kMaxInt || rows > kMaxInt || path_stride > kMaxInt)
      return set_error(ctx, Q35_ERR_UNSUPPORTED, "tree acceptance: at most 256 nodes a request");
    AcceptArgs a;
    a.node_start = node_start;
    a.parents = parents;
    a.draft_tokens = draft_tokens;
    a.sampled_tokens = sampled_tokens;
    a.path = path;
    a.path_count = path_count;
    a.next_token = next_token;
    a.path_stride = static_cast<int>(path_stride);
    a.batch = static_cast<int>(batch);
    a.rows = static_cast<int>(rows);
    a.max_nodes = static_cast<int>(max_nodes);
    const hipError_t e = launch_tree_accept(a, ctx->stream);
    return e == hipSuccess ? Q35_OK : hip_error(ctx, e, "tree acceptance");
  });
}

extern "C" int q35_sample_workspace(q35_context *ctx, size_t rows, size_t vocab, size_t *bytes) {
  return guarded(ctx, [&]() -> int {
    if (bytes == nullptr) return set_error(ctx, Q35_ERR_INVALID, "sampling: no place for the size");
    const int st = draw_check(ctx, rows, vocab);
    if (st == Q35_OK) *bytes = draw_scratch_bytes(static_cast<int>(rows), static_cast<int>(vocab));
    return st;
  });
}

extern "C" int q35_sample_logits(q35_context *ctx, const float *logits, size_t stride, const int32_t *counts,
                                 const float *penalties, const float *temperatures, const int32_t *top_k,
                                 const float *top_p, const float *min_p, const float *uniforms, size_t rows,
                                 size_t vocab, int32_t *out_token, float *out_probability, void *workspace,
                                 size_t workspace_bytes) {
  return guarded(ctx, [&]() -> int {
    if (logits == nullptr || uniforms == nullptr || out_token == nullptr)
      return set_error(ctx, Q35_ERR_INVALID, "sampling: a missing buffer");
    int st = draw_check(ctx, rows, vocab);
    if (st != Q35_OK) return st;
    if (stride < vocab && rows > 1) return set_error(ctx, Q35_ERR_INVALID, "sampling: rows of logits overlap");
    DrawArgs a;
    a.logits = logits;
    a.stride = stride;
    a.counts = counts;
    a.penalties = penalties;
    a.temperatures = temperatures;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.uniforms = uniforms;
    a.rows = static_cast<int>(rows);
    a.vocab = static_cast<int>(vocab);
    a.out_token = out_token;
    a.out_probability = out_probability;
    void *work = nullptr;
    st = workspace_get(ctx, workspace, workspace_bytes, draw_scratch_bytes(a.rows, a.vocab), &work);
    if (st != Q35_OK) return st;
    const hipError_t e = launch_draw(a, work, ctx->stream);
    return e == hipSuccess ? Q35_OK : hip_error(ctx, e, "sampling");
  });
}

extern "C" int q35_cache_copy_pages(q35_context *ctx, uint16_t *k_pool, uint16_t *v_pool, size_t layers,
                                    size_t layer_stride, size_t total_pages, size_t page_tokens, size_t row_elems,
                                    const int32_t *src_pages, const int32_t *dst_pages, const int32_t *tokens,
                                    size_t count) {
  return guarded(ctx, [&]() -> int {
    const int st = pool_check(ctx, k_pool, v_pool, layers, layer_stride, total_pages, page_tokens, row_elems, true);
    if (st != Q35_OK || count == 0) return st;
    if (src_pages == nullptr || dst_pages == nullptr)
      return set_error(ctx, Q35_ERR_INVALID, "page copy: no pages given");
    const int32_t pages = static_cast<int32_t>(total_pages), most = static_cast<int32_t>(page_tokens);
    for (size_t i = 0; i < count; ++i) {
      const int32_t s = src_pages[i], d = dst_pages[i];
      if (s < 0 || s >= pages || d < 0 || d >= pages || (tokens != nullptr && (tokens[i] < 0 || tokens[i] > most)))
        return set_error(ctx, Q35_ERR_INVALID, "page copy: a page outside the pool, or more tokens than a page holds");
    }
    // each page written once, and none that another pair reads: the pairs run
    // in no order
    bool twice = false, both = false;
    if (count <= kComparedPairs) {
      for (size_t i = 0; i < count; ++i) {
        for (size_t j = 0; j < count; ++j) {
          twice |= j < i && dst_pages[j] == dst_pages[i];
          both |= src_pages[j] == dst_pages[i];
        }
      }
    } else {
      std::vector<uint8_t> written(total_pages, 0);
      for (size_t i = 0; i < count; ++i) {
        twice |= written[dst_pages[i]] != 0;
        written[dst_pages[i]] = 1;
      }
      for (size_t i = 0; i < count; ++i) both |= written[src_pages[i]] != 0;
    }
    if (twice) return set_error(ctx, Q35_ERR_INVALID, "page copy: a page is written twice");
    if (both) return set_error(ctx, Q35_ERR_INVALID, "page copy: a page is both read and written");
    PageCopyArgs a;
    a.k_pool = k_pool;
    a.v_pool = v_pool;
    a.layers = static_cast<int>(layers);
    a.page_tokens = most;
    a.row_elems = static_cast<int>(row_elems);
    a.layer_stride = layer_stride;
    return copy_pages(ctx, a, src_pages, dst_pages, tokens, count);
  });
}

extern "C" int q35_cache_compact_rows(q35_context *ctx, uint16_t *k_pool, uint16_t *v_pool, size_t layers,
                                      size_t layer_stride, size_t total_pages, size_t page_tokens, size_t row_elems,
                                      const int32_t *page_table, size_t max_pages, const int32_t *context_lens,
                                      const int32_t *path, size_t path_stride, const int32_t *path_count,
                                      size_t batch) {
  return guarded(ctx, [&]() -> int {
    const int st = pool_check(ctx, k_pool, v_pool, layers, layer_stride, total_pages, page_tokens, row_elems, false);
    if (st != Q35_OK || batch == 0) return st;
    if (page_table == nullptr || context_lens == nullptr || path == nullptr || path_count == nullptr || max_pages == 0 ||
        path_stride == 0)
      return set_error(ctx, Q35_ERR_INVALID, "row compaction: a missing buffer");
    if ((page_tokens & (page_tokens - 1)) != 0 || max_pages > kMaxInt / page_tokens || path_stride > kMaxInt || batch > 65535)
      return set_error(ctx, Q35_ERR_UNSUPPORTED, "row compaction needs a power-of-two page size and at most 65535 requests");
    CompactArgs a;
    a.k_pool = k_pool;
    a.v_pool = v_pool;
    a.layers = static_cast<int>(layers);
    a.row_elems = static_cast<int>(row_elems);
    a.total_pages = static_cast<int>(total_pages);
    a.max_pages = static_cast<int>(max_pages);
    a.page_shift = __builtin_ctzll(page_tokens);
    a.layer_stride = layer_stride;
    a.page_table = page_table;
    a.context_lens = context_lens;
    a.path = path;
    a.path_count = path_count;
    a.path_stride = static_cast<int>(path_stride);
    a.batch = static_cast<int>(batch);
    const hipError_t e = launch_row_compact(a, ctx->stream);
    return e == hipSuccess ? Q35_OK : hip_error(ctx, e, "row compaction");
  });
}
