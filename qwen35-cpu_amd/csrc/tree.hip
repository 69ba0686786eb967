// Attention for trees of drafted tokens over the paged FP16 cache, and the
// path of a tree that its sampled tokens accept.
//
// Request b has c_b context rows in the cache and behind them one row per
// drafted node. Node i sees every context row and the nodes that its mask
// names: s_t = scale * q . k_t over the rows t it sees, p = exp(s - max),
// o = sum p_t v_t / sum p_t, times sigmoid(gate); where the sum of p is zero
// (nothing seen) the output is zero.
#include <algorithm>

#include "q35_device.h"
#include "q35_internal.h"

namespace q35 {
namespace {

constexpr int kTileTokens = 32;   // cache rows per tile
constexpr int kBlockVectors = 32; // query vectors (node, head) per workgroup
constexpr int kTreeWaves = 4;
// Probabilities enter the second product times 2^14, as two binary16 operands
// (22 bits): binary16 then holds them down to 2^-38 of the largest.
constexpr float kProbUnit = 16384.0F;

// Products of 32 cache rows and 32 query vectors on v_mfma_f32_32x32x16_f16,
// with the cache as the A operand in both: S^T[t][m] = sum_d k[t][d] q[m][d]
// and O^T[d][m] = sum_t v[t][d] p[m][t]. Lane l holds column m = l % 32 of
// either result, rows 8(i / 4) + 4(l / 32) + i % 4 in its 16 registers, so the
// softmax of a vector stays in two lanes (l and l ^ 32) and the probabilities
// are the second product's B operand as they lie: k slot (l / 32, i) of step
// ks stands for token 16 ks + 8(i / 4) + 4(l / 32) + i % 4 on both sides.
__device__ __forceinline__ int slot_token(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }

struct TreeRequest {
  int row0, nodes, context, len;  // first row, node rows, context rows, all rows
  bool valid, rows_valid;
};
__device__ __forceinline__ TreeRequest tree_request(const TreeArgs &a, int b) {
  TreeRequest r;
  const int r0 = a.node_start[b], r1 = a.node_start[b + 1], c = a.context_lens[b];
  r.rows_valid = r0 >= 0 && r1 >= r0 && r1 <= a.rows;
  r.row0 = r0;
  r.nodes = r.rows_valid ? r1 - r0 : 0;
  r.context = c;
  r.valid = r.rows_valid && r.nodes <= a.max_nodes && c >= 0 && r.nodes <= a.max_len && c <= a.max_len - r.nodes;
  r.len = r.valid ? c + r.nodes : 0;
  return r;
}

// The rows t .. t + 31 of the request that a node sees, as bits (t a multiple
// of 32 inside the request): the context, then the node's mask words from bit
// t - context on; `end` is one past the last row of the caller's range.
__device__ __forceinline__ uint32_t tree_visible(const uint64_t *words, int word_count, int t, int context, int end) {
  uint32_t bits;
  const int j = t - context;
  if (j <= -kTileTokens) {
    bits = 0xffffffffu;
  } else if (j < 0) {
    const int ctx = -j;  // 1 .. 31 context rows in the tile
    bits = ((1u << ctx) - 1u) | (static_cast<uint32_t>(words[0]) << ctx);
  } else {
    const int w = j >> 6, s = j & 63;
    bits = static_cast<uint32_t>(words[w] >> s);
    if (s > 32 && w + 1 < word_count) bits |= static_cast<uint32_t>(words[w + 1] << (64 - s));
  }
  return end - t < kTileTokens ? bits & ((1u << (end - t)) - 1u) : bits;
}

// DPL halfs of a cache row per lane, 32 lanes to a row
template <int DPL>
struct RowPiece;
template <>
struct RowPiece<8> {
  typedef q35_u32x4 T;
  static __device__ __forceinline__ uint32_t dword(const T &v, int i) { return v[i]; }
  static __device__ __forceinline__ T zero() { return T{0u, 0u, 0u, 0u}; }
};
template <>
struct RowPiece<4> {
  typedef q35_u32x2 T;
  static __device__ __forceinline__ uint32_t dword(const T &v, int i) { return v[i]; }
  static __device__ __forceinline__ T zero() { return T{0u, 0u}; }
};
template <>
struct RowPiece<2> {
  typedef uint32_t T;
  static __device__ __forceinline__ uint32_t dword(const T &v, int) { return v; }
  static __device__ __forceinline__ T zero() { return 0u; }
};

// Whether either binary16 half of a dword is infinite or NaN.
__device__ __forceinline__ bool half2_special(uint32_t w) {
  return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}

// Normalisation and the sigmoid gate of four dims; a zero sum saw nothing.
__device__ __forceinline__ q35_f32x4 tree_finish(q35_f32x4 o, float l, const float *gates) {
  const float inv = 1.0F / (l == 0.0F ? 1.0F : l);
  q35_f32x4 y = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  if (gates != nullptr) {
    const q35_f32x4 x = *reinterpret_cast<const q35_f32x4 *>(gates);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= sigmoid_stable(x[e]);
  }
  return y;
}

// One workgroup per (range of cache rows, 32 query vectors of one KV head,
// request): wavefront w takes the range's tiles w, w + 4, ... with a running
// maximum and sum of its own, operands straight from the cache, and the four
// are joined through LDS at the end.
template <int HD>
__global__ __launch_bounds__(64 * kTreeWaves) Q35_WAVES_PER_EU(1) void tree_attention_kernel(TreeArgs a) {
  constexpr int DPL = HD / 32;    // dims of a value row per lane
  constexpr int KS = HD / 16;     // 16-dim steps of the score product
  constexpr int PART = HD / 4;    // dims joined per round
  constexpr int STRIDE = PART + 4;
  typedef typename RowPiece<DPL>::T Piece;
  constexpr int JOIN = STRIDE > kTileTokens ? STRIDE : kTileTokens;  // floats per wavefront and vector
  __shared__ __align__(16) float join[kTreeWaves * kBlockVectors * JOIN];
  __shared__ float wave_max[kTreeWaves][kBlockVectors], wave_sum_[kTreeWaves][kBlockVectors];
  const int sp = static_cast<int>(blockIdx.x), b = static_cast<int>(blockIdx.z);
  const int g = static_cast<int>(blockIdx.y) % a.kv_heads, mb = static_cast<int>(blockIdx.y) / a.kv_heads;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int qpk = a.heads / a.kv_heads;
  const TreeRequest rq = tree_request(a, b);
  if (!rq.valid) {
    // refused on the device: NaN in the request's rows, where those are known
    if (rq.rows_valid && sp == 0 && mb == 0)
      for (int r = 0; r < rq.nodes; ++r)
        for (int e = tid; e < qpk * HD; e += 64 * kTreeWaves)
          a.out[(static_cast<size_t>(rq.row0 + r) * a.heads + g * qpk) * HD + e] = __uint_as_float(0x7fc00000u);
    return;
  }
  const int vectors = rq.nodes * qpk, m0 = mb * kBlockVectors;
  const int t0 = sp * a.split_tokens;
  if (m0 >= vectors || t0 >= rq.len) return;  // whole workgroup
  const int t1 = min(t0 + a.split_tokens, rq.len);

  // the lane's query vector (spare lanes repeat the last one and see nothing)
  const bool live = m0 + col < vectors;
  const int m = min(m0 + col, vectors - 1), node = m / qpk, u = m - node * qpk;
  const uint64_t *words = a.masks + static_cast<size_t>(rq.row0 + node) * a.mask_words;
  q35_f16x8 qhi[KS], qlo[KS];
  float sscale;
  {
    // the vector as two binary16 operands: 22 bits under its largest value,
    // which a power of two brings to 2^8 (exact, and any fp32 size fits)
    const float *src = a.q + (static_cast<size_t>(rq.row0 + node) * a.heads + g * qpk + u) * HD + 8 * half;
    float x[KS][8], top = 0.0F;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const q35_f32x4 lo = *reinterpret_cast<const q35_f32x4 *>(src + 16 * kk);
      const q35_f32x4 hi = *reinterpret_cast<const q35_f32x4 *>(src + 16 * kk + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[kk][i] = lo[i];
        x[kk][4 + i] = hi[i];
        top = fmaxf(top, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int ex = static_cast<int>(__float_as_uint(top) >> 23);  // biased
    ex = ex == 0 || ex == 255 ? 127 + 8 : max(ex, 20);
    const float down = __uint_as_float(static_cast<uint32_t>(127 + 8 + 127 - ex) << 23);  // 2^(8 - exponent)
    const float up = __uint_as_float(static_cast<uint32_t>(max(ex - 8, 1)) << 23);        // 2^(exponent - 8)
    sscale = a.scale * 1.44269504088896341F * up;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[kk][i] *= down;
      q35_split_f16(x[kk], qhi[kk], qlo[kk]);
    }
  }

  const int shift = a.page_shift, pmask = (1 << shift) - 1;
  const int32_t *table = a.page_table + static_cast<size_t>(b) * a.max_pages;
  const size_t kvw = static_cast<size_t>(a.kv_heads) * HD;
  const uint16_t *kcol = a.k_pool + static_cast<size_t>(g) * HD + 8 * half;
  const uint16_t *vcol = a.v_pool + static_cast<size_t>(g) * HD + DPL * col;
  // the cache row of token t + lane % 32 (rows past the range: the tile's
  // first), and whether its page lies in the pool
  auto cache_row = [&](int t, bool &ok) {
    const int tt = t + col < t1 ? t + col : t;
    const int page = table[tt >> shift];
    ok = static_cast<unsigned>(page) < static_cast<unsigned>(a.total_pages);
    return ((ok ? page : 0) << shift) + (tt & pmask);
  };

  q35_f32x16 acc[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[j][i] = 0.0F;
  float mx = -INFINITY, sum = 0.0F;  // the lane's vector; the sum over the lane's own tokens

  for (int t = t0 + kTileTokens * wave; t < t1; t += kTileTokens * kTreeWaves) {
    bool ok;
    const int row = cache_row(t, ok);
    const uint32_t lost = ~static_cast<uint32_t>(q35_ballot(ok));  // both halves hold the same 32 rows
    const uint16_t *krow = kcol + static_cast<size_t>(row) * kvw;
    q35_u32x4 kraw[KS];
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) kraw[kk] = *reinterpret_cast<const q35_u32x4 *>(krow + 16 * kk);
    Piece vraw[2][8];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int vr = __shfl(row, slot_token(8 * ks + i, half), 64);
        vraw[ks][i] = *reinterpret_cast<const Piece *>(vcol + static_cast<size_t>(vr) * kvw);
      }
    q35_f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0F;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const q35_f16x8 k = q35_f16x8_bits(kraw[kk]);
      s = Q35_MFMA_F32_32X32X16_F16(k, qhi[kk], s);
      s = Q35_MFMA_F32_32X32X16_F16(k, qlo[kk], s);
    }
    uint32_t seen = 0u;
    if (live) seen = t + kTileTokens <= rq.context && t + kTileTokens <= t1 ? 0xffffffffu : tree_visible(words, a.mask_words, t, rq.context, t1);
    float p[16], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int tok = slot_token(i, half);
      float x = s[i] * sscale;
      x = (lost >> tok) & 1u ? NAN : x;  // a page outside the pool
      p[i] = (seen >> tok) & 1u ? x : -INFINITY;
      top = fmaxf(top, p[i]);
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float next = fmaxf(mx, top), base = next == -INFINITY ? 0.0F : next;
    const float keep = mx == next ? 1.0F : exp2f(mx - base);  // 0 at the first seen row
    float part = 0.0F;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = exp2f(p[i] - base);
      part += p[i];
      p[i] *= kProbUnit;
    }
    sum = fmaf(sum, keep, part);
    mx = next;
    if (q35_ballot(keep != 1.0F) != 0ull) {
#pragma unroll
      for (int j = 0; j < DPL; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[j][i] *= keep;
    }
    // Tiles with node rows: a value that is infinite or NaN reaches only the
    // nodes that see its row (0 x inf would reach all), and spare slots hold 0.
    bool special = false;
    if (t + kTileTokens > rq.context) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int tt = t + slot_token(8 * ks + i, half);
          if (tt >= t1) vraw[ks][i] = RowPiece<DPL>::zero();
#pragma unroll
          for (int d = 0; d < DPL / 2; ++d) special |= half2_special(RowPiece<DPL>::dword(vraw[ks][i], d));
        }
      special = q35_ballot(special) != 0ull;
    }
    if (!special) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        q35_f16x8 phi, plo;
        q35_split_f16(p + 8 * ks, phi, plo);
#pragma unroll
        for (int j = 0; j < DPL; ++j) {
          const unsigned sel = (j & 1) ? 0x07060302u : 0x05040100u;
          q35_u32x4 d;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            d[e] = __builtin_amdgcn_perm(RowPiece<DPL>::dword(vraw[ks][2 * e + 1], j >> 1),
                                         RowPiece<DPL>::dword(vraw[ks][2 * e], j >> 1), sel);
          const q35_f16x8 v = q35_f16x8_bits(d);
          acc[j] = Q35_MFMA_F32_32X32X16_F16(v, phi, acc[j]);
          acc[j] = Q35_MFMA_F32_32X32X16_F16(v, plo, acc[j]);
        }
      }
    } else {
      float *pb = join + wave * kTileTokens * kBlockVectors;
#pragma unroll
      for (int i = 0; i < 16; ++i) pb[slot_token(i, half) * kBlockVectors + col] = p[i];
      wave_lds_sync();
      for (int tok = 0; tok < min(kTileTokens, t1 - t); ++tok) {
        const float pt = pb[tok * kBlockVectors + col];
        const uint16_t *vrow = a.v_pool + static_cast<size_t>(__shfl(row, tok, 64)) * kvw + static_cast<size_t>(g) * HD;
        if (!((seen >> tok) & 1u)) continue;
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int j = 0; j < DPL; ++j)
            acc[j][i] = fmaf(pt, half_bits_to_float(vrow[DPL * slot_token(i, half) + j]), acc[j][i]);
      }
      wave_lds_sync();
    }
  }

  // the four wavefronts' parts of each vector
  sum += __shfl_xor(sum, 32, 64);
  if (half == 0) {
    wave_max[wave][col] = mx;
    wave_sum_[wave][col] = sum;
  }
  __syncthreads();
  float all = wave_max[0][col];
#pragma unroll
  for (int w = 1; w < kTreeWaves; ++w) all = fmaxf(all, wave_max[w][col]);
  const float weight = exp2f(mx - (all == -INFINITY ? 0.0F : all)) * (1.0F / kProbUnit);
#pragma unroll
  for (int part = 0; part < 4; ++part) {
    if (part > 0) __syncthreads();  // the last round's sums are read
    float *mine = join + (wave * kBlockVectors + col) * STRIDE;
#pragma unroll
    for (int ii = 0; ii < 4; ++ii)
#pragma unroll
      for (int j = 0; j < DPL; ++j) mine[DPL * (4 * half + ii) + j] = acc[j][4 * part + ii] * weight;
    __syncthreads();
    for (int e = tid; e < kBlockVectors * PART / 4; e += 64 * kTreeWaves) {
      const int v = e / (PART / 4), d = 4 * (e % (PART / 4));
      if (m0 + v >= vectors) continue;
      q35_f32x4 o = *reinterpret_cast<const q35_f32x4 *>(join + v * STRIDE + d);
#pragma unroll
      for (int w = 1; w < kTreeWaves; ++w)
        o += *reinterpret_cast<const q35_f32x4 *>(join + (w * kBlockVectors + v) * STRIDE + d);
      float top = wave_max[0][v];
#pragma unroll
      for (int w = 1; w < kTreeWaves; ++w) top = fmaxf(top, wave_max[w][v]);
      const float base = top == -INFINITY ? 0.0F : top;
      float l = 0.0F;
#pragma unroll
      for (int w = 0; w < kTreeWaves; ++w) l = fmaf(wave_sum_[w][v], exp2f(wave_max[w][v] - base), l);
      const int vn = (m0 + v) / qpk, vu = (m0 + v) - vn * qpk;
      const size_t head = static_cast<size_t>(rq.row0 + vn) * a.heads + g * qpk + vu;
      const int dim = PART * part + d;
      if (a.splits > 1) {
        const size_t at = static_cast<size_t>(sp) * a.rows * a.heads + head;
        *reinterpret_cast<q35_f32x4 *>(a.part_o + at * HD + dim) = o;
        if (dim == 0) *reinterpret_cast<q35_f32x2 *>(a.part_ml + 2 * at) = q35_f32x2{top, l};
      } else {
        *reinterpret_cast<q35_f32x4 *>(a.out + head * HD + dim) =
            tree_finish(o, l, a.gates != nullptr ? a.gates + head * HD + dim : nullptr);
      }
    }
  }
}

// The ranges' parts of one (node, head): weights exp(m_s - M), in range order.
template <int HD>
__global__ __launch_bounds__(HD / 4) void tree_merge_kernel(TreeArgs a) {
  const int h = static_cast<int>(blockIdx.x), i = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  const TreeRequest rq = tree_request(a, b);
  if (!rq.valid || i >= rq.nodes) return;
  const int used = (rq.len + a.split_tokens - 1) / a.split_tokens, d = 4 * threadIdx.x;
  const size_t head = static_cast<size_t>(rq.row0 + i) * a.heads + h, step = static_cast<size_t>(a.rows) * a.heads;
  float top = -INFINITY;
  for (int s = 0; s < used; ++s) top = fmaxf(top, a.part_ml[2 * (s * step + head)]);
  const float base = top == -INFINITY ? 0.0F : top;
  q35_f32x4 o = {0.0F, 0.0F, 0.0F, 0.0F};
  float l = 0.0F;
  for (int s = 0; s < used; ++s) {
    const size_t at = s * step + head;
    const float w = exp2f(a.part_ml[2 * at] - base);
    l = fmaf(a.part_ml[2 * at + 1], w, l);
    const q35_f32x4 x = *reinterpret_cast<const q35_f32x4 *>(a.part_o + at * HD + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], w, o[e]);
  }
  *reinterpret_cast<q35_f32x4 *>(a.out + head * HD + d) =
      tree_finish(o, l, a.gates != nullptr ? a.gates + head * HD + d : nullptr);
}

// ------------------------------------------------------------- acceptance
// One wavefront per request. Node 0 (the request's pending token) is accepted;
// from an accepted node the walk goes to its lowest child whose drafted token
// is the one sampled there, and ends where there is none. Children come after
// their parent, so each step searches behind the node it stands on: all steps
// together read the tree about once. What bounds it is that chain of steps.
__global__ __launch_bounds__(64) void tree_accept_kernel(AcceptArgs a) {
  __shared__ int32_t parent[kMaxTreeNodes], draft[kMaxTreeNodes], sampled[kMaxTreeNodes];
  const int b = static_cast<int>(blockIdx.x), lane = threadIdx.x;
  const int r0 = a.node_start[b], r1 = a.node_start[b + 1];
  const bool valid = r0 >= 0 && r1 >= r0 && r1 <= a.rows && r1 - r0 <= a.max_nodes;
  const int n = valid ? r1 - r0 : 0;
  int32_t *path = a.path + static_cast<size_t>(b) * a.path_stride;
  for (int i = lane; i < n; i += 64) {
    parent[i] = a.parents[r0 + i];
    draft[i] = a.draft_tokens[r0 + i];
    sampled[i] = a.sampled_tokens[r0 + i];
  }
  __syncthreads();
  int count = 0, next = -1;
  if (n > 0) {
    int at = 0;
    for (;;) {  // at grows every turn
      if (lane == 0) path[count] = at;
      ++count;
      next = sampled[at];
      int child = n;
      for (int c0 = (at + 1) & ~63; c0 < n; c0 += 64) {
        const int c = c0 + lane;
        const unsigned long long hit = q35_ballot(c > at && c < n && parent[min(c, n - 1)] == at && draft[min(c, n - 1)] == next);
        if (hit != 0ull) {
          child = c0 + __builtin_ctzll(hit);
          break;
        }
      }
      if (child >= n) break;
      at = child;
    }
  }
  for (int j = count + lane; j < a.max_nodes; j += 64) path[j] = -1;
  if (lane == 0) {
    a.path_count[b] = count;
    a.next_token[b] = next;
  }
}

}  // namespace

hipError_t launch_tree_attention(const TreeArgs &a, hipStream_t stream) {
  const int blocks = (a.max_nodes * (a.heads / a.kv_heads) + kBlockVectors - 1) / kBlockVectors;
  const dim3 grid(a.splits, blocks * a.kv_heads, a.batch), merge(a.heads, a.max_nodes, a.batch);
#define Q35_TREE(HD)                                                                             \
  Q35_LAUNCH((tree_attention_kernel<HD>), grid, dim3(64 * kTreeWaves), 0, stream, a);            \
  if (a.splits > 1) Q35_LAUNCH((tree_merge_kernel<HD>), merge, dim3((HD) / 4), 0, stream, a);
  switch (a.head_dim) {
    case 64: Q35_TREE(64) break;
    case 128: Q35_TREE(128) break;
    case 256: Q35_TREE(256) break;
    default: return hipErrorInvalidValue;
  }
#undef Q35_TREE
  return hipGetLastError();
}

// Ranges of cache rows per request: as many as give each CU two workgroups
// (a workgroup's four wavefronts fill its SIMDs), each of whole rounds of the
// four wavefronts' tiles.
void tree_plan(int batch, int max_nodes, int max_len, int heads, int kv_heads, int cu_count, int *split_tokens, int *splits) {
  constexpr int kRound = kTileTokens * kTreeWaves;
  const long long blocks = static_cast<long long>((max_nodes * (heads / kv_heads) + kBlockVectors - 1) / kBlockVectors) * kv_heads * batch;
  const int rounds = std::max(1, (max_len + kRound - 1) / kRound);
  const int want = static_cast<int>(std::max(1LL, std::min<long long>(rounds, (2LL * cu_count + blocks - 1) / blocks)));
  const int per = (rounds + want - 1) / want;
  *split_tokens = per * kRound;
  *splits = (rounds + per - 1) / per;
}

hipError_t launch_tree_accept(const AcceptArgs &a, hipStream_t stream) {
  Q35_LAUNCH((tree_accept_kernel), dim3(a.batch), dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace q35
