// Attention for trees of drafted tokens over the paged FP16 cache, and the
// path of a tree that its sampled tokens accept.
//
// Request b has c_b context rows in the cache and behind them one row per
// drafted node. Node i sees every context row and the nodes that its mask
// names: s_t = scale * q . k_t over the rows t it sees, p = exp(s - max),
// o = sum p_t v_t / sum p_t, times sigmoid(gate); where the sum of p is zero
// (nothing seen) the output is zero.
//
// What it has to do: read every K and V row once per KV head and 128 query
// vectors, and 4 D operations per vector and row; fp32 queries and
// probabilities enter the products as two binary16 operands, which doubles the
// matrix work and keeps the error at that of fp32 sums (3e-7). Measured, heads
// of 256:
//   1 request, 611 rows of context, 5 nodes, 8 / 2 heads: 15.8 us, latency: 11
//     in the attention (as long without its products), 5 in the merge;
//   16 requests of 64 to 4096 rows, 8 to 16 nodes: 32.5 us, 27 of them in the
//     attention (73 MB, 15 us at a large copy's rate; 29 without the products);
//   64 requests of 1 to 8192 rows, 1 to 23 nodes, 16 / 4 heads: 302 us, 3.7 TB/s
//     of cache rows (1.1 GB, 220 us at a large copy's rate): loads alone take
//     248 us and products alone 243, and they overlap but for a fifth;
//   1 request of 100003 rows, 64 nodes, 16 / 4 heads: 235 to 242 us, 440 TFLOP/s
//     of the formula's, 880 of the matrix units (a large product reaches 1270);
//     matrix units and LDS are each busy for 45% of the cycles; loads alone take
//     128 us.
#include <algorithm>

#include "q35_device.h"
#include "q35_internal.h"

namespace q35 {
namespace {

constexpr int kTileTokens = 32;    // cache rows per tile
constexpr int kStageTokens = 64;   // cache rows per stage: two tiles
constexpr int kGroupVectors = 16;  // query vectors (node, head) per wavefront
constexpr int kTreeWaves = 8;
constexpr int kRowStages = kTreeWaves;  // stages whose rows are resolved at once, one per wavefront
constexpr int kBlockVectors = kTreeWaves * kGroupVectors;  // query vectors per item
// Probabilities are taken times 2^14, the largest then: as two binary16 operands
// (22 bits) they reach down to 2^-38 of it.
constexpr float kProbBinades = 14.0F;

// Products of cache rows and 16 query vectors on v_mfma_f32_16x16x32_f16, with
// the cache as the A operand in both: S^T[t][m] = sum_d k[t][d] q[m][d] and
// O^T[d][m] = sum_t v[t][d] p[m][t]. Lane l holds column m = l % 16 of either
// result, rows 4(l / 16) + i in its 4 registers, so a vector's softmax stays in
// four lanes and the probabilities of a tile's two score products are the
// second product's B operand as they lie: k slot (l / 16, i) stands for the
// tile's token 16(i / 4) + 4(l / 16) + i % 4 on both sides.
__device__ __forceinline__ int slot_token(int i, int quad) { return 16 * (i >> 2) + 4 * quad + (i & 3); }

// A score in binades, and its weight 2^(score - top + 14): the product rounded on
// its own (a contracted difference would leave the rounding of the largest score,
// which an infinite weight could come of where scores are huge), and the 14 added
// to the difference (scores from 2^25 on hold no such step: a reference of top -
// 14 gave weights up to 2^16, past binary16).
__device__ __forceinline__ float score_of(float s, float scale) {
#pragma clang fp contract(off)
  return s * scale;
}
__device__ __forceinline__ float score_weight(float s, float scale, float top) {
#pragma clang fp contract(off)
  const float x = s * scale;
  return Q35_EXP2((x - top) + kProbBinades);
}

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

// Four dims of an output: normalised by the sum l -- a zero sum saw nothing --
// and gated.
__device__ __forceinline__ void tree_store(float *dst, q35_f32x4 y, float l, bool gated, q35_f32x4 gate) {
  const float inv = 1.0F / (l == 0.0F ? 1.0F : l);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] *= inv;
    if (gated) y[e] *= sigmoid_stable(gate[e]);
  }
  *reinterpret_cast<q35_f32x4 *>(dst) = y;
}

__device__ __forceinline__ q35_f32x4 tree_gate(const float *gates, size_t at) {
  return gates != nullptr ? *reinterpret_cast<const q35_f32x4 *>(gates + at) : q35_f32x4{0.0F, 0.0F, 0.0F, 0.0F};
}

// The work is cut into items (request, KV head, block of up to 128 query
// vectors), items one after the other, and an item into units: kItemUnits for
// its beginning and end (queries, first loads and results take about as long as
// five stages) and one per stage of 64 cache rows. Workgroup w of W takes units
// [w T / W, (w + 1) T / W) of all T, so ragged contexts leave every CU the same
// share, whatever the host knew of the lengths. An item whose stages lie inside
// one workgroup's range is finished there; of the others each workgroup with
// some of the stages leaves a part (maximum, sum, unnormalised output) in one of
// its two places: the second where it has the item's first stage, else the first
// (a range has at most one of each).
constexpr int kItemUnits = 5;
__device__ __forceinline__ int item_blocks(const TreeArgs &a, const TreeRequest &r) {
  return (r.nodes * (a.heads / a.kv_heads) + kBlockVectors - 1) / kBlockVectors;
}
__device__ __forceinline__ int item_stages(const TreeRequest &r) { return (r.len + kStageTokens - 1) / kStageTokens; }
__device__ __forceinline__ long long tree_units(const TreeArgs &a, int b) {
  const TreeRequest r = tree_request(a, b);
  return static_cast<long long>(a.kv_heads) * item_blocks(a, r) * (r.nodes > 0 ? item_stages(r) + kItemUnits : 0);
}
// W: the launched workgroups, or as many as there are units, so that no range
// before the last is empty.
__device__ __forceinline__ int unit_groups(const TreeArgs &a, long long total) {
  return total < a.groups ? static_cast<int>(max(total, 1LL)) : a.groups;
}
// (Quotients of whole numbers below 2^52, as kMaxTreeUnits and at most 512
// workgroups leave them: in fp64 they round to no wrong floor -- a quotient short
// of a whole number is short by more than half a step -- and take a tenth of the
// integer code.)
__device__ __forceinline__ long long unit_begin(int w, long long total, int groups) {
  return static_cast<long long>(floor(static_cast<double>(w * total) / groups));
}
__device__ __forceinline__ int unit_group(long long unit, long long total, int groups) {
  return static_cast<int>(floor(static_cast<double>((unit + 1) * groups - 1) / static_cast<double>(total)));
}

// Four dims (from dim 4 f on) of a node's unnormalised output, and the values
// that are not finite in the rows of nodes j0 .. j1 - 1 it sees (`special`: a bit
// for each node with such values), which the products had as zeros: a row that
// weighs anything makes such a sum the value itself.
template <int HD>
__device__ __forceinline__ q35_f32x4 tree_add_special(const TreeArgs &a, const TreeRequest &rq, int b, int g, int node, int f,
                                                      const uint32_t *special, int j0, int j1, q35_f32x4 y) {
  const uint64_t *words = a.masks + static_cast<size_t>(rq.row0 + node) * a.mask_words;
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    if (!((special[j >> 5] >> (j & 31)) & 1u) || !((words[j >> 6] >> (j & 63)) & 1ull)) continue;
    const int t = rq.context + j, page = a.page_table[static_cast<size_t>(b) * a.max_pages + (t >> a.page_shift)];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.total_pages)) continue;  // NaN as it is
    const uint16_t *v = a.v_pool + static_cast<size_t>((page << a.page_shift) + (t & ((1 << a.page_shift) - 1))) * a.kv_heads * HD +
                        static_cast<size_t>(g) * HD + 4 * f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((v[e] & 0x7c00u) == 0x7c00u) y[e] += half_bits_to_float(v[e]);
  }
  return y;
}

// One workgroup of eight wavefronts. A stage's K and V rows go straight from
// the cache to LDS (16 bytes a lane, one stage of 64 rows ahead of the products;
// three stages of 32 rows ahead took 259 instead of 242 us for the long request
// and changed nothing where rows are what counts), each read once for up to 128
// vectors. Each wavefront has a group of 16 vectors and
// takes both tiles of a stage; it keeps its queries and its output in registers
// throughout, two wavefronts to a SIMD, so that one's softmax runs beside the
// other's products. (Groups of 32 vectors would read LDS half as often, but one
// wavefront then fills a SIMD's registers and nothing runs beside it. Where an
// item has at most four groups, two wavefronts to a group, a tile each, were
// slower: 316 against 302 us for 64 requests of up to 8192 rows and 23 nodes.)
//
// In LDS a K row's 16-byte pieces are rotated by xor with the row number, and a
// V row's pairs of pieces, so that the lanes of an operand (16 rows' piece, or
// pair) read distinct banks; the cache is read in the same order (whole rows,
// permuted inside). The value operands, whose lanes need one dim of several
// rows, come out of LDS by transposing reads.
template <int HD>
__global__ __launch_bounds__(64 * kTreeWaves) Q35_WAVES_PER_EU(2) void tree_attention_kernel(TreeArgs a) {
  constexpr int KS = HD / 32;    // 32-dim steps of the score product
  constexpr int PIECES = HD / 8; // 16-byte pieces of a row
  constexpr int NV = HD / 16;    // 16-dim value operands
  constexpr int LOADS = kStageTokens * PIECES / (64 * kTreeWaves);  // pieces of K (and of V) per thread and stage
  constexpr int BLOCK = kStageTokens * HD;  // halfs of a stage's K (or V)
  // (One object: with several the compiler knows which of them the loads to LDS
  // write, and waits for all of those before each read of it. The waits that
  // are needed are the ones at the barriers.)
  __shared__ struct __align__(1024) {
    uint16_t cache[4 * BLOCK];       // [stage % 2][K, V][row][dim]
    int rows[2 * kRowStages][kStageTokens];  // cache rows of two runs of stages (-1: none)
    float sums[kTreeWaves][kGroupVectors];
    long long units[kTreeWaves];
    long long first_unit;
    int first_request, special;
    uint32_t special_nodes[kMaxTreeNodes / 32];
  } sh;
  uint16_t *cache = sh.cache;
  const int tid = threadIdx.x, wave = q35_uniform(tid >> 6), lane = tid & 63, col = lane & 15, quad = lane >> 4;
  const int qpk = a.heads / a.kv_heads, w = static_cast<int>(blockIdx.x);
  const size_t kvw = static_cast<size_t>(a.kv_heads) * HD;
  const int shift = a.page_shift, pmask = (1 << shift) - 1;

  // running unit counts over the requests, a run of them per thread
  const int run = (a.batch + 64 * kTreeWaves - 1) / (64 * kTreeWaves), b0 = min(tid * run, a.batch), b1 = min(b0 + run, a.batch);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += tree_units(a, b);
  long long through = mine;  // inclusive, over the wavefront and then over all
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long long up = __shfl(through, max(lane - d, 0), 64);
    if (lane >= d) through += up;
  }
  if (lane == 63) sh.units[wave] = through;
  __syncthreads();
  long long total = 0;
  for (int v = 0; v < kTreeWaves; ++v) {
    if (v < wave) through += sh.units[v];
    total += sh.units[v];
  }
  const int ranges = unit_groups(a, total);
  const long long begin = unit_begin(min(w, ranges), total, ranges), end = unit_begin(min(w + 1, ranges), total, ranges);
  {
    long long at = through - mine;
    for (int b = b0; b < b1; ++b) {
      const long long n = tree_units(a, b);
      if (w == 0) a.first_units[b] = at;  // for the merge
      if (begin >= at && begin < at + n) {
        sh.first_request = b;
        sh.first_unit = at;
      }
      at += n;
    }
    if (w == 0 && tid == 0) a.first_units[a.batch] = total;
  }
  __syncthreads();
  if (begin >= end) return;  // whole workgroup

  int b = sh.first_request;
  long long base = sh.first_unit;  // the request's first unit
  bool again = false;  // the item's stages once more, its nodes' values that are not finite as zeros
  for (long long unit = begin; unit < end;) {
    const TreeRequest rq = tree_request(a, b);
    const int stages = item_stages(rq), blocks = item_blocks(a, rq);
    const int item_units = stages + kItemUnits;
    const long long request_units = rq.nodes > 0 ? static_cast<long long>(a.kv_heads) * blocks * item_units : 0;
    if (unit >= base + request_units) {  // (a request without units among them)
      base += request_units;
      ++b;
      continue;
    }
    const int item = static_cast<int>(unit - base) / item_units, u0 = static_cast<int>(unit - base) - item * item_units;
    const int u1 = static_cast<int>(min(static_cast<long long>(item_units), u0 + (end - unit)));
    const int s0 = max(0, u0 - kItemUnits), s1 = u1 - kItemUnits;
    unit += u1 - u0;
    if (s1 <= s0) continue;  // only the item's beginning: the next workgroup has its first stage
    const int g = item / blocks, m0 = (item - g * blocks) * kBlockVectors;

    const int vectors = rq.nodes * qpk, groups = min(kTreeWaves, (vectors - m0 + kGroupVectors - 1) / kGroupVectors);
    const bool active = wave < groups;
    const int mg = m0 + kGroupVectors * wave;

    // the lane's query vector (spare lanes repeat the last one and store nothing),
    // asked for before the pages are waited for
    const int m = min(mg + col, vectors - 1), node = m / qpk, u = m - node * qpk;
    const size_t head = static_cast<size_t>(rq.row0 + node) * a.heads + g * qpk + u;
    const uint64_t *words = a.masks + static_cast<size_t>(rq.row0 + node) * a.mask_words;
    q35_f32x4 raw[KS][2];
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i) raw[kk][i] = *reinterpret_cast<const q35_f32x4 *>(a.q + head * HD + 8 * quad + 32 * kk + 4 * i);
    q35_compiler_fence();

    const int32_t *table = a.page_table + static_cast<size_t>(b) * a.max_pages;
    // The cache rows of the stages, a run of kRowStages at a time (a token per
    // thread): token `tid` of run c (past the request: its stage's first), its
    // page, and from that its row.
    auto run_token = [&](int c) {
      const int t = kStageTokens * min(s0 + kRowStages * c + wave, s1 - 1);
      return t + lane < rq.len ? t + lane : t;
    };
    auto run_page = [&](int c) { return table[run_token(c) >> shift]; };
    auto keep_rows = [&](int c, int page) {
      sh.rows[kRowStages * (c & 1) + wave][lane] =
          static_cast<unsigned>(page) < static_cast<unsigned>(a.total_pages) ? (page << shift) + (run_token(c) & pmask) : -1;
    };
    auto stage_rows = [&](int s) { return sh.rows[(s - s0) & (2 * kRowStages - 1)]; };
    auto issue = [&](int s) {
      const int *at = stage_rows(s);
      const uint16_t *kp = a.k_pool + static_cast<size_t>(g) * HD, *vp = a.v_pool + static_cast<size_t>(g) * HD;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 64 * kTreeWaves + tid, r = e / PIECES, slot = e % PIECES;
        const size_t row = static_cast<size_t>(max(at[r], 0)) * kvw;
        uint16_t *to = cache + (s & 1) * 2 * BLOCK + 8 * (i * 64 * kTreeWaves + 64 * wave);
        Q35_LOAD_LDS16(kp + row + 8 * (slot ^ (r & (PIECES - 1))), to);
        Q35_LOAD_LDS16(vp + row + 8 * (slot ^ (2 * r & (PIECES - 1))), to + BLOCK);
      }
    };
    if (!again && tid == 0) sh.special = 0;
    if (again && tid < kMaxTreeNodes / 32) sh.special_nodes[tid] = 0u;
    keep_rows(0, run_page(0));
    int following = run_page(1);
    lds_barrier();
    issue(s0);

    q35_f16x8 qhi[KS], qlo[KS];
    float sscale;
    {
      // the vector as two binary16 operands: 22 bits under its largest value,
      // which a power of two brings to 2^8 (exact, and any fp32 size fits)
      float top = 0.0F;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(raw[kk][i >> 2][i & 3]));
      top = q35_max_rows(top);
      // (after a lift by 2^60 where it is below 2^-100, subnormal or near it)
      const bool small = top < 0x1p-100F;
      if (q35_ballot(small) != 0ull) {
        const float lift = small ? 0x1p60F : 1.0F;
        top *= lift;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
          for (int i = 0; i < 2; ++i) raw[kk][i] *= lift;
      }
      int ex = static_cast<int>(__float_as_uint(top) >> 23);  // biased
      if (ex == 0 || ex == 255) ex = 127 + 8;
      float down = __uint_as_float(static_cast<uint32_t>(127 + 8 + 127 - ex) << 23);  // 2^(8 - exponent)
      const float up = __uint_as_float(static_cast<uint32_t>(ex - 8) << 23);            // 2^(exponent - 8)
      // (neither 0 nor infinite, for products of -inf, of hidden rows, and of 0:
      // at the least the scores, 2^34 at most before, all round to 0)
      sscale = fabsf(a.scale) * up * (small ? 0x1p-60F : 1.0F) * 1.44269504088896341F;
      sscale = fminf(fmaxf(sscale, 0x1p-126F), 3.40282347e38F);
      if (a.scale < 0.0F) down = -down;  // the scores' order is then that of the products
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = raw[kk][i >> 2][i & 3] * down;
        q35_split_f16(x, qhi[kk], qlo[kk]);
      }
    }
    q35_f32x4 acc[NV];  // dims 16 n + 4 quad + i of the lane's vector
#pragma unroll
    for (int n = 0; n < NV; ++n) acc[n] = q35_f32x4{0.0F, 0.0F, 0.0F, 0.0F};
    // the lane's vector: weights are 2^(score - ref + 14); the sum is over its own tokens
    float ref = -INFINITY, sum = 0.0F;

    // 32 rows, K at cache[kb] and V a block behind it, the first of them the
    // request's row t. (Rows past the request repeat one before them under a
    // weight of 0.)
    auto tile = [&](int kb, const int *at, int t) {
      const uint32_t lost = static_cast<uint32_t>(q35_ballot(at[lane & 31] < 0));
      // (the two parts of the queries in sums of their own: four chains of
      // products that do not wait for each other)
      q35_f32x4 s[2], low[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) s[k] = low[k] = q35_f32x4{0.0F, 0.0F, 0.0F, 0.0F};
      int krow[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) krow[k] = kb + (16 * k + col) * HD + 8 * (quad ^ ((16 * k + col) & (PIECES - 1)));
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        q35_f16x8 x[2];  // piece 4 kk + quad of row r lies at that number xor r
#pragma unroll
        for (int k = 0; k < 2; ++k)
          x[k] = q35_f16x8_bits(*reinterpret_cast<const q35_u32x4 *>(cache + (krow[k] ^ (32 * kk))));
#pragma unroll
        for (int k = 0; k < 2; ++k) s[k] = Q35_MFMA_F32_16X16X32_F16(x[k], qhi[kk], s[k]);
#pragma unroll
        for (int k = 0; k < 2; ++k) low[k] = Q35_MFMA_F32_16X16X32_F16(x[k], qlo[kk], low[k]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) s[k] += low[k];
      if (t + kTileTokens > rq.context || lost != 0u) {
        const uint32_t seen = tree_visible(words, a.mask_words, t, rq.context, rq.len);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int tok = slot_token(i, quad);
          float x = (lost >> tok) & 1u ? NAN : s[i >> 2][i & 3];  // a page outside the pool
          s[i >> 2][i & 3] = (seen >> tok) & 1u ? x : -INFINITY;
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, s[i >> 2][i & 3]);
      top = q35_max_rows(top);
      const float next = fmaxf(ref, score_of(top, sscale)), least = next == -INFINITY ? 0.0F : next;
      const float keep = ref == next ? 1.0F : Q35_EXP2(ref - least);  // 0 at the first seen row
      float p[8], sums = 0.0F;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = score_weight(s[i >> 2][i & 3], sscale, least);
        sums += p[i];
      }
      sum = fmaf(sum, keep, sums);
      ref = next;
      if (q35_ballot(keep != 1.0F) != 0ull) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[n][i] *= keep;
      }
      q35_f16x8 phi, plo;
      q35_split_f16(p, phi, plo);
      // dims 16 n .. + 15 of row r: pair n of pieces, at that number xor r
      const int r = 4 * quad + (col >> 2), vrow = kb + BLOCK + r * HD + 16 * (r & (PIECES / 2 - 1)) + 4 * (col & 3);
#pragma unroll
      for (int n0 = 0; n0 < NV; n0 += 4) {  // (four at a time: no product waits for the one before)
        q35_f16x8 x[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint16_t *v = cache + (vrow ^ (16 * (n0 + n)));
          const q35_u32x2 lo = q35_lds_read_tr16(v), hi = q35_lds_read_tr16(v + 16 * HD);
          x[n] = q35_f16x8_bits(q35_u32x4{lo[0], lo[1], hi[0], hi[1]});
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n0 + n] = Q35_MFMA_F32_16X16X32_F16(x[n], phi, acc[n0 + n]);
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n0 + n] = Q35_MFMA_F32_16X16X32_F16(x[n], plo, acc[n0 + n]);
      }
    };

    // One barrier a stage: behind it the stage's loads of all wavefronts are in,
    // and every wavefront is done with the stage before, whose place the next
    // loads take. A run's pages are read most of a run before they are looked at.
    for (int s = s0; s < s1; ++s) {
      const int in_run = (s - s0) & (kRowStages - 1), c = (s - s0) / kRowStages;
      Q35_WAIT_VM(0);
      if (in_run == 1) keep_rows(c + 1, following);
      lds_barrier();
      if (s + 1 < s1) issue(s + 1);
      if (in_run == 2) following = run_page(c + 2);
      const int t = kStageTokens * s;
      if (t + kStageTokens > rq.context) {
        // An infinite or NaN value in a node's row: products with weights of 0
        // would carry it to nodes that do not see the row. Where there is one the
        // stages are gone through again, with zeros in the place of such values
        // (rows past the request, copies of a stage's first, among them).
        const int value = (s & 1) * 2 * BLOCK + BLOCK + 8 * tid, first = t - rq.context + tid / PIECES;
        bool special = false;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int j = first + i * 64 * kTreeWaves / PIECES;
          const q35_u32x4 v = *reinterpret_cast<const q35_u32x4 *>(cache + value + 8 * i * 64 * kTreeWaves);
#pragma unroll
          for (int d = 0; d < 4; ++d)
            special |= j >= 0 && j < rq.nodes && ((v[d] & 0x7c00u) == 0x7c00u || (v[d] & 0x7c000000u) == 0x7c000000u);
        }
        if (special) sh.special = 1;
        if (again) {
#pragma unroll 1
          for (int e = 0; e < 8 * LOADS; ++e) {
            const int j = first + (e >> 3) * 64 * kTreeWaves / PIECES;
            uint16_t *v = cache + value + 8 * (e >> 3) * 64 * kTreeWaves + (e & 7);
            if (j < 0 || (*v & 0x7c00u) != 0x7c00u) continue;
            *v = 0;
            if (j < rq.nodes) atomicOr(&sh.special_nodes[j >> 5], 1u << (j & 31));
          }
          lds_barrier();
        }
      }
      if (active) {
        for (int k = 0; k < 2; ++k)
          if (t + kTileTokens * k < rq.len)
            tile((s & 1) * 2 * BLOCK + kTileTokens * k * HD, stage_rows(s) + kTileTokens * k, t + kTileTokens * k);
      }
    }
    lds_barrier();  // every wavefront is done with the last stage
    if (sh.special != 0 && !again) {
      again = true;
      unit -= u1 - u0;
      continue;
    }

    // Each group's vectors through LDS, [vector][dims] with the 16-byte pieces of
    // a row at their number xor the vector, whose rows then leave whole, dealt
    // over the wavefronts.
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    constexpr int F = HD / 4;
    const bool whole = s0 == 0 && s1 == stages;
    const size_t place = (2 * static_cast<size_t>(w) + (s0 == 0 ? 1 : 0)) * kBlockVectors;
    if (active) {
      q35_f32x4 *result = reinterpret_cast<q35_f32x4 *>(cache) + static_cast<size_t>(wave) * (kGroupVectors * F) + col * F;
#pragma unroll
      for (int n = 0; n < NV; ++n) result[(4 * n + quad) ^ col] = acc[n];
      sh.sums[wave][col] = sum;
      if (!whole && quad == 0) {
        a.part_ml[2 * (place + kGroupVectors * wave + col)] = ref;
        a.part_ml[2 * (place + kGroupVectors * wave + col) + 1] = sum;
      }
    }
    lds_barrier();
    const int count = min(kBlockVectors, vectors - m0);
    const int f = lane & (F - 1);
#pragma unroll 4
    for (int v = wave * (64 / F) + lane / F; v < count; v += kTreeWaves * (64 / F)) {
      q35_f32x4 y = reinterpret_cast<q35_f32x4 *>(cache)[v * F + (f ^ (v & (kGroupVectors - 1)))];
      const int vn = (m0 + v) / qpk, vu = m0 + v - vn * qpk;
      if (again)
        y = tree_add_special<HD>(a, rq, b, g, vn, f, sh.special_nodes, max(kStageTokens * s0 - rq.context, 0),
                                 min(kStageTokens * s1 - rq.context, rq.nodes), y);
      if (whole) {
        const size_t to = (static_cast<size_t>(rq.row0 + vn) * a.heads + g * qpk + vu) * HD + 4 * f;
        tree_store(a.out + to, y, sh.sums[v / kGroupVectors][v & (kGroupVectors - 1)], a.gates != nullptr, tree_gate(a.gates, to));
      } else {
        *reinterpret_cast<q35_f32x4 *>(a.part_o + (place + v) * HD + 4 * f) = y;
      }
    }
    again = false;
    lds_barrier();  // the results and the row lists are free for the next item
  }
}

// One wavefront per (node, head): the parts of its item, weights exp(m_w - M),
// in workgroup order (the workgroups follow from the unit counts). Requests
// that are refused on the device get NaN in their rows, where those are known.
// 5 us at least, its chain of loads; 15 for 64 ragged requests, whose parts,
// gates and outputs are 50 MB (four wavefronts to a workgroup: no change).
template <int HD>
__global__ __launch_bounds__(64) void tree_merge_kernel(TreeArgs a) {
  constexpr int F = HD / 4;  // lanes past the dims repeat them
  const int i = static_cast<int>(blockIdx.x), h = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  const int lane = threadIdx.x, f = lane & (F - 1);
  const TreeRequest rq = tree_request(a, b);
  const long long total = a.first_units[a.batch], base = a.first_units[b];
  if (!rq.valid) {
    for (int r = i; r < rq.nodes; r += static_cast<int>(gridDim.x))
#pragma unroll
      for (int e = 0; e < 4; ++e)
        a.out[(static_cast<size_t>(rq.row0 + r) * a.heads + h) * HD + 4 * f + e] = __uint_as_float(0x7fc00000u);
    return;
  }
  if (i >= rq.nodes) return;
  const int qpk = a.heads / a.kv_heads, g = h / qpk, m = i * qpk + (h - g * qpk), stages = item_stages(rq);
  const long long first =
      base + (static_cast<long long>(g) * item_blocks(a, rq) + m / kBlockVectors) * (stages + kItemUnits) + kItemUnits;
  const int ranges = unit_groups(a, total);
  const int w0 = unit_group(first, total, ranges), w1 = unit_group(first + stages - 1, total, ranges);
  if (w0 == w1) return;  // finished by its workgroup
  const size_t at = m % kBlockVectors;
  auto place = [&](int w) { return (2 * static_cast<size_t>(w) + (w == w0 ? 1 : 0)) * kBlockVectors + at; };
  // 64 parts at a time, a part's maximum and sum per lane; the first parts' rows
  // and the gates are asked for together with the first of those
  constexpr int U = 4;  // parts' rows in flight
  const size_t head = (static_cast<size_t>(rq.row0 + i) * a.heads + h) * HD + 4 * f;
  q35_f32x4 x[U];
  auto ask = [&](int first_part) {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const q35_f32x4 *>(a.part_o + place(min(first_part + u, w1)) * HD + 4 * f);
  };
  q35_f32x2 ml = *reinterpret_cast<const q35_f32x2 *>(a.part_ml + 2 * place(min(w0 + lane, w1)));
  ask(w0);
  const q35_f32x4 gate = tree_gate(a.gates, head);
  q35_compiler_fence();
  float top = ml[0];
  for (int w = w0 + lane + 64; w <= w1; w += 64) top = fmaxf(top, a.part_ml[2 * place(w)]);
  top = group_max<64>(top);
  const float least = top == -INFINITY ? 0.0F : top;
  q35_f32x4 o = {0.0F, 0.0F, 0.0F, 0.0F};
  float l = 0.0F;
  for (int c = w0; c <= w1; c += 64) {
    const int n = min(64, w1 - c + 1);
    if (c > w0) ml = *reinterpret_cast<const q35_f32x2 *>(a.part_ml + 2 * place(min(c + lane, w1)));
    const float weight = lane < n ? Q35_EXP2(ml[0] - least) : 0.0F;
    l += group_sum<64>(lane < n ? ml[1] * weight : 0.0F);
    for (int k = 0; k < n; k += U) {
      if (c + k > w0) ask(c + k);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k + u >= n) break;
        const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), k + u));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[u][e], w, o[e]);
      }
    }
  }
  tree_store(a.out + head, o, l, a.gates != nullptr, gate);
}

// ------------------------------------------------------------- acceptance
// One wavefront per request. Node 0 (the request's pending token) is accepted;
// from an accepted node the walk goes to its lowest child whose drafted token
// is the one sampled there, and ends where there is none. Children come after
// their parent, so each step searches behind the node it stands on: all steps
// together read the tree about once. What bounds it is that chain of steps, and
// for a batch of any size here the launch: 1 to 64 trees of up to 64 nodes 4.1 us.
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
  const dim3 grid(a.groups), merge(a.max_nodes, a.heads, a.batch);
#define Q35_TREE(HD)                                                                  \
  Q35_LAUNCH((tree_attention_kernel<HD>), grid, dim3(64 * kTreeWaves), 0, stream, a); \
  Q35_LAUNCH((tree_merge_kernel<HD>), merge, dim3(64), 0, stream, a);
  switch (a.head_dim) {
    case 64: Q35_TREE(64) break;
    case 128: Q35_TREE(128) break;
    case 256: Q35_TREE(256) break;
    default: return hipErrorInvalidValue;
  }
#undef Q35_TREE
  return hipGetLastError();
}

// Workgroups of a launch: one per CU, but not more than the units that the
// bounds allow.
int tree_groups(int batch, int max_nodes, int max_len, int heads, int kv_heads, int cu_count) {
  return static_cast<int>(std::max(1LL, std::min<long long>(tree_request_units(max_nodes, max_len, heads, kv_heads) * batch, std::min(cu_count, 512))));
}
long long tree_request_units(int max_nodes, int max_len, int heads, int kv_heads) {
  const long long blocks = (static_cast<long long>(max_nodes) * (heads / kv_heads) + kBlockVectors - 1) / kBlockVectors;
  return blocks * kv_heads * ((static_cast<long long>(max_len) + kStageTokens - 1) / kStageTokens + kItemUnits);
}

size_t tree_workspace_bytes(const TreeArgs &a, size_t *part_o, size_t *part_ml) {
  auto align = [](size_t n) { return (n + 255) & ~static_cast<size_t>(255); };
  const size_t parts = 2 * static_cast<size_t>(a.groups) * kBlockVectors;
  *part_o = align((static_cast<size_t>(a.batch) + 1) * 8);
  *part_ml = *part_o + align(parts * a.head_dim * 4);
  return *part_ml + align(parts * 8);
}

hipError_t launch_tree_accept(const AcceptArgs &a, hipStream_t stream) {
  Q35_LAUNCH((tree_accept_kernel), dim3(a.batch), dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace q35
