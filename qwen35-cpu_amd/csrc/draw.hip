// Sampling from logits with given random numbers: per row the repetition
// penalty, then temperature T, top-k, top-p and min-p, and one draw.
//
// Tokens are ordered by value, ties to the lower token (a key: the value's
// ordered bits above the inverted token), and weigh w = exp((x - max) / T).
// Each of the cuts keeps a prefix of that order: top-k its first k tokens,
// top-p the shortest prefix that holds p of their weight, min-p those with
// w >= min_p; the shortest of them counts. The draw is the first token at
// which the running weight passes u times the kept weight. So all there is to
// find are positions in the order, by count or by running weight.
//
// Weights are whole numbers, 2^43 for the largest (from a 64-bit exponential):
// their sums do not depend on the order of the additions, so a row gives the
// same token however its slices and atomics are scheduled, and a sum of 2^20
// tokens fits 64 bits.
//
//   slices: one workgroup per 4096 tokens of a row, which it reads once into
//     registers; counts of its tokens per quarter octave of weight below its own
//     largest (bins on a grid common to the row), the bins' weights, and the
//     tokens of its topmost bins, bin by bin.
//   pick: one workgroup per row joins the slices' bins, finds the bin that
//     each cut falls in, and settles it among that bin's keys -- from the
//     slices' lists, or from the logits where a list does not reach that far.
// Rows with a small top-k ("light") need no weight below its cut: their slices
// leave out the exponentials, and the pick gathers all keys through the cut's
// bin once.
#include "q35_device.h"
#include "q35_internal.h"

namespace q35 {
namespace {

constexpr int kSliceThreads = 256, kSlicePer = 16, kSliceTokens = kSliceThreads * kSlicePer;
constexpr int kBins = 192;    // quarter octaves: a weight below 2^-44 is no whole number left
constexpr int kListed = 1024; // tokens a slice lists
constexpr int kLightTopK = 512;
constexpr int kUnitBits = 43;
constexpr double kUnit = 8796093022208.0;  // 2^43
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64;
constexpr int kParts = kPickThreads;  // parts that a bin of many keys is split into
constexpr int kSettle = 256;          // keys settled by comparing each with each
constexpr int kCached = 2048;         // keys of a light row kept in LDS
constexpr int kMaxSlices = kDrawMaxVocab / kSliceTokens;

struct DrawOptions {
  double inv_t;    // log2(e) / T
  float bin_scale; // bins per unit of x
  int top_k;       // 0: all
  float top_p, min_p;
  bool light;
};

__device__ __forceinline__ DrawOptions draw_options(const DrawArgs &a, int r) {
  DrawOptions o;
  const float t = a.temperatures != nullptr ? a.temperatures[r] : 1.0F;
  const int k = a.top_k != nullptr ? a.top_k[r] : 0;
  const float p = a.top_p != nullptr ? a.top_p[r] : 1.0F, m = a.min_p != nullptr ? a.min_p[r] : 0.0F;
  const bool greedy = !(t > 1.0e-6F);  // the largest logit, as a draw from the first token alone
  o.inv_t = 1.4426950408889634074 / (greedy ? 1.0 : static_cast<double>(t));
  o.bin_scale = fminf(fmaxf(static_cast<float>(4.0 * o.inv_t), 1.0e-30F), 1.0e30F);
  o.top_k = greedy ? 1 : max(k, 0);
  o.top_p = greedy ? 1.0F : p;
  o.min_p = greedy ? 0.0F : m;
  o.light = o.top_k > 0 && o.top_k <= kLightTopK;
  return o;
}

// A token's value: the penalized logit, -inf for NaN, +0 for -0.
__device__ __forceinline__ float draw_value(float x, int count, float penalty) {
  if (count > 0) x = x > 0.0F ? x / penalty : x * penalty;
  return x != x ? -INFINITY : x + 0.0F;
}

// Bins below the bin of the value `top` (at most kBins - 1): the bins are the
// floors of x * scale, so they fall with x whatever the rounding.
__device__ __forceinline__ float bin_floor(float x, float scale) { return floorf(x * scale); }
__device__ __forceinline__ int bins_below(float top, float y) {
  return y == top ? 0 : static_cast<int>(fminf(top - y, static_cast<float>(kBins - 1)));
}

__device__ __forceinline__ double draw_power(float x, float top, double inv_t) {
  return (static_cast<double>(x) - static_cast<double>(top)) * inv_t;
}
// 2^z in units of 2^-43, to the nearest whole number (z <= 0): 2^z = 2^n e^r with
// |r| <= ln(2) / 2, e^r by its series through r^11 (the rest is below 2^-47), and
// the rounding by an addition of 2^52, whose sum holds the number in its low bits.
__device__ __forceinline__ unsigned long long draw_weight(float x, float top, double inv_t) {
  if (x == top) return 1ull << kUnitBits;
  const double z = draw_power(x, top, inv_t);
  if (!(z > -45.0)) return 0ull;
  const double n = rint(z), r = (z - n) * 0.69314718055994530942;
  double e = 1.0 / 39916800.0;
  e = fma(e, r, 1.0 / 3628800.0);
  e = fma(e, r, 1.0 / 362880.0);
  e = fma(e, r, 1.0 / 40320.0);
  e = fma(e, r, 1.0 / 5040.0);
  e = fma(e, r, 1.0 / 720.0);
  e = fma(e, r, 1.0 / 120.0);
  e = fma(e, r, 1.0 / 24.0);
  e = fma(e, r, 1.0 / 6.0);
  e = fma(e, r, 0.5);
  e = fma(e, r, 1.0);
  e = fma(e, r, 1.0);
  const double w = ldexp(e, static_cast<int>(n) + kUnitBits) + 4503599627370496.0;
  return static_cast<unsigned long long>(__double_as_longlong(w)) & 0xfffffffffffffull;
}

// ---------------------------------------------------------------- slices
__global__ __launch_bounds__(kSliceThreads) void draw_slices_kernel(DrawArgs a, DrawScratch w) {
  __shared__ unsigned long long mass[kBins];
  __shared__ unsigned number[kBins];
  __shared__ float tops[kSliceThreads / 64];
  const int s = static_cast<int>(blockIdx.x), r = static_cast<int>(blockIdx.y), tid = threadIdx.x, lane = tid & 63;
  const int t0 = s * kSliceTokens;
  const float *logits = a.logits + static_cast<size_t>(r) * a.stride;
  const float penalty = a.penalties != nullptr ? a.penalties[r] : 1.0F;
  const int32_t *counts = a.counts != nullptr && penalty > 1.0F ? a.counts + static_cast<size_t>(r) * a.vocab : nullptr;
  const DrawOptions o = draw_options(a, r);
  float x[kSlicePer];
  int seen[kSlicePer];
#pragma unroll
  for (int i = 0; i < kSlicePer; ++i) {
    const int t = min(t0 + tid + i * kSliceThreads, a.vocab - 1);
    x[i] = logits[t];
    seen[i] = counts != nullptr ? counts[t] : 0;
  }
  if (tid < kBins) {
    mass[tid] = 0ull;
    number[tid] = 0u;
  }
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSlicePer; ++i) {
    x[i] = t0 + tid + i * kSliceThreads < a.vocab ? draw_value(x[i], seen[i], penalty) : -INFINITY;
    top = fmaxf(top, x[i]);
  }
  top = group_max<64>(top);
  if (lane == 0) tops[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const size_t at = static_cast<size_t>(r) * w.slices + s;
  if (tid == 0) w.top[at] = top;
  if (top == -INFINITY) return;  // whole workgroup: the pick reads nothing else of such a slice
  const float ytop = bin_floor(top, o.bin_scale);
#pragma unroll
  for (int i = 0; i < kSlicePer; ++i) {
    if (x[i] == -INFINITY) continue;
    const int bin = bins_below(ytop, bin_floor(x[i], o.bin_scale));
    atomicAdd(&number[bin], 1u);
    if (!o.light) {
      const unsigned long long m = draw_weight(x[i], top, o.inv_t);
      if (m != 0ull) atomicAdd(&mass[bin], m);
    }
  }
  __syncthreads();
  if (tid < kBins && !o.light) w.mass[at * kBins + tid] = mass[tid];
  // inclusive counts over the bins: three bins per lane of the first wavefront
  if (tid < 64) {
    unsigned n[3];
#pragma unroll
    for (int e = 0; e < 3; ++e) n[e] = number[3 * lane + e];
    n[1] += n[0];
    n[2] += n[1];
    unsigned run = n[2];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const unsigned up = __shfl(run, max(lane - d, 0), 64);
      if (lane >= d) run += up;
    }
    const unsigned before = run - n[2];
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      const unsigned end = before + n[e];
      w.ends[at * kBins + 3 * lane + e] = static_cast<uint16_t>(end);
      // the bin's first place in the list, where the list holds all of it (and
      // some of it may be among the first top_k)
      const unsigned first = e == 0 ? before : before + n[e - 1];
      number[3 * lane + e] = end <= kListed && !(o.light && first >= static_cast<unsigned>(o.top_k)) ? first : 0x80000000u;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSlicePer; ++i) {
    if (x[i] == -INFINITY) continue;
    const int bin = bins_below(ytop, bin_floor(x[i], o.bin_scale));
    if ((number[bin] & 0x80000000u) != 0u) continue;
    const unsigned place = atomicAdd(&number[bin], 1u);
    w.list[at * kListed + place] = static_cast<uint16_t>(tid + i * kSliceThreads);
  }
}

// ------------------------------------------------------------------ pick
struct PickShared {
  float top[kMaxSlices];
  int below[kMaxSlices];                   // bins from the row's top bin to the slice's
  int first[kMaxSlices], end[kMaxSlices];  // the places of a bin's (or of several bins') tokens in each slice's list
  unsigned long long mass[kBins];          // running weight through each bin
  unsigned number[kBins];                  // running count
  unsigned long long part_mass[kParts], cache[kCached];
  unsigned part_number[kParts];
  unsigned long long key[kSettle], weight[kSettle];
  float wave_top[kPickWaves];
  unsigned long long wave_mass[kPickWaves];
  unsigned wave_number[kPickWaves];
  unsigned found;
  int where;
  unsigned long long result_key, result_mass;
};

enum : int { kByCount = 0, kByMass = 1, kByKey = 2 };

struct Picker {
  const DrawArgs &a;
  const DrawScratch &w;
  PickShared &sh;
  DrawOptions o;
  int r, slices;
  float top, ytop, penalty;
  const float *logits;
  const int32_t *counts;
  int cached = -1;  // keys in sh.cache, those of the bins through cached_bin (-1: none)
  int cached_bin = -1;

  __device__ __forceinline__ int bin_at(float x) const { return bins_below(ytop, bin_floor(x, o.bin_scale)); }

  // The list places of bins g0 .. g1 in every slice (then a barrier).
  __device__ __forceinline__ void places(int g0, int g1) const {
    for (int s = threadIdx.x; s < slices; s += kPickThreads) {
      int first = 0, end = 0;
      // the slice's bins: its own bin b is the row's b + below, the last takes
      // all that lies further down
      const int b0 = max(g0 - sh.below[s], 0), b1 = g1 == kBins - 1 ? kBins - 1 : g1 - sh.below[s];
      if (sh.top[s] != -INFINITY && b1 >= 0 && (g1 == kBins - 1 || g0 - sh.below[s] < kBins - 1)) {
        const uint16_t *ends = w.ends + (static_cast<size_t>(r) * w.slices + s) * kBins;
        // (a slice's last bin holds bins of the row beyond g1 too, so a range that
        // ends in it, short of the row's last, takes only what lies before)
        const int last = g1 == kBins - 1 ? kBins - 1 : min(b1, kBins - 2);
        first = b0 > 0 ? ends[b0 - 1] : 0;
        end = ends[last];
      }
      sh.first[s] = first;
      sh.end[s] = max(first, end);
    }
    __syncthreads();
  }
  // f(key) for every key of bins g0 .. g1, from the places in sh.first / sh.end
  template <typename F>
  __device__ __forceinline__ void for_each(int g0, int g1, F f) const {
    if (cached >= 0 && g1 <= cached_bin) {
      for (int e = threadIdx.x; e < cached; e += kPickThreads) {
        const unsigned long long k = sh.cache[e];
        const int bin = bin_at(argmax_key_value(k));
        if (bin >= g0 && bin <= g1) f(k);
      }
      return;
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int s = wave; s < slices; s += kPickWaves) {
      const int first = sh.first[s], end = sh.end[s], t0 = s * kSliceTokens;
      if (first >= end) continue;
      if (end <= kListed && !(o.light && first >= o.top_k)) {
        const uint16_t *list = w.list + (static_cast<size_t>(r) * w.slices + s) * kListed;
        for (int e = first + lane; e < end; e += 64) {
          const int t = t0 + list[e];
          f(argmax_key(draw_value(logits[t], counts != nullptr ? counts[t] : 0, penalty), static_cast<uint32_t>(t)));
        }
      } else {
        constexpr int U = 8;
        for (int e = lane; e < kSliceTokens && t0 + e < a.vocab; e += 64 * U) {
          float x[U];
          int seen[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int t = min(t0 + e + 64 * u, a.vocab - 1);
            x[u] = logits[t];
            seen[u] = counts != nullptr ? counts[t] : 0;
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int t = t0 + e + 64 * u;
            const float v = draw_value(x[u], seen[u], penalty);
            if (e + 64 * u >= kSliceTokens || t >= a.vocab || v == -INFINITY) continue;
            const int bin = bin_at(v);
            if (bin >= g0 && bin <= g1) f(argmax_key(v, static_cast<uint32_t>(t)));
          }
        }
      }
    }
  }

  // Inclusive sums of the threads' (m, c) in thread order.
  __device__ __forceinline__ void running(unsigned long long &m, unsigned &c) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const unsigned long long um = __shfl(m, max(lane - d, 0), 64);
      const unsigned uc = __shfl(c, max(lane - d, 0), 64);
      if (lane >= d) {
        m += um;
        c += uc;
      }
    }
    if (lane == 63) {
      sh.wave_mass[wave] = m;
      sh.wave_number[wave] = c;
    }
    __syncthreads();
    for (int v = 0; v < wave; ++v) {
      m += sh.wave_mass[v];
      c += sh.wave_number[v];
    }
  }
  // sh.mass / sh.number from each bin's own to running sums
  __device__ __forceinline__ void running_bins() const {
    const int tid = threadIdx.x;
    __syncthreads();
    unsigned long long m = tid < kBins ? sh.mass[tid] : 0ull;
    unsigned c = tid < kBins ? sh.number[tid] : 0u;
    running(m, c);
    if (tid < kBins) {
      sh.mass[tid] = m;
      sh.number[tid] = c;
    }
    __syncthreads();
  }

  // The position in bin g at which the running count or weight reaches
  // `target` (kByCount, kByMass), or of the last key at or above it (kByKey):
  // sh.result_key and sh.result_mass, the running weight through it.
  __device__ void settle(int g, int mode, unsigned long long target) const {
    const int tid = threadIdx.x;
    unsigned long long before = g > 0 ? sh.mass[g - 1] : 0ull;
    unsigned above = g > 0 ? sh.number[g - 1] : 0u;
    int n = static_cast<int>(sh.number[g] - above);
    __syncthreads();  // the last settle's readers are done
    if (!(cached >= 0 && g <= cached_bin)) places(g, g);
    unsigned long long low = 0ull, high = ~0ull;
    if (n > kSettle && g < kBins - 1) {
      // keys of values whose x * scale may round into the bin
      const float y = ytop - static_cast<float>(g), x0 = y / o.bin_scale, x1 = (y + 1.0F) / o.bin_scale;
      const float lo = x0 - fabsf(x0) * 1.0e-6F, hi = x1 + fabsf(x1) * 1.0e-6F;
      if (lo > -INFINITY && lo < hi && hi < INFINITY) {
        low = argmax_key(lo, 0xffffffffu);
        high = argmax_key(hi, 0u);
      }
    }
    while (n > kSettle) {  // the range shrinks every turn: keys differ, so n reaches 1 at the latest
      const int shift = max(0, 54 - __builtin_clzll(high - low));
      sh.part_mass[tid] = 0ull;
      sh.part_number[tid] = 0u;
      if (tid == 0) sh.where = -1;
      __syncthreads();
      for_each(g, g, [&](unsigned long long k) {
        if (k < low || k > high) return;
        const int e = kParts - 1 - static_cast<int>((k - low) >> shift);  // descending
        atomicAdd(&sh.part_number[e], 1u);
        const unsigned long long m = draw_weight(argmax_key_value(k), top, o.inv_t);
        if (m != 0ull) atomicAdd(&sh.part_mass[e], m);
      });
      __syncthreads();
      // running sums of the parts up to each, and the part to go on in
      const unsigned long long own_m = sh.part_mass[tid];
      const unsigned own_c = sh.part_number[tid];
      unsigned long long m = own_m;
      unsigned c = own_c;
      running(m, c);
      bool here;
      if (mode == kByCount) {
        here = above + c >= target && above + c - own_c < target;
      } else if (mode == kByMass) {
        here = before + m >= target && before + m - own_m < target;
      } else {
        const unsigned long long k = target < low ? low : target > high ? high : target;
        here = tid == kParts - 1 - static_cast<int>((k - low) >> shift);
      }
      sh.part_mass[tid] = m;
      sh.part_number[tid] = c;
      if (here) sh.where = tid;
      __syncthreads();
      int e = sh.where;
      if (e < 0) {  // the keys' weights round to less than their bin's sum: the last part that weighs, or has keys
        const bool weighs = sh.part_mass[kParts - 1] != 0ull;
        for (int i = 0; i < kParts; ++i) {
          const bool more = weighs ? sh.part_mass[i] != (i > 0 ? sh.part_mass[i - 1] : 0ull)
                                   : sh.part_number[i] != (i > 0 ? sh.part_number[i - 1] : 0u);
          if (more) e = i;
        }
      }
      const unsigned long long m0 = e > 0 ? sh.part_mass[e - 1] : 0ull;
      const unsigned c0 = e > 0 ? sh.part_number[e - 1] : 0u;
      before += m0;
      above += c0;
      n = static_cast<int>(sh.part_number[e] - c0);
      low += static_cast<unsigned long long>(kParts - 1 - e) << shift;
      const unsigned long long last = low + ((1ull << shift) - 1ull);
      high = last < high ? last : high;
      __syncthreads();
    }
    // the keys left, each compared with each: four threads to a key
    if (tid == 0) {
      sh.found = 0u;
      sh.result_key = 0ull;
      sh.result_mass = before;
    }
    __syncthreads();
    for_each(g, g, [&](unsigned long long k) {
      if (k < low || k > high) return;
      const unsigned i = atomicAdd(&sh.found, 1u);
      sh.key[i] = k;
      sh.weight[i] = draw_weight(argmax_key_value(k), top, o.inv_t);
    });
    __syncthreads();
    const int i = tid >> 2, q = tid & 3;
    const unsigned long long mine = i < n ? sh.key[i] : 0ull;
    unsigned long long m = 0ull;
    unsigned c = 0u;
    for (int e = q; e < n; e += 4) {
      if (sh.key[e] >= mine) {
        m += sh.weight[e];
        ++c;
      }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      m += __shfl_xor(m, d, 64);
      c += __shfl_xor(c, d, 64);
    }
    const unsigned long long own = i < n ? sh.weight[i] : 0ull;
    // without a key that meets the condition: the last one that weighs (as above)
    if (q == 0 && i < n && mode == kByMass && own != 0ull) atomicMax(&sh.result_mass, before + m);
    __syncthreads();
    const unsigned long long most = sh.result_mass;
    __syncthreads();
    if (q == 0 && i < n) {
      bool here;
      if (mode == kByCount) here = above + c == target;
      else if (mode == kByMass && most == before) here = c == 1u;
      else if (mode == kByMass) here = own != 0ull && before + m - own < target && (before + m >= target || before + m == most);
      else here = mine >= target && (c == static_cast<unsigned>(n) || !next_at_or_above(mine, target, n));
      if (here) {  // at most the bin's sum, so that no later target passes into the next bin
        sh.result_key = mine;
        sh.result_mass = before + m < sh.mass[g] ? before + m : sh.mass[g];
      }
    }
    __syncthreads();
  }
  // whether a key below `mine` is still at or above the bound
  __device__ __forceinline__ bool next_at_or_above(unsigned long long mine, unsigned long long bound, int n) const {
    bool any = false;
    for (int e = 0; e < n; ++e) any |= sh.key[e] < mine && sh.key[e] >= bound;
    return any;
  }

  // The first bin whose running count or weight reaches the target (the last
  // bin, where rounding leaves none).
  __device__ int bin_of(int mode, unsigned long long target) const {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) sh.where = kBins - 1;
    __syncthreads();
    if (tid < kBins) {
      const unsigned long long here = mode == kByCount ? sh.number[tid] : sh.mass[tid];
      const unsigned long long last = tid == 0 ? 0ull : mode == kByCount ? sh.number[tid - 1] : sh.mass[tid - 1];
      if (here >= target && last < target) sh.where = tid;
    }
    __syncthreads();
    return sh.where;
  }

  // A light row: the weights of the bins through g, and their keys where they
  // are not too many (the bins beyond hold none).
  __device__ __forceinline__ void weigh(int g) {
    const int tid = threadIdx.x, n = static_cast<int>(sh.number[g]);
    __syncthreads();
    if (tid < kBins) sh.mass[tid] = 0ull;
    if (tid == 0) sh.found = 0u;
    places(0, g);
    const bool keep = n <= kCached;
    for_each(0, g, [&](unsigned long long k) {
      const float x = argmax_key_value(k);
      const unsigned long long m = draw_weight(x, top, o.inv_t);
      if (m != 0ull) atomicAdd(&sh.mass[bin_at(x)], m);
      if (keep) sh.cache[atomicAdd(&sh.found, 1u)] = k;
    });
    __syncthreads();
    if (keep) {
      cached = n;
      cached_bin = g;
    }
    // running weights; the counts are running already
    unsigned long long m = tid < kBins ? sh.mass[tid] : 0ull;
    unsigned c = 0u;
    running(m, c);
    if (tid < kBins) sh.mass[tid] = m;
    __syncthreads();
  }
};

__global__ __launch_bounds__(kPickThreads) void draw_pick_kernel(DrawArgs a, DrawScratch w) {
  __shared__ PickShared sh;
  const int r = static_cast<int>(blockIdx.x), tid = threadIdx.x;
  const float penalty = a.penalties != nullptr ? a.penalties[r] : 1.0F;
  Picker p{a,
           w,
           sh,
           draw_options(a, r),
           r,
           w.slices,
           -INFINITY,
           0.0F,
           penalty,
           a.logits + static_cast<size_t>(r) * a.stride,
           a.counts != nullptr && penalty > 1.0F ? a.counts + static_cast<size_t>(r) * a.vocab : nullptr};
  const float u = a.uniforms[r];
  // the row's largest value and each slice's distance from it
  float top = -INFINITY;
  for (int s = tid; s < w.slices; s += kPickThreads) {
    const float x = w.top[static_cast<size_t>(r) * w.slices + s];
    sh.top[s] = x;
    top = fmaxf(top, x);
  }
  top = group_max<64>(top);
  if ((tid & 63) == 0) sh.wave_top[tid >> 6] = top;
  if (tid < kBins) {
    sh.mass[tid] = 0ull;
    sh.number[tid] = 0u;
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kPickWaves; ++v) top = fmaxf(top, sh.wave_top[v]);
  if (top == -INFINITY) {  // whole workgroup: nothing to draw from
    if (tid == 0) {
      a.out_token[r] = -1;
      if (a.out_probability != nullptr) a.out_probability[r] = 0.0F;
    }
    return;
  }
  p.top = top;
  p.ytop = bin_floor(top, p.o.bin_scale);
  for (int s = tid; s < w.slices; s += kPickThreads) sh.below[s] = bins_below(p.ytop, bin_floor(sh.top[s], p.o.bin_scale));
  __syncthreads();
  // the slices' bins, four to a thread, weights brought from each slice's
  // largest to the row's
  for (int e = tid; e < w.slices * (kBins / 4); e += kPickThreads) {
    const int s = e / (kBins / 4), bin = 4 * (e - s * (kBins / 4));
    const float x = sh.top[s];
    if (x == -INFINITY) continue;
    const size_t at = (static_cast<size_t>(r) * w.slices + s) * kBins + bin;
    const q35_u32x2 ends = *reinterpret_cast<const q35_u32x2 *>(w.ends + at);
    unsigned last = bin > 0 ? w.ends[at - 1] : 0u;
    const double scale = x == top ? 1.0 : exp2(fmax(draw_power(x, top, p.o.inv_t), -1000.0));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned end = (ends[k >> 1] >> (16 * (k & 1))) & 0xffffu, n = end - last;
      last = end;
      if (n == 0u) continue;
      const int g = min(kBins - 1, sh.below[s] + bin + k);
      atomicAdd(&sh.number[g], n);
      if (p.o.light) continue;
      const unsigned long long m = static_cast<unsigned long long>(static_cast<double>(w.mass[at + k]) * scale + 0.5);
      if (m != 0ull) atomicAdd(&sh.mass[g], m);
    }
  }
  p.running_bins();
  const unsigned total = sh.number[kBins - 1];
  const int top_k = p.o.top_k > 0 && static_cast<unsigned>(p.o.top_k) < total ? p.o.top_k : 0;
  if (p.o.light) p.weigh(p.bin_of(kByCount, top_k > 0 ? top_k : total));
  unsigned long long kept = sh.mass[kBins - 1];
  if (top_k > 0) {
    p.settle(p.bin_of(kByCount, top_k), kByCount, top_k);
    kept = sh.result_mass;
  }
  unsigned long long cut = kept;
  if (p.o.min_p > 0.0F && top != INFINITY) {
    // the smallest value that weighs min_p, rounded up to fp32
    const double least = static_cast<double>(top) + log2(fmin(static_cast<double>(p.o.min_p), 1.0)) / p.o.inv_t;
    float x = static_cast<float>(least);
    if (static_cast<double>(x) < least) x = nextafterf(x, INFINITY);
    x = fminf(x, top) + 0.0F;
    const int g = x > -INFINITY ? p.bin_at(x) : kBins - 1;
    if (x > -INFINITY && (g == 0 || sh.mass[g - 1] < cut)) {  // (else it lies beyond the first top_k)
      p.settle(g, kByKey, argmax_key(x, 0xffffffffu));
      cut = sh.result_mass < cut ? sh.result_mass : cut;
    }
  }
  if (!(p.o.top_p >= 1.0F)) {
    const double want = ceil(fmax(static_cast<double>(p.o.top_p), 0.0) * static_cast<double>(kept));
    unsigned long long target = want < 1.0 ? 1ull : static_cast<unsigned long long>(want);
    if (target > kept) target = kept;
    if (target < cut) {  // (else it lies beyond the cut there is)
      p.settle(p.bin_of(kByMass, target), kByMass, target);
      cut = sh.result_mass < cut ? sh.result_mass : cut;
    }
  }
  const double at = floor((u > 0.0F ? static_cast<double>(u) : 0.0) * static_cast<double>(cut));
  unsigned long long target = at >= static_cast<double>(cut) ? cut : static_cast<unsigned long long>(at) + 1ull;
  if (target > cut) target = cut;
  p.settle(p.bin_of(kByMass, target), kByMass, target);
  if (tid == 0) {
    const unsigned long long key = sh.result_key;
    const float x = argmax_key_value(key);
    a.out_token[r] = static_cast<int32_t>(argmax_key_index(key));
    if (a.out_probability != nullptr)
      a.out_probability[r] = static_cast<float>((x == top ? 1.0 : exp2(draw_power(x, top, p.o.inv_t))) * kUnit / static_cast<double>(cut));
  }
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

DrawScratch draw_scratch(int rows, int vocab, char *base, size_t *bytes) {
  DrawScratch w;
  w.slices = (vocab + kSliceTokens - 1) / kSliceTokens;
  const size_t n = static_cast<size_t>(rows) * w.slices;
  size_t at = 0;
  auto take = [&](size_t size) {
    char *p = base == nullptr ? nullptr : base + at;
    at += align256(size);
    return p;
  };
  w.mass = reinterpret_cast<unsigned long long *>(take(n * kBins * 8));
  w.list = reinterpret_cast<uint16_t *>(take(n * kListed * 2));
  w.ends = reinterpret_cast<uint16_t *>(take(n * kBins * 2));
  w.top = reinterpret_cast<float *>(take(n * 4));
  *bytes = at;
  return w;
}

}  // namespace

size_t draw_scratch_bytes(int rows, int vocab) {
  size_t bytes = 0;
  (void)draw_scratch(rows, vocab, nullptr, &bytes);
  return bytes;
}

hipError_t launch_draw(const DrawArgs &a, void *scratch, hipStream_t stream) {
  size_t bytes = 0;
  const DrawScratch w = draw_scratch(a.rows, a.vocab, static_cast<char *>(scratch), &bytes);
  Q35_LAUNCH((draw_slices_kernel), dim3(w.slices, a.rows), dim3(kSliceThreads), 0, stream, a, w);
  Q35_LAUNCH((draw_pick_kernel), dim3(a.rows), dim3(kPickThreads), 0, stream, a, w);
  return hipGetLastError();
}

}  // namespace q35
