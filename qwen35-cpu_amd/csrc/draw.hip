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
//   pick: one workgroup per row joins the slices' bins and finds the bins that
//     the cuts fall in. Where at most 2048 keys lie before the nearest cut, it
//     puts those in order -- from the slices' lists, or from the logits where a
//     list does not reach that far -- and every cut and the draw are searches in
//     their running weights. Else each cut is settled among its own bin's keys.
// Rows with a small top-k ("light") need no weight below its cut: their slices
// leave out the exponentials.
//
// The logits (and counts) have to be read once; what bounds many rows is that
// stream, a few rows the chain of dependent steps of two launches. Over 248320
// tokens:
//   256 rows with counts, top-k, top-p and min-p mixed: 110 us, 4.6 TB/s (the
//     slices 101 us, 5.0 TB/s; the pick's rows one to a CU, 15 us);
//   16 rows of a nucleus without top-k: 28 us (slices 15, 5 of them the
//     exponentials in fp64; pick 13: some 1100 keys in order);
//   1 row, top-k 20: 17 us (slices 7, pick 10).
#include "q35_device.h"
#include "q35_internal.h"

namespace q35 {
namespace {

constexpr int kSliceThreads = 256, kSlicePer = 16, kSliceTokens = kSliceThreads * kSlicePer;
constexpr int kBins = 192;    // quarter octaves: a weight below 2^-44 is no whole number left
constexpr int kListed = 1024; // tokens a slice lists
// Light rows: without the rule one row of top-k 20 takes 21 instead of 17 us, 256
// mixed rows 149 instead of 111. A slice lists all that such rows need, but for
// ties and for a cut in the row's last bin, which takes all that lies further down.
constexpr int kLightTopK = 512;
constexpr int kUnitBits = 43;
constexpr double kUnit = 8796093022208.0;  // 2^43
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64;
constexpr int kParts = kPickThreads;  // parts that a bin of many keys is split into
constexpr int kSettle = 256;          // keys settled by comparing each with each
// Keys put in order at once, two per thread. (Settling each cut in its own bin
// instead: one row of top-k 20 45 against 18 us, 16 rows of a nucleus 53 against
// 28.)
constexpr int kOrdered = 2 * kPickThreads;
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
// 2^(z + shift) for z in [-1000, 0]: 2^z = 2^n e^r with |r| <= ln(2) / 2, e^r by
// its series through r^11 (the rest is below 2^-47).
__device__ __forceinline__ double draw_exp2(double z, int shift) {
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
  return ldexp(e, static_cast<int>(n) + shift);
}
// A weight in units of 2^-43, to the nearest whole number: rounded by an
// addition of 2^52, whose sum holds the number in its low bits.
__device__ __forceinline__ unsigned long long draw_weight(float x, float top, double inv_t) {
  if (x == top) return 1ull << kUnitBits;
  const double z = draw_power(x, top, inv_t);
  if (!(z > -45.0)) return 0ull;
  return static_cast<unsigned long long>(__double_as_longlong(draw_exp2(z, kUnitBits) + 4503599627370496.0)) & 0xfffffffffffffull;
}

// ---------------------------------------------------------------- slices
typedef unsigned Four __attribute__((vector_size(16), aligned(4)));

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
  // four tokens at a time (rows need not be aligned to more than 4 bytes, which
  // such loads take); the row's last slice token by token
  auto token = [&](int i) { return 4 * (tid + (i >> 2) * kSliceThreads) + (i & 3); };
  if (t0 + kSliceTokens <= a.vocab) {
#pragma unroll
    for (int i = 0; i < kSlicePer; i += 4) {
      const Four v = *reinterpret_cast<const Four *>(logits + t0 + token(i));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i + e] = __uint_as_float(v[e]);
    }
#pragma unroll
    for (int i = 0; i < kSlicePer; i += 4) {
      Four v = {0u, 0u, 0u, 0u};
      if (counts != nullptr) v = *reinterpret_cast<const Four *>(counts + t0 + token(i));
#pragma unroll
      for (int e = 0; e < 4; ++e) seen[i + e] = static_cast<int>(v[e]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kSlicePer; ++i) {
      const int t = min(t0 + token(i), a.vocab - 1);
      x[i] = logits[t];
      seen[i] = counts != nullptr ? counts[t] : 0;
    }
  }
  if (tid < kBins) {
    mass[tid] = 0ull;
    number[tid] = 0u;
  }
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSlicePer; ++i) {
    x[i] = t0 + token(i) < a.vocab ? draw_value(x[i], seen[i], penalty) : -INFINITY;
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
  unsigned nth[kSlicePer];  // the token's number in its bin
#pragma unroll
  for (int i = 0; i < kSlicePer; ++i) {
    if (x[i] == -INFINITY) continue;
    const int bin = bins_below(ytop, bin_floor(x[i], o.bin_scale));
    nth[i] = atomicAdd(&number[bin], 1u);
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
    const unsigned first = number[bin];
    if ((first & 0x80000000u) != 0u) continue;
    w.list[at * kListed + first + nth[i]] = static_cast<uint16_t>(token(i));
  }
}

// ------------------------------------------------------------------ pick
struct PickShared {
  float top[kMaxSlices];
  int below[kMaxSlices];                     // bins from the row's top bin to the slice's
  double scale[kMaxSlices];                  // the slice's largest weight
  int first[kMaxSlices];                     // a range of bins' first place in each slice's list (-1: not listed)
  int start[kMaxSlices + 1];                 // listed tokens of the range before each slice
  unsigned long long mass[kBins];            // running weight through each bin
  unsigned number[kBins], next[kBins];       // running count; the next free place
  unsigned long long key[kOrdered], sorted[kOrdered];  // key: running weights, once sorted holds the keys
  unsigned long long part_mass[kParts];
  unsigned part_number[kParts];
  float wave_top[kPickWaves];
  unsigned long long wave_mass[kPickWaves];
  unsigned wave_number[kPickWaves];
  unsigned found;
  int where;
  unsigned long long result_key, result_mass;
};

enum : int { kByCount = 0, kByMass = 1, kByKey = 2 };

struct Picker {
  PickShared &sh;
  DrawOptions o;
  int slices, vocab;
  float top, ytop, penalty;
  const float *logits;
  const int32_t *counts;
  const uint16_t *ends, *list;  // the row's

  __device__ __forceinline__ int bin_at(float x) const { return bins_below(ytop, bin_floor(x, o.bin_scale)); }

  // The list places of bins g0 .. g1 in every slice (then a barrier).
  __device__ __forceinline__ void places(int g0, int g1) const {
    const int s = threadIdx.x;
    int first = 0, last = 0, end = 0;  // tokens before the range, before its last bin, and through it
    if (s < slices && sh.top[s] != -INFINITY) {
      // the slice's bins: its own bin b is the row's b + below, the last takes
      // all that lies further down (so a range that ends in it, short of the
      // row's last, takes only what lies before)
      const int below = sh.below[s], b0 = max(g0 - below, 0), b1 = g1 == kBins - 1 ? kBins - 1 : min(g1 - below, kBins - 2);
      if (b1 >= b0) {
        first = b0 > 0 ? ends[s * kBins + b0 - 1] : 0;
        last = b1 > b0 ? ends[s * kBins + b1 - 1] : first;
        end = max(first, static_cast<int>(ends[s * kBins + b1]));
      }
    }
    // (a light row's slice leaves out each bin behind top_k others: where the row's
    // last bin takes several of the slice's, the first of them alone says nothing)
    const bool listed = end <= kListed && !(o.light && last >= o.top_k && end > o.top_k);
    unsigned long long unused = 0ull;
    unsigned through = listed ? end - first : 0;
    running(unused, through);
    if (s < slices) {
      sh.first[s] = listed || first == end ? first : -1;
      sh.start[s + 1] = static_cast<int>(through);
    }
    if (s == 0) sh.start[0] = 0;
    __syncthreads();
  }
  // f(key) for every key of bins g0 .. g1, from what places() left
  template <typename F>
  __device__ __forceinline__ void for_each(int g0, int g1, F f) const {
    const int listed = sh.start[slices];
#pragma unroll 1
    for (int i = threadIdx.x; i < listed; i += kPickThreads) {
      int s = 0;  // the last slice that starts at or before i
#pragma unroll
      for (int step = kMaxSlices / 2; step > 0; step >>= 1)
        if (s + step < slices && sh.start[s + step] <= i) s += step;
      const int t = s * kSliceTokens + list[s * kListed + sh.first[s] + i - sh.start[s]];
      f(argmax_key(draw_value(logits[t], counts != nullptr ? counts[t] : 0, penalty), static_cast<uint32_t>(t)));
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll 1
    for (int s = wave; s < slices; s += kPickWaves) {
      if (sh.first[s] >= 0) continue;
      constexpr int U = 8;
      const int t0 = s * kSliceTokens;
#pragma unroll 1
      for (int e = lane; e < kSliceTokens && t0 + e < vocab; e += 64 * U) {
        float x[U];
        int seen[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = min(t0 + e + 64 * u, vocab - 1);
          x[u] = logits[t];
          seen[u] = counts != nullptr ? counts[t] : 0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = t0 + e + 64 * u;
          const float v = draw_value(x[u], seen[u], penalty);
          if (t >= vocab || v == -INFINITY) continue;
          const int bin = bin_at(v);
          if (bin >= g0 && bin <= g1) f(argmax_key(v, static_cast<uint32_t>(t)));
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
  // sh.mass / sh.number from each bin's own to running sums: three bins per lane
  // of the first wavefront
  __device__ __forceinline__ void running_bins() const {
    static_assert(kBins == 3 * 64, "three bins per lane");
    const int lane = threadIdx.x;
    __syncthreads();
    if (lane < 64) {
      unsigned long long m[3], run_m = 0ull;
      unsigned c[3], run_c = 0u;
#pragma unroll
      for (int e = 0; e < 3; ++e) {
        m[e] = run_m += sh.mass[3 * lane + e];
        c[e] = run_c += sh.number[3 * lane + e];
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const unsigned long long um = __shfl(run_m, max(lane - d, 0), 64);
        const unsigned uc = __shfl(run_c, max(lane - d, 0), 64);
        if (lane >= d) {
          run_m += um;
          run_c += uc;
        }
      }
#pragma unroll
      for (int e = 0; e < 3; ++e) {
        sh.mass[3 * lane + e] = run_m - m[2] + m[e];
        sh.number[3 * lane + e] = run_c - c[2] + c[e];
      }
    }
    __syncthreads();
  }

  // The keys through bin g, all n of them (at most kOrdered), in sh.sorted, and
  // their running weights in sh.key: bin by bin to begin with, then each key's
  // place by comparing it with its bin's.
  __device__ __forceinline__ void in_order(int g, int n) const {
    const int tid = threadIdx.x;
    if (tid < kBins) sh.next[tid] = tid > 0 ? sh.number[tid - 1] : 0u;
    places(0, g);
    for_each(0, g, [&](unsigned long long k) { sh.key[atomicAdd(&sh.next[bin_at(argmax_key_value(k))], 1u)] = k; });
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < n; i += kPickThreads) {
      const unsigned long long k = sh.key[i];
      const int bin = bin_at(argmax_key_value(k)), end = static_cast<int>(sh.number[bin]);
      int place = bin > 0 ? static_cast<int>(sh.number[bin - 1]) : 0;
#pragma unroll 4
      for (int e = place; e < end; ++e) place += sh.key[e] > k ? 1 : 0;
      sh.sorted[place] = k;
    }
    __syncthreads();
    static_assert(kOrdered == 2 * kPickThreads, "two keys per thread");
    unsigned long long m = 0ull, last = 0ull;
#pragma unroll 1
    for (int i = 2 * tid; i < min(n, 2 * tid + 2); ++i) m += last = draw_weight(argmax_key_value(sh.sorted[i]), top, o.inv_t);
    const bool both = 2 * tid + 1 < n;
    unsigned unused = 0u;
    running(m, unused);
    if (both) sh.key[2 * tid + 1] = m;
    if (2 * tid < n) sh.key[2 * tid] = both ? m - last : m;
    __syncthreads();
  }
  // The first of places 0 .. n - 1 that satisfies f, which holds for all after one
  // it holds for; n - 1 if none does. Every wavefront looks for itself.
  template <typename F>
  __device__ __forceinline__ int first_place(int n, F f) const {
    static_assert(kOrdered == 64 * 32, "64 lanes look at every 32nd");
    const int lane = threadIdx.x & 63;
    int e = 32 * lane + 31;
    const int c = 32 * __builtin_ctzll(q35_ballot(e >= n - 1 || f(min(e, n - 1))));
    e = c + (lane & 31);
    return c + __builtin_ctzll(q35_ballot(e >= n - 1 || f(min(e, n - 1))));
  }

  // The position in bin g at which the running count or weight reaches
  // `target` (kByCount, kByMass), or of the last key at or above it (kByKey):
  // sh.result_key and sh.result_mass, the running weight through it.
  __device__ __forceinline__ void settle(int g, int mode, unsigned long long target) const {
    const int tid = threadIdx.x;
    unsigned long long before = g > 0 ? sh.mass[g - 1] : 0ull;
    unsigned above = g > 0 ? sh.number[g - 1] : 0u;
    int n = static_cast<int>(sh.number[g] - above);
    __syncthreads();  // the last settle's readers are done
    places(g, g);
    unsigned long long low = 0ull, high = ~0ull;
    if (n > kSettle && g < kBins - 1) {
      // keys of values whose x * scale may round into the bin: a product is off by
      // 2^-24 of it, or, below 2^-126, by its whole size (-0 is in the bin of 0)
      const float y = ytop - static_cast<float>(g), x0 = y / o.bin_scale, x1 = (y + 1.0F) / o.bin_scale;
      const float tiny = 1.17549435e-38F / o.bin_scale;
      const float lo = x0 - fabsf(x0) * 1.0e-6F - tiny, hi = x1 + fabsf(x1) * 1.0e-6F + tiny;
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
      sh.sorted[i] = draw_weight(argmax_key_value(k), top, o.inv_t);
    });
    __syncthreads();
    const int i = tid >> 2, q = tid & 3;
    const unsigned long long mine = i < n ? sh.key[i] : 0ull;
    unsigned long long m = 0ull;
    unsigned c = 0u;
    for (int e = q; e < n; e += 4) {
      if (sh.key[e] >= mine) {
        m += sh.sorted[e];
        ++c;
      }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      m += __shfl_xor(m, d, 64);
      c += __shfl_xor(c, d, 64);
    }
    const unsigned long long own = i < n ? sh.sorted[i] : 0ull;
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
  __device__ __forceinline__ int bin_of(int mode, unsigned long long target) const {
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

  // A light row: the running weights of the bins through g (the bins beyond hold
  // none); the counts are running already.
  __device__ __forceinline__ void weigh(int g) const {
    const int tid = threadIdx.x;
    if (tid < kBins) sh.mass[tid] = 0ull;
    places(0, g);
    for_each(0, g, [&](unsigned long long k) {
      const float x = argmax_key_value(k);
      const unsigned long long m = draw_weight(x, top, o.inv_t);
      if (m != 0ull) atomicAdd(&sh.mass[bin_at(x)], m);
    });
    __syncthreads();
    unsigned long long m = tid < kBins ? sh.mass[tid] : 0ull;
    unsigned unused = 0u;
    running(m, unused);
    if (tid < kBins) sh.mass[tid] = m;
    __syncthreads();
  }
};

// The place of a drawn number in a weight of `cut`: 1 .. cut.
__device__ __forceinline__ unsigned long long draw_target(float u, unsigned long long cut) {
  const double at = floor((u > 0.0F ? static_cast<double>(u) : 0.0) * static_cast<double>(cut));
  return at >= static_cast<double>(cut) ? cut : min(static_cast<unsigned long long>(at) + 1ull, cut);
}
__device__ __forceinline__ unsigned long long draw_nucleus(float top_p, unsigned long long kept) {
  const double want = ceil(fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(kept));
  return want < 1.0 ? 1ull : min(static_cast<unsigned long long>(want), kept);
}

// The draw where a cut has too many keys before it to put them in order: every
// cut is settled in its own bin. Leaves the key in sh.result_key and returns the
// weight drawn from. (Apart from the kernel, whose instructions are all fetched
// anew by every launch: this is the part that it seldom reaches.)
__device__ __attribute__((noinline)) unsigned long long draw_settled(Picker p, unsigned top_k, unsigned total, float least, float u) {
  PickShared &sh = p.sh;
  if (p.o.light) p.weigh(p.bin_of(kByCount, top_k > 0u ? top_k : total));
  unsigned long long kept = sh.mass[kBins - 1];
  unsigned long long cut = kept;
  // the first top_k, the keys from `least` on, the nucleus, the drawn one
#pragma unroll 1
  for (int step = 0; step < 4; ++step) {
    int mode = kByMass, g = 0;
    unsigned long long target = 0ull;
    if (step == 0) {
      if (top_k == 0u) continue;
      mode = kByCount;
      target = top_k;
    } else if (step == 1) {
      if (least == -INFINITY) continue;
      g = p.bin_at(least);
      if (g > 0 && sh.mass[g - 1] >= cut) continue;  // beyond the first top_k
      mode = kByKey;
      target = argmax_key(least, 0xffffffffu);
    } else if (step == 2) {
      if (p.o.top_p >= 1.0F) continue;
      target = draw_nucleus(p.o.top_p, kept);
      if (target >= cut) continue;
    } else {
      target = draw_target(u, cut);
    }
    if (mode != kByKey) g = p.bin_of(mode, target);
    p.settle(g, mode, target);
    if (step == 0) kept = cut = sh.result_mass;
    else if (step < 3 && sh.result_mass < cut) cut = sh.result_mass;
  }
  return cut;
}

__global__ __launch_bounds__(kPickThreads) void draw_pick_kernel(DrawArgs a, DrawScratch w) {
  __shared__ PickShared sh;
  const int r = static_cast<int>(blockIdx.x), tid = threadIdx.x, slices = w.slices;
  const size_t row = static_cast<size_t>(r) * slices;
  const float penalty = a.penalties != nullptr ? a.penalties[r] : 1.0F;
  Picker p{sh,
           draw_options(a, r),
           slices,
           a.vocab,
           -INFINITY,
           0.0F,
           penalty,
           a.logits + static_cast<size_t>(r) * a.stride,
           a.counts != nullptr && penalty > 1.0F ? a.counts + static_cast<size_t>(r) * a.vocab : nullptr,
           w.ends + row * kBins,
           w.list + row * kListed};
  const float u = a.uniforms[r];
  // the slices' bins, four to a thread, U times; the first are asked for together
  // with the slices' largest values
  constexpr int U = 3, kFours = kBins / 4;
  const int fours = slices * kFours;
  q35_u32x2 ends[U];
  unsigned last[U];
  q35_u64x2 mass[U][2];
  auto ask = [&](int e0) {
#pragma unroll
    for (int v = 0; v < U; ++v) {
      const int at = 4 * min(e0 + v * kPickThreads, fours - 1);
      ends[v] = *reinterpret_cast<const q35_u32x2 *>(p.ends + at);
      last[v] = p.ends[max(at - 1, 0)];
      if (p.o.light) continue;
      mass[v][0] = *reinterpret_cast<const q35_u64x2 *>(w.mass + row * kBins + at);
      mass[v][1] = *reinterpret_cast<const q35_u64x2 *>(w.mass + row * kBins + at + 2);
    }
  };
  // the row's largest value and each slice's distance from it
  const float own = tid < slices ? w.top[row + tid] : -INFINITY;
  ask(tid);
  float top = group_max<64>(own);
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
  if (tid < slices) {
    sh.top[tid] = own;
    sh.below[tid] = bins_below(p.ytop, bin_floor(own, p.o.bin_scale));
    sh.scale[tid] = own == top ? 1.0 : draw_exp2(fmax(draw_power(own, top, p.o.inv_t), -1000.0), 0);
  }
  __syncthreads();
  // weights brought from each slice's largest to the row's
#pragma unroll 1
  for (int e0 = tid; e0 < fours; e0 += U * kPickThreads) {
    if (e0 != tid) ask(e0);
#pragma unroll
    for (int v = 0; v < U; ++v) {
      const int e = e0 + v * kPickThreads, s = e / kFours, bin = 4 * (e - s * kFours);
      if (e >= fours || sh.top[s] == -INFINITY) continue;
      unsigned before = bin > 0 ? last[v] : 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned end = (ends[v][k >> 1] >> (16 * (k & 1))) & 0xffffu, n = end - before;
        before = end;
        if (n == 0u) continue;
        const int g = min(kBins - 1, sh.below[s] + bin + k);
        atomicAdd(&sh.number[g], n);
        if (p.o.light) continue;
        const unsigned long long own_mass = mass[v][k >> 1][k & 1];
        const unsigned long long m = static_cast<unsigned long long>(static_cast<double>(own_mass) * sh.scale[s] + 0.5);
        if (m != 0ull) atomicAdd(&sh.mass[g], m);
      }
    }
  }
  p.running_bins();
  const unsigned total = sh.number[kBins - 1];
  const unsigned top_k = p.o.top_k > 0 && static_cast<unsigned>(p.o.top_k) < total ? p.o.top_k : 0u;
  // the smallest value that weighs min_p, rounded up to fp32 (-inf: no such cut)
  float least = -INFINITY;
  if (p.o.min_p > 0.0F && top != INFINITY) {
    const double x = static_cast<double>(top) + log2(fmin(static_cast<double>(p.o.min_p), 1.0)) / p.o.inv_t;
    least = static_cast<float>(x);
    if (static_cast<double>(least) < x) least = nextafterf(least, INFINITY);
    // (at an infinite temperature every weight is 1)
    least = p.o.inv_t > 0.0 ? fminf(least, top) + 0.0F : -INFINITY;
  }
  // The bin through which keys have to be put in order: the first top_k's, whose
  // weight the nucleus needs, or the nearest cut's, or that of the drawn key.
  const bool by_count = p.o.light || top_k > 0u;
  int g = kBins - 1;
  if (top_k > 0u) {
    g = p.bin_of(kByCount, top_k);
  } else if (!by_count) {
    const unsigned long long all = sh.mass[kBins - 1];
    if (least != -INFINITY) g = p.bin_at(least);
    if (!(p.o.top_p >= 1.0F)) g = min(g, p.bin_of(kByMass, draw_nucleus(p.o.top_p, all)));
    else if (least == -INFINITY) g = p.bin_of(kByMass, draw_target(u, all));
  }
  const int n = static_cast<int>(sh.number[g]);
  unsigned long long cut;
  if (n <= kOrdered) {
    p.in_order(g, n);
    const unsigned long long *running = sh.key, most = running[n - 1];
    auto place_of = [&](unsigned long long target) {
      target = min(target, most);  // (the bins' weights, rounded once more, may pass the keys')
      return p.first_place(n, [&](int e) { return running[e] >= target; });
    };
    const unsigned long long kept = top_k > 0u ? running[top_k - 1] : by_count ? most : sh.mass[kBins - 1];
    cut = kept;
    if (least != -INFINITY) {
      const unsigned long long bound = argmax_key(least, 0xffffffffu);
      const int e = p.first_place(n, [&](int i) { return sh.sorted[i] < bound; });
      cut = min(cut, running[e > 0 && sh.sorted[e] < bound ? e - 1 : e]);
    }
    if (!(p.o.top_p >= 1.0F)) cut = min(cut, running[place_of(draw_nucleus(p.o.top_p, kept))]);
    const int e = place_of(draw_target(u, cut));
    if (tid == 0) sh.result_key = sh.sorted[e];
  } else {
    cut = draw_settled(p, top_k, total, least, u);
  }
  if (tid == 0) {
    const unsigned long long key = sh.result_key;
    const float x = argmax_key_value(key);
    a.out_token[r] = static_cast<int32_t>(argmax_key_index(key));
    if (a.out_probability != nullptr)
      a.out_probability[r] = static_cast<float>((x == top ? 1.0 : draw_exp2(fmax(draw_power(x, top, p.o.inv_t), -1000.0), 0)) * kUnit / static_cast<double>(cut));
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
