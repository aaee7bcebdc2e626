// One state per row of logits, drawn at a given uniform number: bn_draw_states of include/bn_hip.h.
//
//   w_i = exp((x_i - max x) / T)                  order: x decreasing, ties by ascending index
//   A = the first k of the order                  W = sum_A w
//   P = those of A with less than p W before them in the order
//   K = those of P with w_i >= m                  state = min{i in K : sum_{j in K, j <= i} w_j > u W_K}
//
// P and K are prefixes of the order: a row's kept states are those above a threshold, a key (the logit
// as an integer that sorts like it) and, among the states on that key, an index.
//
// Rows of up to 1024 states live in the registers of a group of 1 to 64 lanes, 16 states per lane, and
// are sorted there (draw_short).  Longer rows take two launches.  The first (block_summaries) reads the
// logits once, all rows cut over the whole GPU, and leaves of every 64 states the largest key and, where
// a row's total weight will be needed, their weight relative to it.  The second (draw_long, a block per
// row) works on those: without filters the prefix sums of 1/64 of the row lead to the 64 states that are
// looked at again; with filters the largest keys of the 64s bound the threshold from below (the k largest
// of them are k states of the row), and only the 64s that reach the bound are read again.  Where more
// than 1024 states pass the bound, the threshold is found by counts and weights in bins of keys, 12 bits
// of the key at a time.
//
// Cumulative weights decide indices, so weights are doubles everywhere, summed in an order that depends
// on the row alone.  Bins are filled by atomics, whose order varies: they add integers (the weight times a
// power of two), whose sum does not.
#pragma once

#include <algorithm>
#include <type_traits>

#include "row_values.h"

namespace bn_draw {

using namespace bn_rows;

// A logit as an unsigned integer that sorts like it; -0 and +0 are one key, no state has key 0.
template <typename W>
struct KeyOf;
template <>
struct KeyOf<float> {
  using Key = uint32_t;
  static __device__ __forceinline__ Key key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  }
  static __device__ __forceinline__ float value(Key k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
  }
};
template <>
struct KeyOf<double> {
  using Key = uint64_t;
  static __device__ __forceinline__ Key key(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
  }
  static __device__ __forceinline__ double value(Key k) {
    return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
  }
};
template <typename T>
using KeyType = typename KeyOf<typename Value<T>::Wide>::Key;

template <typename T>
__device__ __forceinline__ KeyType<T> key_at(const T* x, int64_t i) {
  return KeyOf<typename Value<T>::Wide>::key(Value<T>::widen(x[i]));
}

// NaN or +inf: the row has no distribution
__device__ __forceinline__ bool undrawable(float x) { return !(x < INFINITY); }
__device__ __forceinline__ bool undrawable(double x) { return !(x < (double)INFINITY); }

struct Draws {
  const void* logits;
  int64_t rows;
  int64_t width;
  int64_t stride;
  const int64_t* counts;
  const void* uniforms;
  int32_t uniform_dtype;
  bn_draw_filters filters;
  void* block_keys;     // [rows][blocks_per_row], long rows
  double* block_sums;   // [rows][blocks_per_row]
  int64_t blocks_per_row;
  int32_t* out;
};

// A row's settings, clamped so that any value in a row's own array means something: no top-k outside
// [1, n), no top-p outside (0, 1) but "only the first" at p <= 0, min-p within [0, 1].
struct Setting {
  double temperature;  // 0: the largest logit
  int64_t top_k;       // n: off
  double top_p;        // 2: off
  double min_p;        // 0: off
  double uniform;
  int64_t n;
  bool valid;
  __device__ __forceinline__ bool has_top_k() const { return top_k < n; }
  __device__ __forceinline__ bool has_top_p() const { return top_p < 1.0; }
};

__device__ __forceinline__ int64_t row_states(const Draws& a, int64_t r) {
  if (!a.counts) return a.width;
  const int64_t n = a.counts[r];
  return n < 0 ? 0 : (n > a.width ? a.width : n);
}

__device__ __forceinline__ Setting row_setting(const Draws& a, int64_t r) {
  Setting s;
  s.n = row_states(a, r);
  s.uniform = a.uniform_dtype == BN_F32 ? (double)static_cast<const float*>(a.uniforms)[r]
                                        : static_cast<const double*>(a.uniforms)[r];
  s.temperature = a.filters.temperature_dev ? a.filters.temperature_dev[r] : a.filters.temperature;
  s.top_k = a.filters.top_k_dev ? a.filters.top_k_dev[r] : a.filters.top_k;
  s.top_p = a.filters.top_p_dev ? a.filters.top_p_dev[r] : a.filters.top_p;
  s.min_p = a.filters.min_p_dev ? a.filters.min_p_dev[r] : a.filters.min_p;
  s.valid = s.n > 0 && s.uniform >= 0.0 && s.uniform <= 1.0 && s.temperature >= 0.0 && !isinf(s.temperature);
  if (s.top_k <= 0 || s.top_k > s.n) s.top_k = s.n;
  if (!(s.top_p < 1.0)) s.top_p = 2.0;
  if (s.top_p < 0.0) s.top_p = 0.0;
  s.min_p = s.min_p > 0.0 ? fmin(s.min_p, 1.0) : 0.0;
  return s;
}

// exp((x - best) / T) for x <= best, as 2^t with t = (x - best) log2(e) / T: 2^t = 2^round(t) * 2^f with a
// polynomial of degree 10 in f (interpolating (2^f - 1) / f at the Chebyshev nodes of [-1/2, 1/2]: 6e-16
// relative, exactly 1 at f = 0).  17 double instructions, which run beside the loads that feed them; the
// library's exp took twice that.
struct Weight {
  double best;
  double rate;  // log2(e) / T; a T below 1e-290 acts like one (0 for what is below the maximum)
  __device__ __forceinline__ Weight(double best_, double temperature)
      : best(best_), rate(1.4426950408889634074 / fmax(temperature, 1e-290)) {}
  __device__ __forceinline__ double operator()(double x) const {
    const double t = fmax((x - best) * rate, -2200.0);  // 2^-2200 is 0, and -inf stays out of the polynomial
    const double whole = rint(t);
    const double f = t - whole;
    double p = 7.070977866508138e-09;
    p = fma(p, f, 1.0205905413765595e-07);
    p = fma(p, f, 1.3215451633221434e-06);
    p = fma(p, f, 1.5252672924850737e-05);
    p = fma(p, f, 0.00015403530424776529);
    p = fma(p, f, 0.0013333558200794592);
    p = fma(p, f, 0.009618129107618665);
    p = fma(p, f, 0.05550410866465167);
    p = fma(p, f, 0.24022650695910075);
    p = fma(p, f, 0.6931471805599462);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)whole);
  }
  template <typename Key>
  __device__ __forceinline__ double of_key(Key k) const;
};
template <>
__device__ __forceinline__ double Weight::of_key<uint32_t>(uint32_t k) const {
  return (*this)((double)KeyOf<float>::value(k));
}
template <>
__device__ __forceinline__ double Weight::of_key<uint64_t>(uint64_t k) const {
  return (*this)(KeyOf<double>::value(k));
}

// ---- lanes ------------------------------------------------------------------------------------

// Exclusive prefix sum over the G lanes of a group, and the group's total.
template <int G>
__device__ __forceinline__ double group_scan(double v, double* total) {
  const int lane = threadIdx.x % G;
  double upto = v;
#pragma unroll
  for (int d = 1; d < G; d <<= 1) {
    const double left = __shfl_up(upto, d, G);
    if (lane >= d) upto += left;
  }
  *total = __shfl(upto, G - 1, G);
  const double before = __shfl_up(upto, 1, G);
  return lane == 0 ? 0.0 : before;
}
template <int G, typename U, typename Combine>
__device__ __forceinline__ U group_all(U v, Combine combine) {
#pragma unroll
  for (int d = 1; d < G; d <<= 1) v = combine(v, (U)__shfl_xor(v, d, 64));
  return v;
}

// ---- a row in registers: E states in each of G lanes --------------------------------------------

// What is sorted: (key, slot) with larger keys and, on one key, lower slots first.  A 32-bit key and a
// slot below 1024 are 42 bits: as the mantissa of a double they are exchanged by one v_max_f64 and one
// v_min_f64.
struct Packed {
  double v;
  static __device__ __forceinline__ Packed make(uint32_t key, int slot) {
    const uint32_t low = (key << 10) | (uint32_t)(1023 - slot);
    return {__longlong_as_double((long long)(((uint64_t)(0x43300000u | (key >> 22)) << 32) | low))};
  }
  __device__ __forceinline__ uint32_t key() const {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return (uint32_t)(b >> 10);
  }
  __device__ __forceinline__ bool above(const Packed& o) const { return v > o.v; }
  static __device__ __forceinline__ void order(Packed& hi, Packed& lo) {
    double big, small;  // never NaN: no canonicalisation needed, which fmax would bring
    asm("v_max_f64 %0, %1, %2" : "=v"(big) : "v"(hi.v), "v"(lo.v));
    asm("v_min_f64 %0, %1, %2" : "=v"(small) : "v"(hi.v), "v"(lo.v));
    hi.v = big;
    lo.v = small;
  }
  template <int MASK>
  __device__ __forceinline__ Packed other() const { return {lane_xor<MASK>(v)}; }
  __device__ __forceinline__ Packed shuffled(int mask) const { return {__shfl_xor(v, mask, 64)}; }
};
struct Wide64 {
  uint64_t k;
  uint32_t slot;
  static __device__ __forceinline__ Wide64 make(uint64_t key, int slot) { return {key, (uint32_t)slot}; }
  __device__ __forceinline__ uint64_t key() const { return k; }
  __device__ __forceinline__ bool above(const Wide64& o) const { return k > o.k || (k == o.k && slot < o.slot); }
  static __device__ __forceinline__ void order(Wide64& hi, Wide64& lo) {
    const Wide64 a = hi, b = lo;
    const bool swap = b.above(a);
    hi = swap ? b : a;
    lo = swap ? a : b;
  }
  template <int MASK>
  __device__ __forceinline__ Wide64 other() const { return {lane_xor<MASK>(k), lane_xor<MASK>(slot)}; }
  __device__ __forceinline__ Wide64 shuffled(int mask) const {
    return {(uint64_t)__shfl_xor((unsigned long long)k, mask, 64), (uint32_t)__shfl_xor((int)slot, mask, 64)};
  }
};
template <typename Key>
struct Sorted;
template <>
struct Sorted<uint32_t> { using Type = Packed; };
template <>
struct Sorted<uint64_t> { using Type = Wide64; };

template <int MASK, int E, bool MIRROR, typename C>
__device__ __forceinline__ void exchange_lanes(C (&c)[E], bool lower) {
  C o[E];
#pragma unroll
  for (int j = 0; j < E; ++j) o[j] = c[MIRROR ? E - 1 - j : j].template other<MASK>();
#pragma unroll
  for (int j = 0; j < E; ++j)
    if (o[j].above(c[j]) == lower) c[j] = o[j];  // no two are equal: the slots differ
}

template <int STRIDE, int E, typename C>
__device__ __forceinline__ void half_cleaners(C (&c)[E], int lane) {
  if constexpr (STRIDE >= 1) {
    if constexpr (STRIDE >= E) {
      exchange_lanes<STRIDE / E, E, false>(c, (lane & (STRIDE / E)) == 0);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((j & STRIDE) == 0) C::order(c[j], c[j | STRIDE]);
    }
    half_cleaners<STRIDE / 2, E>(c, lane);
  }
}

// Bitonic sort of G * E entries, the largest first (position lane * E + j); every merge starts by comparing
// mirrored positions, so that all exchanges point the same way.
template <int K, int G, int E, typename C>
__device__ __forceinline__ void sort_group(C (&c)[E], int lane) {
  if constexpr (K <= G * E) {
    if constexpr (K <= E) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((j ^ (K - 1)) > j) C::order(c[j], c[j ^ (K - 1)]);
    } else {
      exchange_lanes<K / E - 1, E, true>(c, (lane & (K / E / 2)) == 0);
    }
    half_cleaners<K / 4, E>(c, lane);
    sort_group<K * 2, G, E>(c, lane);
  }
}

// The draw among states held by a group of lanes, key[j] of slot lane * E + j, 0 where there is none; slots
// ascend with the states' indices.  `total`: the weight that top-p is a share of, when top-k is off and
// states outside the group hold some of it; negative: the group's.  Returns the slot, the same in every lane.
template <int G, int E, typename Key>
__device__ int draw_in_group(const Key (&key)[E], const Setting& s, const Weight& weight, double row_total) {
  using C = typename Sorted<Key>::Type;
  const int lane = threadIdx.x % G;
  const bool filtered = s.has_top_k() || s.has_top_p();
  C floor = C::make(0, 0);
  // rows of one wave differ in their settings: the wave sorts if any of them has to
  if (__any(filtered)) {
    C c[E];
#pragma unroll
    for (int j = 0; j < E; ++j) c[j] = C::make(key[j], lane * E + j);
    sort_group<2, G, E>(c, lane);
    double w[E], here = 0.0, all;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[j] = lane * E + j < s.top_k && c[j].key() != 0 ? weight.of_key(c[j].key()) : 0.0;
      here += w[j];
    }
    double before = group_scan<G>(here, &all);
    const double target = s.top_p * (row_total >= 0.0 ? row_total : all);
    // the last kept entry: the first one, and those with less than the target before them
    C last = C::make(0, 0);
    bool any = false;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int at = lane * E + j;
      if (at < s.top_k && c[j].key() != 0 && (at == 0 || before < target)) {
        last = c[j];
        any = true;
      }
      before += w[j];
    }
    // kept entries are a prefix of the order: of the lanes' last ones the lowest is the threshold
    if (!any) last = C::make((Key)~(Key)0, 0);
#pragma unroll
    for (int d = 1; d < G; d <<= 1) {
      const C o = last.shuffled(d);
      if (last.above(o)) last = o;
    }
    if (filtered) floor = last;
  }
  double w[E], here = 0.0, all;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const C c = C::make(key[j], lane * E + j);
    w[j] = 0.0;
    if (key[j] != 0 && !floor.above(c)) {
      w[j] = weight.of_key(key[j]);
      if (w[j] < s.min_p) w[j] = 0.0;
    }
    here += w[j];
  }
  double upto = group_scan<G>(here, &all);
  const double target = s.uniform * all;
  int pick = INT32_MAX, last = -1;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    upto += w[j];
    if (w[j] > 0.0) {
      last = lane * E + j;
      if (upto > target && pick == INT32_MAX) pick = last;
    }
  }
  pick = group_all<G>(pick, [](int p, int q) { return p < q ? p : q; });
  last = group_all<G>(last, [](int p, int q) { return p > q ? p : q; });
  return pick == INT32_MAX ? last : pick;  // u = 1, or the sums' rounding: the last kept state
}

// The lowest slot that holds `best`.
template <int G, int E, typename Key>
__device__ __forceinline__ int first_in_group(const Key (&key)[E], Key best) {
  int first = INT32_MAX;
#pragma unroll
  for (int j = E - 1; j >= 0; --j)
    if (key[j] == best) first = (int)(threadIdx.x % G) * E + j;
  return group_all<G>(first, [](int p, int q) { return p < q ? p : q; });
}

constexpr int kShortThreads = 256;

// Rows of up to G * E states.
template <typename T, int G, int E>
__global__ void __launch_bounds__(kShortThreads) draw_short(const Draws a) {
  using W = typename Value<T>::Wide;
  using Key = KeyType<T>;
  constexpr int V = Value<T>::kVec;
  constexpr int kRows = kShortThreads / G;
  const int lane = threadIdx.x % G;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.rows; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t r = r0 + threadIdx.x / G;
    if (r >= a.rows) continue;  // whole groups leave together
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    const Setting s = row_setting(a, r);
    const int n = (int)s.n, first = lane * E;
    Key key[E];
    bool bad = false;
    Key best = 0;
    const auto take = [&](int j, T v) {
      const W wide = Value<T>::widen(v);
      bad |= undrawable(wide);
      key[j] = KeyOf<W>::key(wide);
      best = best > key[j] ? best : key[j];
    };
    if (E >= V && first + E <= n) {
#pragma unroll
      for (int k = 0; k + V <= E; k += V) {
        const Pack<T> p = load_pack(x + first + k);
#pragma unroll
        for (int j = 0; j < V; ++j) take(k + j, p.v[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        key[j] = 0;
        if (first + j < n) take(j, x[first + j]);
      }
    }
#pragma unroll
    for (int d = 1; d < G; d <<= 1) {
      const Key o = (Key)__shfl_xor((typename std::conditional<sizeof(Key) == 8, unsigned long long, unsigned>::type)best, d, 64);
      best = best > o ? best : o;
    }
    bad = group_all<G>((int)bad, [](int p, int q) { return p | q; }) != 0;
    const double largest = (double)KeyOf<W>::value(best);
    const bool valid = s.valid && !bad && !isinf(largest);
    const bool greedy = s.temperature == 0.0;
    const Weight weight(valid ? largest : 0.0, greedy ? 1.0 : s.temperature);
    int pick = draw_in_group<G, E>(key, s, weight, -1.0);
    if (greedy) pick = first_in_group<G, E>(key, best);
    if (lane == 0) a.out[r] = valid ? pick : -1;
  }
}

// ---- long rows: summaries of 64 states -----------------------------------------------------------

constexpr int kBlock = 64;          // states per summary
constexpr int kShortStates = 1024;  // rows beyond this are long
constexpr int kSummaryThreads = 256;

// A wave summarises V blocks per pack (64 lanes of V states), kPacks packs at a time.
template <typename T, int PACKS>
__global__ void __launch_bounds__(kSummaryThreads) block_summaries(const Draws a, int64_t tiles_per_row) {
  using W = typename Value<T>::Wide;
  using Key = KeyType<T>;
  constexpr int V = Value<T>::kVec;
  constexpr int kLanes = kBlock / V;  // lanes of a block
  constexpr int64_t kWaveStates = 64 * V;
  constexpr int64_t kTile = kWaveStates * PACKS * (kSummaryThreads / 64);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tiles = a.rows * tiles_per_row;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t r = tile / tiles_per_row;
    const int64_t start = (tile - r * tiles_per_row) * kTile + wave * kWaveStates * PACKS;
    const int64_t n = row_states(a, r);
    if (start >= n) continue;
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    const Setting s = row_setting(a, r);
    // top-k draws from the k largest alone; greedy rows need no weights at all
    const bool sums = !s.has_top_k() && s.temperature > 0.0;
    Key* keys = static_cast<Key*>(a.block_keys) + r * a.blocks_per_row;
    W v[PACKS][V];
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
      const int64_t i = start + k * kWaveStates + lane * V;
      if (i + V <= n) {
        const Pack<T> p = load_pack(x + i);
#pragma unroll
        for (int j = 0; j < V; ++j) v[k][j] = Value<T>::widen(p.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[k][j] = i + j < n ? Value<T>::widen(x[i + j]) : (W)-INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
      const int64_t i = start + k * kWaveStates + lane * V;
      bool bad = false;
      W best = v[k][0];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        bad |= undrawable(v[k][j]);
        best = fmax(best, v[k][j]);
      }
      best = lanes_max<kLanes>(best);
      const uint64_t bad_lanes = __ballot(bad) >> (lane & ~(kLanes - 1));
      bad = (bad_lanes & ((kLanes == 64 ? 0ull : (1ull << kLanes)) - 1)) != 0;
      double sum = 0.0;
      if (sums) {
        const Weight weight(isinf(best) || bad ? 0.0 : (double)best, s.temperature);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += weight((double)v[k][j]);
        sum = lanes_sum<kLanes>(sum);
      }
      if (lane % kLanes == 0 && i < n) {
        // the largest key there is marks a block that makes its row undrawable
        keys[i / kBlock] = bad ? (Key)~(Key)0 : KeyOf<W>::key(best);
        if (sums) a.block_sums[r * a.blocks_per_row + i / kBlock] = sum;
      }
    }
  }
}

// ---- long rows: the draw ----------------------------------------------------------------------------

constexpr int kCandidates = 1024;  // states that one wave draws among
constexpr int kListed = 512;       // blocks they may come from

template <typename Key, int THREADS>
struct Shared {
  static constexpr int kBins = 4 * THREADS;
  unsigned long long mass[kBins];
  uint32_t count[kBins];
  Key candidate[kCandidates];
  int32_t candidate_index[kCandidates];
  int32_t listed[kListed];
  double sums[THREADS / 64];
  unsigned long long words[THREADS / 64];
  long long answer[4];
};

template <int THREADS, typename U, typename Combine>
__device__ __forceinline__ U block_all(U v, unsigned long long* lds, Combine combine) {
  static_assert(sizeof(U) == 8, "one word per wave");
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = combine(v, (U)__shfl_xor(v, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) reinterpret_cast<U*>(lds)[threadIdx.x >> 6] = v;
  __syncthreads();
  U out = reinterpret_cast<U*>(lds)[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) out = combine(out, reinterpret_cast<U*>(lds)[w]);
  return out;
}
constexpr auto kMax = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
constexpr auto kMin = [](unsigned long long p, unsigned long long q) { return p < q ? p : q; };
constexpr auto kSum = [](unsigned long long p, unsigned long long q) { return p + q; };

// Exclusive prefix sum of one value per thread, and the block's total.
template <int THREADS, typename U>
__device__ __forceinline__ U block_scan(U v, unsigned long long* lds, U* total) {
  static_assert(sizeof(U) == 8, "one word per wave");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  U upto = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const U left = (U)__shfl_up(upto, d, 64);
    if (lane >= d) upto += left;
  }
  __syncthreads();
  if (lane == 63) reinterpret_cast<U*>(lds)[wave] = upto;
  __syncthreads();
  U base = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w == wave) base = sum;
    sum += reinterpret_cast<U*>(lds)[w];
  }
  *total = sum;
  U before = (U)__shfl_up(upto, 1, 64);
  if (lane == 0) before = 0;
  return base + before;
}

// Calls fn(index, key) for all n states of a row in memory.
template <typename T, int THREADS, typename Fn>
__device__ __forceinline__ void for_each_state(const T* x, int64_t n, Fn fn) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  const int64_t packs = n / V;
#pragma unroll 2
  for (int64_t k = threadIdx.x; k < packs; k += THREADS) {
    const Pack<T> p = load_pack(x + k * V);
#pragma unroll
    for (int j = 0; j < V; ++j) fn(k * V + j, KeyOf<W>::key(Value<T>::widen(p.v[j])));
  }
  const int64_t i = packs * V + threadIdx.x;
  if (i < n) fn(i, KeyOf<W>::key(Value<T>::widen(x[i])));
}

// A weight as an integer: times 2^scale_bits, which lets n of them add up within 62 bits and one be
// rounded by adding 2^52.
__device__ __forceinline__ int mass_bits(int64_t n) {
  const int room = 62 - (64 - __clzll((unsigned long long)n));
  return room < 50 ? room : 50;
}
__device__ __forceinline__ unsigned long long mass_of(double w, int bits) {
  const double shifted = ldexp(w, bits) + 4503599627370496.0;
  return (unsigned long long)__double_as_longlong(shifted) & 0xFFFFFFFFFFFFFull;
}

template <typename Key>
struct Bin {
  Key low, high;              // keys of the bin
  unsigned long long above;   // count or mass of the bins above it
  unsigned long long states;  // in it
  bool reached;               // the target is reached in it or above; else it is the lowest that holds a state
};

// The bin of keys in [low, high] in which the count (BY_MASS: the mass) from the top, `above` included,
// reaches `target`.  each(fn) calls fn(key) for every key there is; keys outside the range are passed over.
// States on `floor` (nothing lies below it) have mass floor_mass together.
template <bool BY_MASS, int THREADS, typename Key, typename Each, typename Mass>
__device__ Bin<Key> find_bin(Shared<Key, THREADS>& lds, Each each, Mass mass, Key low, Key high,
                             unsigned long long above, double target, Key floor, unsigned long long floor_mass) {
  constexpr int kBins = Shared<Key, THREADS>::kBins;
  constexpr int kLog = THREADS == 1024 ? 12 : THREADS == 512 ? 11 : 10;
  static_assert((1 << kLog) == kBins, "four bins per thread");
  const Key range = high - low;
  const int bits = range == 0 ? 0 : (sizeof(Key) == 8 ? 64 - __clzll((unsigned long long)range) : 32 - __clz((int)(uint32_t)range));
  const int shift = bits > kLog ? bits - kLog : 0;
  __syncthreads();
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    lds.count[b * THREADS + threadIdx.x] = 0;
    lds.mass[b * THREADS + threadIdx.x] = 0;
  }
  __syncthreads();
  each([&](Key k) {
    if (k < low || k > high) return;
    const int bin = (int)((k - low) >> shift);
    atomicAdd(&lds.count[bin], 1u);
    if (BY_MASS && k != floor) atomicAdd(&lds.mass[bin], mass(k));
  });
  __syncthreads();
  if (BY_MASS && threadIdx.x == 0 && floor >= low && floor <= high) lds.mass[(int)((floor - low) >> shift)] += floor_mass;
  __syncthreads();
  // thread t holds bins kBins - 1 - 4 t downwards
  unsigned long long own[4], sum = 0, total;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int bin = kBins - 1 - 4 * (int)threadIdx.x - b;
    own[b] = BY_MASS ? lds.mass[bin] : (unsigned long long)lds.count[bin];
    sum += own[b];
  }
  unsigned long long before = above + block_scan<THREADS>(sum, lds.words, &total);
  unsigned long long found = ~0ull, lowest = 0, found_above = 0, lowest_above = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int at = 4 * (int)threadIdx.x + b;
    if (lds.count[kBins - 1 - at] != 0) {
      if (found == ~0ull && (double)(before + own[b]) >= target) {
        found = (unsigned long long)at;
        found_above = before;
      }
      lowest = (unsigned long long)at + 1;
      lowest_above = before;
    }
    before += own[b];
  }
  const unsigned long long first = block_all<THREADS>(found, lds.words, kMin);
  const unsigned long long last = block_all<THREADS>(lowest, lds.words, kMax);
  const unsigned long long at = first != ~0ull ? first : last - 1;
  if (threadIdx.x == (unsigned)(at / 4)) lds.answer[0] = (long long)(first != ~0ull ? found_above : lowest_above);
  __syncthreads();
  const int bin = kBins - 1 - (int)at;
  Bin<Key> out;
  out.low = low + ((Key)bin << shift);
  const Key top = out.low + (((Key)1 << shift) - 1);
  out.high = top > high || top < out.low ? high : top;
  out.above = (unsigned long long)lds.answer[0];
  out.states = lds.count[bin];
  out.reached = first != ~0ull;
  return out;
}

// Finds the state at which a cumulative sum exceeds its target: segment sums in index order first, then the
// 64 * PER states of one segment by one wave.  sum_of(segment) is the segment's weight, weight_at(index) a
// state's (0: not kept).
template <int THREADS, int PER, typename Lds, typename SumOf, typename WeightAt>
__device__ int64_t locate(Lds& lds, int64_t segments, double uniform, SumOf sum_of, WeightAt weight_at) {
  const int64_t each = (segments + THREADS - 1) / THREADS;
  const int64_t begin = std::min<int64_t>((int64_t)threadIdx.x * each, segments);
  const int64_t end = std::min<int64_t>(begin + each, segments);
  double here = 0.0, total;
  int64_t last_filled = -1;
  for (int64_t q = begin; q < end; ++q) {
    const double s = sum_of(q);
    here += s;
    if (s > 0.0) last_filled = q;
  }
  const double left = block_scan<THREADS>(here, lds.words, &total);
  const double target = uniform * total;
  // u = 1, or the sums' rounding: the last segment that holds anything
  const bool mine = here > 0.0 && left + here > target;
  unsigned long long owner = block_all<THREADS>(mine ? (unsigned long long)threadIdx.x : ~0ull, lds.words, kMin);
  const bool none = owner == ~0ull;
  if (none) owner = block_all<THREADS>(here > 0.0 ? (unsigned long long)threadIdx.x + 1 : 0ull, lds.words, kMax) - 1;
  if (threadIdx.x == (unsigned)owner) {
    double upto = left;
    int64_t segment = last_filled;
    double before = left;
    for (int64_t q = begin; q < end; ++q) {
      const double s = sum_of(q);
      if (s > 0.0 && (q == last_filled || (!none && upto + s > target))) {
        segment = q;
        before = upto;
        break;
      }
      upto += s;
    }
    lds.answer[1] = segment;
    lds.answer[2] = __double_as_longlong(before);
  }
  __syncthreads();
  const int64_t start = lds.answer[1] * (64 * PER);
  if (threadIdx.x < 64) {
    double w[PER], sum = 0.0, all;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      w[j] = weight_at(start + (int64_t)threadIdx.x * PER + j);
      sum += w[j];
    }
    double upto = __longlong_as_double(lds.answer[2]) + group_scan<64>(sum, &all);
    int pick = INT32_MAX, last = -1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      upto += w[j];
      if (w[j] > 0.0) {
        last = (int)threadIdx.x * PER + j;
        if (!none && upto > target && pick == INT32_MAX) pick = last;
      }
    }
    pick = group_all<64>(pick, [](int p, int q) { return p < q ? p : q; });
    last = group_all<64>(last, [](int p, int q) { return p > q ? p : q; });
    if (threadIdx.x == 0) lds.answer[3] = start + (pick == INT32_MAX ? last : pick);
  }
  __syncthreads();
  return lds.answer[3];
}

template <int E, typename Key, int THREADS>
__device__ __forceinline__ int draw_among_candidates(const Shared<Key, THREADS>& lds, int count, const Setting& s,
                                                     const Weight& weight, double row_total) {
  Key key[E];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const int at = (int)(threadIdx.x & 63) * E + j;
    key[j] = at < count ? lds.candidate[at] : (Key)0;
  }
  return draw_in_group<64, E>(key, s, weight, row_total);
}

// One row, by the whole block; the same answer in every thread.
template <typename T, int THREADS>
__device__ int64_t draw_row(const Draws& a, int64_t r, Shared<KeyType<T>, THREADS>& lds) {
  using W = typename Value<T>::Wide;
  using Key = KeyType<T>;
  constexpr int V = Value<T>::kVec;
  const T* x = static_cast<const T*>(a.logits) + r * a.stride;
  Setting s = row_setting(a, r);
  if (!s.valid) return -1;
  const int64_t n = s.n;
  const int64_t blocks = (n + kBlock - 1) / kBlock;
  const Key* keys = static_cast<const Key*>(a.block_keys) + r * a.blocks_per_row;
  double* sums = a.block_sums + r * a.blocks_per_row;

  unsigned long long best = 0, least = ~0ull;
  for (int64_t b = threadIdx.x; b < blocks; b += THREADS) {
    best = kMax(best, (unsigned long long)keys[b]);
    least = kMin(least, (unsigned long long)keys[b]);
  }
  best = block_all<THREADS>(best, lds.words, kMax);
  if ((Key)best == (Key)~(Key)0) return -1;
  const double largest = (double)KeyOf<W>::value((Key)best);
  if (isinf(largest)) return -1;

  if (s.temperature == 0.0) {
    unsigned long long block = ~0ull;
    for (int64_t b = threadIdx.x; b < blocks && block == ~0ull; b += THREADS)
      if ((unsigned long long)keys[b] == best) block = (unsigned long long)b;
    block = block_all<THREADS>(block, lds.words, kMin);
    const int64_t i = (int64_t)block * kBlock + (threadIdx.x & 63);
    const uint64_t hits = __ballot(i < n && key_at(x, std::min(i, n - 1)) == (Key)best);
    return (int64_t)block * kBlock + __ffsll((unsigned long long)hits) - 1;
  }

  const Weight weight(largest, s.temperature);
  const auto block_sum_of = [&](int64_t b) { return sums[b] * weight.of_key(keys[b]); };
  if (!s.has_top_k() && !s.has_top_p() && s.min_p == 0.0)
    return locate<THREADS, 1>(lds, blocks, s.uniform, block_sum_of, [&](int64_t i) {
      return i < n ? weight.of_key(key_at(x, std::min(i, n - 1))) : 0.0;
    });

  // ---- a floor below which nothing is kept
  least = block_all<THREADS>(least, lds.words, kMin);
  const int bits = mass_bits(n);
  const auto mass = [&](Key k) { return mass_of(weight.of_key(k), bits); };
  const auto each_block = [&](auto fn) {
    for (int64_t b = threadIdx.x; b < blocks; b += THREADS) fn(keys[b]);
  };
  Key floor = 1;
  const auto raise_floor = [&](double least_weight) {  // only states of at least this weight are kept
    const double step = s.temperature * log(least_weight);
    // room for this line's roundings and the one to W
    const W bound = (W)(largest + step - 1e-6 * (fabs(largest) + fabs(step) + 1e-6 * s.temperature));
    if (bound < (W)largest && !isinf(bound)) floor = std::max(floor, KeyOf<W>::key(bound));
  };
  double row_total = -1.0;  // W, where it is the whole row's
  if (s.has_top_k()) {
    // the largest keys of k blocks are k states: the k-th state's key is not below the k-th of them
    if (s.top_k < blocks)
      floor = find_bin<false>(lds, each_block, mass, (Key)least, (Key)best, 0ull, (double)s.top_k, (Key)0, 0ull).low;
  } else if (s.has_top_p()) {
    double here = 0.0;
    const int64_t each = (blocks + THREADS - 1) / THREADS;
    for (int64_t b = (int64_t)threadIdx.x * each; b < std::min<int64_t>((int64_t)(threadIdx.x + 1) * each, blocks); ++b)
      here += block_sum_of(b);
    (void)block_scan<THREADS>(here, lds.words, &row_total);
    // the states below (1 - p) W / n hold less than the share that is left out
    const double lowest = largest + s.temperature * log(fmax((1.0 - s.top_p) * row_total / (double)n, 1e-300)) -
                          1e-6 * (fabs(largest) + 1.0);
    const W bound = (W)fmax(lowest, -(double)INFINITY);
    if (bound < (W)largest && !isinf(bound)) floor = std::max(floor, KeyOf<W>::key(bound));
    // and blocks' largest states that hold the share by themselves do too
    const Bin<Key> bin = find_bin<true>(lds, each_block, mass, (Key)least, (Key)best, 0ull,
                                        s.top_p * ldexp(row_total, bits) * (1.0 + 1e-9), (Key)0, 0ull);
    if (bin.reached) floor = std::max(floor, bin.low);
  }
  // (with top-k and top-p together W is the weight of all top-k states, those that min-p drops among them)
  if (s.min_p > 0.0 && !(s.has_top_k() && s.has_top_p())) raise_floor(s.min_p);

  // ---- few states at or above it: one wave draws among them
  {
    const int64_t each = (blocks + THREADS - 1) / THREADS;
    const int64_t begin = std::min<int64_t>((int64_t)threadIdx.x * each, blocks), end = std::min<int64_t>(begin + each, blocks);
    unsigned long long passing = 0, listed;
    for (int64_t b = begin; b < end; ++b) passing += keys[b] >= floor;
    unsigned long long at = block_scan<THREADS>(passing, lds.words, &listed);
    if (listed <= kListed) {
      for (int64_t b = begin; b < end; ++b)
        if (keys[b] >= floor) lds.listed[at++] = (int32_t)b;
      __syncthreads();
      // counts per listed block, their prefix sums, then the states in order of their index
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
      for (int q = wave; q < (int)listed; q += THREADS / 64) {
        const int64_t i = (int64_t)lds.listed[q] * kBlock + lane;
        const uint64_t hits = __ballot(i < n && key_at(x, std::min(i, n - 1)) >= floor);
        if (lane == 0) lds.count[q] = (uint32_t)__popcll(hits);
      }
      __syncthreads();
      unsigned long long mine = 0, candidates;
      constexpr int kPer = (kListed + THREADS - 1) / THREADS;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int q = (int)threadIdx.x * kPer + j;
        if (q < (int)listed) mine += lds.count[q];
      }
      unsigned long long before = block_scan<THREADS>(mine, lds.words, &candidates);
      if (candidates <= kCandidates) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int q = (int)threadIdx.x * kPer + j;
          if (q < (int)listed) {
            const uint32_t c = lds.count[q];
            lds.count[q] = (uint32_t)before;
            before += c;
          }
        }
        __syncthreads();
        for (int q = wave; q < (int)listed; q += THREADS / 64) {
          const int64_t i = (int64_t)lds.listed[q] * kBlock + lane;
          const Key k = key_at(x, std::min(i, n - 1));
          const bool hit = i < n && k >= floor;
          const uint64_t hits = __ballot(hit);
          if (hit) {
            const int to = (int)lds.count[q] + __popcll(hits & ((1ull << lane) - 1));
            lds.candidate[to] = k;
            lds.candidate_index[to] = (int32_t)i;
          }
        }
        __syncthreads();
        if (threadIdx.x < 64) {
          const int count = (int)candidates;
          int slot;
          if (count <= 64)
            slot = draw_among_candidates<1>(lds, count, s, weight, row_total);
          else if (count <= 256)
            slot = draw_among_candidates<4>(lds, count, s, weight, row_total);
          else
            slot = draw_among_candidates<16>(lds, count, s, weight, row_total);
          if (threadIdx.x == 0) lds.answer[3] = lds.candidate_index[slot];
        }
        __syncthreads();
        return lds.answer[3];
      }
    }
  }

  // ---- many: the threshold by counts and masses over the whole row
  const auto each_state = [&](auto fn) {
    for_each_state<T, THREADS>(x, n, [&](int64_t, Key k) { fn(k); });
  };
  Key threshold = floor;
  unsigned long long kept_ties = 0, ties = 0;  // of the states on `threshold`; equal: all of them
  if (s.has_top_k()) {
    Bin<Key> bin{floor, (Key)best, 0ull, 0ull, true};
    do {
      bin = find_bin<false>(lds, each_state, mass, bin.low, bin.high, bin.above, (double)s.top_k, (Key)0, 0ull);
    } while (bin.low != bin.high);
    threshold = bin.low;
    ties = bin.states;
    kept_ties = (unsigned long long)s.top_k - bin.above;
  }
  if (s.has_top_p()) {
    const Key lowest = s.has_top_k() ? threshold : (Key)0;  // the key whose states are not all in A
    const unsigned long long lowest_mass = s.has_top_k() ? kept_ties * mass(threshold) : 0ull;
    double target = s.top_p * ldexp(row_total, bits);
    if (s.has_top_k()) {
      unsigned long long all = 0;
      for_each_state<T, THREADS>(x, n, [&](int64_t, Key k) {
        if (k > threshold) all += mass(k);
      });
      target = s.top_p * (double)(block_all<THREADS>(all, lds.words, kSum) + lowest_mass);
    }
    Bin<Key> bin{threshold, (Key)best, 0ull, 0ull, true};
    do {
      bin = find_bin<true>(lds, each_state, mass, bin.low, bin.high, bin.above, target, lowest, lowest_mass);
    } while (bin.low != bin.high);
    const unsigned long long in_a = bin.low == lowest && s.has_top_k() ? kept_ties : bin.states;
    const double each = (double)mass(bin.low), above = (double)bin.above;
    unsigned long long keep = in_a;
    if (each > 0.0) keep = (unsigned long long)fmin(fmax(ceil((target - above) / each), 1.0), (double)in_a);
    while (keep > 1 && above + (double)(keep - 1) * each >= target) --keep;
    while (keep < in_a && above + (double)keep * each < target) ++keep;
    threshold = bin.low;
    ties = bin.states;
    kept_ties = keep;
  }
  int64_t last_tie = n;
  if (kept_ties < ties) {  // the index of the last kept state on the threshold
    constexpr int64_t kStep = (int64_t)THREADS * V;
    unsigned long long seen = 0;
    for (int64_t base = 0; base < n && seen < kept_ties; base += kStep) {
      const int64_t i = base + (int64_t)threadIdx.x * V;
      unsigned long long mine = 0, all;
      uint32_t on = 0;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i + j < n && key_at(x, i + j) == threshold) {
          on |= 1u << j;
          ++mine;
        }
      unsigned long long before = seen + block_scan<THREADS>(mine, lds.words, &all);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (on >> j & 1) {
          if (++before == kept_ties) lds.answer[0] = i + j;
        }
      seen += all;
    }
    __syncthreads();
    last_tie = lds.answer[0];
  }
  // ---- the draw: sums of 64 V kept states in index order (they take the place of the block sums)
  const auto kept_weight = [&](int64_t i, Key k) {
    if (k < threshold || (k == threshold && i > last_tie)) return 0.0;
    const double w = weight.of_key(k);
    return w >= s.min_p ? w : 0.0;
  };
  const int64_t segments = (n + 64 * V - 1) / (64 * V);
  __syncthreads();
  for (int64_t q = threadIdx.x >> 6; q < segments; q += THREADS / 64) {
    const int64_t i = q * 64 * V + (int64_t)(threadIdx.x & 63) * V;
    double sum = 0.0;
    if (i + V <= n) {
      const Pack<T> p = load_pack(x + i);
#pragma unroll
      for (int j = 0; j < V; ++j) sum += kept_weight(i + j, KeyOf<W>::key(Value<T>::widen(p.v[j])));
    } else {
      for (int j = 0; j < V; ++j)
        if (i + j < n) sum += kept_weight(i + j, key_at(x, i + j));
    }
    sum = lanes_sum<64>(sum);
    if ((threadIdx.x & 63) == 0) sums[q] = sum;
  }
  __syncthreads();
  return locate<THREADS, V>(lds, segments, s.uniform, [&](int64_t q) { return sums[q]; }, [&](int64_t i) {
    return i < n ? kept_weight(i, key_at(x, std::min(i, n - 1))) : 0.0;
  });
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) draw_long(const Draws a) {
  __shared__ Shared<KeyType<T>, THREADS> lds;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int64_t state = draw_row<T, THREADS>(a, r, lds);
    if (threadIdx.x == 0) a.out[r] = (int32_t)state;
    __syncthreads();
  }
}

constexpr int64_t kMaxStates = 1 << 24;
constexpr int64_t kMaxBlocks = 1 << 20;

template <typename T, int G, int E>
void launch_short(const Draws& a, hipStream_t s) {
  const int64_t per_block = kShortThreads / G;
  hipLaunchKernelGGL((draw_short<T, G, E>), dim3((uint32_t)std::min((a.rows + per_block - 1) / per_block, kMaxBlocks)),
                     dim3(kShortThreads), 0, s, a);
}

template <typename T>
void launch_long(const Draws& a, hipStream_t s) {
  constexpr int kPacks = 4;
  constexpr int64_t kTile = (int64_t)64 * Value<T>::kVec * kPacks * (kSummaryThreads / 64);
  const int64_t tiles = (a.width + kTile - 1) / kTile;
  hipLaunchKernelGGL((block_summaries<T, kPacks>), dim3((uint32_t)std::min(a.rows * tiles, kMaxBlocks)),
                     dim3(kSummaryThreads), 0, s, a, tiles);
  const dim3 grid((uint32_t)std::min(a.rows, kMaxBlocks));
  if (a.width <= 16384)
    hipLaunchKernelGGL((draw_long<T, 256>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((draw_long<T, 512>), grid, dim3(512), 0, s, a);
}

template <typename T>
hipError_t launch(const Draws& a, hipStream_t s) {
  if (a.width <= 4) launch_short<T, 1, 4>(a, s);
  else if (a.width <= 8) launch_short<T, 1, 8>(a, s);
  else if (a.width <= 16) launch_short<T, 1, 16>(a, s);
  else if (a.width <= 32) launch_short<T, 2, 16>(a, s);
  else if (a.width <= 64) launch_short<T, 4, 16>(a, s);
  else if (a.width <= 128) launch_short<T, 8, 16>(a, s);
  else if (a.width <= 256) launch_short<T, 16, 16>(a, s);
  else if (a.width <= 512) launch_short<T, 32, 16>(a, s);
  else if (a.width <= kShortStates) launch_short<T, 64, 16>(a, s);
  else launch_long<T>(a, s);
  return hipGetLastError();
}

// one translation unit per type (draw_f32.hip, ...), so that they are compiled side by side
hipError_t launch_f32(const Draws& a, hipStream_t s);
hipError_t launch_f64(const Draws& a, hipStream_t s);
hipError_t launch_f16(const Draws& a, hipStream_t s);
hipError_t launch_bf16(const Draws& a, hipStream_t s);


}  // namespace bn_draw
