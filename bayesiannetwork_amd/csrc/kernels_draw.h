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
// Rows of up to 2048 states live in the registers of a group of 1 to 64 lanes, 16 states per lane (32 beyond
// 1024), and are sorted there (draw_short).  Longer rows take two launches.  The first (block_summaries) reads
// the logits once, all rows cut over the whole GPU, and leaves of every 64 states the largest key (up to 16384
// states: of every 16) and, where a row's total weight will be needed, their weight relative to it.  The second
// (draw_long, a block per row) works on those: without filters the prefix sums of 1/64 of the row lead to the 64
// states that are looked at again; with filters the largest keys bound the threshold from below (the k largest
// of them are k states of the row), and only the pieces that reach the bound are read again.  Rows that have
// more than 512 states above the bound are left to a third kernel (draw_wide; with a small top-k the same
// block goes on); where such rows of a small batch
// have top-p alone, its passes over the row are shared by 32 blocks first (draw_wide_masses, draw_wide_sums).
//
// Cumulative weights decide indices, so weights are doubles, summed in an order that depends on the call's
// sizes alone; rows in registers take floats first, with a bound on what they are wrong by, and make the
// comparisons again in doubles that are closer than that.  Bins are filled by atomics, whose order varies: they add
// integers (the weight times a power of two), whose sum does not.  Where these decide a border they are of 2^-49 of
// the largest weight for at most 4096 states, and a pair of them (ByMassAndRest) for a whole row: a border is
// off by less than 1e-11 of the row's weight.
#pragma once

#include <algorithm>
#include <cstdint>
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

struct RowState;
struct SharedRow;

struct Draws {
  const void* logits;
  int64_t rows;
  int64_t width;
  int64_t stride;
  const int64_t* counts;
  const void* uniforms;
  int32_t uniform_dtype;
  bn_draw_filters filters;
  // long rows: the workspace
  double* block_sums;     // [rows][sums_per_row]
  RowState* row_states;   // [rows]
  SharedRow* shared;      // [rows], or null where a block does a row by itself
  void* piece_keys;       // [rows][pieces_per_row]
  int64_t pieces_per_row;
  int64_t sums_per_row;   // blocks and two more: draw_wide's segments, of 128 states at least, take two entries each
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

// exp((x - best) / T) for x <= best, as 2^t with t = (x - best) log2(e) / T: 2^t = 2^k * 2^f, k = round(t), with
// a polynomial of degree 9 in f (interpolating (2^f - 1) / f at the Chebyshev nodes of [-1/2, 1/2]: 4e-14
// relative, exactly 1 at f = 0).  k comes from adding 1.5 * 2^52, whose sum carries it in its low bits, and goes
// into an exponent by shifting: 17 of the 30 instructions that block_summaries spends on a state, and it is bound by
// their issue, 5.3 cycles each (256 x 131072 bfloat16, every row weighed: 33 us; profiles/row_operators_counters.txt).
struct Weight {
  double best;
  double rate;    // log2(e) / T; T is taken within 1e-290 .. 1e290
  double lowest;  // x - best from which on the weight is 0: t = -1023, whose exponent field is 0
  __device__ __forceinline__ Weight(double best_, double temperature)
      : best(best_), rate(1.4426950408889634074 / fmin(fmax(temperature, 1e-290), 1e290)), lowest(-1023.0 / rate) {}
  __device__ __forceinline__ double operator()(double x) const {
    constexpr double kShift = 6755399441055744.0;
    const double d = fmax(x - best, lowest);
    const double shifted = fma(d, rate, kShift);
    const double f = fma(d, rate, kShift - shifted);
    double p = 1.0203121063391729e-07;
    p = fma(p, f, 1.3255224878668817e-06);
    p = fma(p, f, 1.525268684626772e-05);
    p = fma(p, f, 0.00015403455852453838);
    p = fma(p, f, 0.0013333558179043112);
    p = fma(p, f, 0.009618129159402558);
    p = fma(p, f, 0.055504108664760424);
    p = fma(p, f, 0.2402265069581299);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    const uint32_t k = (uint32_t)(uint64_t)__double_as_longlong(shifted);
    return p * __hiloint2double((int)((k + 1023u) << 20), 0);
  }
  // In single precision.  Three roundings of t (the difference, the rate, their product) and the exponential's own:
  // wrong by less than (3 * ln 2 * |t| + 4) * 2^-24 of the weight, and 0 below 2^-126.  Rates beyond 1e30 either way
  // are left to doubles.
  template <typename W>
  __device__ __forceinline__ float rough(W x) const {
    return __builtin_amdgcn_exp2f((float)(x - (W)best) * (float)rate);
  }
  __device__ __forceinline__ bool rough_is_usable() const { return rate > 1e-30 && rate < 1e30; }
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
template <int G, typename U>
__device__ __forceinline__ U group_scan(U v, U* total) {
  const U upto = lanes_scan<G>(v);
  *total = __shfl(upto, G - 1, G);
  return lane_before<G>(upto);
}

// ---- a row in registers: E states in each of G lanes --------------------------------------------

// a and b in descending order.  (Plain v_max / v_min: fmax would first make NaNs of signalling ones quiet,
// and a row with a NaN is not drawn anyway.)
__device__ __forceinline__ void order(float& a, float& b) {
  float hi, lo;
  asm("v_max_f32 %0, %1, %2" : "=v"(hi) : "v"(a), "v"(b));
  asm("v_min_f32 %0, %1, %2" : "=v"(lo) : "v"(a), "v"(b));
  a = hi;
  b = lo;
}
__device__ __forceinline__ void order(double& a, double& b) {
  double hi, lo;
  asm("v_max_f64 %0, %1, %2" : "=v"(hi) : "v"(a), "v"(b));
  asm("v_min_f64 %0, %1, %2" : "=v"(lo) : "v"(a), "v"(b));
  a = hi;
  b = lo;
}

// The larger of two where `keep` is +infinity, the smaller where it is -infinity.
__device__ __forceinline__ float one_of(float a, float b, float keep) {
  float out;
  asm("v_med3_f32 %0, %1, %2, %3" : "=v"(out) : "v"(a), "v"(b), "v"(keep));
  return out;
}
__device__ __forceinline__ double one_of(double a, double b, double keep) {
  order(a, b);
  return keep > 0.0 ? a : b;
}

template <int MASK, int E, bool MIRROR, typename W>
__device__ __forceinline__ void exchange_lanes(W (&c)[E], bool lower) {
  const W keep = lower ? INFINITY : -INFINITY;
  // two at a time, since a mirrored pair reads each other's place
  static_assert(!MIRROR || E == 1 || E % 2 == 0, "mirrored in pairs");
#pragma unroll
  for (int j = 0; j < (E + 1) / 2; ++j) {
    const int k = E - 1 - j;
    const W at_j = lane_xor<MASK>(c[MIRROR ? k : j]), at_k = lane_xor<MASK>(c[MIRROR ? j : k]);
    c[j] = one_of(c[j], at_j, keep);
    if (k != j) c[k] = one_of(c[k], at_k, keep);
  }
}

template <int STRIDE, int E, typename W>
__device__ __forceinline__ void half_cleaners(W (&c)[E], int lane) {
  if constexpr (STRIDE >= 1) {
    if constexpr (STRIDE >= E) {
      exchange_lanes<STRIDE / E, E, false>(c, (lane & (STRIDE / E)) == 0);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((j & STRIDE) == 0) order(c[j], c[j | STRIDE]);
    }
    half_cleaners<STRIDE / 2, E>(c, lane);
  }
}

// Bitonic sort of G * E logits, the largest first (position lane * E + j); every merge starts by comparing
// mirrored positions, so that all exchanges point the same way.  Logits alone: which of the equal ones are
// kept is told by counting them afterwards, and an exchange costs two instructions of the full rate.
template <int K, int G, int E, typename W>
__device__ __forceinline__ void sort_group(W (&c)[E], int lane) {
  if constexpr (K <= G * E) {
    if constexpr (K <= E) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((j ^ (K - 1)) > j) order(c[j], c[j ^ (K - 1)]);
    } else {
      exchange_lanes<K / E - 1, E, true>(c, (lane & (K / E / 2)) == 0);
    }
    half_cleaners<K / 4, E>(c, lane);
    sort_group<K * 2, G, E>(c, lane);
  }
}

// Sums over a row's weights in R.  Doubles decide every comparison; floats, at a quarter of the cost, those that are
// not close, and tell where one is, so that the wave makes it again in doubles.  Of a sum of G * E <= 2048 floats the
// weights' errors make (3 * ln 2 * 11 + 4) * 2^-24 at most (the mean |t| of weights that are shares of a sum with a 1
// in it stays below log2 of their number), its additions 2 E + 6 roundings, and both sides of a comparison have them.
template <typename R, int E>
struct Sums {
  static constexpr bool kRough = sizeof(R) == 4;
  static constexpr R kSlack = kRough ? (R)((80 + 4 * E) * 0x1p-24) : (R)0;
  template <typename W>
  __device__ __forceinline__ static R weight_of(const Weight& weight, W x) {
    if constexpr (kRough)
      return weight.rough(x);
    else
      return weight((double)x);
  }
};

// The prefix of an order that top-p keeps: its length and the last one's logit in this lane.  Returns whether a float
// is too close to tell.
template <typename R, int G, int E, typename W>
__device__ __forceinline__ bool keep_share(const W (&c)[E], int top, const Setting& s, const Weight& weight,
                                           double row_total, int* length, W* last) {
  using S = Sums<R, E>;
  const int lane = threadIdx.x % G, mine = top - lane * E;
  R w[E], here = 0, all;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    w[j] = j < mine ? S::weight_of(weight, c[j]) : (R)0;
    here += w[j];
  }
  R before = group_scan<G>(here, &all);
  const double whole = row_total >= 0.0 ? row_total : (double)all;
  const R target = (R)(s.top_p * whole);
  R nearest = lane == 0 ? (R)INFINITY : fabs(before - target);
  *length = 0;
  *last = INFINITY;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    // those with less than the target before them, and the first one in any case
    const bool kept = j < mine && ((j == 0 && lane == 0) || before < target);
    *length += kept;
    *last = kept ? c[j] : *last;
    before += w[j];
    if (S::kRough) nearest = fmin(nearest, fabs(before - target));
  }
  return S::kRough && !(nearest > S::kSlack * (R)whole);  // a NaN is close to anything
}

// The draw among the states of at least min-p of the largest weight that are kept: all of them (kAll), those down to
// a threshold, or those above it and the first `ties` of those on it.  The slot, or -1 if a float is too close to tell
// (or none is left).
enum Keep { kAll, kDownTo, kTies };
template <typename R, Keep KEEP, int G, int E, typename W>
__device__ __forceinline__ int draw_kept(const W (&x)[E], const Setting& s, const Weight& weight, W threshold, int ties) {
  using S = Sums<R, E>;
  const int lane = threadIdx.x % G;
  int on_threshold = 0;
  if (KEEP == kTies) {  // ties are kept in the order of their slots
#pragma unroll
    for (int j = 0; j < E; ++j) on_threshold += x[j] == threshold;
    on_threshold = lanes_scan<G>(on_threshold) - on_threshold;  // in the lanes before
  }
  const R min_p = (R)s.min_p;
  bool close = false;
  R w[E], here = 0, all;
  if (S::kRough && __any(s.min_p > 0.0)) {
    R nearest = INFINITY;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[j] = S::weight_of(weight, x[j]);
      nearest = fmin(nearest, fabs(w[j] - min_p));
      w[j] = w[j] >= min_p ? w[j] : (R)0;
    }
    close = s.min_p > 0.0 && !(nearest > (R)2e-5 * min_p);  // |t| is below 126
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[j] = S::weight_of(weight, x[j]);
      if (!S::kRough) w[j] = w[j] >= min_p ? w[j] : (R)0;
    }
  }
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if (KEEP == kDownTo) w[j] = x[j] >= threshold ? w[j] : (R)0;
    if (KEEP == kTies) {
      const bool tie = x[j] == threshold;
      w[j] = x[j] > threshold || (tie && on_threshold < ties) ? w[j] : (R)0;
      on_threshold += tie;
    }
    here += w[j];
  }
  R upto = group_scan<G>(here, &all);
  const R target = (R)(s.uniform * (double)all);
  int pick = INT32_MAX, last = -1;
  if constexpr (S::kRough) {
    // a lane that starts beyond the target is not the one; borders of lanes are borders too, and so is 0
    int below = upto > target ? E : 0;
    R nearest = fmin(target, fabs(upto - target));
#pragma unroll
    for (int j = 0; j < E; ++j) {
      upto += w[j];
      below += upto <= target;
      nearest = fmin(nearest, fabs(upto - target));
    }
    if (below < E) pick = lane * E + below;
    if (close || !(nearest > S::kSlack * all)) pick = -1;
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      upto += w[j];
      if (w[j] > 0) {
        last = lane * E + j;
        if (upto > target && pick == INT32_MAX) pick = last;
      }
    }
  }
  pick = lanes_all<G>(pick, [](int p, int q) { return p < q ? p : q; });
  if (S::kRough) return pick == INT32_MAX ? -1 : pick;
  last = lanes_all<G>(last, [](int p, int q) { return p > q ? p : q; });
  return pick == INT32_MAX ? last : pick;  // u = 1, or the sums' rounding: the last kept state
}

// The draw among `count` states held by a group of lanes, x[j] of slot lane * E + j (-inf beyond the count);
// slots ascend with the states' indices.  `row_total`: the weight that top-p is a share of, when top-k is off
// and states outside the group hold some of it; negative: the group's.  Returns the slot, the same in every
// lane.  FILTER: some row may have a top-k or top-p.
template <bool FILTER, int G, int E, typename W>
__device__ int draw_in_group(const W (&x)[E], int count, const Setting& s, const Weight& weight, double row_total) {
  const int lane = threadIdx.x % G;
  const auto least = [](W p, W q) { return fmin(p, q); };
  const auto add = [](int p, int q) { return p + q; };
  const bool usable = weight.rough_is_usable();
  W threshold = -INFINITY;
  int ties = INT32_MAX;  // states on the threshold that are kept
  bool all_ties = true;
  // rows of one wave differ in their settings: the wave sorts if any of them has to
  const bool filtered = s.has_top_k() || s.has_top_p();
  if (FILTER && __any(filtered)) {
    W c[E];
#pragma unroll
    for (int j = 0; j < E; ++j) c[j] = x[j];
    sort_group<2, G, E>(c, lane);
    // the kept ones are a prefix of the order: its length, and the last one's logit
    const int top = (int)(s.top_k < count ? s.top_k : count);
    int length = 0;
    W last = INFINITY;
    if (__any(s.has_top_p())) {
      const bool close = keep_share<float, G, E>(c, top, s, weight, row_total, &length, &last);
      if (__any((close || !usable) && s.has_top_p()))
        keep_share<double, G, E>(c, top, s, weight, row_total, &length, &last);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const bool kept = lane * E + j < top;
        length += kept;
        last = kept ? c[j] : last;
      }
    }
    length = lanes_all<G>(length, add);
    last = lanes_all<G>(last, least);
    int above = 0, down_to = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      above += c[j] > last;
      down_to += c[j] >= last;
    }
    above = lanes_all<G>(above, add);
    down_to = lanes_all<G>(down_to, add);
    if (filtered) {
      threshold = last;
      ties = length - above;
      all_ties = down_to == length;
    }
  }
  int pick;
  if (!FILTER)
    pick = draw_kept<float, kAll, G, E>(x, s, weight, threshold, ties);
  else if (__all(all_ties))
    pick = draw_kept<float, kDownTo, G, E>(x, s, weight, threshold, ties);
  else
    pick = draw_kept<float, kTies, G, E>(x, s, weight, threshold, ties);
  if (!__any(pick < 0 || !usable)) return pick;
  return draw_kept<double, FILTER ? kTies : kAll, G, E>(x, s, weight, threshold, ties);
}

// The lowest slot that holds `best`.
template <int G, int E, typename W>
__device__ __forceinline__ int first_in_group(const W (&x)[E], W best) {
  int first = INT32_MAX;
#pragma unroll
  for (int j = E - 1; j >= 0; --j)
    if (x[j] == best) first = (int)(threadIdx.x % G) * E + j;
  return lanes_all<G>(first, [](int p, int q) { return p < q ? p : q; });
}

constexpr int kShortThreads = 256;

// Rows of up to G * E states.
template <typename T, bool FILTER, int G, int E>
__global__ void __launch_bounds__(kShortThreads, 2) draw_short(const Draws a, int64_t first_row) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  constexpr int kRows = kShortThreads / G;
  const int lane = threadIdx.x % G;
  const int64_t r = first_row + (int64_t)blockIdx.x * kRows + threadIdx.x / G;
  if (r >= a.rows) return;  // whole groups leave together
  const T* row = static_cast<const T*>(a.logits) + r * a.stride;
  const Setting s = row_setting(a, r);
  const int n = (int)s.n, first = lane * E;
  W x[E];
  if (E >= V && n >= V) {  // (nothing behind the row's n states is read)
    Raw raw[E / V > 0 ? E / V : 1];
#pragma unroll
    for (int k = 0; k < E / V; ++k) raw[k] = raw_of(load_pack(row + pack_start(first + k * V, n, V)));
#pragma unroll
    for (int k = 0; k < E / V; ++k) {
      const int from = first + k * V, by = from - pack_start(from, n, V);
      if (__any(by > 0 && by < V)) raw[k] = moved_down<sizeof(T)>(raw[k], by);
      const Pack<T> p = pack_of<T>(raw[k]);
#pragma unroll
      for (int j = 0; j < V; ++j) x[k * V + j] = from + j < n ? Value<T>::widen(p.v[j]) : (W)-INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = first + j < n ? Value<T>::widen(row[first + j]) : (W)-INFINITY;
  }
  bool bad = false;
  W best = -INFINITY;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    bad |= undrawable(x[j]);
    best = fmax(best, x[j]);
  }
  best = lanes_max<G>(best);
  bad = lanes_all<G>((int)bad, [](int p, int q) { return p | q; }) != 0;
  const bool valid = s.valid && !bad && !isinf(best);
  const bool greedy = s.temperature == 0.0;
  const Weight weight(valid ? (double)best : 0.0, greedy ? 1.0 : s.temperature);
  int pick = draw_in_group<FILTER, G, E>(x, n, s, weight, -1.0);
  if (greedy) pick = first_in_group<G, E>(x, best);
  if (lane == 0) a.out[r] = valid ? pick : -1;
}

// ---- long rows: summaries ------------------------------------------------------------------------

constexpr int kBlock = 64;          // states whose weights are added up
constexpr int kShortStates = 2048;  // rows beyond this are long
constexpr int kSummaryThreads = 256;

// States that a largest key is kept of: the fewer, the closer the floor that the keys give, and up to 16384
// states there are few blocks.
constexpr int64_t kSmallPieceStates = 16384;
inline int piece_states(int64_t num_states) { return num_states <= kSmallPieceStates ? 16 : kBlock; }

// A wave summarises V blocks per pack (64 lanes of V states), PACKS packs at a time.
template <typename T, int PIECE, int PACKS>
__global__ void __launch_bounds__(kSummaryThreads) block_summaries(const Draws a, int64_t tiles_per_row) {
  using W = typename Value<T>::Wide;
  using Key = KeyType<T>;
  constexpr int V = Value<T>::kVec;
  constexpr int kLanes = kBlock / V, kPieceLanes = PIECE / V;
  constexpr int kWaveStates = 64 * V;
  constexpr int kTile = kWaveStates * PACKS * (kSummaryThreads / 64);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tiles = a.rows * tiles_per_row;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t r = tile / tiles_per_row;
    const int start = (int)(tile - r * tiles_per_row) * kTile + wave * kWaveStates * PACKS;
    const int n = (int)row_states(a, r);
    if (start >= n) continue;
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    const Setting s = row_setting(a, r);
    // top-k draws from the k largest alone, min-p from those near the largest; greedy rows need no weights at all
    const bool sums = !s.has_top_k() && (s.has_top_p() || s.min_p == 0.0) && s.temperature > 0.0;
    Key* keys = static_cast<Key*>(a.piece_keys) + r * a.pieces_per_row;
    Raw raw[PACKS];
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
      const int i = start + k * kWaveStates + lane * V;
      if (i + V <= n) {
        raw[k] = raw_of(load_pack(x + i));
      } else {
        Pack<T> p;
#pragma unroll
        for (int j = 0; j < V; ++j) p.v[j] = i + j < n ? x[i + j] : Value<T>::round(-INFINITY);
        raw[k] = raw_of(p);
      }
    }
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
      const int i = start + k * kWaveStates + lane * V;
      bn_rows::kept(raw[k]);
      const Pack<T> p = pack_of<T>(raw[k]);
      W v[V];
      bool spoilt = false;
      W best = -INFINITY;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = Value<T>::widen(p.v[j]);
        best = fmax(best, v[j]);
        spoilt |= undrawable(v[j]);
      }
      best = lanes_max<kPieceLanes>(best);
      const uint64_t bad_lanes = __ballot(spoilt) >> (lane & ~(kPieceLanes - 1));
      const bool bad = (bad_lanes & ((1ull << kPieceLanes) - 1)) != 0;
      // the largest key there is marks a piece that makes its row undrawable
      if (lane % kPieceLanes == 0 && i < n) keys[i / PIECE] = bad ? (Key)~(Key)0 : KeyOf<W>::key(best);
      if (sums) {
        if constexpr (PIECE < kBlock) best = lanes_max<kLanes>(best);
        const Weight weight(isinf(best) ? 0.0 : (double)best, s.temperature);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) sum += weight((double)v[j]);
        sum = lanes_sum<kLanes>(sum);
        if (lane % kLanes == 0 && i < n) a.block_sums[r * a.sums_per_row + i / kBlock] = sum;
      }
    }
  }
}

// ---- long rows: the draw ----------------------------------------------------------------------------

// What draw_long found out about a row that draw_wide has to finish.
struct RowState {
  unsigned long long best, floor;  // keys: the largest, and one below which nothing is kept
  double total;                    // weight of the whole row, where top-k is off
  long long pending;               // 0: the row is drawn
};

// What the blocks that share a row's second and third pass leave for the last one.
constexpr int kShares = 32;  // at most a wave's lanes
constexpr int kShareThreads = 256;
constexpr int kRoughBins = 4 * kShareThreads;
constexpr int kSharedRoom = 4096;  // states around the threshold
struct SharedRow {
  unsigned long long mass[kRoughBins];
  double certain[kShares];
  unsigned long long listed;
  uint64_t key[kSharedRoom];
  int32_t index[kSharedRoom];
};

constexpr int kCandidates = 512;  // states that one wave draws among
constexpr int kListed = 512;      // pieces they may come from
constexpr int kLongThreads = 256;

template <int THREADS>
struct Bins {
  static constexpr int kThreads = THREADS;
  static constexpr int kBins = 4 * THREADS;
  unsigned long long words[THREADS / 64];
  long long answer[4];
  unsigned long long mass[kBins];
  uint32_t count[kBins];
};

template <int THREADS, typename U, typename Combine>
__device__ __forceinline__ U block_all(U v, unsigned long long* lds, Combine combine) {
  static_assert(sizeof(U) == 8, "one word per wave");
  v = lanes_all<64>(v, combine);
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
// two 32-bit minima at once
constexpr auto kMinOfHalves = [](unsigned long long p, unsigned long long q) {
  const uint32_t hi = (uint32_t)(p >> 32) < (uint32_t)(q >> 32) ? (uint32_t)(p >> 32) : (uint32_t)(q >> 32);
  const uint32_t lo = (uint32_t)p < (uint32_t)q ? (uint32_t)p : (uint32_t)q;
  return ((unsigned long long)hi << 32) | lo;
};

// Exclusive prefix sum of one value per thread, and the block's total.
template <int THREADS, typename U>
__device__ __forceinline__ U block_scan(U v, unsigned long long* lds, U* total) {
  static_assert(sizeof(U) == 8, "one word per wave");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const U upto = lanes_scan<64>(v);
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
  return base + lane_before<64>(upto);
}

// A weight as an integer: times a power of two that lets n of them add up within 62 bits and one be rounded
// by adding 2^52.
__device__ __forceinline__ double mass_scale(int n) {
  const int room = 62 - (32 - __clz(n));
  return ldexp(1.0, room < 50 ? room : 50);
}
__device__ __forceinline__ unsigned long long mass_of(double w, double scale) {
  const double shifted = w * scale + 4503599627370496.0;
  return (unsigned long long)__double_as_longlong(shifted) & 0xFFFFFFFFFFFFFull;
}

// What find_bin adds up by bin: states,
struct ByCount {
  const uint32_t* count;
  __device__ __forceinline__ void clear(int) const {}
  template <typename Key>
  __device__ __forceinline__ void add(int, Key) const {}
  __device__ __forceinline__ double of(int bin) const { return (double)count[bin]; }
};
// their weights as integers,
struct ByMass {
  const Weight& weight;
  unsigned long long* mass;
  double scale, unit = 1.0 / scale;  // powers of two
  __device__ __forceinline__ void clear(int bin) const { mass[bin] = 0; }
  template <typename Key>
  __device__ __forceinline__ void add(int bin, Key k) const {
    atomicAdd(&mass[bin], mass_of(weight.of_key(k), scale));
  }
  __device__ __forceinline__ double of(int bin) const { return (double)mass[bin] * unit; }
};
// or as integers and what these leave of each weight, as integers again.  One integer per weight has room for
// 2^-37 of the largest at 2^24 states: a tail of weights below half of that counts as nothing, however much it
// holds together.  Two have room for 2^-74.
struct ByMassAndRest {
  const Weight& weight;
  unsigned long long* mass;
  unsigned long long* rest;
  double scale, unit = 1.0 / scale;
  __device__ __forceinline__ void clear(int bin) const { mass[bin] = rest[bin] = 0; }
  template <typename Key>
  __device__ __forceinline__ void add(int bin, Key k) const {
    const double scaled = weight.of_key(k) * scale, whole = floor(scaled);
    atomicAdd(&mass[bin], mass_of(whole, 1.0));
    if (scaled != whole) atomicAdd(&rest[bin], mass_of(scaled - whole, scale));
  }
  __device__ __forceinline__ double of(int bin) const { return ((double)mass[bin] + (double)rest[bin] * unit) * unit; }
};

// A bin, and what lies above it.
struct Found {
  int bin;
  double above;               // count or weight of the bins above
  unsigned long long states;  // in the bin
  bool reached;               // the target is reached in it; else it is the lowest that holds a state
};

// The bin in which what `by` adds up from the top, `above` included, reaches `target`.  each(fn)
// calls fn(key) for every key there is; bin_of(key) is its bin, ascending with the key, or negative.
template <typename Lds, typename Each, typename BinOf, typename By>
__device__ __forceinline__ Found find_bin(Lds& lds, Each each, BinOf bin_of, By by, double above, double target) {
  constexpr int THREADS = Lds::kThreads, kBins = Lds::kBins;
  __syncthreads();
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    lds.count[b * THREADS + threadIdx.x] = 0;
    by.clear(b * THREADS + (int)threadIdx.x);
  }
  __syncthreads();
  each([&](auto k) {
    const int bin = bin_of(k);
    if (bin < 0) return;
    atomicAdd(&lds.count[bin], 1u);
    by.add(bin, k);
  });
  __syncthreads();
  // thread t holds bins kBins - 1 - 4 t downwards
  double own[4], sum = 0.0, total;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    own[b] = by.of(kBins - 1 - 4 * (int)threadIdx.x - b);
    sum += own[b];
  }
  double before = above + block_scan<THREADS>(sum, lds.words, &total);
  // the first bin that reaches the target and, counted from the other end, the last one that holds a state
  uint32_t found = ~0u, lowest = ~0u;
  double found_above = 0.0, lowest_above = 0.0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint32_t at = 4 * threadIdx.x + b;
    if (lds.count[kBins - 1 - at] != 0) {
      if (found == ~0u && before + own[b] >= target) {
        found = at;
        found_above = before;
      }
      lowest = kBins - 1 - at;
      lowest_above = before;
    }
    before += own[b];
  }
  const unsigned long long both = block_all<THREADS>(((unsigned long long)found << 32) | lowest, lds.words, kMinOfHalves);
  const bool reached = (uint32_t)(both >> 32) != ~0u;
  const int at = reached ? (int)(both >> 32) : kBins - 1 - (int)std::min((uint32_t)both, (uint32_t)kBins - 1);
  if (threadIdx.x == (unsigned)(at / 4)) lds.answer[0] = __double_as_longlong(reached ? found_above : lowest_above);
  __syncthreads();
  return {kBins - 1 - at, __longlong_as_double(lds.answer[0]), lds.count[kBins - 1 - at], reached};
}

// A range of keys, what lies above it and how many states it holds.
template <typename Key>
struct KeyRange {
  Key low, high;
  double above;
  unsigned long long states;
  bool reached;
};

// find_bin with as many bins of equal width as there are for the keys of a range; narrows it to the one found.
template <typename Lds, typename Key, typename Each, typename By>
__device__ __forceinline__ void narrow(Lds& lds, KeyRange<Key>& range, Each each, By by, double target) {
  constexpr int kLog = Lds::kThreads == 1024 ? 12 : 10;
  static_assert((1 << kLog) == Lds::kBins, "four bins per thread");
  const Key low = range.low, high = range.high, span = high - low;
  const int bits = sizeof(Key) == 8 ? 64 - __clzll((long long)span) : 32 - __clz((int)(uint32_t)span);
  const int shift = bits > kLog ? bits - kLog : 0;
  const Found f = find_bin(
      lds, each, [&](Key k) { return k < low || k > high ? -1 : (int)((k - low) >> shift); }, by, range.above, target);
  range.low = low + ((Key)f.bin << shift);
  const Key top = range.low + (((Key)1 << shift) - 1);
  range.high = top > high || top < range.low ? high : top;
  range.above = f.above;
  range.states = f.states;
  range.reached = f.reached;
}

// The logit of a floor; 1, below all states' keys, stands for none.
template <typename W, typename Key>
__device__ __forceinline__ double floor_value(Key floor) {
  const double v = floor == 1 ? -INFINITY : (double)KeyOf<W>::value(floor);
  return v > -INFINITY ? v : -INFINITY;
}

// Finds the state at which a cumulative sum exceeds its target: segment sums in index order first, then the
// 64 * PER states of one segment by one wave.  sum_of(segment) is the segment's weight, weight_at(index) a
// state's (0: not kept).
template <int PER, typename Lds, typename SumOf, typename WeightAt>
__device__ __forceinline__ int locate(Lds& lds, int segments, double uniform, SumOf sum_of, WeightAt weight_at) {
  constexpr int THREADS = Lds::kThreads;
  const int each = (segments + THREADS - 1) / THREADS;
  const int begin = std::min((int)threadIdx.x * each, segments);
  const int end = std::min(begin + each, segments);
  double here = 0.0, total;
  int last_filled = -1;
  for (int q = begin; q < end; ++q) {
    const double s = sum_of(q);
    here += s;
    if (s > 0.0) last_filled = q;
  }
  const double left = block_scan<THREADS>(here, lds.words, &total);
  const double target = uniform * total;
  // the first thread whose segments exceed the target; u = 1, or the sums' rounding: the last that holds anything
  const uint32_t over = here > 0.0 && left + here > target ? threadIdx.x : ~0u;
  const uint32_t filled = here > 0.0 ? THREADS - 1 - threadIdx.x : ~0u;
  const unsigned long long both = block_all<THREADS>(((unsigned long long)over << 32) | filled, lds.words, kMinOfHalves);
  const bool none = (uint32_t)(both >> 32) == ~0u;
  const uint32_t owner = none ? THREADS - 1 - std::min((uint32_t)both, (uint32_t)THREADS - 1) : (uint32_t)(both >> 32);
  if (threadIdx.x == owner) {
    double before = left;
    int segment = begin;
    for (; segment < last_filled; ++segment) {
      const double s = sum_of(segment);
      if (!none && before + s > target) break;
      before += s;
    }
    lds.answer[1] = segment;
    lds.answer[2] = __double_as_longlong(before);
  }
  __syncthreads();
  const int start = (int)lds.answer[1] * (64 * PER);
  if (threadIdx.x < 64) {
    double w[PER], sum = 0.0, all;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      w[j] = weight_at(start + (int)threadIdx.x * PER + j);
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
    pick = lanes_all<64>(pick, [](int p, int q) { return p < q ? p : q; });
    last = lanes_all<64>(last, [](int p, int q) { return p > q ? p : q; });
    if (threadIdx.x == 0) lds.answer[3] = start + (pick == INT32_MAX ? last : pick);
  }
  __syncthreads();
  return (int)lds.answer[3];
}

constexpr int kStaged = 2048;  // summaries kept in LDS: all of a row of up to 131072 states

template <typename Key>
struct LongShared {
  static constexpr int kThreads = kLongThreads;
  static constexpr int kBins = 4 * kLongThreads;
  unsigned long long words[kLongThreads / 64];
  long long answer[4];
  Key piece_key[kStaged];
  union {
    double block_sum[kStaged];  // done with before the others are written
    struct {
      unsigned long long mass[kBins];
      uint32_t count[kBins];
      int32_t index[kCandidates];
      int32_t listed[kListed];
      uint8_t hits[kListed * kBlock * sizeof(Key) / 16];  // per pack of a listed piece, at least 16 / sizeof(Key) states
    };
  };
};

// The draw by one wave among the states of a list.
template <int E, typename T>
__device__ __forceinline__ int draw_among(const T* row, const int32_t* index, int count, const Setting& s,
                                          const Weight& weight, double row_total) {
  typename Value<T>::Wide x[E];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const int at = (int)(threadIdx.x & 63) * E + j;
    x[j] = at < count ? Value<T>::widen(row[index[at]]) : (typename Value<T>::Wide)-INFINITY;
  }
  return draw_in_group<true, 64, E>(x, count, s, weight, row_total);
}

// One row, by the whole block, from its summaries; the same answer in every thread: the state, -1, or -2 for
// a row that is left to draw_wide, with what it needs in `state`.
template <typename T, int PIECE>
__device__ __forceinline__ int draw_row(const Draws& a, int64_t r, LongShared<KeyType<T>>& lds, RowState& state) {
  using W = typename Value<T>::Wide;
  using Key = KeyType<T>;
  constexpr int V = Value<T>::kVec;
  constexpr int THREADS = kLongThreads;
  const T* x = static_cast<const T*>(a.logits) + r * a.stride;
  const int n = (int)row_states(a, r);
  const int pieces = (n + PIECE - 1) / PIECE, blocks = (n + kBlock - 1) / kBlock;
  const Key* keys = static_cast<const Key*>(a.piece_keys) + r * a.pieces_per_row;
  const double* sums = a.block_sums + r * a.sums_per_row;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool staged = pieces <= kStaged;

  unsigned long long best = 0, least = ~0ull;
#pragma unroll 8
  for (int b = threadIdx.x; b < pieces; b += THREADS) {
    const Key k = keys[b];
    best = kMax(best, (unsigned long long)k);
    least = kMin(least, (unsigned long long)k);
    if (staged) lds.piece_key[b] = k;
  }
  const Setting s = row_setting(a, r);  // (its loads on their way together with the summaries)
  if (!s.valid) return -1;
  best = block_all<THREADS>(best, lds.words, kMax);
  if ((Key)best == (Key)~(Key)0) return -1;
  const double largest = (double)KeyOf<W>::value((Key)best);
  if (isinf(largest)) return -1;
  const auto key_of = [&](int b) { return staged ? lds.piece_key[b] : keys[b]; };

  if (s.temperature == 0.0) {
    unsigned long long piece = ~0ull;
    for (int b = threadIdx.x; b < pieces && piece == ~0ull; b += THREADS)
      if (key_of(b) == (Key)best) piece = (unsigned long long)b;
    piece = block_all<THREADS>(piece, lds.words, kMin);
    const int i = (int)piece * PIECE + lane % PIECE;
    const uint64_t hits = __ballot(i < n && key_at(x, std::min(i, n - 1)) == (Key)best);
    return (int)piece * PIECE + __ffsll((unsigned long long)hits) - 1;
  }

  // ---- weights of the blocks, where the whole row's counts
  const Weight weight(largest, s.temperature);
  const bool plain = !s.has_top_k() && !s.has_top_p() && s.min_p == 0.0;
  const auto block_weight = [&](int b) {  // a block's sum is relative to its largest state
    Key k = key_of(b * (kBlock / PIECE));
#pragma unroll
    for (int q = 1; q < kBlock / PIECE; ++q)
      if (b * (kBlock / PIECE) + q < pieces) k = std::max(k, key_of(b * (kBlock / PIECE) + q));
    return sums[b] * weight.of_key(k);
  };
  const auto block_sum_of = [&](int b) { return staged ? lds.block_sum[b] : block_weight(b); };
  double row_total = -1.0;  // W, where it is the whole row's
  if (plain || (s.has_top_p() && !s.has_top_k())) {
    if (staged) {
#pragma unroll 8
      for (int b = threadIdx.x; b < blocks; b += THREADS) lds.block_sum[b] = block_weight(b);
      __syncthreads();
    }
    if (plain)
      return locate<1>(lds, blocks, s.uniform, block_sum_of, [&](int i) {
        return i < n ? weight.of_key(key_at(x, std::min(i, n - 1))) : 0.0;
      });
    double here = 0.0;
    const int each = (blocks + THREADS - 1) / THREADS;
    for (int b = (int)threadIdx.x * each; b < std::min((int)(threadIdx.x + 1) * each, blocks); ++b) here += block_sum_of(b);
    (void)block_scan<THREADS>(here, lds.words, &row_total);
  }

  // ---- a floor below which nothing is kept
  least = block_all<THREADS>(least, lds.words, kMin);
  const auto each_piece = [&](auto fn) {
    for (int b = threadIdx.x; b < pieces; b += THREADS) fn(key_of(b));
  };
  Key floor = 1;
  const auto raise_floor = [&](double least_weight) {  // only states of at least this weight are kept
    const double step = s.temperature * log(least_weight);
    // room for this line's roundings and the one to W
    const W bound = (W)(largest + step - 1e-6 * (fabs(largest) + fabs(step) + 1e-6 * s.temperature));
    if (bound < (W)largest && !isinf(bound)) floor = std::max(floor, KeyOf<W>::key(bound));
  };
  if (s.has_top_k()) {
    // the largest keys of k pieces are k states: the k-th state's key is not below the k-th of them
    if (s.top_k < pieces) {
      KeyRange<Key> range{(Key)least, (Key)best, 0.0, 0ull, true};
      narrow(lds, range, each_piece, ByCount{lds.count}, (double)s.top_k);
      floor = range.low;
    }
  } else if (s.has_top_p()) {
    // the states below (1 - p) W / n hold less than the share that is left out
    raise_floor((1.0 - s.top_p) * row_total / (double)n);
    // and where pieces' largest states hold the share by themselves, nothing below those is kept
    // (with room for the sums' roundings and for the integers', half a unit per piece)
    KeyRange<Key> range{std::max(floor, (Key)least), (Key)best, 0.0, 0ull, true};
    const double scale = mass_scale(n);
    narrow(lds, range, each_piece, ByMass{weight, lds.mass, scale},
           s.top_p * row_total * (1.0 + 1e-9) + (double)pieces / scale);
    if (range.reached) floor = std::max(floor, range.low);
  }
  // (with top-k and top-p together W is the weight of all top-k states, those that min-p drops among them)
  if (s.min_p > 0.0 && !(s.has_top_k() && s.has_top_p())) raise_floor(s.min_p);

  // ---- few states at or above it: one wave draws among them
  const int each = (pieces + THREADS - 1) / THREADS;
  const int begin = std::min((int)threadIdx.x * each, pieces), end = std::min(begin + each, pieces);
  unsigned long long passing = 0, listed;
  for (int b = begin; b < end; ++b) passing += key_of(b) >= floor;
  unsigned long long at = block_scan<THREADS>(passing, lds.words, &listed);
  if (listed <= kListed) {
    for (int b = begin; b < end; ++b)
      if (key_of(b) >= floor) lds.listed[at++] = b;
    __syncthreads();
    // V states in each of PIECE / V lanes per listed piece: which are at or above the floor, as bits, and their
    // number; prefix sums; then their indices in order.  A block has a SIMD per wave, so that this is bound by a
    // wave's own instructions and waits: logits are compared, not keys, up to four packs per lane are on their way at
    // once, and the second half works on the bits alone (row of 500 listed pieces: 15.7 -> 6.5 us).
    constexpr int kLanes = PIECE / V, kTogether = 64 / kLanes, kStride = THREADS / 64 * kTogether, kAhead = 4;
    static_assert(sizeof(lds.hits) >= kListed * kLanes, "a byte per pack");
    const int part = lane % kLanes, slots = (int)listed * kLanes;
    const W lowest = (W)floor_value<W>(floor);
    const auto first_of = [&](int from) { return n < V ? 0 : pack_start(from, n, V); };
    for (int base = wave * kTogether; base < (int)listed; base += kAhead * kStride) {
      Raw raw[kAhead];
      int from[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int q = std::min(base + u * kStride + lane / kLanes, (int)listed - 1);
        from[u] = lds.listed[q] * PIECE + part * V;
        if (n >= V) {
          raw[u] = raw_of(load_pack(x + first_of(from[u])));
        } else {
          Pack<T> p;
#pragma unroll
          for (int j = 0; j < V; ++j) p.v[j] = j < n ? x[j] : Value<T>::round(-INFINITY);
          raw[u] = raw_of(p);
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (base + u * kStride >= (int)listed) break;
        const int q = base + u * kStride + lane / kLanes, first = first_of(from[u]);
        const Pack<T> p = pack_of<T>(raw[u]);
        uint32_t hits = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) hits |= (uint32_t)(Value<T>::widen(p.v[j]) >= lowest) << j;
        hits = hits >> std::min(from[u] - first, V) << std::min(from[u] - first, V);
        if (n < V) hits &= (1u << n) - 1;
        if (q >= (int)listed) hits = 0;
        const int count = lanes_all<kLanes>(__popc(hits), [](int p, int q) { return p + q; });
        if (q < (int)listed) {
          lds.hits[q * kLanes + part] = (uint8_t)hits;
          if (part == 0) lds.count[q] = (uint32_t)count;
        }
      }
    }
    __syncthreads();
    constexpr int kPer = kListed / THREADS;
    unsigned long long mine = 0, candidates;
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
      for (int base = wave * 64; base < slots; base += THREADS) {
        const int q = (base + lane) / kLanes;
        uint32_t hits = base + lane < slots ? lds.hits[base + lane] : 0u;
        int to = lanes_scan<kLanes>((int)__popc(hits)) - (int)__popc(hits);
        if (hits == 0) continue;
        to += (int)lds.count[q];
        const int first = first_of(lds.listed[q] * PIECE + part * V);
        for (; hits != 0; hits &= hits - 1) lds.index[to++] = first + __ffs((int)hits) - 1;
      }
      __syncthreads();
      if (wave == 0) {
        const int count = (int)candidates;
        int slot;
        if (count <= 64)
          slot = draw_among<1>(x, lds.index, count, s, weight, row_total);
        else if (count <= 256)
          slot = draw_among<4>(x, lds.index, count, s, weight, row_total);
        else
          slot = draw_among<8>(x, lds.index, count, s, weight, row_total);
        if (lane == 0) lds.answer[3] = lds.index[slot];
      }
      __syncthreads();
      return (int)lds.answer[3];
    }
  }
  state = {best, (unsigned long long)floor, row_total, 1};
  return -2;
}

// ---- long rows that keep many states ----------------------------------------------------------------

// Calls fn(index, logit) for the states [begin, end) of a row in memory; begin is a multiple of a pack.
template <typename T, int THREADS, typename Fn>
__device__ __forceinline__ void for_each_state(const T* x, int begin, int end, Fn fn) {
  constexpr int V = Value<T>::kVec;
#pragma unroll 2
  for (int i = begin + (int)threadIdx.x * V; i + V <= end; i += THREADS * V) {
    const Pack<T> p = load_pack(x + i);
#pragma unroll
    for (int j = 0; j < V; ++j) fn(i + j, Value<T>::widen(p.v[j]));
  }
  const int i = begin + (end - begin) / V * V + (int)threadIdx.x;
  if (i < end) fn(i, Value<T>::widen(x[i]));
}

// Bins of equal width in the logit (in the key they would be wide near the maximum, where the weight is, and
// narrow around 0).  All that lies at or below `low` is in bin 0.
template <typename W>
struct Steps {
  W low, per_bin_inverse;
  int last;
  __device__ __forceinline__ Steps(double floor, double best, double temperature, int bins) : last(bins - 1) {
    // weights are 0 from 750 T below the maximum on
    low = (W)fmax(floor, best - 750.0 * temperature);
    if (!(low > -INFINITY)) low = (W)floor;
    per_bin_inverse = (W)((double)bins / (best - (double)low));
    if (!(per_bin_inverse > (W)0) || isinf(per_bin_inverse)) per_bin_inverse = 0;
  }
  __device__ __forceinline__ int bin(W x) const {
    return x > low ? (int)fmin((x - low) * per_bin_inverse, (W)last) : 0;
  }
};

template <typename Key, int ROOM>
struct Listed {
  static constexpr int kRoom = ROOM;
  union {
    struct {
      Key key[kRoom];
      int32_t index[kRoom];
    };
    unsigned long long rest[kRoom];  // of the bins' masses, where there is no list
  };
  uint32_t count;  // those that found no room counted too
  __device__ __forceinline__ void add(int i, Key k) {
    const uint32_t at = atomicAdd(&count, 1u);
    if (at >= kRoom) return;
    key[at] = k;
    index[at] = i;
  }
};

// The states of a prefix of the order: keys above `key`, and those on it up to an index.
template <typename Key>
struct Prefix {
  Key key;
  int last;
  __device__ __forceinline__ bool has(int i, Key k) const { return k > key || (k == key && i <= last); }
};

// The index of the `kept`-th state, in ascending index, on a key; all of them are in the list if `in_list`.
template <typename T, int THREADS, int ROOM>
__device__ __forceinline__ int last_kept(const T* x, int n, KeyType<T> key, unsigned long long kept, Bins<THREADS>& lds,
                         const Listed<KeyType<T>, ROOM>& list, bool in_list) {
  constexpr int V = Value<T>::kVec;
  if (in_list) {
    const uint32_t count = list.count;
    const auto each = [&](auto fn) {
      for (uint32_t q = threadIdx.x; q < count; q += THREADS)
        if (list.key[q] == key) fn(~(uint32_t)list.index[q]);
    };
    KeyRange<uint32_t> range{~(uint32_t)n, ~0u, 0.0, 0ull, true};
    do {
      narrow(lds, range, each, ByCount{lds.count}, (double)kept);
    } while (range.low != range.high && range.states > 1);
    each([&](uint32_t i) {
      if (i >= range.low && i <= range.high) lds.answer[1] = (long long)~i;
    });
    __syncthreads();
    return (int)lds.answer[1];
  }
  unsigned long long seen = 0;
  for (int base = 0; base < n && seen < kept; base += THREADS * V) {
    const int i = base + (int)threadIdx.x * V;
    unsigned long long mine = 0, all;
    uint32_t on = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i + j < n && key_at(x, i + j) == key) {
        on |= 1u << j;
        ++mine;
      }
    unsigned long long before = seen + block_scan<THREADS>(mine, lds.words, &all);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (on >> j & 1) {
        if (++before == kept) lds.answer[0] = i + j;
      }
    seen += all;
  }
  __syncthreads();
  return (int)lds.answer[0];
}

// A row that is left, as every block that works on it sees it.
template <typename T>
struct WideRow {
  using W = typename Value<T>::Wide;
  using Key = KeyType<T>;
  static constexpr int V = Value<T>::kVec;
  static constexpr int kSegment = 64 * V;  // states whose sum a wave takes
  const T* x;
  Setting s;
  int n, segments;
  Key best, floor;
  double largest;
  Weight weight;
  Steps<W> steps;
  double* sums;               // the block sums have served: one entry per segment, what certainly is kept of it,
  unsigned long long* extra;  // and what the states around the threshold add, as integers of 2^-50
  __device__ __forceinline__ WideRow(const Draws& a, int64_t r, const RowState& state, int bins)
      : x(static_cast<const T*>(a.logits) + r * a.stride),
        s(row_setting(a, r)),
        n((int)s.n),
        segments((n + kSegment - 1) / kSegment),
        best((Key)state.best),
        floor((Key)state.floor),
        largest((double)KeyOf<W>::value(best)),
        weight(largest, s.temperature),
        steps(floor_value<W>(floor), largest, s.temperature, bins),
        sums(a.block_sums + r * a.sums_per_row),
        extra(reinterpret_cast<unsigned long long*>(sums + segments)) {}
};
constexpr double kListScale = 1125899906842624.0;  // 2^50: at most 4096 weights add up

// Masses by logit of a prefix's states in [begin, end), from weights of single precision (of double where the
// temperature leaves that no room).
constexpr double kRoughScale = 274877906944.0;  // 2^38: 2^24 weights add up within 62 bits
template <typename T, int THREADS>
__device__ __forceinline__ void add_rough_masses(const WideRow<T>& row, const Prefix<KeyType<T>>& in, int begin, int end,
                                 unsigned long long* mass) {
  using W = typename Value<T>::Wide;
  const bool usable = row.weight.rough_is_usable();
  for_each_state<T, THREADS>(row.x, begin, end, [&](int i, W v) {
    if (!in.has(i, KeyOf<W>::key(v))) return;
    const double w = usable ? (double)row.weight.rough(v) : row.weight((double)v);
    atomicAdd(&mass[row.steps.bin(v)], mass_of(w, kRoughScale));
  });
}

// The bins around the threshold at which the mass from the top reaches `target`: what lies above these is kept,
// what lies below is not.  Three roundings of the exponent t make a rough weight wrong by 3 * 2^-24 * ln 2 * |t|,
// the exponential itself by 2^-22; a sum that starts with the largest weight, 1, has a mean |t| of 25 at most
// (2^24 states of weight 2^-24 double it), so it is off by less than 4e-6 of itself, a fifth of kSlack, and by
// the integers' rounding.  Where all bins together stay below the target (min-p has raised the floor over states
// that the share counts), there is no threshold: bins 0..-1, with every state above them.
template <int THREADS>
__device__ __forceinline__ int2 bins_around(const unsigned long long* mass, double target, int n, unsigned long long* words) {
  constexpr int kBins = 4 * THREADS;
  constexpr double kSlack = 2e-5;
  const double rounding = (double)n + 1.0, goal = target * kRoughScale;
  unsigned long long own[4], sum = 0, total;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    own[b] = mass[kBins - 1 - 4 * (int)threadIdx.x - b];
    sum += own[b];
  }
  unsigned long long upto = block_scan<THREADS>(sum, words, &total);
  uint32_t first = ~0u, last = ~0u;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint32_t at = 4 * threadIdx.x + b;
    upto += own[b];
    if (first == ~0u && (double)upto * (1.0 + kSlack) + rounding >= goal) first = at;
    if (last == ~0u && (double)upto * (1.0 - kSlack) - rounding >= goal) last = at;
  }
  const unsigned long long ends = block_all<THREADS>(((unsigned long long)first << 32) | last, words, kMinOfHalves);
  if ((uint32_t)(ends >> 32) == ~0u) return make_int2(0, -1);
  const int lowest = std::min((uint32_t)ends, (uint32_t)kBins - 1);
  const int highest = std::min((int)std::min((uint32_t)(ends >> 32), (uint32_t)kBins - 1), lowest);
  return make_int2(kBins - 1 - lowest, kBins - 1 - highest);
}

// Weights of a prefix's states in the bins above one: their sum over the segments [begin, end), and by segment
// those that min-p leaves.  others(index, key) is called for its states in the bins lowest..above.
template <typename T, int THREADS, typename Others>
__device__ __forceinline__ double add_up(const WideRow<T>& row, const Prefix<KeyType<T>>& in, int lowest, int above, int begin, int end,
                         unsigned long long* words, Others others) {
  using W = typename Value<T>::Wide;
  using Key = KeyType<T>;
  constexpr int V = Value<T>::kVec;
  const int lane = threadIdx.x & 63;
  const auto load = [&](int q) {
    const int i = (q * 64 + lane) * V;
    Pack<T> p;
    if (i + V <= row.n) {
      p = load_pack(row.x + i);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) p.v[j] = i + j < row.n ? row.x[i + j] : Value<T>::round(-INFINITY);
    }
    return raw_of(p);
  };
  double all = 0.0;
  int q = begin + (int)(threadIdx.x >> 6);
  Raw next = load(q);  // the segment after this one is on its way while this one is worked on
  for (; q < end; q += THREADS / 64) {
    Raw raw = next;
    next = load(q + THREADS / 64);
    bn_rows::kept(raw);
    const Pack<T> p = pack_of<T>(raw);
    const int i = (q * 64 + lane) * V;
    double drawn = 0.0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const W v = Value<T>::widen(p.v[j]);
      const Key k = KeyOf<W>::key(v);
      if (!in.has(i + j, k)) continue;
      const int bin = row.steps.bin(v);
      if (bin > above) {
        const double w = row.weight((double)v);
        all += w;
        drawn += w >= row.s.min_p ? w : 0.0;
      } else if (bin >= lowest) {
        others(i + j, k);
      }
    }
    drawn = lanes_sum<64>(drawn);
    if (lane == 0) {
      row.sums[q] = drawn;
      row.extra[q] = 0;
    }
  }
  double total;
  (void)block_scan<THREADS>(all, words, &total);  // (its barriers also publish the segments' sums)
  return total;
}
template <typename T, int THREADS>
__device__ __forceinline__ double add_up(const WideRow<T>& row, const Prefix<KeyType<T>>& in, unsigned long long* words) {
  return add_up<T, THREADS>(row, in, 0, -1, 0, row.segments, words, [](int, KeyType<T>) {});
}

// A wide row's last steps: what top-p keeps of a prefix when the states around the threshold are listed, and the draw.
template <typename T, int THREADS, int ROOM>
struct Settling {
  using Key = KeyType<T>;
  using Sum = unsigned long long;
  const WideRow<T>& row;
  Bins<THREADS>& lds;
  Listed<Key, ROOM>& list;
  __device__ __forceinline__ Settling(const WideRow<T>& row_, Bins<THREADS>& lds_, Listed<Key, ROOM>& list_)
      : row(row_), lds(lds_), list(list_) {}

  template <typename Fn>
  __device__ __forceinline__ void each_listed(Fn fn) const {
    const uint32_t count = list.count;
    for (uint32_t q = threadIdx.x; q < count; q += THREADS) fn(list.key[q]);
  }

  // The key at which the weight reaches `reach`, among the listed ones.
  __device__ __forceinline__ void narrow_listed(KeyRange<Key>& range, double reach) {
    // the list's own range, which is a bin or two, instead of all keys
    Sum low = ~0ull, high = 0;
    each_listed([&](Key k) {
      low = kMin(low, (Sum)k);
      high = kMax(high, (Sum)k);
    });
    range.low = (Key)block_all<THREADS>(low, lds.words, kMin);
    range.high = (Key)block_all<THREADS>(high, lds.words, kMax);
    const ByMass by{row.weight, lds.mass, mass_scale(ROOM)};
    do {
      narrow(lds, range, [&](auto fn) { each_listed(fn); }, by, reach);
    } while (range.low != range.high);
  }

  // Ends `kept` in the states on the range's key: those with less than the target before them, one at least.
  __device__ __forceinline__ void end_on_key(Prefix<Key>& kept, const KeyRange<Key>& range, double reach, bool in_list) {
    const double each = row.weight.of_key(range.low);
    Sum ties = range.states;
    if (each > 0.0) ties = (Sum)fmin(fmax(ceil((reach - range.above) / each), 1.0), (double)range.states);
    const int bound = range.low == kept.key ? kept.last : row.n;
    kept.key = range.low;
    kept.last = ties < range.states ? last_kept<T>(row.x, row.n, range.low, ties, lds, list, in_list) : bound;
  }

  // The segments hold what lies above the bins around the threshold, the list what lies in them.
  __device__ __forceinline__ void add_listed(const Prefix<Key>& kept) {
    const uint32_t count = list.count;
    for (uint32_t q = threadIdx.x; q < count; q += THREADS)
      if (kept.has(list.index[q], list.key[q])) {
        const double w = row.weight.of_key(list.key[q]);
        if (w >= row.s.min_p) atomicAdd(&row.extra[list.index[q] / WideRow<T>::kSegment], mass_of(w, kListScale));
      }
  }

  // The state drawn from a prefix, once the segments' sums are there.
  __device__ __forceinline__ int drawn(const Prefix<Key>& kept) {
    __syncthreads();
    return locate<WideRow<T>::V>(
        lds, row.segments, row.s.uniform,
        [&](int q) {
          const Sum more = __hip_atomic_load(&row.extra[q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          return row.sums[q] + (double)more / kListScale;
        },
        [&](int i) {
          if (i >= row.n) return 0.0;
          const Key k = key_at(row.x, std::min(i, row.n - 1));
          const double w = kept.has(i, k) ? row.weight.of_key(k) : 0.0;
          return w >= row.s.min_p ? w : 0.0;
        });
  }
};

// A row with top-p alone whose passes the blocks of draw_wide_masses and draw_wide_sums have shared, from what these
// have left.
template <typename T, int THREADS>
__device__ __forceinline__ int draw_shared_row(const WideRow<T>& row, const SharedRow& shared, double row_total, Bins<THREADS>& lds,
                               Listed<KeyType<T>, kSharedRoom>& list) {
  using Key = KeyType<T>;
  Settling<T, THREADS, kSharedRoom> settling(row, lds, list);
  const int lane = threadIdx.x & 63;  // one load for all shares, and the same tree in every wave
  const double certain = lanes_sum<64>(lane < kShares ? shared.certain[lane] : 0.0);
  const uint32_t count = (uint32_t)shared.listed;
  for (uint32_t q = threadIdx.x; q < count; q += THREADS) {
    list.key[q] = (Key)shared.key[q];
    list.index[q] = shared.index[q];
  }
  if (threadIdx.x == 0) list.count = count;
  __syncthreads();
  Prefix<Key> kept{row.floor, row.n};
  KeyRange<Key> range{row.floor, row.best, certain, 0ull, true};
  const double reach = row.s.top_p * row_total;
  if (count != 0) {  // none: the share is not reached, all of the prefix is kept
    settling.narrow_listed(range, reach);
    settling.end_on_key(kept, range, reach, true);
    settling.add_listed(kept);
  }
  return settling.drawn(kept);
}

// One row by the whole block, over the row in memory: one pass weighs its states roughly, by logit, a second
// one adds up what is certainly kept, and the few thousand states around the threshold are settled in LDS.
template <typename T, int THREADS, int ROOM>
__device__ __forceinline__ int draw_wide_row(const WideRow<T>& row, double row_total, Bins<THREADS>& lds, Listed<KeyType<T>, ROOM>& list) {
  using W = typename Value<T>::Wide;
  using Key = KeyType<T>;
  using Sum = unsigned long long;
  const Setting& s = row.s;
  const int n = row.n;
  const T* x = row.x;
  Settling<T, THREADS, ROOM> settling(row, lds, list);
  const ByCount by_count{lds.count};

  // the states of a prefix in bins lowest..highest, by key
  const auto each_in = [&](const Prefix<Key>& in, int lowest, int highest, auto fn) {
    for_each_state<T, THREADS>(x, 0, n, [&](int i, W v) {
      const int bin = row.steps.bin(v);
      if (bin < lowest || bin > highest) return;
      const Key k = KeyOf<W>::key(v);
      if (in.has(i, k)) fn(i, k);
    });
  };
  const auto clear_list = [&]() {
    __syncthreads();
    if (threadIdx.x == 0) list.count = 0;
    __syncthreads();
  };
  const auto fill_list = [&](const Prefix<Key>& in, int lowest, int highest, Key low, Key high) {
    clear_list();
    each_in(in, lowest, highest, [&](int i, Key k) {
      if (k >= low && k <= high) list.add(i, k);
    });
    __syncthreads();
  };
  const auto each_listed = [&](auto fn) { settling.each_listed(fn); };

  // ---- top-k: the k-th key by counting
  Prefix<Key> kept{row.floor, n};
  if (s.has_top_k()) {
    const Prefix<Key> all = kept;
    const auto each_state = [&](auto fn) {
      for_each_state<T, THREADS>(x, 0, n, [&](int, W v) {
        if (KeyOf<W>::key(v) >= all.key) fn(v);
      });
    };
    const Found f = find_bin(lds, each_state, [&](W v) { return row.steps.bin(v); }, by_count, 0.0, (double)s.top_k);
    KeyRange<Key> range{row.floor, row.best, f.above, f.states, true};
    const auto each_key = [&](auto fn) {
      each_in(all, f.bin, f.bin, [&](int, Key k) { fn(k); });
    };
    while (range.low != range.high && range.states > ROOM) narrow(lds, range, each_key, by_count, (double)s.top_k);
    const bool in_list = range.states <= ROOM;
    if (in_list) {
      fill_list(all, f.bin, f.bin, range.low, range.high);
      while (range.low != range.high) narrow(lds, range, each_listed, by_count, (double)s.top_k);
    }
    kept.key = range.low;
    const Sum ties = (Sum)s.top_k - (Sum)range.above;
    if (ties < range.states) kept.last = last_kept<T>(x, n, range.low, ties, lds, list, in_list);
  }

  bool added = false;
  if (s.has_top_p()) {
    const double reach = s.top_p * (s.has_top_k() ? add_up<T, THREADS>(row, kept, lds.words) : row_total);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 4; ++b) lds.mass[b * THREADS + threadIdx.x] = 0;
    __syncthreads();
    add_rough_masses<T, THREADS>(row, kept, 0, n, lds.mass);
    __syncthreads();
    const int2 around = bins_around<THREADS>(lds.mass, reach, n, lds.words);
    clear_list();
    const double certain = add_up<T, THREADS>(row, kept, around.x, around.y, 0, row.segments, lds.words,
                                              [&](int i, Key k) { list.add(i, k); });
    KeyRange<Key> range{kept.key, row.best, certain, 0ull, true};
    const bool whole_list = list.count <= ROOM;  // the list holds all those around the threshold
    bool in_list = whole_list;                   // ... those on its key
    if (!in_list) {
      const auto each_key = [&](auto fn) {
        each_in(kept, around.x, around.y, [&](int, Key k) { fn(k); });
      };
      static_assert(ROOM >= Bins<THREADS>::kBins, "the list's memory holds the rests");
      const ByMassAndRest by{row.weight, lds.mass, list.rest, mass_scale(n)};
      do {
        narrow(lds, range, each_key, by, reach);
      } while (range.low != range.high && range.states > ROOM);
      in_list = range.states <= ROOM;
      if (in_list) fill_list(kept, around.x, around.y, range.low, range.high);
    }
    if (list.count != 0) {  // none: the share is not reached, all of the prefix is kept
      if (in_list) settling.narrow_listed(range, reach);
      settling.end_on_key(kept, range, reach, in_list);
      if (whole_list) settling.add_listed(kept);
    }
    added = whole_list;
  }
  if (!added) (void)add_up<T, THREADS>(row, kept, lds.words);
  return settling.drawn(kept);
}

// The second launch.  ALONE: it draws the rows with many states as well, a block's threads over all of the row.
template <typename T, int PIECE, bool ALONE>
__global__ void __launch_bounds__(kLongThreads) draw_long(const Draws a, int64_t first_row) {
  using Key = KeyType<T>;
  __shared__ union {
    LongShared<Key> few;
    struct {
      Bins<kLongThreads> lds;
      Listed<Key, 4 * kLongThreads> list;
    } many;
  } space;
  const int64_t r = first_row + blockIdx.x;
  RowState state{};
  int drawn = draw_row<T, PIECE>(a, r, space.few, state);
  if constexpr (ALONE) {
    if (drawn < -1) {
      __syncthreads();
      const WideRow<T> row(a, r, state, Bins<kLongThreads>::kBins);
      drawn = draw_wide_row<T>(row, state.total, space.many.lds, space.many.list);
    }
    if (threadIdx.x == 0) a.out[r] = drawn;
    return;
  }
  if (threadIdx.x == 0) {
    if (drawn >= -1) a.out[r] = drawn;
    a.row_states[r] = state;
  }
  if (drawn < -1 && a.shared) {
    for (int b = threadIdx.x; b < kRoughBins; b += kLongThreads) a.shared[r].mass[b] = 0;
    if (threadIdx.x == 0) a.shared[r].listed = 0;
  }
}

// A row whose passes were shared is left with short lists, over which fewer waves meet sooner: the others of its
// block end (serving batch of 256 x 131072: 30 -> 14.5 us).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) draw_wide(const Draws a, int64_t first_row) {
  using Key = KeyType<T>;
  constexpr bool kMayShare = THREADS > kShareThreads;
  constexpr int kSharedList = kMayShare ? kSharedRoom : 1;
  __shared__ union {
    struct {
      Bins<THREADS> lds;
      Listed<Key, 4 * THREADS> list;
    } whole;
    struct {
      Bins<kShareThreads> lds;
      Listed<Key, kSharedList> list;
    } shared;
  } space;
  const int64_t r = first_row + blockIdx.x;
  const RowState state = a.row_states[r];
  if (!state.pending) return;
  if constexpr (kMayShare) {
    const Setting s = row_setting(a, r);
    if (a.shared && s.has_top_p() && !s.has_top_k() && a.shared[r].listed <= (unsigned long long)kSharedRoom) {
      if (threadIdx.x >= kShareThreads) return;
      const WideRow<T> row(a, r, state, kRoughBins);
      const int drawn = draw_shared_row<T, kShareThreads>(row, a.shared[r], state.total, space.shared.lds, space.shared.list);
      if (threadIdx.x == 0) a.out[r] = drawn;
      return;
    }
  }
  const WideRow<T> row(a, r, state, Bins<THREADS>::kBins);
  const int drawn = draw_wide_row<T>(row, state.total, space.whole.lds, space.whole.list);
  if (threadIdx.x == 0) a.out[r] = drawn;
}

// The same passes over a row with top-p alone, by kShares blocks: a block is bound by its arithmetic (a row of
// 131072 states took one block 110 us), and a call of few rows leaves most of the GPU idle.
template <typename T>
__global__ void __launch_bounds__(kShareThreads) draw_wide_masses(const Draws a) {
  __shared__ unsigned long long mass[kRoughBins];
  const int64_t r = blockIdx.x / kShares;
  const int share = blockIdx.x % kShares;
  const RowState state = a.row_states[r];
  if (!state.pending) return;
  const WideRow<T> row(a, r, state, kRoughBins);
  if (!row.s.has_top_p() || row.s.has_top_k()) return;
  for (int b = threadIdx.x; b < kRoughBins; b += kShareThreads) mass[b] = 0;
  __syncthreads();
  const int each = (row.segments + kShares - 1) / kShares * WideRow<T>::kSegment;
  const int begin = std::min(share * each, row.n), end = std::min(begin + each, row.n);
  add_rough_masses<T, kShareThreads>(row, Prefix<KeyType<T>>{row.floor, row.n}, begin, end, mass);
  __syncthreads();
  for (int b = threadIdx.x; b < kRoughBins; b += kShareThreads)
    if (mass[b] != 0) atomicAdd(&a.shared[r].mass[b], mass[b]);
}

template <typename T>
__global__ void __launch_bounds__(kShareThreads) draw_wide_sums(const Draws a) {
  using Key = KeyType<T>;
  constexpr int kRoom = 1024;
  __shared__ unsigned long long words[kShareThreads / 64], base;
  __shared__ Listed<Key, kRoom> list;
  const int64_t r = blockIdx.x / kShares;
  const int share = blockIdx.x % kShares;
  const RowState state = a.row_states[r];
  if (!state.pending) return;
  const WideRow<T> row(a, r, state, kRoughBins);
  if (!row.s.has_top_p() || row.s.has_top_k()) return;
  SharedRow& shared = a.shared[r];
  const int2 around = bins_around<kShareThreads>(shared.mass, row.s.top_p * state.total, row.n, words);
  const int each = (row.segments + kShares - 1) / kShares;
  const int begin = std::min(share * each, row.segments), end = std::min(begin + each, row.segments);
  const Prefix<Key> in{row.floor, row.n};
  if (threadIdx.x == 0) list.count = 0;
  __syncthreads();
  const double certain = add_up<T, kShareThreads>(row, in, around.x, around.y, begin, end, words,
                                                  [&](int i, Key k) { list.add(i, k); });
  // the share's states around the threshold go behind those of the shares before
  if (threadIdx.x == 0) {
    shared.certain[share] = certain;
    base = atomicAdd(&shared.listed, list.count > kRoom ? kSharedRoom + 1ull : (unsigned long long)list.count);
  }
  __syncthreads();
  const uint32_t count = list.count;
  if (count > kRoom || base + count > kSharedRoom) return;  // draw_wide sees from their number that some are missing
  for (uint32_t q = threadIdx.x; q < count; q += kShareThreads) {
    shared.key[base + q] = (uint64_t)list.key[q];
    shared.index[base + q] = list.index[q];
  }
}

constexpr int64_t kMaxStates = 1 << 24;
constexpr int64_t kMaxBlocks = 1 << 20;

template <typename T, int G, int E>
void launch_short(const Draws& a, hipStream_t s) {
  const int64_t per_block = kShortThreads / G;
  const bn_draw_filters& f = a.filters;
  const bool filter = f.top_k_dev || f.top_p_dev || (f.top_k > 0 && f.top_k < a.width) || f.top_p < 1.0;
  for (int64_t r = 0; r < a.rows; r += kMaxBlocks * per_block) {
    const dim3 grid((uint32_t)std::min((a.rows - r + per_block - 1) / per_block, kMaxBlocks));
    if (filter)
      hipLaunchKernelGGL((draw_short<T, true, G, E>), grid, dim3(kShortThreads), 0, s, a, r);
    else
      hipLaunchKernelGGL((draw_short<T, false, G, E>), grid, dim3(kShortThreads), 0, s, a, r);
  }
}

// 16 states per lane take the fewest instructions per row; where that leaves SIMDs (1024) with less than four
// waves, 4 states per lane make four times as many.
template <typename T, int G>
void launch_short_rows(const Draws& a, hipStream_t s) {
  if (G * 4 <= 64 && a.rows * G < 64 * 4096)
    launch_short<T, std::min(G * 4, 64), 4>(a, s);
  else
    launch_short<T, G, 16>(a, s);
}

template <typename T, int PIECE>
void launch_summaries_and_draw(const Draws& a, bool alone, hipStream_t s) {
  constexpr int kPacks = 4;
  constexpr int64_t kTile = (int64_t)64 * Value<T>::kVec * kPacks * (kSummaryThreads / 64);
  const int64_t tiles = (a.width + kTile - 1) / kTile;
  hipLaunchKernelGGL((block_summaries<T, PIECE, kPacks>), dim3((uint32_t)std::min(a.rows * tiles, kMaxBlocks)),
                     dim3(kSummaryThreads), 0, s, a, tiles);
  for (int64_t r = 0; r < a.rows; r += kMaxBlocks) {
    const dim3 grid((uint32_t)std::min(a.rows - r, kMaxBlocks));
    if (alone)
      hipLaunchKernelGGL((draw_long<T, PIECE, true>), grid, dim3(kLongThreads), 0, s, a, r);
    else
      hipLaunchKernelGGL((draw_long<T, PIECE, false>), grid, dim3(kLongThreads), 0, s, a, r);
  }
}

template <typename T>
void launch_long(Draws a, hipStream_t s) {
  const bn_draw_filters& f = a.filters;
  // a row may have top-p alone: without top-k, or with one that is no less than the row's states
  const bool top_p = f.top_p_dev || f.top_p < 1.0;
  // A small top-k leaves few states in all but the rarest rows (ties at the k-th, or most of the k largest in a few
  // pieces), and so little of those that a block of draw_long finishes them in less time than draw_wide's launch and
  // meetings of 16 waves take: no third launch then (32000 bfloat16 states, k = 256 / 257: 16.5 / 18.2 us, sorted 49 /
  // 63).  A top-k of 5000 is left to it: 105 us for a row of 131072, 303 with 256 threads.
  const bool filtered = f.top_k_dev || top_p || f.min_p_dev || f.top_k > 0 || f.min_p > 0.0;
  const bool alone = !f.top_k_dev && f.top_k > 0 && f.top_k <= kCandidates / 2;
  if (alone || !(top_p && (f.top_k_dev || f.top_k == 0 || f.top_k >= a.width || a.counts))) a.shared = nullptr;
  if (a.width <= kSmallPieceStates)
    launch_summaries_and_draw<T, 16>(a, alone, s);
  else
    launch_summaries_and_draw<T, kBlock>(a, alone, s);
  if (alone || !filtered) return;
  if (a.shared) {
    const dim3 grid((uint32_t)(a.rows * kShares));
    hipLaunchKernelGGL(draw_wide_masses<T>, grid, dim3(kShareThreads), 0, s, a);
    hipLaunchKernelGGL(draw_wide_sums<T>, grid, dim3(kShareThreads), 0, s, a);
  }
  for (int64_t r = 0; r < a.rows; r += kMaxBlocks) {
    const dim3 grid((uint32_t)std::min(a.rows - r, kMaxBlocks));
    if (a.width <= kSmallPieceStates)
      hipLaunchKernelGGL((draw_wide<T, 256>), grid, dim3(256), 0, s, a, r);
    else
      hipLaunchKernelGGL((draw_wide<T, 1024>), grid, dim3(1024), 0, s, a, r);
  }
}

// Rows of which several blocks take a share: long ones, and no more of them than leave CUs (256) idle.
inline bool rows_are_shared(int64_t rows, int64_t num_states) { return num_states > kSmallPieceStates && rows <= 512; }

template <typename T>
hipError_t launch(const Draws& a, hipStream_t s) {
  if (a.width <= 4) launch_short<T, 1, 4>(a, s);
  else if (a.width <= 16) launch_short_rows<T, 1>(a, s);
  else if (a.width <= 32) launch_short_rows<T, 2>(a, s);
  else if (a.width <= 64) launch_short_rows<T, 4>(a, s);
  else if (a.width <= 128) launch_short_rows<T, 8>(a, s);
  else if (a.width <= 256) launch_short_rows<T, 16>(a, s);
  else if (a.width <= 512) launch_short<T, 32, 16>(a, s);
  else if (a.width <= 1024) launch_short<T, 64, 16>(a, s);
  else if (a.width <= kShortStates) launch_short<T, 64, 32>(a, s);
  else launch_long<T>(a, s);
  return hipGetLastError();
}

// one translation unit per type (draw_f32.hip, ...), so that they are compiled side by side
hipError_t launch_f32(const Draws& a, hipStream_t s);
hipError_t launch_f64(const Draws& a, hipStream_t s);
hipError_t launch_f16(const Draws& a, hipStream_t s);
hipError_t launch_bf16(const Draws& a, hipStream_t s);


}  // namespace bn_draw
