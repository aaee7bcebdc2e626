// One state per row of logits, drawn at a given uniform number: bn_draw_states of include/bn_hip.h.
//
//   w_i = exp((x_i - max x) / T)                  order: x decreasing, ties by ascending index
//   A = the first k of the order                  W = sum_A w
//   P = those of A with less than p W before them in the order
//   K = those of P with w_i >= m                  state = min{i in K : sum_{j in K, j <= i} w_j > u W_K}
//
// P and K are prefixes of the order, so a row's kept states are those above a threshold: a key (the
// logit as an integer that sorts like it) and, among the states on that key, an index.  The threshold is
// found digit by digit: 256 bins of counts and masses over the states that share the digits found so far.
// Masses are 64-bit integers (w scaled by a power of two), so the atomics that add them up give the same
// sums in any order; the cumulative sums of the draw itself are doubles in a fixed order.
#include "../../include/bn_hip.h"

#include <algorithm>
#include <cmath>
#include <string>

#include <hip/hip_runtime.h>

#include "error.h"
#include "row_values.h"

namespace {

using namespace bn_rows;

// A logit as an unsigned integer that sorts like it; -0 and +0 are one key.
template <typename W>
struct KeyOf;
template <>
struct KeyOf<float> {
  using Key = uint32_t;
  static constexpr int kBits = 32;
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
  static constexpr int kBits = 64;
  static __device__ __forceinline__ Key key(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
  }
  static __device__ __forceinline__ double value(Key k) {
    return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
  }
};

struct Draws {
  const void* logits;
  int64_t rows;
  int64_t width;
  int64_t stride;
  const int64_t* counts;
  const void* uniforms;
  int32_t uniform_dtype;
  bn_draw_filters filters;
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
};

__device__ __forceinline__ Setting row_setting(const Draws& a, int64_t r) {
  Setting s;
  s.n = a.width;
  if (a.counts) {
    const int64_t n = a.counts[r];
    s.n = n < 0 ? 0 : (n > a.width ? a.width : n);
  }
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

__device__ __forceinline__ double weight_of(double x, double best, double temperature) {
  return exp((x - best) / temperature);
}

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 256;

struct Shared {
  uint32_t count[kBins];
  unsigned long long mass[kBins];
  double sums[kWaves];
  unsigned long long words[kWaves];
  long long answer[4];
};

template <typename Combine, typename U>
__device__ __forceinline__ U block_all(U v, U* lds, Combine combine) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = combine(v, (U)__shfl_xor(v, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  U out = lds[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) out = combine(out, lds[w]);
  return out;
}

// Exclusive prefix sum of one double per thread, and the block's total.
__device__ __forceinline__ double block_scan(double v, double* lds, double* total) {
  double upto = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double left = __shfl_up(upto, d, 64);
    if ((int)(threadIdx.x & 63) >= d) upto += left;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = upto;
  __syncthreads();
  double base = 0.0, sum = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == (int)(threadIdx.x >> 6)) base = sum;
    sum += lds[w];
  }
  *total = sum;
  double before = __shfl_up(upto, 1, 64);
  if ((threadIdx.x & 63) == 0) before = 0.0;
  return base + before;
}

// What is kept of a row: keys above `key`, states on it up to index `last_tie`, weights from `min_p`.
template <typename Key>
struct Threshold {
  Key key;
  int64_t last_tie;
};

template <typename T>
struct Row {
  using W = typename Value<T>::Wide;
  using Key = typename KeyOf<W>::Key;
  const T* x;
  Setting s;
  double best;
  double scale;  // of the integer masses
  __device__ __forceinline__ Key key(int64_t i) const { return KeyOf<W>::key(Value<T>::widen(x[i])); }
  __device__ __forceinline__ double weight(Key k) const {
    return weight_of((double)KeyOf<W>::value(k), best, s.temperature);
  }
  __device__ __forceinline__ unsigned long long mass(Key k) const {
    return (unsigned long long)llrint(weight(k) * scale);
  }
};

// Walks the digits of the threshold key among the row's keys >= floor.  BY_MASS: the first key of the
// order at which the mass reaches `target` (states on `floor` count floor_ties times); else the
// `target`-th key.  Answers the key, how many states on it are kept and how many lie on it.
template <typename T, bool BY_MASS>
__device__ void find_threshold(const Row<T>& row, typename Row<T>::Key floor, int64_t floor_ties, double target,
                               Shared& lds, typename Row<T>::Key* key_out, int64_t* kept_out, int64_t* ties_out,
                               double* above_out) {
  using Key = typename Row<T>::Key;
  constexpr int kBits = KeyOf<typename Row<T>::W>::kBits;
  Key prefix = 0;
  double above = 0.0;  // mass or count of the keys above the prefix
  for (int shift = kBits - 8; shift >= 0; shift -= 8) {
    __syncthreads();
    lds.count[threadIdx.x] = 0;
    lds.mass[threadIdx.x] = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < row.s.n; i += kThreads) {
      const Key k = row.key(i);
      if (k < floor || (shift + 8 < kBits && (k >> (shift + 8)) != prefix)) continue;
      const int bin = (int)((k >> shift) & 255);
      atomicAdd(&lds.count[bin], 1u);
      if (BY_MASS && k != floor) atomicAdd(&lds.mass[bin], row.mass(k));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      const bool holds_floor = shift + 8 >= kBits || (floor >> (shift + 8)) == prefix;
      int bin = kBins - 1;
      for (;; --bin) {
        double here = (double)lds.count[bin];
        if (BY_MASS) {
          unsigned long long m = lds.mass[bin];
          if (holds_floor && bin == (int)((floor >> shift) & 255)) m += (unsigned long long)floor_ties * row.mass(floor);
          here = (double)m;
        }
        if (bin == 0) break;
        if (lds.count[bin] == 0) continue;
        if (above + here >= target) break;
        bool more = false;  // the last bin that holds anything takes what rounding leaves over
        for (int b = bin - 1; b >= 0 && !more; --b) more = lds.count[b] != 0;
        if (!more) break;
        above += here;
      }
      lds.answer[0] = bin;
      lds.sums[0] = above;
      lds.answer[1] = lds.count[bin];
    }
    __syncthreads();
    prefix = (Key)((shift + 8 >= kBits ? (Key)0 : (Key)(prefix << 8)) | (Key)lds.answer[0]);
    above = lds.sums[0];
    *ties_out = lds.answer[1];
  }
  *key_out = prefix;
  *above_out = above;
  if (BY_MASS) {
    const int64_t here = prefix == floor ? floor_ties : *ties_out;
    const double each = (double)row.mass(prefix);
    int64_t keep = each > 0.0 ? (int64_t)fmin(ceil((target - above) / each), (double)here) : here;
    if (keep < 1) keep = 1;
    while (keep > 1 && above + (double)(keep - 1) * each >= target) --keep;
    while (keep < here && above + (double)keep * each < target) ++keep;
    *kept_out = keep;
  } else {
    *kept_out = (int64_t)(target - above);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) draw_rows(const Draws a) {
  using R = Row<T>;
  using Key = typename R::Key;
  using W = typename R::W;
  __shared__ Shared lds;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    __syncthreads();
    R row;
    row.x = static_cast<const T*>(a.logits) + r * a.stride;
    row.s = row_setting(a, r);
    const int64_t n = row.s.n;
    // the largest logit; NaN and +inf make the row undrawable
    unsigned long long best = 0, bad = 0;
    for (int64_t i = threadIdx.x; i < n; i += kThreads) {
      const W x = Value<T>::widen(row.x[i]);
      if (isnan(x) || (isinf(x) && x > 0)) bad = 1;
      const unsigned long long k = KeyOf<W>::key(x);
      best = best > k ? best : k;
    }
    const auto larger = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
    best = block_all(best, lds.words, larger);
    bad = block_all(bad, lds.words, larger);
    row.best = (double)KeyOf<W>::value((Key)best);
    if (!row.s.valid || bad || isinf(row.best)) {
      if (threadIdx.x == 0) a.out[r] = -1;
      continue;
    }
    if (row.s.temperature == 0.0) {
      unsigned long long first = ~0ull;
      for (int64_t i = threadIdx.x; i < n; i += kThreads)
        if (row.key(i) == (Key)best) {
          first = (unsigned long long)i;
          break;
        }
      first = block_all(first, lds.words, [](unsigned long long p, unsigned long long q) { return p < q ? p : q; });
      if (threadIdx.x == 0) a.out[r] = (int32_t)first;
      continue;
    }
    row.scale = ldexp(1.0, 62 - (64 - __clzll((unsigned long long)n)));

    Threshold<Key> t{0, n};
    int64_t kept_ties = n, ties = n;  // of the states on t.key
    double above = 0.0;
    if (row.s.top_k < n) find_threshold<T, false>(row, 0, 0, (double)row.s.top_k, lds, &t.key, &kept_ties, &ties, &above);
    if (row.s.top_p < 1.0) {
      unsigned long long total = 0;
      for (int64_t i = threadIdx.x; i < n; i += kThreads) {
        const Key k = row.key(i);
        if (k > t.key) total += row.mass(k);
      }
      total = block_all(total, lds.words, [](unsigned long long p, unsigned long long q) { return p + q; });
      int64_t floor_ties = kept_ties;
      if (row.s.top_k >= n) floor_ties = 0;  // no state has key 0
      total += (unsigned long long)floor_ties * (floor_ties ? row.mass(t.key) : 0ull);
      const Key floor = t.key;
      const double target = row.s.top_p * (double)total;
      find_threshold<T, true>(row, floor, floor_ties, target, lds, &t.key, &kept_ties, &ties, &above);
    }
    if (kept_ties < ties) {  // the index of the last kept state on the key
      int64_t seen = 0;
      for (int64_t base = 0; base < n; base += kThreads) {
        const int64_t i = base + threadIdx.x;
        const bool on = i < n && row.key(i) == t.key;
        double total;
        const int64_t before = seen + (int64_t)block_scan(on ? 1.0 : 0.0, lds.sums, &total);
        if (on && before == kept_ties - 1) lds.answer[2] = i;
        seen += (int64_t)total;
        __syncthreads();
        if (seen >= kept_ties) break;
      }
      __syncthreads();
      t.last_tie = lds.answer[2];
    }

    const auto kept_weight = [&](int64_t i) {
      if (i >= n) return 0.0;
      const Key k = row.key(i);
      if (k < t.key || (k == t.key && i > t.last_tie)) return 0.0;
      const double w = row.weight(k);
      return w >= row.s.min_p ? w : 0.0;
    };
    double total = 0.0;
    for (int64_t base = 0; base < n; base += kThreads) {
      double here;
      (void)block_scan(kept_weight(base + threadIdx.x), lds.sums, &here);
      total += here;
    }
    const double target = row.s.uniform * total;
    double before = 0.0;
    unsigned long long pick = ~0ull;
    int64_t last = -1;
    for (int64_t base = 0; base < n && pick == ~0ull; base += kThreads) {
      const int64_t i = base + threadIdx.x;
      const double w = kept_weight(i);
      double here;
      const double left = block_scan(w, lds.sums, &here);
      if (w > 0.0) last = i;
      unsigned long long mine = w > 0.0 && before + left + w > target ? (unsigned long long)i : ~0ull;
      before += here;
      if (before > target)
        pick = block_all(mine, lds.words, [](unsigned long long p, unsigned long long q) { return p < q ? p : q; });
    }
    if (pick == ~0ull) {  // u = 1, or the sums' rounding: the last kept state
      pick = block_all((unsigned long long)(last + 1), lds.words, larger) - 1;
    }
    if (threadIdx.x == 0) a.out[r] = (int32_t)pick;
  }
}

using bn::fail;

#define BN_HIP_CHECK(expr)                                                            \
  do {                                                                                \
    hipError_t err__ = (expr);                                                        \
    if (err__ != hipSuccess)                                                          \
      return fail(BN_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(err__));  \
  } while (0)

constexpr int64_t kMaxStates = 1 << 24;
constexpr int64_t kMaxBlocks = 1 << 20;

int check_draws(int dtype, const Draws& a) {
  const size_t es = dtype_bytes(dtype);
  if (es == 0) return fail(BN_ERR_INVALID, "dtype must be BN_F32, BN_F64, BN_F16 or BN_BF16");
  if (a.rows < 0 || a.rows > (int64_t)1 << 40) return fail(BN_ERR_INVALID, "bad number of rows");
  if (a.width < 1 || a.width > kMaxStates) return fail(BN_ERR_INVALID, "num_states must be in 1..2^24");
  if (a.stride < 0) return fail(BN_ERR_INVALID, "negative row stride");
  const bn_draw_filters& f = a.filters;
  if (!f.temperature_dev && !(f.temperature >= 0.0 && !std::isinf(f.temperature)))
    return fail(BN_ERR_INVALID, "temperature must be finite and not negative");
  if (!f.top_k_dev && f.top_k < 0) return fail(BN_ERR_INVALID, "top_k must not be negative");
  if (!f.top_p_dev && !(f.top_p > 0.0 && f.top_p <= 1.0)) return fail(BN_ERR_INVALID, "top_p must be in (0, 1]");
  if (!f.min_p_dev && !(f.min_p >= 0.0 && f.min_p <= 1.0)) return fail(BN_ERR_INVALID, "min_p must be in [0, 1]");
  return BN_OK;
}

}  // namespace

extern "C" {

int64_t bn_draw_states_workspace_bytes(int dtype, int64_t rows, int64_t num_states) {
  if (dtype_bytes(dtype) == 0 || rows < 0 || num_states < 1 || num_states > kMaxStates) return -1;
  return 8;
}

int bn_draw_states(int dtype, const void* logits_dev, int64_t rows, int64_t num_states, int64_t row_stride,
                   const int64_t* row_states_dev, int uniform_dtype, const void* uniforms_dev,
                   const bn_draw_filters* filters, void* workspace_dev, int32_t* out_dev, void* stream) {
  if (!filters) return fail(BN_ERR_INVALID, "filters is null");
  Draws a{logits_dev, rows, num_states, row_stride, row_states_dev, uniforms_dev, uniform_dtype, *filters, out_dev};
  if (int rc = check_draws(dtype, a)) return rc;
  if (uniform_dtype != BN_F32 && uniform_dtype != BN_F64)
    return fail(BN_ERR_INVALID, "uniform_dtype must be BN_F32 or BN_F64");
  if (rows == 0) return BN_OK;
  if (!logits_dev || !uniforms_dev || !workspace_dev || !out_dev) return fail(BN_ERR_INVALID, "null argument");
  if (reinterpret_cast<uintptr_t>(logits_dev) % dtype_bytes(dtype))
    return fail(BN_ERR_INVALID, "row address not aligned to its type");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((uint32_t)std::min(rows, kMaxBlocks));
  switch (dtype) {
    case BN_F32: hipLaunchKernelGGL(draw_rows<float>, grid, dim3(kThreads), 0, s, a); break;
    case BN_F64: hipLaunchKernelGGL(draw_rows<double>, grid, dim3(kThreads), 0, s, a); break;
    case BN_F16: hipLaunchKernelGGL(draw_rows<__half>, grid, dim3(kThreads), 0, s, a); break;
    default: hipLaunchKernelGGL(draw_rows<__hip_bfloat16>, grid, dim3(kThreads), 0, s, a); break;
  }
  BN_HIP_CHECK(hipGetLastError());
  return BN_OK;
}

}  // extern "C"
