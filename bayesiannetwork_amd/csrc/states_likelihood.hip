// Log-likelihood of one state per row of logits, and its gradient: bn_states_log_likelihood* of
// include/bn_hip.h.
//
//   ll_r        = x_{r,s_r} - L_r,   L_r = log sum_i exp(x_{r,i})
//   d ll / dx_i = [i = s_r] - exp(x_{r,i} - L_r)
//
// Bound by memory: each logit is read once, and written once where the gradient is asked for.  A row
// belongs to a group of 4 to 64 lanes (short rows) or to a block; what a row's lanes can keep in
// registers between the sum and the gradient is not read again.
#include "../../include/bn_hip.h"

#include <algorithm>
#include <cmath>
#include <string>

#include <hip/hip_runtime.h>

#include "error.h"
#include "row_values.h"

namespace {

using namespace bn_rows;

// Arguments of every kernel here.
struct Rows {
  const void* logits;
  int64_t rows;
  int64_t width;           // states of a full row
  int64_t stride;          // elements between rows
  const int64_t* counts;   // states of each row, or null: width
  const void* states;
  int32_t state_bytes;     // 1 (unsigned), 4 or 8
  double* totals;          // [rows][2], a row's Total: written by the forward pass, read by the backward pass
  const void* weights;     // d loss / d ll, or null: 1
  int64_t weights_stride;
  void* ll;
  void* gradient;
  int64_t gradient_stride;
};

enum Mode { kForward, kBoth, kBackward };

__device__ __forceinline__ float exp_wide(float t) { return __builtin_amdgcn_exp2f(t * 1.44269502162933349609f); }
__device__ __forceinline__ double exp_wide(double t) { return exp(t); }

// exp(t), t <= 0, for gradients.  With float32 logits the roundings of t log2(e) are made good (five instructions;
// without it a gradient of 64 states was off by 1.2e-7 of its norm, with it by 4e-8).  They hardly
// move a sum of exponentials, and what 16-bit logits lead to is rounded far above them.
template <typename T>
__device__ __forceinline__ float exp_precise(float t) {
  constexpr float kLog2e = 1.44269502162933349609f, kRest = 1.92596303e-8f;  // together log2(e) to 48 bits
  if (sizeof(T) == 2) return exp_wide(t);
  const float y = t * kLog2e;
  const float e = __builtin_amdgcn_exp2f(y);
  // NaN or infinite where y is infinite: any finite number does, since e is 0 there
  const float r = fminf(fmaxf(fmaf(t, kRest, fmaf(t, kLog2e, -y)), -1.0f), 1.0f);
  return fmaf(e, r * 0.693147180559945f, e);
}
template <typename T>
__device__ __forceinline__ double exp_precise(double t) {
  return exp(t);
}

__device__ __forceinline__ int64_t row_count(const Rows& a, int64_t r) {
  if (!a.counts) return a.width;
  const int64_t n = a.counts[r];
  return n < 0 ? 0 : (n > a.width ? a.width : n);
}

// The row's state, -1 where it is none of the row's n states (an unobserved row).
__device__ __forceinline__ int64_t row_state(const Rows& a, int64_t r, int64_t n) {
  int64_t s;
  if (a.state_bytes == 8)
    s = static_cast<const int64_t*>(a.states)[r];
  else if (a.state_bytes == 4)
    s = static_cast<const int32_t*>(a.states)[r];
  else
    s = static_cast<const uint8_t*>(a.states)[r];
  return s >= 0 && s < n ? s : -1;
}

// A row's largest logit and sum of exp(x - best).  `best` is -inf and `sum` 0 for a row without possible
// states; NaN or +inf among the logits has made `sum` NaN.  The two are kept apart all the way: in
// best + log(sum) a row of logits near the type's lowest value (all masked) would lose its sum.
template <typename W>
struct Total {
  W best;
  W sum;
  __device__ __forceinline__ W reference() const { return isinf(best) && best < 0 ? (W)0 : best; }
};

// ll of a row, in double: the difference to the largest logit is not rounded together with the
// logarithm, so a row whose state is nearly certain keeps its small value down to the last bit of the sum (6e-8 for
// all types but float64).  `target` is the state's logit.
template <typename T, typename W>
__device__ __forceinline__ void finish_row(const Rows& a, int64_t r, bool observed, W target, const Total<W>& total) {
  double ll = 0.0;
  if (observed)
    ll = total.sum == (W)0 ? -INFINITY : ((double)target - (double)total.reference()) - log((double)total.sum);
  if (a.ll) static_cast<W*>(a.ll)[r] = (W)ll;
  if (a.totals) {
    a.totals[2 * r] = (double)total.best;
    a.totals[2 * r + 1] = (double)total.sum;
  }
}

// Gradient of a row: weight * ([i = state] - exp(x_i - best) / sum), 0 for a row that was not observed.
template <typename T>
struct Slope {
  using W = typename Value<T>::Wide;
  W reference, scale, weight;
  bool observed;
  __device__ __forceinline__ W at(W x, bool is_state) const {
    const W p = exp_precise<T>(x - reference) * scale;
    return weight * ((is_state ? (W)1 : (W)0) - p);
  }
};

template <typename T>
__device__ __forceinline__ typename Value<T>::Wide row_weight(const Rows& a, int64_t r) {
  using W = typename Value<T>::Wide;
  return a.weights ? static_cast<const W*>(a.weights)[r * a.weights_stride] : (W)1;
}

template <typename T, typename W>
__device__ __forceinline__ Slope<T> slope_from_total(W weight, bool observed, const Total<W>& total) {
  // sum 0: no possible state, no gradient
  const bool none = total.sum == (W)0;
  return {total.reference(), none ? (W)0 : (W)1 / total.sum, none ? (W)0 : weight, observed};
}

// The gradient at the V states from i on, of which the row has n (x: their logits); the row's state is `at`
// places behind i.  0 beyond the row.
template <typename T>
__device__ __forceinline__ Pack<T> gradient_pack(const Slope<T>& slope, Pack<T> x, int64_t at, int64_t inside) {
  constexpr int V = Value<T>::kVec;
  const int place = (uint64_t)at < (uint64_t)V ? (int)at : -1;
  if (!slope.observed) inside = 0;
  if (inside >= V) {
#pragma unroll
    for (int j = 0; j < V; ++j) x.v[j] = Value<T>::round(slope.at(Value<T>::widen(x.v[j]), place == j));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      x.v[j] = Value<T>::round(j < inside ? slope.at(Value<T>::widen(x.v[j]), place == j) : (typename Value<T>::Wide)0);
  }
  return x;
}

// Stores the part of a pack that lies inside a row of `width` states.
template <bool STREAM, typename T, typename Index>
__device__ __forceinline__ void store_row_pack(T* out, Index i, Index width, const Pack<T>& p) {
  constexpr int V = Value<T>::kVec;
  if (i + V <= width) {
    if (STREAM)
      store_pack_streamed(out + i, p);
    else
      store_pack(out + i, p);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i + j < width) out[i + j] = p.v[j];
  }
}

// The V logits from i on, -inf where the row's n states have ended.
template <typename T, typename Index>
__device__ __forceinline__ Pack<T> row_pack(const T* x, Index i, Index n) {
  constexpr int V = Value<T>::kVec;
  Pack<T> p;
  if (i + V <= n) {
    p = load_pack(x + i);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) p.v[j] = i + j < n ? x[i + j] : Value<T>::round(-INFINITY);
  }
  return p;
}

// The same as registers that stay packed.
template <typename T, typename Index>
__device__ __forceinline__ Raw row_raw(const T* x, Index i, Index n) {
  Raw raw;
  if (i + Value<T>::kVec <= n) {
    raw = raw_of(load_pack(x + i));
  } else {
    raw = raw_of(row_pack(x, i, n));
  }
  return raw;
}

// ---- short rows: LANES lanes hold a row as PACKS packs each -----------------------------------

// A group takes KEEP rows, all loaded before the first is worked on; the logarithms of their sums (a hundred
// double instructions, whatever the number of lanes that need one) are left to the end, where lane k has
// row k's.  (The gradient goes past the caches' order as in rows_in_block: 131072 x 64 float32 13.8 us, 17.9 us
// otherwise.)
template <typename T, int LANES, int PACKS, int KEEP, int MODE>
__global__ void __launch_bounds__(256) rows_in_lanes(const Rows a) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  constexpr int kRowsPerBlock = 256 / LANES * KEEP;
  static_assert(KEEP <= LANES, "one lane per kept row");
  const int lane = threadIdx.x % LANES, width = (int)a.width;
  for (int64_t r0 = (int64_t)blockIdx.x * kRowsPerBlock; r0 < a.rows; r0 += (int64_t)gridDim.x * kRowsPerBlock) {
    const int64_t base = r0 + (int64_t)(threadIdx.x / LANES) * KEEP;
    if (base >= a.rows) continue;  // whole groups leave together: the exchanges below stay within a group
    // lane k < KEEP knows row base + k
    const int64_t own = base + lane;
    const bool owner = lane < KEEP && own < a.rows;
    int own_count = 0, own_state = -1;
    W own_target = 0, own_weight = 0;
    if (owner) {
      own_count = (int)row_count(a, own);
      own_state = (int)row_state(a, own, own_count);
      if (own_state >= 0) own_target = Value<T>::widen(static_cast<const T*>(a.logits)[own * a.stride + own_state]);
      if (MODE == kBoth) own_weight = row_weight<T>(a, own);
    }
    Raw raw[KEEP][PACKS];
#pragma unroll
    for (int q = 0; q < KEEP; ++q) {
      const T* x = static_cast<const T*>(a.logits) + (base + q) * a.stride;
      const int n = __shfl(own_count, q, LANES);
#pragma unroll
      for (int k = 0; k < PACKS; ++k) raw[q][k] = row_raw(x, (k * LANES + lane) * V, n);
    }
    Total<W> own_total{(W)-INFINITY, (W)0};
#pragma unroll
    for (int q = 0; q < KEEP; ++q) {
      W best = -INFINITY;
#pragma unroll
      for (int k = 0; k < PACKS; ++k) {
        kept(raw[q][k]);
        const Pack<T> p = pack_of<T>(raw[q][k]);
#pragma unroll
        for (int j = 0; j < V; ++j) best = fmax(best, Value<T>::widen(p.v[j]));
      }
      Total<W> total;
      total.best = lanes_max<LANES>(best);
      const W reference = total.reference();
      W sum = 0;
#pragma unroll
      for (int k = 0; k < PACKS; ++k) {
        kept(raw[q][k]);
        const Pack<T> p = pack_of<T>(raw[q][k]);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += exp_wide(Value<T>::widen(p.v[j]) - reference);
      }
      total.sum = lanes_sum<LANES>(sum);
      if (lane == q) own_total = total;
      if constexpr (MODE == kBoth) {
        if (base + q >= a.rows) continue;
        const int n = __shfl(own_count, q, LANES), state = __shfl(own_state, q, LANES);
        const Slope<T> slope = slope_from_total<T>(__shfl(own_weight, q, LANES), state >= 0, total);
        T* out = static_cast<T*>(a.gradient) + (base + q) * a.gradient_stride;
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
          const int i = (k * LANES + lane) * V;
          kept(raw[q][k]);
          if (i < width)
            store_row_pack<true>(out, i, width, gradient_pack(slope, pack_of<T>(raw[q][k]), state - i, n - i));
        }
      }
    }
    if (owner) finish_row<T>(a, own, own_state >= 0, own_target, own_total);
  }
}

// ---- long rows: a block per row ---------------------------------------------------------------

template <int THREADS, typename W>
__device__ __forceinline__ W block_max(W v, W* lds) {
  v = lanes_max<64>(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  W m = lds[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) m = fmax(m, lds[w]);
  return m;
}

template <int THREADS, typename W>
__device__ __forceinline__ W block_sum(W v, W* lds) {
  v = lanes_sum<64>(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  W s = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) s += lds[w];
  return s;
}

// Log-likelihood and gradient of rows that a block's registers hold.  A thread takes its logits' exponentials
// relative to its own largest one and keeps them; once the block has agreed on the row's maximum and sum, one
// factor per thread turns them into the gradient.  So every logit costs one exponential, and its register is
// free again before the block has met: the next row's logits are requested then and arrive while this row is
// reduced and written.  4096 rows of 64000 bfloat16 states, 1.05 GB, take 191 us, 5.5 TB/s, in a long run of calls
// (a copy of the same tensors 196; the first 50 calls, as in profiles/row_operators_kernels.txt, 203); loading, reducing
// and storing one after the other took 353 us (a CU holds one such row, and its memory pipe idled in
// between), reading the row twice instead 318 us.
// The gradient is stored past the caches' order, which takes 13 us from that and 1.6 from 1000 rows of
// 5003 float32 (9.7 us now), where what reads it next is no slower for it (18.7 against 20.7 us together); between about
// 100 and 256 MB the next reader loses more than is won here (4096 x 16000: 44 against 46 us alone, 99
// against 92 together).
// HOLD: false where the exponentials do not fit the registers beside the logits.  They are taken twice then, and
// the next row is requested as this one is written.
//
// A row is up to PACKS rounds of THREADS whole packs, by uniform addresses and without checks, and a rest of
// less than a round with them (checks in the unrolled rounds cost more registers than the row itself).
template <typename T, int THREADS, int PACKS, bool HOLD>
__global__ void __launch_bounds__(THREADS) rows_in_block(const Rows a) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  constexpr int kWaves = THREADS / 64;
  constexpr int kRound = THREADS * V;  // states
  __shared__ W maxima[2][kWaves], sums[2][kWaves];  // by turns: one barrier per row is enough
  const int width = (int)a.width;
  const uint32_t place = threadIdx.x * V;  // of this thread's pack in every round
  const auto load = [&](const T* x, int k, int n) {
    Raw raw;
    if ((k + 1) * kRound <= n) {
      raw = raw_of(load_pack((x + k * kRound) + place));
    } else {
      Pack<T> none;
#pragma unroll
      for (int j = 0; j < V; ++j) none.v[j] = Value<T>::round(-INFINITY);
      raw = raw_of(none);
    }
    return raw;
  };
  int64_t r = blockIdx.x;
  if (r >= a.rows) return;
  int n = (int)row_count(a, r);
  Raw raw[PACKS], rest;
  {
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
#pragma unroll
    for (int k = 0; k < PACKS; ++k) raw[k] = load(x, k, n);
    rest = row_raw(x, n / kRound * kRound + (int)place, n);
  }
  for (int turn = 0;; turn ^= 1) {
    const int64_t next = r + gridDim.x;
    const bool more = next < a.rows;
    const int next_n = more ? (int)row_count(a, next) : 0;
    const int state = (int)row_state(a, r, n);
    const W weight = row_weight<T>(a, r);
    // the thread whose pack holds the row's state also writes its gradient, after the pack
    const bool owner = (int)threadIdx.x == (state >= 0 ? state / V % THREADS : 0);
    W target = 0;
    if (owner && state >= 0) target = Value<T>::widen(static_cast<const T*>(a.logits)[r * a.stride + state]);
    W own = -INFINITY;
    const auto raise = [&](Raw& from) {
      kept(from);
      const Pack<T> p = pack_of<T>(from);
#pragma unroll
      for (int j = 0; j < V; ++j) own = fmax(own, Value<T>::widen(p.v[j]));
    };
#pragma unroll
    for (int k = 0; k < PACKS; ++k) raise(raw[k]);
    raise(rest);
    const W reference = own == (W)-INFINITY ? (W)0 : own;
    W e[HOLD ? PACKS + 1 : 1][V], sum = 0;
    const auto add = [&](Raw& from, int k) {
      kept(from);
      const Pack<T> p = pack_of<T>(from);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const W power = exp_precise<T>(Value<T>::widen(p.v[j]) - reference);
        if (HOLD) e[HOLD ? k : 0][j] = power;
        sum += power;
      }
    };
    const T* next_x = static_cast<const T*>(a.logits) + next * a.stride;
    const auto load_next = [&](int k) {  // nothing if there is no next row
      if (k < PACKS)
        raw[k < PACKS ? k : 0] = load(next_x, k, next_n);
      else
        rest = row_raw(next_x, next_n / kRound * kRound + (int)place, next_n);
    };
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
      add(raw[k], k);
      if (HOLD) load_next(k);
    }
    add(rest, PACKS);
    if (HOLD) load_next(PACKS);
    // (a thread or wave without possible states has sum 0 and stays out through the factor 0; NaN stays in)
    const W wave_best = lanes_max<64>(own);
    const W wave_sum = lanes_sum<64>(sum * (own == (W)-INFINITY ? (W)0 : exp_wide(own - wave_best)));
    if ((threadIdx.x & 63) == 0) {
      maxima[turn][threadIdx.x >> 6] = wave_best;
      sums[turn][threadIdx.x >> 6] = wave_sum;
    }
    __syncthreads();  // every thread has read its logits, the owner the state's: the gradient may replace them
    Total<W> total{(W)-INFINITY, (W)0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total.best = fmax(total.best, maxima[turn][w]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      total.sum += sums[turn][w] * (maxima[turn][w] == (W)-INFINITY ? (W)0 : exp_wide(maxima[turn][w] - total.best));
    const Slope<T> slope = slope_from_total<T>(weight, state >= 0, total);
    const W factor = (own == (W)-INFINITY ? (W)0 : exp_precise<T>(own - total.best)) * slope.scale * -slope.weight;
    T* out = static_cast<T*>(a.gradient) + r * a.gradient_stride;
    const auto gradient_of = [&](Raw& from, int k) {
      Pack<T> g;
      if (HOLD) {
#pragma unroll
        for (int j = 0; j < V; ++j) g.v[j] = Value<T>::round(e[HOLD ? k : 0][j] * factor);
      } else {
        kept(from);
        const Pack<T> p = pack_of<T>(from);
#pragma unroll
        for (int j = 0; j < V; ++j) g.v[j] = Value<T>::round(exp_precise<T>(Value<T>::widen(p.v[j]) - reference) * factor);
      }
      return g;
    };
    int written = 0;  // states behind which the gradient is 0
    if (state >= 0) {
#pragma unroll
      for (int k = 0; k < PACKS; ++k) {
        if ((k + 1) * kRound <= n) store_pack_streamed((out + k * kRound) + place, gradient_of(raw[k], k));
        if (!HOLD) load_next(k);
      }
      const int i = n / kRound * kRound + (int)place;
      if (i < n) store_row_pack<false>(out, i, n, gradient_of(rest, PACKS));
      written = n;
    } else if (!HOLD) {
#pragma unroll
      for (int k = 0; k < PACKS; ++k) load_next(k);
    }
    if (!HOLD) load_next(PACKS);
    for (int i = written + (int)threadIdx.x; i < width; i += THREADS) out[i] = Value<T>::round((W)0);
    if (owner) {
      if (state >= 0) out[state] = Value<T>::round(slope.at(target, true));
      finish_row<T>(a, r, state >= 0, target, total);
    }
    if (!more) return;
    r = next;
    n = next_n;
  }
}

// Longer rows, or rows that only need their sum: one pass with a running maximum, whose change rescales the
// sum, and (both) a second one over the row in memory.
template <typename T, int THREADS, int AHEAD, int MODE>
__global__ void __launch_bounds__(THREADS) rows_streamed(const Rows a) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  __shared__ W maxima[THREADS / 64], sums[THREADS / 64];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    const int64_t n = row_count(a, r);
    const int64_t state = row_state(a, r, n);
    W target = 0;
    if (threadIdx.x == 0 && state >= 0) target = Value<T>::widen(x[state]);
    // AHEAD packs are worked on while the next ones arrive, with one look at the maximum for all of them
    Total<W> own{(W)-INFINITY, (W)0};
    constexpr int64_t kStep = (int64_t)THREADS * V * AHEAD;
    Raw next[AHEAD];
    const auto load = [&](int64_t start) {
      if (start + kStep <= n) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) next[k] = raw_of(load_pack((x + start + k * THREADS * V) + threadIdx.x * V));
      } else {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) next[k] = row_raw(x, start + (int64_t)(k * THREADS + threadIdx.x) * V, n);
      }
    };
    load(0);
    for (int64_t start = 0; start < n; start += kStep) {
      Raw raw[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) raw[k] = next[k];
      load(start + kStep);
      W best = own.best;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        kept(raw[k]);
        const Pack<T> p = pack_of<T>(raw[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) best = fmax(best, Value<T>::widen(p.v[j]));
      }
      if (best > own.best) {
        if (own.sum != (W)0) own.sum *= exp_wide(own.best - best);  // 0 stays 0 while best was -inf
        own.best = best;
      }
      const W reference = own.reference();
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        kept(raw[k]);
        const Pack<T> p = pack_of<T>(raw[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) own.sum += exp_wide(Value<T>::widen(p.v[j]) - reference);
      }
    }
    Total<W> total;
    total.best = block_max<THREADS>(own.best, maxima);
    if (own.sum != (W)0) own.sum *= exp_wide(own.reference() - total.reference());
    total.sum = block_sum<THREADS>(own.sum, sums);
    if constexpr (MODE == kBoth) {
      const Slope<T> slope = slope_from_total<T>(row_weight<T>(a, r), state >= 0, total);
      T* out = static_cast<T*>(a.gradient) + r * a.gradient_stride;
#pragma unroll 2
      for (int64_t i = (int64_t)threadIdx.x * V; i < a.width; i += THREADS * V)
        store_row_pack<true>(out, i, a.width, gradient_pack(slope, row_pack(x, i, n), state - i, n - i));
    }
    if (threadIdx.x == 0) finish_row<T>(a, r, state >= 0, target, total);
    __syncthreads();  // the next row writes maxima and sums
  }
}

// ---- the backward pass on its own: elementwise, from the rows' totals --------------------------

constexpr int kBackwardThreads = 256;

// Index: uint32_t where all packs can be counted in 32 bits, whose division is five times cheaper.
template <typename T, typename Index>
__global__ void __launch_bounds__(kBackwardThreads) rows_backward(const Rows a, Index packs_per_row, Index packs) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  const Index step = (Index)gridDim.x * kBackwardThreads;
  Index q = (Index)blockIdx.x * kBackwardThreads + threadIdx.x;
  if (q >= packs) return;
  while (true) {
    const int64_t r = q / packs_per_row;
    const int64_t i = (int64_t)(q - (Index)r * packs_per_row) * V;
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    const int64_t n = row_count(a, r);
    const Pack<T> p = row_pack(x, i, n);
    const Total<W> total{(W)a.totals[2 * r], (W)a.totals[2 * r + 1]};
    const int64_t state = row_state(a, r, n);
    const Slope<T> slope = slope_from_total<T>(row_weight<T>(a, r), state >= 0, total);
    store_row_pack<false>(static_cast<T*>(a.gradient) + r * a.gradient_stride, i, a.width,
                   gradient_pack(slope, p, state - i, n - i));
    if (packs - q <= step) return;
    q += step;
  }
}

// ---- launches -----------------------------------------------------------------------------------

using bn::fail;

#define BN_HIP_CHECK(expr)                                                            \
  do {                                                                                \
    hipError_t err__ = (expr);                                                        \
    if (err__ != hipSuccess)                                                          \
      return fail(BN_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(err__));  \
  } while (0)

constexpr int64_t kMaxBlocks = 1 << 20;

template <typename T, int LANES, int PACKS, int KEEP, int MODE>
void launch_lanes(const Rows& a, hipStream_t s) {
  const int64_t per_block = 256 / LANES * KEEP;
  const int64_t blocks = std::min((a.rows + per_block - 1) / per_block, kMaxBlocks);
  hipLaunchKernelGGL((rows_in_lanes<T, LANES, PACKS, KEEP, MODE>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
}

template <typename T, int LANES, int PACKS, int MODE>
void launch_short(const Rows& a, hipStream_t s) {
  constexpr int kKeep = std::min(LANES, PACKS == 4 ? 2 : 4);
  // several rows per group once that leaves every SIMD (1024) four waves (131072 x 64 float32, forward: 14.6 us at
  // one row per group, 10.4 at two, 8.9 at four and at eight)
  if (kKeep > 1 && a.rows * LANES >= (int64_t)64 * 4096 * kKeep)
    launch_lanes<T, LANES, PACKS, kKeep, MODE>(a, s);
  else
    launch_lanes<T, LANES, PACKS, 1, MODE>(a, s);
}

template <typename T, int THREADS, int PACKS, bool HOLD = true>
void launch_block(const Rows& a, hipStream_t s) {
  // as many blocks as the 256 CUs' registers hold at a time
  constexpr int64_t kPerCu = PACKS == 16 ? 1 : PACKS == 8 ? 768 / THREADS : 1024 / THREADS;
  hipLaunchKernelGGL((rows_in_block<T, THREADS, PACKS, HOLD>), dim3((uint32_t)std::min<int64_t>(a.rows, 256 * kPerCu)),
                     dim3(THREADS), 0, s, a);
}

// Forward, us at 256 threads with 2 packs ahead / 512 with 4: 4096 x 32000 bfloat16 45 / 58, 4096 x 5003 float32
// 17 / 28, 2048 x 128000 bfloat16 103 / 97, 8 x 128000 18 / 13; both, 1024 x 128000 float32: 322 / 285.
template <typename T, int THREADS, int AHEAD, int MODE>
void launch_streamed(const Rows& a, hipStream_t s) {
  hipLaunchKernelGGL((rows_streamed<T, THREADS, AHEAD, MODE>), dim3((uint32_t)std::min(a.rows, kMaxBlocks)),
                     dim3(THREADS), 0, s, a);
}

template <typename T, int MODE>
int launch_forward(const Rows& a, hipStream_t s) {
  constexpr int64_t V = Value<T>::kVec;
  const int64_t packs = (a.width + V - 1) / V;
  if (packs <= 1) launch_short<T, 1, 1, MODE>(a, s);
  else if (packs <= 2) launch_short<T, 2, 1, MODE>(a, s);
  else if (packs <= 4) launch_short<T, 4, 1, MODE>(a, s);
  else if (packs <= 8) launch_short<T, 8, 1, MODE>(a, s);
  else if (packs <= 16) launch_short<T, 16, 1, MODE>(a, s);
  else if (packs <= 32) launch_short<T, 32, 1, MODE>(a, s);
  else if (packs <= 64) launch_short<T, 64, 1, MODE>(a, s);
  else if (packs <= 128) launch_short<T, 64, 2, MODE>(a, s);
  else if (packs <= 256) launch_short<T, 64, 4, MODE>(a, s);
  else if (MODE == kBoth && packs <= 256 * 4) launch_block<T, 256, 4>(a, s);
  else if (MODE == kBoth && packs <= 256 * 8) launch_block<T, 256, 8>(a, s);
  else if (MODE == kBoth && packs <= 512 * 8) launch_block<T, 512, 8>(a, s);
  else if (MODE == kBoth && packs <= 512 * 16) launch_block<T, 512, 16>(a, s);
  else if (MODE == kBoth && packs <= 1024 * 16) launch_block<T, 1024, 16, false>(a, s);
  else if (packs <= 8192) launch_streamed<T, 256, 2, MODE>(a, s);
  else launch_streamed<T, 512, 4, MODE>(a, s);
  BN_HIP_CHECK(hipGetLastError());
  return BN_OK;
}

template <typename T>
int launch_backward(const Rows& a, hipStream_t s) {
  constexpr int64_t V = Value<T>::kVec;
  const int64_t per_row = (a.width + V - 1) / V, packs = a.rows * per_row;
  const dim3 grid((uint32_t)std::min((packs + kBackwardThreads - 1) / kBackwardThreads, kMaxBlocks));
  if (packs < (int64_t)1 << 32)
    hipLaunchKernelGGL((rows_backward<T, uint32_t>), grid, dim3(kBackwardThreads), 0, s, a, (uint32_t)per_row,
                       (uint32_t)packs);
  else
    hipLaunchKernelGGL((rows_backward<T, uint64_t>), grid, dim3(kBackwardThreads), 0, s, a, (uint64_t)per_row,
                       (uint64_t)packs);
  BN_HIP_CHECK(hipGetLastError());
  return BN_OK;
}

template <typename T>
int launch(const Rows& a, int mode, hipStream_t s) {
  if (mode == kForward) return launch_forward<T, kForward>(a, s);
  if (mode == kBoth) return launch_forward<T, kBoth>(a, s);
  return launch_backward<T>(a, s);
}

int launch_any(int dtype, const Rows& a, int mode, hipStream_t s) {
  switch (dtype) {
    case BN_F32: return launch<float>(a, mode, s);
    case BN_F64: return launch<double>(a, mode, s);
    case BN_F16: return launch<__half>(a, mode, s);
    default: return launch<__hip_bfloat16>(a, mode, s);
  }
}

int check_rows(int dtype, const Rows& a) {
  const size_t es = dtype_bytes(dtype);
  if (es == 0) return fail(BN_ERR_INVALID, "dtype must be BN_F32, BN_F64, BN_F16 or BN_BF16");
  if (a.rows < 0 || a.width < 1) return fail(BN_ERR_INVALID, "rows must not be negative and num_states must be positive");
  if (a.width > (int64_t)1 << 40 || a.rows > (int64_t)1 << 40) return fail(BN_ERR_INVALID, "too many rows or states");
  if (a.state_bytes != 1 && a.state_bytes != 4 && a.state_bytes != 8)
    return fail(BN_ERR_INVALID, "states must be of 1, 4 or 8 bytes");
  if (a.rows == 0) return BN_OK;
  if (!a.logits || !a.states) return fail(BN_ERR_INVALID, "null argument");
  if (a.stride < 0) return fail(BN_ERR_INVALID, "negative row stride");
  if (reinterpret_cast<uintptr_t>(a.logits) % es || reinterpret_cast<uintptr_t>(a.gradient) % es)
    return fail(BN_ERR_INVALID, "row address not aligned to its type");
  return BN_OK;
}

// The gradient may replace the logits, row for row, or have columns of its own between them (the same stride); any
// other overlap would change a row that is still read.
int check_gradient(int dtype, const Rows& a) {
  if (a.rows == 0) return BN_OK;
  if (!a.gradient) return fail(BN_ERR_INVALID, "null argument");
  if (a.rows > 1 && a.gradient_stride < a.width)
    return fail(BN_ERR_INVALID, "the gradient's rows overlap: gradient_stride is below num_states");
  const uintptr_t es = dtype_bytes(dtype);
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.logits), g = reinterpret_cast<uintptr_t>(a.gradient);
  const uintptr_t x_end = x + ((uintptr_t)(a.rows - 1) * a.stride + a.width) * es;
  const uintptr_t g_end = g + ((uintptr_t)(a.rows - 1) * a.gradient_stride + a.width) * es;
  const bool same = x == g && (a.rows == 1 || a.stride == a.gradient_stride);
  const uintptr_t row = (uintptr_t)a.width * es, pitch = (uintptr_t)a.stride * es;
  bool between = false;
  if (a.stride == a.gradient_stride && a.stride >= 2 * a.width) {
    const uintptr_t behind = g >= x ? (g - x) % pitch : pitch - (x - g) % pitch;  // of a row's start, within the pitch
    between = behind >= row && behind <= pitch - row;
  }
  if (!same && !between && x < g_end && g < x_end)
    return fail(BN_ERR_INVALID, "the gradient lies over the logits without being the same rows");
  return BN_OK;
}

}  // namespace

extern "C" {

int bn_states_log_likelihood(int dtype, const void* logits_dev, int64_t rows, int64_t num_states, int64_t row_stride,
                             const int64_t* row_states_dev, const void* states_dev, int32_t state_bytes,
                             void* ll_out_dev, double* totals_out_dev, void* stream) {
  Rows a{};
  a.logits = logits_dev;
  a.rows = rows;
  a.width = num_states;
  a.stride = row_stride;
  a.counts = row_states_dev;
  a.states = states_dev;
  a.state_bytes = state_bytes;
  a.ll = ll_out_dev;
  a.totals = totals_out_dev;
  if (int rc = check_rows(dtype, a)) return rc;
  if (rows == 0) return BN_OK;
  if (!ll_out_dev) return fail(BN_ERR_INVALID, "null argument");
  return launch_any(dtype, a, kForward, static_cast<hipStream_t>(stream));
}

int bn_states_log_likelihood_gradient(int dtype, const void* logits_dev, int64_t rows, int64_t num_states,
                                      int64_t row_stride, const int64_t* row_states_dev, const void* states_dev,
                                      int32_t state_bytes, const double* totals_dev, const void* weights_dev,
                                      int64_t weights_stride, void* ll_out_dev, void* gradient_out_dev,
                                      int64_t gradient_stride, void* stream) {
  Rows a{};
  a.logits = logits_dev;
  a.rows = rows;
  a.width = num_states;
  a.stride = row_stride;
  a.counts = row_states_dev;
  a.states = states_dev;
  a.state_bytes = state_bytes;
  a.totals = const_cast<double*>(totals_dev);
  a.weights = weights_dev;
  a.weights_stride = weights_stride;
  a.ll = totals_dev ? nullptr : ll_out_dev;
  a.gradient = gradient_out_dev;
  a.gradient_stride = gradient_stride;
  if (int rc = check_rows(dtype, a)) return rc;
  if (weights_dev && weights_stride < 0) return fail(BN_ERR_INVALID, "negative weight stride");
  if (int rc = check_gradient(dtype, a)) return rc;
  if (rows == 0) return BN_OK;
  if (totals_dev && ll_out_dev)
    return fail(BN_ERR_INVALID, "ll_out is written together with the totals: pass either totals or ll_out");
  return launch_any(dtype, a, totals_dev ? kBackward : kBoth, static_cast<hipStream_t>(stream));
}

}  // extern "C"
