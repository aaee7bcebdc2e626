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

__device__ __forceinline__ float exp_wide(float t) { return __builtin_amdgcn_exp2f(t * 1.44269504088896340736f); }
__device__ __forceinline__ double exp_wide(double t) { return exp(t); }

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

// ll of the row, in double: the difference to the largest logit is not rounded together with the
// logarithm, so a row whose state is nearly certain keeps its small value's digits
template <typename T, typename W>
__device__ __forceinline__ void finish_row(const Rows& a, int64_t r, const T* x, int64_t state, const Total<W>& total) {
  using Out = typename Value<T>::Wide;
  double ll = 0.0;
  if (state >= 0) {
    const double target = (double)Value<T>::widen(x[state]);
    ll = total.sum == (W)0 ? -INFINITY : (target - (double)total.reference()) - log((double)total.sum);
  }
  if (a.ll) static_cast<Out*>(a.ll)[r] = (Out)ll;
  if (a.totals) {
    a.totals[2 * r] = (double)total.best;
    a.totals[2 * r + 1] = (double)total.sum;
  }
}

// Gradient of a row: weight * ([i = state] - exp(x_i - best) / sum).
template <typename W>
struct Slope {
  W reference, scale, weight;
  int64_t state;
  __device__ __forceinline__ W at(W x, int64_t i) const {
    const W p = exp_wide(x - reference) * scale;
    return weight * ((i == state ? (W)1 : (W)0) - p);
  }
};

template <typename T>
__device__ __forceinline__ typename Value<T>::Wide row_weight(const Rows& a, int64_t r) {
  using W = typename Value<T>::Wide;
  return a.weights ? static_cast<const W*>(a.weights)[r * a.weights_stride] : (W)1;
}

template <typename T, typename W>
__device__ __forceinline__ Slope<W> slope_from_total(const Rows& a, int64_t r, int64_t state, const Total<W>& total) {
  // sum 0 (no possible state): scale 0 and weight 0 below
  const W weight = total.sum == (W)0 ? (W)0 : row_weight<T>(a, r);
  const W scale = total.sum == (W)0 ? (W)0 : (W)1 / total.sum;
  return {total.reference(), scale, weight, state};
}

// ---- short rows: LANES lanes hold a row as PACKS packs each -----------------------------------

template <typename T, int LANES, int PACKS, int MODE>
__global__ void __launch_bounds__(256) rows_in_lanes(const Rows a) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  constexpr int kRowsPerBlock = 256 / LANES;
  const int lane = threadIdx.x % LANES;
  for (int64_t r0 = (int64_t)blockIdx.x * kRowsPerBlock; r0 < a.rows; r0 += (int64_t)gridDim.x * kRowsPerBlock) {
    const int64_t r = r0 + threadIdx.x / LANES;
    if (r >= a.rows) continue;  // whole groups leave together: the shuffles below stay within a group
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    const int64_t n = row_count(a, r);
    const int64_t state = row_state(a, r, n);
    W v[PACKS * V];
    W best = -INFINITY;
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
      const int64_t i = (int64_t)(k * LANES + lane) * V;
      if (i + V <= n) {
        const Pack<T> p = load_pack(x + i);
#pragma unroll
        for (int j = 0; j < V; ++j) v[k * V + j] = Value<T>::widen(p.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[k * V + j] = i + j < n ? Value<T>::widen(x[i + j]) : (W)-INFINITY;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) best = fmax(best, v[k * V + j]);
    }
    Total<W> total;
    total.best = lanes_max<LANES>(best);
    const W reference = total.reference();
    W sum = 0;
#pragma unroll
    for (int k = 0; k < PACKS * V; ++k) sum += exp_wide(v[k] - reference);
    total.sum = lanes_sum<LANES>(sum);
    if (lane == 0) finish_row<T>(a, r, x, state, total);
    if constexpr (MODE == kBoth) {
      const Slope<W> slope = slope_from_total<T>(a, r, state, total);
      T* out = static_cast<T*>(a.gradient) + r * a.gradient_stride;
#pragma unroll
      for (int k = 0; k < PACKS; ++k) {
        const int64_t i = (int64_t)(k * LANES + lane) * V;
        Pack<T> p;
#pragma unroll
        for (int j = 0; j < V; ++j)
          p.v[j] = Value<T>::round(state >= 0 && i + j < n ? slope.at(v[k * V + j], i + j) : (W)0);
        if (i + V <= a.width) {
          store_pack(out + i, p);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (i + j < a.width) out[i + j] = p.v[j];
        }
      }
    }
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
  __syncthreads();
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
  __syncthreads();
  return s;
}

// Two or three passes over the row in memory: maximum, sum and (both) the gradient.
template <typename T, int THREADS, int MODE>
__global__ void __launch_bounds__(THREADS) rows_streamed(const Rows a) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  __shared__ W lds[THREADS / 64];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    const int64_t n = row_count(a, r);
    const int64_t state = row_state(a, r, n);
    const int64_t packs = n / V;
    W best = -INFINITY;
    for (int64_t k = threadIdx.x; k < packs; k += THREADS) {
      const Pack<T> p = load_pack(x + k * V);
#pragma unroll
      for (int j = 0; j < V; ++j) best = fmax(best, Value<T>::widen(p.v[j]));
    }
    const int64_t tail = packs * V + threadIdx.x;
    if (tail < n) best = fmax(best, Value<T>::widen(x[tail]));
    Total<W> total;
    total.best = block_max<THREADS>(best, lds);
    const W reference = total.reference();
    W sum = 0;
    for (int64_t k = threadIdx.x; k < packs; k += THREADS) {
      const Pack<T> p = load_pack(x + k * V);
#pragma unroll
      for (int j = 0; j < V; ++j) sum += exp_wide(Value<T>::widen(p.v[j]) - reference);
    }
    if (tail < n) sum += exp_wide(Value<T>::widen(x[tail]) - reference);
    total.sum = block_sum<THREADS>(sum, lds);
    if (threadIdx.x == 0) finish_row<T>(a, r, x, state, total);
    if constexpr (MODE == kBoth) {
      __syncthreads();  // finish_row reads the state's logit, which the gradient may overwrite
      const Slope<W> slope = slope_from_total<T>(a, r, state, total);
      T* out = static_cast<T*>(a.gradient) + r * a.gradient_stride;
      const int64_t out_packs = a.width / V;
      for (int64_t k = threadIdx.x; k < out_packs; k += THREADS) {
        const int64_t i = k * V;
        Pack<T> p;
        if (k < packs) p = load_pack(x + i);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          W g = 0;
          if (state >= 0 && i + j < n) g = slope.at(Value<T>::widen(k < packs ? p.v[j] : x[i + j]), i + j);
          p.v[j] = Value<T>::round(g);
        }
        store_pack(out + i, p);
      }
      const int64_t i = out_packs * V + threadIdx.x;
      if (i < a.width) out[i] = Value<T>::round(state >= 0 && i < n ? slope.at(Value<T>::widen(x[i]), i) : (W)0);
    }
  }
}

// ---- the backward pass on its own: elementwise, from the rows' totals ----------------------

// A block takes kPacksPerBlock packs of the output, row after row.
constexpr int kBackwardThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kBackwardThreads) rows_backward(const Rows a, int64_t packs_per_row) {
  using W = typename Value<T>::Wide;
  constexpr int V = Value<T>::kVec;
  const int64_t total_packs = a.rows * packs_per_row;
  for (int64_t q = (int64_t)blockIdx.x * kBackwardThreads + threadIdx.x; q < total_packs;
       q += (int64_t)gridDim.x * kBackwardThreads) {
    const int64_t r = q / packs_per_row;
    const int64_t i = (q - r * packs_per_row) * V;
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    T* out = static_cast<T*>(a.gradient) + r * a.gradient_stride;
    const int64_t n = row_count(a, r);
    const int64_t state = row_state(a, r, n);
    const Total<W> total{(W)a.totals[2 * r], (W)a.totals[2 * r + 1]};
    const Slope<W> slope = slope_from_total<T>(a, r, state, total);
    Pack<T> p;
    const bool whole = i + V <= n;
    if (whole) p = load_pack(x + i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      W g = 0;
      if (state >= 0 && i + j < n) g = slope.at(Value<T>::widen(whole ? p.v[j] : x[i + j]), i + j);
      p.v[j] = Value<T>::round(g);
    }
    if (i + V <= a.width) {
      store_pack(out + i, p);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i + j < a.width) out[i + j] = p.v[j];
    }
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

template <typename T, int LANES, int PACKS, int MODE>
void launch_lanes(const Rows& a, hipStream_t s) {
  const int64_t per_block = 256 / LANES;
  const int64_t blocks = std::min((a.rows + per_block - 1) / per_block, kMaxBlocks);
  hipLaunchKernelGGL((rows_in_lanes<T, LANES, PACKS, MODE>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
}

template <typename T, int MODE>
int launch_forward(const Rows& a, hipStream_t s) {
  constexpr int64_t V = Value<T>::kVec;
  const int64_t packs = (a.width + V - 1) / V;
  if (packs <= 1) launch_lanes<T, 1, 1, MODE>(a, s);
  else if (packs <= 2) launch_lanes<T, 2, 1, MODE>(a, s);
  else if (packs <= 4) launch_lanes<T, 4, 1, MODE>(a, s);
  else if (packs <= 8) launch_lanes<T, 8, 1, MODE>(a, s);
  else if (packs <= 16) launch_lanes<T, 16, 1, MODE>(a, s);
  else if (packs <= 32) launch_lanes<T, 32, 1, MODE>(a, s);
  else if (packs <= 64) launch_lanes<T, 64, 1, MODE>(a, s);
  else if (packs <= 128) launch_lanes<T, 64, 2, MODE>(a, s);
  else if (packs <= 256) launch_lanes<T, 64, 4, MODE>(a, s);
  else
    hipLaunchKernelGGL((rows_streamed<T, 512, MODE>), dim3((uint32_t)std::min(a.rows, kMaxBlocks)), dim3(512), 0, s, a);
  BN_HIP_CHECK(hipGetLastError());
  return BN_OK;
}

template <typename T>
int launch_backward(const Rows& a, hipStream_t s) {
  constexpr int64_t V = Value<T>::kVec;
  const int64_t packs = (a.width + V - 1) / V;
  const int64_t blocks = std::min((a.rows * packs + kBackwardThreads - 1) / kBackwardThreads, kMaxBlocks);
  hipLaunchKernelGGL(rows_backward<T>, dim3((uint32_t)blocks), dim3(kBackwardThreads), 0, s, a, packs);
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

// The gradient may replace the logits, row for row; any other overlap would change a row that is still read.
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
  if (!same && x < g_end && g < x_end)
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
