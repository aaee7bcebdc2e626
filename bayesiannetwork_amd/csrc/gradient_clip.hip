// Global gradient norm over many tensors, and clipping: bn_gradient_set_* of include/bn_hip.h.
//
//   norm = sqrt(sum over all tensors and elements of g^2)
//   out  = g * (norm > max_norm ? max_norm / norm : 1)
//
// Bound by memory: every gradient is read for the norm and, since no element can be scaled before the
// last one has been seen, read again for the copy.  A set lists its tensors once, cut into chunks of
// at most 8 KiB that one wave streams with 16-byte loads; tensors of any number, size and type are
// then two launches (785 tables of 20 elements: 2.7 + 3.4 us).  Neighbours in memory are joined before they
// are cut, so a model whose tables are slices of one buffer is one tensor to the kernels; what precedes the
// first cache line of an output is a chunk of its own, since 16-byte stores across lines cost twice.
//
// The second pass takes the chunks from the last to the first: what the first pass read last is still in the
// 256 MB cache.  Sets that do not fit it store past it.  8 x 64 MiB float32, copied: 267 us (in the same order
// and through the cache 316; reading and writing 1.6 GB without any reuse would be 300).
//
// Squares are summed in double: the square of any float32 is finite there, and the conversions keep
// up with the loads several times over.  Those of float64 gradients may leave double's range on either side while
// the norm does not: such tensors are summed at three scales, and the one that fits is taken.  A wave's chunks, a
// block's waves and the blocks are summed in an order that depends on the set alone - no atomics, the same bits
// every time.
#include "../../include/bn_hip.h"

#include <algorithm>
#include <cmath>
#include <new>
#include <string>
#include <vector>

#include <hip/hip_runtime.h>

#include "error.h"
#include "row_values.h"

namespace {

using namespace bn_rows;

struct Chunk {
  const void* source;
  void* output;
  int32_t count;  // elements
  int32_t dtype;
};

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kChunkBytes = 8192;
constexpr int kMaxBlocks = 1024;  // 4 blocks of 4 waves on each of 256 CUs
constexpr uintptr_t kLine = 128;  // bytes of a cache line
constexpr int64_t kCacheBytes = (int64_t)256 << 20;

// Sums of squares: as they are, and of float64 gradients also times 2^-600 and 2^600 each.  Where the first overflows
// all that counts is in the second; where it is below 2^-800 there is no other type's element but zeros, and
// none that the third has no room for.
constexpr double kDown = 0x1p-600, kUp = 0x1p600, kTiny = 0x1p-800;
struct Squares {
  double sum = 0.0, large = 0.0, small = 0.0;
  template <typename T>
  __device__ __forceinline__ void add(T v) {
    const double x = (double)Value<T>::widen(v);
    sum = fma(x, x, sum);
    if constexpr (sizeof(T) == 8) {
      large = fma(x * kDown, x * kDown, large);
      small = fma(x * kUp, x * kUp, small);
    }
  }
};

template <typename T>
__device__ __forceinline__ void chunk_squares(const Chunk& c, int lane, Squares& squares) {
  constexpr int V = Value<T>::kVec;
  const T* g = static_cast<const T*>(c.source);
  Squares own;  // summed by itself: a chunk's order is the same wherever it is taken
  const int packs = c.count / V;
#pragma unroll 4
  for (int i = lane; i < packs; i += 64) {
    const Pack<T> p = load_pack(g + (size_t)i * V);
#pragma unroll
    for (int j = 0; j < V; ++j) own.add(p.v[j]);
  }
  const int i = packs * V + lane;
  if (i < c.count) own.add(g[i]);
  squares.sum += own.sum;
  if constexpr (sizeof(T) == 8) {
    squares.large += own.large;
    squares.small += own.small;
  }
}

// max_norm / norm, or 1.  Where double has no room for that quotient (the other types' products are 0 then) float64
// gradients are divided by the norm and multiplied by max_norm, in the order that stays in range: |g| <= norm.
struct Factor {
  double factor;
  double before = 1.0, inverse, after = 1.0;
  __device__ __forceinline__ Factor(double norm, double max_norm) {
    // a NaN norm leaves no gradient usable: every element becomes NaN; an infinite one gives factor 0
    factor = inverse = norm <= max_norm ? 1.0 : max_norm / norm;
    if (factor < 0x1p-900 && !isinf(norm)) {
      const double down = norm > 1.0 ? kDown : 1.0;
      before = down * fmax(max_norm, 1.0);
      inverse = 1.0 / (norm * down);
      after = fmin(max_norm, 1.0);
    }
  }
};

template <typename T>
__device__ __forceinline__ T scaled(T v, const Factor& f) {
  // one product in double; the 16-bit types pass through float32 on the way, whose step is 2^-13 (half)
  // and 2^-16 (bfloat16) of theirs
  if constexpr (sizeof(T) == 8)
    return v * f.before * f.inverse * f.after;
  else
    return Value<T>::round((float)((double)Value<T>::widen(v) * f.factor));
}

template <typename T, bool STREAM>
__device__ __forceinline__ void chunk_scale(const Chunk& c, int lane, const Factor& factor) {
  constexpr int V = Value<T>::kVec;
  const T* g = static_cast<const T*>(c.source);
  T* out = static_cast<T*>(c.output);
  const int packs = c.count / V;
#pragma unroll 4
  for (int i = lane; i < packs; i += 64) {
    Pack<T> p = load_pack(g + (size_t)i * V);
#pragma unroll
    for (int j = 0; j < V; ++j) p.v[j] = scaled<T>(p.v[j], factor);
    if (STREAM)
      store_pack_streamed(out + (size_t)i * V, p);
    else
      store_pack(out + (size_t)i * V, p);
  }
  const int i = packs * V + lane;
  if (i < c.count) out[i] = scaled<T>(g[i], factor);
}

// sum over the block, the same in every thread (a barrier between one sum and the next is the caller's)
__device__ __forceinline__ double block_sum(double v, double* lds) {
  v = lanes_sum<64>(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += lds[w];
  return total;
}

// `partials`: every block's sum; where the set has float64 gradients (`doubles`), then the large and the small ones.
__global__ void __launch_bounds__(kThreads) gradient_squares(const Chunk* __restrict__ chunks, int64_t n_chunks,
                                                            int doubles, double* __restrict__ partials) {
  __shared__ double lds[kWaves];
  const int lane = threadIdx.x & 63;
  Squares squares;
  for (int64_t k = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); k < n_chunks; k += (int64_t)gridDim.x * kWaves) {
    const Chunk c = chunks[k];
    switch (c.dtype) {
      case BN_F32: chunk_squares<float>(c, lane, squares); break;
      case BN_F64: chunk_squares<double>(c, lane, squares); break;
      case BN_F16: chunk_squares<__half>(c, lane, squares); break;
      default: chunk_squares<__hip_bfloat16>(c, lane, squares); break;
    }
  }
  const double total = block_sum(squares.sum, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
  if (doubles) {
    __syncthreads();
    const double large = block_sum(squares.large, lds);
    __syncthreads();
    const double small = block_sum(squares.small, lds);
    if (threadIdx.x == 0) {
      partials[gridDim.x + blockIdx.x] = large;
      partials[2 * gridDim.x + blockIdx.x] = small;
    }
  }
}

__device__ __forceinline__ double norm_of(const double* __restrict__ partials, int n_partials, int doubles, double* lds) {
  const auto total = [&](const double* from) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < n_partials; i += kThreads) sum += from[i];
    return block_sum(sum, lds);
  };
  const double sum = total(partials);
  const bool over = isinf(sum);
  if (!doubles || !(over || sum < kTiny)) return sqrt(sum);
  __syncthreads();
  return sqrt(total(partials + (over ? 1 : 2) * n_partials)) * (over ? kUp : kDown);
}

__global__ void __launch_bounds__(kThreads) gradient_norm_finish(const double* __restrict__ partials, int n_partials,
                                                                int doubles, double* __restrict__ norm_out) {
  __shared__ double lds[kWaves];
  const double norm = norm_of(partials, n_partials, doubles, lds);
  if (threadIdx.x == 0) *norm_out = norm;
}

// STREAM: gradients and outputs together exceed the cache.
template <bool STREAM>
__global__ void __launch_bounds__(kThreads) gradient_scale(const Chunk* __restrict__ chunks, int64_t n_chunks,
                                                          const double* __restrict__ partials, int n_partials,
                                                          int doubles, double max_norm, double* __restrict__ norm_out) {
  __shared__ double lds[kWaves];
  const double norm = norm_of(partials, n_partials, doubles, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const Factor factor(norm, max_norm);
  const int lane = threadIdx.x & 63;
  for (int64_t k = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); k < n_chunks; k += (int64_t)gridDim.x * kWaves) {
    const Chunk c = chunks[n_chunks - 1 - k];
    switch (c.dtype) {
      case BN_F32: chunk_scale<float, STREAM>(c, lane, factor); break;
      case BN_F64: chunk_scale<double, STREAM>(c, lane, factor); break;
      case BN_F16: chunk_scale<__half, STREAM>(c, lane, factor); break;
      default: chunk_scale<__hip_bfloat16, STREAM>(c, lane, factor); break;
    }
  }
}

struct Range {
  uintptr_t begin, end;
  int32_t tensor;
};

}  // namespace

struct bn_gradient_set {
  int device = 0;
  int64_t n_chunks = 0;
  int64_t bytes = 0;  // of all gradients
  int blocks = 1;
  int doubles = 0;  // whether any gradient is of float64
  Chunk* d_chunks = nullptr;
};

namespace {

using bn::fail;

#define BN_HIP_CHECK(expr)                                                            \
  do {                                                                                \
    hipError_t err__ = (expr);                                                        \
    if (err__ != hipSuccess)                                                          \
      return fail(BN_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(err__));  \
  } while (0)

// Every output must be its own gradient's memory or memory that nothing else in the set uses: a block
// that scales one tensor must not change what another still reads or writes.
int check_overlap(int32_t n, const int32_t* dtypes, const int64_t* sizes, const void* const* sources,
                  void* const* outputs) {
  std::vector<Range> out, in;
  for (int32_t t = 0; t < n; ++t) {
    if (sizes[t] == 0) continue;
    const uintptr_t bytes = (uintptr_t)sizes[t] * dtype_bytes(dtypes[t]);
    const uintptr_t o = reinterpret_cast<uintptr_t>(outputs[t]), s = reinterpret_cast<uintptr_t>(sources[t]);
    out.push_back({o, o + bytes, t});
    in.push_back({s, s + bytes, t});
  }
  const auto by_begin = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  std::sort(out.begin(), out.end(), by_begin);
  std::sort(in.begin(), in.end(), by_begin);
  for (size_t i = 1; i < out.size(); ++i)
    if (out[i].begin < out[i - 1].end)
      return fail(BN_ERR_INVALID, "outputs " + std::to_string(out[i - 1].tensor) + " and " +
                                      std::to_string(out[i].tensor) + " share memory");
  // outputs are disjoint from here on; sweep both lists for outputs that meet a gradient not their own
  size_t first = 0;
  for (const Range& s : in) {
    while (first < out.size() && out[first].end <= s.begin) ++first;
    for (size_t i = first; i < out.size() && out[i].begin < s.end; ++i)
      if (out[i].tensor != s.tensor || out[i].begin != s.begin)
        return fail(BN_ERR_INVALID, "output " + std::to_string(out[i].tensor) + " lies over gradient " +
                                        std::to_string(s.tensor));
  }
  return BN_OK;
}

int build_set(int32_t n, const int32_t* dtypes, const int64_t* sizes, const void* const* sources,
              void* const* outputs, bn_gradient_set* set) {
  if (int rc = check_overlap(n, dtypes, sizes, sources, outputs)) return rc;
  std::vector<Chunk> chunks;
  int32_t t = 0;
  while (t < n) {
    const int64_t es = (int64_t)dtype_bytes(dtypes[t]);
    const char* s = static_cast<const char*>(sources[t]);
    char* o = static_cast<char*>(outputs[t]);
    int64_t count = sizes[t];
    int32_t last = t;
    // the next tensor continues this one in both arrays: one run
    while (count > 0 && last + 1 < n && dtypes[last + 1] == dtypes[t] && sizes[last + 1] > 0 &&
           static_cast<const char*>(sources[last + 1]) == s + count * es &&
           static_cast<char*>(outputs[last + 1]) == o + count * es)
      count += sizes[++last];
    set->bytes += count * es;
    if (dtypes[t] == BN_F64 && count > 0) set->doubles = 1;
    int64_t here = (int64_t)((kLine - reinterpret_cast<uintptr_t>(o) % kLine) % kLine) / es;
    if (here == 0) here = kChunkBytes / es;
    for (int64_t done = 0; done < count; done += here, here = kChunkBytes / es) {
      here = std::min(count - done, here);
      chunks.push_back({s + done * es, o + done * es, (int32_t)here, dtypes[t]});
    }
    t = last + 1;
  }
  set->n_chunks = (int64_t)chunks.size();
  set->blocks = (int)std::min<int64_t>(std::max<int64_t>((set->n_chunks + kWaves - 1) / kWaves, 1), kMaxBlocks);
  BN_HIP_CHECK(hipGetDevice(&set->device));
  if (!chunks.empty()) {
    BN_HIP_CHECK(hipMalloc(reinterpret_cast<void**>(&set->d_chunks), chunks.size() * sizeof(Chunk)));
    BN_HIP_CHECK(hipMemcpy(set->d_chunks, chunks.data(), chunks.size() * sizeof(Chunk), hipMemcpyHostToDevice));
  }
  return BN_OK;
}

int launch_squares(const bn_gradient_set* set, double* partials, hipStream_t s) {
  int device = -1;
  if (hipGetDevice(&device) != hipSuccess || device != set->device)
    return fail(BN_ERR_STATE, "the gradient set belongs to another HIP device than the current one");
  hipLaunchKernelGGL(gradient_squares, dim3(set->blocks), dim3(kThreads), 0, s, set->d_chunks, set->n_chunks, set->doubles,
                     partials);
  BN_HIP_CHECK(hipGetLastError());
  return BN_OK;
}

}  // namespace

extern "C" {

int bn_gradient_set_create(int32_t num_tensors, const int32_t* dtypes, const int64_t* sizes,
                           const void* const* gradients_dev, void* const* outputs_dev, bn_gradient_set** out_set) {
  if (!out_set) return fail(BN_ERR_INVALID, "out_set is null");
  *out_set = nullptr;
  if (num_tensors < 0) return fail(BN_ERR_INVALID, "negative number of tensors");
  if (num_tensors > 0 && (!dtypes || !sizes || !gradients_dev || !outputs_dev))
    return fail(BN_ERR_INVALID, "null argument");
  for (int32_t t = 0; t < num_tensors; ++t) {
    const size_t es = dtype_bytes(dtypes[t]);
    if (es == 0) return fail(BN_ERR_INVALID, "dtype must be BN_F32, BN_F64, BN_F16 or BN_BF16");
    if (sizes[t] < 0 || sizes[t] > ((int64_t)1 << 48)) return fail(BN_ERR_INVALID, "bad tensor size");
    if (sizes[t] == 0) continue;
    if (!gradients_dev[t] || !outputs_dev[t]) return fail(BN_ERR_INVALID, "null tensor address");
    if (reinterpret_cast<uintptr_t>(gradients_dev[t]) % es || reinterpret_cast<uintptr_t>(outputs_dev[t]) % es)
      return fail(BN_ERR_INVALID, "tensor address not aligned to its type");
  }
  bn_gradient_set* set = new (std::nothrow) bn_gradient_set();
  if (!set) return fail(BN_ERR_INVALID, "out of host memory");
  int rc;
  try {
    rc = build_set(num_tensors, dtypes, sizes, gradients_dev, outputs_dev, set);
  } catch (const std::bad_alloc&) {
    rc = fail(BN_ERR_INVALID, "out of host memory");
  }
  if (rc) {
    if (set->d_chunks) (void)hipFree(set->d_chunks);
    delete set;
    return rc;
  }
  *out_set = set;
  return BN_OK;
}

int bn_gradient_set_destroy(bn_gradient_set* set) {
  if (!set) return BN_OK;
  // the last reference to a set may go while some stream is being captured, which hipFree would end otherwise
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  (void)hipThreadExchangeStreamCaptureMode(&mode);
  int prev = 0;
  (void)hipGetDevice(&prev);
  (void)hipSetDevice(set->device);
  if (set->d_chunks) (void)hipFree(set->d_chunks);
  (void)hipSetDevice(prev);
  (void)hipThreadExchangeStreamCaptureMode(&mode);
  delete set;
  return BN_OK;
}

int64_t bn_gradient_set_workspace_bytes(const bn_gradient_set* set) {
  return set ? (int64_t)set->blocks * (set->doubles ? 3 : 1) * (int64_t)sizeof(double) : -1;
}

int bn_gradient_set_norm(bn_gradient_set* set, void* workspace_dev, double* norm_out_dev, void* stream) {
  if (!set || !workspace_dev || !norm_out_dev) return fail(BN_ERR_INVALID, "null argument");
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* partials = static_cast<double*>(workspace_dev);
  if (int rc = launch_squares(set, partials, s)) return rc;
  hipLaunchKernelGGL(gradient_norm_finish, dim3(1), dim3(kThreads), 0, s, partials, set->blocks, set->doubles,
                     norm_out_dev);
  BN_HIP_CHECK(hipGetLastError());
  return BN_OK;
}

int bn_gradient_set_clip(bn_gradient_set* set, double max_norm, void* workspace_dev, double* norm_out_dev,
                         void* stream) {
  if (!set || !workspace_dev || !norm_out_dev) return fail(BN_ERR_INVALID, "null argument");
  if (!(max_norm > 0.0) || std::isinf(max_norm)) return fail(BN_ERR_INVALID, "max_norm must be positive and finite");
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* partials = static_cast<double*>(workspace_dev);
  if (int rc = launch_squares(set, partials, s)) return rc;
  if (2 * set->bytes > kCacheBytes)
    hipLaunchKernelGGL(gradient_scale<true>, dim3(set->blocks), dim3(kThreads), 0, s, set->d_chunks, set->n_chunks,
                       partials, set->blocks, set->doubles, max_norm, norm_out_dev);
  else
    hipLaunchKernelGGL(gradient_scale<false>, dim3(set->blocks), dim3(kThreads), 0, s, set->d_chunks, set->n_chunks,
                       partials, set->blocks, set->doubles, max_norm, norm_out_dev);
  BN_HIP_CHECK(hipGetLastError());
  return BN_OK;
}

}  // extern "C"
