// bn_draw_states of include/bn_hip.h: argument checks and dispatch over the logits' types
// (kernels_draw.h, one translation unit per type).
#include "../../include/bn_hip.h"

#include <algorithm>
#include <cmath>
#include <string>

#include "error.h"
#include "kernels_draw.h"

namespace {

using namespace bn_draw;
using bn::fail;

#define BN_HIP_CHECK(expr)                                                            \
  do {                                                                                \
    hipError_t err__ = (expr);                                                        \
    if (err__ != hipSuccess)                                                          \
      return fail(BN_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(err__));  \
  } while (0)

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

// Workspace of long rows: block sums, row states and piece keys of all rows.
int64_t blocks_per_row(int64_t num_states) { return num_states <= kShortStates ? 0 : (num_states + kBlock - 1) / kBlock; }
int64_t pieces_per_row(int64_t num_states) {
  const int64_t piece = piece_states(num_states);
  return num_states <= kShortStates ? 0 : (num_states + piece - 1) / piece;
}

}  // namespace

extern "C" {

int64_t bn_draw_states_workspace_bytes(int dtype, int64_t rows, int64_t num_states) {
  if (dtype_bytes(dtype) == 0 || rows < 0 || rows > (int64_t)1 << 40 || num_states < 1 || num_states > kMaxStates) return -1;
  const int64_t key_bytes = dtype == BN_F64 ? 8 : 4;
  const int64_t blocks = blocks_per_row(num_states);
  if (blocks == 0) return 0;
  return rows * ((blocks + 2) * (int64_t)sizeof(double) + (int64_t)sizeof(RowState) +
                 (rows_are_shared(rows, num_states) ? (int64_t)sizeof(SharedRow) : 0) + pieces_per_row(num_states) * key_bytes);
}

int bn_draw_states(int dtype, const void* logits_dev, int64_t rows, int64_t num_states, int64_t row_stride,
                   const int64_t* row_states_dev, int uniform_dtype, const void* uniforms_dev,
                   const bn_draw_filters* filters, void* workspace_dev, int32_t* out_dev, void* stream) {
  if (!filters) return fail(BN_ERR_INVALID, "filters is null");
  Draws a{};
  a.logits = logits_dev;
  a.rows = rows;
  a.width = num_states;
  a.stride = row_stride;
  a.counts = row_states_dev;
  a.uniforms = uniforms_dev;
  a.uniform_dtype = uniform_dtype;
  a.filters = *filters;
  a.out = out_dev;
  if (int rc = check_draws(dtype, a)) return rc;
  if (uniform_dtype != BN_F32 && uniform_dtype != BN_F64)
    return fail(BN_ERR_INVALID, "uniform_dtype must be BN_F32 or BN_F64");
  if (rows == 0) return BN_OK;
  a.pieces_per_row = pieces_per_row(num_states);
  if (!logits_dev || !uniforms_dev || !out_dev || (a.pieces_per_row > 0 && !workspace_dev))
    return fail(BN_ERR_INVALID, "null argument");
  if (reinterpret_cast<uintptr_t>(logits_dev) % dtype_bytes(dtype))
    return fail(BN_ERR_INVALID, "row address not aligned to its type");
  if (reinterpret_cast<uintptr_t>(workspace_dev) % 8) return fail(BN_ERR_INVALID, "workspace not aligned to 8 bytes");
  if (a.pieces_per_row > 0) {
    a.sums_per_row = blocks_per_row(num_states) + 2;
    a.block_sums = static_cast<double*>(workspace_dev);
    a.row_states = reinterpret_cast<RowState*>(a.block_sums + rows * a.sums_per_row);
    void* rest = a.row_states + rows;
    if (rows_are_shared(rows, num_states)) {
      a.shared = static_cast<SharedRow*>(rest);
      rest = a.shared + rows;
    }
    a.piece_keys = rest;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case BN_F32: BN_HIP_CHECK(launch_f32(a, s)); break;
    case BN_F64: BN_HIP_CHECK(launch_f64(a, s)); break;
    case BN_F16: BN_HIP_CHECK(launch_f16(a, s)); break;
    default: BN_HIP_CHECK(launch_bf16(a, s)); break;
  }
  return BN_OK;
}

}  // extern "C"
