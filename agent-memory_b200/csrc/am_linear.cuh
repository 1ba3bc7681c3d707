// Launch parameters and device helpers of the 4-bit linear layers and the expert routing.
#pragma once

#include "am_common.cuh"

namespace am {

// y = x W^T over 4-bit weights, plain or gated (up != null), for one matrix or per expert.
struct LinearParams {
  const uint32_t* codes[2];   // [0] the matrix (gate), [1] its partner (up) or null
  const uint32_t* params[2];  // [rows of weights][pstride]: half2 (scale * 2^(24-e), bias * 2^-e)
  const float* row_scale[2];  // [rows of weights]: 2^e
  int32_t n_out, n_in, groups, pstride;
  int32_t experts;
  int32_t bf16;               // activations and outputs: bf16 (1) or fp16 (0)
  const uint16_t* x;
  int64_t x_stride;
  int32_t x_rows;
  const int32_t* offsets;     // [experts + 1] or null (one matrix, rows [0, rows))
  const int32_t* order;       // [rows] or null: output row r comes from x row order[r] / top_k
  int32_t top_k;
  int32_t rows;               // output rows
  uint16_t* out;
  int64_t out_stride;
  int32_t* status;
};

struct RouteParams {
  const void* logits;
  int32_t dtype;
  int64_t stride;
  int32_t tokens, n_experts, top_k, normalize;
  int32_t* experts;
  float* weights;
  int32_t* offsets;
  int32_t* order;
  int32_t* positions;
  int32_t* ws;
};

struct CombineParams {
  const uint16_t* y;
  const uint16_t* residual;
  uint16_t* out;
  int64_t y_stride, residual_stride, out_stride;
  const float* weights;
  const int32_t* positions;
  int32_t y_rows, tokens, top_k, width, bf16;
  int32_t* status;
};

// Rows [lo, hi) of expert e, clamped to [0, rows).
__device__ __forceinline__ void expert_range(const LinearParams& p, int e, int& lo, int& hi) {
  if (p.offsets == nullptr) {
    lo = 0;
    hi = p.rows;
  } else {
    lo = min(max(p.offsets[e], 0), p.rows);
    hi = min(max(p.offsets[e + 1], lo), p.rows);
  }
}

// The x row that output row r is made from; -1 (and the status bit) for a bad order entry.
__device__ __forceinline__ int source_row(const LinearParams& p, int r) {
  if (p.order == nullptr) return r;
  const int pair = p.order[r];
  const int t = pair / p.top_k;
  if (pair < 0 || t >= p.x_rows) {
    flag_status(p.status, AM_STATUS_BAD_POSITION);
    return -1;
  }
  return t;
}

__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

}  // namespace am
