// Linear layers over 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k], W = scale * code + bias
// per group of 64 inputs; gated: silu(x G^T) * (x U^T); and both per expert over rows sorted
// by expert.
#include "am_internal.h"
#include "am_linear.cuh"

namespace am {

// ---------------------------------------------------------------- weight parameters
// One warp per weight row: the row's exponent e is the smallest with every |scale| * 2^(24-e)
// and |bias| * 2^-e at most 2^15 (fp16 holds up to 65504), then the groups' pairs are scaled by
// powers of two and stored as fp16.
__device__ __forceinline__ int exponent_above(float v) {  // least e with v < 2^e (v > 0, finite)
  int e;
  frexpf(v, &e);
  return e;
}

template <bool BF16>
__global__ void __launch_bounds__(128) weight_pack_kernel(const uint16_t* scales, const uint16_t* biases,
                                                          int64_t rows, int groups, uint32_t* params,
                                                          float* row_scale) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const uint16_t* s = scales + row * groups;
  const uint16_t* b = biases + row * groups;
  float ms = 0.0f, mb = 0.0f;
  for (int g = lane; g < groups; g += 32) {
    ms = fmaxf(ms, fabsf(h2f<BF16>(s[g])));
    mb = fmaxf(mb, fabsf(h2f<BF16>(b[g])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ms = fmaxf(ms, __shfl_xor_sync(0xffffffffu, ms, o));
    mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, o));
  }
  constexpr float kMax = 3.0e38f;  // an infinite scale or bias stays infinite in the params
  int e = -126;
  if (ms > 0.0f) e = max(e, exponent_above(fminf(ms, kMax)) + 24 - 15);
  if (mb > 0.0f) e = max(e, exponent_above(fminf(mb, kMax)) - 15);
  if (ms == 0.0f && mb == 0.0f) e = 0;
  e = min(e, 127);
  if (lane == 0) row_scale[row] = ldexpf(1.0f, e);
  const int pstride = (groups + 3) & ~3;
  for (int g = lane; g < pstride; g += 32) {
    uint32_t v = 0;
    if (g < groups) v = pack_half2(ldexpf(h2f<BF16>(s[g]), 24 - e), ldexpf(h2f<BF16>(b[g]), -e));
    params[row * pstride + g] = v;
  }
}

cudaError_t launch_weight_pack(const void* scales, const void* biases, bool bf16, int64_t rows, int groups,
                               uint32_t* params, float* row_scale, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
  const auto* s = static_cast<const uint16_t*>(scales);
  const auto* b = static_cast<const uint16_t*>(biases);
  if (bf16)
    weight_pack_kernel<true><<<grid, 128, 0, stream>>>(s, b, rows, groups, params, row_scale);
  else
    weight_pack_kernel<false><<<grid, 128, 0, stream>>>(s, b, rows, groups, params, row_scale);
  return cudaGetLastError();
}

// ---------------------------------------------------------------- plain kernel
// One warp per output column and eight rows: lanes stride over the groups' words, fp32 products.
constexpr int kPlainRows = 8;

__global__ void __launch_bounds__(256) linear_plain_kernel(const LinearParams p) {
  const int e = blockIdx.z;
  int lo, hi;
  expert_range(p, e, lo, hi);
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (n >= p.n_out) return;
  const int64_t wrow = (int64_t)e * p.n_out + n;
  for (int r0 = lo + blockIdx.y * kPlainRows; r0 < hi; r0 += gridDim.y * kPlainRows) {
    const uint16_t* xr[kPlainRows];
#pragma unroll
    for (int m = 0; m < kPlainRows; ++m) {
      const int src = r0 + m < hi ? source_row(p, r0 + m) : -1;
      xr[m] = src >= 0 ? p.x + (int64_t)src * p.x_stride : nullptr;
    }
    float acc[2][kPlainRows] = {};
    for (int which = 0; which < (p.codes[1] != nullptr ? 2 : 1); ++which) {
      const uint32_t* wc = p.codes[which] + wrow * (p.n_in / 8);
      for (int w = lane; w < p.n_in / 8; w += 32) {
        const __half2 sb = *reinterpret_cast<const __half2*>(&p.params[which][wrow * p.pstride + w / 8]);
        const float s = __low2float(sb) * 5.9604644775390625e-8f, b = __high2float(sb);  // 2^-24
        const uint32_t code = wc[w];
        float wv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) wv[i] = fmaf(static_cast<float>((code >> (4 * i)) & 15u), s, b);
#pragma unroll
        for (int m = 0; m < kPlainRows; ++m) {
          if (xr[m] == nullptr) continue;
          const uint4 xv = *reinterpret_cast<const uint4*>(xr[m] + w * 8);
          const uint32_t u[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            acc[which][m] = fmaf(h2f_rt(static_cast<uint16_t>(u[i / 2] >> (16 * (i & 1))), p.bf16), wv[i],
                                 acc[which][m]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < kPlainRows; ++m) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        acc[0][m] += __shfl_xor_sync(0xffffffffu, acc[0][m], o);
        acc[1][m] += __shfl_xor_sync(0xffffffffu, acc[1][m], o);
      }
      if (lane == 0 && r0 + m < hi) {
        float y = acc[0][m] * p.row_scale[0][wrow];
        if (p.codes[1] != nullptr) y = silu_mul(y, acc[1][m] * p.row_scale[1][wrow]);
        store_out(p.out, (int64_t)(r0 + m) * p.out_stride + n, y, p.bf16 ? AM_DTYPE_BF16 : AM_DTYPE_F16);
      }
    }
  }
}

cudaError_t launch_linear(const LinearParams& p, cudaStream_t stream) {
  if (p.rows == 0 || p.n_out == 0) return cudaSuccess;
  const int row_blocks = min((p.rows + kPlainRows - 1) / kPlainRows, 1024);
  dim3 grid((p.n_out + 7) / 8, p.offsets != nullptr ? min(row_blocks, 64) : row_blocks, p.experts);
  linear_plain_kernel<<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace am
