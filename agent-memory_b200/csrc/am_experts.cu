// Routing of tokens to experts (top-k, softmax weights, stable counting sort) and the weighted
// sum of the experts' rows.
#include "am_internal.h"
#include "am_linear.cuh"

namespace am {

// ---------------------------------------------------------------- top-k of one token (a warp)
// Lane i holds logits i, i + 32, ...  (as ordered integers); each round takes the largest, the
// lower index first.  NaN counts as -inf.
constexpr int kMaxExperts = 1024, kMaxTopK = 32;

__device__ __forceinline__ float load_logit(const RouteParams& p, int64_t i) {
  const float v = p.dtype == AM_DTYPE_F32 ? static_cast<const float*>(p.logits)[i]
                                          : h2f_rt(static_cast<const uint16_t*>(p.logits)[i],
                                                   p.dtype == AM_DTYPE_BF16);
  return v != v ? -INFINITY : v;
}

// exp(v - top) where equal infinities count as equal logits
__device__ __forceinline__ float weight_of(float v, float top) {
  return top == -INFINITY ? 0.0f : (v == top ? 1.0f : expf(v - top));
}

// After this, lane j < top_k holds the j-th chosen expert and its weight.
template <int PER>
__device__ __forceinline__ void route_token(const RouteParams& p, int t, int lane, int& my_e, float& my_w) {
  float v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    v[i] = e < p.n_experts ? load_logit(p, (int64_t)t * p.stride + e) : -INFINITY;
  }
  uint32_t taken = 0;
  float top = 0.0f, my_v = -INFINITY, sum = 0.0f;
  my_e = 0;
  for (int j = 0; j < p.top_k; ++j) {
    float best = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 32 + lane;
      if (e < p.n_experts && !((taken >> i) & 1) && (at == 0x7fffffff || v[i] > best)) {
        best = v[i];
        at = e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ob = __shfl_xor_sync(0xffffffffu, best, o);
      const int oa = __shfl_xor_sync(0xffffffffu, at, o);
      if (oa != 0x7fffffff && (at == 0x7fffffff || ob > best || (ob == best && oa < at))) {
        best = ob;
        at = oa;
      }
    }
    if (j == 0) top = best;
    if ((at & 31) == lane) taken |= 1u << (at >> 5);
    if (j == lane) {
      my_e = at;
      my_v = best;
    }
    if (p.normalize) sum += weight_of(best, top);
  }
  if (!p.normalize) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * 32 + lane < p.n_experts) sum += weight_of(v[i], top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  my_w = sum > 0.0f ? weight_of(my_v, top) / sum : 0.0f;
}

// One CTA: top-k of every token, then the counting sort by one thread per expert.
__global__ void __launch_bounds__(1024) route_plain_kernel(const RouteParams p) {
  __shared__ int32_t start[kMaxExperts + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int t = warp; t < p.tokens; t += 32) {
    int e;
    float w;
    route_token<32>(p, t, lane, e, w);
    if (lane < p.top_k) {
      p.experts[(int64_t)t * p.top_k + lane] = e;
      p.weights[(int64_t)t * p.top_k + lane] = w;
    }
  }
  __syncthreads();
  const int pairs = p.tokens * p.top_k;
  const int me = threadIdx.x;
  int count = 0;
  if (me < p.n_experts)
    for (int i = 0; i < pairs; ++i) count += p.experts[i] == me;
  if (me < p.n_experts) start[me + 1] = count;
  __syncthreads();
  if (me == 0) {
    start[0] = 0;
    for (int e = 0; e < p.n_experts; ++e) start[e + 1] += start[e];
  }
  __syncthreads();
  if (me < p.n_experts) {
    int at = start[me];
    for (int i = 0; i < pairs; ++i)
      if (p.experts[i] == me) {
        p.order[at] = i;
        p.positions[i] = at++;
      }
  }
  for (int e = me; e <= p.n_experts; e += 1024) p.offsets[e] = start[e];
}

cudaError_t launch_route(const RouteParams& p, cudaStream_t stream) {
  route_plain_kernel<<<1, 1024, 0, stream>>>(p);
  return cudaGetLastError();
}

// ---------------------------------------------------------------- combine
__global__ void __launch_bounds__(256) combine_plain_kernel(const CombineParams p) {
  const int t = blockIdx.x;
  for (int c = blockIdx.y * 256 + threadIdx.x; c < p.width; c += gridDim.y * 256) {
    float acc = p.residual != nullptr ? h2f_rt(p.residual[(int64_t)t * p.residual_stride + c], p.bf16) : 0.0f;
    float sum = 0.0f;
    for (int j = 0; j < p.top_k; ++j) {
      const int at = p.positions[(int64_t)t * p.top_k + j];
      if (at < 0 || at >= p.y_rows) {
        flag_status(p.status, AM_STATUS_BAD_POSITION);
        continue;
      }
      sum = fmaf(p.weights[(int64_t)t * p.top_k + j], h2f_rt(p.y[(int64_t)at * p.y_stride + c], p.bf16), sum);
    }
    store_out(p.out, (int64_t)t * p.out_stride + c, acc + sum, p.bf16 ? AM_DTYPE_BF16 : AM_DTYPE_F16);
  }
}

cudaError_t launch_combine(const CombineParams& p, cudaStream_t stream) {
  combine_plain_kernel<<<dim3(p.tokens, min((p.width + 255) / 256, 64)), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace am
