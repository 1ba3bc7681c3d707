// Routing of tokens to experts (top-k, softmax weights, stable counting sort) and the weighted
// sum of the experts' rows.
#include <algorithm>

#include "am_internal.h"
#include "am_linear.cuh"

namespace am {

// Launches with programmatic stream serialization (the kernels wait in griddep_wait before they
// touch memory) and, where cluster > 1, thread-block clusters of that size.
template <typename K, typename P>
static cudaError_t launch_chained(K kfn, const P& p, dim3 grid, int threads, int smem, int cluster,
                                  cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kfn, p);
}

// ---------------------------------------------------------------- routing
// 1. Top-k by a warp a token: each round takes the largest logit (as an ordered integer) and the
//    lowest index that has it, two warp reductions.  NaN counts as -inf.
// 2. A stable counting sort by expert of the (token, slot) pairs in one cluster of up to 8 CTAs: a
//    warp walks its contiguous part 32 pairs at a time (match_any ranks equal experts among the
//    lanes) with counters per (warp, expert); the counters' prefix over warps, CTAs (distributed
//    shared memory) and experts gives the places.
// Up to 16 tokens one CTA of 8 warps does both; more go through a top-k launch over all SMs first (16
// tokens of 64 experts: 5.9 us and 6.6, 32: 8.5 and 6.7; 4096 of 32 experts: 22 and 10.2).  Both are
// bound by the launches and the barriers: 1 token of 64 experts takes 4.2 us, and the data of 4096
// are 0.8 MB.
__device__ __forceinline__ float load_logit(const RouteParams& p, int64_t i) {
  const float v = p.dtype == AM_DTYPE_F32 ? static_cast<const float*>(p.logits)[i]
                                          : h2f_rt(static_cast<const uint16_t*>(p.logits)[i],
                                                   p.dtype == AM_DTYPE_BF16);
  return v != v ? -INFINITY : v + 0.0f;  // (-0 and 0 are equal: one key)
}

// Floats as unsigned integers in the same order (all above 0), and back.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// exp(v - top), where equal infinities count as equal logits.
__device__ __forceinline__ float weight_of(float v, float top) {
  return top == -INFINITY ? 0.0f : (v == top ? 1.0f : expf(v - top));
}

// A warp routes token t (PER * 32 >= n_experts); lane j writes slot j.
template <int PER>
__device__ __forceinline__ void route_token(const RouteParams& p, int t, int lane) {
  float v[PER];
  uint32_t key[PER];  // 0: taken, or no expert
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    v[i] = e < p.n_experts ? load_logit(p, (int64_t)t * p.stride + e) : -INFINITY;
    key[i] = e < p.n_experts ? ordered(v[i]) : 0u;
  }
  float top = 0.0f, sum = 0.0f, my_v = -INFINITY;
  int my_e = 0;
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(0xffffffffu, best);
    uint32_t at = 0xffffffffu;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (key[i] == best) at = i * 32 + lane;
    at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * 32 + lane == static_cast<int>(at)) key[i] = 0;
    const float bv = unordered(best);
    if (j == 0) top = bv;
    if (j == lane) {
      my_v = bv;
      my_e = static_cast<int>(at);
    }
    if (p.normalize) sum += weight_of(bv, top);
  }
  if (!p.normalize) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * 32 + lane < p.n_experts) sum += weight_of(v[i], top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (lane < p.top_k) {
    p.experts[(int64_t)t * p.top_k + lane] = my_e;
    p.weights[(int64_t)t * p.top_k + lane] = sum > 0.0f ? weight_of(my_v, top) / sum : 0.0f;
  }
}

template <int PER>
__global__ void __launch_bounds__(256) route_topk_kernel(const __grid_constant__ RouteParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t < p.tokens) route_token<PER>(p, t, threadIdx.x & 31);
}

constexpr int kRouteHeld = 4096;  // pairs of a CTA whose expert and rank stay in shared memory

// Shared memory: counters [warps][n_experts], totals and first places [n_experts], a word a warp,
// then the held pairs' expert and rank.  PER > 0: the top-k too, by a CTA of 256 threads.
template <int PER>
__global__ void __launch_bounds__(PER > 0 ? 256 : 1024) route_sort_kernel(const __grid_constant__ RouteParams p) {
  extern __shared__ int32_t counts[];
  const int E = p.n_experts, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int threads = blockDim.x, warps = threads >> 5;
  int32_t* totals = counts + warps * E;
  int32_t* first = totals + E;
  int32_t* carry = first + E;
  int32_t* held_e = carry + 32;
  const int rank = blockIdx.x, ctas = gridDim.x;  // one cluster
  const int t0 = static_cast<int>((int64_t)p.tokens * rank / ctas);
  const int t1 = static_cast<int>((int64_t)p.tokens * (rank + 1) / ctas);
  const int i0 = t0 * p.top_k, n = (t1 - t0) * p.top_k;
  const bool held = n <= kRouteHeld;
  int32_t* held_r = held_e + (held ? n : 0);
  for (int i = tid; i < warps * E; i += threads) counts[i] = 0;
  griddep_launch_dependents();
  griddep_wait();
  if constexpr (PER > 0) {
    for (int t = t0 + warp; t < t1; t += warps) route_token<PER>(p, t, lane);
  }
  __syncthreads();

  // places among the warp's pairs of the same expert, and the warp's counts
  const int a = static_cast<int>((int64_t)n * warp / warps), b = static_cast<int>((int64_t)n * (warp + 1) / warps);
  int32_t* mine = counts + warp * E;
  for (int i = a; i < b; i += 32) {
    const bool live = i + lane < b;
    const int e = live ? p.experts[i0 + i + lane] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (live) {
      const int r = mine[e] + before;
      if (held) {
        held_e[i + lane] = e;
        held_r[i + lane] = r;
      } else {
        p.positions[i0 + i + lane] = r;
      }
    }
    __syncwarp();
    if (live && before == 0) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  // exclusive prefix over the warps (a lane a warp); the CTA's totals
  for (int e = warp; e < E; e += warps) {
    const int c = lane < warps ? counts[lane * E + e] : 0;
    int incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane < warps) counts[lane * E + e] = incl - c;
    if (lane == 31) totals[e] = incl;
  }
  if (ctas > 1)
    cluster_sync_all();
  else
    __syncthreads();
  // first place of every expert (scan over the experts, a chunk of `threads` at a time) plus what
  // the CTAs before this one hold of it
  int base = 0;
  for (int e0 = 0; e0 < E; e0 += threads) {
    const int e = e0 + tid;
    int all = 0, before = 0;
    if (e < E) {
      if (ctas > 1) {
        const uint32_t addr = smem_u32(&totals[e]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int v = c < ctas ? __float_as_int(ld_dsmem_f32(dsmem_addr(addr, c))) : 0;
          before += c < rank ? v : 0;
          all += v;
        }
      } else {
        all = totals[e];
      }
    }
    int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) carry[warp] = incl;
    __syncthreads();
    const int cw = lane < warps ? carry[lane] : 0;
    const int start = base + __reduce_add_sync(0xffffffffu, lane < warp ? cw : 0) + incl - all;
    base += __reduce_add_sync(0xffffffffu, cw);
    if (e < E) {
      if (rank == 0) p.offsets[e] = start;
      first[e] = start + before;
    }
    __syncthreads();
  }
  if (rank == 0 && tid == 0) p.offsets[E] = base;
  for (int i = a + lane; i < b; i += 32) {
    const int e = held ? held_e[i] : p.experts[i0 + i];
    const int pos = (held ? held_r[i] : p.positions[i0 + i]) + mine[e] + first[e];
    p.positions[i0 + i] = pos;
    p.order[pos] = i0 + i;
  }
  if (ctas > 1) cluster_sync_all();  // peers have read this CTA's totals
}

template <int PER>
static cudaError_t launch_sort(const RouteParams& p, int ctas, int threads, cudaStream_t stream) {
  const int held = static_cast<int>(std::min<int64_t>(((int64_t)p.tokens + ctas - 1) / ctas * p.top_k, kRouteHeld));
  const int smem = (threads / 32 * p.n_experts + 2 * p.n_experts + 32 + 2 * held) * 4;
  auto kfn = route_sort_kernel<PER>;
  if (smem > 48 * 1024) {
    // once per device, to what the largest call needs: host threads share the attribute, and one that
    // set it to its own call's size could lower it between another's setting and launch
    constexpr int kLargest = (34 * 1024 + 32 + 2 * kRouteHeld) * 4;  // 1024 experts, 32 warps
    static unsigned long long done = 0;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (!bit || !(__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) {
      err = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, kLargest);
      if (err != cudaSuccess) return err;
      if (bit) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
    }
  }
  return launch_chained(kfn, p, dim3(ctas), threads, smem, ctas, stream);
}

template <int PER>
static cudaError_t launch_route_t(const RouteParams& p, cudaStream_t stream) {
  if (p.tokens <= 16) return launch_sort<PER>(p, 1, 256, stream);
  const cudaError_t err =
      launch_chained(route_topk_kernel<PER>, p, dim3((p.tokens - 1) / 8 + 1), 256, 0, 1, stream);
  if (err != cudaSuccess) return err;
  int ctas = 1;  // a CTA for every 1024 pairs: one pair a thread
  while (ctas < 8 && (int64_t)p.tokens * p.top_k > ctas * 1024) ctas *= 2;
  return launch_sort<0>(p, ctas, 1024, stream);
}

cudaError_t launch_route(const RouteParams& p, cudaStream_t stream) {
  if (p.n_experts <= 32) return launch_route_t<1>(p, stream);
  if (p.n_experts <= 64) return launch_route_t<2>(p, stream);
  if (p.n_experts <= 128) return launch_route_t<4>(p, stream);
  if (p.n_experts <= 256) return launch_route_t<8>(p, stream);
  return launch_route_t<32>(p, stream);
}

// ---------------------------------------------------------------- combine
// HBM-bound.  A CTA takes a part of a token's row, a thread VEC columns of it, with the loads of four rows at
// once; the experts' rows are read here for the last time and leave the caches first.  4096 tokens of
// 4 rows of 2880: 21 us, 6.7 TB/s (without the hint 24; with columns dealt out over whole CTAs, a
// division a thread, 29).
template <int VEC>
struct Columns;
template <>
struct Columns<8> {
  using T = uint4;
};
template <>
struct Columns<1> {
  using T = uint16_t;
};

template <int VEC>
__device__ __forceinline__ void add_columns(float (&acc)[VEC], typename Columns<VEC>::T u, float w, bool bf16) {
  if constexpr (VEC == 1) {
    acc[0] = fmaf(w, h2f_rt(u, bf16), acc[0]);
  } else {
    const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, h2f_rt(static_cast<uint16_t>(q[i >> 1] >> (16 * (i & 1))), bf16), acc[i]);
  }
}

template <int VEC>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ CombineParams p) {
  using T = typename Columns<VEC>::T;
  griddep_launch_dependents();
  griddep_wait();
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  if (c >= p.width) return;
  for (uint32_t t = blockIdx.x; t < static_cast<uint32_t>(p.tokens); t += gridDim.x) {  // (up to 2^31 - 1)
    const float* w = p.weights + (int64_t)t * p.top_k;
    const int32_t* at = p.positions + (int64_t)t * p.top_k;
    T res{};
    if (p.residual != nullptr) res = *reinterpret_cast<const T*>(p.residual + (int64_t)t * p.residual_stride + c);
    float acc[VEC] = {};
    for (int j0 = 0; j0 < p.top_k; j0 += 4) {
      T y[4];
      float wj[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = T{};
        wj[j] = 0.0f;
        if (j0 + j < p.top_k) {
          const int row = at[j0 + j];
          if (row >= 0 && row < p.y_rows) {
            wj[j] = w[j0 + j];
            y[j] = __ldlu(reinterpret_cast<const T*>(p.y + (int64_t)row * p.y_stride + c));
          } else {
            flag_status(p.status, AM_STATUS_BAD_POSITION);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) add_columns<VEC>(acc, y[j], wj[j], p.bf16);
    }
    if (p.residual != nullptr) add_columns<VEC>(acc, res, 1.0f, p.bf16);
    uint16_t* dst = p.out + (int64_t)t * p.out_stride + c;
    if constexpr (VEC == 1) {
      dst[0] = p.bf16 ? f2h<true>(acc[0]) : f2h<false>(acc[0]);
    } else {
      uint32_t o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        o[k] = static_cast<uint32_t>(p.bf16 ? f2h<true>(acc[2 * k]) : f2h<false>(acc[2 * k])) |
               static_cast<uint32_t>(p.bf16 ? f2h<true>(acc[2 * k + 1]) : f2h<false>(acc[2 * k + 1])) << 16;
      *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

cudaError_t launch_combine(const CombineParams& p, cudaStream_t stream) {
  auto wide = [](const void* ptr, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && stride % 8 == 0;
  };
  // 16-byte columns where every row allows them (8x fewer, 8x larger accesses than one by one)
  const bool vec = p.width % 8 == 0 && wide(p.y, p.y_stride) && wide(p.out, p.out_stride) &&
                   (p.residual == nullptr || wide(p.residual, p.residual_stride));
  // CTAs of equal parts of a token's row, 256 columns or vectors at most
  const int cols = vec ? p.width / 8 : p.width, parts = (cols - 1) / 256 + 1;
  if (parts > 65535) return cudaErrorNotSupported;
  const int threads = ((cols + parts - 1) / parts + 31) & ~31;
  const dim3 grid(std::min(p.tokens, 1 << 20), parts);
  return vec ? launch_chained(combine_kernel<8>, p, grid, threads, 0, 1, stream)
             : launch_chained(combine_kernel<1>, p, grid, threads, 0, 1, stream);
}

}  // namespace am
