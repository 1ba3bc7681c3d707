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
// One cluster of up to 8 CTAs, each with a contiguous part of the tokens, in one launch: a token's
// work is a few hundred cycles of shuffles, so the launch and the barriers cost more than the data
// (4096 tokens of 32 experts are 0.5 MB), and a second launch more than the SMs left idle.
//
// 1. Top-k by a team of TEAM lanes a token (TEAM * PER >= n_experts): each round takes the maximum
//    of 64-bit keys (the logit as an ordered integer, then the complemented index: ties go to
//    the lower one) over the team.  NaN counts as -inf.
// 2. A stable counting sort by expert of the (token, slot) pairs: a warp walks its contiguous part
//    32 pairs at a time (match_any ranks equal experts among the lanes) with counters per
//    (warp, expert); the counters' prefix over warps, CTAs (distributed shared memory) and
//    experts gives the places.
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

// Routes token t (t < 0: only takes part in the shuffles).  Slot j is written by lane j % TEAM.
template <int TEAM, int PER>
__device__ __forceinline__ void route_token(const RouteParams& p, int t, int lane) {
  constexpr int SLOTS = 32 / TEAM;  // top_k <= 32
  const int l = lane & (TEAM - 1);
  float v[PER];
  uint64_t key[PER];  // 0: taken, or no expert
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * TEAM + l;
    v[i] = t >= 0 && e < p.n_experts ? load_logit(p, (int64_t)t * p.stride + e) : -INFINITY;
    key[i] = e < p.n_experts ? (static_cast<uint64_t>(ordered(v[i])) << 32) | static_cast<uint32_t>(~e) : 0;
  }
  float top = 0.0f, sum = 0.0f, mine[SLOTS];
  int mine_e[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    mine[s] = -INFINITY;
    mine_e[s] = 0;
  }
  for (int j = 0; j < p.top_k; ++j) {
    uint64_t best = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = key[i] > best ? key[i] : best;
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] == best) key[i] = 0;
    const float bv = unordered(static_cast<uint32_t>(best >> 32));
    if (j == 0) top = bv;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (j == s * TEAM + l) {
        mine[s] = bv;
        mine_e[s] = static_cast<int>(~static_cast<uint32_t>(best));
      }
    if (p.normalize) sum += weight_of(bv, top);
  }
  if (!p.normalize) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * TEAM + l < p.n_experts) sum += weight_of(v[i], top);
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int j = s * TEAM + l;
    if (t >= 0 && j < p.top_k) {
      p.experts[(int64_t)t * p.top_k + j] = mine_e[s];
      p.weights[(int64_t)t * p.top_k + j] = sum > 0.0f ? weight_of(mine[s], top) / sum : 0.0f;
    }
  }
}

// Shared memory: counters [warps][n_experts], this CTA's totals [n_experts], one word a warp.
template <int TEAM, int PER>
__global__ void __launch_bounds__(1024) route_kernel(const __grid_constant__ RouteParams p) {
  extern __shared__ int32_t counts[];
  const int E = p.n_experts, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int threads = blockDim.x, warps = threads >> 5;
  int32_t* totals = counts + warps * E;
  int32_t* carry = totals + E;
  const int rank = blockIdx.x, ctas = gridDim.x;  // one cluster
  const int t0 = static_cast<int>((int64_t)p.tokens * rank / ctas);
  const int t1 = static_cast<int>((int64_t)p.tokens * (rank + 1) / ctas);
  for (int i = tid; i < warps * E; i += threads) counts[i] = 0;
  griddep_launch_dependents();
  griddep_wait();

  constexpr int TEAMS = 32 / TEAM;  // of a warp
  for (int t = t0 + warp * TEAMS; t < t1; t += warps * TEAMS) {
    const int mine = t + lane / TEAM;
    route_token<TEAM, PER>(p, mine < t1 ? mine : -1, lane);
  }
  __syncthreads();

  // places among the warp's pairs of the same expert, and the warp's counts
  const int i0 = t0 * p.top_k, n = (t1 - t0) * p.top_k;
  const int a = i0 + static_cast<int>((int64_t)n * warp / warps), b = i0 + static_cast<int>((int64_t)n * (warp + 1) / warps);
  int32_t* mine = counts + warp * E;
  for (int i = a; i < b; i += 32) {
    const bool live = i + lane < b;
    const int e = live ? p.experts[i + lane] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (live) p.positions[i + lane] = mine[e] + before;
    __syncwarp();
    if (live && before == 0) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  // exclusive prefix over the warps; the CTA's totals
  for (int e = tid; e < E; e += threads) {
    int run = 0;
    for (int w = 0; w < warps; ++w) {
      const int c = counts[w * E + e];
      counts[w * E + e] = run;
      run += c;
    }
    totals[e] = run;
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
      const uint32_t addr = smem_u32(&totals[e]);
      for (int c = 0; c < ctas; ++c) {
        const int v = ctas > 1 ? __float_as_int(ld_dsmem_f32(dsmem_addr(addr, c))) : totals[e];
        before += c < rank ? v : 0;
        all += v;
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
    int pre = 0, sum = 0;
    for (int w = 0; w < warps; ++w) {
      pre += w < warp ? carry[w] : 0;
      sum += carry[w];
    }
    const int start = base + pre + incl - all;
    base += sum;
    if (e < E) {
      if (rank == 0) p.offsets[e] = start;
      for (int w = 0; w < warps; ++w) counts[w * E + e] += start + before;
    }
    __syncthreads();
  }
  if (rank == 0 && tid == 0) p.offsets[E] = base;
  for (int i = a + lane; i < b; i += 32) {
    const int pos = p.positions[i] + mine[p.experts[i]];
    p.positions[i] = pos;
    p.order[pos] = i;
  }
  if (ctas > 1) cluster_sync_all();  // peers have read this CTA's totals
}

template <int TEAM, int PER>
static cudaError_t launch_route_t(const RouteParams& p, cudaStream_t stream) {
  // a CTA for every 64 tokens; few tokens in a small CTA, whose barriers are cheaper
  int ctas = 1;
  while (ctas < 8 && p.tokens > ctas * 64) ctas *= 2;
  const int threads = p.tokens * TEAM <= 256 ? 256 : 1024;
  const int smem = (threads / 32 * p.n_experts + p.n_experts + 32) * 4;
  auto kfn = route_kernel<TEAM, PER>;
  if (smem > 48 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return err;
  }
  return launch_chained(kfn, p, dim3(ctas), threads, smem, ctas, stream);
}

cudaError_t launch_route(const RouteParams& p, cudaStream_t stream) {
  if (p.n_experts <= 32) return launch_route_t<8, 4>(p, stream);
  if (p.n_experts <= 64) return launch_route_t<16, 4>(p, stream);
  if (p.n_experts <= 128) return launch_route_t<32, 4>(p, stream);
  if (p.n_experts <= 256) return launch_route_t<32, 8>(p, stream);
  return launch_route_t<32, 32>(p, stream);
}

// ---------------------------------------------------------------- combine
// HBM-bound: a thread sums VEC columns of a token, its rows' loads issued four at a time.
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
  const int cols = p.width / VEC;
  const int64_t all = (int64_t)p.tokens * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int t = static_cast<int>(i / cols), c = static_cast<int>(i - (int64_t)t * cols) * VEC;
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
            y[j] = *reinterpret_cast<const T*>(p.y + (int64_t)row * p.y_stride + c);
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
  const int64_t all = (int64_t)p.tokens * (vec ? p.width / 8 : p.width);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((all + 255) / 256, 1 << 20));
  return vec ? launch_chained(combine_kernel<8>, p, dim3(grid), 256, 0, 1, stream)
             : launch_chained(combine_kernel<1>, p, dim3(grid), 256, 0, 1, stream);
}

}  // namespace am
