// Linear layers over 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k], W = scale * code + bias
// per group of 64 inputs; gated: silu(x G^T) * (x U^T); and both per expert over rows sorted
// by expert.
#include <algorithm>

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

// ---------------------------------------------------------------- few tokens (HBM-bound)
// Up to 8 tokens of one matrix or expert: y^T = W x^T on mma.sync m16n8k16 with the weights as the A
// operand straight from their packed words.  tcgen05 would take the dequantized weights through
// TMEM; here a weight is used for at most 8 tokens and the kernel is bound by the bytes of the
// codes, so the operand that needs no staging wins.
//
// * Dequantization: one AND turns two nibbles of a word into fp16 subnormals code * 2^-24 (or
//   * 2^-20), one packed FMA with (scale * 2^24 or 2^20, bias) makes the two weights, rounded
//   once: 9 operations for 8 weights.  The row's exponent (am_q4_weight_pack) keeps scale * 2^24
//   inside fp16 and is undone on the fp32 result.
// * The inputs of a group of 64 are permuted over the MMA's k slots so that lane t of a quad owns
//   words 2t and 2t + 1 of its row.  The activations are staged in the same order, as fp16 under
//   a power of two per token (exact), in fragment order: one 16-byte load per two MMAs.
// * A CTA of 16 warps a SM.  wk of them split the inputs (each stages only its own slice of the
//   activations, so nothing waits for the whole CTA before the sums), the others take further
//   row tiles; with long inputs CK CTAs of a cluster split them again.  Every warp streams its
//   slices of the row tiles (16 rows x up to 4 groups a stage) through a private cp.async ring:
//   the warps of a SM keep 70 to 110 KB in flight, across tile and expert ends.
// * Partial sums meet in shared memory every few tiles, in a fixed order.
// * The work of all experts is one sequence of row tiles, cut evenly over the CTAs.
// * Before griddepcontrol.wait the CTA only asks L2 for its first codes (a prefetch reads
//   nothing, so it may run before the previous kernel is done).
constexpr int kFewWarps = 16;
constexpr int kFewTokens = 8;
constexpr int kFewStage = 16 * 128 + 16 * 16;  // codes and parameters of 16 rows x 4 groups

struct FewParams {
  LinearParams p;
  int32_t wk;       // warps along the inputs (1, 2, 4, 8 or 16)
  int32_t ck;       // CTAs of a cluster along the inputs
  int32_t tiles;    // positions of one item: row tiles / (16 / wk), rounded up
  int32_t batch;    // positions between two sums
  int32_t slice;    // groups of a warp's slice, at most
  int32_t x_stride; // staged bytes of a warp's activations
};

template <int MT, int D>
__global__ void __launch_bounds__(kFewWarps * 32, 1) linear_few_kernel(const __grid_constant__ FewParams f) {
  constexpr bool GATED = MT == 2;
  constexpr int STAGE = MT * kFewStage;
  const LinearParams& p = f.p;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int rank = f.ck > 1 ? static_cast<int>(blockIdx.x) % f.ck : 0;
  const int cluster = static_cast<int>(blockIdx.x) / f.ck, clusters = static_cast<int>(gridDim.x) / f.ck;
  const int wk = f.wk, wr_n = kFewWarps / wk;
  const int kslice = warp % wk, wr = warp / wk;
  uint8_t* ring = smem + warp * (D * STAGE);
  uint8_t* sx = smem + kFewWarps * D * STAGE + warp * f.x_stride;
  float* red = reinterpret_cast<float*>(smem + kFewWarps * (D * STAGE + f.x_stride));
  const int row_tiles = (p.n_out + 15) >> 4;
  // this warp's groups
  const int slices = wk * f.ck, slot = rank * wk + kslice;
  const int ga = p.groups * slot / slices, gb = p.groups * (slot + 1) / slices;
  const int stages = (gb - ga + 3) >> 2;  // of one row tile

  griddep_launch_dependents();
  if (p.offsets == nullptr) {  // L2 prefetch of the CTA's first tiles: a lane pair a row
    const int64_t pos0 = (int64_t)f.tiles * cluster / clusters;
    const int64_t n = (pos0 * wr_n + wr) * 16 + (lane >> 1);
    if (n < p.n_out) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const char* c = reinterpret_cast<const char*>(p.codes[i] + n * (p.n_in / 8));
        for (int g = ga + (lane & 1) * 4; g < gb; g += 8)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(c + g * 32));
      }
    }
  }
  griddep_wait();
  const int items = count_items<kFewTokens>(p);
  const int64_t total = (int64_t)items * f.tiles;
  const int64_t p0 = total * cluster / clusters, p1 = total * (cluster + 1) / clusters;

  // ---- load side: walks the positions [p0, p1) a few stages ahead of the sums.  A lane fetches 16
  // bytes of rows lane / 8 + 4 j of the tile and a parameter of rows lane / 4 + 8 j.
  int l_left = static_cast<int>(p1 - p0);
  int l_item = static_cast<int>(p0 / f.tiles);
  int l_pos = static_cast<int>(p0 - (int64_t)l_item * f.tiles);  // position in the item
  int l_stage = 0, l_buf = 0, l_e = 0;
  const int row_bytes = p.n_in / 2;
  const int64_t tile_bytes = (int64_t)wr_n * 16 * row_bytes, tile_params = (int64_t)wr_n * 16 * p.pstride;
  const uint8_t* l_codes = nullptr;   // this lane's first chunk of the tile, matrix 0
  const uint32_t* l_params = nullptr;
  const int64_t codes_diff = GATED ? reinterpret_cast<const uint8_t*>(p.codes[1]) - reinterpret_cast<const uint8_t*>(p.codes[0]) : 0;
  const int64_t params_diff = GATED ? p.params[1] - p.params[0] : 0;
  const uint32_t l_dst = smem_u32(ring) + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);  // row + 4: chunk ^ 4
  const uint32_t l_pdst = smem_u32(ring) + 2048 + (lane >> 2) * 16 + (lane & 3) * 4;
  auto l_open = [&]() {  // pointers of position l_pos of item l_item
    int lo, hi;
    l_e = find_item<kFewTokens>(p, l_item, lo, hi);
    const int64_t row = (int64_t)max(l_e, 0) * p.n_out + (int64_t)(l_pos * wr_n + wr) * 16;
    l_codes = reinterpret_cast<const uint8_t*>(p.codes[0]) + (row + (lane >> 3)) * row_bytes + ga * 32 + (lane & 7) * 16;
    l_params = p.params[0] + (row + (lane >> 2)) * p.pstride + ga + (lane & 3);
  };
  if (l_left > 0) l_open();
  auto fetch = [&]() {
    if (l_left > 0) {
      const int first_row = (l_pos * wr_n + wr) * 16;
      const int ng = min(4, gb - ga - 4 * l_stage);
      const uint32_t dst = l_dst + l_buf * STAGE, pdst = l_pdst + l_buf * STAGE;
      const uint8_t* src = l_codes + l_stage * 128;
      const uint32_t* psrc = l_params + l_stage * 4;
      const int rows = p.n_out - first_row;  // rows past the matrix are neither loaded nor stored
      if ((lane & 7) < 2 * ng) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((lane >> 3) + 4 * j < rows)
              cp_async16_s((dst ^ ((j & 1) << 6)) + i * kFewStage + j * 512, src + i * codes_diff + j * 4 * row_bytes);
      }
      if ((lane & 3) < ng) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if ((lane >> 2) + 8 * j < rows)
              cp_async4_s(pdst + i * kFewStage + j * 128, psrc + i * params_diff + j * 8 * p.pstride);
      }
      if (++l_stage == stages) {
        l_stage = 0;
        --l_left;
        l_codes += tile_bytes;
        l_params += tile_params;
        if (++l_pos == f.tiles) {
          l_pos = 0;
          ++l_item;
          if (l_left > 0) l_open();
        }
      }
      if (++l_buf == D) l_buf = 0;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < D - 1; ++i) fetch();

  // ---- compute side
  int item = -1, e = 0, lo = 0, hi = 0, m = 0, buf = 0;
  float scale2[2] = {};  // powers of two of tokens 2 t4 and 2 t4 + 1
  // this warp's slice of the item's activations: largest |x| of a token to [2^14, 2^15), fragment order
  auto stage_x = [&]() {
    const int vecs = (gb - ga) * 8;  // 16-byte vectors of a token's slice
    __syncwarp();
    for (int tok = 0; tok < m; ++tok) {
      const int row = source_row(p, lo + tok);
      const uint4* src = reinterpret_cast<const uint4*>(p.x + (int64_t)max(row, 0) * p.x_stride + ga * 64);
      float inv = 1.0f, sc = 1.0f;
      if (p.bf16) {
        uint32_t mx = 0;
        if (row >= 0)
          for (int v = lane; v < vecs; v += 32) mx = max(mx, max_abs_bits(src[v]));
        const int ex = row_exponent(__reduce_max_sync(0xffffffffu, mx));
        inv = exp2f(static_cast<float>(-ex));
        sc = exp2f(static_cast<float>(ex));
      }
      if (tok == 2 * t4) scale2[0] = sc;
      if (tok == 2 * t4 + 1) scale2[1] = sc;
      for (int v = lane; v < vecs; v += 32) {
        uint4 o = make_uint4(0, 0, 0, 0);
        if (row >= 0) o = p.bf16 ? permute_bf16(src[v], inv) : permute_f16(src[v]);
        // word c of the group: lane c / 2 of the quad, half c & 1
        const int grp = v >> 3, c = v & 7;
        reinterpret_cast<uint4*>(sx)[((grp * 2 + (c & 1)) * m + tok) * 4 + (c >> 1)] = o;
      }
    }
    __syncwarp();
  };

  // byte offsets of this lane's two words of group q in a row pair's stage
  uint32_t woff[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) woff[q] = g8 * 128 + (((2 * q + (t4 >> 1)) ^ g8) << 4) + (t4 & 1) * 8;
  int left = static_cast<int>(p1 - p0), it = static_cast<int>(p0 / f.tiles);
  int tile0 = static_cast<int>(p0 - (int64_t)it * f.tiles);
  while (left > 0) {
    // a batch: positions of one item
    if (it != item) {
      e = find_item<kFewTokens>(p, it, lo, hi);
      item = it;
      m = hi - lo;
      stage_x();
    }
    const int nb = min(min(f.batch, f.tiles - tile0), left);
    for (int b = 0; b < nb; ++b) {
      float acc[MT][4] = {};
      const int tile = (tile0 + b) * wr_n + wr;
      for (int st = 0; st < stages; ++st) {
        fetch();
        cp_async_wait<D - 1>();
        __syncwarp();
        if (tile < row_tiles) {
          const uint8_t* src = ring + buf * STAGE;
          const int ng = min(4, gb - ga - 4 * st);
          uint4 pq[MT][2];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              pq[i][h] = *reinterpret_cast<const uint4*>(src + i * kFewStage + 2048 + (g8 + 8 * h) * 16);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (q >= ng) break;
            const uint4* bx = reinterpret_cast<const uint4*>(sx) + (4 * st + q) * 8 * m;
            uint4 b0 = make_uint4(0, 0, 0, 0), b1 = b0;
            if (g8 < m) {
              b0 = bx[g8 * 4 + t4];
              b1 = bx[(m + g8) * 4 + t4];
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t a[2][2][4];  // [row half][word][pair]
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint2 w = *reinterpret_cast<const uint2*>(src + i * kFewStage + woff[q] + h * 1024);
                const uint32_t v = q == 0 ? pq[i][h].x : q == 1 ? pq[i][h].y : q == 2 ? pq[i][h].z : pq[i][h].w;
                const uint32_t s24 = __byte_perm(v, v, 0x1010), bb = __byte_perm(v, v, 0x3232);
                const uint32_t s20 = hfma2_bits(s24, 0x2c002c00u, 0x80008000u);  // * 2^-4
                dequant_word(w.x, s24, s20, bb, a[h][0]);
                dequant_word(w.y, s24, s20, bb, a[h][1]);
              }
              mma_f16_16816(acc[i], a[0][0][0], a[1][0][0], a[0][0][1], a[1][0][1], b0.x, b0.y);
              mma_f16_16816(acc[i], a[0][0][2], a[1][0][2], a[0][0][3], a[1][0][3], b0.z, b0.w);
              mma_f16_16816(acc[i], a[0][1][0], a[1][1][0], a[0][1][1], a[1][1][1], b1.x, b1.y);
              mma_f16_16816(acc[i], a[0][1][2], a[1][1][2], a[0][1][3], a[1][1][3], b1.z, b1.w);
            }
          }
        }
        __syncwarp();  // the stage is read before it is loaded again
        if (++buf == D) buf = 0;
      }
      // partial sums [batch][matrix][wr][slice][token][16 rows]
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int tok = 2 * t4 + (c & 1);
          if (tok < m)
            red[((((b * MT + i) * wr_n + wr) * wk + kslice) * m + tok) * 16 + g8 + 8 * (c >> 1)] =
                acc[i][c] * scale2[c & 1];
        }
    }
    // ---- sums over the slices, the row's power of two, the gate, the output
    if (f.ck > 1)
      cluster_sync_all();
    else
      __syncthreads();
    const int outs = nb * wr_n * 16 * m;
    const uint32_t red_addr = smem_u32(red);
    for (int o = tid + rank * kFewWarps * 32; o < outs; o += kFewWarps * 32 * f.ck) {
      const int r = o & 15, rest = o >> 4;
      const int w = rest % wr_n, bt = rest / wr_n;  // rows fastest over the tiles of a position
      const int b = bt % nb, tok = bt / nb;
      const int n = ((tile0 + b) * wr_n + w) * 16 + r;
      if (n >= p.n_out) continue;
      float sum[2];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int at = (((b * MT + i) * wr_n + w) * wk * m + tok) * 16 + r;
        float s = 0.0f;
        if (f.ck > 1) {
          for (int c = 0; c < f.ck; ++c) {
            const uint32_t base = dsmem_addr(red_addr, c) + at * 4;
#pragma unroll 4
            for (int k = 0; k < wk; ++k) s += ld_dsmem_f32(base + k * m * 64);
          }
        } else {
#pragma unroll 4
          for (int k = 0; k < wk; ++k) s += red[at + k * m * 16];
        }
        sum[i] = s * p.row_scale[i][(int64_t)e * p.n_out + n];
      }
      const float y = GATED ? silu_mul(sum[0], sum[1]) : sum[0];
      p.out[(int64_t)(lo + tok) * p.out_stride + n] = p.bf16 ? f2h<true>(y) : f2h<false>(y);
    }
    if (f.ck > 1)
      cluster_sync_all();
    else
      __syncthreads();
    left -= nb;
    if ((tile0 += nb) == f.tiles) {
      tile0 = 0;
      ++it;
    }
  }
}

constexpr int kFewSmem = 220 * 1024;

template <int MT, int D>
static cudaError_t launch_few_t(const FewParams& f, int smem, int ctas, int dev, cudaStream_t stream) {
  static unsigned long long done = 0;
  auto kfn = linear_few_kernel<MT, D>;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) {
    cudaError_t err = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
    if (err != cudaSuccess) return err;
    if (bit) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kFewWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = f.ck;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = f.ck > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kfn, f);
}

// Which kernel: the mean number of rows of a matrix decides (a grouped call's counts are on the
// device).
bool linear_uses_tensor_tiles(int rows, int experts, bool grouped) {
  const int mean = grouped ? (rows + experts - 1) / experts : rows;
  return mean > kFewTokens;
}

cudaError_t launch_linear_few(const LinearParams& p, cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return err;
  const int mt = p.codes[1] != nullptr ? 2 : 1;
  const int tok = min(p.rows, kFewTokens);
  const int64_t items = p.offsets != nullptr ? (int64_t)min(p.experts, p.rows) + p.rows / kFewTokens
                                             : (p.rows + kFewTokens - 1) / kFewTokens;
  FewParams f{};
  f.p = p;
  // Slices along the inputs: up to 16 warps with at least 4 groups (a whole stage) each.
  f.wk = 1;
  while (f.wk < kFewWarps && p.groups >= f.wk * 8) f.wk *= 2;
  const int row_tiles = (p.n_out + 15) / 16;
  const int wr_n = kFewWarps / f.wk;
  f.tiles = (row_tiles + wr_n - 1) / wr_n;
  f.batch = std::max(1, std::min(16, 32 / (mt * tok)));  // 32 KB of sums
  const int red = f.batch * mt * kFewWarps * tok * 64;
  // A cluster splits the inputs when the activations of a CTA would leave no room for two stages.
  f.ck = 1;
  for (;; f.ck *= 2) {
    f.slice = (p.groups + f.wk * f.ck - 1) / (f.wk * f.ck);
    f.x_stride = f.slice * 128 * tok;
    if (f.ck == 8 || kFewWarps * (2 * mt * kFewStage + f.x_stride) + red <= kFewSmem) break;
  }
  const int room = kFewSmem - red - kFewWarps * f.x_stride;
  const int d = min(mt == 2 ? 3 : 5, room / (kFewWarps * mt * kFewStage));
  if (d < 2) return cudaErrorNotSupported;  // (more than 8 x 16 x 19 groups of 64 inputs)
  const int smem = kFewWarps * (d * mt * kFewStage + f.x_stride) + red;
  const int ctas = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(items * f.tiles, sms / f.ck))) * f.ck;
  if (mt == 2) return d == 2 ? launch_few_t<2, 2>(f, smem, ctas, dev, stream) : launch_few_t<2, 3>(f, smem, ctas, dev, stream);
  switch (d) {
    case 2: return launch_few_t<1, 2>(f, smem, ctas, dev, stream);
    case 3: return launch_few_t<1, 3>(f, smem, ctas, dev, stream);
    case 4: return launch_few_t<1, 4>(f, smem, ctas, dev, stream);
    default: return launch_few_t<1, 5>(f, smem, ctas, dev, stream);
  }
}

}  // namespace am
