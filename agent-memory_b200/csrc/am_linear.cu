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

// ---------------------------------------------------------------- few tokens (HBM-bound)
// Up to 8 * NT tokens of one matrix or expert: y^T = W x^T on mma.sync m16n8k16 with the weights as
// the A operand straight from their packed words.  tcgen05 would take the dequantized weights
// through TMEM or shared memory; here a weight is used for at most 32 tokens and the kernel is
// bound by the bytes of the codes, so the operand that needs no staging wins.
//
// * Dequantization: one AND turns two nibbles of a word into fp16 subnormals code * 2^-24 (or
//   * 2^-20), one packed FMA with (scale * 2^24 or 2^20, bias) makes the two weights, rounded
//   once: 9 operations for 8 weights.  The row's exponent (am_q4_weight_pack) keeps scale * 2^24
//   inside fp16 and is undone on the fp32 result.
// * The inputs of a group of 64 are permuted over the MMA's k slots so that lane t of a quad owns
//   words 2t and 2t + 1 of its row: 8-byte loads, four lanes a 32-byte sector.  The
//   activations are staged in the same order, as fp16 under a power of two per token
//   (exact), in fragment order: one conflict-free 16-byte load per two MMAs.
// * A warp owns MT tiles of 16 weight rows (gated: one of each matrix) and a range of groups; WK
//   of a CTA's 8 warps and CK CTAs of a cluster split the inputs, partial sums meet in shared
//   memory (in a fixed order: results do not depend on timing).  A CTA walks row tiles with
//   stride gridDim.x and loads GQ groups ahead, across tile ends.
// * Before griddepcontrol.wait the CTA only asks L2 for its first codes (a prefetch reads
//   nothing, so it may run before the previous kernel is done).
constexpr int kFewWarps = 8;
constexpr int kFewSmemX = 96 * 1024;  // staged activations; longer inputs go in several stages

struct FewParams {
  LinearParams p;
  int32_t wk;         // warps along the inputs (1, 2, 4 or 8)
  int32_t ck;         // CTAs of a cluster along the inputs
  int32_t tiles;      // row tiles of a matrix for one CTA (8 / wk warps x 16 rows x (gated ? 1 : MT))
  int32_t x_groups;   // groups staged at a time (a multiple of 4)
};

__device__ __forceinline__ uint2 ld_codes(const uint32_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

template <int NT, int MT, bool GATED, int GQ>
__global__ void __launch_bounds__(kFewWarps * 32, 2) linear_few_kernel(const __grid_constant__ FewParams f) {
  static_assert(!GATED || MT == 2, "a gated warp holds one tile of each matrix");
  constexpr int TOK = 8 * NT;
  const LinearParams& p = f.p;
  extern __shared__ __align__(16) uint8_t smem[];
  // [0, TOK) token exponents as floats, [TOK, 2 TOK) token maxima, then the staged activations /
  // the partial sums
  float* tok_scale = reinterpret_cast<float*>(smem);
  int* tok_max = reinterpret_cast<int*>(smem) + TOK;
  int* tok_row = reinterpret_cast<int*>(smem) + 2 * TOK;
  uint8_t* sx = smem + 3 * TOK * 4;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int rank = f.ck > 1 ? static_cast<int>(blockIdx.x) % f.ck : 0;  // clusters lie along x
  const int first_tile = static_cast<int>(blockIdx.x) / f.ck;
  const int tile_step = static_cast<int>(gridDim.x) / f.ck;
  const int wk = f.wk, wr_n = kFewWarps / wk;
  const int kslice = warp % wk, wr = warp / wk;
  const int rows_per_warp = GATED ? 16 : 16 * MT;
  const int rows_per_cta = rows_per_warp * wr_n;
  // this CTA's and this warp's quads of groups
  const int quads = p.pstride >> 2;
  const int cq0 = quads * rank / f.ck, cq1 = quads * (rank + 1) / f.ck;

  griddep_launch_dependents();
  if (p.offsets == nullptr) {  // L2 prefetch of the first tile's codes: rows tid / wk.., 128 bytes each step
    const int r = tid >> 1;
    const int64_t n = (int64_t)first_tile * rows_per_cta + r;
    if (r < rows_per_cta && n < p.n_out) {
      const char* c = reinterpret_cast<const char*>(p.codes[0] + n * (p.n_in / 8));
      const int b1 = min(cq1 * 128, p.n_in / 2);
      for (int b = cq0 * 128 + (tid & 1) * 128; b < b1; b += 256)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(c + b));
    }
  }
  griddep_wait();

  int lo, hi;
  const int e = find_item<TOK>(p, blockIdx.y, lo, hi);
  if (e < 0) return;  // the whole cluster: it shares blockIdx.y
  const int m = hi - lo;
  const uint32_t* codes[MT];
  const uint32_t* params[MT];
  const int64_t wbase = (int64_t)e * p.n_out;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    codes[i] = p.codes[GATED ? i : 0];
    params[i] = p.params[GATED ? i : 0];
  }

  if (tid < TOK) {
    tok_row[tid] = tid < m ? source_row(p, lo + tid) : -1;
    tok_max[tid] = 0;
  }
  __syncthreads();
  // token exponents: the largest |x| over this CTA's inputs goes to [2^14, 2^15)
  const int xg0 = cq0 * 4, xg1 = min(cq1 * 4, p.groups);
  if (p.bf16) {
    const int vecs = (xg1 - xg0) * 8;  // 16-byte vectors of a token
    for (int i = tid; i < ((vecs + 31) & ~31) * m; i += kFewWarps * 32) {
      const int tok = i / ((vecs + 31) & ~31), v = i % ((vecs + 31) & ~31);
      uint32_t mx = 0;
      const int row = tok_row[tok];
      if (v < vecs && row >= 0) {
        const uint4 u = *reinterpret_cast<const uint4*>(p.x + (int64_t)row * p.x_stride + xg0 * 64 + v * 8);
        mx = max_abs_bits(u);
      }
      mx = __reduce_max_sync(0xffffffffu, mx);
      if (lane == 0) atomicMax(&tok_max[tok], static_cast<int>(mx));
    }
    __syncthreads();
  }
  if (tid < TOK) {
    const int ex = p.bf16 ? row_exponent(tok_max[tid]) : 0;
    tok_scale[tid] = exp2f(static_cast<float>(ex));
    tok_max[tid] = __float_as_int(exp2f(static_cast<float>(-ex)));
  }
  __syncthreads();
  const float* tok_inv = reinterpret_cast<const float*>(tok_max);

  const int x_groups = f.x_groups;
  float acc[MT][NT][4];
  uint2 cw[2][MT][GQ][2];  // codes: rows g8 and g8 + 8
  uint32_t pw[2][MT][2][GQ];

  auto weight_row = [&](int tile, int i, int half) -> int {
    const int n = tile * rows_per_cta + wr * rows_per_warp + (GATED ? 0 : 16 * i) + g8 + 8 * half;
    return min(n, p.n_out - 1);  // rows past the matrix repeat its last one; their sums are not stored
  };
  auto load_step = [&](int buf, int tile, int gs) {  // groups gs .. gs + GQ - 1
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t row = wbase + weight_row(tile, i, h);
        const uint32_t* c = codes[i] + row * (p.n_in / 8) + gs * 8 + 2 * t4;
#pragma unroll
        for (int q = 0; q < GQ; ++q) cw[buf][i][q][h] = gs + q < p.groups ? ld_codes(c + q * 8) : make_uint2(0, 0);
        const uint32_t* pp = params[i] + row * p.pstride + gs;
        if constexpr (GQ == 4) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(pp));
          pw[buf][i][h][0] = v.x;
          pw[buf][i][h][1] = v.y;
          pw[buf][i][h][2] = v.z;
          pw[buf][i][h][3] = v.w;
        } else {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(pp));
          pw[buf][i][h][0] = v.x;
          pw[buf][i][h][1] = v.y;
        }
      }
  };
  auto compute_step = [&](int buf, int gs, int stage0) {
#pragma unroll
    for (int q = 0; q < GQ; ++q) {
      if (gs + q >= p.groups) break;
      const uint4* bx = reinterpret_cast<const uint4*>(sx) + (int64_t)(gs + q - stage0) * 8 * m;
      uint32_t bf[NT][2][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (n * 8 + g8 < m) v = bx[(h * m + n * 8 + g8) * 4 + t4];
          bf[n][h][0] = v.x;
          bf[n][h][1] = v.y;
          bf[n][h][2] = v.z;
          bf[n][h][3] = v.w;
        }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint32_t s24[2], s20[2], bb[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t v = pw[buf][i][h][q];
          s24[h] = __byte_perm(v, v, 0x1010);
          bb[h] = __byte_perm(v, v, 0x3232);
          s20[h] = hfma2_bits(s24[h], 0x2c002c00u, 0x80008000u);  // * 2^-4
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t a0[4], a1[4];
          dequant_word(w == 0 ? cw[buf][i][q][0].x : cw[buf][i][q][0].y, s24[0], s20[0], bb[0], a0);
          dequant_word(w == 0 ? cw[buf][i][q][1].x : cw[buf][i][q][1].y, s24[1], s20[1], bb[1], a1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16_16816(acc[i][n], a0[0], a1[0], a0[1], a1[1], bf[n][w][0], bf[n][w][1]);
            mma_f16_16816(acc[i][n], a0[2], a1[2], a0[3], a1[3], bf[n][w][2], bf[n][w][3]);
          }
        }
      }
    }
  };

  // stage groups [s0, s1) of the activations in fragment order
  auto stage_x = [&](int s0, int s1) {
    const int n = (s1 - s0) * 8;
    for (int i = tid; i < n * m; i += kFewWarps * 32) {
      const int tok = i / n, v = i % n;  // v: 8 inputs of the token
      const int grp = v >> 3, c = v & 7;
      const int row = tok_row[tok];
      uint4 o = make_uint4(0, 0, 0, 0);
      if (row >= 0) {
        const uint4 u = *reinterpret_cast<const uint4*>(p.x + (int64_t)row * p.x_stride + (int64_t)s0 * 64 + v * 8);
        o = p.bf16 ? permute_bf16(u, tok_inv[tok]) : permute_f16(u);
      }
      // word c of the group: lane c / 2 of the quad, half c & 1
      reinterpret_cast<uint4*>(sx)[((int64_t)grp * 2 + (c & 1)) * m * 4 + tok * 4 + (c >> 1)] = o;
    }
  };

  bool staged_all = (xg1 - xg0) <= x_groups;
  if (staged_all) stage_x(xg0, xg1);
  // partial sums: [matrix or half][warp row][k slice][token][16 rows]; at the same offset in
  // every CTA of a cluster
  float* red = reinterpret_cast<float*>(sx + (size_t)x_groups * 128 * m);
  for (int tile = first_tile; tile < f.tiles; tile += tile_step) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][n][c] = 0.0f;
    for (int s0 = xg0; s0 < xg1; s0 += x_groups) {
      const int s1 = min(s0 + x_groups, xg1);
      if (!staged_all) {
        __syncthreads();  // the previous stage is read
        stage_x(s0, s1);
      }
      // this warp's steps of GQ groups
      const int sq = (s1 - s0 + 3) >> 2;
      const int a = s0 + 4 * (sq * kslice / wk), b = min(s0 + 4 * (sq * (kslice + 1) / wk), s1);
      if (a < b) load_step(0, tile, a);
      __syncthreads();  // the activations are staged (and the last tile's sums are read)
      int gs = a;
      while (gs < b) {
        if (gs + GQ < b) load_step(1, tile, gs + GQ);
        compute_step(0, gs, s0);
        gs += GQ;
        if (gs >= b) break;
        if (gs + GQ < b) load_step(0, tile, gs + GQ);
        compute_step(1, gs, s0);
        gs += GQ;
      }
    }
    // partial sums to shared memory: acc[i][n] = rows g8 (+8), tokens 8 n + 2 t4 (+1)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int tok = n * 8 + 2 * t4 + (c & 1);
          if (tok < m) red[(((i * wr_n + wr) * wk + kslice) * m + tok) * 16 + g8 + 8 * (c >> 1)] = acc[i][n][c];
        }
    if (f.ck > 1)
      cluster_sync_all();
    else
      __syncthreads();
    // sums over the slices, scales, the gate, the output: one thread per (row, token), rows fastest
    const int rows_out = rows_per_cta;
    const uint32_t red_addr = smem_u32(red);
    for (int o = tid + rank * kFewWarps * 32; o < rows_out * m; o += kFewWarps * 32 * f.ck) {
      const int tok = o / rows_out, rr = o % rows_out;
      const int w_r = rr / rows_per_warp, in_warp = rr % rows_per_warp;
      const int n = tile * rows_per_cta + rr;
      if (n >= p.n_out) continue;
      float sum[2];
#pragma unroll
      for (int which = 0; which < (GATED ? 2 : 1); ++which) {
        const int i = GATED ? which : in_warp >> 4;
        const int at = ((i * wr_n + w_r) * wk * m + tok) * 16 + (in_warp & 15);
        float s = 0.0f;
        if (f.ck > 1) {
          for (int c = 0; c < f.ck; ++c) {
            float part = 0.0f;
            const uint32_t base = dsmem_addr(red_addr, c);
            for (int k = 0; k < wk; ++k) part += ld_dsmem_f32(base + (at + k * m * 16) * 4);
            s += part * ld_dsmem_f32(dsmem_addr(smem_u32(&tok_scale[tok]), c));
          }
        } else {
          for (int k = 0; k < wk; ++k) s += red[at + k * m * 16];
          s *= tok_scale[tok];
        }
        sum[which] = s * p.row_scale[which][wbase + n];
      }
      const float y = GATED ? silu_mul(sum[0], sum[1]) : sum[0];
      p.out[(int64_t)(lo + tok) * p.out_stride + n] = p.bf16 ? f2h<true>(y) : f2h<false>(y);
    }
    if (f.ck > 1) cluster_sync_all();  // peers have read this CTA's sums
  }
}

template <int NT, int MT, bool GATED, int GQ>
static cudaError_t launch_few_t(const LinearParams& p, int items, cudaStream_t stream) {
  constexpr int TOK = 8 * NT;
  FewParams f{};
  f.p = p;
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return err;
  // Split of the work: enough warps along the inputs that every SM has two CTAs' worth of warps,
  // at least one quad of groups (256 inputs) each.
  const int warp_rows = GATED ? 16 : 16 * MT;
  const int64_t row_warps = (int64_t)((p.n_out + warp_rows - 1) / warp_rows) * items;
  const int quads = p.pstride / 4;
  const int slots = sms * 2 * kFewWarps;
  int split = 1;
  while (split < 64 && split * 2 <= quads && row_warps * split < slots) split *= 2;
  // a long row of tiles: halving a warp's work evens the last round out
  while (split < 8 && split * 2 <= quads) {
    const double per = (double)row_warps * split / slots;
    if (per >= 8.0 || ceil(per) / per < 1.06) break;
    split *= 2;
  }
  const int tok = min(p.offsets != nullptr ? TOK : p.rows, TOK);
  f.wk = min(split, kFewWarps);
  f.ck = split / f.wk;
  const int x_limit = kFewSmemX / (128 * tok) & ~3;
  while (f.ck < 8 && (quads + f.ck - 1) / f.ck * 4 > x_limit && f.ck * 2 <= quads) f.ck *= 2;
  f.x_groups = min(x_limit, (quads + f.ck - 1) / f.ck * 4);
  const int rows_per_cta = warp_rows * (kFewWarps / f.wk);
  f.tiles = (p.n_out + rows_per_cta - 1) / rows_per_cta;
  const int smem = 3 * TOK * 4 + f.x_groups * 128 * tok + kFewWarps * MT * 16 * tok * 4;
  static unsigned long long done = 0;
  auto kfn = linear_few_kernel<NT, MT, GATED, GQ>;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) {
    err = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               3 * TOK * 4 + kFewSmemX + kFewWarps * MT * 16 * TOK * 4);
    if (err != cudaSuccess) return err;
    if (bit) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
  }
  const int per_sm = smem > 110 * 1024 ? 1 : 2;
  const int ctas = max(1, min(f.tiles, (sms * per_sm) / max(1, f.ck * items)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas * f.ck, items);
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

template <int NT>
static cudaError_t launch_few(const LinearParams& p, cudaStream_t stream) {
  const int tok = 8 * NT;
  const int64_t items = p.offsets != nullptr ? (int64_t)min(p.experts, p.rows) + p.rows / tok
                                             : (p.rows + tok - 1) / tok;
  constexpr int GQ = 2;
  if (items > 65535) return cudaErrorInvalidConfiguration;
  if (p.codes[1] != nullptr) return launch_few_t<NT, 2, true, GQ>(p, static_cast<int>(items), stream);
  if constexpr (NT == 1) return launch_few_t<NT, 1, false, 4>(p, static_cast<int>(items), stream);
  return launch_few_t<NT, 2, false, GQ>(p, static_cast<int>(items), stream);
}

// Which kernel: the mean number of rows of a matrix decides (a grouped call's counts are on the
// device).
bool linear_uses_tensor_tiles(int rows, int experts, bool grouped) {
  const int mean = grouped ? (rows + experts - 1) / experts : rows;
  return mean > 8;
}

cudaError_t launch_linear_few(const LinearParams& p, cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  const int mean = p.offsets != nullptr ? (p.rows + p.experts - 1) / p.experts : p.rows;
  if (mean <= 8) return launch_few<1>(p, stream);
  if (mean <= 16) return launch_few<2>(p, stream);
  return launch_few<4>(p, stream);
}

}  // namespace am
