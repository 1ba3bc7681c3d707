// Linear layers over 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k], W = scale * code + bias
// per group of 64 inputs; gated: silu(x G^T) * (x U^T); and both per expert over rows sorted
// by expert.
#include <algorithm>
#include <climits>

#include "am_internal.h"
#include "am_linear.cuh"

namespace am {

int sm_count(int* device) {
  static int counts[64] = {};
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  *device = dev;
  if (dev < 64) n = __atomic_load_n(&counts[dev], __ATOMIC_RELAXED);
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) __atomic_store_n(&counts[dev], n, __ATOMIC_RELAXED);
  return n;
}

// ---------------------------------------------------------------- weight parameters
// One warp per weight row: the row's exponent e is the smallest with every |scale| * 2^(24-e)
// and |bias| * 2^(20-e) at most 2^15 (fp16 holds up to 65504), then the groups' pairs are scaled by
// these powers of two and stored as fp16.  The two reach their limit together at |bias| =
// 16 scale, just above what a quantizer of 16 levels gives (0 to -15 scale), so both have fp16's
// whole range below the row's largest: with L the larger of max |scale| and max |bias| / 16, a
// scale is exact from 2^-28 L and a bias from 2^-24 L on (those of bf16 8 times further down).
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
  if (mb > 0.0f) e = max(e, exponent_above(fminf(mb, kMax)) + 20 - 15);
  if (ms == 0.0f && mb == 0.0f) e = 0;
  e = min(e, 127);
  if (lane == 0) row_scale[row] = ldexpf(1.0f, e);
  const int pstride = (groups + 3) & ~3;
  for (int g = lane; g < pstride; g += 32) {
    uint32_t v = 0;
    if (g < groups) v = pack_half2(ldexpf(h2f<BF16>(s[g]), 24 - e), ldexpf(h2f<BF16>(b[g]), 20 - e));
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
// Up to 8 tokens of one matrix or expert: y^T = W x^T on mma.sync m16n8k16 with the codes as the A
// operand straight from their packed words.  tcgen05 would take dequantized weights through
// TMEM; here a weight is used for at most 8 tokens and the kernel is bound by the bytes of the
// codes, so the operand that needs no staging wins.
//
// * Per group of 64 inputs y += scale * (codes . x) + bias * sum(x), the first dot product on
//   the tensor cores (exact products, fp32 sums), the rest in fp32: no weight is rounded.  One
//   AND turns two nibbles of a word into fp16 subnormals code * 2^-24, or 16 code * 2^-24 for
//   the odd nibbles, whose activations are staged divided by 16: 5 integer operations for 8
//   weights; the parameters hold scale * 2^24 and bias * 2^20 (am_q4_weight_pack).
// * The inputs of a group are permuted over the MMA's k slots so that lane t of a quad owns words
//   2t and 2t + 1 of its row.  The activations are staged in the same order, as fp16 under a
//   power of two per token and slice (exact), in fragment order, with their group sums.
// * A CTA of 16 warps a SM.  wk of them split the inputs, the others take further row tiles; when
//   the activations do not fit, CK CTAs of a cluster split the inputs again.  Every warp
//   streams its slices of the row tiles (16 rows x up to 4 groups a stage) through a private
//   cp.async ring: the warps of a SM keep 74 to 110 KB in flight, across tile and expert ends.
// * Partial sums meet in shared memory every few tiles, in a fixed order.
// * The work of all experts is one sequence of row tiles, cut evenly over the CTAs.
// * What bounds it (ncu, 128256x4096): no unit alone.  1 token 56 us, 5.3 TB/s (a plain read of the
//   bytes 45.7): issue slots 65 % busy (70 instructions a warp for 16 weight rows x 64 inputs), ALU
//   60 %, shared memory 55 %.  8 tokens 70 us: shared memory 70 % (23 wavefronts for the same piece, 8
//   of them the activations read again for every row tile), issue 60 % (83 instructions), DRAM 50 %.
//   Small matrices by a start of 3 us: 1 token 4096x4096 5.6 us; 8 tokens 4096x14336 14.9.
// * Before griddepcontrol.wait the CTA only asks L2 for its first codes (a prefetch reads
//   nothing, so it may run before the previous kernel is done).
constexpr int kFewWarps = 16, kFewLogWarps = 4;
constexpr int kFewTokens = 8;
constexpr int kFewCodes = 16 * 128, kFewPar = 16 * 16;  // bytes of 16 rows x 4 groups

struct FewParams {
  LinearParams p;
  int32_t lwk;    // log2 of the warps along the inputs (1 to 16)
  int32_t lck;    // log2 of the CTAs of a cluster along the inputs (1 to 8)
  int32_t tiles;  // positions of one item: row tiles / (16 / wk), rounded up
  int32_t batch;  // positions between two sums
};

// Ring depth of a warp: what leaves room for the activations of a few thousand inputs.
template <bool GATED, int TK>
constexpr int kFewDepth = GATED ? 2 : (TK == 8 ? 3 : 4);

// D = A x B with a zero accumulator.
__device__ __forceinline__ void mma_f16_16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// D += A x B (as mma_f16_16816, free to be scheduled among other tiles' operations).
__device__ __forceinline__ void mma_f16_16816_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight activations of a token times `f` (a power of two) in the order of the A operand, the odd
// inputs of a word divided by 16; `sum` gets their fp32 sum (of the scaled values).
template <bool BF16>
__device__ __forceinline__ uint4 stage_inputs(uint4 u, float f, float& sum) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float v[8];
  sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = h2f<BF16>(static_cast<uint16_t>(w[j])) * f;
    v[2 * j + 1] = h2f<BF16>(static_cast<uint16_t>(w[j] >> 16)) * f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sum += v[j];
  constexpr float k = 0.0625f;
  return make_uint4(pack_half2(v[0], v[4]), pack_half2(v[1] * k, v[5] * k), pack_half2(v[2], v[6]),
                    pack_half2(v[3] * k, v[7] * k));
}

// The share [p0, p0 + n) of `total` positions of one of the clusters.
__device__ __forceinline__ void few_share(int total, int cluster, int clusters, int& p0, int& n) {
  const int each = total / clusters, more = total - each * clusters;
  p0 = each * cluster + min(cluster, more);
  n = each + (cluster < more);
}

// The positions of this CTA's cluster again, as far as their tokens are not finite (store_nonfinite; by the
// CTAs whose inputs those are).
static __device__ __noinline__ void few_store_nonfinite(const FewParams& f, int tk) {
  const LinearParams& p = f.p;
  const int clusters = static_cast<int>(gridDim.x) >> f.lck, cluster = static_cast<int>(blockIdx.x) >> f.lck;
  const int items = p.offsets == nullptr ? (p.rows + tk - 1) / tk : count_items(p, tk);
  const int rows = 16 << (kFewLogWarps - f.lwk);
  int p0, n_pos;
  few_share(items * f.tiles, cluster, clusters, p0, n_pos);
  for (int q = p0; q < p0 + n_pos; ++q) {
    int lo, hi;
    const int e = find_item(p, q / f.tiles, tk, lo, hi);
    store_nonfinite(p, nullptr, e, lo, hi, q % f.tiles * rows, (q % f.tiles + 1) * rows);
  }
}

// TK: tokens of an item, padded to 1, 2, 4 or 8.
template <bool GATED, int TK>
__global__ void __launch_bounds__(kFewWarps * 32, 1) linear_few_kernel(const __grid_constant__ FewParams f) {
  constexpr int TROWS = 16;          // output rows of a tile
  constexpr int MT = GATED ? 2 : 1;  // matrices
  constexpr int D = kFewDepth<GATED, TK>;
  constexpr int XG = 128 * TK;  // staged bytes of a group
  const LinearParams& p = f.p;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g8 = lane >> 2, t4 = lane & 3;
  const int rank = static_cast<int>(blockIdx.x) & ((1 << f.lck) - 1);
  const int cluster = static_cast<int>(blockIdx.x) >> f.lck, clusters = static_cast<int>(gridDim.x) >> f.lck;
  const int lwr = kFewLogWarps - f.lwk, wr_n = 1 << lwr, wk = 1 << f.lwk;
  const int kslice = warp & (wk - 1), wr = warp >> f.lwk;
  // this CTA's groups [ca, cb) and this warp's [ga, gb): whole quads (16 bytes of parameters)
  const int quads = p.pstride >> 2, lsl = f.lwk + f.lck;
  const int ca = (quads * rank >> f.lck) * 4, cb = min((quads * (rank + 1) >> f.lck) * 4, p.groups);
  const int qa = quads * ((rank << f.lwk) + kslice) >> lsl, qb = quads * ((rank << f.lwk) + kslice + 1) >> lsl;
  const int ga = qa * 4, gb = min(qb * 4, p.groups);
  const int stages = qb - qa;  // of one row tile
  const int cta_groups = ((quads + (1 << f.lck) - 1) >> f.lck) * 4;  // at most
  constexpr int STAGE = MT * (kFewCodes + kFewPar);
  uint8_t* ring = smem + warp * (D * STAGE);
  uint8_t* sx = smem + kFewWarps * D * STAGE;  // [group][half][TK][4] x 16 bytes
  float* sxsum = reinterpret_cast<float*>(sx + cta_groups * XG);     // [group][TK], times 2^-20
  float* sxmax = sxsum + cta_groups * TK;  // [warp]: largest |x| of its part of a token, as bits
  volatile int* marked = reinterpret_cast<volatile int*>(sxmax + kFewWarps);  // a token is not finite
  float* red = sxmax + kFewWarps + 4;
  *marked = 0;  // (by every thread; stage_x has a barrier before it is set)
  const int row_tiles = (p.n_out + TROWS - 1) / TROWS;

  griddep_launch_dependents();
  // positions [p0, p0 + n_pos) of the sequence of all items' positions
  int items = (p.rows + TK - 1) / TK, p0, n_pos;
  auto share = [&]() { few_share(items * f.tiles, cluster, clusters, p0, n_pos); };
  if (p.offsets == nullptr) {
    share();
    // L2 prefetch of the first tiles' codes: a lane pair a row
    if (p0 < f.tiles) {
#pragma unroll 1
      for (int i = 0; i < MT; ++i) {
        const int64_t n = (int64_t)((p0 << lwr) + wr) * TROWS + (lane >> 1);
        if (n < p.n_out) {
          const char* c = reinterpret_cast<const char*>(p.codes[i] + n * (p.n_in / 8));
          for (int g = ga + (lane & 1) * 4; g < min(gb, ga + 16); g += 8)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(c + g * 32));
        }
      }
    }
  }
  // ---- load side: walks the positions [p0, p1) D - 1 stages ahead of the sums.  A lane fetches 16
  // bytes of rows lane / 8 + 4 j of the tile, lanes 0 to 15 the parameters of a row.  (cp.async:
  // tensor-map boxes of 16 rows reached 3.5 TB/s here, these copies 6.1.)
  const int row_bytes = p.n_in / 2;
  const int64_t codes4 = (int64_t)4 * row_bytes;  // bytes to the next j
  const int64_t tile_bytes = (int64_t)wr_n * TROWS * row_bytes - stages * 128;  // from a tile's end to the next
  const int64_t tile_par = (int64_t)wr_n * TROWS * p.pstride * 4 - stages * 16;
  const uint8_t *l_codes = nullptr, *l_par = nullptr;  // this lane's bytes of the next stage, matrix 0
  const int64_t codes_diff =  // from a matrix to its partner
      GATED ? reinterpret_cast<const uint8_t*>(p.codes[1]) - reinterpret_cast<const uint8_t*>(p.codes[0]) : 0;
  const int64_t par_diff =
      GATED ? reinterpret_cast<const uint8_t*>(p.params[1]) - reinterpret_cast<const uint8_t*>(p.params[0]) : 0;
  // chunk c of row r at c ^ 2 (r % 4): the eight bytes a lane reads of four rows lie in distinct banks
  const uint32_t l_dst0 = smem_u32(ring) + (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3) << 1)) << 4);
  const uint32_t l_pdst0 = smem_u32(ring) + 2048 + (lane & 15) * 16;
  int item0, l_left, l_item, l_pos;  // (l_pos: position in the item)
  int l_stage = 0;
  uint32_t l_off = 0;  // of the next stage's buffer
  int l_rows = 0;      // weight rows from the tile's first one to the matrix's end
  auto l_open = [&]() {  // position l_pos of item l_item
    int lo, hi;
    const int e = find_item(p, l_item, TK, lo, hi);
    const int first = (l_pos * wr_n + wr) * TROWS;
    const int64_t row = (int64_t)max(e, 0) * p.n_out + first;
    l_rows = p.n_out - first;
    l_codes = reinterpret_cast<const uint8_t*>(p.codes[0]) + (row + (lane >> 3)) * row_bytes + qa * 128 + (lane & 7) * 16;
    l_par = reinterpret_cast<const uint8_t*>(p.params[0]) + ((row + (lane & 15)) * p.pstride + qa * 4) * 4;
  };
  auto l_begin = [&]() {
    item0 = p0 / f.tiles;
    l_left = n_pos;
    l_item = item0;
    l_pos = p0 - item0 * f.tiles;
    if (l_left > 0) l_open();
  };
  if (p.offsets == nullptr) l_begin();
  auto fetch = [&]() {
    if (l_left > 0) {
      const uint32_t dst = l_dst0 + l_off, pdst = l_pdst0 + l_off;
      // rows past the matrix are neither loaded nor stored, groups past the last neither loaded nor used
      const int chunks = min(8, (p.groups - (qa + l_stage) * 4) * 2);
      if (l_rows >= TROWS && chunks == 8) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const uint8_t* src = l_codes + i * codes_diff;
          cp_async16_s(dst + i * (kFewCodes + kFewPar), src);
          cp_async16_s(dst + i * (kFewCodes + kFewPar) + 512, src + codes4);
          cp_async16_s(dst + i * (kFewCodes + kFewPar) + 1024, src + 2 * codes4);
          cp_async16_s(dst + i * (kFewCodes + kFewPar) + 1536, src + 3 * codes4);
          if (lane < 16) cp_async16_ca_s(pdst + i * (kFewCodes + kFewPar), l_par + i * par_diff);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < MT; ++i) {
          for (int j = 0; j < 4; ++j)
            if ((lane >> 3) + 4 * j < l_rows && (lane & 7) < chunks)
              cp_async16_s(dst + i * (kFewCodes + kFewPar) + j * 512, l_codes + i * codes_diff + j * codes4);
          if (lane < min(l_rows, 16)) cp_async16_ca_s(pdst + i * (kFewCodes + kFewPar), l_par + i * par_diff);
        }
      }
      l_codes += 128;
      l_par += 16;
      if ((l_off += STAGE) == D * STAGE) l_off = 0;
      if (++l_stage == stages) {
        l_stage = 0;
        --l_left;
        l_codes += tile_bytes;
        l_par += tile_par;
        l_rows -= wr_n * TROWS;
        if (++l_pos == f.tiles) {
          l_pos = 0;
          ++l_item;
          if (l_left > 0) l_open();
        }
      }
    }
    cp_async_commit();
  };

  // ---- compute side
  int item = -1, e = 0, lo = 0, hi = 0, m = 0, buf = 0;
  // The item's activations of this CTA's inputs, the largest |x| of a token to [2^14, 2^15): 16 / TK
  // warps a token.  A lane holds its first XH vectors of 8 from the maximum to the conversion (4096
  // inputs at 8 tokens), the others are read twice.  They are asked for before the item's codes:
  // their way from L2 and the issue of the first copies take a microsecond each (1 token
  // 4096x4096 5.9 -> 5.5 us, 8 tokens 8.8 -> 7.5).  The gated kernel has no registers for eight.
  constexpr int WPT = kFewWarps / TK, XH = TK == 8 && !GATED ? 8 : 4;
  const int vecs = (cb - ca) * 8;  // 16-byte vectors of a token
  const int x_tok = warp / WPT, v0 = warp % WPT * 32 + lane;
  uint4 held[XH];
  auto open_item = [&](int i) {
    e = find_item(p, i, TK, lo, hi);
    item = i;
    m = hi - lo;
    const int x_row = x_tok < m ? source_row(p, lo + x_tok) : -1;
    const uint4* x_src = reinterpret_cast<const uint4*>(p.x + (int64_t)max(x_row, 0) * p.x_stride + (int64_t)ca * 64);
#pragma unroll
    for (int j = 0; j < XH; ++j) {
      held[j] = make_uint4(0, 0, 0, 0);
      if (x_row >= 0 && v0 + j * 32 * WPT < vecs) held[j] = x_src[v0 + j * 32 * WPT];
    }
  };
  griddep_wait();
  if (p.offsets != nullptr) {
    items = count_items(p, TK);
    share();
    l_begin();
  }
  if (n_pos > 0) open_item(item0);
#pragma unroll 1
  for (int i = 0; i < D - 1; ++i) fetch();

  auto stage_x = [&]() {
    const int x_tok = warp / WPT, v0 = warp % WPT * 32 + lane, vecs = (cb - ca) * 8;
    const int x_row = x_tok < m ? source_row(p, lo + x_tok) : -1;
    const uint4* x_src = reinterpret_cast<const uint4*>(p.x + (int64_t)max(x_row, 0) * p.x_stride + (int64_t)ca * 64);
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < XH; ++j) mx = max(mx, max_abs_bits(held[j]));
    if (x_row >= 0) {
#pragma unroll 4
      for (int v = v0 + XH * 32 * WPT; v < vecs; v += 32 * WPT) mx = max(mx, max_abs_bits(x_src[v]));
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane == 0) sxmax[warp] = __uint_as_float(mx);
    __syncthreads();
    if (x_tok < m) {
      const uint32_t all = lane < WPT ? __float_as_uint(sxmax[x_tok * WPT + lane]) : 0u;
      mx = __reduce_max_sync(0xffffffffu, all);
      if (mx >= nonfinite_bits(p)) *marked = 1;
      const float inv = exp2_int(-(p.bf16 ? row_exponent(mx) : row_exponent_f16(mx)));
      auto convert = [&](int v, uint4 u) {  // (u is zero where v is past the end)
        float sum;
        const uint4 o = p.bf16 ? stage_inputs<true>(u, inv, sum) : stage_inputs<false>(u, inv, sum);
#pragma unroll
        for (int s = 1; s < 8; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        // word c of the group: lane c / 2 of the quad, half c & 1
        const int grp = v >> 3, c = v & 7;
        if (v < vecs) {
          *reinterpret_cast<uint4*>(sx + grp * XG + ((c & 1) * TK + x_tok) * 64 + (c >> 1) * 16) = o;
          if (c == 0) sxsum[grp * TK + x_tok] = sum * 0x1p-20f;  // (what the biases are multiplied by)
        }
      };
#pragma unroll
      for (int j = 0; j < XH; ++j)
        if (v0 - lane + j * 32 * WPT < vecs) convert(v0 + j * 32 * WPT, held[j]);
#pragma unroll 2
      for (int v = v0 + XH * 32 * WPT; v - lane < vecs; v += 32 * WPT)
        convert(v, x_row >= 0 && v < vecs ? x_src[v] : make_uint4(0, 0, 0, 0));
    }
    __syncthreads();
  };

  // byte offsets of this lane's two words of group q in a row pair's stage, and of its token's
  // activations and its two columns' sums in a group
  uint32_t woff[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) woff[q] = g8 * 128 + (((2 * q + (t4 >> 1)) ^ ((g8 & 3) << 1)) << 4) + (t4 & 1) * 8;
  const uint8_t* xlane = sx + (ga - ca) * XG + (g8 & (TK - 1)) * 64 + t4 * 16;
  const float* slane = sxsum + (ga - ca) * TK + ((2 * t4) & (TK - 1));
  int left = n_pos, it = item0, staged = -1, tile0 = p0 - item0 * f.tiles;
  float tscale[2] = {};  // powers of two of this lane's columns
  while (left > 0) {
    // a batch: positions of one item
    if (it != staged) {
      if (it != item) open_item(it);
      staged = it;
      stage_x();  // (the last batch ended with a barrier after its last read of the activations)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t mx = 0;
#pragma unroll
        for (int k = 0; k < WPT; ++k) mx = max(mx, __float_as_uint(sxmax[((2 * t4 + c) & (TK - 1)) * WPT + k]));
        tscale[c] = exp2_int(p.bf16 ? row_exponent(mx) : row_exponent_f16(mx));
      }
    }
    const int nb = min(min(f.batch, f.tiles - tile0), left);
    for (int b = 0; b < nb; ++b) {
      float acc[MT][4] = {};
      const int tile = ((tile0 + b) << lwr) + wr;
      // the rows' powers of two, needed after the sums
      float rs[MT][2];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = tile * TROWS + g8 + 8 * h;
          rs[i][h] = n < p.n_out ? __ldg(p.row_scale[i] + (int64_t)e * p.n_out + n) : 0.0f;
        }
      const uint8_t* xs = xlane;
      const float* ss = slane;
      for (int st = 0; st < stages; ++st) {
        fetch();
        cp_async_wait<D - 1>();
        __syncwarp();
        if (tile < row_tiles) {
          const uint8_t* src = ring + buf;
          uint4 pq[MT][2];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              pq[i][h] = *reinterpret_cast<const uint4*>(src + i * (kFewCodes + kFewPar) + 2048 + (g8 + 8 * h) * 16);
          auto group = [&](int q) {
            // column g8 of B: the columns past TK are never read, and a 16-byte load costs a
            // pass of shared memory for every eight lanes that take part
            uint4 b0 = make_uint4(0, 0, 0, 0), b1 = b0;
            if (TK == 8 || g8 < TK) {
              b0 = *reinterpret_cast<const uint4*>(xs + q * XG);
              b1 = *reinterpret_cast<const uint4*>(xs + q * XG + TK * 64);
            }
            float2 sm;
            if constexpr (TK == 1)
              sm = make_float2(ss[q], 0.0f);
            else
              sm = *reinterpret_cast<const float2*>(ss + q * TK);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t a[2][8];  // [row half][pair]
              float sc[2], bi[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint2 w = *reinterpret_cast<const uint2*>(src + i * (kFewCodes + kFewPar) + woff[q] + h * 1024);
                const uint32_t v = q == 0 ? pq[i][h].x : q == 1 ? pq[i][h].y : q == 2 ? pq[i][h].z : pq[i][h].w;
                const float2 sb = __half22float2(*reinterpret_cast<const __half2*>(&v));
                sc[h] = sb.x;
                bi[h] = sb.y;
                const uint32_t wh = w.x >> 8, xh = w.y >> 8;
                a[h][0] = w.x & 0x000f000fu;
                a[h][1] = w.x & 0x00f000f0u;
                a[h][2] = wh & 0x000f000fu;
                a[h][3] = wh & 0x00f000f0u;
                a[h][4] = w.y & 0x000f000fu;
                a[h][5] = w.y & 0x00f000f0u;
                a[h][6] = xh & 0x000f000fu;
                a[h][7] = xh & 0x00f000f0u;
              }
              float d[4];
              mma_f16_16816_zero(d, a[0][0], a[1][0], a[0][1], a[1][1], b0.x, b0.y);
              mma_f16_16816_add(d, a[0][2], a[1][2], a[0][3], a[1][3], b0.z, b0.w);
              mma_f16_16816_add(d, a[0][4], a[1][4], a[0][5], a[1][5], b1.x, b1.y);
              mma_f16_16816_add(d, a[0][6], a[1][6], a[0][7], a[1][7], b1.z, b1.w);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                acc[i][2 * h] = fmaf(bi[h], sm.x, fmaf(sc[h], d[2 * h], acc[i][2 * h]));
                if constexpr (TK > 1) acc[i][2 * h + 1] = fmaf(bi[h], sm.y, fmaf(sc[h], d[2 * h + 1], acc[i][2 * h + 1]));
              }
            }
          };
          const int ng = gb - ga - 4 * st;
          if (ng >= 4) {
#pragma unroll
            for (int q = 0; q < 4; ++q) group(q);
          } else {
            group(0);
            if (ng > 1) group(1);
            if (ng > 2) group(2);
          }
          xs += 4 * XG;
          ss += 4 * TK;
        }
        __syncwarp();  // the stage is read before it is loaded again
        if ((buf += STAGE) == D * STAGE) buf = 0;
      }
      // partial sums [batch][matrix][wr][slice][token][16 rows]
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int tok = 2 * t4 + (c & 1);
        if (tok < TK) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
            red[(((((((b * MT + i) << lwr) + wr) << f.lwk) + kslice) * TK + tok) << 4) + g8 + 8 * (c >> 1)] =
                acc[i][c] * (tscale[c & 1] * rs[i][c >> 1]);
        }
      }
    }
    // ---- sums over the slices, the gate, the output: rows fastest, then tiles of a position, tokens
    if (f.lck > 0)
      cluster_sync_all();
    else
      __syncthreads();
    constexpr int LROWS = 4, LTK = TK == 1 ? 0 : TK == 2 ? 1 : TK == 4 ? 2 : 3;
    const int outs = nb << (lwr + LROWS + LTK);
    const uint32_t red_addr = smem_u32(red);
    for (int o = tid + rank * kFewWarps * 32; o < outs; o += kFewWarps * 32 << f.lck) {
      const int r = o & (TROWS - 1), w = (o >> LROWS) & (wr_n - 1), rest = o >> (LROWS + lwr);
      const int tok = rest & (TK - 1), b = rest >> LTK;
      const int n = (((tile0 + b) << lwr) + w) * TROWS + r;
      if (n >= p.n_out || tok >= m) continue;
      float sum[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int at = ((((((b * MT + i) << lwr) + w) << f.lwk) * TK + tok) << 4) + r;
        float s = 0.0f;
        if (f.lck > 0) {
          for (int c = 0; c < 1 << f.lck; ++c) {
            const uint32_t base = dsmem_addr(red_addr, c) + at * 4;
#pragma unroll 4
            for (int k = 0; k < wk; ++k) s += ld_dsmem_f32(base + k * TK * 64);
          }
        } else {
#pragma unroll 4
          for (int k = 0; k < wk; ++k) s += red[at + k * TK * 16];
        }
        sum[i] = s;
      }
      const float y = GATED ? silu_mul(sum[0], sum[MT - 1]) : sum[0];
      p.out[(int64_t)(lo + tok) * p.out_stride + n] = p.bf16 ? f2h<true>(y) : f2h<false>(y);
    }
    if (f.lck > 0)
      cluster_sync_all();
    else
      __syncthreads();
    left -= nb;
    if ((tile0 += nb) == f.tiles) {
      tile0 = 0;
      ++it;
    }
  }
  if (*marked) few_store_nonfinite(f, TK);  // (every thread cleared it, and the last batch ended with a barrier)
}

constexpr int kFewSmem = 227 * 1024;
constexpr int kFewCluster = 8;  // CTAs, at most, that split the inputs

// Tokens of an item: all rows of a plain call; for experts twice their mean number (one with
// more reads its weights again).  One token of 64 experts: 10.1 us with items of one token, 10.3
// with items of eight; 16 tokens, items of four and eight: 42.9 and 45.1.
static int few_tokens(int rows, int experts, bool grouped) {
  const int64_t tok = grouped ? (2 * (int64_t)rows + experts - 1) / experts : rows;
  return tok <= 1 ? 1 : tok <= 2 ? 2 : tok <= 4 ? 4 : kFewTokens;
}

// Positions between two sums: 16 KB of sums.
constexpr int few_batch(bool gated, int tk) { return 16 / ((gated ? 2 : 1) * tk); }

// Shared memory of a CTA where `ck` of them split the inputs (quads of groups): the warps' rings, the
// activations with their group sums, the partial sums.
template <bool GATED, int TK>
static int64_t few_smem(int quads, int ck) {
  constexpr int MT = GATED ? 2 : 1;
  constexpr int64_t ring = kFewWarps * kFewDepth<GATED, TK> * MT * (kFewCodes + kFewPar);
  constexpr int64_t red = few_batch(GATED, TK) * MT * kFewWarps * TK * 64;
  return ring + (int64_t)((quads + ck - 1) / ck) * 4 * (128 + 4) * TK + (kFewWarps + 4) * 4 + red;
}

// Whether the largest cluster holds the activations of a call: up to 49152 inputs at 8 tokens (a gated
// pair 32768), 65536 at 4, 131072 at 2 and 264192 at 1.
static bool few_fits(int tok, bool gated, int n_in) {
  const int quads = ((n_in / 64) + 3) / 4;
  int64_t smem = 0;
  if (tok == 1) smem = gated ? few_smem<true, 1>(quads, kFewCluster) : few_smem<false, 1>(quads, kFewCluster);
  if (tok == 2) smem = gated ? few_smem<true, 2>(quads, kFewCluster) : few_smem<false, 2>(quads, kFewCluster);
  if (tok == 4) smem = gated ? few_smem<true, 4>(quads, kFewCluster) : few_smem<false, 4>(quads, kFewCluster);
  if (tok == 8) smem = gated ? few_smem<true, 8>(quads, kFewCluster) : few_smem<false, 8>(quads, kFewCluster);
  return smem <= kFewSmem;
}

template <bool GATED, int TK>
static cudaError_t launch_few_t(FewParams& f, cudaStream_t stream) {
  const LinearParams& p = f.p;
  // items a grouped call is likely to have, and has at most
  const int64_t likely = p.offsets != nullptr ? std::min(p.experts, p.rows) : (p.rows + TK - 1) / TK;
  const int64_t items = p.offsets != nullptr ? likely + p.rows / TK : likely;
  int dev = 0;
  const int sms = sm_count(&dev);
  if (sms == 0) return cudaErrorInvalidDevice;
  cudaError_t err = cudaSuccess;
  static unsigned long long done = 0;
  auto kfn = linear_few_kernel<GATED, TK>;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) {
    err = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem);
    if (err != cudaSuccess) return err;
    if (bit) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
  }
  f.batch = few_batch(GATED, TK);
  const int quads = p.pstride / 4;
  int ck = 1;
  while (ck < kFewCluster && few_smem<GATED, TK>(quads, ck) > kFewSmem) ck *= 2;
  if (few_smem<GATED, TK>(quads, ck) > kFewSmem) return cudaErrorNotSupported;  // (few_fits said it would)
  const int smem = static_cast<int>(few_smem<GATED, TK>(quads, ck));
  // Warps along the inputs: the split whose CTAs finish first, a position costing its groups and
  // about one and a half groups' time for the sums; a warp gets at least a whole stage.
  const int row_tiles = (p.n_out + 15) / 16;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(sms / ck * ck));
  cfg.blockDim = dim3(kFewWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ck;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ck > 1 ? 2 : 1;
  // CTAs, or clusters, that run at once: clusters lie within a GPC, so fewer of 4 or 8 fit than the SMs hold
  // (8 tokens 8192x28672 in clusters of 8: 55.8 us with 18 of them, 52.6 with the 15 that fit)
  int ctas = sms;
  if (ck > 1) {
    static int fit[64][4];  // by log2 of the cluster, once known
    const int i = ck == 2 ? 1 : ck == 4 ? 2 : 3;
    ctas = dev < 64 ? __atomic_load_n(&fit[dev][i], __ATOMIC_RELAXED) : 0;
    if (ctas == 0) {
      err = cudaOccupancyMaxActiveClusters(&ctas, kfn, &cfg);
      if (err != cudaSuccess) return err;
      if (ctas == 0) return cudaErrorNotSupported;
      if (dev < 64) __atomic_store_n(&fit[dev][i], ctas, __ATOMIC_RELAXED);
    }
  }
  double best = 0.0;
  int wk = 1;
  for (int k = 1; k <= kFewWarps; k *= 2) {
    if (k > 1 && quads < k * ck) break;
    const int wr = kFewWarps / k;
    const int64_t positions = (int64_t)((row_tiles + wr - 1) / wr) * likely;
    const double rounds = static_cast<double>((positions + ctas - 1) / ctas);
    const double cost = rounds * ((quads + k * ck - 1) / (k * ck) * 4 + 1.5);
    if (k == 1 || cost < best) {
      best = cost;
      wk = k;
    }
  }
  auto log2_of = [](int v) { return 31 - __builtin_clz(v); };
  f.lwk = log2_of(wk);
  f.lck = log2_of(ck);
  const int wr = kFewWarps / wk;
  f.tiles = (row_tiles + wr - 1) / wr;
  if (items * f.tiles > INT_MAX) return cudaErrorNotSupported;
  cfg.gridDim = dim3(static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(items * f.tiles, ctas)) * ck));
  return cudaLaunchKernelEx(&cfg, kfn, f);
}

template <bool GATED>
static cudaError_t launch_few(FewParams& f, int tok, cudaStream_t stream) {
  switch (tok) {
    case 1: return launch_few_t<GATED, 1>(f, stream);
    case 2: return launch_few_t<GATED, 2>(f, stream);
    case 4: return launch_few_t<GATED, 4>(f, stream);
    default: return launch_few_t<GATED, 8>(f, stream);
  }
}

// Which kernel.  One matrix: this one up to 8 tokens (4096x4096 at 8: 7.6 us, the tiles 12.8; 28672x8192
// 42 and 39); a gated pair, whose sums at 8 tokens cost more than the tiles' longer start once the
// pair is large, up to 4 of those (8 tokens, 33 million weights: 13.1 and 14.5 us; 117 million: 29.2 and
// 24.4).  Experts: up to a mean of two rows (a grouped call's counts are on the device; 64 experts
// of 2048x1408: mean 2 31.8 and 30.0 us, mean 1 24.1 and 25.4; 8 of 4096x14336 gated: mean 2 103
// and 109, mean 3 143 and 111).  In each case only where the activations fit.
bool linear_uses_tensor_tiles(int rows, int experts, bool grouped, bool gated, int n_out, int n_in) {
  if (grouped ? (rows - 1) / experts >= 2
              : rows > kFewTokens || (gated && rows > 4 && 2LL * n_out * n_in > 56000000))
    return true;
  return !few_fits(few_tokens(rows, experts, grouped), gated, n_in);
}

cudaError_t launch_linear_few(const LinearParams& p, cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  FewParams f{};
  f.p = p;
  const int tok = few_tokens(p.rows, p.experts, p.offsets != nullptr);
  return p.codes[1] != nullptr ? launch_few<true>(f, tok, stream) : launch_few<false>(f, tok, stream);
}

}  // namespace am
