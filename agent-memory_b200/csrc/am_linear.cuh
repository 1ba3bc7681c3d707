// Launch parameters and device helpers of the 4-bit linear layers and the expert routing.
#pragma once

#include "am_common.cuh"

namespace am {

// y = x W^T over 4-bit weights, plain or gated (up != null), for one matrix or per expert.
struct LinearParams {
  const uint32_t* codes[2];   // [0] the matrix (gate), [1] its partner (up) or null
  const uint32_t* params[2];  // [rows of weights][pstride]: half2 (scale * 2^(24-e), bias * 2^(20-e))
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
  uint64_t wait_ns;           // limit of the bounded waits
  // tensor-tile kernel: the activations as fp16 rows [rows][n_in] in its input order and their
  // powers of two, in the caller's workspace; tensor maps of them and of the codes
  uint16_t* xh;
  float* xscale;
  alignas(64) CUtensorMap tmap_w[2];
  alignas(64) CUtensorMap tmap_x;
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

// The x row that output row r (of pair order[r]) is made from; -1 (and the status bit) for a bad order
// entry.
__device__ __forceinline__ int source_row_of(const LinearParams& p, int pair) {
  if (p.order == nullptr) return pair;
  const int t = pair / p.top_k;
  if (pair < 0 || t >= p.x_rows) {
    flag_status(p.status, AM_STATUS_BAD_POSITION);
    return -1;
  }
  return t;
}
__device__ __forceinline__ int source_row(const LinearParams& p, int r) {
  return source_row_of(p, p.order != nullptr ? p.order[r] : r);
}

__device__ __forceinline__ uint32_t hfma2_bits(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// The four weight pairs of one word: inputs (0, 4), (1, 5), (2, 6), (3, 7) of its eight.  BITS: the bits of
// a code that count.
template <uint32_t BITS = 15>
__device__ __forceinline__ void dequant_word(uint32_t w, uint32_t s24, uint32_t s20, uint32_t b, uint32_t (&o)[4]) {
  constexpr uint32_t EVEN = BITS * 0x00010001u, ODD = BITS * 0x00100010u;
  const uint32_t h = w >> 8;
  o[0] = hfma2_bits(w & EVEN, s24, b);
  o[1] = hfma2_bits(w & ODD, s20, b);
  o[2] = hfma2_bits(h & EVEN, s24, b);
  o[3] = hfma2_bits(h & ODD, s20, b);
}

// How the tensor-core tiles round a weight scale * code + bias to fp16.  PARTS == 1: once, an error of
// 1.8e-4 of the product (normal weights) beside the output's own rounding of 2.1e-4 in fp16 and
// 1.7e-3 in bf16.  A gated fp16 output takes that error twice, 1.6 times its own rounding in all:
// there a weight is the sum of two parts with an MMA each, scale * (code / 4 * 4 - 8), which is exact,
// and scale * (code % 4) + (bias + 8 * scale), together 1.0e-4: 1.2 times.
constexpr int weight_parts(bool gated, bool bf16) { return gated && !bf16 ? 2 : 1; }

// The 64 weights of a group's row as fp16 pairs: part `part` of PARTS.
template <int PARTS>
__device__ __forceinline__ void dequant_group(const uint4& w0, const uint4& w1, uint32_t params, int part,
                                              uint32_t (&o)[32]) {
  const uint32_t s24 = __byte_perm(params, params, 0x1010);
  uint32_t b = hfma2_bits(__byte_perm(params, params, 0x3232), 0x00100010u, 0x80008000u);  // * 2^-20
  const uint32_t s20 = hfma2_bits(s24, 0x2c002c00u, 0x80008000u);  // * 2^-4
  // 8 * scale = s24 * 2^-21
  if (PARTS == 2) b = part == 0 ? hfma2_bits(s24, 0x00080008u, b) : hfma2_bits(s24, 0x80088008u, 0x80008000u);
  const uint32_t words[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t d[4];
    if (PARTS == 1)
      dequant_word(words[j], s24, s20, b, d);
    else if (part == 0)
      dequant_word<3>(words[j], s24, s20, b, d);
    else
      dequant_word<12>(words[j], s24, s20, b, d);
#pragma unroll
    for (int q = 0; q < 4; ++q) o[4 * j + q] = d[q];
  }
}

// Activations under a power of two: the largest |bf16| of eight as its 15 bits, the exponent that
// takes a row's largest to [2^14, 2^15) (zero rows and the smallest numbers: 2^-126), and eight
// inputs as fp16 pairs (0, 4), (1, 5), (2, 6), (3, 7), the order of dequant_word.
__device__ __forceinline__ uint32_t max_abs_bits(uint4 u) {
  const uint32_t a = __vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu);
  const uint32_t b = __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu);
  const uint32_t c = __vmaxu2(a, b);
  return max(c & 0xffffu, c >> 16);
}
__device__ __forceinline__ int row_exponent(uint32_t max_bits) {
  return max(min(max(static_cast<int>(max_bits >> 7), 1), 254) - 127 - 14, -126);
}
// 2^e for e in [-126, 127].
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }
// The same for fp16 bits.
__device__ __forceinline__ int row_exponent_f16(uint32_t max_bits) {
  const float v = fminf(__half2float(__ushort_as_half(static_cast<uint16_t>(max_bits))), 65504.0f);
  return v > 0.0f ? ilogbf(v) - 14 : 0;
}
__device__ __forceinline__ uint4 permute_f16(uint4 u) {
  return make_uint4(__byte_perm(u.x, u.z, 0x5410), __byte_perm(u.x, u.z, 0x7632), __byte_perm(u.y, u.w, 0x5410),
                    __byte_perm(u.y, u.w, 0x7632));
}
__device__ __forceinline__ uint4 permute_bf16(uint4 u, float f) {
  auto lo = [f](uint32_t w) { return __uint_as_float(w << 16) * f; };
  auto hi = [f](uint32_t w) { return __uint_as_float(w & 0xffff0000u) * f; };
  return make_uint4(pack_half2(lo(u.x), lo(u.z)), pack_half2(hi(u.x), hi(u.z)), pack_half2(lo(u.y), lo(u.w)),
                    pack_half2(hi(u.y), hi(u.w)));
}

// Work items of a call: pieces of at most `tok` rows of one expert.  The warp's lanes agree.
__device__ __forceinline__ int count_items(const LinearParams& p, int tok) {
  if (p.offsets == nullptr) return (p.rows + tok - 1) / tok;
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int e = lane; e < p.experts; e += 32) {
    int a, b;
    expert_range(p, e, a, b);
    n += (b - a + tok - 1) / tok;
  }
  return __reduce_add_sync(0xffffffffu, n);
}

// Item `item`: rows [lo, hi) of one expert, whose rows are cut evenly into as few items as hold them.
// Returns the expert, or -1 past the last item.  All lanes of a warp call it.
__device__ __forceinline__ int find_item(const LinearParams& p, int item, int tok, int& lo, int& hi) {
  if (p.offsets == nullptr) {
    const int n = (p.rows + tok - 1) / tok, per = n > 0 ? (p.rows + n - 1) / n : 0;
    lo = item * per;
    hi = min(lo + per, p.rows);
    return item < n ? 0 : -1;
  }
  // each warp scans the experts, 32 at a time
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    int a = 0, b = 0;
    if (e0 + lane < p.experts) expert_range(p, e0 + lane, a, b);
    const int n = (b - a + tok - 1) / tok;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    if (item < base + total) {
      const bool mine = item >= base + incl - n && item < base + incl;
      const int src = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
      const int per = n > 0 ? (b - a + n - 1) / n : 0;
      const int first = a + (item - (base + incl - n)) * per;
      lo = __shfl_sync(0xffffffffu, first, src);
      hi = __shfl_sync(0xffffffffu, min(first + per, b), src);
      return e0 + src;
    }
    base += total;
  }
  return -1;
}

// silu(g) * u by the fast exponential (off by up to 2 + 1.2 |g| ulp) and division (2 ulp): 2^-18 of
// silu at g = -20, beside the output's own rounding of 2^-12 (fp16) or 2^-9.  Below g = -87.3 it
// is 0, where |silu| is less than 1.1e-36.
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

// Two outputs as a pair of the call's type.
__device__ __forceinline__ uint32_t pack_out(const LinearParams& p, float x, float y) {
  if (p.bf16) {
    const __nv_bfloat162 z = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&z);
  }
  return pack_half2(x, y);
}

// ---- tokens with infinite or NaN activations
// The kernels' sums are not what the formula gives there: a scale and a bias meet an infinity apart, a
// weight that rounds to zero or is the sum of two parts makes it a NaN.  A kernel that has seen such
// a token stores its outputs again behind the others.

// The least fp16 or bf16 bits (without the sign) that are no finite number.
__device__ __forceinline__ uint32_t nonfinite_bits(const LinearParams& p) { return p.bf16 ? 0x7f80u : 0x7c00u; }

// The product of weight row `wrow` with x row `x_row` as far as infinite and NaN activations determine it
// (under the weight row's power of two); false where there is none.
__device__ __forceinline__ bool nonfinite_sum(const LinearParams& p, int matrix, int64_t wrow, int x_row, float& sum) {
  const uint16_t* x = p.x + (int64_t)x_row * p.x_stride;
  const uint32_t* codes = p.codes[matrix] + wrow * (p.n_in / 8);
  const uint32_t* params = p.params[matrix] + wrow * p.pstride;
  const uint32_t limit = nonfinite_bits(p);
  bool any = false;
  sum = 0.0f;
#pragma unroll 1
  for (int k = 0; k < p.n_in; k += 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(x + k);
    if (max_abs_bits(u) < limit) continue;
    any = true;
    const uint32_t v = params[k >> 6];
    const float2 sb = __half22float2(*reinterpret_cast<const __half2*>(&v));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = (w[j >> 1] >> (16 * (j & 1))) & 0xffffu;
      if ((bits & 0x7fffu) < limit) continue;
      const float code = static_cast<float>((codes[k >> 3] >> (4 * j)) & 15u);
      sum += h2f_rt(static_cast<uint16_t>(bits), p.bf16) * fmaf(code * 0x1p-24f, sb.x, sb.y * 0x1p-20f);
    }
    if (isnan(sum)) break;  // (and stays so)
  }
  return any;
}

// Stores again such tokens among output rows [lo, hi), weight rows [n0, n1) of expert e, by the whole
// CTA.  scale (or null): the tokens' powers of two from row lo on; linear_rows_kernel gives such a
// token a NaN.
__device__ __forceinline__ void store_nonfinite(const LinearParams& p, const float* scale, int e, int lo, int hi, int n0,
                                                int n1) {
  for (int r = lo + static_cast<int>(threadIdx.x >> 5); r < hi; r += blockDim.x >> 5) {
    if (scale != nullptr && !isnan(scale[r - lo])) continue;
    const int x_row = source_row(p, r);
    if (x_row < 0) continue;
    for (int n = n0 + static_cast<int>(threadIdx.x & 31); n < min(n1, p.n_out); n += 32) {
      float y, u;
      if (!nonfinite_sum(p, 0, (int64_t)e * p.n_out + n, x_row, y)) break;
      if (p.codes[1] != nullptr) {
        nonfinite_sum(p, 1, (int64_t)e * p.n_out + n, x_row, u);
        y = silu_mul(y, u);
      }
      p.out[(int64_t)r * p.out_stride + n] = p.bf16 ? f2h<true>(y) : f2h<false>(y);
    }
  }
}

// The same for the tiles of CTA `cta` of `ctas`: items of `tok` rows x row_tiles tiles, of which this CTA
// makes weight rows [row0, row0 + rows) of every tile_rows, and tokens rank / ck to (rank + 1) / ck.
__device__ __forceinline__ void store_nonfinite_tiles(const LinearParams& p, int tok, int row_tiles, int tile_rows,
                                                          int row0, int rows, int cta, int ctas, int rank, int ck) {
  griddep_wait();
  const int tiles = count_items(p, tok) * row_tiles;
  for (int tile = cta; tile < tiles; tile += ctas) {
    int lo, hi;
    const int e = find_item(p, tile / row_tiles, tok, lo, hi);
    const int n0 = tile % row_tiles * tile_rows + row0, t0 = lo + (hi - lo) * rank / ck;
    store_nonfinite(p, p.xscale + t0, e, t0, lo + (hi - lo) * (rank + 1) / ck, n0, n0 + rows);
  }
}

// Bytes between tokens of a warp's 32 output rows in shared memory: 64, and 16 against bank conflicts.
constexpr int kOutPitch = 80;

// A warp writes output rows row0 .. row0 + 31 (weight rows) of 8 * BLOCKS tokens from `tok` on: q[j][i]
// holds in mma fragments (thread (g, t): weight row 8 i + g, tokens 8 j + 2 t, + 1) pairs of
// tokens.  They are transposed through 8 * BLOCKS * kOutPitch bytes of shared memory at `so`; a
// token's 32 rows leave as 64 bytes.
template <int BLOCKS>
__device__ __forceinline__ void store_tokens(const LinearParams& p, uint8_t* so, const uint32_t (&q)[BLOCKS][4], int tok,
                                             int hi, int row0) {
  const int lane = threadIdx.x & 31;
  const bool wide = (p.out_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  const int left = p.n_out - (row0 + (lane & 3) * 8);  // from this lane's 8 output rows on
  const uint32_t st = smem_u32(so) + (lane & 7) * kOutPitch + (lane >> 3) * 16;
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) stsm_x4_trans(st + j * 8 * kOutPitch, q[j][0], q[j][1], q[j][2], q[j][3]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
    const int at = tok + j * 8 + (lane >> 2);
    const uint4 d = *reinterpret_cast<const uint4*>(so + (j * 8 + (lane >> 2)) * kOutPitch + (lane & 3) * 16);
    if (at < hi && left > 0) {
      uint16_t* dst = p.out + (int64_t)at * p.out_stride + row0 + (lane & 3) * 8;
      if (wide && left >= 8) {
        *reinterpret_cast<uint4*>(dst) = d;
      } else {
        const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) dst[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
  __syncwarp();
}

// The same for 16 output rows of 16 tokens: q[j][h] are rows 8 h .. 8 h + 7 of tokens 8 j .. 8 j + 7, through
// 16 * kOutPitch16 bytes at `so`; a token's 16 rows leave as 32 bytes.
constexpr int kOutPitch16 = 48;
__device__ __forceinline__ void store_tokens_16(const LinearParams& p, uint8_t* so, const uint32_t (&q)[2][2], int tok,
                                                int hi, int row0) {
  const int lane = threadIdx.x & 31;
  const bool wide = (p.out_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  const int left = p.n_out - (row0 + (lane & 1) * 8);
  stsm_x4_trans(smem_u32(so) + ((lane >> 4) * 8 + (lane & 7)) * kOutPitch16 + ((lane >> 3) & 1) * 16, q[0][0], q[0][1],
                q[1][0], q[1][1]);
  __syncwarp();
  const int at = tok + (lane >> 1);
  const uint4 d = *reinterpret_cast<const uint4*>(so + (lane >> 1) * kOutPitch16 + (lane & 1) * 16);
  if (at < hi && left > 0) {
    uint16_t* dst = p.out + (int64_t)at * p.out_stride + row0 + (lane & 1) * 8;
    if (wide && left >= 8) {
      *reinterpret_cast<uint4*>(dst) = d;
    } else {
      const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) dst[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
    }
  }
  __syncwarp();
}

// Position in a ring of N buffers and the parity of its current round.
template <int N>
struct Ring {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      ph ^= 1u;
    }
  }
};

}  // namespace am
