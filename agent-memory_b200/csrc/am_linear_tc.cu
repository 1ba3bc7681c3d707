// Linear layers over 4-bit weights for more than a few tokens: tcgen05 tensor tiles.
//
// y^T = W x^T: weight rows are the M side (128 lanes of TMEM), tokens the N side, so a weight is
// dequantized once for up to 128 tokens, straight into the TMEM operand.
//
// 1. linear_rows_kernel writes the activations as fp16 rows of the workspace, in output order (a
//    grouped call's tokens are gathered here: tile::gather4 loads in the tile kernel measured
//    2.5x slower than plain boxes, ~75 clocks per four rows), each under a power of two (exact
//    for fp16 and bf16 values) and with its inputs in the order in which the dequantization
//    below produces the weights.
// 2. linear_tiles_kernel: a CTA owns two 128-row weight tiles (plain: 256 rows of the matrix;
//    gated: 128 rows of each matrix) and NT tokens of one matrix or expert.
//    * one thread streams the codes (TMA, 128 rows x 256 inputs a box, 128-byte swizzle), one
//      the activations (TMA boxes of NT rows x 64 inputs);
//    * warps 0-7 dequantize: a thread owns a weight row; 64 codes a step become 32 registers of
//      fp16 pairs (9 operations for 8 weights, see am_linear.cu) and go to TMEM with one
//      tcgen05.st -- no shared-memory round trip, and the MMA reads its A operand there;
//    * two threads, one a weight tile, issue tcgen05.mma (kind::f16, M = 128, N = NT, K = 16).
//    The accumulators are read back by the dequantization warps, scaled by the row's and the
//    token's powers of two, gated, rounded once and stored.  A CTA walks the tiles with stride
//    gridDim.x; the loads of its next tile run during the output of the last one.
//    With few tiles the inputs are split over the CTAs of a cluster, whose fp32 sums meet in
//    distributed shared memory, in rank order.
// Every wait is bounded (LinearParams::wait_ns); on timeout the kernel flags AM_STATUS_TIMEOUT,
// lets its copies and MMAs in flight finish, frees its TMEM and returns.
//
// The codes and parameters are read before griddepcontrol.wait: linear_rows_kernel starts only
// when everything before it in the stream is complete (it is launched without programmatic
// serialization), and it writes nothing but the activations.
#include <algorithm>
#include <climits>

#include "am_internal.h"
#include "am_linear.cuh"
#include "am_tcgen05.cuh"

namespace am {

// ---------------------------------------------------------------- activations
__global__ void __launch_bounds__(128) linear_rows_kernel(const __grid_constant__ LinearParams p) {
  __shared__ uint32_t wmax[4];
  griddep_launch_dependents();
  const int row = blockIdx.x, tid = threadIdx.x;
  const int from = source_row(p, row);
  const uint4* src = reinterpret_cast<const uint4*>(p.x + (int64_t)max(from, 0) * p.x_stride);
  uint4* dst = reinterpret_cast<uint4*>(p.xh + (int64_t)row * p.n_in);
  const int vecs = p.n_in / 8;
  if (from < 0) {
    for (int i = tid; i < vecs; i += 128) dst[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) p.xscale[row] = 1.0f;
    return;
  }
  if (!p.bf16) {
    for (int i = tid; i < vecs; i += 128) {
      const uint4 u = src[i];
      dst[i] = permute_f16(u);
    }
    if (tid == 0) p.xscale[row] = 1.0f;
    return;
  }
  uint32_t mx = 0;
  for (int i = tid; i < vecs; i += 128) mx = max(mx, max_abs_bits(src[i]));
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((tid & 31) == 0) wmax[tid >> 5] = mx;
  __syncthreads();
  mx = max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3]));
  const int ex = row_exponent(mx);
  const float inv = exp2f(static_cast<float>(-ex));
  for (int i = tid; i < vecs; i += 128) dst[i] = permute_bf16(src[i], inv);
  if (tid == 0) p.xscale[row] = exp2f(static_cast<float>(ex));
}

// ---------------------------------------------------------------- tiles
template <int NT>
struct TilesLayout {
  // 128 tokens: one CTA a SM, 512 TMEM columns; fewer: two CTAs a SM of 256 columns each
  static constexpr int CTAS = NT == 128 ? 1 : 2;
  static constexpr uint32_t TMEM_COLS = 512 / CTAS;
  static constexpr int SP = NT == 128 ? 2 : 1;             // slabs (64 inputs) of a pipeline step
  static constexpr int CS = NT == 128 ? 3 : 2;             // code stages (256 rows x 256 inputs)
  static constexpr int XS = NT == 128 ? 3 : (NT == 64 ? 5 : 8);  // activation steps (NT x 64 SP inputs)
  static constexpr int AB = (TMEM_COLS - 2 * NT) / (64 * SP);    // TMEM operand buffers (2 tiles x 32 SP columns)
  static constexpr int DW = 8 * SP;                        // dequantization warps: 8 a slab of the step
  static constexpr int THREADS = 32 * (DW + 4);            // + codes, activations, two MMA warps
  static constexpr int CSTAGE = 2 * 128 * 128;
  static constexpr int XSLAB = NT * 128;
  static constexpr int OFF_C = 0;
  static constexpr int OFF_X = OFF_C + CS * CSTAGE;
  static constexpr int OFF_END = OFF_X + XS * SP * XSLAB;
  static constexpr int RED = 2 * NT * 128 * 4;             // fp32 sums of a split (over the rings)
  static constexpr int OFF_OUT = OFF_END > RED ? OFF_END : RED;  // 1 KB a dequantization warp
  static constexpr int OFF_SCALE = OFF_OUT + DW * 1024;    // two tiles' token scales
  static constexpr int OFF_BAR = OFF_SCALE + 2 * NT * 4;
  static constexpr int B_CFULL = 0, B_CEMPTY = CS, B_XFULL = 2 * CS, B_XEMPTY = B_XFULL + XS;
  static constexpr int B_AFULL = B_XEMPTY + XS, B_AEMPTY = B_AFULL + AB, B_DFULL = B_AEMPTY + AB;
  static constexpr int B_DEMPTY = B_DFULL + 1, B_SFULL = B_DEMPTY + 1, B_SEMPTY = B_SFULL + 2;
  static constexpr int B_DRAIN = B_SEMPTY + 2, B_COUNT = B_DRAIN + 2;
  static constexpr int SMEM = OFF_BAR + B_COUNT * 8 + 16;
  static constexpr int A_COL = 2 * NT;  // D[tile] at tile * NT, A[buffer][tile] at A_COL + 32 SP (2 b + tile)
  static_assert(AB >= 2, "the operand needs two buffers");
  static_assert((SMEM + 1024) * CTAS <= 233472 && SMEM <= 232448, "shared memory of a SM");
  // Arrivals that complete a phase of barrier i.
  static __device__ int arrivals(int i) {
    if (i >= B_CEMPTY && i < B_CEMPTY + CS) return DW;
    if (i >= B_XEMPTY && i < B_XEMPTY + XS) return 2;
    if (i >= B_AFULL && i < B_AFULL + AB) return DW;
    if (i >= B_AEMPTY && i < B_AEMPTY + AB) return 2;
    if (i == B_DFULL) return 2;
    if (i == B_DEMPTY) return DW;
    if (i >= B_SEMPTY && i < B_SEMPTY + 2) return DW;
    return 1;
  }
};

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

struct TilesParams {
  LinearParams p;
  int32_t ck;         // CTAs of a cluster that split the inputs (then a CTA has one tile)
  int32_t row_tiles;  // tiles of CTA_ROWS weight rows
};

template <int NT, bool GATED>
__global__ void __launch_bounds__(TilesLayout<NT>::THREADS, TilesLayout<NT>::CTAS)
    linear_tiles_kernel(const __grid_constant__ TilesParams f) {
  using LY = TilesLayout<NT>;
  constexpr int CS = LY::CS, XS = LY::XS, AB = LY::AB, SP = LY::SP, DW = LY::DW;
  constexpr int CODES_WARP = DW, X_WARP = DW + 1, MMA_WARP = DW + 2;
  constexpr int STEPS = 4 / SP;  // steps of a code stage
  const LinearParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s_base = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + LY::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + LY::OFF_BAR + LY::B_COUNT * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + LY::OFF_BAR + LY::B_COUNT * 8 + 4);
  float* tok_scale = reinterpret_cast<float*>(smem + LY::OFF_SCALE);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  auto wait = [&](int i, uint32_t parity) { return wait_or_abort(bar(i), parity, p.wait_ns, abort_flag); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  griddep_launch_dependents();
  if (s_base & 1023u) {  // swizzled tiles need a 1024-byte aligned window (the whole grid returns)
    if (tid == 0) flag_status(p.status, AM_STATUS_BAD_POSITION);
    return;
  }
  const int rank = f.ck > 1 ? static_cast<int>(blockIdx.x) % f.ck : 0;
  const int first = static_cast<int>(blockIdx.x) / f.ck, step = static_cast<int>(gridDim.x) / f.ck;
  const int tiles = count_items(p, NT) * f.row_tiles;
  if (first >= tiles) return;  // the whole cluster
  constexpr int CTA_ROWS = GATED ? 128 : 256;
  // this CTA's inputs: quads of groups [q0, q1), slabs of 64 inputs, steps of SP slabs
  const int quads = p.pstride >> 2;
  const int q0 = quads * rank / f.ck, q1 = quads * (rank + 1) / f.ck;
  const int slabs = min(q1 * 4, p.groups) - q0 * 4;
  const int steps = (slabs + SP - 1) / SP;

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "r"(LY::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  } else if (warp == CODES_WARP) {
    for (int i = lane; i < LY::B_COUNT; i += 32) mbar_init(bar(i), LY::arrivals(i));
    if (lane == 0) *abort_flag = 0;
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

  int issued_c = 0, issued_x = 0;  // loads issued (their own threads' counts)
  bool mma_issued = false;
  bool ok = true;
  if (warp == CODES_WARP) {
    Ring<CS> ring;
    for (int tile = first; tile < tiles; tile += step) {
      int lo, hi;
      const int e = find_item(p, tile / f.row_tiles, NT, lo, hi);
      const int y = e * p.n_out + tile % f.row_tiles * CTA_ROWS;
      if (lane == 0) {
        for (int c = q0; c < q1; ++c) {
          ok = wait(LY::B_CEMPTY + ring.s, ring.ph ^ 1u);
          if (!ok) break;
          const uint32_t full = bar(LY::B_CFULL + ring.s), dst = s_base + LY::OFF_C + ring.s * LY::CSTAGE;
          mbar_arrive_expect_tx(full, LY::CSTAGE);
          tma_load_2d(dst, &p.tmap_w[0], c * 128, y, full);
          tma_load_2d(dst + LY::CSTAGE / 2, &p.tmap_w[GATED ? 1 : 0], c * 128, GATED ? y : y + 128, full);
          ++issued_c;
          ring.next();
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
    }
  } else if (warp == X_WARP) {
    griddep_wait();  // the activations are written
    Ring<XS> ring;
    int k = 0;
    for (int tile = first; tile < tiles && ok; tile += step, ++k) {
      int lo, hi;
      find_item(p, tile / f.row_tiles, NT, lo, hi);
      for (int i = 0; i < steps; ++i) {
        ok = __all_sync(0xffffffffu, wait(LY::B_XEMPTY + ring.s, ring.ph ^ 1u));
        if (!ok) break;
        const uint32_t full = bar(LY::B_XFULL + ring.s), dst = s_base + LY::OFF_X + ring.s * SP * LY::XSLAB;
        const int n = min(SP, slabs - i * SP);
        if (lane == 0) {
          mbar_arrive_expect_tx(full, n * LY::XSLAB);
          for (int s = 0; s < n; ++s)
            tma_load_2d(dst + s * LY::XSLAB, &p.tmap_x, (q0 * 4 + i * SP + s) * 128, lo, full);
        }
        ++issued_x;
        ring.next();
        if (i == min(XS, steps) - 1) {  // behind the first loads: the tokens' powers of two
          const int b = k & 1;
          ok = __all_sync(0xffffffffu, wait(LY::B_SEMPTY + b, ((k >> 1) & 1) ^ 1));
          if (!ok) break;
          for (int j = lane; j < NT; j += 32) tok_scale[b * NT + j] = lo + j < hi ? p.xscale[lo + j] : 0.0f;
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(LY::B_SFULL + b));
        }
      }
    }
  } else if (warp >= MMA_WARP) {
    // Two issuing threads, one a weight tile: the waits and commits of one hide behind the MMAs
    // of the other (one thread for both left the tensor pipe idle half of the time).
    if (lane == 0) {
      constexpr uint32_t ID = tc::idesc(128, NT, false);
      const int t = warp - MMA_WARP;
      const uint32_t d = tmem + t * NT;
      Ring<XS> xr;
      Ring<AB> ar;
      uint32_t dph = 1;
      for (int tile = first; tile < tiles && ok; tile += step, dph ^= 1u) {
        ok = wait(LY::B_DEMPTY, dph);
        for (int i = 0; i < steps && ok; ++i) {
          ok = wait(LY::B_XFULL + xr.s, xr.ph) && wait(LY::B_AFULL + ar.s, ar.ph);
          if (!ok) break;
          tc::fence_after();
          const uint64_t xd = tc::sdesc(s_base + LY::OFF_X + xr.s * SP * LY::XSLAB, 16, 1024);
          const uint32_t a = tmem + LY::A_COL + ar.s * 64 * SP + t * 32;
          // (descriptor addresses count 16-byte units: 32 bytes of a swizzled row are 16 inputs)
          tc::mma_ts(d, a, xd, ID, i > 0 ? 1u : 0u);
#pragma unroll
          for (int ks = 1; ks < 4; ++ks) tc::mma_ts(d, a + ks * 8, xd + ks * 2, ID, 1u);
          if (SP == 2 && 2 * i + 1 < slabs) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) tc::mma_ts(d, a + 64 + ks * 8, xd + LY::XSLAB / 16 + ks * 2, ID, 1u);
          }
          mma_issued = true;
          tc::commit(bar(LY::B_XEMPTY + xr.s));
          tc::commit(bar(LY::B_AEMPTY + ar.s));
          xr.next();
          ar.next();
        }
        if (ok) tc::commit(bar(LY::B_DFULL));
      }
    }
  } else {
    // ---- dequantization: one weight row of tile t a thread, slab `group` of every step.  A slab's
    // store into TMEM completes while the next one is dequantized, and only then is it handed
    // to the MMA threads.
    const int group = warp >> 3, t = (warp >> 2) & 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t a_base = tmem + LY::A_COL + group * 64 + t * 32 + lane_base;
    Ring<CS> cr;
    Ring<AB> ar;
    int stored = -1;  // buffer of the store in flight
    auto publish = [&]() {
      if (stored >= 0) {
        tc::tmem_wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(LY::B_AFULL + stored));
      }
    };
    int k = 0;
    for (int tile = first; tile < tiles && ok; tile += step, ++k) {
      int lo, hi;
      const int e = find_item(p, tile / f.row_tiles, NT, lo, hi);
      const int n0 = tile % f.row_tiles * CTA_ROWS;
      const int64_t wrow = (int64_t)e * p.n_out + min(n0 + (GATED ? 0 : t * 128) + r, p.n_out - 1);
      const uint4* prow = reinterpret_cast<const uint4*>(p.params[GATED ? t : 0] + wrow * p.pstride);
      uint4 pv = __ldg(prow + q0);
      for (int c = q0; c < q1; ++c) {
        const uint4 pnext = __ldg(prow + min(c + 1, q1 - 1));
        ok = __all_sync(0xffffffffu, wait(LY::B_CFULL + cr.s, cr.ph));
        if (!ok) break;
        const uint8_t* crow = smem + LY::OFF_C + cr.s * LY::CSTAGE + t * (LY::CSTAGE / 2) + r * 128;
        const uint32_t pw[4] = {pv.x, pv.y, pv.z, pv.w};
        const int in_stage = min(4, slabs - 4 * (c - q0));
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          if (st * SP >= in_stage) break;
          const int s = st * SP + group;
          uint32_t o[32];
          if (s < in_stage) {
            const uint4 w0 = *reinterpret_cast<const uint4*>(crow + (((2 * s) ^ (r & 7)) << 4));
            const uint4 w1 = *reinterpret_cast<const uint4*>(crow + (((2 * s + 1) ^ (r & 7)) << 4));
            const uint32_t ps = SP == 1 || group == 0 ? pw[st * SP] : pw[(st * SP + 1) & 3];
            const uint32_t s24 = __byte_perm(ps, ps, 0x1010), bb = __byte_perm(ps, ps, 0x3232);
            const uint32_t s20 = hfma2_bits(s24, 0x2c002c00u, 0x80008000u);
            const uint32_t words[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint32_t d[4];
              dequant_word(words[j], s24, s20, bb, d);
#pragma unroll
              for (int q = 0; q < 4; ++q) o[4 * j + q] = d[q];
            }
          }
          publish();
          ok = __all_sync(0xffffffffu, wait(LY::B_AEMPTY + ar.s, ar.ph ^ 1u));
          if (!ok) break;
          tc::fence_after();
          if (s < in_stage) tc::tmem_st32_nowait(a_base + ar.s * 64 * SP, o);
          stored = ar.s;
          ar.next();
        }
        if (!ok) break;
        __syncwarp();  // the stage's codes are in registers
        if (lane == 0) mbar_arrive(bar(LY::B_CEMPTY + cr.s));
        cr.next();
        pv = pnext;
      }
      if (!ok) break;
      publish();
      stored = -1;
      const int b = k & 1;
      ok = __all_sync(0xffffffffu, wait(LY::B_DFULL, k & 1) && wait(LY::B_SFULL + b, (k >> 1) & 1));
      if (!ok) break;
      tc::fence_after();
      if (f.ck > 1) {
        // ---- fp32 sums to shared memory, [tile][token][128 rows]
        constexpr int COLS = NT / SP;
        float* red = reinterpret_cast<float*>(smem) + t * NT * 128 + r;
#pragma unroll 1
        for (int cb = group * COLS; cb < (group + 1) * COLS; cb += 16) {
          float v[16];
          tc::tmem_ld16(tmem + t * NT + cb + lane_base, v);
#pragma unroll
          for (int j = 0; j < 16; ++j) red[(cb + j) * 128] = v[j];
        }
        break;
      }
      // ---- output: lane = weight row, columns = tokens; 16 tokens at a time through the warp's
      // own shared memory, so that a token's 32 rows leave as 64 bytes
      constexpr int PARTS = GATED ? DW / 4 : DW / 8;  // warps that share a lane quarter (and tile)
      constexpr int COLS = NT / PARTS;
      const int part = GATED ? warp >> 2 : group;
      const int row0 = n0 + (GATED ? 0 : t * 128) + quarter * 32;
      const int64_t wr = (int64_t)e * p.n_out + min(row0 + lane, p.n_out - 1);
      const float rs0 = p.row_scale[0][wr], rs1 = GATED ? p.row_scale[1][wr] : 0.0f;
      uint16_t* so = reinterpret_cast<uint16_t*>(smem + LY::OFF_OUT + warp * 1024);
      const bool wide = (p.out_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
#pragma unroll 1
      for (int cb = part * COLS; cb < (part + 1) * COLS; cb += 16) {
        if (lo + cb >= hi) break;
        float g[16], u[16];
        tc::tmem_ld16(tmem + (GATED ? 0 : t * NT) + cb + lane_base, g);
        if constexpr (GATED) tc::tmem_ld16(tmem + NT + cb + lane_base, u);
        const float4* ts4 = reinterpret_cast<const float4*>(tok_scale + b * NT + cb);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float4 tv = ts4[j >> 2];
          const float ts = (j & 3) == 0 ? tv.x : (j & 3) == 1 ? tv.y : (j & 3) == 2 ? tv.z : tv.w;
          g[j] *= rs0 * ts;
          if constexpr (GATED) g[j] = silu_mul(g[j], u[j] * (rs1 * ts));
        }
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          uint32_t h;
          if (p.bf16) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(g[j], g[j + 1]);
            h = *reinterpret_cast<const uint32_t*>(&v);
          } else {
            h = pack_half2(g[j], g[j + 1]);
          }
          so[j * 32 + lane] = static_cast<uint16_t>(h);
          so[(j + 1) * 32 + lane] = static_cast<uint16_t>(h >> 16);
        }
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int tok = h * 8 + (lane >> 2), col = (lane & 3) * 8;
          const int left = p.n_out - (row0 + col);
          const uint4 d = *reinterpret_cast<const uint4*>(so + tok * 32 + col);
          if (lo + cb + tok < hi && left > 0) {
            uint16_t* dst = p.out + (int64_t)(lo + cb + tok) * p.out_stride + row0 + col;
            if (wide && left >= 8) {
              *reinterpret_cast<uint4*>(dst) = d;
            } else {
              const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (j < left) dst[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
            }
          }
        }
        __syncwarp();
      }
      // the accumulators and the tokens' scales are read
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(LY::B_DEMPTY));
        mbar_arrive(bar(LY::B_SEMPTY + b));
      }
    }
  }
  if (!ok) *abort_flag = 1;
  __syncwarp();
  if (f.ck > 1) {
    // the ranks' sums of a token and row, added in rank order; a rank finishes its share of the
    // tokens, two rows a thread
    griddep_wait();
    cluster_sync_all();
    if (!*abort_flag) {
      int lo, hi;
      const int e = find_item(p, first / f.row_tiles, NT, lo, hi);
      const int n0 = first % f.row_tiles * CTA_ROWS;
      const int m = hi - lo;
      const int t0 = m * rank / f.ck, t1 = m * (rank + 1) / f.ck;
      constexpr int PAIRS = CTA_ROWS / 2;
      const bool wide = (p.out_stride & 1) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 3) == 0;
      for (int o = tid; o < PAIRS * (t1 - t0); o += LY::THREADS) {
        const int tok = t0 + o / PAIRS, rr = (o % PAIRS) * 2;
        const int row = n0 + rr;
        if (row >= p.n_out) continue;
        const uint32_t at = s_base + (((GATED ? 0 : rr >> 7) * NT + tok) * 128 + (rr & 127)) * 4;
        float2 a[8], b[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          a[c] = c < f.ck ? ld_dsmem_f32x2(dsmem_addr(at, c)) : make_float2(0.0f, 0.0f);
          if constexpr (GATED) b[c] = c < f.ck ? ld_dsmem_f32x2(dsmem_addr(at + NT * 128 * 4, c)) : make_float2(0.0f, 0.0f);
        }
#pragma unroll
        for (int c = 1; c < 8; ++c) {
          a[0].x += a[c].x;
          a[0].y += a[c].y;
          if constexpr (GATED) {
            b[0].x += b[c].x;
            b[0].y += b[c].y;
          }
        }
        const float ts = tok_scale[tok];
        const int64_t wr = (int64_t)e * p.n_out + row;
        const bool two = row + 1 < p.n_out;
        float y0 = a[0].x * (p.row_scale[0][wr] * ts), y1 = two ? a[0].y * (p.row_scale[0][wr + 1] * ts) : 0.0f;
        if constexpr (GATED) {
          y0 = silu_mul(y0, b[0].x * (p.row_scale[1][wr] * ts));
          if (two) y1 = silu_mul(y1, b[0].y * (p.row_scale[1][wr + 1] * ts));
        }
        const uint32_t h0 = p.bf16 ? f2h<true>(y0) : f2h<false>(y0), h1 = p.bf16 ? f2h<true>(y1) : f2h<false>(y1);
        uint16_t* dst = p.out + (int64_t)(lo + tok) * p.out_stride + row;
        if (wide && two) {
          *reinterpret_cast<uint32_t*>(dst) = h0 | (h1 << 16);
        } else {
          dst[0] = static_cast<uint16_t>(h0);
          if (two) dst[1] = static_cast<uint16_t>(h1);
        }
      }
    }
    cluster_sync_all();
  }

  // ---- teardown: after an abort, this CTA's loads and MMAs in flight finish (bounded) first
  __syncthreads();
  if (*abort_flag) {
    constexpr uint64_t kDrainNs = 100000000ull;
    if (warp == CODES_WARP && lane == 0)
      for (int j = max(0, issued_c - CS); j < issued_c; ++j)
        mbar_wait_bounded(bar(LY::B_CFULL + j % CS), (j / CS) & 1, kDrainNs);
    if (warp == X_WARP && lane == 0)
      for (int j = max(0, issued_x - XS); j < issued_x; ++j)
        mbar_wait_bounded(bar(LY::B_XFULL + j % XS), (j / XS) & 1, kDrainNs);
    if (warp >= MMA_WARP && lane == 0 && mma_issued) {
      tc::commit(bar(LY::B_DRAIN + warp - MMA_WARP));
      mbar_wait_bounded(bar(LY::B_DRAIN + warp - MMA_WARP), 0, kDrainNs);
    }
    if (tid == 0) flag_status(p.status, AM_STATUS_TIMEOUT);
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(LY::TMEM_COLS));
  }
}

// ---------------------------------------------------------------- host
// Pairs of SMs where a matrix's mean number of rows fills most of a pair's 256 tokens and the tiles
// fill the pairs.
bool linear_uses_pairs(int rows, int experts, int n_out, bool grouped, bool gated) {
  const int mean = grouped ? (rows + experts - 1) / experts : rows;
  const int64_t tiles = (int64_t)((n_out + (gated ? 127 : 255)) / (gated ? 128 : 256)) *
                        (grouped ? rows / 256 : (rows + 255) / 256);
  return mean > 192 && tiles >= 64;
}

int linear_token_tile(int rows, int experts, bool grouped) {
  const int mean = grouped ? (rows + experts - 1) / experts : rows;
  return mean <= 32 ? 32 : (mean <= 64 ? 64 : 128);
}

template <int NT, bool GATED>
static cudaError_t launch_tiles_t(const LinearParams& p, int64_t items, cudaStream_t stream) {
  using LY = TilesLayout<NT>;
  int dev = 0;
  const int sms = sm_count(&dev);
  if (sms == 0) return cudaErrorInvalidDevice;
  cudaError_t err = cudaSuccess;
  auto kfn = linear_tiles_kernel<NT, GATED>;
  static unsigned long long done = 0;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) {
    err = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, LY::SMEM);
    if (err != cudaSuccess) return err;
    if (bit) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
  }
  const int rows_per_cta = GATED ? 128 : 256;
  const int row_tiles = (p.n_out + rows_per_cta - 1) / rows_per_cta;
  if (row_tiles * items > INT_MAX) return cudaErrorNotSupported;
  const int quads = p.pstride / 4;
  TilesParams f{};
  f.p = p;
  f.ck = 1;
  while (f.ck < 8 && (int64_t)row_tiles * items * f.ck * 2 <= (int64_t)sms * LY::CTAS && f.ck * 4 <= quads) f.ck *= 2;
  cudaLaunchConfig_t cfg = {};
  f.row_tiles = row_tiles;
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(row_tiles * items * f.ck, (int64_t)sms * LY::CTAS)));
  cfg.blockDim = dim3(LY::THREADS);
  cfg.dynamicSmemBytes = LY::SMEM;
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
static cudaError_t launch_tiles(const LinearParams& p, cudaStream_t stream) {
  const int64_t items = p.offsets != nullptr ? (int64_t)min(p.experts, p.rows) + p.rows / NT
                                             : ((int64_t)p.rows + NT - 1) / NT;
  return p.codes[1] != nullptr ? launch_tiles_t<NT, true>(p, items, stream) : launch_tiles_t<NT, false>(p, items, stream);
}

cudaError_t launch_linear_tiles(const LinearParams& p, bool pairs, cudaStream_t stream) {
  linear_rows_kernel<<<p.rows, 128, 0, stream>>>(p);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  if (pairs) return launch_linear_pair(p, stream);
  switch (linear_token_tile(p.rows, p.experts, p.offsets != nullptr)) {
    case 32: return launch_tiles<32>(p, stream);
    case 64: return launch_tiles<64>(p, stream);
    default: return launch_tiles<128>(p, stream);
  }
}

}  // namespace am
