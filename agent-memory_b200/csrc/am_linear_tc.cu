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
// Up to 64 tokens two CTAs share a SM.  No unit is saturated (ncu, 37 tokens 65536x4096 gated, 85 us:
// issue slots 59 % busy, tensor pipe 48 %, shared memory 35 %, DRAM 45 %; most stalls wait for the
// TMEM stores and barriers): what bounds it is the latency of a slab's chain, codes to
// commit, which two CTAs hide only in part.  At 128 tokens the tensor pipe is 62 % busy.  37 tokens
// 15360x3840 gated 26 us, 2.6 TB/s; 128 tokens 14336x4096 gated 33 us.  With few tiles the
// start, the activations' launch and the join take 10 us: 37 tokens 4096x4096 13 us.
// Every wait is bounded (LinearParams::wait_ns); on timeout the kernel flags AM_STATUS_TIMEOUT,
// lets its copies and MMAs in flight finish, frees its TMEM and returns.
//
// The codes and parameters are read before griddepcontrol.wait: linear_rows_kernel lets this grid start
// only after its own wait, when everything before it in the stream is complete, and it writes
// nothing but the activations.
#include <algorithm>
#include <climits>

#include "am_internal.h"
#include "am_linear.cuh"
#include "am_tcgen05.cuh"

namespace am {

// ---------------------------------------------------------------- activations
// A team of TEAM threads a row (a warp up to 2048 inputs, else the CTA): all of its 16-byte vectors are
// loaded before the first is used and stay in registers between the maximum and the conversion
// (up to kRowVectors a thread; longer rows are read twice).
constexpr int kRowThreads = 256, kRowVectors = 8;

template <int TEAM>
__global__ void __launch_bounds__(kRowThreads) linear_rows_kernel(const __grid_constant__ LinearParams p) {
  __shared__ uint32_t wmax[kRowThreads / 32];
  griddep_wait();
  griddep_launch_dependents();  // (not earlier: the next grid reads the weights before its own wait)
  const int row = blockIdx.x * (kRowThreads / TEAM) + threadIdx.x / TEAM, tid = threadIdx.x % TEAM;
  if (row >= p.rows) return;  // (whole teams)
  // rows that no expert holds are left alone: their order entries mean nothing (all three loads at once)
  const int pair = p.order != nullptr ? p.order[row] : row;
  const int held_lo = p.offsets != nullptr ? p.offsets[0] : 0;
  const int held_hi = p.offsets != nullptr ? p.offsets[p.experts] : p.rows;
  if (row < held_lo || row >= held_hi) return;
  const int from = source_row_of(p, pair);
  const uint4* src = reinterpret_cast<const uint4*>(p.x + (int64_t)max(from, 0) * p.x_stride);
  uint4* dst = reinterpret_cast<uint4*>(p.xh + (int64_t)row * p.n_in);
  const int vecs = from < 0 ? 0 : p.n_in / 8;
  const bool held = vecs <= TEAM * kRowVectors;
  uint4 u[kRowVectors];
  uint32_t mx = 0;
  for (int i0 = 0; i0 < vecs; i0 += TEAM * kRowVectors) {
#pragma unroll
    for (int j = 0; j < kRowVectors; ++j) {
      const int i = i0 + j * TEAM + tid;
      u[j] = i < vecs ? src[i] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < kRowVectors; ++j) mx = max(mx, max_abs_bits(u[j]));
    if (!p.bf16) {  // fp16 values stay as they are
#pragma unroll
      for (int j = 0; j < kRowVectors; ++j) {
        const int i = i0 + j * TEAM + tid;
        if (i < vecs) dst[i] = permute_f16(u[j]);
      }
    }
  }
  if (from < 0) {
    if (tid == 0) p.xscale[row] = 1.0f;
    for (int i = tid; i < p.n_in / 8; i += TEAM) dst[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
  if constexpr (TEAM > 32) {
    if ((tid & 31) == 0) wmax[tid >> 5] = mx;
    __syncthreads();
    mx = __reduce_max_sync(0xffffffffu, wmax[tid & (TEAM / 32 - 1)]);
  }
  // (a row with an infinity or a NaN is marked by a NaN as its power of two)
  if (!p.bf16) {
    if (tid == 0) p.xscale[row] = mx < 0x7c00u ? 1.0f : __int_as_float(0x7fffffff);
    return;
  }
  const int ex = row_exponent(mx);
  const float inv = exp2_int(-ex);
  for (int i0 = 0; i0 < vecs; i0 += TEAM * kRowVectors) {
#pragma unroll
    for (int j = 0; j < kRowVectors; ++j) {
      const int i = i0 + j * TEAM + tid;
      if (i < vecs) dst[i] = permute_bf16(held ? u[j] : src[i], inv);
    }
  }
  if (tid == 0) p.xscale[row] = mx < 0x7f80u ? exp2_int(ex) : __int_as_float(0x7fffffff);
}

// ---------------------------------------------------------------- tiles
template <int NT>
struct TilesLayout {
  // 128 tokens: one CTA a SM, 512 TMEM columns; fewer: two CTAs a SM of 256 columns each
  static constexpr int CTAS = NT == 128 ? 1 : 2;
  static constexpr uint32_t TMEM_COLS = 512 / CTAS;
  static constexpr int SP = NT == 128 ? 2 : 1;             // slabs (64 inputs) of a pipeline step
  static constexpr int CS = NT == 128 ? 3 : 2;             // code stages (256 rows x 256 inputs)
  static constexpr int XS = NT == 128 ? 3 : (NT == 64 ? 4 : 8);  // activation steps (NT x 64 SP inputs)
  static constexpr int AB = (TMEM_COLS - 2 * NT) / (64 * SP);    // TMEM operand buffers (2 tiles x 32 SP columns)
  static constexpr int DW = 8 * SP;                        // dequantization warps: 8 a slab of the step
  static constexpr int THREADS = 32 * (DW + 4);            // + codes, activations, two MMA warps
  static constexpr int CSTAGE = 2 * 128 * 128;
  static constexpr int XSLAB = NT * 128;
  static constexpr int OFF_C = 0;
  static constexpr int OFF_X = OFF_C + CS * CSTAGE;
  static constexpr int OFF_END = OFF_X + XS * SP * XSLAB;
  static constexpr int RED = 2 * NT * 128 * 4;             // fp32 sums of a split (over the rings)
  static constexpr int OFF_OUT = OFF_END > RED ? OFF_END : RED;  // kOutPitch bytes a token of a warp
  static constexpr int OFF_SCALE = OFF_OUT + DW * 16 * kOutPitch;  // two tiles' token scales
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

struct TilesParams {
  LinearParams p;
  int32_t ck;         // CTAs of a cluster that split the inputs (then a CTA has one tile)
  int32_t row_tiles;  // tiles of CTA_ROWS weight rows
};

// (out of line and with nothing kept for it: the kernel's loops do not notice)
template <int NT, int CTA_ROWS>
__device__ __noinline__ void tiles_store_nonfinite(const TilesParams& f) {
  const int b = static_cast<int>(blockIdx.x);
  store_nonfinite_tiles(f.p, NT, f.row_tiles, CTA_ROWS, 0, CTA_ROWS, b / f.ck, static_cast<int>(gridDim.x) / f.ck, b % f.ck,
                        f.ck);
}

template <int NT, bool GATED, int PARTS>
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
  volatile int* nonfinite = abort_flag + 1;  // one of this CTA's tokens is not finite
  float* tok_scale = reinterpret_cast<float*>(smem + LY::OFF_SCALE);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  // (loads wait long, the others mostly not at all)
  auto wait_long = [&](int i, uint32_t parity) { return wait_or_abort(bar(i), parity, p.wait_ns, abort_flag); };
  auto wait = [&](int i, uint32_t parity) { return wait_warp(bar(i), parity, p.wait_ns, abort_flag); };
  // (the warp index by a shuffle: uniform to the compiler, which then keeps the MMA operands in
  // uniform registers)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  griddep_launch_dependents();
  if (s_base & 1023u) {  // swizzled tiles need a 1024-byte aligned window (the whole grid returns)
    if (tid == 0) flag_status(p.status, AM_STATUS_BAD_POSITION);
    griddep_wait();
    return;
  }
  const int rank = f.ck > 1 ? static_cast<int>(blockIdx.x) % f.ck : 0;
  const int first = static_cast<int>(blockIdx.x) / f.ck, step = static_cast<int>(gridDim.x) / f.ck;
  const int tiles = count_items(p, NT) * f.row_tiles;
  if (first >= tiles) {  // the whole cluster
    griddep_wait();  // (a grid may not be complete before the one it depends on: the next one waits for this one only)
    return;
  }
  constexpr int CTA_ROWS = GATED ? 128 : 256;
  // this CTA's inputs: quads of groups [q0, q1), slabs of 64 inputs, steps of SP slabs
  const int quads = p.pstride >> 2;
  const int q0 = quads * rank / f.ck, q1 = quads * (rank + 1) / f.ck;
  const int slabs = min(q1 * 4, p.groups) - q0 * 4;
  const int steps = (slabs + SP - 1) / SP * PARTS;  // (a step's parts follow one another)

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "r"(LY::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  } else if (warp == CODES_WARP) {
    for (int i = lane; i < LY::B_COUNT; i += 32) mbar_init(bar(i), LY::arrivals(i));
    if (lane == 0) *abort_flag = *nonfinite = 0;
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

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
          ok = wait_long(LY::B_CEMPTY + ring.s, ring.ph ^ 1u);
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
        ok = __all_sync(0xffffffffu, wait_long(LY::B_XEMPTY + ring.s, ring.ph ^ 1u));
        if (!ok) break;
        const uint32_t full = bar(LY::B_XFULL + ring.s), dst = s_base + LY::OFF_X + ring.s * SP * LY::XSLAB;
        const int n = min(SP, slabs - i / PARTS * SP);
        if (lane == 0) {
          mbar_arrive_expect_tx(full, n * LY::XSLAB);
          for (int s = 0; s < n; ++s)
            tma_load_2d(dst + s * LY::XSLAB, &p.tmap_x, (q0 * 4 + i / PARTS * SP + s) * 128, lo, full);
        }
        ++issued_x;
        ring.next();
        if (i == min(XS, steps) - 1) {  // behind the first loads: the tokens' powers of two
          const int b = k & 1;
          ok = wait(LY::B_SEMPTY + b, ((k >> 1) & 1) ^ 1);
          if (!ok) break;
          bool marked = false;
          for (int j = lane; j < NT; j += 32) {
            const float ts = lo + j < hi ? p.xscale[lo + j] : 0.0f;
            tok_scale[b * NT + j] = ts;
            marked |= isnan(ts);
          }
          if (__any_sync(0xffffffffu, marked)) *nonfinite = 1;  // (the warp together: a divergent store made the loops spill)
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(LY::B_SFULL + b));
        }
      }
    }
  } else if (warp >= MMA_WARP) {
    // Two issuing warps, one a weight tile: the waits and commits of one hide behind the MMAs of the other
    // (one for both left the tensor pipe idle half of the time).  The whole warp runs the loop,
    // converged, and one lane issues: with a divergent loop every operand of every MMA moves to a
    // uniform register first.
    constexpr uint32_t ID = tc::idesc(128, NT, false);
    const bool lead = elect_one();
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
        if (lead) {
          // (descriptor addresses count 16-byte units: 32 bytes of a swizzled row are 16 inputs)
          tc::mma_ts(d, a, xd, ID, i > 0 ? 1u : 0u);
#pragma unroll
          for (int ks = 1; ks < 4; ++ks) tc::mma_ts(d, a + ks * 8, xd + ks * 2, ID, 1u);
          if (SP == 2 && 2 * (i / PARTS) + 1 < slabs) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) tc::mma_ts(d, a + 64 + ks * 8, xd + LY::XSLAB / 16 + ks * 2, ID, 1u);
          }
          tc::commit(bar(LY::B_XEMPTY + xr.s));
          tc::commit(bar(LY::B_AEMPTY + ar.s));
        }
        mma_issued = lead;
        xr.next();
        ar.next();
      }
      if (ok && lead) tc::commit(bar(LY::B_DFULL));
    }
  } else {
    // ---- dequantization: one weight row of tile t a thread, slab `group` of every step
    const int group = SP == 1 ? 0 : warp >> 3, t = (warp >> 2) & 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t a_base = tmem + LY::A_COL + group * 64 + t * 32 + lane_base;
    Ring<CS> cr;
    Ring<AB> ar;
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
        ok = wait(LY::B_CFULL + cr.s, cr.ph);
        if (!ok) break;
        const uint8_t* crow = smem + LY::OFF_C + cr.s * LY::CSTAGE + t * (LY::CSTAGE / 2) + r * 128;
        const uint32_t pw[4] = {pv.x, pv.y, pv.z, pv.w};
        const int in_stage = min(4, slabs - 4 * (c - q0));
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          if (st * SP >= in_stage) break;
          const int s = st * SP + group;
          uint4 w0, w1;
          if (s < in_stage) {
            w0 = *reinterpret_cast<const uint4*>(crow + (((2 * s) ^ (r & 7)) << 4));
            w1 = *reinterpret_cast<const uint4*>(crow + (((2 * s + 1) ^ (r & 7)) << 4));
          }
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            uint32_t o[32];
            if (s < in_stage)
              dequant_group<PARTS>(w0, w1, SP == 1 || group == 0 ? pw[st * SP] : pw[(st * SP + 1) & 3], part, o);
            ok = wait(LY::B_AEMPTY + ar.s, ar.ph ^ 1u);
            if (!ok) break;
            tc::fence_after();
            if (s < in_stage) tc::tmem_st32(a_base + ar.s * 64 * SP, o);  // (17 cycles with its wait)
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(LY::B_AFULL + ar.s));
            ar.next();
          }
          if (!ok) break;
        }
        if (!ok) break;
        __syncwarp();  // the stage's codes are in registers
        if (lane == 0) mbar_arrive(bar(LY::B_CEMPTY + cr.s));
        cr.next();
        pv = pnext;
      }
      if (!ok) break;
      const int b = k & 1;
      ok = wait(LY::B_DFULL, k & 1) && wait(LY::B_SFULL + b, (k >> 1) & 1);
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
      // ---- output: 16 tokens at a time, from mma fragments (thread (g8, t4): rows g8 + 8 i, tokens 2 t4, + 1
      // of eight)
      constexpr int SHARES = GATED ? DW / 4 : DW / 8;  // warps that share a lane quarter (and tile)
      constexpr int COLS = NT / SHARES;
      const int part = GATED ? warp >> 2 : group;
      const int g8 = lane >> 2, t4 = lane & 3;
      const int row0 = n0 + (GATED ? 0 : t * 128) + quarter * 32;
      float rs[GATED ? 2 : 1][4];
#pragma unroll
      for (int m = 0; m < (GATED ? 2 : 1); ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          rs[m][i] = __ldg(p.row_scale[m] + (int64_t)e * p.n_out + min(row0 + g8 + 8 * i, p.n_out - 1));
      uint8_t* so = smem + LY::OFF_OUT + warp * 16 * kOutPitch;
#pragma unroll 1
      for (int cb = part * COLS; cb < (part + 1) * COLS; cb += 16) {
        if (lo + cb >= hi) break;
        float v[GATED ? 2 : 1][2][8];  // [matrix][16 rows][token block, row g8 or g8 + 8, token]
#pragma unroll
        for (int m = 0; m < (GATED ? 2 : 1); ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            tc::tmem_ld_16x16_nowait(tmem + (GATED ? m * NT : t * NT) + cb + lane_base + (static_cast<uint32_t>(16 * h) << 16),
                                     v[m][h]);
        float2 ts[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) ts[j] = *reinterpret_cast<const float2*>(tok_scale + b * NT + cb + 8 * j + 2 * t4);
        tc::tmem_wait_ld();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float f = (i & 1) ? ts[i >> 2].y : ts[i >> 2].x;
            const int r4 = 2 * h + ((i >> 1) & 1);
            v[0][h][i] *= rs[0][r4] * f;
            if constexpr (GATED) v[0][h][i] = silu_mul(v[0][h][i], v[1][h][i] * (rs[1][r4] * f));
          }
        uint32_t q[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            q[j][2 * h] = pack_out(p, v[0][h][4 * j], v[0][h][4 * j + 1]);
            q[j][2 * h + 1] = pack_out(p, v[0][h][4 * j + 2], v[0][h][4 * j + 3]);
          }
        store_tokens(p, so, q, lo + cb, hi, row0);
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
    // the ranks' sums of a token and row, added in rank order; a rank finishes its share of the tokens,
    // a thread four rows of every TL-th of them
    griddep_wait();
    int lo, hi;
    const int e = find_item(p, first / f.row_tiles, NT, lo, hi);
    const int n0 = first % f.row_tiles * CTA_ROWS;
    constexpr int QUADS = CTA_ROWS / 4, TL = LY::THREADS / QUADS;
    const int rr = tid % QUADS * 4, tl = tid / QUADS, row = n0 + rr;
    float rs[GATED ? 2 : 1][4];
#pragma unroll
    for (int m = 0; m < (GATED ? 2 : 1); ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) rs[m][i] = __ldg(p.row_scale[m] + (int64_t)e * p.n_out + min(row + i, p.n_out - 1));
    cluster_sync_all();
    if (!*abort_flag && tl < TL) {
      // a rank that gave up has no sums: then nothing is stored (a lane asks one rank, ahead of the first
      // sums, and the warp votes behind them; a lane asking all ranks cost 0.35 us)
      int gave_up = 0;
      if (lane < f.ck) gave_up = __float_as_int(ld_dsmem_f32(dsmem_addr(smem_u32(const_cast<const int*>(abort_flag)), lane)));
      const int m = hi - lo;
      const int t0 = m * rank / f.ck, t1 = m * (rank + 1) / f.ck;
      const bool wide = (p.out_stride & 3) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7) == 0 && row + 4 <= p.n_out;
      const uint32_t at0 = s_base + ((GATED ? 0 : rr >> 7) * NT * 128 + (rr & 127)) * 4;
      for (int tok = t0 + tl; tok < t1; tok += TL) {
        float4 s[GATED ? 2 : 1] = {};
#pragma unroll 8
        for (int c = 0; c < f.ck; ++c) {
          const uint32_t at = dsmem_addr(at0, c) + tok * 512;
#pragma unroll
          for (int k = 0; k < (GATED ? 2 : 1); ++k) {
            const float4 v = ld_dsmem_f32x4(at + k * NT * 512);
            s[k].x += v.x;
            s[k].y += v.y;
            s[k].z += v.z;
            s[k].w += v.w;
          }
        }
        if (__any_sync(0xffffffffu, gave_up)) break;
        const float ts = tok_scale[tok];
        float y[4] = {s[0].x, s[0].y, s[0].z, s[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] *= rs[0][i] * ts;
        if constexpr (GATED) {
          const float w[4] = {s[1].x, s[1].y, s[1].z, s[1].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = silu_mul(y[i], w[i] * (rs[1][i] * ts));
        }
        uint16_t* dst = p.out + (int64_t)(lo + tok) * p.out_stride + row;
        if (wide) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack_out(p, y[0], y[1]), pack_out(p, y[2], y[3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row + i < p.n_out) dst[i] = p.bf16 ? f2h<true>(y[i]) : f2h<false>(y[i]);
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
    if (warp >= MMA_WARP && mma_issued) {
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
  if (*nonfinite) tiles_store_nonfinite<NT, CTA_ROWS>(f);
}

// ---------------------------------------------------------------- host
// Pairs of SMs where a matrix's mean number of rows passes the single tile's 128 tokens and the tiles
// fill the pairs (experts, 32 of 2880x2880 gated: mean 96 147 us and 125 single, mean 144 167 and 222;
// one matrix, 512 tokens: 14336x4096 gated, 224 tiles, 96 and 102; 4096x14336, 32 tiles, 59 and 50).
bool linear_uses_pairs(int rows, int experts, int n_out, bool grouped, bool gated) {
  const int mean = grouped ? (rows + experts - 1) / experts : rows;
  const int64_t tiles = (int64_t)((n_out + (gated ? 127 : 255)) / (gated ? 128 : 256)) *
                        (grouped ? rows / 256 : (rows + 255) / 256);
  return mean > 128 && tiles >= 64;
}

// Tokens of a tile: what holds the rows of a matrix, for experts twice their mean up to 64 (32 of 2880x2880
// gated, mean 8: 73 us with 32 tokens and 77 with 64, mean 32: 102 and 82, mean 96: 149 with 64 and
// 125 with 128).  One matrix of few tiles is cut into 64 up to 128 tokens, for more SMs to work (128
// tokens: 4096x4096, 32 tiles, 14.3 us and 16.9 uncut; 14336x4096, 112, 25.4 and 23.1).
int linear_token_tile(int rows, int experts, int n_out, bool grouped, bool gated) {
  const int mean = grouped ? (rows + experts - 1) / experts : rows;
  if (mean <= (grouped ? 16 : 32)) return 32;
  if (mean <= 64) return 64;
  const int tile_rows = gated ? 128 : 256;
  return !grouped && mean <= 128 && (n_out + tile_rows - 1) / tile_rows <= 32 ? 64 : 128;
}

template <int NT, bool GATED, int PARTS>
static cudaError_t launch_tiles_t(const LinearParams& p, int64_t items, cudaStream_t stream) {
  using LY = TilesLayout<NT>;
  int dev = 0;
  const int sms = sm_count(&dev);
  if (sms == 0) return cudaErrorInvalidDevice;
  cudaError_t err = cudaSuccess;
  auto kfn = linear_tiles_kernel<NT, GATED, PARTS>;
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
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(LY::THREADS);
  cfg.dynamicSmemBytes = LY::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  // The inputs are split while all tiles still run at once: clusters lie within a GPC, so fewer of 8 fit than
  // the SMs would hold (128 tokens 4096x4096, 16 tiles: 29 us in clusters of 8 that came in two
  // waves, 16.9 in clusters of 4).
  static int fit[64][4];  // clusters of 2^i that fit on a device, once known
  const int64_t tiles = row_tiles * items;
  f.ck = 1;
  f.row_tiles = row_tiles;
  for (int i = 1; i < 4 && (4 << (i - 1)) <= quads && (tiles << i) <= (int64_t)sms * LY::CTAS; ++i) {
    int n = dev < 64 ? __atomic_load_n(&fit[dev][i], __ATOMIC_RELAXED) : 0;
    if (n == 0) {
      cfg.gridDim = dim3(static_cast<unsigned>(sms * LY::CTAS) >> i << i);
      attr[1].val.clusterDim.x = 1 << i;
      cfg.numAttrs = 2;
      err = cudaOccupancyMaxActiveClusters(&n, kfn, &cfg);
      if (err != cudaSuccess) return err;
      if (dev < 64) __atomic_store_n(&fit[dev][i], n, __ATOMIC_RELAXED);
    }
    if (tiles > n) break;
    f.ck = 1 << i;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(tiles * f.ck, (int64_t)sms * LY::CTAS)));
  attr[1].val.clusterDim.x = f.ck;
  cfg.numAttrs = f.ck > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kfn, f);
}

template <int NT>
static cudaError_t launch_tiles(const LinearParams& p, cudaStream_t stream) {
  const int64_t items = p.offsets != nullptr ? (int64_t)min(p.experts, p.rows) + p.rows / NT
                                             : ((int64_t)p.rows + NT - 1) / NT;
  const bool gated = p.codes[1] != nullptr;
  if (weight_parts(gated, p.bf16) == 2) return launch_tiles_t<NT, true, 2>(p, items, stream);
  return gated ? launch_tiles_t<NT, true, 1>(p, items, stream) : launch_tiles_t<NT, false, 1>(p, items, stream);
}

cudaError_t launch_linear_tiles(const LinearParams& p, bool pairs, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const int team = p.n_in <= 32 * 8 * kRowVectors ? 32 : kRowThreads;
  cfg.gridDim = dim3((p.rows + kRowThreads / team - 1) / (kRowThreads / team));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, team == 32 ? linear_rows_kernel<32> : linear_rows_kernel<kRowThreads>, p);
  if (err != cudaSuccess) return err;
  if (pairs) return launch_linear_pair(p, stream);
  switch (linear_token_tile(p.rows, p.experts, p.n_out, p.offsets != nullptr, p.codes[1] != nullptr)) {
    case 32: return launch_tiles<32>(p, stream);
    case 64: return launch_tiles<64>(p, stream);
    default: return launch_tiles<128>(p, stream);
  }
}

}  // namespace am
