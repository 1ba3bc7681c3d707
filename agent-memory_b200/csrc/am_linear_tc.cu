// Linear layers over 4-bit weights for more than a few tokens: tcgen05 tensor tiles.
//
// y^T = W x^T: weight rows are the M side (128 lanes of TMEM), tokens the N side, so a weight is
// dequantized once for up to 128 tokens, straight into the TMEM operand.
//
// 1. linear_rows_kernel writes the activations as fp16 rows of the workspace, each under a power
//    of two (exact for fp16 and bf16 values) and with its inputs in the order in which the
//    dequantization below produces the weights.
// 2. linear_tiles_kernel: a CTA owns two 128-row weight tiles (plain: 256 rows of the matrix;
//    gated: 128 rows of each matrix) and NT tokens of one matrix or expert.
//    * one thread streams the codes (TMA, 128 rows x 256 inputs a box, 128-byte swizzle), one
//      warp the activations (TMA boxes of NT rows x 64 inputs; through `order` by
//      tile::gather4, four rows an instruction; rows past the item or behind a bad index lie
//      outside the map and read as zeros);
//    * warps 0-7 dequantize: a thread owns a weight row; 64 codes a step become 32 registers of
//      fp16 pairs (9 operations for 8 weights, see am_linear.cu) and go to TMEM with one
//      tcgen05.st -- no shared-memory round trip, and the MMA reads its A operand there;
//    * one thread issues tcgen05.mma (kind::f16, M = 128, N = NT, K = 16) over both tiles.
//    The accumulators are read back by the dequantization warps, scaled by the row's and the
//    token's powers of two, gated, rounded once and stored.
//    With few tiles the inputs are split over the CTAs of a cluster, whose fp32 sums meet in
//    distributed shared memory, in rank order.
// Every wait is bounded (LinearParams::wait_ns); on timeout the kernel flags AM_STATUS_TIMEOUT,
// lets its copies and MMAs in flight finish, frees its TMEM and returns.
//
// The codes and parameters are read before griddepcontrol.wait: linear_rows_kernel starts only
// when everything before it in the stream is complete (it is launched without programmatic
// serialization), and it writes nothing but the activations.
#include "am_internal.h"
#include "am_linear.cuh"
#include "am_tcgen05.cuh"

namespace am {

// ---------------------------------------------------------------- activations
__global__ void __launch_bounds__(128) linear_rows_kernel(const __grid_constant__ LinearParams p) {
  __shared__ uint32_t wmax[4];
  griddep_launch_dependents();
  const int row = blockIdx.x, tid = threadIdx.x;
  const uint4* src = reinterpret_cast<const uint4*>(p.x + (int64_t)row * p.x_stride);
  uint4* dst = reinterpret_cast<uint4*>(p.xh + (int64_t)row * p.n_in);
  const int vecs = p.n_in / 8;
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
  static constexpr int CS = NT == 128 ? 3 : 2;              // code stages (256 rows x 256 inputs)
  static constexpr int XS = NT == 128 ? 6 : (NT == 64 ? 5 : 8);  // activation slabs (NT x 64 inputs)
  static constexpr int AB = (TMEM_COLS - 2 * NT) / 64;      // TMEM operand buffers (2 tiles x 32 columns)
  static constexpr int DG = NT == 128 ? 2 : 1;              // groups of 8 dequantization warps, slabs in turn
  static constexpr int DW = 8 * DG;
  static constexpr int THREADS = 32 * (DW + 3);             // + codes, activations, MMA
  static constexpr int CSTAGE = 2 * 128 * 128;
  static constexpr int XSLAB = NT * 128;
  static constexpr int OFF_C = 0;
  static constexpr int OFF_X = OFF_C + CS * CSTAGE;
  static constexpr int OFF_END = OFF_X + XS * XSLAB;
  static constexpr int RED = 2 * NT * 128 * 4;              // fp32 sums of a split (over the rings)
  static constexpr int OFF_BAR = OFF_END > RED ? OFF_END : RED;
  static constexpr int B_CFULL = 0, B_CEMPTY = CS, B_XFULL = 2 * CS, B_XEMPTY = B_XFULL + XS;
  static constexpr int B_AFULL = B_XEMPTY + XS, B_AEMPTY = B_AFULL + AB, B_DFULL = B_AEMPTY + AB;
  static constexpr int B_DRAIN = B_DFULL + 1, B_SCALE = B_DRAIN + 1, B_COUNT = B_SCALE + 1;
  static constexpr int OFF_SCALE = OFF_BAR + B_COUNT * 8 + 16;
  static constexpr int SMEM = OFF_SCALE + NT * 4;
  static constexpr int A_COL = 2 * NT;  // D[tile] at tile * NT, A[buffer][tile] at A_COL + 64 b + 32 tile
  static_assert(AB >= 2 && (DG == 1 || AB % DG == 0), "the operand needs two buffers");
  static_assert(SMEM * CTAS <= 232448 - 1024 * (CTAS - 1), "shared memory of a SM");
};

// gather4 load of four rows of a map with one-row boxes of 128 bytes.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int x, int r0, int r1, int r2,
                                            int r3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%2, %3, %4, %5, %6}], [%7];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
      : "memory");
}

struct TilesParams {
  LinearParams p;
  int32_t ck;  // CTAs of a cluster that split the inputs
};

template <int NT, bool GATED>
__global__ void __launch_bounds__(TilesLayout<NT>::THREADS, TilesLayout<NT>::CTAS)
    linear_tiles_kernel(const __grid_constant__ TilesParams f) {
  using LY = TilesLayout<NT>;
  constexpr int CS = LY::CS, XS = LY::XS, AB = LY::AB;
  constexpr int DW = LY::DW, DG = LY::DG;
  constexpr int CODES_WARP = DW, X_WARP = DW + 1, MMA_WARP = DW + 2;
  const LinearParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s_base = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + LY::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + LY::OFF_BAR + LY::B_COUNT * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + LY::OFF_BAR + LY::B_COUNT * 8 + 4);
  float* tok_scale = reinterpret_cast<float*>(smem + LY::OFF_SCALE);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (s_base & 1023u) {  // swizzled tiles need a 1024-byte aligned window (the whole grid returns)
    if (tid == 0) flag_status(p.status, AM_STATUS_BAD_POSITION);
    return;
  }
  int lo, hi;
  const int e = find_item<NT>(p, blockIdx.y, lo, hi);
  if (e < 0) return;  // the whole cluster: it shares blockIdx.y
  const int rank = f.ck > 1 ? static_cast<int>(blockIdx.x) % f.ck : 0;
  const int tile = static_cast<int>(blockIdx.x) / f.ck;
  constexpr int CTA_ROWS = GATED ? 128 : 256;
  const int n0 = tile * CTA_ROWS;
  // this CTA's inputs: quads of groups [q0, q1), slabs of 64 inputs
  const int quads = p.pstride >> 2;
  const int q0 = quads * rank / f.ck, q1 = quads * (rank + 1) / f.ck;
  const int slabs = min(q1 * 4, p.groups) - q0 * 4;

  if (tid == 0) {
    for (int i = 0; i < LY::B_COUNT; ++i) {
      const bool c_empty = i >= LY::B_CEMPTY && i < LY::B_CEMPTY + CS;
      const bool a_full = i >= LY::B_AFULL && i < LY::B_AFULL + AB;
      mbar_init(bar(i), c_empty ? DW : (a_full ? 8 : 1));
    }
    fence_mbar_init();
    *abort_flag = 0;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "r"(LY::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

  int issued_c = 0, issued_x = 0;  // loads in flight (their own threads' counts)
  bool mma_issued = false;
  if (warp == CODES_WARP) {
    if (lane == 0) {
      const int y = e * p.n_out + n0;
      bool ok = true;
      for (int c = 0; c < q1 - q0; ++c) {
        const int s = c % CS;
        if (c >= CS) ok = wait_or_abort(bar(LY::B_CEMPTY + s), ((c - CS) / CS) & 1, p.wait_ns, abort_flag);
        if (!ok) break;
        mbar_arrive_expect_tx(bar(LY::B_CFULL + s), LY::CSTAGE);
        const uint32_t dst = s_base + LY::OFF_C + s * LY::CSTAGE;
        tma_load_2d(dst, &p.tmap_w[0], (q0 + c) * 128, y, bar(LY::B_CFULL + s));
        tma_load_2d(dst + LY::CSTAGE / 2, &p.tmap_w[GATED ? 1 : 0], (q0 + c) * 128, GATED ? y : y + 128,
                    bar(LY::B_CFULL + s));
        issued_c = c + 1;
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == X_WARP) {
    int rows4[4] = {};
    if (p.order != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = lo + 4 * lane + j;
        const int src = 4 * lane < NT && r < hi ? source_row(p, r) : -1;
        rows4[j] = src >= 0 ? src : p.x_rows;  // past the map: zeros
      }
    }
    griddep_wait();  // the activations are written
    bool ok = true;
    auto scales = [&]() {  // the tokens' powers of two, for the epilogue
      for (int j = lane; j < NT; j += 32) {
        const int r = lo + j;
        float v = 0.0f;
        if (r < hi) {
          const int src = p.order != nullptr ? p.order[r] / p.top_k : r;
          if (src >= 0 && src < p.x_rows) v = p.xscale[src];
        }
        tok_scale[j] = v;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(LY::B_SCALE));
    };
    for (int i = 0; i < slabs; ++i) {
      if (i == min(XS, slabs) - 1) scales();  // behind the first loads
      const int s = i % XS;
      if (i >= XS) ok = wait_or_abort(bar(LY::B_XEMPTY + s), ((i - XS) / XS) & 1, p.wait_ns, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      const uint32_t dst = s_base + LY::OFF_X + s * LY::XSLAB;
      if (lane == 0) mbar_arrive_expect_tx(bar(LY::B_XFULL + s), LY::XSLAB);
      __syncwarp();
      if (p.order != nullptr) {
        if (4 * lane < NT)
          tma_gather4(dst + lane * 512, &p.tmap_x, (q0 * 4 + i) * 128, rows4[0], rows4[1], rows4[2], rows4[3],
                      bar(LY::B_XFULL + s));
      } else if (lane == 0) {
        tma_load_2d(dst, &p.tmap_x, (q0 * 4 + i) * 128, lo, bar(LY::B_XFULL + s));
      }
      issued_x = i + 1;
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == MMA_WARP) {
    if (lane == 0) {
      constexpr uint32_t ID = tc::idesc(128, NT, false);
      bool ok = true;
      for (int i = 0; i < slabs && ok; ++i) {
        const int b = i % AB, s = i % XS;
        ok = wait_or_abort(bar(LY::B_XFULL + s), (i / XS) & 1, p.wait_ns, abort_flag) &&
             wait_or_abort(bar(LY::B_AFULL + b), (i / AB) & 1, p.wait_ns, abort_flag);
        if (!ok) break;
        tc::fence_after();
        const uint32_t xs = s_base + LY::OFF_X + s * LY::XSLAB;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            tc::mma_ts(tmem + t * NT, tmem + LY::A_COL + b * 64 + t * 32 + ks * 8, tc::sdesc(xs + ks * 32, 16, 1024),
                       ID, (i > 0 || ks > 0) ? 1u : 0u);
        mma_issued = true;
        tc::commit(bar(LY::B_XEMPTY + s));
        tc::commit(bar(LY::B_AEMPTY + b));
      }
      if (ok) tc::commit(bar(LY::B_DFULL));
      if (!ok) *abort_flag = 1;
    }
  } else {
    // ---- dequantization: one weight row of tile t a thread, 64 inputs (a slab) at a time; with two
    // groups of warps each takes every other slab.  A slab's store into TMEM completes while
    // the next one is dequantized, and only then is it handed to the MMA thread.
    const int group = warp >> 3, t = (warp >> 2) & 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int n = min(n0 + (GATED ? 0 : t * 128) + r, p.n_out - 1);
    const uint32_t* prow = p.params[GATED ? t : 0] + ((int64_t)e * p.n_out + n) * p.pstride;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t a_base = tmem + LY::A_COL + t * 32 + lane_base;
    uint4 pv = __ldg(reinterpret_cast<const uint4*>(prow) + q0);
    bool ok = true;
    int stored = -1;  // buffer of the store in flight
    auto publish = [&]() {
      if (stored >= 0) {
        tc::tmem_wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(LY::B_AFULL + stored));
      }
    };
    for (int c = 0; c < q1 - q0 && ok; ++c) {
      const int cs = c % CS;
      const uint4 pnext = c + 1 < q1 - q0 ? __ldg(reinterpret_cast<const uint4*>(prow) + q0 + c + 1) : pv;
      ok = __all_sync(0xffffffffu, wait_or_abort(bar(LY::B_CFULL + cs), (c / CS) & 1, p.wait_ns, abort_flag));
      if (!ok) break;
      const uint8_t* crow = smem + LY::OFF_C + cs * LY::CSTAGE + t * (LY::CSTAGE / 2) + r * 128;
      const uint32_t pw[4] = {pv.x, pv.y, pv.z, pv.w};
      const int in_stage = min(4, slabs - 4 * c);
#pragma unroll
      for (int s4 = 0; s4 < 4; s4 += DG) {
        const int s = s4 + group;
        if (s >= in_stage) break;
        const int i = 4 * c + s, b = i % AB;
        const uint4 w0 = *reinterpret_cast<const uint4*>(crow + (((2 * s) ^ (r & 7)) << 4));
        const uint4 w1 = *reinterpret_cast<const uint4*>(crow + (((2 * s + 1) ^ (r & 7)) << 4));
        const uint32_t ps = DG == 1 ? pw[s4] : (group == 0 ? pw[s4] : pw[(s4 + 1) & 3]);
        const uint32_t s24 = __byte_perm(ps, ps, 0x1010), bb = __byte_perm(ps, ps, 0x3232);
        const uint32_t s20 = hfma2_bits(s24, 0x2c002c00u, 0x80008000u);
        const uint32_t words[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
        uint32_t o[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t d[4];
          dequant_word(words[j], s24, s20, bb, d);
#pragma unroll
          for (int k = 0; k < 4; ++k) o[4 * j + k] = d[k];
        }
        publish();
        if (i >= AB) {
          ok = __all_sync(0xffffffffu,
                          wait_or_abort(bar(LY::B_AEMPTY + b), ((i - AB) / AB) & 1, p.wait_ns, abort_flag));
          if (!ok) break;
          tc::fence_after();
        }
        tc::tmem_st32_nowait(a_base + b * 64, o);
        stored = b;
      }
      __syncwarp();  // the stage's codes are in registers
      if (lane == 0) mbar_arrive(bar(LY::B_CEMPTY + cs));
      pv = pnext;
    }
    if (ok) {
      publish();
      ok = __all_sync(0xffffffffu, wait_or_abort(bar(LY::B_DFULL), 0, p.wait_ns, abort_flag) &&
                                       wait_or_abort(bar(LY::B_SCALE), 0, p.wait_ns, abort_flag));
    }
    if (!ok) *abort_flag = 1;
    // the output warps meet here also after an abort (each may have seen it at another step)
    tc::fence_after();
    if (f.ck == 1) {
      // ---- output: lane = weight row, columns = tokens; rounded values to shared memory as
      // [token][row], then whole rows of them to global memory
      constexpr int PARTS = GATED ? DW / 4 : DW / 8;  // warps that share a lane quarter (and tile)
      constexpr int COLS = NT / PARTS;
      const int part = GATED ? warp >> 2 : group;
      const int row = n0 + (GATED ? 0 : t * 128) + r;
      const int64_t wr = (int64_t)e * p.n_out + min(row, p.n_out - 1);
      const float rs0 = p.row_scale[0][wr], rs1 = GATED ? p.row_scale[1][wr] : 0.0f;
      uint16_t* so = reinterpret_cast<uint16_t*>(smem);
      if (ok) {
#pragma unroll 1
        for (int cb = part * COLS; cb < (part + 1) * COLS; cb += 16) {
          if (lo + cb >= hi) break;
          float g[16], u[16];
          tc::tmem_ld16(tmem + (GATED ? 0 : t * NT) + cb + lane_base, g);
          if constexpr (GATED) tc::tmem_ld16(tmem + NT + cb + lane_base, u);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float ts = tok_scale[cb + j];
            const float y = GATED ? silu_mul(g[j] * (rs0 * ts), u[j] * (rs1 * ts)) : g[j] * (rs0 * ts);
            so[(cb + j) * CTA_ROWS + (GATED ? 0 : t * 128) + r] = p.bf16 ? f2h<true>(y) : f2h<false>(y);
          }
        }
      }
      asm volatile("bar.sync 1, %0;\n" ::"n"(DW * 32) : "memory");
      if (!*abort_flag) {
        const int m = hi - lo;
        const bool wide = (p.out_stride & 7) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
        constexpr int VPR = CTA_ROWS / 8;  // 16-byte vectors of a token
        for (int v = tid; v < m * VPR; v += DW * 32) {
          const int tok = v / VPR, col = (v % VPR) * 8;
          const int left = p.n_out - (n0 + col);
          if (left <= 0) continue;
          const uint4 d = *reinterpret_cast<const uint4*>(so + tok * CTA_ROWS + col);
          uint16_t* dst = p.out + (int64_t)(lo + tok) * p.out_stride + n0 + col;
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
    } else if (ok) {
      // ---- fp32 sums to shared memory, [tile][token][128 rows]
      constexpr int COLS = NT / DG;
      float* red = reinterpret_cast<float*>(smem) + t * NT * 128 + r;
#pragma unroll 1
      for (int cb = group * COLS; cb < (group + 1) * COLS; cb += 16) {
        float v[16];
        tc::tmem_ld16(tmem + t * NT + cb + lane_base, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) red[(cb + j) * 128] = v[j];
      }
    }
  }
  __syncwarp();
  if (f.ck > 1) {
    // the ranks' sums of a token and row, added in rank order; a rank finishes its share of the
    // tokens, two rows a thread
    cluster_sync_all();
    if (!*abort_flag) {
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
    if (warp == MMA_WARP && lane == 0 && mma_issued) {
      tc::commit(bar(LY::B_DRAIN));
      mbar_wait_bounded(bar(LY::B_DRAIN), 0, kDrainNs);
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
int linear_token_tile(int rows, int experts, bool grouped) {
  const int mean = grouped ? (rows + experts - 1) / experts : rows;
  return mean <= 32 ? 32 : (mean <= 64 ? 64 : 128);
}

template <int NT, bool GATED>
static cudaError_t launch_tiles_t(const LinearParams& p, int64_t items, cudaStream_t stream) {
  using LY = TilesLayout<NT>;
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return err;
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
  const int quads = p.pstride / 4;
  TilesParams f{};
  f.p = p;
  f.ck = 1;
  while (f.ck < 8 && (int64_t)row_tiles * items * f.ck * 2 <= (int64_t)sms * LY::CTAS && f.ck * 4 <= quads) f.ck *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(row_tiles * f.ck, static_cast<unsigned>(items));
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
  if (items > 65535) return cudaErrorInvalidConfiguration;
  return p.codes[1] != nullptr ? launch_tiles_t<NT, true>(p, items, stream) : launch_tiles_t<NT, false>(p, items, stream);
}

cudaError_t launch_linear_tiles(const LinearParams& p, cudaStream_t stream) {
  linear_rows_kernel<<<p.x_rows, 128, 0, stream>>>(p);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  switch (linear_token_tile(p.rows, p.experts, p.offsets != nullptr)) {
    case 32: return launch_tiles<32>(p, stream);
    case 64: return launch_tiles<64>(p, stream);
    default: return launch_tiles<128>(p, stream);
  }
}

}  // namespace am
