// Linear layers over 4-bit weights for many tokens: tcgen05 on pairs of SMs (cta_group::2).
//
// The tiles of am_linear_tc.cu with twice the tokens: two CTAs of a cluster share one product of 256
// weight rows x up to 256 tokens.  Each dequantizes 128 of the rows into its own TMEM and loads
// half of the tokens' activations; the leader's MMAs (M = 256) read the operands of both.  A
// weight is dequantized once for 256 tokens instead of 128, and an activation is brought into
// shared memory and read from it for 256 weight rows by each SM: at the power cap that these sizes
// run at, the work saved beside the MMAs is clock rate gained for them.
//
// Per CTA: one thread streams the codes (plain: 128 rows of the matrix; gated: 64 rows of each, 16 and
// 16 alternating in TMEM, so that one thread reads a row's gate and its partner), one the
// activations; their full barrier, shared with the dequantized operand's, is the leader's.  8
// warps dequantize (two groups of 4, a 64-input slab of a step each) and write the output: TMEM holds
// the 256-column accumulator and eight operand slabs.  The MMA shape follows the item: N is its tokens
// rounded up to 32.  4096 tokens 14336x4096 gated: 668 us, 1.44 PFLOP/s, in a burst and 780 at the power
// cap, which bounds it (ncu, 2048 tokens 16384x4096 gated: tensor pipe 81 % busy, issue slots 34 %); a tile of few inputs is bound by its output (32 experts 2880x2880 gated, 512
// rows each: 510 to 540 us, 1.0 to 1.07 PFLOP/s).  Waits are bounded as in am_linear_tc.cu; the CTAs of a pair leave together.
#include <algorithm>
#include <climits>

#include "am_internal.h"
#include "am_linear.cuh"
#include "am_tcgen05.cuh"

namespace am {

namespace tc2 {

// D (TMEM of both CTAs) [+]= A (TMEM of both, 128 rows each) x B (shared memory of both, N / 2 rows
// each, at the same offset).  Issued by the leader.
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t id, uint32_t accum) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(b), "r"(id), "r"(accum));
}

// Arrive on both CTAs' copy of `bar` once every MMA this thread issued before has completed.
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// Tile load into this CTA's shared memory that completes on the leader's copy of `bar`.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar & 0xFEFFFFFFu)
      : "memory");
}

// Arrive on an mbarrier of the cluster (address from mapa).  What it hands over is TMEM, ordered by the
// tcgen05 fences around the arrival and the wait; a cluster-scope release of all memory before it
// would cost 320 cycles an arrival instead of 8 (measured).
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(addr) : "memory");
}

}  // namespace tc2

template <bool GATED>
struct PairLayout {
  static constexpr int CS = 4;               // code stages (128 rows x 256 inputs)
  static constexpr int ST = 4;               // steps in flight: two slabs (64 inputs) of operand and activations
  static constexpr int DW = 8;               // dequantization warps: 4 a slab of a step
  static constexpr int THREADS = 32 * (DW + 3);  // + codes, activations, MMA
  static constexpr int CSTAGE = 128 * 128;
  static constexpr int XSLAB = 128 * 128;    // 128 tokens x 64 inputs
  static constexpr int OFF_C = 0;
  static constexpr int OFF_X = OFF_C + CS * CSTAGE;
  static constexpr int OFF_OUT = OFF_X + ST * 2 * XSLAB;           // kOutPitch bytes a token of a warp
  static constexpr int OUT = 16 * (GATED ? kOutPitch16 : kOutPitch);
  static constexpr int OFF_SCALE = OFF_OUT + DW * OUT;             // two tiles' token scales
  static constexpr int OFF_BAR = OFF_SCALE + 2 * 256 * 4;
  // FULL: a step's operand is in the TMEM of both CTAs and its activations in their shared memory (the
  // leader's copy); EMPTY: the step's MMAs are done (both copies).
  static constexpr int B_CFULL = 0, B_CEMPTY = CS, B_FULL = 2 * CS, B_EMPTY = B_FULL + ST;
  static constexpr int B_DFULL = B_EMPTY + ST, B_DEMPTY = B_DFULL + 1, B_SFULL = B_DEMPTY + 1, B_SEMPTY = B_SFULL + 2;
  static constexpr int B_DRAIN = B_SEMPTY + 2, B_COUNT = B_DRAIN + 1;
  static constexpr int SMEM = OFF_BAR + B_COUNT * 8 + 16;
  static constexpr int A_COL = 256;  // D at 0, A[step][slab] at A_COL + 32 (2 step + slab)
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  static __device__ int arrivals(int i) {
    if (i >= B_CEMPTY && i < B_CEMPTY + CS) return DW;
    if (i >= B_FULL && i < B_FULL + ST) return 2 * DW + 1;  // both CTAs' warps, the activations' thread
    if (i == B_DEMPTY) return 2 * DW;
    if (i >= B_SEMPTY && i < B_SEMPTY + 2) return DW;
    return 1;
  }
};

struct PairParams {
  LinearParams p;
  int32_t row_tiles;    // tiles of 256 weight rows (gated: 128 of each matrix)
  int32_t tile_tokens;  // tokens of an item, at most: a multiple of 32 up to 256
};

// (out of line and with nothing kept for it: the kernel's loops do not notice)
template <int CTA_ROWS>
__device__ __noinline__ void pair_store_nonfinite(const PairParams& f) {
  const int b = static_cast<int>(blockIdx.x);
  store_nonfinite_tiles(f.p, f.tile_tokens, f.row_tiles, 2 * CTA_ROWS, (b & 1) * CTA_ROWS, CTA_ROWS, b >> 1,
                        static_cast<int>(gridDim.x) >> 1, 0, 1);
}

template <bool GATED, int PARTS>
__global__ void __launch_bounds__(PairLayout<GATED>::THREADS, 1) linear_pair_kernel(const __grid_constant__ PairParams f) {
  using LY = PairLayout<GATED>;
  constexpr int CS = LY::CS, ST = LY::ST, DW = LY::DW;
  constexpr int CODES_WARP = DW, X_WARP = DW + 1, MMA_WARP = DW + 2;
  constexpr int CTA_ROWS = GATED ? 64 : 128;  // output rows of a CTA
  const LinearParams& p = f.p;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s_base = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + LY::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + LY::OFF_BAR + LY::B_COUNT * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + LY::OFF_BAR + LY::B_COUNT * 8 + 4);
  volatile int* nonfinite = abort_flag + 1;  // one of this CTA's tokens is not finite
  float* tok_scale = reinterpret_cast<float*>(smem + LY::OFF_SCALE);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
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
  const int rank = static_cast<int>(blockIdx.x) & 1;
  const int first = static_cast<int>(blockIdx.x) >> 1, step = static_cast<int>(gridDim.x) >> 1;
  const int tiles = count_items(p, f.tile_tokens) * f.row_tiles;
  if (first >= tiles) {  // both CTAs of the pair
    griddep_wait();  // (a grid may not be complete before the one it depends on: the next one waits for this one only)
    return;
  }
  const int stages = p.pstride >> 2;  // quads of groups
  const int slabs = p.groups, steps = (slabs + 1) / 2 * PARTS;  // (a step's parts follow one another)

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(tmem_slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::);
  } else if (warp == CODES_WARP) {
    for (int i = lane; i < LY::B_COUNT; i += 32) mbar_init(bar(i), LY::arrivals(i));
    if (lane == 0) *abort_flag = *nonfinite = 0;
    fence_mbar_init();
  }
  tc::fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before either arrives on the other's
  tc::fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  int issued_c = 0, issued_x = 0;  // loads issued (their own threads' counts)
  bool mma_issued = false;
  bool ok = true;
  if (warp == CODES_WARP) {
    Ring<CS> ring;
    for (int tile = first; tile < tiles && ok; tile += step) {
      int lo, hi;
      const int e = find_item(p, tile / f.row_tiles, f.tile_tokens, lo, hi);
      const int y = e * p.n_out + tile % f.row_tiles * 2 * CTA_ROWS + rank * CTA_ROWS;
      if (lane == 0) {
        for (int c = 0; c < stages; ++c) {
          ok = wait_quick(bar(LY::B_CEMPTY + ring.s), ring.ph ^ 1u, p.wait_ns, abort_flag);
          if (!ok) break;
          const uint32_t full = bar(LY::B_CFULL + ring.s), dst = s_base + LY::OFF_C + ring.s * LY::CSTAGE;
          mbar_arrive_expect_tx(full, LY::CSTAGE);
          am::tma_load_2d(dst, &p.tmap_w[0], c * 128, y, full);
          am::tma_load_2d(dst + LY::CSTAGE / 2, &p.tmap_w[GATED ? 1 : 0], c * 128, GATED ? y : y + 64, full);
          ++issued_c;
          ring.next();
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
  } else if (warp == X_WARP) {
    griddep_wait();  // the activations are written
    Ring<ST> ring;
    int k = 0;
    for (int tile = first; tile < tiles && ok; tile += step, ++k) {
      int lo, hi;
      find_item(p, tile / f.row_tiles, f.tile_tokens, lo, hi);
      const int half = ((hi - lo + 31) & ~31) >> 1;  // tokens of a CTA
      const int y = lo + rank * half;
      for (int i = 0; i < steps; ++i) {
        ok = wait(LY::B_EMPTY + ring.s, ring.ph ^ 1u);
        if (!ok) break;
        const uint32_t dst = s_base + LY::OFF_X + ring.s * 2 * LY::XSLAB;
        const int n = min(2, slabs - i / PARTS * 2);
        if (lane == 0) {
          const uint32_t full = bar(LY::B_FULL + ring.s);
          if (rank == 0) mbar_arrive_expect_tx(full, 2 * n * LY::XSLAB);  // both CTAs' bytes
          for (int s = 0; s < n; ++s) tc2::tma_load_2d(dst + s * LY::XSLAB, &p.tmap_x, (i / PARTS * 2 + s) * 128, y, full);
        }
        ++issued_x;
        ring.next();
        if (i == min(ST, steps) - 1) {  // behind the first loads: the tokens' powers of two
          const int b = k & 1;
          ok = wait(LY::B_SEMPTY + b, ((k >> 1) & 1) ^ 1);
          if (!ok) break;
          bool marked = false;
          for (int j = lane; j < 256; j += 32) {
            const float ts = lo + j < hi ? p.xscale[lo + j] : 0.0f;
            tok_scale[b * 256 + j] = ts;
            marked |= isnan(ts);
          }
          if (__any_sync(0xffffffffu, marked)) *nonfinite = 1;  // (the warp together: a divergent store made the loops spill)
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(LY::B_SFULL + b));
        }
      }
    }
  } else if (warp == MMA_WARP) {
    const bool lead = elect_one();
    Ring<ST> ring;
    uint32_t dph = 1;
    for (int tile = first; tile < tiles && ok && rank == 0; tile += step, dph ^= 1u) {
      int lo, hi;
      find_item(p, tile / f.row_tiles, f.tile_tokens, lo, hi);
      const uint32_t id = tc::idesc(256, (hi - lo + 31) & ~31, false);
      // One wait and one commit a step (8 MMAs of 128 cycles); the wait for step i + 1 stands before the
      // last MMAs of step i.  (With separate barriers for operand and activations the issuing thread
      // itself took 1450 cycles a step.)  The warp stays converged and one lane issues, as in
      // linear_tiles_kernel.
      ok = wait(LY::B_DEMPTY, dph) && wait(LY::B_FULL + ring.s, ring.ph);
      for (int i = 0; i < steps && ok; ++i) {
        tc::fence_after();
        const uint64_t xd = tc::sdesc(s_base + LY::OFF_X + ring.s * 2 * LY::XSLAB, 16, 1024);
        const uint32_t a = tmem + LY::A_COL + ring.s * 64, done = bar(LY::B_EMPTY + ring.s);
        const bool both = 2 * (i / PARTS) + 1 < slabs;
        ring.next();
        if (lead) {
          // (descriptor addresses count 16-byte units: 32 bytes of a swizzled row are 16 inputs)
          tc2::mma_ts(tmem, a, xd, id, i > 0 ? 1u : 0u);
#pragma unroll
          for (int ks = 1; ks < 4; ++ks) tc2::mma_ts(tmem, a + ks * 8, xd + ks * 2, id, 1u);
          if (both) {
            tc2::mma_ts(tmem, a + 32, xd + LY::XSLAB / 16, id, 1u);
            tc2::mma_ts(tmem, a + 40, xd + LY::XSLAB / 16 + 2, id, 1u);
          }
        }
        mma_issued = lead;
        if (i + 1 < steps) ok = wait(LY::B_FULL + ring.s, ring.ph);
        if (lead) {
          if (both) {
            tc2::mma_ts(tmem, a + 48, xd + LY::XSLAB / 16 + 4, id, 1u);
            tc2::mma_ts(tmem, a + 56, xd + LY::XSLAB / 16 + 6, id, 1u);
          }
          tc2::commit(done);
        }
      }
      if (ok && lead) tc2::commit(bar(LY::B_DFULL));
    }
  } else {
    // ---- dequantization (as in linear_tiles_kernel): a weight row a thread, slab `group` of every step
    const int group = warp >> 2, quarter = warp & 3;
    const int which = GATED ? lane >> 4 : 0;                          // the matrix of this lane's row
    const int rr = GATED ? quarter * 16 + (lane & 15) : quarter * 32 + lane;  // output row within the CTA
    const int r = which * 64 + rr;                                    // row of the code stage
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t a_base = tmem + LY::A_COL + group * 32 + lane_base;
    const uint32_t lead_full = dsmem_addr(bar(LY::B_FULL), 0), lead_dempty = dsmem_addr(bar(LY::B_DEMPTY), 0);
    Ring<CS> cr;
    Ring<ST> ring;
    const uint4* prow = nullptr;  // parameters of this thread's weight row, a code stage each
    uint4 pv = make_uint4(0, 0, 0, 0);
    auto dequant = [&](int c0, int c1) {  // code stages [c0, c1)
      for (int c = c0; c < c1 && ok; ++c) {
        const uint32_t ps[2] = {group == 0 ? pv.x : pv.y, group == 0 ? pv.z : pv.w};
        pv = __ldg(prow + min(c + 1, stages - 1));
        ok = wait(LY::B_CFULL + cr.s, cr.ph);
        if (!ok) break;
        const uint8_t* crow = smem + LY::OFF_C + cr.s * LY::CSTAGE + r * 128;
        const int in_stage = min(4, slabs - 4 * c);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          if (st * 2 >= in_stage) break;
          const int s = st * 2 + group;
          uint4 w0, w1;
          if (s < in_stage) {
            w0 = *reinterpret_cast<const uint4*>(crow + (((2 * s) ^ (r & 7)) << 4));
            w1 = *reinterpret_cast<const uint4*>(crow + (((2 * s + 1) ^ (r & 7)) << 4));
          }
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            uint32_t o[32];
            if (s < in_stage) dequant_group<PARTS>(w0, w1, ps[st], part, o);
            ok = wait(LY::B_EMPTY + ring.s, ring.ph ^ 1u);
            if (!ok) break;
            tc::fence_after();
            if (s < in_stage) tc::tmem_st32(a_base + ring.s * 64, o);
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc2::arrive_cluster(lead_full + ring.s * 8);
            ring.next();
          }
          if (!ok) break;
        }
        if (!ok) break;
        __syncwarp();  // the stage's codes are in registers
        if (lane == 0) mbar_arrive(bar(LY::B_CEMPTY + cr.s));
        cr.next();
      }
    };
    // ---- output of the k-th tile: group g takes every other 16 tokens.  The accumulators come in mma
    // fragments (thread (g8, t4): rows g8 + 8 i, tokens 2 t4, + 1 of eight; gated: of the gate for i < 2 and
    // of its partner above), leave transposed through the warp's own shared memory, a token's 32
    // rows as 64 bytes (gated 16, 32).
    auto output = [&](int k, int lo, int hi, int n0, int64_t wbase) {
      const int b = k & 1;
      const int g8 = lane >> 2, t4 = lane & 3;
      const int row0 = n0 + quarter * (GATED ? 16 : 32);  // of the warp's
      float rs[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        rs[i] = __ldg(p.row_scale[GATED ? i >> 1 : 0] + wbase + min(row0 + g8 + 8 * (GATED ? i & 1 : i), p.n_out - 1));
      ok = ok && wait(LY::B_DFULL, k & 1) && wait(LY::B_SFULL + b, (k >> 1) & 1);
      if (!ok) return;
      tc::fence_after();
      uint8_t* so = smem + LY::OFF_OUT + warp * LY::OUT;
      float next[2][8];  // the next 16 tokens, loaded behind this one's work: [16 rows][token block, row
                         // g8 or g8 + 8, token]
      auto load = [&](int cb) {
        tc::tmem_ld_16x16_nowait(tmem + cb + lane_base, next[0]);
        tc::tmem_ld_16x16_nowait(tmem + cb + lane_base + (16u << 16), next[1]);
      };
      if (lo + group * 16 < hi) load(group * 16);
#pragma unroll 1
      for (int cb = group * 16; lo + cb < hi; cb += 32) {
        float v[2][8];
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[0][i] = next[0][i];
          v[1][i] = next[1][i];
        }
        if (lo + cb + 32 < hi) load(cb + 32);
        float2 ts[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) ts[j] = *reinterpret_cast<const float2*>(tok_scale + b * 256 + cb + 8 * j + 2 * t4);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[h][i] *= rs[2 * h + ((i >> 1) & 1)] * ((i & 1) ? ts[i >> 2].y : ts[i >> 2].x);
        if constexpr (GATED) {
          uint32_t q[2][2];  // [token block][8 rows]: pairs of tokens
#pragma unroll
          for (int i = 0; i < 8; i += 2)
            q[i >> 2][(i >> 1) & 1] = pack_out(p, silu_mul(v[0][i], v[1][i]), silu_mul(v[0][i + 1], v[1][i + 1]));
          store_tokens_16(p, so, q, lo + cb, hi, row0);
        } else {
          uint32_t q[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              q[j][2 * h] = pack_out(p, v[h][4 * j], v[h][4 * j + 1]);
              q[j][2 * h + 1] = pack_out(p, v[h][4 * j + 2], v[h][4 * j + 3]);
            }
          store_tokens(p, so, q, lo + cb, hi, row0);
        }
      }
      // the accumulator and the tokens' scales are read
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        tc2::arrive_cluster(lead_dempty);
        mbar_arrive(bar(LY::B_SEMPTY + b));
      }
    };
    // The first ST steps of a tile are dequantized before the output of the one before it: they fill
    // the operand buffers while its last MMAs run, and the next MMAs start with the output done.
    constexpr int AHEAD = LY::ST / (2 * PARTS);  // stages
    int k = 0, lo = 0, hi = 0, n0 = 0;
    int64_t wbase = 0;
    for (int tile = first; tile < tiles && ok; tile += step, ++k) {
      int lo_n, hi_n;
      const int e = find_item(p, tile / f.row_tiles, f.tile_tokens, lo_n, hi_n);
      const int n0_n = tile % f.row_tiles * 2 * CTA_ROWS + rank * CTA_ROWS;
      const int64_t wbase_n = (int64_t)e * p.n_out;
      prow = reinterpret_cast<const uint4*>(p.params[which] + (wbase_n + min(n0_n + rr, p.n_out - 1)) * p.pstride);
      pv = __ldg(prow);
      dequant(0, min(AHEAD, stages));
      if (ok && k > 0) output(k - 1, lo, hi, n0, wbase);
      if (ok) dequant(min(AHEAD, stages), stages);
      lo = lo_n;
      hi = hi_n;
      n0 = n0_n;
      wbase = wbase_n;
    }
    if (ok && k > 0) output(k - 1, lo, hi, n0, wbase);
  }
  if (!ok) *abort_flag = 1;
  __syncthreads();

  // ---- teardown: after an abort, this CTA's loads (and the leader's MMAs) in flight finish (bounded);
  // then both CTAs are done with each other's memory
  if (*abort_flag) {
    constexpr uint64_t kDrainNs = 100000000ull;
    if (warp == CODES_WARP && lane == 0)
      for (int j = max(0, issued_c - CS); j < issued_c; ++j)
        mbar_wait_bounded(bar(LY::B_CFULL + j % CS), (j / CS) & 1, kDrainNs);
    if (warp == X_WARP && lane == 0 && rank == 0)  // (both CTAs' loads complete on the leader's barriers)
      for (int j = max(0, issued_x - ST); j < issued_x; ++j)
        mbar_wait_bounded(bar(LY::B_FULL + j % ST), (j / ST) & 1, kDrainNs);
    if (warp == MMA_WARP && mma_issued) {
      tc2::commit(bar(LY::B_DRAIN));
      mbar_wait_bounded(bar(LY::B_DRAIN), 0, kDrainNs);
    }
    if (tid == 0) flag_status(p.status, AM_STATUS_TIMEOUT);
  }
  tc::fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 0) {
    tc::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
  }
  if (*nonfinite) pair_store_nonfinite<CTA_ROWS>(f);
}

// ---------------------------------------------------------------- host
template <bool GATED, int PARTS>
static cudaError_t launch_pair_t(const PairParams& f, int clusters, int dev, cudaStream_t stream) {
  auto kfn = linear_pair_kernel<GATED, PARTS>;
  static unsigned long long done = 0;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!bit || !(__atomic_load_n(&done, __ATOMIC_ACQUIRE) & bit)) {
    const cudaError_t err = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, PairLayout<GATED>::SMEM);
    if (err != cudaSuccess) return err;
    if (bit) __atomic_fetch_or(&done, bit, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(PairLayout<GATED>::THREADS);
  cfg.dynamicSmemBytes = PairLayout<GATED>::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kfn, f);
}

cudaError_t launch_linear_pair(const LinearParams& p, cudaStream_t stream) {
  int dev = 0;
  const int sms = sm_count(&dev);
  if (sms == 0) return cudaErrorInvalidDevice;
  const bool gated = p.codes[1] != nullptr;
  const int rows = gated ? 128 : 256, parts = weight_parts(gated, p.bf16);
  PairParams f{};
  f.p = p;
  f.row_tiles = (p.n_out + rows - 1) / rows;
  const int pairs = sms / 2;
  f.tile_tokens = 256;
  int64_t items = p.offsets != nullptr ? (int64_t)std::min(p.experts, p.rows) + p.rows / 256 : 0;
  if (p.offsets == nullptr) {
    // One matrix: the cut of the tokens that ends first.  A step of 128 inputs measured 4.6 cycles a token
    // (1178 for 256), 950 at least (the MMA thread), a tile's start and output 8000.
    const double steps = (p.groups + 1) / 2 * parts;
    double best = 0.0;
    for (int n = (p.rows + 255) / 256, tries = 0; tries < 12; ++n, ++tries) {
      const int tokens = ((p.rows + n - 1) / n + 31) & ~31;
      const int64_t tiles = (int64_t)f.row_tiles * ((p.rows + tokens - 1) / tokens);
      const double cost = (double)((tiles + pairs - 1) / pairs) * (steps * std::max(4.6 * tokens, 950.0) + 8000.0);
      if (tries == 0 || cost < best) {
        best = cost;
        f.tile_tokens = tokens;
      }
    }
    items = (p.rows + f.tile_tokens - 1) / f.tile_tokens;
  }
  if (f.row_tiles * items > INT_MAX) return cudaErrorNotSupported;
  const int clusters = static_cast<int>(std::min<int64_t>(f.row_tiles * items, pairs));
  if (parts == 2) return launch_pair_t<true, 2>(f, clusters, dev, stream);
  return gated ? launch_pair_t<true, 1>(f, clusters, dev, stream) : launch_pair_t<false, 1>(f, clusters, dev, stream);
}

}  // namespace am
