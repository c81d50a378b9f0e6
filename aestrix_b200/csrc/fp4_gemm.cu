// fp4_gemm.cu — many bf16 rows times microscaled 4-bit weights on CTA pairs:
// y = x W^T, act(x Wg^T) * (x Wu^T), and the gradients dx = dy W.
//
// Tensor-bound (tcgen05.mma.cta_group::2, bf16 operands, 256 x 256 output
// tiles, persistent). CTA r of a pair holds x rows [128 r, 128 r + 128) of the
// tile (A, by TMA) and decodes its 128 of the tile's 256 columns of B from
// records in shared memory; both halves feed one MMA, each CTA receives its
// 128 rows of f32 accumulators in tensor memory, two buffers of 256 columns,
// so that the epilogue of one tile overlaps the main loop of the next.
// A K step is 64 wide. Forward (K = columns of W): CTA r decodes rows of one
// record, 64 columns a step, into a K-major tile; the gated form's rank 0
// takes the gate's record and rank 1 the up projection's, so that both
// projections of 128 outputs lie in one accumulator. Backward (K = rows of W):
// a record is 128 rows of K and 256 output columns; CTA r decodes its 128
// columns of 64 rows a step. The bytes a decoded row leaves in shared memory
// are the same either way; the MMA reads them as an MN-major operand.
// Decoded values are exact in bf16 (at most 6 significant bits), so no
// rounding enters before the f32 sums; tensor scales are applied to those.
//   warp 0      producer of the A boxes
//   warp 1      MMA issuer (even CTA only)
//   warp 2      tensor-memory allocation
//   warp 3      producer of the records (one bulk copy each)
//   warps 4-11  epilogue (tensor-memory lane quadrant = warp % 4; half of the
//               columns each)
//   warps 12-27 decode: four groups of four warps, two per unit (below); with
//               two groups a unit took 1.05 us, nearly all of it one group's
//               latency
// A unit of the pipeline is two K steps, decoded by two groups; the next unit by
// the other two. Barriers: an A box lands on afull (five places); the decode
// warps write their step's part of B and arrive on the even CTA's bready (three
// units; both CTAs' sixteen warps, and the odd CTA's warp 1 for its A boxes);
// the MMA thread waits for that and for its own boxes, issues eight MMAs and
// commits once, to `done` of both CTAs, which frees the unit's A and B. `done`
// has six barriers, a multiple of both rings' units and even, so that each wait
// knows its phase although a group sees every other unit. A record is released
// (rempty) by the decode warps that read it.
// Tiles that would leave a last wave of the clusters mostly empty are split
// along K evenly over the clusters; their f32 pieces go to the workspace and
// join_kernel adds them in order and applies the epilogue.
// Each kernel lets the stream's next one set up behind it (0.5 to 1 us a call).
// Tensor memory is taken after the wait for the previous kernel: that one may
// hold some, or not have taken its own yet.
// Measured in the 2 ms after a pause, and in a loop, where the power cap leaves
// 1.6 GHz (1.75 the gradient): 512 rows gated 4096 -> 9216 56 us (1.4 PFLOP/s) and
// 64, 1111 rows 9216 -> 4104 82 and 93 (tiles of 256 use 82 % of the products), 512
// rows back through 4096 -> 7680 31.5 and 33 (60 tiles on 74 pairs). The tensor pipe
// is busy 63 to 66 % of the kernel.
#include <algorithm>

#include "fp4_internal.h"
#include "fp4_tile.cuh"

namespace aex {
namespace fp4 {

constexpr int kGThreads = 896;
constexpr int kGA = 5;      // places for A boxes, one K step each
constexpr int kGB = 3;      // units (two steps) of decoded B
constexpr int kGDone = 6;
constexpr int kGRecs = 2;
constexpr int kGTile = 128 * 64 * 2;  // one operand of one CTA and step
constexpr int kGOffB = kGA * kGTile;
constexpr int kGRecSlot = rec_bytes(AEX_FP4_NV);
constexpr int kGOffRec = kGOffB + kGB * 2 * kGTile;
constexpr int kGOffBar = kGOffRec + kGRecs * kGRecSlot;
// afull[A], bready[B], done[6], rfull[R], rempty[R], accf[2], acce[2], drain
constexpr int kGNumBars = kGA + kGB + kGDone + 2 * kGRecs + 5;
constexpr int kGSmem = kGOffBar + kGNumBars * 8 + 16 + 1024;
static_assert(kGSmem <= 232448, "fp4 GEMM exceeds the shared-memory limit");

enum GemmMode : int { kPlain = 0, kGatedFwd = 1, kGatedGrad = 2, kDgrad = 3 };

// The gated projection's gradients in place of its result.
struct GradOut {
  float fold0, fold1;  // the tensor scales that dg and du take on
  const uint16_t* dh;
  int64_t lddh;
  uint16_t* dg;
  uint16_t* du;
  int64_t ldg;
};

struct GemmParams {
  const uint8_t* w0;
  const uint8_t* w1;
  int k_blocks;  // records along the columns of a weight
  int n_tiles;   // records along its rows
  TileWork work;
  TileOut o;
  GradOut grad;
  uint32_t zero;  // 0 (arrive_after_loads)
  int* status;
};

// dh of 8 columns (col a multiple of 8), zeros past the last. Plain loads: the previous kernel, which may have written
// it, ran when this one was set up, and the read-only path is for what nobody writes meanwhile.
__device__ __forceinline__ uint4 grad_load(const TileOut& o, const GradOut& p, int64_t row, int col) {
  const int left = o.cols - col;
  uint32_t d[4] = {0, 0, 0, 0};
  const uint16_t* src = p.dh + row * p.lddh + col;
  if (left >= 8) return *reinterpret_cast<const uint4*>(src);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    d[i] = (2 * i < left ? src[2 * i] : 0u) | ((2 * i + 1 < left ? static_cast<uint32_t>(src[2 * i + 1]) : 0u) << 16);
  return make_uint4(d[0], d[1], d[2], d[3]);
}

// dg, du of 8 columns from g, u (already scaled) and dh. They are rounded to bf16 here, as operands of the tensor
// core's next product (what bf16 leaves of them would take that product a second time). So dx is off by 0.0023 of its
// size (1024 rows, 4096 -> 9216), where its own last rounding alone comes to 0.0017.
__device__ __forceinline__ void grad8(const TileOut& o, const GradOut& p, int64_t row, int col, const float* g,
                                      const float* u, const uint4& dh) {
  if (col >= o.cols) return;
  const uint32_t d[4] = {dh.x, dh.y, dh.z, dh.w};
  uint32_t og[4], ou[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a[2], b[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float gi = g[2 * i + e], ui = u[2 * i + e];
      const float dv = e ? bf16hi_to_f32(d[i]) : bf16lo_to_f32(d[i]);
      const float sg = sigmoid<true>(sigmoid_arg(gi, o.activation));
      const float act = gi * sg;
      a[e] = dv * ui * fmaf(act * (1.f - sg), sigmoid_arg_slope(gi, o.activation), sg) * p.fold0;
      b[e] = dv * act * p.fold1;
    }
    og[i] = pack_bf16x2(a[0], a[1]);
    ou[i] = pack_bf16x2(b[0], b[1]);
  }
  // dg and du have rows of whole vectors: the columns past the last are written, never read
  *reinterpret_cast<uint4*>(p.dg + row * p.ldg + col) = make_uint4(og[0], og[1], og[2], og[3]);
  *reinterpret_cast<uint4*>(p.du + row * p.ldg + col) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
}

template <int kFormat, int kMode>
__global__ void __launch_bounds__(kGThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tm0, const __grid_constant__ CUtensorMap tm1,
                const __grid_constant__ GemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kGOffBar);
  uint64_t* afull = bars;
  uint64_t* bready = afull + kGA;
  uint64_t* done = bready + kGB;
  uint64_t* rfull = done + kGDone;
  uint64_t* rempty = rfull + kGRecs;
  uint64_t* accf = rempty + kGRecs;
  uint64_t* acce = accf + 2;
  uint64_t* drain = acce + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kGNumBars);
  __shared__ int abort_flag;
  constexpr bool kBack = kMode == kDgrad;
  constexpr int kRec = rec_bytes(kFormat);
  constexpr int kUnits = kBack ? 1 : 2;  // units (two K steps) per record

  const int warp = static_cast<int>(warp_id_uniform());
  const int lane = static_cast<int>(lane_id());
  const uint32_t rank = cluster_ctarank();
  const int cluster = static_cast<int>(blockIdx.x >> 1);
  const int clusters = static_cast<int>(gridDim.x >> 1);

  launch_dependents();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kGA; ++s) mbar_init(&afull[s], 1);
    for (int s = 0; s < kGB; ++s) mbar_init(&bready[s], 2 * 8 + 1);
    for (int s = 0; s < kGDone; ++s) mbar_init(&done[s], 1);
    for (int s = 0; s < kGRecs; ++s) {
      mbar_init(&rfull[s], 1);
      mbar_init(&rempty[s], kBack ? 8 : 16);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf[b], 1);
      mbar_init(&acce[b], 2 * 8);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm0);
    if (kBack) prefetch_tmap(&tm1);
  }
  wait_dependency();  // what it reads may be the previous kernel's, and so may the tensor memory
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  // The producers touch this CTA's barriers alone: they start at once and take part in the cluster's barrier when done.
  cluster_arrive();
  if (warp != 0 && warp != 3) cluster_wait();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------ A producer
      const uint32_t done0 = smem_u32(&done[0]);
      int g = 0;  // K steps so far
      bool ok = true;
      TilePiece t;
      for (int i = 0; ok && p.work.piece(cluster, clusters, i, &t); ++i) {
        const int row0 = t.mt * 256 + static_cast<int>(rank) * 128;
        for (int k = t.r0 * kUnits * 2; k < t.r1 * kUnits * 2; ++k, ++g) {
          if (g >= kGA) {
            const int u = (g - kGA) >> 1;  // the unit that used this place
            if (!mbar_wait_cl(done0 + 8 * (u % kGDone), (u / kGDone) & 1, &abort_flag, p.status, kDevTimeoutTma)) {
              ok = false;
              break;
            }
          }
          const int s = g % kGA;
          mbar_arrive_expect_tx(&afull[s], kGTile);
          // dgrad: the second weight's rows follow the first's (p.n_tiles records of two steps)
          const bool second = kBack && k >= 2 * p.n_tiles;
          tma_load_2d(smem + s * kGTile, second ? &tm1 : &tm0, &afull[s], (second ? k - 2 * p.n_tiles : k) * 64, row0);
        }
      }
      if (!ok) {
        // The copies in flight land before the CTA can exit.
        for (int j = (g > kGA ? g - kGA : 0); j < g; ++j) {
          const uint32_t a = smem_u32(&afull[j % kGA]);
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(a, (j / kGA) & 1) && globaltimer_ns() - t0 < kWaitTimeoutNs) {
          }
        }
      }
    }
    __syncwarp();
    cluster_wait();
  } else if (warp == 3) {
    if (lane == 0) {
      // ------------------------------------------------- record producer
      uint32_t s = 0, ph = 0;
      int g = 0;
      bool ok = true;
      TilePiece t;
      for (int i = 0; ok && p.work.piece(cluster, clusters, i, &t); ++i) {
        for (int r = t.r0; r < t.r1; ++r, ++g) {
          if (g >= kGRecs && !mbar_wait(&rempty[s], ph ^ 1, &abort_flag, p.status, kDevTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint8_t* w = p.w0;
          int rt, kb;
          if (kBack) {
            const bool second = r >= p.n_tiles;
            if (second) w = p.w1;
            rt = second ? r - p.n_tiles : r;
            kb = t.nt;
          } else {
            kb = r;
            if (kMode == kPlain) {
              rt = min(2 * t.nt + static_cast<int>(rank), p.n_tiles - 1);  // an odd last tile: columns nobody stores
            } else {
              rt = t.nt;
              if (rank) w = p.w1;
            }
          }
          mbar_arrive_expect_tx(&rfull[s], kRec);
          bulk_load(smem + kGOffRec + s * kGRecSlot, w + (static_cast<size_t>(rt) * p.k_blocks + kb) * kRec, kRec,
                    &rfull[s]);
          if (++s == kGRecs) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) {
        for (int j = (g > kGRecs ? g - kGRecs : 0); j < g; ++j) {
          const uint32_t a = smem_u32(&rfull[j % kGRecs]);
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(a, (j / kGRecs) & 1) && globaltimer_ns() - t0 < kWaitTimeoutNs) {
          }
        }
      }
    }
    __syncwarp();
    cluster_wait();
  } else if (warp == 1) {
    if (lane == 0 && rank == 1) {
      // ------------------------------------- "A landed" of the odd CTA
      const uint32_t afull0 = smem_u32(&afull[0]);
      const uint32_t lead = mapa_shared(smem_u32(&bready[0]), 0);
      uint32_t as = 0, aph = 0, bs = 0;
      bool ok = true;
      TilePiece t;
      for (int i = 0; ok && p.work.piece(cluster, clusters, i, &t); ++i)
        for (int u = t.r0 * kUnits; u < t.r1 * kUnits && ok; ++u) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && mbar_wait_cl(afull0 + 8 * as, aph, &abort_flag, p.status, kDevTimeoutTma);
            if (++as == kGA) {
              as = 0;
              aph ^= 1;
            }
          }
          if (ok) mbar_arrive_cluster(lead + 8 * bs);
          if (++bs == kGB) bs = 0;
        }
    } else if (lane == 0) {
      // ------------------------------------------------------------- MMA
      constexpr uint32_t kIdesc = idesc_bf16_f32(256, 256, false, kBack);
      constexpr uint32_t kBStep = kBack ? 128 : 2;  // 16 K rows of an MN-major tile: 2 KB; of a K-major one: 32 B
      const uint32_t s0 = smem_u32(smem);
      const uint32_t bready0 = smem_u32(&bready[0]), afull0 = smem_u32(&afull[0]), done0 = smem_u32(&done[0]);
      const uint64_t da0 = sdesc_sw128(s0, 16, 1024);
      const uint64_t db0 = sdesc_sw128(s0 + kGOffB, kBack ? 8192 : 16, 1024);
      uint32_t as = 0, aph = 0, bs = 0, bph = 0, ds = 0;
      bool ok = true;
      TilePiece t;
      for (int i = 0; ok && p.work.piece(cluster, clusters, i, &t); ++i) {
        const int b = i & 1;
        if (i >= 2 && !mbar_wait_cl(smem_u32(&acce[b]), ((i >> 1) + 1) & 1, &abort_flag, p.status, kDevTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + b * 256;
        const int n = (t.r1 - t.r0) * kUnits;
        for (int u = 0; u < n; ++u) {
          if (!mbar_wait_cl(bready0 + 8 * bs, bph, &abort_flag, p.status, kDevTimeoutMma)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!mbar_wait_cl(afull0 + 8 * as, aph, &abort_flag, p.status, kDevTimeoutMma)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t da = da0 + ((as * kGTile) >> 4), db = db0 + (((2 * bs + h) * kGTile) >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_ss_pair(d, da + kk * 2, db + kk * kBStep, kIdesc, (u > 0 || h > 0 || kk > 0) ? 1u : 0u);
            if (++as == kGA) {
              as = 0;
              aph ^= 1;
            }
          }
          if (!ok) break;
          umma_commit_both(done0 + 8 * ds);
          if (++ds == kGDone) ds = 0;
          if (++bs == kGB) {
            bs = 0;
            bph ^= 1;
          }
        }
        if (!ok) break;
        umma_commit_both(smem_u32(&accf[b]));
      }
      // Waited for on abort too: no MMA is in flight at the teardown.
      umma_commit_pair(smem_u32(drain));
      int no_abort = 0;
      mbar_wait_cl(smem_u32(drain), 0, &no_abort, p.status, kDevTimeoutMma);
    }
  } else if (warp >= 4 && warp < 12) {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3, half = (warp - 4) >> 2;
    TilePiece t;
    for (int i = 0; p.work.piece(cluster, clusters, i, &t); ++i) {
      const int b = i & 1;
      const int in_tile = static_cast<int>(rank) * 128 + quad * 32 + lane;
      const int64_t row = static_cast<int64_t>(t.mt) * 256 + in_tile;
      // dh is loaded sixteen columns ahead (1411 rows, 160 -> 9008: 73.9 us when it was loaded where it is used, 69.3)
      uint4 dh[2];
      const int dcol = t.nt * 128 + 64 * half;
      const bool grad = kMode == kGatedGrad && t.slot < 0 && row < p.o.m;
      if (kMode == kGatedGrad) {
        dh[0] = dh[1] = make_uint4(0, 0, 0, 0);
        if (grad) dh[0] = grad_load(p.o, p.grad, row, dcol), dh[1] = grad_load(p.o, p.grad, row, dcol + 8);
      }
      if (!mbar_wait_warp_cl(smem_u32(&accf[b]), (i >> 1) & 1, &abort_flag, p.status, kDevTimeoutEpilogue)) break;
      tc_fence_after();
      const uint32_t tbase = tmem + (static_cast<uint32_t>(quad * 32) << 16) + b * 256;
      if (t.slot >= 0) {
        store_piece(p.work, t.slot, in_tile, row < p.o.m, half, tbase);
      } else if (kMode != kGatedGrad) {
        tile_half<kMode == kGatedFwd>(p.o, row, t.nt, half, tbase);
      } else {
#pragma unroll 1
        for (int c = 0; c < 64; c += 16) {
          float g[16], u[16];
          const uint4 d0 = dh[0], d1 = dh[1];
          if (grad && c + 16 < 64) {
            dh[0] = grad_load(p.o, p.grad, row, dcol + c + 16);
            dh[1] = grad_load(p.o, p.grad, row, dcol + c + 24);
          }
          tmem_read<16>(tbase + 64 * half + c, g);
          tmem_read<16>(tbase + 128 + 64 * half + c, u);
          if (grad) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              g[e] *= p.o.alpha0;
              u[e] *= p.o.alpha1;
            }
            grad8(p.o, p.grad, row, dcol + c, g, u, d0);
            grad8(p.o, p.grad, row, dcol + c + 8, g + 8, u + 8, d1);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acce[b]), 0));
    }
  } else if (warp >= 12) {
    // -------------------------------------------------------------- decode
    const int group = ((warp - 12) >> 2) & 1, turn = (warp - 12) >> 3;
    const int dt = (warp & 3) * 32 + lane;
    const uint32_t done0 = smem_u32(&done[0]);
    const uint32_t bready_lead0 = mapa_shared(smem_u32(&bready[0]), 0);
    uint32_t bs = 0, ds = kGDone - kGB, dph = 1, rs = 0, rph = 0;  // ds: the unit kGB before this one
    int g = 0;                                                     // units so far
    bool ok = true;
    TilePiece t;
    for (int i = 0; ok && p.work.piece(cluster, clusters, i, &t); ++i) {
      const int n = (t.r1 - t.r0) * kUnits;
      for (int u = 0; u < n; ++u, ++g) {
        const uint32_t cb = bs, cds = ds, cdph = dph, crs = rs, crph = rph;
        if (++bs == kGB) bs = 0;
        if (++ds == kGDone) {
          ds = 0;
          dph ^= 1;
        }
        if ((u & (kUnits - 1)) == kUnits - 1 && ++rs == kGRecs) {
          rs = 0;
          rph ^= 1;
        }
        if ((g & 1) != turn) continue;
        const int k = 2 * u + group;  // this group's step, from the piece's first
        if (!mbar_wait_warp(&rfull[crs], crph, &abort_flag, p.status, kDevTimeoutProducer)) {
          ok = false;
          break;
        }
        const uint8_t* rec = smem + kGOffRec + crs * kGRecSlot;
        // r: row of the record; cp: its 64-column part; dst: that row in B
        int r, cp;
        uint8_t* dst = smem + kGOffB + (2 * cb + group) * kGTile;
        if (kBack) {
          r = (k & 1) * 64 + (dt & 63);
          cp = 2 * static_cast<int>(rank) + (dt >> 6);
          dst += (dt >> 6) * 8192 + (dt & 63) * 128;
        } else {
          r = dt;
          cp = k & 3;
          dst += dt * 128;
        }
        const int sw = r & 7;  // the row's swizzle, in the record and in B (a multiple of 8 rows apart)
        const uint4 c0 = *reinterpret_cast<const uint4*>(rec + r * 128 + (((2 * cp) ^ sw) << 4));
        const uint4 c1 = *reinterpret_cast<const uint4*>(rec + r * 128 + (((2 * cp + 1) ^ sw) << 4));
        uint32_t sc;
        if (kFormat == AEX_FP4_NV)
          sc = *reinterpret_cast<const uint32_t*>(rec + scale_off(r, cp));
        else
          sc = *reinterpret_cast<const uint16_t*>(rec + scale_off(r, cp >> 1) + (cp & 1) * 2);
        // this warp's only read of the record
        arrive_after_loads(smem_u32(&rempty[crs]), c0.x | c0.y | c0.z | c0.w | c1.x | c1.y | c1.z | c1.w | sc, p.zero,
                           lane);
        if (g >= kGB && !mbar_wait_warp_cl(done0 + 8 * cds, cdph, &abort_flag, p.status, kDevTimeoutMma)) {
          ok = false;
          break;
        }
        const uint32_t ws[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        if (kFormat == AEX_FP4_MX && (sc & 0xFFu) <= 128u && (sc >> 8) <= 128u) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t s2 = mx_scale_from_tiny(j < 4 ? sc & 0xFFu : sc >> 8);
            *reinterpret_cast<uint4*>(dst + ((j ^ sw) << 4)) =
                make_uint4(mul_bf16x2(code_pair_tiny(ws[j], 0), s2), mul_bf16x2(code_pair_tiny(ws[j], 1), s2),
                           mul_bf16x2(code_pair_tiny(ws[j], 2), s2), mul_bf16x2(code_pair_tiny(ws[j], 3), s2));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            // nvfp4: a scale every two words, mxfp4: every four
            const uint32_t s2 =
                scale_pair<kFormat>((sc >> (kFormat == AEX_FP4_NV ? 8 * (j >> 1) : 8 * (j >> 2))) & 0xFFu);
            *reinterpret_cast<uint4*>(dst + ((j ^ sw) << 4)) =
                make_uint4(decode_pair<kFormat>(ws[j], 0, s2), decode_pair<kFormat>(ws[j], 1, s2),
                           decode_pair<kFormat>(ws[j], 2, s2), decode_pair<kFormat>(ws[j], 3, s2));
          }
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(bready_lead0 + 8 * cb);
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // no peer access to this CTA's shared or tensor memory after this point
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

template <int kMode>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ GemmParams p) {
  constexpr bool kGated = kMode == kGatedFwd || kMode == kGatedGrad;
  join_tile<kGated>(p.work, p.o.m, [&](int64_t row, int nt, int c, const float* v, const float* u) {
    if (kMode == kGatedGrad) {
      float g[8], h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] = v[e] * p.o.alpha0;
        h[e] = u[e] * p.o.alpha1;
      }
      grad8(p.o, p.grad, row, nt * 128 + c, g, h, grad_load(p.o, p.grad, row, nt * 128 + c));
    } else {
      finish<kGated, 8>(p.o, row, nt, c, v, u);
    }
  });
}

// A thread takes eight columns, a warp 256 of a row: its loads of two bytes share their sectors by way of L1. The
// gradient of 512 rows takes 37.1 us with it and 31.7 without at 4097 -> 7680, 76.8 and 65.8 at 18431 -> 4096.
constexpr int kPadRows = 8;  // rows of a block
__global__ void __launch_bounds__(32 * kPadRows)
    pad_rows_kernel(const uint16_t* __restrict__ src, int64_t ld, int rows, int cols, uint16_t* __restrict__ dst,
                    int64_t ldd) {
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x) * 8;
  if (col >= ldd) return;
  const int have = static_cast<int>(min(static_cast<int64_t>(8), cols - col));
  for (int64_t row = static_cast<int64_t>(blockIdx.y) * kPadRows + threadIdx.y; row < rows;
       row += static_cast<int64_t>(gridDim.y) * kPadRows) {
    const uint16_t* s = src + row * ld + col;
    uint32_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < have ? s[e] : 0u;
    *reinterpret_cast<uint4*>(dst + row * ldd + col) =
        make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
}

namespace {

int x_map(aex_ctx* ctx, CUtensorMap* tm, const void* x, int64_t ldx, int rows, int cols) {
  uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  uint64_t strides[1] = {static_cast<uint64_t>(ldx) * 2};
  uint32_t box[2] = {64, 128};
  return make_tmap(ctx, tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int kFormat, int kMode>
int launch_gemm(aex_ctx* ctx, const CUtensorMap& tm0, const CUtensorMap& tm1, GemmParams p, const TilePlan& plan,
                void* pieces, cudaStream_t s) {
  p.work = tile_work(plan, pieces);
  p.status = ctx->d_status;
  auto kern = gemm_kernel<kFormat, kMode>;
  static SmemOptIn opt_in;
  if (int r = opt_in(ctx, reinterpret_cast<const void*>(kern), kGSmem)) return r;
  if (int r = launch_pairs(ctx, reinterpret_cast<const void*>(kern), plan.clusters, kGThreads, kGSmem, true, s,
                           const_cast<CUtensorMap*>(&tm0), const_cast<CUtensorMap*>(&tm1), &p))
    return r;
  if (plan.split)
    return launch_after(ctx, reinterpret_cast<const void*>(join_kernel<kMode>),
                        join_blocks(p.work, kMode == kGatedFwd || kMode == kGatedGrad), kJoinThreads, s, &p);
  return AEX_OK;
}

template <int kMode>
int by_format(aex_ctx* ctx, int format, const CUtensorMap& tm0, const CUtensorMap& tm1, const GemmParams& p,
              const TilePlan& plan, void* pieces, cudaStream_t s) {
  return format == AEX_FP4_MX ? launch_gemm<AEX_FP4_MX, kMode>(ctx, tm0, tm1, p, plan, pieces, s)
                              : launch_gemm<AEX_FP4_NV, kMode>(ctx, tm0, tm1, p, plan, pieces, s);
}

GemmParams weight_params(const aex_fp4weight* w0, const aex_fp4weight* w1) {
  GemmParams p{};
  p.w0 = w0->records;
  p.w1 = w1 ? w1->records : nullptr;
  p.k_blocks = w0->k_blocks;
  p.n_tiles = w0->n_tiles;
  return p;
}

float unit_of(int format) {
  return format == AEX_FP4_MX ? decode_unit<AEX_FP4_MX>() : decode_unit<AEX_FP4_NV>();
}

// Microseconds of the main loop per record: four K steps forward, two backward (B200).
constexpr double kForwardUs = 1.5, kBackwardUs = 0.75;

}  // namespace

TilePlan plan_gemm(const aex_fp4weight* w, bool gated, int m) {
  return plan_tiles(w->clusters, m, gated ? w->n_tiles : (w->n_tiles + 1) / 2, w->k_blocks, kForwardUs);
}
TilePlan plan_dgrad(const aex_fp4weight* w, bool two, int m) {
  return plan_tiles(w->clusters, m, w->k_blocks, w->n_tiles * (two ? 2 : 1), kBackwardUs);
}

int gemm_clusters(aex_ctx* ctx, int* out) {
  auto kern = gemm_kernel<AEX_FP4_NV, kPlain>;
  AEX_CUDA_TRY(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGSmem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * (ctx->sm_count / 2), 1, 1);
  cfg.blockDim = dim3(kGThreads, 1, 1);
  cfg.dynamicSmemBytes = kGSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  AEX_CUDA_TRY(ctx, cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
  if (n <= 0) return set_error(ctx, AEX_ERR_UNSUPPORTED, "the fp4 CTA-pair GEMM cannot be resident on this device");
  *out = n;
  return AEX_OK;
}

int run_gemm(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  const aex_fp4weight* w = j.w0;
  CUtensorMap tm;
  if (int r = x_map(ctx, &tm, j.x, j.ldx, j.m, w->k)) return r;
  GemmParams p = weight_params(w, j.w1);
  p.o.m = j.m;
  p.o.cols = w->n;
  p.o.alpha0 = unit_of(w->format) * w->tensor_scale;
  p.o.alpha1 = j.w1 ? unit_of(w->format) * j.w1->tensor_scale : 0.f;
  p.o.activation = j.activation;
  p.o.y = j.y;
  p.o.ldy = j.ldy;
  p.o.y_f32 = j.y_f32;
  p.o.vec = vec_ok(j.y, j.ldy, j.y_f32);
  const TilePlan plan = plan_gemm(w, j.w1 != nullptr, j.m);
  return j.w1 ? by_format<kGatedFwd>(ctx, w->format, tm, tm, p, plan, j.pieces, s)
              : by_format<kPlain>(ctx, w->format, tm, tm, p, plan, j.pieces, s);
}

int pad_rows(aex_ctx* ctx, const void* src, int64_t ld, int rows, int cols, void* dst, int64_t ldd, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((ldd / 8 + 31) / 32),
                  static_cast<unsigned>(std::min((rows - 1) / kPadRows + 1, 65535)));
  pad_rows_kernel<<<grid, dim3(32, kPadRows), 0, s>>>(static_cast<const uint16_t*>(src), ld, rows, cols,
                                                      static_cast<uint16_t*>(dst), ldd);
  return check_launch(ctx, "fp4 pad_rows_kernel");
}

int run_gated_grad(aex_ctx* ctx, const aex_fp4weight* wg, const aex_fp4weight* wu, int activation, const void* x,
                   int64_t ldx, int m, const void* dh, int64_t lddh, uint16_t* dg, uint16_t* du, int64_t ld,
                   void* pieces, cudaStream_t s) {
  CUtensorMap tm;
  if (int r = x_map(ctx, &tm, x, ldx, m, wg->k)) return r;
  GemmParams p = weight_params(wg, wu);
  p.o.m = m;
  p.o.cols = wg->n;
  p.o.alpha0 = unit_of(wg->format) * wg->tensor_scale;
  p.o.alpha1 = unit_of(wg->format) * wu->tensor_scale;
  p.o.activation = activation;
  p.grad.fold0 = wg->tensor_scale;
  p.grad.fold1 = wu->tensor_scale;
  p.grad.dh = static_cast<const uint16_t*>(dh);
  p.grad.lddh = lddh;
  p.grad.dg = dg;
  p.grad.du = du;
  p.grad.ldg = ld;
  return by_format<kGatedGrad>(ctx, wg->format, tm, tm, p, plan_gemm(wg, true, m), pieces, s);
}

int run_dgrad(aex_ctx* ctx, const aex_fp4weight* w0, const aex_fp4weight* w1, const void* d0, int64_t ld0,
              const void* d1, int64_t ld1, int m, float alpha, void* dx, bool dx_f32, int64_t lddx, void* pieces,
              cudaStream_t s) {
  CUtensorMap tm0, tm1;
  if (int r = x_map(ctx, &tm0, d0, ld0, m, w0->n)) return r;
  tm1 = tm0;
  if (w1)
    if (int r = x_map(ctx, &tm1, d1, ld1, m, w1->n)) return r;
  GemmParams p = weight_params(w0, w1);
  p.o.m = m;
  p.o.cols = w0->k;
  p.o.alpha0 = unit_of(w0->format) * alpha;
  p.o.y = dx;
  p.o.ldy = lddx;
  p.o.y_f32 = dx_f32;
  p.o.vec = vec_ok(dx, lddx, dx_f32);
  return by_format<kDgrad>(ctx, w0->format, tm0, tm1, p, plan_dgrad(w0, w1 != nullptr, m), pieces, s);
}

}  // namespace fp4
}  // namespace aex
