// fp4_block.cu — many rows, both operands in microscaled 4 bits: y = x W^T and
// act(x Wg^T) * (x Wu^T) by block-scaled tensor-core products.
//
// Tensor-bound (tcgen05.mma.cta_group::2 kind::mxf4nvf4 / mxf4, K = 64 per
// instruction, 256 x 256 output tiles, persistent). The tensor core takes codes
// and scales as they are: CTA r of a pair holds the record of x rows
// [128 r, 128 r + 128) of the tile (A) and of its 128 of the tile's 256 weight
// rows (B; gated: rank 0 the gate's, rank 1 the up projection's), by plain bulk
// copies, since a record is already the swizzled operand image. The scales go
// from shared to tensor memory (tcgen05.cp, 512 bytes for 128 rows x 4 scales),
// issued by the thread that issues the products, whose order with them the
// hardware keeps; each CTA holds the scales of its A rows and of all 256 B rows.
//   warp 0   producer (both CTAs)
//   warp 1   even CTA: MMA issuer; odd CTA: forwards "landed" to the even CTA
//   warp 2   tensor-memory allocation
//   warps 4-11 epilogue (tensor-memory lane quadrant = warp % 4; half of the
//            columns each)
// Tensor memory holds 512 columns, two accumulators of 256 and the scales of a
// step (48) do not fit: the accumulators overlap by 48 columns, [0, 256) and
// [208, 464). The epilogue reads those first and hands them back (`ovl`), so
// that the next tile's products wait for a fifth of the epilogue only (with one
// accumulator they waited for all of it: 157 us for 4608 rows gated, 129 now).
// Barriers per 256-column step (stage s): the copies land on each CTA's full[s];
// the odd CTA's forwarder arrives on the even CTA's peer[s]; the MMA thread
// waits for both, issues the copies of scales and four products, and commits to
// both CTAs' empty[s]. Tiles are dealt out as in the dequantizing GEMM.
// Measured, the rows' quantisation included (17 and 12 us of it): 4608 rows 4096
// -> 12288 nvfp4 99 us (4.7 PFLOP/s) in the 2 ms after a pause, 117 us (4.0) in a
// loop, where the power cap leaves 1.43 GHz; gated 4096 -> 9216 mxfp4 132 us (5.3)
// and 152 (4.6). The tensor pipe is busy 70 and 74 % of the kernel.
#include <algorithm>

#include "fp4_internal.h"
#include "fp4_tile.cuh"

namespace aex {
namespace fp4 {

constexpr int kBThreads = 384;
constexpr int kBStages = 5;
constexpr int kBOffB = kRecCodes;
constexpr int kBOffSfa = 2 * kRecCodes;
constexpr int kBOffSfb = kBOffSfa + 2048;
constexpr int kBStage = kBOffSfb + 2 * 2048;  // 38 KB
static_assert(kBStage % 1024 == 0, "operand tiles start on 1024-byte boundaries");
constexpr int kBOffBar = kBStages * kBStage;
// full[S], peer[S], empty[S], accf[2], acce[2], ovl, drain
constexpr int kBNumBars = 3 * kBStages + 6;
constexpr int kBSmem = kBOffBar + kBNumBars * 8 + 16 + 1024;
static_assert(kBSmem <= 232448, "fp4 block GEMM exceeds the shared-memory limit");
// tensor memory: the accumulators, then the scales of a step
constexpr uint32_t kBAcc1 = 208;
constexpr int kBOvl = 256 - kBAcc1;      // columns that both accumulators use
constexpr uint32_t kBSfa = kBAcc1 + 256;  // 4 columns per group of 128 rows x 4 scales
constexpr uint32_t kBSfb = kBSfa + 16;    // 8 columns per group of 256 rows x 4 scales
static_assert(kBSfb + 32 == 512, "tensor memory");

struct BlockParams {
  const uint8_t* x;
  const uint8_t* w0;
  const uint8_t* w1;
  int k_blocks;
  int x_tiles;  // records along the rows of x
  int n_tiles;  // records along the rows of a weight
  TileWork work;
  TileOut o;
  int* status;
};

// Instruction descriptor of the 4-bit block-scaled kinds: scale id of B [4,6),
// A and B type e2m1 = 1 at [7,10) and [10,12), N >> 3 [17,23), scale type bit
// 23 (1: E8M0), M >> 7 [27,29), scale id of A [29,31).
__host__ __device__ constexpr uint32_t idesc_fp4(int M, int N, bool e8m0, uint32_t scale_id) {
  return (scale_id << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         ((e8m0 ? 1u : 0u) << 23) | (static_cast<uint32_t>(M >> 7) << 27) | (scale_id << 29);
}

// Shared-memory descriptor of 512 contiguous bytes as 32 rows of 16 (no
// swizzle: 8-row core matrices of 128 bytes, 128 bytes apart).
__device__ __forceinline__ uint64_t sdesc_scales(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(8) << 16) |
         (static_cast<uint64_t>(8) << 32) | (static_cast<uint64_t>(1) << 46);
}

// In both CTAs of the pair: 32 rows x 16 bytes -> 4 columns, in all four lane
// quadrants.
__device__ __forceinline__ void tmem_cp_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

template <int kFormat>
__device__ __forceinline__ void umma_fp4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                              uint32_t sfb, uint32_t accumulate) {
  if (kFormat == AEX_FP4_MX)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

template <int kFormat, bool kGated>
__global__ void __launch_bounds__(kBThreads, 1) block_kernel(const __grid_constant__ BlockParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kBOffBar);
  uint64_t* peer = full + kBStages;
  uint64_t* empty = peer + kBStages;
  uint64_t* accf = empty + kBStages;
  uint64_t* acce = accf + 2;
  uint64_t* ovl = acce + 2;
  uint64_t* drain = ovl + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + kBNumBars);
  __shared__ int abort_flag;
  constexpr int kRec = rec_bytes(kFormat);
  constexpr int kScales = rec_scales(kFormat);
  constexpr int kGroups = kScales / 512;  // scale groups of a record: 4 (nvfp4) or 2 (mxfp4)

  const int warp = static_cast<int>(warp_id_uniform());
  const int lane = static_cast<int>(lane_id());
  const uint32_t rank = cluster_ctarank();
  const int cluster = static_cast<int>(blockIdx.x >> 1);
  const int clusters = static_cast<int>(gridDim.x >> 1);

  launch_dependents();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kBStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&peer[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf[b], 1);
      mbar_init(&acce[b], 2 * 8);
    }
    mbar_init(ovl, 2 * 4);
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  // Before the wait, as the GEMM must not: the kernel before this one is always quantize_kernel, launched without
  // setting up early and without tensor memory, so whatever held some on this stream has ended.
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_dependency();  // x's records are written

  if (warp == 0) {
    if (lane == 0) {
      // -------------------------------------------------------- producer
      const uint32_t empty0 = smem_u32(&empty[0]);
      uint32_t s = 0, ph = 0;
      int g = 0;
      bool ok = true;
      TilePiece t;
      for (int i = 0; ok && p.work.piece(cluster, clusters, i, &t); ++i) {
        const int mt = t.mt, nt = t.nt;
        const size_t step = static_cast<size_t>(kRec);
        // past the last tile of rows or outputs: any record, its results are not stored
        const uint8_t* xa = p.x + static_cast<size_t>(min(2 * mt + static_cast<int>(rank), p.x_tiles - 1)) * p.k_blocks * step;
        const uint8_t *b0, *b1;
        if (kGated) {
          b0 = p.w0 + static_cast<size_t>(nt) * p.k_blocks * step;
          b1 = p.w1 + static_cast<size_t>(nt) * p.k_blocks * step;
        } else {
          b0 = p.w0 + static_cast<size_t>(2 * nt) * p.k_blocks * step;
          b1 = p.w0 + static_cast<size_t>(min(2 * nt + 1, p.n_tiles - 1)) * p.k_blocks * step;
        }
        for (int k = t.r0; k < t.r1; ++k, ++g) {
          if (g >= kBStages && !mbar_wait_cl(empty0 + 8 * s, ph ^ 1, &abort_flag, p.status, kDevTimeoutTma)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * kBStage;
          const size_t at = static_cast<size_t>(k) * step;
          mbar_arrive_expect_tx(&full[s], 2 * kRecCodes + 3 * kScales);
          bulk_load(st, xa + at, kRecCodes, &full[s]);
          bulk_load(st + kBOffB, (rank ? b1 : b0) + at, kRecCodes, &full[s]);
          bulk_load(st + kBOffSfa, xa + at + kRecCodes, kScales, &full[s]);
          bulk_load(st + kBOffSfb, b0 + at + kRecCodes, kScales, &full[s]);
          bulk_load(st + kBOffSfb + 2048, b1 + at + kRecCodes, kScales, &full[s]);
          if (++s == kBStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) {
        for (int j = (g > kBStages ? g - kBStages : 0); j < g; ++j) {
          const uint32_t a = smem_u32(&full[j % kBStages]);
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(a, (j / kBStages) & 1) && globaltimer_ns() - t0 < kWaitTimeoutNs) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 1) {
      // ------------------------------------------------- forwarder (odd CTA)
      const uint32_t lead = mapa_shared(smem_u32(&peer[0]), 0);
      uint32_t s = 0, ph = 0;
      bool ok = true;
      TilePiece t;
      for (int i = 0; ok && p.work.piece(cluster, clusters, i, &t); ++i)
        for (int k = t.r0; k < t.r1; ++k) {
          if (!mbar_wait_cl(smem_u32(&full[s]), ph, &abort_flag, p.status, kDevTimeoutTma)) {
            ok = false;
            break;
          }
          mbar_arrive_cluster(lead + 8 * s);
          if (++s == kBStages) {
            s = 0;
            ph ^= 1;
          }
        }
    } else if (lane == 0) {
      // ----------------------------------------------------- MMA (even CTA)
      const uint32_t s0 = smem_u32(smem);
      const uint64_t da0 = sdesc_sw128(s0, 16, 1024);
      const uint64_t db0 = sdesc_sw128(s0 + kBOffB, 16, 1024);
      const uint64_t dsa0 = sdesc_scales(s0 + kBOffSfa);
      const uint64_t dsb0 = sdesc_scales(s0 + kBOffSfb);
      uint32_t s = 0, ph = 0;
      bool ok = true;
      TilePiece t;
      for (int i = 0; ok && p.work.piece(cluster, clusters, i, &t); ++i) {
        // this accumulator's previous tile is read, and of the other's the columns they share
        const int b = i & 1;
        if ((i >= 2 && !mbar_wait_cl(smem_u32(&acce[b]), ((i >> 1) + 1) & 1, &abort_flag, p.status, kDevTimeoutMma)) ||
            (i >= 1 && !mbar_wait_cl(smem_u32(ovl), (i + 1) & 1, &abort_flag, p.status, kDevTimeoutMma))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + b * kBAcc1;
        for (int k = t.r0; k < t.r1; ++k) {
          if (!mbar_wait_cl(smem_u32(&full[s]), ph, &abort_flag, p.status, kDevTimeoutMma) ||
              !mbar_wait_cl(smem_u32(&peer[s]), ph, &abort_flag, p.status, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t off = (s * kBStage) >> 4;
#pragma unroll
          for (int gq = 0; gq < kGroups; ++gq) {
            tmem_cp_scales_pair(tmem + kBSfa + 4 * gq, dsa0 + off + gq * 32);
            tmem_cp_scales_pair(tmem + kBSfb + 8 * gq, dsb0 + off + gq * 32);
            tmem_cp_scales_pair(tmem + kBSfb + 8 * gq + 4, dsb0 + off + 128 + gq * 32);
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            // mxfp4: a group's four scales serve two products, the second takes bytes 2 and 3
            const int gq = kFormat == AEX_FP4_MX ? kk >> 1 : kk;
            const uint32_t idesc = idesc_fp4(256, 256, kFormat == AEX_FP4_MX, kFormat == AEX_FP4_MX ? (kk & 1) * 2 : 0);
            umma_fp4_pair<kFormat>(d, da0 + off + kk * 2, db0 + off + kk * 2, idesc, tmem + kBSfa + 4 * gq,
                                   tmem + kBSfb + 8 * gq, (k > t.r0 || kk > 0) ? 1u : 0u);
          }
          umma_commit_both(smem_u32(&empty[s]));
          if (++s == kBStages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        umma_commit_both(smem_u32(&accf[b]));
      }
      umma_commit_pair(smem_u32(drain));
      int no_abort = 0;
      mbar_wait_cl(smem_u32(drain), 0, &no_abort, p.status, kDevTimeoutMma);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t ovl_lead = mapa_shared(smem_u32(ovl), 0);
    TilePiece t;
    for (int i = 0; p.work.piece(cluster, clusters, i, &t); ++i) {
      const int b = i & 1;
      if (!mbar_wait_warp_cl(smem_u32(&accf[b]), (i >> 1) & 1, &abort_flag, p.status, kDevTimeoutEpilogue)) break;
      tc_fence_after();
      const int in_tile = static_cast<int>(rank) * 128 + quad * 32 + lane;
      const int64_t row = static_cast<int64_t>(t.mt) * 256 + in_tile;
      const bool live = row < p.o.m;
      const uint32_t tbase = tmem + (static_cast<uint32_t>(quad * 32) << 16) + b * kBAcc1;
      // The shared columns are the last of accumulator 0, in half 1, and the first of accumulator 1, in half 0.
      const bool mine = half != b;
      const int o0 = b ? 0 : static_cast<int>(kBAcc1);  // first shared column of this accumulator
      float sh[kBOvl];
      if (mine) {
        tmem_read<kBOvl>(tbase + o0, sh);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(ovl_lead);
      }
      if (kGated && t.slot < 0) {
        // outputs [64 half, ..): the shared columns are up columns 80..127 (accumulator 0) or gate columns 0..47
        if (mine) {
#pragma unroll
          for (int e = 0; e < kBOvl; e += 16) {
            const int c = (b ? 0 : static_cast<int>(kBAcc1) - 128) + e;
            float v[16];
            tmem_read<16>(tbase + (b ? 128 : 0) + c, v);
            if (live) finish<true, 16>(p.o, row, t.nt, c, b ? sh + e : v, b ? v : sh + e);
          }
        }
        const int c0 = mine && half == 0 ? kBOvl : 64 * half;
        const int c1 = mine && half == 1 ? static_cast<int>(kBAcc1) - 128 : 64 * half + 64;
#pragma unroll 1
        for (int c = c0; c < c1; c += 16) {
          uint32_t g[16], u[16];
          tmem_ld16(tbase + c, g);
          tmem_ld16(tbase + 128 + c, u);
          tmem_wait_ld();
          if (live) finish<true, 16>(p.o, row, t.nt, c, reinterpret_cast<float*>(g), reinterpret_cast<float*>(u));
        }
      } else {
        auto emit = [&](int c, const float* v) {
          if (!live) return;
          if (t.slot < 0)
            finish<false, 16>(p.o, row, t.nt, c, v, nullptr);
          else
            store_piece16(p.work, t.slot, in_tile, c, v);
        };
        if (mine) {
#pragma unroll
          for (int e = 0; e < kBOvl; e += 16) emit(o0 + e, sh + e);
        }
        const int c0 = mine && half == 0 ? kBOvl : 128 * half;
        const int c1 = mine && half == 1 ? static_cast<int>(kBAcc1) : 128 * half + 128;
#pragma unroll 1
        for (int c = c0; c < c1; c += 16) {
          float v[16];
          tmem_read<16>(tbase + c, v);
          emit(c, v);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acce[b]), 0));
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

template <bool kGated>
__global__ void __launch_bounds__(kJoinThreads) block_join_kernel(const __grid_constant__ BlockParams p) {
  join_tile<kGated>(p.work, p.o.m, [&](int64_t row, int nt, int c, const float* v, const float* u) {
    finish<kGated, 8>(p.o, row, nt, c, v, u);
  });
}

namespace {

template <int kFormat, bool kGated>
int launch_block(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  const aex_fp4weight* w = j.w0;
  const TilePlan plan = plan_block(w, kGated, j.m);
  BlockParams p{};
  p.x = j.x_records;
  p.w0 = w->records;
  p.w1 = kGated ? j.w1->records : nullptr;
  p.k_blocks = w->k_blocks;
  p.x_tiles = (j.m - 1) / kRecRows + 1;
  p.n_tiles = w->n_tiles;
  p.work = tile_work(plan, j.pieces);
  p.o.m = j.m;
  p.o.cols = w->n;
  p.o.alpha0 = static_cast<float>(static_cast<double>(j.x_scale) * w->tensor_scale);
  p.o.alpha1 = kGated ? static_cast<float>(static_cast<double>(j.x_scale) * j.w1->tensor_scale) : 0.f;
  p.o.activation = j.activation;
  p.o.y = j.y;
  p.o.ldy = j.ldy;
  p.o.y_f32 = j.y_f32;
  p.o.vec = vec_ok(j.y, j.ldy, j.y_f32);
  p.status = ctx->d_status;
  auto kern = block_kernel<kFormat, kGated>;
  static SmemOptIn opt_in;
  if (int r = opt_in(ctx, reinterpret_cast<const void*>(kern), kBSmem)) return r;
  if (int r = launch_pairs(ctx, reinterpret_cast<const void*>(kern), plan.clusters, kBThreads, kBSmem, true, s, &p))
    return r;
  if (plan.split)
    return launch_after(ctx, reinterpret_cast<const void*>(block_join_kernel<kGated>), join_blocks(p.work, kGated),
                        kJoinThreads, s, &p);
  return AEX_OK;
}

// Microseconds of the main loop per record (B200).
constexpr double kBlockUs = 0.37;

}  // namespace

TilePlan plan_block(const aex_fp4weight* w, bool gated, int m) {
  return plan_tiles(w->clusters, m, gated ? w->n_tiles : (w->n_tiles + 1) / 2, w->k_blocks, kBlockUs);
}

int run_block(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  if (j.w0->format == AEX_FP4_MX)
    return j.w1 ? launch_block<AEX_FP4_MX, true>(ctx, j, s) : launch_block<AEX_FP4_MX, false>(ctx, j, s);
  return j.w1 ? launch_block<AEX_FP4_NV, true>(ctx, j, s) : launch_block<AEX_FP4_NV, false>(ctx, j, s);
}

}  // namespace fp4
}  // namespace aex
