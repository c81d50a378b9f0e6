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
//   warps 4-7 epilogue (tensor-memory lane quadrant = warp % 4)
// Barriers per 256-column step (stage s): the copies land on each CTA's full[s];
// the odd CTA's forwarder arrives on the even CTA's peer[s]; the MMA thread
// waits for both, issues the copies of scales and four products, and commits to
// the even CTA's empty[s], whose producer forwards it to the odd CTA's.
#include <algorithm>

#include "fp4_internal.h"
#include "fp4_tile.cuh"

namespace aex {
namespace fp4 {

constexpr int kBThreads = 256;
constexpr int kBStages = 5;
constexpr int kBOffB = kRecCodes;
constexpr int kBOffSfa = 2 * kRecCodes;
constexpr int kBOffSfb = kBOffSfa + 2048;
constexpr int kBStage = kBOffSfb + 2 * 2048;  // 38 KB
static_assert(kBStage % 1024 == 0, "operand tiles start on 1024-byte boundaries");
constexpr int kBOffBar = kBStages * kBStage;
// full[S], peer[S], empty[S], accf, acce, drain
constexpr int kBNumBars = 3 * kBStages + 3;
constexpr int kBSmem = kBOffBar + kBNumBars * 8 + 16 + 1024;
static_assert(kBSmem <= 232448, "fp4 block GEMM exceeds the shared-memory limit");
// tensor memory: the accumulator, then the scales of a stage
constexpr uint32_t kBSfa = 256;       // 4 columns per group of 128 rows x 4 scales
constexpr uint32_t kBSfb = kBSfa + 16;  // 8 columns per group of 256 rows x 4 scales

struct BlockParams {
  const uint8_t* x;
  const uint8_t* w0;
  const uint8_t* w1;
  int k_blocks;
  int x_tiles;  // records along the rows of x
  int n_tiles;  // records along the rows of a weight
  int m_tiles, tiles;
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
  uint64_t* acce = accf + 1;
  uint64_t* drain = acce + 1;
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

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kBStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&peer[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(accf, 1);
    mbar_init(acce, 2 * 4);
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // -------------------------------------------------------- producer
      const uint32_t empty0 = smem_u32(&empty[0]);
      const uint32_t peer_empty0 = mapa_shared(empty0, 1);
      uint32_t s = 0, ph = 0;
      int g = 0;
      bool ok = true;
      for (int t = cluster; t < p.tiles && ok; t += clusters) {
        const int mt = t % p.m_tiles, nt = t / p.m_tiles;
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
        for (int k = 0; k < p.k_blocks; ++k, ++g) {
          if (g >= kBStages) {
            if (!mbar_wait_cl(empty0 + 8 * s, ph ^ 1, &abort_flag, p.status, kDevTimeoutTma)) {
              ok = false;
              break;
            }
            if (rank == 0) mbar_arrive_cluster(peer_empty0 + 8 * s);
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
      for (int t = cluster; t < p.tiles && ok; t += clusters)
        for (int k = 0; k < p.k_blocks; ++k) {
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
      int i = 0;
      bool ok = true;
      for (int t = cluster; t < p.tiles && ok; t += clusters, ++i) {
        if (i >= 1 && !mbar_wait_cl(smem_u32(acce), (i + 1) & 1, &abort_flag, p.status, kDevTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int k = 0; k < p.k_blocks; ++k) {
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
            umma_fp4_pair<kFormat>(tmem, da0 + off + kk * 2, db0 + off + kk * 2, idesc, tmem + kBSfa + 4 * gq,
                                   tmem + kBSfb + 8 * gq, (k > 0 || kk > 0) ? 1u : 0u);
          }
          umma_commit_pair(smem_u32(&empty[s]));
          if (++s == kBStages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        umma_commit_pair(smem_u32(accf));
        umma_commit_pair(mapa_shared(smem_u32(accf), 1));
      }
      umma_commit_pair(smem_u32(drain));
      int no_abort = 0;
      mbar_wait_cl(smem_u32(drain), 0, &no_abort, p.status, kDevTimeoutMma);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3;
    int i = 0;
    for (int t = cluster; t < p.tiles; t += clusters, ++i) {
      if (!mbar_wait_warp_cl(smem_u32(accf), i & 1, &abort_flag, p.status, kDevTimeoutEpilogue)) break;
      tc_fence_after();
      const int64_t row = static_cast<int64_t>(t % p.m_tiles) * 256 + rank * 128 + quad * 32 + lane;
      tile_rows<kGated>(p.o, row, t / p.m_tiles, tmem + (static_cast<uint32_t>(quad * 32) << 16));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(acce), 0));
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

namespace {

template <int kFormat, bool kGated>
int launch_block(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  const aex_fp4weight* w = j.w0;
  BlockParams p{};
  p.x = j.workspace;
  p.w0 = w->records;
  p.w1 = kGated ? j.w1->records : nullptr;
  p.k_blocks = w->k_blocks;
  p.x_tiles = (j.m - 1) / kRecRows + 1;
  p.n_tiles = w->n_tiles;
  p.m_tiles = (j.m - 1) / 256 + 1;
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * (kGated ? w->n_tiles : (w->n_tiles + 1) / 2);
  if (tiles > 0x3FFFFFFF) return set_error(ctx, AEX_ERR_UNSUPPORTED, "fp4 GEMM: %lld output tiles", (long long)tiles);
  p.tiles = static_cast<int>(tiles);
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
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kBThreads, 1, 1);
  cfg.dynamicSmemBytes = kBSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (ctx->fp4_clusters <= 0) {
    cfg.gridDim = dim3(2 * (ctx->sm_count / 2), 1, 1);
    int n = 0;
    AEX_CUDA_TRY(ctx, cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    if (n <= 0) return set_error(ctx, AEX_ERR_UNSUPPORTED, "the fp4 CTA-pair GEMM cannot be resident on this device");
    ctx->fp4_clusters = n;
  }
  cfg.gridDim = dim3(2 * std::min(p.tiles, ctx->fp4_clusters), 1, 1);
  AEX_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kern, p));
  return check_launch(ctx, "fp4 block_kernel");
}

}  // namespace

int run_block(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  if (j.w0->format == AEX_FP4_MX)
    return j.w1 ? launch_block<AEX_FP4_MX, true>(ctx, j, s) : launch_block<AEX_FP4_MX, false>(ctx, j, s);
  return j.w1 ? launch_block<AEX_FP4_NV, true>(ctx, j, s) : launch_block<AEX_FP4_NV, false>(ctx, j, s);
}

}  // namespace fp4
}  // namespace aex
