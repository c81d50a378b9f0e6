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
//   warps 4-7   epilogue (tensor-memory lane quadrant = warp % 4)
//   warps 8-15  decode: two groups of four warps, alternate K steps
// Barriers per step (stage s): the A box lands on afull[s]; a decode warp waits
// for it and for its record, writes its part of B and arrives on the even
// CTA's bready[s] (both CTAs' four warps of a group); the MMA thread waits for
// that, issues four MMAs and commits to the even CTA's empty[s], whose A
// producer forwards it to the odd CTA. A record is released (rempty) by all
// eight decode warps.
#include <algorithm>

#include "fp4_internal.h"
#include "fp4_tile.cuh"

namespace aex {
namespace fp4 {

constexpr int kGThreads = 512;
constexpr int kGStages = 5;
constexpr int kGRecs = 3;
constexpr int kGTile = 128 * 64 * 2;  // one operand of one CTA and step
constexpr int kGStage = 2 * kGTile;
constexpr int kGRecSlot = rec_bytes(AEX_FP4_NV);
constexpr int kGOffRec = kGStages * kGStage;
constexpr int kGOffBar = kGOffRec + kGRecs * kGRecSlot;
// afull[S], bready[S], empty[S], rfull[R], rempty[R], accf[2], acce[2], drain
constexpr int kGNumBars = 3 * kGStages + 2 * kGRecs + 5;
constexpr int kGSmem = kGOffBar + kGNumBars * 8 + 16 + 1024;
static_assert(kGSmem <= 232448, "fp4 GEMM exceeds the shared-memory limit");

enum GemmMode : int { kPlain = 0, kGatedFwd = 1, kGatedGrad = 2, kDgrad = 3 };

struct GemmParams {
  const uint8_t* w0;
  const uint8_t* w1;
  int k_blocks;  // records along the columns of a weight
  int n_tiles;   // records along its rows
  int m_tiles, tiles;
  int recs;      // records per tile and CTA (dgrad: of both weights)
  TileOut o;
  // gated gradient
  float fold0, fold1;  // the tensor scales that dg and du take on
  const uint16_t* dh;
  int64_t lddh;
  uint16_t* dg;
  uint16_t* du;
  int64_t ldg;
  int* status;
};

// dg, du of 8 columns (col a multiple of 8) from g, u (already scaled).
__device__ __forceinline__ void grad8(const GemmParams& p, int64_t row, int col, const float* g, const float* u) {
  const int left = p.o.cols - col;
  if (left <= 0) return;
  const uint16_t* src = p.dh + row * p.lddh + col;
  uint32_t d[4];
  if (left >= 8) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(src));
    d[0] = q.x, d[1] = q.y, d[2] = q.z, d[3] = q.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      d[i] = (2 * i < left ? src[2 * i] : 0u) | ((2 * i + 1 < left ? static_cast<uint32_t>(src[2 * i + 1]) : 0u) << 16);
  }
  uint32_t og[4], ou[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a[2], b[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float gi = g[2 * i + e], ui = u[2 * i + e];
      const float dv = e ? bf16hi_to_f32(d[i]) : bf16lo_to_f32(d[i]);
      const float sg = sigmoid<true>(sigmoid_arg(gi, p.o.activation));
      const float act = gi * sg;
      a[e] = dv * ui * fmaf(act * (1.f - sg), sigmoid_arg_slope(gi, p.o.activation), sg) * p.fold0;
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
  uint64_t* bready = afull + kGStages;
  uint64_t* empty = bready + kGStages;
  uint64_t* rfull = empty + kGStages;
  uint64_t* rempty = rfull + kGRecs;
  uint64_t* accf = rempty + kGRecs;
  uint64_t* acce = accf + 2;
  uint64_t* drain = acce + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kGNumBars);
  __shared__ int abort_flag;
  constexpr bool kBack = kMode == kDgrad;
  constexpr int kRec = rec_bytes(kFormat);
  constexpr int kSteps = kBack ? 2 : 4;  // K steps per record

  const int warp = static_cast<int>(warp_id_uniform());
  const int lane = static_cast<int>(lane_id());
  const uint32_t rank = cluster_ctarank();
  const int cluster = static_cast<int>(blockIdx.x >> 1);
  const int clusters = static_cast<int>(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kGStages; ++s) {
      mbar_init(&afull[s], 1);
      mbar_init(&bready[s], 2 * 4);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kGRecs; ++s) {
      mbar_init(&rfull[s], 1);
      mbar_init(&rempty[s], 8);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf[b], 1);
      mbar_init(&acce[b], 2 * 4);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm0);
    if (kBack) prefetch_tmap(&tm1);
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int steps = p.recs * kSteps;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------ A producer
      const uint32_t empty0 = smem_u32(&empty[0]);
      const uint32_t peer_empty0 = mapa_shared(empty0, 1);
      uint32_t s = 0, ph = 0;
      int g = 0;
      bool ok = true;
      for (int t = cluster; t < p.tiles && ok; t += clusters) {
        const int row0 = (t % p.m_tiles) * 256 + static_cast<int>(rank) * 128;
        for (int k = 0; k < steps; ++k, ++g) {
          if (g >= kGStages) {
            if (!mbar_wait_cl(empty0 + 8 * s, ph ^ 1, &abort_flag, p.status, kDevTimeoutTma)) {
              ok = false;
              break;
            }
            if (rank == 0) mbar_arrive_cluster(peer_empty0 + 8 * s);
          }
          mbar_arrive_expect_tx(&afull[s], kGTile);
          // dgrad: the second weight's rows follow the first's (p.n_tiles records of two steps)
          const bool second = kBack && k >= 2 * p.n_tiles;
          tma_load_2d(smem + s * kGStage, second ? &tm1 : &tm0, &afull[s], (second ? k - 2 * p.n_tiles : k) * 64, row0);
          if (++s == kGStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) {
        for (int j = (g > kGStages ? g - kGStages : 0); j < g; ++j) {
          const uint32_t a = smem_u32(&afull[j % kGStages]);
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(a, (j / kGStages) & 1) && globaltimer_ns() - t0 < kWaitTimeoutNs) {
          }
        }
      }
    }
  } else if (warp == 3) {
    if (lane == 0) {
      // ------------------------------------------------- record producer
      uint32_t s = 0, ph = 0;
      int g = 0;
      bool ok = true;
      for (int t = cluster; t < p.tiles && ok; t += clusters) {
        const int nt = t / p.m_tiles;
        for (int i = 0; i < p.recs; ++i, ++g) {
          if (g >= kGRecs && !mbar_wait(&rempty[s], ph ^ 1, &abort_flag, p.status, kDevTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint8_t* w = p.w0;
          int rt, kb;
          if (kBack) {
            const bool second = i >= p.n_tiles;
            if (second) w = p.w1;
            rt = second ? i - p.n_tiles : i;
            kb = nt;
          } else {
            kb = i;
            if (kMode == kPlain) {
              rt = min(2 * nt + static_cast<int>(rank), p.n_tiles - 1);  // an odd last tile: columns nobody stores
            } else {
              rt = nt;
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
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // ------------------------------------------------------------- MMA
      constexpr uint32_t kIdesc = idesc_bf16_f32(256, 256, false, kBack);
      constexpr uint32_t kBStep = kBack ? 128 : 2;  // 16 K rows of an MN-major tile: 2 KB; of a K-major one: 32 B
      const uint32_t s0 = smem_u32(smem);
      const uint32_t bready0 = smem_u32(&bready[0]);
      const uint32_t empty0 = smem_u32(&empty[0]);
      const uint64_t da0 = sdesc_sw128(s0, 16, 1024);
      const uint64_t db0 = sdesc_sw128(s0 + kGTile, kBack ? 8192 : 16, 1024);
      uint32_t s = 0, ph = 0;
      int i = 0;
      bool ok = true;
      for (int t = cluster; t < p.tiles && ok; t += clusters, ++i) {
        const int b = i & 1;
        if (i >= 2 && !mbar_wait_cl(smem_u32(&acce[b]), ((i >> 1) + 1) & 1, &abort_flag, p.status, kDevTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + b * 256;
        for (int k = 0; k < steps; ++k) {
          if (!mbar_wait_cl(bready0 + 8 * s, ph, &abort_flag, p.status, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t off = (s * kGStage) >> 4;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_ss_pair(d, da0 + off + kk * 2, db0 + off + kk * kBStep, kIdesc, (k > 0 || kk > 0) ? 1u : 0u);
          umma_commit_pair(empty0 + 8 * s);
          if (++s == kGStages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        umma_commit_pair(smem_u32(&accf[b]));
        umma_commit_pair(mapa_shared(smem_u32(&accf[b]), 1));
      }
      // Waited for on abort too: no MMA is in flight at the teardown.
      umma_commit_pair(smem_u32(drain));
      int no_abort = 0;
      mbar_wait_cl(smem_u32(drain), 0, &no_abort, p.status, kDevTimeoutMma);
    }
  } else if (warp >= 4 && warp < 8) {
    // ------------------------------------------------------------ epilogue
    const int quad = warp & 3;
    int i = 0;
    for (int t = cluster; t < p.tiles; t += clusters, ++i) {
      const int nt = t / p.m_tiles;
      const int b = i & 1;
      if (!mbar_wait_warp_cl(smem_u32(&accf[b]), (i >> 1) & 1, &abort_flag, p.status, kDevTimeoutEpilogue)) break;
      tc_fence_after();
      const int64_t row = static_cast<int64_t>(t % p.m_tiles) * 256 + rank * 128 + quad * 32 + lane;
      const uint32_t tbase = tmem + (static_cast<uint32_t>(quad * 32) << 16) + b * 256;
      if (kMode != kGatedGrad) {
        tile_rows<kMode == kGatedFwd>(p.o, row, nt, tbase);
      } else {
#pragma unroll 1
        for (int c0 = 0; c0 < 128; c0 += 32) {
          uint32_t gr[32], ur[32];
          tmem_ld32(tbase + c0, gr);
          tmem_ld32(tbase + 128 + c0, ur);
          tmem_wait_ld();
          if (row < p.o.m) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              float g[8], u[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                g[i] = __uint_as_float(gr[e + i]) * p.o.alpha0;
                u[i] = __uint_as_float(ur[e + i]) * p.o.alpha1;
              }
              grad8(p, row, nt * 128 + c0 + e, g, u);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acce[b]), 0));
    }
  } else if (warp >= 8) {
    // -------------------------------------------------------------- decode
    const int group = (warp - 8) >> 2;
    const int dt = ((warp - 8) & 3) * 32 + lane;
    const uint32_t afull0 = smem_u32(&afull[0]);
    const uint32_t bready_lead0 = mapa_shared(smem_u32(&bready[0]), 0);
    uint32_t s = 0, ph = 0, rs = 0, rph = 0;
    bool ok = true;
    for (int t = cluster; t < p.tiles && ok; t += clusters) {
      for (int k = 0; k < steps; ++k) {
        const uint32_t cs = s, cph = ph, crs = rs, crph = rph;
        if (++s == kGStages) {
          s = 0;
          ph ^= 1;
        }
        const bool last_of_rec = (k & (kSteps - 1)) == kSteps - 1;
        if (last_of_rec && ++rs == kGRecs) {
          rs = 0;
          rph ^= 1;
        }
        if ((k & 1) != group) continue;  // steps per tile are even: the groups keep alternating
        if (!mbar_wait_warp(&rfull[crs], crph, &abort_flag, p.status, kDevTimeoutProducer) ||
            !mbar_wait_warp_cl(afull0 + 8 * cs, cph, &abort_flag, p.status, kDevTimeoutProducer)) {
          ok = false;
          break;
        }
        const uint8_t* rec = smem + kGOffRec + crs * kGRecSlot;
        // r: row of the record; cp: its 64-column part; dst: that row in B
        int r, cp;
        uint8_t* dst = smem + cs * kGStage + kGTile;
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
        // This warp's last read of the record: group 1 takes its last step, group 0 the one before.
        if ((k & (kSteps - 1)) >= kSteps - 2) {
          __syncwarp();
          if (lane == 0) mbar_arrive_addr(smem_u32(&rempty[crs]));
        }
        const uint32_t ws[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // nvfp4: a scale every two words, mxfp4: every four
          const uint32_t s2 = scale_pair<kFormat>((sc >> (kFormat == AEX_FP4_NV ? 8 * (j >> 1) : 8 * (j >> 2))) & 0xFFu);
          *reinterpret_cast<uint4*>(dst + ((j ^ sw) << 4)) =
              make_uint4(decode_pair<kFormat>(ws[j], 0, s2), decode_pair<kFormat>(ws[j], 1, s2),
                         decode_pair<kFormat>(ws[j], 2, s2), decode_pair<kFormat>(ws[j], 3, s2));
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(bready_lead0 + 8 * cs);
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

namespace {

int x_map(aex_ctx* ctx, CUtensorMap* tm, const void* x, int64_t ldx, int rows, int cols) {
  uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  uint64_t strides[1] = {static_cast<uint64_t>(ldx) * 2};
  uint32_t box[2] = {64, 128};
  return make_tmap(ctx, tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int kFormat, int kMode>
int launch_gemm(aex_ctx* ctx, const CUtensorMap& tm0, const CUtensorMap& tm1, GemmParams p, int64_t col_tiles,
                cudaStream_t s) {
  p.m_tiles = (p.o.m - 1) / 256 + 1;
  const int64_t tiles = p.m_tiles * col_tiles;
  if (tiles > 0x3FFFFFFF) return set_error(ctx, AEX_ERR_UNSUPPORTED, "fp4 GEMM: %lld output tiles", (long long)tiles);
  p.tiles = static_cast<int>(tiles);
  p.status = ctx->d_status;
  auto kern = gemm_kernel<kFormat, kMode>;
  static SmemOptIn opt_in;
  if (int r = opt_in(ctx, reinterpret_cast<const void*>(kern), kGSmem)) return r;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kGThreads, 1, 1);
  cfg.dynamicSmemBytes = kGSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // One CTA per SM (shared memory); clusters of two that fit at once.
  if (ctx->fp4_clusters <= 0) {
    cfg.gridDim = dim3(2 * (ctx->sm_count / 2), 1, 1);
    int n = 0;
    AEX_CUDA_TRY(ctx, cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    if (n <= 0) return set_error(ctx, AEX_ERR_UNSUPPORTED, "the fp4 CTA-pair GEMM cannot be resident on this device");
    ctx->fp4_clusters = n;
  }
  cfg.gridDim = dim3(2 * std::min(p.tiles, ctx->fp4_clusters), 1, 1);
  AEX_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kern, tm0, tm1, p));
  return check_launch(ctx, "fp4 gemm_kernel");
}

template <int kMode>
int by_format(aex_ctx* ctx, int format, const CUtensorMap& tm0, const CUtensorMap& tm1, const GemmParams& p,
              int64_t col_tiles, cudaStream_t s) {
  return format == AEX_FP4_MX ? launch_gemm<AEX_FP4_MX, kMode>(ctx, tm0, tm1, p, col_tiles, s)
                              : launch_gemm<AEX_FP4_NV, kMode>(ctx, tm0, tm1, p, col_tiles, s);
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

}  // namespace

int run_gemm(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  const aex_fp4weight* w = j.w0;
  CUtensorMap tm;
  if (int r = x_map(ctx, &tm, j.x, j.ldx, j.m, w->k)) return r;
  GemmParams p = weight_params(w, j.w1);
  p.o.m = j.m;
  p.o.cols = w->n;
  p.recs = w->k_blocks;
  p.o.alpha0 = unit_of(w->format) * w->tensor_scale;
  p.o.alpha1 = j.w1 ? unit_of(w->format) * j.w1->tensor_scale : 0.f;
  p.o.activation = j.activation;
  p.o.y = j.y;
  p.o.ldy = j.ldy;
  p.o.y_f32 = j.y_f32;
  p.o.vec = vec_ok(j.y, j.ldy, j.y_f32);
  return j.w1 ? by_format<kGatedFwd>(ctx, w->format, tm, tm, p, w->n_tiles, s)
              : by_format<kPlain>(ctx, w->format, tm, tm, p, (w->n_tiles + 1) / 2, s);
}

int run_gated_grad(aex_ctx* ctx, const aex_fp4weight* wg, const aex_fp4weight* wu, int activation, const void* x,
                   int64_t ldx, int m, const void* dh, int64_t lddh, uint16_t* dg, uint16_t* du, int64_t ld,
                   cudaStream_t s) {
  CUtensorMap tm;
  if (int r = x_map(ctx, &tm, x, ldx, m, wg->k)) return r;
  GemmParams p = weight_params(wg, wu);
  p.o.m = m;
  p.o.cols = wg->n;
  p.recs = wg->k_blocks;
  p.o.alpha0 = unit_of(wg->format) * wg->tensor_scale;
  p.o.alpha1 = unit_of(wg->format) * wu->tensor_scale;
  p.fold0 = wg->tensor_scale;
  p.fold1 = wu->tensor_scale;
  p.o.activation = activation;
  p.dh = static_cast<const uint16_t*>(dh);
  p.lddh = lddh;
  p.dg = dg;
  p.du = du;
  p.ldg = ld;
  return by_format<kGatedGrad>(ctx, wg->format, tm, tm, p, wg->n_tiles, s);
}

int run_dgrad(aex_ctx* ctx, const aex_fp4weight* w0, const aex_fp4weight* w1, const void* d0, int64_t ld0,
              const void* d1, int64_t ld1, int m, float alpha, void* dx, bool dx_f32, int64_t lddx, cudaStream_t s) {
  CUtensorMap tm0, tm1;
  if (int r = x_map(ctx, &tm0, d0, ld0, m, w0->n)) return r;
  tm1 = tm0;
  if (w1)
    if (int r = x_map(ctx, &tm1, d1, ld1, m, w1->n)) return r;
  GemmParams p = weight_params(w0, w1);
  p.o.m = m;
  p.o.cols = w0->k;
  p.recs = w0->n_tiles * (w1 ? 2 : 1);
  p.o.alpha0 = unit_of(w0->format) * alpha;
  p.o.y = dx;
  p.o.ldy = lddx;
  p.o.y_f32 = dx_f32;
  p.o.vec = vec_ok(dx, lddx, dx_f32);
  return by_format<kDgrad>(ctx, w0->format, tm0, tm1, p, w0->k_blocks, s);
}

}  // namespace fp4
}  // namespace aex
