// fp4_small.cu — products of few rows (at most 16) with microscaled 4-bit
// weights: y = x W^T, or act(x Wg^T) * (x Wu^T).
//
// HBM-bound: the weight is read once. A CTA owns 128 weight rows (one column of
// records; the gated form one of each weight) and one K split of a
// thread-block cluster; a producer warp streams its records through a ring of
// shared-memory slots by bulk copies, eight compute warps take 16 rows each.
// The codes are decoded to bf16 pairs in registers (value * scale is exact:
// at most 6 significant bits) and multiplied on the tensor cores by
// mma.sync.m16n8k16 with the activations as the 8-column operand: at 1 to 8
// rows the work on a decoded pair is the same, and the decoding (2.5 integer
// and 1 multiply instructions per pair) is what the issue slots go to. tcgen05
// would need its operand written back to shared memory, which at these row
// counts costs more than the product.
// Sums: the tensor core's f32 accumulators truncate, so each 256-column block
// is summed there (16 steps) and then added to f32 registers; the K splits are
// added in rank order through distributed shared memory (no atomics).
// f32 activations enter as three bf16 columns (the top, middle and low 8 bits
// of the significand, by truncation: their sum is x exactly), so the products
// stay exact. Quantized activations are rounded while they are staged.
#include <algorithm>

#include "fp4.cuh"
#include "fp4_internal.h"

namespace aex {
namespace fp4 {

constexpr int kSmWarps = 8;
constexpr int kSmCompute = kSmWarps * 32;
constexpr int kSmThreads = kSmCompute + 32;
constexpr int kSmMaxSplit = 8;
constexpr size_t kSmXBudget = 68 * 1024;  // staged activations of one phase

struct SmallParams {
  const uint8_t* w0;
  const uint8_t* w1;
  const void* x;
  int64_t ldx;
  int x_f32, quantize;
  float x_scale, inv_6ts;
  int m, k, n, k_blocks;
  int kb_per_split;
  int kb_phase;  // records' worth of columns staged at a time
  int slots;
  float alpha0, alpha1;  // what the two accumulators are multiplied by
  int activation;
  void* y;
  int64_t ldy;
  int y_f32;
  int* status;
};

__host__ __device__ constexpr int sm_slot_bytes(int format, bool gated) { return rec_bytes(format) * (gated ? 2 : 1); }

__device__ __forceinline__ void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The 16-byte unit u (8 columns) of a 256-column block sits at unit sm_pos(u)
// of its staged column: the four lanes of a row quad read units 8t + 4h + w
// (t the lane) together, so those four are neighbours.
__device__ __forceinline__ int sm_pos(int u) { return ((u & 7) << 2) | (u >> 3); }

// Stages columns [k0, k0 + 256 nkb) of the m rows; `pitch` bytes per column.
template <int kFormat>
__device__ __forceinline__ void sm_stage(const SmallParams& p, uint8_t* xs, int pitch, int k0, int nkb, int t) {
  if (p.quantize) {
    const int upr = nkb * 16, items = p.m * upr;
    for (int i0 = 0; i0 < items; i0 += kSmCompute) {
      const int i = i0 + t;
      const int mr = i / upr, c = i % upr, col = k0 + c * 16;
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0.f;
      if (i < items && col < p.k) {
        if (p.x_f32) {
          const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + mr * p.ldx + col);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 f = __ldg(s + e);
            v[4 * e] = f.x;
            v[4 * e + 1] = f.y;
            v[4 * e + 2] = f.z;
            v[4 * e + 3] = f.w;
          }
        } else {
          const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + mr * p.ldx + col);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint4 u = __ldg(s + e);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              v[8 * e + 2 * j] = bf16lo_to_f32(w[j]);
              v[8 * e + 2 * j + 1] = bf16hi_to_f32(w[j]);
            }
          }
        }
      }
      uint32_t w[2], sb;
      quantize16<kFormat, true>(v, p.x_scale, p.inv_6ts, w, &sb);
      if (i < items) {
        const uint32_t s2 = scale_pair<kFormat>(sb);
        uint8_t* dst = xs + mr * pitch + (c >> 4) * 512;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4*>(dst + sm_pos((c & 15) * 2 + h) * 16) =
              make_uint4(decode_pair<kFormat>(w[h], 0, s2), decode_pair<kFormat>(w[h], 1, s2),
                         decode_pair<kFormat>(w[h], 2, s2), decode_pair<kFormat>(w[h], 3, s2));
      }
    }
  } else {
    const int upr = nkb * 32, items = p.m * upr;
    for (int i = t; i < items; i += kSmCompute) {
      const int mr = i / upr, c = i % upr, col = k0 + c * 8;
      const int off = (c >> 5) * 512 + sm_pos(c & 31) * 16;
      if (p.x_f32) {
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (col < p.k) {
          const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + mr * p.ldx + col);
          const float4 a = __ldg(s), b = __ldg(s + 1);
          f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        }
        uint32_t hi[8], mid[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t u = __float_as_uint(f[e]);
          hi[e] = u & 0xFFFF0000u;
          const float r1 = f[e] - __uint_as_float(hi[e]);
          mid[e] = __float_as_uint(r1) & 0xFFFF0000u;
          lo[e] = __float_as_uint(r1 - __uint_as_float(mid[e])) & 0xFFFF0000u;
          if ((u & 0x7F800000u) == 0x7F800000u) {  // infinity, NaN: the top column alone carries it
            if (u & 0x007FFFFFu) hi[e] = 0x7FC00000u;
            mid[e] = lo[e] = 0u;
          }
        }
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          const uint32_t* b = part == 0 ? hi : part == 1 ? mid : lo;
          *reinterpret_cast<uint4*>(xs + (3 * mr + part) * pitch + off) =
              make_uint4(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632),
                         __byte_perm(b[4], b[5], 0x7632), __byte_perm(b[6], b[7], 0x7632));
        }
      } else {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (col < p.k)
          u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + mr * p.ldx + col));
        *reinterpret_cast<uint4*>(xs + mr * pitch + off) = u;
      }
    }
  }
}

// One record against the staged columns of its block: acc += (16 rows of this
// warp) x (8 kT columns). xb: this lane's column (of tile 0) and quad position.
template <int kFormat, int kT>
__device__ __forceinline__ void sm_record(const uint4* codes, const uint32_t* scales, const uint8_t* xb, int pitch,
                                          int cols, int g, int t, float (*acc)[4]) {
  float c[kT][4];
#pragma unroll
  for (int i = 0; i < kT; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t wa[4] = {codes[h].x, codes[h].y, codes[h].z, codes[h].w};
    const uint32_t wb[4] = {codes[2 + h].x, codes[2 + h].y, codes[2 + h].z, codes[2 + h].w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      // nvfp4: scales of columns 32h + 16(w / 2) in byte 2h + w / 2; mxfp4: byte h of the lane's pair
      const int sh = kFormat == AEX_FP4_NV ? 8 * (2 * h + (w >> 1)) : 8 * (2 * (t & 1) + h);
      const uint32_t sa = scale_pair<kFormat>((scales[0] >> sh) & 0xFFu);
      const uint32_t sb = scale_pair<kFormat>((scales[1] >> sh) & 0xFFu);
      uint32_t pa[4], pb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pa[j] = decode_pair<kFormat>(wa[w], j, sa);
        pb[j] = decode_pair<kFormat>(wb[w], j, sb);
      }
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        uint4 b = make_uint4(0, 0, 0, 0);
        if (8 * i + g < cols) b = *reinterpret_cast<const uint4*>(xb + 8 * i * pitch + (h * 4 + w) * 64);
        mma_bf16(c[i], pa[0], pb[0], pa[1], pb[1], b.x, b.y);
        mma_bf16(c[i], pa[2], pb[2], pa[3], pb[3], b.z, b.w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] += c[i][e];
}

template <int kFormat, int kT, bool kGated>
__global__ void __launch_bounds__(kSmThreads) small_kernel(const __grid_constant__ SmallParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kSlot = sm_slot_bytes(kFormat, kGated);
  constexpr int kRec = rec_bytes(kFormat);
  const int slots = p.slots;
  uint8_t* ring = smem;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + slots * kSlot);
  uint64_t* empty = full + slots;
  uint8_t* xs = reinterpret_cast<uint8_t*>(full) + 128;  // at most 8 slots
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rt = blockIdx.x, split = blockIdx.y;
  const int kb0 = split * p.kb_per_split;
  const int nkb = max(0, min(p.k_blocks, kb0 + p.kb_per_split) - kb0);
  const int parts = p.x_f32 && !p.quantize ? 3 : 1;
  const int cols = p.m * parts;
  if (tid == 0) {
    abort_flag = 0;
    for (int s = 0; s < slots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kSmWarps);
    }
    fence_barrier_init();
  }
  __syncthreads();
  float acc0[kT][4], acc1[kGated ? kT : 1][4];
#pragma unroll
  for (int i = 0; i < kT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc0[i][e] = 0.f;
      if (kGated) acc1[i][e] = 0.f;
    }
  int issued = 0;
  if (warp == kSmWarps) {
    if (lane == 0) {
      for (int b = 0; b < nkb; ++b) {
        const int s = b % slots;
        if (b >= slots && !mbar_wait(&empty[s], ((b / slots) - 1) & 1, &abort_flag, p.status, kDevTimeoutProducer))
          break;
        const size_t at = (static_cast<size_t>(rt) * p.k_blocks + kb0 + b) * kRec;
        mbar_arrive_expect_tx(&full[s], kSlot);
        bulk_load(ring + s * kSlot, p.w0 + at, kRec, &full[s]);
        if (kGated) bulk_load(ring + s * kSlot + kRec, p.w1 + at, kRec, &full[s]);
        issued = b + 1;
      }
    }
    __syncwarp();
  } else {
    const int g = lane >> 2, t = lane & 3;
    const int pitch = p.kb_phase * 512 + 64;
    const int row = warp * 16 + g;  // and row + 8
    bool ok = true;
    for (int b = 0; b < nkb; ++b) {
      const int in_phase = b % p.kb_phase;
      if (in_phase == 0) {
        if (b) asm volatile("bar.sync 1, %0;" ::"n"(kSmCompute) : "memory");  // the previous columns are used
        sm_stage<kFormat>(p, xs, pitch, (kb0 + b) * kRecK, min(p.kb_phase, nkb - b), tid);
        asm volatile("bar.sync 1, %0;" ::"n"(kSmCompute) : "memory");
      }
      const int s = b % slots;
      if (ok) ok = mbar_wait_warp(&full[s], (b / slots) & 1, &abort_flag, p.status, kDevTimeoutTma);
      if (!ok) continue;  // the barriers above still see every warp
      const uint8_t* xb = xs + g * pitch + in_phase * 512 + t * 16;
      uint4 codes[kGated ? 8 : 4];
      uint32_t sc[kGated ? 4 : 2];
#pragma unroll
      for (int q = 0; q < (kGated ? 2 : 1); ++q) {
        const uint8_t* rec = ring + s * kSlot + q * kRec;
#pragma unroll
        for (int r8 = 0; r8 < 2; ++r8) {
          const uint8_t* rp = rec + (row + 8 * r8) * 128;
          codes[4 * q + 2 * r8] = *reinterpret_cast<const uint4*>(rp + (((2 * t) ^ g) << 4));
          codes[4 * q + 2 * r8 + 1] = *reinterpret_cast<const uint4*>(rp + (((2 * t + 1) ^ g) << 4));
          sc[2 * q + r8] = *reinterpret_cast<const uint32_t*>(
              rec + scale_off(row + 8 * r8, kFormat == AEX_FP4_NV ? t : t >> 1));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_addr(smem_u32(&empty[s]));  // the warp's reads of the slot are done
      sm_record<kFormat, kT>(codes, sc, xb, pitch, cols, g, t, acc0);
      if (kGated) sm_record<kFormat, kT>(codes + 4, sc + 2, xb, pitch, cols, g, t, acc1);
    }
  }
  __syncthreads();  // every copy has landed and been read: the ring becomes the partial sums [cols][128]
  if (abort_flag) {
    // A wait ran out: the copies in flight land before the ring is written or the CTA exits.
    for (int b = max(0, issued - slots); b < issued; ++b) {
      const uint32_t a = smem_u32(&full[b % slots]);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(a, (b / slots) & 1) && globaltimer_ns() - t0 < kWaitTimeoutNs) {
      }
    }
    __syncthreads();
  }
  float* part0 = reinterpret_cast<float*>(ring);
  float* part1 = part0 + cols * kRecRows;
  if (warp < kSmWarps) {
    const int g = lane >> 2, t = lane & 3, row = warp * 16 + g;
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 8 * i + 2 * t + (e & 1), r = row + (e >> 1) * 8;
        if (c < cols) {
          part0[c * kRecRows + r] = acc0[i][e];
          if (kGated) part1[c * kRecRows + r] = acc1[i][e];
        }
      }
  }
  cluster_sync_all();
  const int nsplit = static_cast<int>(gridDim.y);
  const uint32_t a0 = smem_u32(part0), a1 = smem_u32(part1);
  for (int i = split * kSmThreads + tid; i < p.m * kRecRows; i += nsplit * kSmThreads) {
    const int mr = i / kRecRows, r = i % kRecRows;
    const int64_t col = static_cast<int64_t>(rt) * kRecRows + r;
    if (col >= p.n) continue;
    float v0 = 0.f, v1 = 0.f;
    for (int c = 0; c < nsplit; ++c)
      for (int q = 0; q < parts; ++q) {
        const uint32_t off = ((mr * parts + q) * kRecRows + r) * 4;
        v0 += ld_shared_cluster_f32(mapa_shared(a0 + off, c));
        if (kGated) v1 += ld_shared_cluster_f32(mapa_shared(a1 + off, c));
      }
    v0 *= p.alpha0;
    if (kGated) {
      v1 *= p.alpha1;
      v0 = v0 * sigmoid<false>(sigmoid_arg(v0, p.activation)) * v1;
    }
    if (p.y_f32)
      static_cast<float*>(p.y)[static_cast<int64_t>(mr) * p.ldy + col] = v0;
    else
      static_cast<uint16_t*>(p.y)[static_cast<int64_t>(mr) * p.ldy + col] =
          static_cast<uint16_t>(pack_bf16x2(v0, 0.f) & 0xFFFFu);
  }
  __syncwarp();
  cluster_sync_all();  // every CTA's shared memory stays until its peers have read it
}

namespace {

template <int kFormat, int kT, bool kGated>
int launch_small(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  const aex_fp4weight* w = j.w0;
  const int cols = j.m * (j.x_f32 && !j.quantize ? 3 : 1);
  SmallParams p{};
  p.w0 = w->records;
  p.w1 = kGated ? j.w1->records : nullptr;
  p.x = j.x;
  p.ldx = j.ldx;
  p.x_f32 = j.x_f32;
  p.quantize = j.quantize;
  p.x_scale = j.x_scale;
  p.inv_6ts = static_cast<float>(1.0 / (6.0 * static_cast<double>(j.x_scale)));
  p.m = j.m;
  p.k = w->k;
  p.n = w->n;
  p.k_blocks = w->k_blocks;
  const double unit = decode_unit<kFormat>() * (j.quantize ? decode_unit<kFormat>() * static_cast<double>(j.x_scale) : 1.0);
  p.alpha0 = static_cast<float>(unit * w->tensor_scale);
  p.alpha1 = kGated ? static_cast<float>(unit * j.w1->tensor_scale) : 0.f;
  p.activation = j.activation;
  p.y = j.y;
  p.ldy = j.ldy;
  p.y_f32 = j.y_f32;
  p.status = ctx->d_status;

  auto kern = small_kernel<kFormat, kT, kGated>;
  constexpr int kSlot = sm_slot_bytes(kFormat, kGated);
  constexpr int kMaxSmem = 226 * 1024;
  AEX_CUDA_TRY(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
  // K split: the largest whose CTAs run in one wave (more copies in flight per
  // weight row), else the one of the fewest waves.
  int best_split = 0, best_slots = 0, best_phase = 0;
  int64_t best_waves = 0;
  size_t best_smem = 0;
  for (int sp = 1; sp <= std::min(kSmMaxSplit, w->k_blocks); ++sp) {
    const int kb = (w->k_blocks + sp - 1) / sp;
    if ((w->k_blocks + kb - 1) / kb != sp) continue;  // an empty split
    const int slots = std::min(kb, 4);
    int phase = kb;
    while (phase > 1 && static_cast<size_t>(cols) * (phase * 512 + 64) > kSmXBudget) phase = (phase + 1) / 2;
    // the partial sums take the ring's place
    const size_t partial = static_cast<size_t>(cols) * kRecRows * 4 * (kGated ? 2 : 1);
    size_t smem = static_cast<size_t>(slots) * kSlot + 128 + static_cast<size_t>(cols) * (phase * 512 + 64);
    smem = std::max(smem, partial);
    const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>(4, (227 * 1024) / (smem + 1024)));
    const int64_t waves = (static_cast<int64_t>(w->n_tiles) * sp + per_sm * ctx->sm_count - 1) / (per_sm * ctx->sm_count);
    if (!best_split || waves <= best_waves) {
      best_split = sp;
      best_waves = waves;
      best_slots = slots;
      best_phase = phase;
      best_smem = smem;
    }
  }
  p.kb_per_split = (w->k_blocks + best_split - 1) / best_split;
  p.kb_phase = best_phase;
  p.slots = best_slots;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(w->n_tiles, best_split, 1);
  cfg.blockDim = dim3(kSmThreads, 1, 1);
  cfg.dynamicSmemBytes = best_smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = best_split;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AEX_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kern, p));
  return check_launch(ctx, "fp4 small_kernel");
}

template <int kFormat, bool kGated>
int pick_tiles(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  const int cols = j.m * (j.x_f32 && !j.quantize ? 3 : 1);
  if (cols <= 8) return launch_small<kFormat, 1, kGated>(ctx, j, s);
  if (cols <= 16) return launch_small<kFormat, 2, kGated>(ctx, j, s);
  return launch_small<kFormat, 6, kGated>(ctx, j, s);  // 17..48 columns: f32 rows
}

}  // namespace

int run_small(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  if (j.w0->format == AEX_FP4_MX)
    return j.w1 ? pick_tiles<AEX_FP4_MX, true>(ctx, j, s) : pick_tiles<AEX_FP4_MX, false>(ctx, j, s);
  return j.w1 ? pick_tiles<AEX_FP4_NV, true>(ctx, j, s) : pick_tiles<AEX_FP4_NV, false>(ctx, j, s);
}

}  // namespace fp4
}  // namespace aex
