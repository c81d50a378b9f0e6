// fp4_small.cu — products of few rows (at most 16) with microscaled 4-bit
// weights: y = x W^T, or act(x Wg^T) * (x Wu^T).
//
// The weight is read once, and the work on its codes takes longer than that: one
// row 4096 -> 9216 nvfp4 8.1 us (2.6 TB/s), 3 f32 rows 4096 -> 18431 mxfp4 15.7 us
// (2.6). Half to two thirds of the issue slots are taken; the rest is latency (staging,
// the first records, the sum over the cluster). A CTA owns 128 weight rows (one
// column of records; the gated form one of each weight) and one K split of a
// thread-block cluster; a producer warp streams its records through a ring of
// shared-memory slots by bulk copies, compute warps take 16 rows each, up to
// three sets of eight warps that take turns at the records (one set left the
// SM's schedulers idle over half of the time). The number of slots is a multiple
// of the sets, or enough for every record: a slot's records then all belong to
// one set, which so sees every phase of the slot's barriers.
// The codes are decoded in registers and multiplied on the tensor cores by
// mma.sync.m16n8k16 with the activations as the 8-column operand: at 1 to 8
// rows the work on a decoded pair is the same, and the decoding is what the
// issue slots go to. (tcgen05 would need its operand written back to shared
// memory, which at these row counts costs more than the product.)
//
// Decoding to f16, not bf16: a pair of e2m1 codes becomes an f16 pair in one
// conversion, against four integer operations to a bf16 pair (measured on one
// SM sub-partition: two cycles each). So the activations have to be f16 too.
// Each row's 256 columns of a record are scaled by a power of two that puts the
// largest magnitude into [2^14, 2^15); 11 bits of significand down to 2^-24
// then hold bf16 values over 31 binades exactly. Whether they do is checked
// value by value as they are staged; a record's columns for which they do not
// (or that hold an infinity or NaN) are staged as bf16 and take the integer
// decoding, which covers every value. Both products of bf16 rows are exact.
// f32 rows take two columns, 11 + 11 bits and the sign between them, each with a
// scale of its own: a value is held to within 2^-23 of itself, less than its
// f32 products' sums lose, and checked as well (a third column for the last bit
// cost 3 rows, 4096 -> 18431, 19.8 us against 15.1). As bf16: 8 + 8 + 8 bits, by
// truncation, the last 8 in a second product.
// Scales: nvfp4, 16 columns: into the decoded pair (2 + 4 bits, exact in f16);
// mxfp4, 32 columns: exponents that f16 does not hold, so one column block is
// summed over two products and enters the f32 sum times its scale.
// Sums: the tensor core's f32 accumulators truncate, so a record is summed
// there (16 steps) and then added to f32 registers; the K splits are added in
// rank order through distributed shared memory (no atomics).
#include <cuda_fp16.h>

#include <algorithm>

#include "fp4.cuh"
#include "fp4_internal.h"

namespace aex {
namespace fp4 {

// Sets of eight compute warps, by the registers that 8 kT activation columns take.
__host__ __device__ constexpr int sm_ways(int kT) { return kT == 1 ? 3 : 2; }
__host__ __device__ constexpr int sm_warps(int kT) { return 8 * sm_ways(kT); }
__host__ __device__ constexpr int sm_threads(int kT) { return sm_warps(kT) * 32 + 32; }
constexpr int kSmMaxSplit = 8;
constexpr int kSmSmem = 226 * 1024;

struct SmallParams {
  const uint8_t* w0;
  const uint8_t* w1;
  const void* x;
  int64_t ldx;
  int x_f32, quantize;
  float x_scale, inv_6ts;
  int m, k, n, k_blocks;
  int m_inv;     // i / m = i * m_inv >> 16 for i <= 512
  int kb_per_split;
  int kb_phase;  // records' worth of columns staged at a time
  int slots;
  float alpha0, alpha1;  // what the two accumulators are multiplied by
  int activation;
  void* y;
  int64_t ldy;
  int y_f32;
  uint32_t zero;  // 0 (arrive_after_loads)
  int* status;
};

__host__ __device__ constexpr int sm_slot_bytes(int format, bool gated) { return rec_bytes(format) * (gated ? 2 : 1); }

// d (+)= a b, one 16 x 8 x 16 product; pa, pb: the pairs of rows g and g + 8.
template <bool kBf16>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* pa, const uint32_t* pb, uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(pa[0]), "r"(pb[0]), "r"(pa[1]), "r"(pb[1]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(pa[0]), "r"(pb[0]), "r"(pa[1]), "r"(pb[1]), "r"(b0), "r"(b1));
}
template <bool kBf16>
__device__ __forceinline__ void mma16816_first(float* d, const uint32_t* pa, const uint32_t* pb, uint32_t b0,
                                               uint32_t b1) {
  if (kBf16)
    asm volatile(
        "{\n\t.reg .f32 z;\n\tmov.f32 z, 0f00000000;\n\t"
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {z,z,z,z};\n\t}"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(pa[0]), "r"(pb[0]), "r"(pa[1]), "r"(pb[1]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "{\n\t.reg .f32 z;\n\tmov.f32 z, 0f00000000;\n\t"
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {z,z,z,z};\n\t}"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(pa[0]), "r"(pb[0]), "r"(pa[1]), "r"(pb[1]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float lds_f32(uint32_t a) { return __uint_as_float(lds32(a)); }

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Two e4m3 bytes (the low half of v) as an f16 pair.
__device__ __forceinline__ uint32_t e4m3_pair_f16(uint32_t v) {
  uint32_t d;
  asm("{\n\t.reg .b16 t, u;\n\tmov.b32 {t, u}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ float f16_value(uint32_t b) { return __half2float(__ushort_as_half(static_cast<uint16_t>(b))); }

// Where a lane quad finds its operand: the 16-byte unit u (8 columns) of a
// record's 256 columns sits at unit sm_pos(u) of its staged column, so that the
// four lanes of a quad read neighbours. mxfp4: lane t takes word t of a chunk
// of 32 columns, the natural order; nvfp4: words of chunks 2t and 2t + 1.
template <int kFormat>
__device__ __forceinline__ int sm_pos(int u) {
  return kFormat == AEX_FP4_MX ? u : ((u & 7) << 2) | (u >> 3);
}

// Staged activations of a phase: columns of `pitch` bytes at xs, f32 rows' third
// parts (wide records only) `third` bytes on, then per column and record the
// factor that undoes its scale; *wide: a bit per record.
struct SmStage {
  uint8_t* xs;
  float* factor;  // [kb_phase][cols]
  uint32_t* wide;
  int pitch, cols, third;
};

__device__ __forceinline__ uint32_t cvt_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Stages columns 8l..8l+7 of a row and record as f16 halves: bf16 rows, eight
// values w. False unless every value is held exactly. 2^k takes the largest of
// the record into [2^14, 2^15); f16 then holds all of a value's 8 bits down to
// 2^-17, which is 31 binades below.
__device__ __forceinline__ bool sm_stage_bf16(const uint4& q, uint8_t* dst, float* factor, int lane) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t top2 = 0, low2 = 0xFFFFFFFFu;  // of the two halves: the largest magnitude, the smallest less one
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t mag = w[j] & 0x7FFF7FFFu;
    top2 = __vmaxu2(top2, mag);
    low2 = __vminu2(low2, (mag + 0x7FFF7FFFu) ^ 0x80008000u);  // a zero becomes 0xFFFF
  }
  const uint32_t top = __reduce_max_sync(0xffffffffu, max(top2 & 0xFFFFu, top2 >> 16));
  const int e0 = top ? static_cast<int>(top >> 7) - 127 : 14;
  const bool fits = e0 >= -48 && e0 <= 62;
  const int k = fits ? 14 - e0 : 0;
  const float up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
  float v[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = bf16lo_to_f32(w[j]) * up;
    v[2 * j + 1] = bf16hi_to_f32(w[j]) * up;
  }
  *reinterpret_cast<uint4*>(dst) =
      make_uint4(cvt_f16x2(v[0], v[2]), cvt_f16x2(v[4], v[6]), cvt_f16x2(v[1], v[3]), cvt_f16x2(v[5], v[7]));
  if (lane == 0) *factor = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
  return fits && min(low2 & 0xFFFFu, low2 >> 16) + 1 >= static_cast<uint32_t>(e0 + 127 - 31) << 7;
}

// The same of f32 values v in kParts halves: one holds them exactly (quantized
// ones) or the record is wide, two to within 2^-23 of each value.
template <int kParts>
__device__ __forceinline__ bool sm_stage_f32(const float* v, uint8_t* dst, int pitch, float* factor, int lane) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
  top = __reduce_max_sync(0xffffffffu, top);
  // outside 2^-48 .. 2^62 (and for what is not finite) bf16
  const int e0 = top ? static_cast<int>(top >> 23) - 127 : 14;
  bool held = e0 >= -48 && e0 <= 62;
  const int k = held ? 14 - e0 : 0;
  const float up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    r[e] = v[e] * up;
    held &= !(r[e] == 0.f && v[e] != 0.f);
  }
  float down = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    constexpr int kFirst[4] = {0, 4, 1, 5};
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = kFirst[j];
      h[j] = cvt_f16x2(r[e], r[e + 2]);
      r[e] = (r[e] - f16_value(h[j] & 0xFFFFu)) * 2048.f;  // what is left, to the next part's scale
      r[e + 2] = (r[e + 2] - f16_value(h[j] >> 16)) * 2048.f;
    }
    *reinterpret_cast<uint4*>(dst + part * pitch) = make_uint4(h[0], h[1], h[2], h[3]);
    if (lane == 0) factor[part] = down;
    down *= 1.f / 2048.f;
  }
  constexpr float most = kParts == 2 ? 0.5f : 0.f;  // what two parts leave stands 2^22 too high
#pragma unroll
  for (int e = 0; e < 8; ++e) held &= fabsf(r[e]) <= most * fabsf(v[e] * up);
  return held;
}

// Columns 8l..8l+7 of item i's row and record, as they stand (zeros past the last column and item). Plain loads: the
// read-only path is for what nobody writes while the kernel runs, and this one is set up while the previous runs.
struct SmItem {
  int b, mr;
  uint4 lo, hi;
};
__device__ __forceinline__ SmItem sm_fetch(const SmallParams& p, int kb0, int i, int items, int lane) {
  SmItem t;
  t.b = i * p.m_inv >> 16;
  t.mr = i - t.b * p.m;
  t.lo = t.hi = make_uint4(0, 0, 0, 0);
  const int col = (kb0 + t.b) * kRecK + lane * 8;
  if (i < items && col < p.k) {
    if (p.x_f32) {
      const uint4* s = reinterpret_cast<const uint4*>(static_cast<const float*>(p.x) + t.mr * p.ldx + col);
      t.lo = s[0];
      t.hi = s[1];
    } else {
      t.lo = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + t.mr * p.ldx + col);
    }
  }
  return t;
}
// Its values, quantized where that is asked for.
template <int kFormat>
__device__ __forceinline__ void sm_values(const SmallParams& p, const SmItem& t, float* v) {
  if (p.x_f32) {
    const uint32_t w[8] = {t.lo.x, t.lo.y, t.lo.z, t.lo.w, t.hi.x, t.hi.y, t.hi.z, t.hi.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[e]);
  } else {
    const uint32_t w[4] = {t.lo.x, t.lo.y, t.lo.z, t.lo.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = bf16lo_to_f32(w[j]);
      v[2 * j + 1] = bf16hi_to_f32(w[j]);
    }
  }
  if (p.quantize) {
    uint32_t top = 0, w, d[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    const float s = scale_to_f32<kFormat>(quantize_cols<kFormat, 8, false>(v, top, p.x_scale, p.inv_6ts, &w));
    decode_f16(w, d);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = f16_value(d[j] & 0xFFFFu) * s;  // exact
      v[2 * j + 1] = f16_value(d[j] >> 16) * s;
    }
  }
}

// One warp per row and record; notes in *wide which records need bf16.
template <int kFormat, int kParts>
__device__ __forceinline__ void sm_stage(const SmallParams& p, const SmStage& st, int kb0, int nkb, int warp, int warps,
                                         int lane) {
  const int items = p.m * nkb;
  const auto place = [&](const SmItem& t) {
    return st.xs + t.mr * kParts * st.pitch + t.b * 512 + sm_pos<kFormat>(lane) * 16;
  };
  const auto note = [&](const SmItem& t, bool held) {
    if (!__all_sync(0xffffffffu, held) && lane == 0) atomicOr(st.wide, 1u << t.b);
  };
  if (kParts == 1 && !p.x_f32 && !p.quantize) {
    constexpr int kAhead = 4;  // items whose loads are on their way at once
#pragma unroll 1
    for (int i = warp; i < items; i += kAhead * warps) {
      SmItem t[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) t[j] = sm_fetch(p, kb0, i + j * warps, items, lane);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i + j * warps < items)
          note(t[j], sm_stage_bf16(t[j].lo, place(t[j]), st.factor + t[j].b * st.cols + t[j].mr, lane));
    }
    return;
  }
  SmItem next = sm_fetch(p, kb0, warp, items, lane);
#pragma unroll 1
  for (int i = warp; i < items; i += warps) {
    const SmItem t = next;
    next = sm_fetch(p, kb0, i + warps, items, lane);
    float v[8];
    sm_values<kFormat>(p, t, v);
    note(t, sm_stage_f32<kParts>(v, place(t), st.pitch, st.factor + t.b * st.cols + t.mr * kParts, lane));
  }
}

// Stages the records of `only` again, as bf16 (not inlined: it is rare, and its registers cost the main loop some).
template <int kFormat, int kParts>
__device__ __noinline__ void sm_stage_wide(const SmallParams& p, SmStage st, int kb0, int nkb, uint32_t only,
                                           int warp, int warps, int lane) {
  const int items = p.m * nkb;
#pragma unroll 1
  for (int i = warp; i < items; i += warps) {
    const SmItem t = sm_fetch(p, kb0, i, items, lane);
    if (!((only >> t.b) & 1u)) continue;
    float v[8];
    sm_values<kFormat>(p, t, v);
    uint8_t* dst = st.xs + t.mr * kParts * st.pitch + t.b * 512 + sm_pos<kFormat>(lane) * 16;
    uint32_t h[8];
#pragma unroll 1
    for (int part = 0; part < (kParts == 2 ? 3 : 1); ++part) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // the top 8 bits, exactly what there is where x has no more; an infinity or NaN is in the first part alone
        const uint32_t u = __float_as_uint(v[e]);
        const bool special = (u & 0x7F800000u) == 0x7F800000u;
        h[e] = special && (u & 0x007FFFFFu) ? 0x7FC0u : u >> 16;
        v[e] = special ? 0.f : v[e] - __uint_as_float(u & 0xFFFF0000u);
      }
      const uint4 o = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
      if (part < 2) {
        *reinterpret_cast<uint4*>(dst + part * st.pitch) = o;
        if (lane == 0)
          st.factor[t.b * st.cols + t.mr * kParts + part] = kFormat == AEX_FP4_NV ? 128.f : 1.f;
      } else {
        *reinterpret_cast<uint4*>(dst + st.third) = o;
        *reinterpret_cast<uint4*>(dst + st.third + st.pitch) = make_uint4(0, 0, 0, 0);
      }
    }
  }
}

// One record against the staged columns: acc += (16 rows of this warp) x (8 kT
// columns). codes: nvfp4, chunks 2t and 2t + 1 of row g, then of row g + 8;
// mxfp4, [chunk / 2] words of (chunk, row). xb: per 8 columns this lane's column
// and its place in a quad; fb: per 8 columns the factors of this lane's two.
template <int kFormat, int kT, bool kWide>
__device__ __forceinline__ void sm_record(const uint4* codes, const uint32_t* scales, const uint32_t* xb, uint32_t off,
                                          const uint32_t (*fb)[2], uint32_t foff, float (*acc)[4]) {
  float c[kT][4], f[kT][2];
#pragma unroll
  for (int i = 0; i < kT; ++i) {
    f[i][0] = lds_f32(fb[i][0] + foff);
    f[i][1] = lds_f32(fb[i][1] + foff);
  }
  if (kFormat == AEX_FP4_NV) {
    float d[kT][4];  // a second chain of sums: the products of one chain wait for one another
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // the two blocks of chunk 2t + h, both rows
      const uint32_t fa = kWide ? 0 : e4m3_pair_f16(scales[0] >> (16 * h));
      const uint32_t fc = kWide ? 0 : e4m3_pair_f16(scales[1] >> (16 * h));
      const uint32_t wa[4] = {codes[h].x, codes[h].y, codes[h].z, codes[h].w};
      const uint32_t wb[4] = {codes[2 + h].x, codes[2 + h].y, codes[2 + h].z, codes[2 + h].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t pa[4], pb[4];
        if (kWide) {
          const int sh = 16 * h + 8 * (w >> 1);
          const uint32_t sa = scale_pair<kFormat>((scales[0] >> sh) & 0xFFu);
          const uint32_t sb = scale_pair<kFormat>((scales[1] >> sh) & 0xFFu);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            pa[j] = decode_pair<kFormat>(wa[w], j, sa);
            pb[j] = decode_pair<kFormat>(wb[w], j, sb);
          }
        } else {
          const uint32_t sel = (w >> 1) ? 0x3232u : 0x1010u;
          const uint32_t sa = __byte_perm(fa, 0, sel), sb = __byte_perm(fc, 0, sel);
          decode_f16(wa[w], pa);
          decode_f16(wb[w], pb);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            pa[j] = mul_f16x2(pa[j], sa);
            pb[j] = mul_f16x2(pb[j], sb);
          }
        }
#pragma unroll
        for (int i = 0; i < kT; ++i) {
          const uint4 b = lds128(xb[i] + off + (h * 4 + w) * 64);
          if (h == 0 && w == 0) {
            mma16816_first<kWide>(c[i], pa, pb, b.x, b.y);
            mma16816_first<kWide>(d[i], pa + 2, pb + 2, b.z, b.w);
          } else {
            mma16816<kWide>(c[i], pa, pb, b.x, b.y);
            mma16816<kWide>(d[i], pa + 2, pb + 2, b.z, b.w);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[i][e] += d[i][e];
  } else {
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) {
      const uint4 q = codes[ch >> 1];
      const uint32_t wa = (ch & 1) ? q.z : q.x, wb = (ch & 1) ? q.w : q.y;
      // the scale byte as 2^(byte - 127): 0 is the subnormal, 255 infinity, which the multiplication makes NaN
      const uint32_t sel = 0x0444u | (static_cast<uint32_t>(ch & 3) << 12);
      float sa = __uint_as_float(max(__byte_perm(scales[2 * (ch >> 2)], 0, sel) >> 1, 0x00400000u));
      float sb = __uint_as_float(max(__byte_perm(scales[2 * (ch >> 2) + 1], 0, sel) >> 1, 0x00400000u));
      sa = fmaf(sa, 0.f, sa);
      sb = fmaf(sb, 0.f, sb);
      uint32_t pa[4], pb[4];
      if (kWide) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          pa[j] = mul_bf16x2(code_pair_tiny(wa, j), kBf16x2_2p126);
          pb[j] = mul_bf16x2(code_pair_tiny(wb, j), kBf16x2_2p126);
        }
      } else {
        decode_f16(wa, pa);
        decode_f16(wb, pb);
      }
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        const uint4 b = lds128(xb[i] + off + ch * 64);
        float d[4];
        mma16816_first<kWide>(d, pa, pb, b.x, b.y);
        mma16816<kWide>(d, pa + 2, pb + 2, b.z, b.w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // the column's own scale first: what is then multiplied is the f32 product's size, whatever the exponents
          const float s = e < 2 ? sa : sb, v = d[e] * f[i][e & 1];
          c[i][e] = ch == 0 ? v * s : fmaf(v, s, c[i][e]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kT; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc[i][e] = kFormat == AEX_FP4_NV ? fmaf(c[i][e], f[i][e & 1], acc[i][e]) : acc[i][e] + c[i][e];
  }
}

__device__ __forceinline__ uint4 ldmatrix_x4(uint32_t addr) {
  uint4 r;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(addr)
               : "memory");
  return r;
}

// Where this lane finds its codes and scales in a record (rows row0 + g and row0 + g + 8).
struct SmLane {
  uint32_t code[4], scale;
};
template <int kFormat>
__device__ __forceinline__ SmLane sm_lane(int row0, int g, int t, int lane) {
  SmLane o;
  if (kFormat == AEX_FP4_NV) {
#pragma unroll
    for (int h = 0; h < 2; ++h) o.code[h] = o.code[2 + h] = (row0 + g) * 128 + (((2 * t + h) ^ g) << 4);
    o.scale = scale_off(row0 + g, t);
  } else {
    // matrix i of four (8 rows x 16 bytes, addresses from lanes 8i..8i+7): chunk c + (i >> 1), row half i & 1;
    // lane (g, t) receives word t of row g of each
    const int row = row0 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
    for (int c2 = 0; c2 < 4; ++c2) o.code[c2] = row * 128 + (((2 * c2 + (lane >> 4)) ^ (row & 7)) << 4);
    o.scale = scale_off(row0 + g, 0);
  }
  return o;
}
template <int kFormat>
__device__ __forceinline__ void sm_load(uint32_t rec, const SmLane& o, uint4* codes, uint32_t* scales) {
  if (kFormat == AEX_FP4_NV) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      codes[h] = lds128(rec + o.code[h]);
      codes[2 + h] = lds128(rec + o.code[h] + 8 * 128);
    }
    scales[0] = lds32(rec + o.scale);
    scales[1] = lds32(rec + o.scale + 8 * 16);  // row + 8: in the same group of 32 rows
  } else {
#pragma unroll
    for (int c2 = 0; c2 < 4; ++c2) codes[c2] = ldmatrix_x4(rec + o.code[c2]);
#pragma unroll
    for (int q = 0; q < 4; ++q) scales[q] = lds32(rec + o.scale + (q >> 1) * 512 + (q & 1) * 8 * 16);
  }
}

template <int kFormat, int kT, bool kGated, int kParts>
__global__ void __launch_bounds__(sm_threads(kT)) small_kernel(const __grid_constant__ SmallParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kSlot = sm_slot_bytes(kFormat, kGated);
  constexpr int kRec = rec_bytes(kFormat);
  constexpr int kSmWarps = sm_warps(kT), kSmCompute = kSmWarps * 32, kSmThreads = sm_threads(kT);
  constexpr int kWays = sm_ways(kT);  // the warps that share 16 rows take turns at the records
  const int slots = p.slots;
  uint8_t* ring = smem;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + slots * kSlot);
  uint64_t* empty = full + slots;
  __shared__ int abort_flag;
  __shared__ uint32_t wide;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rt = blockIdx.x, split = blockIdx.y;
  const int kb0 = split * p.kb_per_split;
  const int nkb = max(0, min(p.k_blocks, kb0 + p.kb_per_split) - kb0);
  const int cols = p.m * kParts;
  SmStage st;
  st.xs = reinterpret_cast<uint8_t*>(full) + 128;  // at most 8 slots
  st.pitch = p.kb_phase * 512 + 64;
  st.third = cols * st.pitch;
  st.factor = reinterpret_cast<float*>(st.xs + kParts * cols * st.pitch);  // two parts: a third's columns in between
  st.wide = &wide;
  st.cols = cols;
  launch_dependents();
  if (tid == 0) {
    abort_flag = 0;
    wide = 0;
    for (int s = 0; s < slots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 8);
    }
    fence_barrier_init();
  }
  wait_dependency();  // x, and the weight, may be the previous kernel's
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
    const int row0 = (warp & 7) * 16, set = warp >> 3;
    const SmLane at = sm_lane<kFormat>(row0, g, t, lane);
    // A column past the last reads the last one's: its sums are not stored.
    uint32_t xb[kT], fb[kT][2];
#pragma unroll
    for (int i = 0; i < kT; ++i) {
      xb[i] = smem_u32(st.xs) + min(8 * i + g, cols - 1) * st.pitch + t * 16;
#pragma unroll
      for (int e = 0; e < 2; ++e) fb[i][e] = smem_u32(st.factor) + min(8 * i + 2 * t + e, cols - 1) * 4;
    }
    const uint32_t ring0 = smem_u32(ring), full0 = smem_u32(full), empty0 = smem_u32(empty);
    bool ok = true;
    uint32_t wide_now = 0;
    // slot s and its phase bit, and the record's place in the staged columns, advance with b
    uint32_t s = 0, ph = 0;
    int in_phase = 0, turn = 0;
#pragma unroll 1
    for (int b = 0; b < nkb; ++b, ++in_phase) {
      if (in_phase == p.kb_phase) in_phase = 0;
      if (in_phase == 0) {
        const int count = min(p.kb_phase, nkb - b);
        if (b) {
          asm volatile("bar.sync 1, %0;" ::"n"(kSmCompute) : "memory");  // the previous columns are used
          if (tid == 0) wide = 0;
          asm volatile("bar.sync 1, %0;" ::"n"(kSmCompute) : "memory");
        }
        sm_stage<kFormat, kParts>(p, st, kb0 + b, count, warp, kSmWarps, lane);
        asm volatile("bar.sync 1, %0;" ::"n"(kSmCompute) : "memory");
        wide_now = *reinterpret_cast<volatile uint32_t*>(&wide);
        if (wide_now) {
          sm_stage_wide<kFormat, kParts>(p, st, kb0 + b, count, wide_now, warp, kSmWarps, lane);
          asm volatile("bar.sync 1, %0;" ::"n"(kSmCompute) : "memory");
        }
      }
      const uint32_t cs = s, cph = ph;
      if (++s == static_cast<uint32_t>(slots)) {
        s = 0;
        ph ^= 1;
      }
      const bool mine = turn == set;
      if (++turn == kWays) turn = 0;
      if (!mine) continue;
      if (ok) ok = mbar_wait_warp_addr(full0 + 8 * cs, cph, &abort_flag, p.status, kDevTimeoutTma);
      if (!ok) continue;  // the barriers above still see every warp
      const uint32_t off = in_phase * 512, foff = in_phase * cols * 4;
      const bool narrow = !((wide_now >> in_phase) & 1u);
      const int passes = kParts == 1 || narrow ? 1 : kParts;  // the second: the third parts of f32 rows
#pragma unroll 1
      for (int pass = 0; pass < passes; ++pass) {
        uint32_t all = 0;
#pragma unroll
        for (int q = 0; q < (kGated ? 2 : 1); ++q) {
          uint4 codes[4];
          uint32_t sc[kFormat == AEX_FP4_NV ? 2 : 4];
          sm_load<kFormat>(ring0 + cs * kSlot + q * kRec, at, codes, sc);
#pragma unroll
          for (int i = 0; i < 4; ++i) all |= codes[i].x | codes[i].y | codes[i].z | codes[i].w;
#pragma unroll
          for (int i = 0; i < (kFormat == AEX_FP4_NV ? 2 : 4); ++i) all |= sc[i];
          if (q == (kGated ? 1 : 0) && pass == passes - 1)
            arrive_after_loads(empty0 + 8 * cs, all, p.zero, lane);  // the warp's reads of the slot are done
          if (narrow)
            sm_record<kFormat, kT, false>(codes, sc, xb, off, fb, foff, q ? acc1 : acc0);
          else
            sm_record<kFormat, kT, true>(codes, sc, xb, off + pass * st.third, fb, foff, q ? acc1 : acc0);
        }
      }
    }
  }
  __syncthreads();  // every copy has landed and been read: the ring becomes the partial sums [ways][cols][128]
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
  float* part1 = part0 + kWays * cols * kRecRows;
  if (warp < kSmWarps) {
    const int g = lane >> 2, t = lane & 3, row = (warp & 7) * 16 + g, set = warp >> 3;
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c0 = 8 * i + 2 * t + (e & 1), c = set * cols + c0, r = row + (e >> 1) * 8;
        if (c0 < cols) {
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
      for (int q = 0; q < kWays * kParts; ++q) {
        const uint32_t off = (((q % kWays) * cols + mr * kParts + q / kWays) * kRecRows + r) * 4;
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

template <int kFormat, int kT, bool kGated, int kParts>
int launch_small(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  const aex_fp4weight* w = j.w0;
  const int cols = j.m * kParts;
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
  p.m_inv = 65536 / j.m + 1;
  p.k = w->k;
  p.n = w->n;
  p.k_blocks = w->k_blocks;
  const double unit = j.quantize ? static_cast<double>(j.x_scale) : 1.0;
  p.alpha0 = static_cast<float>(unit * w->tensor_scale);
  p.alpha1 = kGated ? static_cast<float>(unit * j.w1->tensor_scale) : 0.f;
  p.activation = j.activation;
  p.y = j.y;
  p.ldy = j.ldy;
  p.y_f32 = j.y_f32;
  p.status = ctx->d_status;

  auto kern = small_kernel<kFormat, kT, kGated, kParts>;
  constexpr int kSlot = sm_slot_bytes(kFormat, kGated);
  static SmemOptIn opt_in;
  if (int r = opt_in(ctx, reinterpret_cast<const void*>(kern), kSmSmem)) return r;
  // K split: the one that leaves the busiest SM the fewest records (CTAs that share an SM share its schedulers), the
  // smallest of those (less to add up). 72 row tiles of 16 records (B200, one row): split 2, 144 CTAs.
  int best_split = 1;
  int64_t best_load = INT64_MAX;
  for (int sp = 1; sp <= std::min(kSmMaxSplit, w->k_blocks); ++sp) {
    const int kb = (w->k_blocks + sp - 1) / sp;
    if ((w->k_blocks + kb - 1) / kb != sp) continue;  // an empty split
    const int64_t load = (static_cast<int64_t>(w->n_tiles) * sp + ctx->sm_count - 1) / ctx->sm_count * kb;
    if (load < best_load) {
      best_split = sp;
      best_load = load;
    }
  }
  const int kb = (w->k_blocks + best_split - 1) / best_split;
  constexpr int kSlots = !kGated ? 6 : sm_ways(kT) == 3 ? 3 : 4;
  static_assert(kSlots % sm_ways(kT) == 0, "a slot's records belong to one set of warps");
  const int best_slots = std::min(kb, kSlots);
  const size_t x_budget = kSmSmem - static_cast<size_t>(best_slots) * kSlot - 128;
  int best_phase = std::min(kb, 32);  // a bit each in the mask of wide records
  const auto staged = [&](int phase) { return static_cast<size_t>(cols) * (kParts * (phase * 512 + 64) + phase * 4); };
  while (best_phase > 1 && staged(best_phase) > x_budget) best_phase = (best_phase + 1) / 2;
  // the partial sums take the ring's place
  const size_t best_smem =
      std::max(static_cast<size_t>(best_slots) * kSlot + 128 + staged(best_phase),
               static_cast<size_t>(cols) * kRecRows * 4 * sm_ways(kT) * (kGated ? 2 : 1));
  p.kb_per_split = (w->k_blocks + best_split - 1) / best_split;
  p.kb_phase = best_phase;
  p.slots = best_slots;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(w->n_tiles, best_split, 1);
  cfg.blockDim = dim3(sm_threads(kT), 1, 1);
  cfg.dynamicSmemBytes = best_smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = best_split;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // set up behind the previous kernel
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  AEX_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, kern, p));
  return check_launch(ctx, "fp4 small_kernel");
}

template <int kFormat, bool kGated>
int pick_tiles(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  if (!j.x_f32 || j.quantize)
    return j.m <= 8 ? launch_small<kFormat, 1, kGated, 1>(ctx, j, s) : launch_small<kFormat, 2, kGated, 1>(ctx, j, s);
  // f32 rows: eight a launch, sixteen columns (32 columns leave registers for one set of warps: 51 us for 16 rows,
  // 4096 -> 18431, against 48 for two launches)
  for (int r = 0; r < j.m; r += 8) {
    Job part = j;
    part.m = std::min(8, j.m - r);
    part.x = static_cast<const float*>(j.x) + r * j.ldx;
    part.y = static_cast<uint8_t*>(j.y) + r * j.ldy * (j.y_f32 ? 4 : 2);
    if (int rc = part.m <= 4 ? launch_small<kFormat, 1, kGated, 2>(ctx, part, s)
                             : launch_small<kFormat, 2, kGated, 2>(ctx, part, s))
      return rc;
  }
  return AEX_OK;
}

}  // namespace

int run_small(aex_ctx* ctx, const Job& j, cudaStream_t s) {
  if (j.w0->format == AEX_FP4_MX)
    return j.w1 ? pick_tiles<AEX_FP4_MX, true>(ctx, j, s) : pick_tiles<AEX_FP4_MX, false>(ctx, j, s);
  return j.w1 ? pick_tiles<AEX_FP4_NV, true>(ctx, j, s) : pick_tiles<AEX_FP4_NV, false>(ctx, j, s);
}

}  // namespace fp4
}  // namespace aex
