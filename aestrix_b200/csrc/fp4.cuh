// fp4.cuh — the microscaled 4-bit form shared by the fp4 kernels: its rounding,
// its decoding and the tile layout ("records") the products read.
//
// A value is code * scale (* one f32 per tensor for nvfp4): e2m1 codes 0, 0.5,
// 1, 1.5, 2, 3, 4, 6 with a sign bit, and per block of columns one scale byte,
// mxfp4: 2^(byte - 127) for 32 columns (255: NaN); nvfp4: e4m3 for 16 columns
// (bit 7 ignored, 0x7F: NaN).
//
// Record layout. A matrix is cut into records of 128 rows x 256 columns, zero
// past its rows (weights only) and columns; record (rt, kb) of a matrix with
// k_blocks = ceil(k / 256) starts at byte (rt * k_blocks + kb) * record bytes:
//   [0, 16384)   codes, 128 bytes a row, as the tensor core's 128-byte swizzle
//                wants them: 16-byte chunk c (columns 32c..32c+31) of row r at
//                r * 128 + ((c ^ (r & 7)) << 4). Eight codes a 32-bit word, the
//                nibbles of a word permuted as in the affine layout (nibble i
//                holds column 2i for i < 4, 2(i - 4) + 1 above), so that one
//                shift and mask yields two adjacent columns in the halves of a
//                word. The permutation stays inside 8 columns, hence inside a
//                block: a product of two matrices in this layout is unchanged.
//   [16384, ..)  scale bytes in groups of 512, the order the tensor core's
//                scale operand wants: row r, scale j of the group at
//                (r % 32) * 16 + (r / 32) * 4 + j. nvfp4: one group per 64
//                columns (4 groups); mxfp4: one per 128 columns (2 groups).
// One bulk copy moves a record (both regions are contiguous), and the same
// bytes serve the block-scaled tensor-core product, the dequantizing GEMM and
// the small-row kernel.
#pragma once
#include "fp4_internal.h"
#include "sm100.cuh"

namespace aex {
namespace fp4 {

// ------------------------------------------------------------------ rounding
// e2m1 rounding of |x| / unit to nearest, ties to the even code, decided as in
// real arithmetic although the quotient is not exact in f32: every border lies
// on the bf16 grid (at most 3 significant bits), so the approximate quotient
// rounded to bf16 is the border itself whenever it is near one, and the sign
// of the fused x - border * s * tensor_scale (border * s is exact in f32: 8 + 4
// bits) says which side x is on; otherwise it lies on the same side of every
// border as the quotient. The same argument holds for the e4m3 scale (borders
// of at most 5 bits, border * 6 exact). Requires 2^-100 <= tensor_scale <=
// 2^100, so that no residual that matters underflows.
__device__ __forceinline__ float settle(float approx, float border_unit, float tensor_scale, float x) {
  const float rt = __bfloat162float(__float2bfloat16_rn(approx));
  const float e = __fmaf_rn(-(rt * border_unit), tensor_scale, x);
  const int d = (e > 0.f) - (e < 0.f);
  return __int_as_float(__float_as_int(rt) + d);
}

__device__ __forceinline__ uint32_t e4m3_sat(float v) {  // v >= 0, to nearest even, at most 448
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xFFu;
}

// e4m3 byte -> f32 (bit 7 ignored): the bits, shifted into f32 exponent and
// mantissa, are the value times 2^-120, subnormals included.
__device__ __forceinline__ float e4m3_to_f32(uint32_t b) {
  b &= 0x7Fu;
  const float v = __uint_as_float(b << 20) * 0x1p120f;
  return b == 0x7Fu ? __uint_as_float(0x7FC00000u) : v;
}

// E8M0 byte -> f32 (255: NaN; 0: 2^-127, subnormal).
__device__ __forceinline__ float e8m0_to_f32(uint32_t b) {
  return b == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(b == 255u ? 0x7FC00000u : b << 23);
}

template <int kFormat>
__device__ __forceinline__ float scale_to_f32(uint32_t b) {
  return kFormat == AEX_FP4_MX ? e8m0_to_f32(b) : e4m3_to_f32(b);
}

// Eight values as one word of codes, in the order of the columns or (kPermute) of the records.
template <bool kPermute>
__device__ __forceinline__ uint32_t code_word(const float* p) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(p[0]), "f"(p[kPermute ? 2 : 1]), "f"(p[kPermute ? 4 : 2]), "f"(p[kPermute ? 6 : 3]),
        "f"(p[kPermute ? 1 : 4]), "f"(p[kPermute ? 3 : 5]), "f"(p[kPermute ? 5 : 6]), "f"(p[7]));
  return w;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes and scale byte of kN (8 or 16) columns v of one row; the block's other
// columns are with this lane's neighbours (lane ^ 1, and for a fourth part
// lane ^ 2); all lanes of a warp call it. top: the bits of the largest |v| of
// these columns (an infinity or NaN among them: at least 0x7F800000, which makes
// the block's scale a NaN and its codes 0). inv_6ts is 1 / (6 tensor_scale)
// rounded to f32.
// mxfp4: v over a power of two is exact. nvfp4, tensor_scale a power of two: the
// unit has 4 significant bits, and a quotient that is rounded correctly (a
// reciprocal rounded to nearest, one residual) is a border only if v is. Any
// other tensor_scale: v is multiplied by the reciprocal 2^-21 above and below;
// the approximations are off by at most 1.25 * 2^-22 (2^-23 the reciprocal, 2^-24
// each the roundings of the unit, of the reciprocal moved, of the product), so
// where both give the same codes they are the quotients', and where not the
// eight values are settled exactly. (Settling every value cost 21 us for 4608 x
// 4096.)
template <int kFormat, int kN, bool kPermute>
__device__ __forceinline__ uint32_t quantize_cols(const float* v, uint32_t top, float tensor_scale, float inv_6ts,
                                                  uint32_t* codes) {
#pragma unroll
  for (int o = 1; o < block_of(kFormat) / kN; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool bad = top >= 0x7F800000u;
  const float amax = bad ? 0.f : __uint_as_float(top);
  float q[kN];
  if (kFormat == AEX_FP4_MX) {
    // floor(log2 amax) - 2, biased: the exponent field less 2 (subnormals, and what is below 2^-125, take byte 0)
    const int ex = max(static_cast<int>(__float_as_uint(amax) >> 23) - 2, 0);
    const float inv = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);  // 2^(127 - ex), ex <= 252
#pragma unroll
    for (int i = 0; i < kN; ++i) q[i] = v[i] * inv;
#pragma unroll
    for (int h = 0; h < kN / 8; ++h) codes[h] = bad ? 0u : code_word<kPermute>(q + 8 * h);
    return bad ? 0xFFu : static_cast<uint32_t>(ex);
  }
  const uint32_t sb = e4m3_sat(settle(amax * inv_6ts, 6.f, tensor_scale, amax));
  const float s = e4m3_to_f32(sb), unit = s * tensor_scale;
  if ((__float_as_uint(tensor_scale) & 0x007FFFFFu) == 0) {
    const float inv = __frcp_rn(unit);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float r = v[i] * inv;
      q[i] = fmaf(fmaf(-r, unit, v[i]), inv, r);
      if (!(fabsf(r) < 8.f)) q[i] = r;  // beyond the largest code (the residual of a huge one may be no number)
    }
#pragma unroll
    for (int h = 0; h < kN / 8; ++h) codes[h] = code_word<kPermute>(q + 8 * h);
  } else {
    const float inv = rcp_approx(unit);
    const float up = inv * (1.f + 0x1p-21f), down = inv * (1.f - 0x1p-21f);
#pragma unroll
    for (int h = 0; h < kN / 8; ++h) {
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = v[8 * h + i] * up;
        b[i] = v[8 * h + i] * down;
      }
      codes[h] = code_word<kPermute>(a);
      if (codes[h] != code_word<kPermute>(b) && sb) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = v[8 * h + i];
          a[i] = copysignf(settle(fabsf(x) * inv, s, tensor_scale, fabsf(x)), x);
        }
        codes[h] = code_word<kPermute>(a);
      }
    }
  }
  if (bad || sb == 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) q[i] = bad ? 0.f : copysignf(0.f, v[i]);
#pragma unroll
    for (int h = 0; h < kN / 8; ++h) codes[h] = code_word<kPermute>(q + 8 * h);
  }
  return bad ? 0x7Fu : sb;
}

// ------------------------------------------------------------------ decoding
// The eight codes of a word as four f16 pairs: byte b of a record word holds
// columns (0, 2), (4, 6), (1, 3), (5, 7) of its eight. (In the
// order of the columns: byte b holds columns 2b and 2b + 1.)
__device__ __forceinline__ void decode_f16(uint32_t w, uint32_t* d) {
  asm("{\n\t.reg .b8 t0, t1, t2, t3;\n\t"
      "mov.b32 {t0, t1, t2, t3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, t0;\n\tcvt.rn.f16x2.e2m1x2 %1, t1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, t2;\n\tcvt.rn.f16x2.e2m1x2 %3, t3;\n\t}"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(w));
}

// Columns (2j, 2j + 1) of a record word as a bf16 pair, times 2^-126: the three
// magnitude bits of a code, placed at the border of exponent and mantissa, are
// its value in units of 2^-126 (0.5 is a bf16 subnormal there).
__device__ __forceinline__ uint32_t code_pair_tiny(uint32_t w, int j) {
  const uint32_t mag = j == 0 ? w << 6 : j == 1 ? w << 2 : j == 2 ? w >> 2 : w >> 6;
  return (mag & 0x01C001C0u) | ((w << (12 - 4 * j)) & 0x80008000u);
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ void st_global_32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

constexpr uint32_t kBf16x2_2p126 = 0x7E807E80u;  // 2^126 in both halves

// The scale as the bf16 pair that decode_pair multiplies by. nvfp4: s * 2^119
// (at most 1.75 * 2^127), so that one multiplication takes the pair from
// 2^-126 to 2^-7 times its value, exactly (2 + 4 significant bits);
// the products undo the 2^-7. mxfp4: 2^e itself (0: subnormal; 255: NaN).
template <int kFormat>
__device__ __forceinline__ uint32_t scale_pair(uint32_t byte) {
  if (kFormat == AEX_FP4_MX) {
    const uint32_t b = byte == 0 ? 0x0040u : byte == 255u ? 0x7FC0u : byte << 7;
    return b | (b << 16);
  }
  const float s = e4m3_to_f32(byte) * 0x1p119f;
  return __byte_perm(__float_as_uint(s), 0, 0x3232);
}

// What the decoded pairs are to be multiplied by in the end.
template <int kFormat>
__host__ __device__ constexpr float decode_unit() {
  return kFormat == AEX_FP4_MX ? 1.f : 128.f;
}

// mxfp4 scales of at most 2 (byte <= 128) take the pair to its value in one
// multiplication: 2^(byte - 127 + 126) is a bf16.
__device__ __forceinline__ uint32_t mx_scale_from_tiny(uint32_t byte) { return (byte + 126u) * 0x00800080u; }

template <int kFormat>
__device__ __forceinline__ uint32_t decode_pair(uint32_t w, int j, uint32_t scale2) {
  uint32_t p = code_pair_tiny(w, j);
  if (kFormat == AEX_FP4_MX) p = mul_bf16x2(p, kBf16x2_2p126);  // the exponents of mxfp4 do not fit one step
  return mul_bf16x2(p, scale2);
}

// -------------------------------------------------------------- activation
// act(g) = g * sigmoid(z): silu z = g; gelu (tanh form) z = sqrt(8 / pi) (g + 0.044715 g^3), since
// (1 + tanh(y)) / 2 = sigmoid(2 y).
__device__ __forceinline__ float sigmoid_arg(float g, int activation) {
  constexpr float kA = 1.5957691216057308f;  // sqrt(8 / pi)
  return activation == AEX_ACT_SILU ? g : kA * fmaf(0.044715f * g * g, g, g);
}
__device__ __forceinline__ float sigmoid_arg_slope(float g, int activation) {
  constexpr float kA = 1.5957691216057308f;
  // It is multiplied by g s (1 - s), which is 0 long before |g| = 64: a square that overflowed would make that a NaN.
  const float c = fminf(fabsf(g), 64.f);
  return activation == AEX_ACT_SILU ? 1.f : kA * fmaf(3.f * 0.044715f * c, c, 1.f);
}

// kFast: to about 2^-20 of the value; 0 where z is below -87 (the quotient's divisor is above 2^126).
template <bool kFast>
__device__ __forceinline__ float sigmoid(float z) {
  return kFast ? __fdividef(1.f, 1.f + __expf(-z)) : 1.f / (1.f + expf(-z));
}

}  // namespace fp4
}  // namespace aex
