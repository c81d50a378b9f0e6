// fp4_quant.cu — to the microscaled 4-bit form and back, and the weight handle
// of the fp4 products.
//
// All three kernels are streams: a thread owns 16 columns of a row, which is one
// nvfp4 block or, with its neighbouring lane, one mxfp4 block, so the block's
// largest magnitude needs no shared memory and every element is read and
// written once. 4608 x 9216 bf16 -> nvfp4 takes 21.5 us (5.1 TB/s; bound by the
// rounding's instructions, three quarters of the issue slots; two values a
// multiplication gained 0.9 us here and nothing in the products), -> mxfp4 17.1 us
// (6.3 TB/s, HBM), back from nvfp4 18.2 us (6.0 TB/s, HBM).
#include <cuda_fp16.h>

#include <algorithm>
#include <new>

#include "fp4.cuh"
#include "fp4_internal.h"

namespace aex {
namespace fp4 {

constexpr int kThreads = 256;

__device__ __forceinline__ void ldg256(const void* p, uint32_t* v) {
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p));
}

// 32 bytes, in one load where the address allows.
__device__ __forceinline__ void load32(const void* p, bool whole, uint32_t* w) {
  if (whole) {
    ldg256(p, w);
  } else {
    const uint4 a = __ldg(static_cast<const uint4*>(p)), b = __ldg(static_cast<const uint4*>(p) + 1);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  }
}

// 16 elements of a row as f32, and the bits of the largest magnitude.
template <bool kF32>
__device__ __forceinline__ uint32_t load16(const void* x, int64_t at, bool whole, float* v) {
  if (kF32) {
    uint32_t w[16], top = 0;
    const float* p = static_cast<const float*>(x) + at;
    load32(p, whole, w);
    load32(p + 8, whole, w + 8);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[i] = __uint_as_float(w[i]);
      top = max(top, w[i] & 0x7FFFFFFFu);
    }
    return top;
  }
  uint32_t w[8], top = 0;  // two 16-bit maxima at a time: bits without the sign are ordered as magnitudes
  load32(static_cast<const uint16_t*>(x) + at, whole, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
    v[2 * i] = bf16lo_to_f32(w[i]);
    v[2 * i + 1] = bf16hi_to_f32(w[i]);
  }
  return max(top << 16, top & 0xFFFF0000u);
}

__device__ __forceinline__ uint32_t divide(uint32_t u, const FastDiv& f) {
  return f.div == 1 ? u : __umulhi(u, f.mul) >> f.shift;
}

// x [rows, k] -> codes [rows, k/2] and scales [rows, k/block] (kRecords: the
// record layout in `codes`, columns padded with zeros to whole records; rows
// past the last are left as they are; x starts at row `first` of the first
// records). `upr` units of 16 columns a row (even); rows * upr < 2^31
// (slice_rows).
template <int kFormat, bool kF32, bool kRecords>
__global__ void __launch_bounds__(kThreads, 8) quantize_kernel(const void* __restrict__ x, int64_t ldx, int rows, int k,
                                                            uint32_t first, FastDiv upr, int whole,
                                                            float tensor_scale, float inv_6ts,
                                                            uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales) {
  if (kRecords) launch_dependents();  // the product that reads the records waits for them itself
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t row = divide(u, upr), c = u - row * upr.div;  // an mxfp4 pair (u even, u + 1) is one row's
  const bool live = row < static_cast<uint32_t>(rows);
  const int col = static_cast<int>(c) * 16;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  uint32_t top = 0;
  if (live && col < k) top = load16<kF32>(x, static_cast<int64_t>(row) * ldx + col, whole != 0, v);
  uint32_t w[2];
  const uint32_t sb = quantize_cols<kFormat, 16, kRecords>(v, top, tensor_scale, inv_6ts, w);
  if (!live) return;
  if (kRecords) {
    const uint32_t at = first + row;
    const int r = static_cast<int>(at % kRecRows);
    uint8_t* rec = codes + (static_cast<size_t>(at / kRecRows) * (upr.div / 16) + c / 16) * rec_bytes(kFormat);
    const int cu = static_cast<int>(c % 16);  // unit inside the record
    *reinterpret_cast<uint2*>(rec + r * 128 + (((cu >> 1) ^ (r & 7)) << 4) + (cu & 1) * 8) = make_uint2(w[0], w[1]);
    if (kFormat == AEX_FP4_NV)
      rec[scale_off(r, cu >> 2) + (cu & 3)] = static_cast<uint8_t>(sb);
    else if (!(cu & 1))
      rec[scale_off(r, cu >> 3) + ((cu >> 1) & 3)] = static_cast<uint8_t>(sb);
  } else {
    reinterpret_cast<uint2*>(codes)[u] = make_uint2(w[0], w[1]);
    if (kFormat == AEX_FP4_NV)
      scales[u] = static_cast<uint8_t>(sb);
    else if (!(u & 1))
      scales[u >> 1] = static_cast<uint8_t>(sb);
  }
}

__device__ __forceinline__ uint32_t nibble_compress(uint32_t x) {  // 4 bytes < 16 -> 4 nibbles
  x = (x | (x >> 4)) & 0x00FF00FFu;
  return (x | (x >> 8)) & 0x0000FFFFu;
}
__device__ __forceinline__ uint32_t permute_word(uint32_t w) {
  return nibble_compress(w & 0x0F0F0F0Fu) | (nibble_compress((w >> 4) & 0x0F0F0F0Fu) << 16);
}
__device__ __forceinline__ uint32_t nibble_spread(uint32_t x) {  // 4 nibbles -> the low nibbles of 4 bytes
  x = (x | (x << 8)) & 0x00FF00FFu;
  return (x | (x << 4)) & 0x0F0F0F0Fu;
}
__device__ __forceinline__ uint32_t restore_word(uint32_t w) {  // inverse of permute_word
  return nibble_spread(w & 0xFFFFu) | (nibble_spread(w >> 16) << 4);
}

// x rounded so that one more rounding, to bf16, is that of the exact product
// c * tensor_scale: to odd, which keeps the side of every bf16 tie.
__device__ __forceinline__ float product_to_odd(float c, float tensor_scale) {
  const float p = __fmul_rz(c, tensor_scale);
  return __fmaf_rn(c, tensor_scale, -p) != 0.f ? __uint_as_float(__float_as_uint(p) | 1u) : p;
}

// Four bytes of a and b by the nibbles of sel's low half (__byte_perm without its masking of bit 3).
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}

// The values of 16 codes as bf16 pairs in the order of the columns. A block has
// eight magnitudes: s and 1.5 s times the tensor scale, each rounded once, and
// powers of two of them (exact: tensor scales and block scales leave room). The
// codes select their bytes (a third of the instructions of a product and a
// rounding for each).
__device__ __forceinline__ void bf16_by_table(uint2 codes, float s, float tensor_scale, uint32_t* o) {
  const float a = __bfloat162float(__float2bfloat16_rn(product_to_odd(s, tensor_scale)));
  const float b = __bfloat162float(__float2bfloat16_rn(product_to_odd(1.5f * s, tensor_scale)));
  const float m[8] = {a * 0.f, a * 0.5f, a, b, a * 2.f, b * 2.f, a * 4.f, b * 4.f};
  uint32_t lo[2], hi[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t p = __byte_perm(__float_as_uint(m[4 * h]), __float_as_uint(m[4 * h + 1]), 0x7362);
    const uint32_t q = __byte_perm(__float_as_uint(m[4 * h + 2]), __float_as_uint(m[4 * h + 3]), 0x7362);
    lo[h] = __byte_perm(p, q, 0x5410);
    hi[h] = __byte_perm(p, q, 0x7632);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t w = (q & 2 ? codes.y : codes.x) >> (16 * (q & 1)), idx = w & 0x7777u;
    // a selector with bit 3 set repeats the sign of the selected byte: 0xFF for a negative code, 0x80 for others
    const uint32_t sign = prmt(0x80808080u, 0x80808080u, w) << 1;
    const uint32_t l4 = prmt(lo[0], lo[1], idx);
    const uint32_t h4 = prmt(hi[0], hi[1], idx) | (sign & 0x80808080u);
    o[2 * q] = __byte_perm(l4, h4, 0x5140);
    o[2 * q + 1] = __byte_perm(l4, h4, 0x7362);
  }
}

// Codes -> values, out [rows, k] (row pitch ldo). kRecords: from the record
// layout, from row `first` of the first records on. One thread per 16 columns.
template <int kFormat, bool kF32, bool kRecords>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales, int rows,
                                                              uint32_t first, FastDiv upr, int k_blocks,
                                                              float tensor_scale, void* __restrict__ out,
                                                              int64_t ldo, int whole) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t row = divide(u, upr), c = u - row * upr.div;
  if (row >= static_cast<uint32_t>(rows)) return;
  uint2 w;
  uint32_t sb;
  if (kRecords) {
    const uint32_t in = first + row;
    const int r = static_cast<int>(in % kRecRows), cu = static_cast<int>(c % 16);
    const uint8_t* rec = codes + (static_cast<size_t>(in / kRecRows) * k_blocks + c / 16) * rec_bytes(kFormat);
    w = *reinterpret_cast<const uint2*>(rec + r * 128 + (((cu >> 1) ^ (r & 7)) << 4) + (cu & 1) * 8);
    sb = kFormat == AEX_FP4_NV ? rec[scale_off(r, cu >> 2) + (cu & 3)] : rec[scale_off(r, cu >> 3) + ((cu >> 1) & 3)];
  } else {
    w = __ldg(reinterpret_cast<const uint2*>(codes) + u);
    sb = __ldg(scales + (kFormat == AEX_FP4_NV ? u : u >> 1));
  }
  const float s = scale_to_f32<kFormat>(sb);
  if (kRecords) w = make_uint2(restore_word(w.x), restore_word(w.y));
  const int64_t at = static_cast<int64_t>(row) * ldo + static_cast<int64_t>(c) * 16;
  uint32_t o[16];
  if (kF32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t d[4];
      decode_f16(h ? w.y : w.x, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t half = i & 1 ? d[i >> 1] >> 16 : d[i >> 1] & 0xFFFFu;
        // code * scale is exact (2 + 4 bits), so this is one rounding
        o[8 * h + i] =
            __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(half))) * s * tensor_scale);
      }
    }
  } else {
    bf16_by_table(w, s, tensor_scale, o);
  }
  uint8_t* dst = static_cast<uint8_t*>(out) + at * (kF32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < (kF32 ? 16 : 8); i += 8) {
    if (whole) {
      st_global_32(dst + 4 * i, o + i);
    } else {
      *reinterpret_cast<uint4*>(dst + 4 * i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      *reinterpret_cast<uint4*>(dst + 4 * i + 16) = make_uint4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
    }
  }
}

// Rows as stored (codes, scales) -> records, zero past n and k. One CTA per
// record, a thread per 16 columns at a time.
template <int kFormat>
__global__ void __launch_bounds__(kThreads) records_kernel(const uint8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales, int n, int k,
                                                           int k_blocks, uint8_t* __restrict__ records) {
  const int rt = static_cast<int>(blockIdx.x / k_blocks), kb = static_cast<int>(blockIdx.x % k_blocks);
  uint8_t* rec = records + static_cast<size_t>(blockIdx.x) * rec_bytes(kFormat);
  constexpr int kBlock = block_of(kFormat);
  for (int i = threadIdx.x; i < kRecRows * 16; i += kThreads) {
    const int r = i >> 4, cu = i & 15;
    const int64_t row = static_cast<int64_t>(rt) * kRecRows + r;
    const int col = kb * kRecK + cu * 16;
    uint2 w = make_uint2(0, 0);
    uint32_t sb = 0;
    if (row < n && col < k) {
      w = __ldg(reinterpret_cast<const uint2*>(codes + row * (k / 2) + col / 2));
      sb = scales[row * (k / kBlock) + col / kBlock];
      if (kFormat == AEX_FP4_NV) sb &= 0x7Fu;
    }
    *reinterpret_cast<uint2*>(rec + r * 128 + (((cu >> 1) ^ (r & 7)) << 4) + (cu & 1) * 8) =
        make_uint2(permute_word(w.x), permute_word(w.y));
    if (kFormat == AEX_FP4_NV)
      rec[scale_off(r, cu >> 2) + (cu & 3)] = static_cast<uint8_t>(sb);
    else if (!(cu & 1))
      rec[scale_off(r, cu >> 3) + ((cu >> 1) & 3)] = static_cast<uint8_t>(sb);
  }
}

namespace {

template <int kFormat, bool kF32, bool kRecords>
int launch_quantize(aex_ctx* ctx, const void* x, int64_t ldx, int rows, int k, float ts, uint8_t* codes,
                    uint8_t* scales, cudaStream_t s) {
  const uint32_t upr = kRecords ? static_cast<uint32_t>(records_along(k)) * 16 : static_cast<uint32_t>(k / 16);
  const int64_t step = slice_rows(upr);
  const float inv = static_cast<float>(1.0 / (6.0 * static_cast<double>(ts)));
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    const int nr = static_cast<int>(std::min<int64_t>(step, rows - r0));
    const uint32_t blocks = static_cast<uint32_t>((static_cast<int64_t>(nr) * upr + kThreads - 1) / kThreads);
    const uint8_t* xs = static_cast<const uint8_t*>(x) + r0 * ldx * (kF32 ? 4 : 2);
    uint8_t* cs = kRecords ? codes + static_cast<size_t>(r0 / kRecRows) * (upr / 16) * rec_bytes(kFormat)
                           : codes + static_cast<size_t>(r0) * upr * 8;
    uint8_t* ss = kRecords ? nullptr : scales + static_cast<size_t>(r0) * (k / block_of(kFormat));
    const int whole = (reinterpret_cast<uintptr_t>(xs) | static_cast<uint64_t>(ldx * (kF32 ? 4 : 2))) % 32 == 0;
    const auto first = static_cast<uint32_t>(r0 % kRecRows);
    quantize_kernel<kFormat, kF32, kRecords>
        <<<blocks, kThreads, 0, s>>>(xs, ldx, nr, k, first, fast_div(upr), whole, ts, inv, cs, ss);
    if (int r = check_launch(ctx, "fp4 quantize_kernel")) return r;
  }
  return AEX_OK;
}

template <int kFormat, bool kF32, bool kRecords>
int launch_dequantize(aex_ctx* ctx, const uint8_t* codes, const uint8_t* scales, int rows, int k, float ts, void* out,
                      int64_t ldo, cudaStream_t s) {
  const uint32_t upr = static_cast<uint32_t>(k / 16);
  const int k_blocks = records_along(k);
  const int64_t step = slice_rows(upr);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    const int nr = static_cast<int>(std::min<int64_t>(step, rows - r0));
    const uint32_t blocks = static_cast<uint32_t>((static_cast<int64_t>(nr) * upr + kThreads - 1) / kThreads);
    const uint8_t* cs = kRecords ? codes + static_cast<size_t>(r0 / kRecRows) * k_blocks * rec_bytes(kFormat)
                                 : codes + static_cast<size_t>(r0) * upr * 8;
    const uint8_t* ss = kRecords ? nullptr : scales + static_cast<size_t>(r0) * (k / block_of(kFormat));
    uint8_t* os = static_cast<uint8_t*>(out) + r0 * ldo * (kF32 ? 4 : 2);
    const int whole = (reinterpret_cast<uintptr_t>(os) | static_cast<uint64_t>(ldo * (kF32 ? 4 : 2))) % 32 == 0;
    const auto first = static_cast<uint32_t>(r0 % kRecRows);
    dequantize_kernel<kFormat, kF32, kRecords>
        <<<blocks, kThreads, 0, s>>>(cs, ss, nr, first, fast_div(upr), k_blocks, ts, os, ldo, whole);
    if (int r = check_launch(ctx, "fp4 dequantize_kernel")) return r;
  }
  return AEX_OK;
}

template <bool kRecords>
int dispatch_dequantize(aex_ctx* ctx, const uint8_t* codes, const uint8_t* scales, int rows, int k, int format,
                        float ts, void* out, int out_dtype, int64_t ldo, cudaStream_t s) {
  const bool f32 = out_dtype == AEX_DTYPE_F32;
  if (format == AEX_FP4_MX)
    return f32 ? launch_dequantize<AEX_FP4_MX, true, kRecords>(ctx, codes, scales, rows, k, ts, out, ldo, s)
               : launch_dequantize<AEX_FP4_MX, false, kRecords>(ctx, codes, scales, rows, k, ts, out, ldo, s);
  return f32 ? launch_dequantize<AEX_FP4_NV, true, kRecords>(ctx, codes, scales, rows, k, ts, out, ldo, s)
             : launch_dequantize<AEX_FP4_NV, false, kRecords>(ctx, codes, scales, rows, k, ts, out, ldo, s);
}

}  // namespace

int check_format(aex_ctx* ctx, int format, float tensor_scale) {
  if (format != AEX_FP4_MX && format != AEX_FP4_NV)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "format must be AEX_FP4_MX or AEX_FP4_NV");
  if (format == AEX_FP4_MX && tensor_scale != 1.f)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "mxfp4 has no tensor scale: it must be 1");
  if (!(tensor_scale >= 0x1p-100f && tensor_scale <= 0x1p100f))
    return set_error(ctx, AEX_ERR_INVALID_ARG, "tensor_scale must lie in [2^-100, 2^100]");
  return AEX_OK;
}

int check_matrix(aex_ctx* ctx, const char* name, const void* p, int dtype, int64_t ld, int rows, int cols) {
  if (!p) return set_error(ctx, AEX_ERR_INVALID_ARG, "%s is NULL", name);
  if (dtype != AEX_DTYPE_BF16 && dtype != AEX_DTYPE_F32)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "%s: dtype must be AEX_DTYPE_BF16 or AEX_DTYPE_F32", name);
  if (rows <= 0) return set_error(ctx, AEX_ERR_INVALID_ARG, "%s: the number of rows must be positive", name);
  if ((reinterpret_cast<uintptr_t>(p) & 15) || ld < cols || ld % (dtype == AEX_DTYPE_F32 ? 4 : 8))
    return set_error(ctx, AEX_ERR_INVALID_ARG,
                     "%s must be 16-byte aligned, its row pitch at least %d elements and a multiple of 16 bytes", name,
                     cols);
  return AEX_OK;
}

int quantize_records(aex_ctx* ctx, const void* x, bool f32, int64_t ldx, int m, int k, int format, float ts,
                     uint8_t* records, cudaStream_t s) {
  if (format == AEX_FP4_MX)
    return f32 ? launch_quantize<AEX_FP4_MX, true, true>(ctx, x, ldx, m, k, ts, records, nullptr, s)
               : launch_quantize<AEX_FP4_MX, false, true>(ctx, x, ldx, m, k, ts, records, nullptr, s);
  return f32 ? launch_quantize<AEX_FP4_NV, true, true>(ctx, x, ldx, m, k, ts, records, nullptr, s)
             : launch_quantize<AEX_FP4_NV, false, true>(ctx, x, ldx, m, k, ts, records, nullptr, s);
}

}  // namespace fp4
}  // namespace aex

extern "C" {

int aex_fp4_quantize(aex_ctx* ctx, const void* x, int x_dtype, int64_t ldx, int rows, int k, int format,
                     float tensor_scale, uint8_t* codes, uint8_t* scales, aex_stream stream) {
  using namespace aex;
  if (!ctx) return set_error(ctx, AEX_ERR_INVALID_ARG, "NULL ctx");
  if (int r = fp4::check_format(ctx, format, tensor_scale)) return r;
  if (k <= 0 || k % 32) return set_error(ctx, AEX_ERR_INVALID_ARG, "k must be a positive multiple of 32 (k=%d)", k);
  if (int r = fp4::check_matrix(ctx, "x", x, x_dtype, ldx, rows, k)) return r;
  if (!codes || !scales || (reinterpret_cast<uintptr_t>(codes) & 15))
    return set_error(ctx, AEX_ERR_INVALID_ARG, "codes (16-byte aligned) and scales must not be NULL");
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  auto s = static_cast<cudaStream_t>(stream);
  const bool f32 = x_dtype == AEX_DTYPE_F32;
  if (format == AEX_FP4_MX)
    return f32 ? fp4::launch_quantize<AEX_FP4_MX, true, false>(ctx, x, ldx, rows, k, tensor_scale, codes, scales, s)
               : fp4::launch_quantize<AEX_FP4_MX, false, false>(ctx, x, ldx, rows, k, tensor_scale, codes, scales, s);
  return f32 ? fp4::launch_quantize<AEX_FP4_NV, true, false>(ctx, x, ldx, rows, k, tensor_scale, codes, scales, s)
             : fp4::launch_quantize<AEX_FP4_NV, false, false>(ctx, x, ldx, rows, k, tensor_scale, codes, scales, s);
}

int aex_fp4_dequantize(aex_ctx* ctx, const uint8_t* codes, const uint8_t* scales, int rows, int k, int format,
                       float tensor_scale, void* out, int out_dtype, int64_t ldo, aex_stream stream) {
  using namespace aex;
  if (!ctx) return set_error(ctx, AEX_ERR_INVALID_ARG, "NULL ctx");
  if (int r = fp4::check_format(ctx, format, tensor_scale)) return r;
  if (k <= 0 || k % 32) return set_error(ctx, AEX_ERR_INVALID_ARG, "k must be a positive multiple of 32 (k=%d)", k);
  if (!codes || !scales || (reinterpret_cast<uintptr_t>(codes) & 15))
    return set_error(ctx, AEX_ERR_INVALID_ARG, "codes (16-byte aligned) and scales must not be NULL");
  if (int r = fp4::check_matrix(ctx, "out", out, out_dtype, ldo, rows, k)) return r;
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  return fp4::dispatch_dequantize<false>(ctx, codes, scales, rows, k, format, tensor_scale, out, out_dtype, ldo,
                                         static_cast<cudaStream_t>(stream));
}

int aex_fp4weight_create(aex_ctx* ctx, const uint8_t* codes, const uint8_t* scales, int n, int k, int format,
                         float tensor_scale, aex_fp4weight** out, aex_stream stream) {
  using namespace aex;
  if (!ctx || !out) return set_error(ctx, AEX_ERR_INVALID_ARG, "NULL ctx/out");
  *out = nullptr;
  if (int r = fp4::check_format(ctx, format, tensor_scale)) return r;
  if (n <= 0 || k <= 0 || k % 32)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "n must be positive and k a positive multiple of 32 (n=%d k=%d)", n, k);
  if (!codes || !scales || (reinterpret_cast<uintptr_t>(codes) & 15))
    return set_error(ctx, AEX_ERR_INVALID_ARG, "codes (16-byte aligned) and scales must not be NULL");
  const int64_t n_tiles = (static_cast<int64_t>(n) + fp4::kRecRows - 1) / fp4::kRecRows;
  const int64_t k_blocks = fp4::records_along(k);
  if (n_tiles * k_blocks > 0x7FFFFFFF)
    return set_error(ctx, AEX_ERR_UNSUPPORTED, "fp4 weight of %d x %d is too large", n, k);
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  AEX_CUDA_TRY(ctx, cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture));
  if (capture != cudaStreamCaptureStatusNone)  // a graph would lay the weight out at its replays only
    return set_error(ctx, AEX_ERR_UNSUPPORTED, "a weight cannot be created on a stream that is being captured");
  int clusters = 0;
  if (int r = fp4::gemm_clusters(ctx, &clusters)) return r;
  auto* w = new (std::nothrow) aex_fp4weight();
  if (!w) return set_error(ctx, AEX_ERR_OOM, "host allocation failed");
  w->device = ctx->device;
  w->n = n;
  w->k = k;
  w->format = format;
  w->tensor_scale = tensor_scale;
  w->n_tiles = static_cast<int>(n_tiles);
  w->clusters = clusters;
  w->k_blocks = static_cast<int>(k_blocks);
  w->bytes = static_cast<size_t>(n_tiles * k_blocks) * fp4::rec_bytes(format);
  cudaError_t e = cudaMalloc(&w->records, w->bytes);
  if (e != cudaSuccess) {
    delete w;
    return cuda_error(ctx, e, "cudaMalloc(fp4 records)");
  }
  const auto blocks = static_cast<unsigned>(n_tiles * k_blocks);
  auto s = static_cast<cudaStream_t>(stream);
  if (format == AEX_FP4_MX)
    fp4::records_kernel<AEX_FP4_MX><<<blocks, fp4::kThreads, 0, s>>>(codes, scales, n, k, w->k_blocks, w->records);
  else
    fp4::records_kernel<AEX_FP4_NV><<<blocks, fp4::kThreads, 0, s>>>(codes, scales, n, k, w->k_blocks, w->records);
  if (int r = check_launch(ctx, "fp4 records_kernel")) {
    cudaFree(w->records);
    delete w;
    return r;
  }
  *out = w;
  return AEX_OK;
}

void aex_fp4weight_destroy(aex_fp4weight* w) {
  if (!w) return;
  int cur = -1;
  cudaGetDevice(&cur);
  cudaSetDevice(w->device);
  cudaDeviceSynchronize();
  cudaFree(w->records);
  if (cur >= 0) cudaSetDevice(cur);
  delete w;
}

int aex_fp4weight_shape(const aex_fp4weight* w, int* n, int* k) {
  if (!w || !n || !k) return AEX_ERR_INVALID_ARG;
  *n = w->n;
  *k = w->k;
  return AEX_OK;
}

int aex_fp4weight_dequantize(aex_ctx* ctx, const aex_fp4weight* w, void* out, int out_dtype, int64_t ldo,
                             aex_stream stream) {
  using namespace aex;
  if (!ctx || !w) return set_error(ctx, AEX_ERR_INVALID_ARG, "NULL argument");
  if (ctx->device != w->device) return set_error(ctx, AEX_ERR_INVALID_ARG, "weight lives on another device");
  if (int r = fp4::check_matrix(ctx, "out", out, out_dtype, ldo, w->n, w->k)) return r;
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  return fp4::dispatch_dequantize<true>(ctx, w->records, nullptr, w->n, w->k, w->format, w->tensor_scale, out,
                                        out_dtype, ldo, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
