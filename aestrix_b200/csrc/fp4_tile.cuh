// fp4_tile.cuh — what the two tensor-core GEMMs with microscaled 4-bit weights
// share: the result's description and the epilogue of a tile.
#pragma once
#include "fp4.cuh"

namespace aex {
namespace fp4 {

struct TileOut {
  int m, cols;
  float alpha0, alpha1;  // what the accumulators (the gate's and the up projection's) are multiplied by
  int activation;
  void* y;
  int64_t ldy;
  int y_f32;
  int vec;  // rows of y are whole 16-byte vectors
};

// 32 columns [col, col + 32) of one row.
template <bool kF32>
__device__ __forceinline__ void store32(const TileOut& p, int64_t row, int col, const float* v) {
  if (kF32) {
    float* o = static_cast<float*>(p.y) + row * p.ldy + col;
    if (p.vec && col + 32 <= p.cols) {
#pragma unroll
      for (int i = 0; i < 32; i += 4)
        *reinterpret_cast<float4*>(o + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (col + i < p.cols) o[i] = v[i];
    }
  } else {
    uint16_t* o = static_cast<uint16_t*>(p.y) + row * p.ldy + col;
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    if (p.vec && col + 32 <= p.cols) {
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<uint4*>(o + 2 * i) = make_uint4(pk[i], pk[i + 1], pk[i + 2], pk[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (col + i < p.cols) o[i] = static_cast<uint16_t>((i & 1) ? pk[i >> 1] >> 16 : pk[i >> 1] & 0xFFFFu);
    }
  }
}

// A row's 256 accumulator columns starting at tensor-memory address tbase, as
// columns [256 nt, ..) of y, or (gated) 128 of the gate and 128 of the up
// projection as columns [128 nt, ..).
template <bool kGated>
__device__ __forceinline__ void tile_rows(const TileOut& p, int64_t row, int nt, uint32_t tbase) {
  if (!kGated) {
#pragma unroll 1
    for (int c0 = 0; c0 < 256; c0 += 32) {
      uint32_t r[32];
      tmem_ld32(tbase + c0, r);
      tmem_wait_ld();
      const int col = nt * 256 + c0;
      if (row < p.m && col < p.cols) {
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]) * p.alpha0;
        if (p.y_f32)
          store32<true>(p, row, col, v);
        else
          store32<false>(p, row, col, v);
      }
    }
  } else {
#pragma unroll 1
    for (int c0 = 0; c0 < 128; c0 += 32) {
      uint32_t gr[32], ur[32];
      tmem_ld32(tbase + c0, gr);
      tmem_ld32(tbase + 128 + c0, ur);
      tmem_wait_ld();
      const int col = nt * 128 + c0;
      if (row < p.m && col < p.cols) {
        float v[32];
        if (p.y_f32) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float g = __uint_as_float(gr[e]) * p.alpha0, u = __uint_as_float(ur[e]) * p.alpha1;
            v[e] = g * sigmoid<false>(sigmoid_arg(g, p.activation)) * u;
          }
          store32<true>(p, row, col, v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float g = __uint_as_float(gr[e]) * p.alpha0, u = __uint_as_float(ur[e]) * p.alpha1;
            v[e] = g * sigmoid<true>(sigmoid_arg(g, p.activation)) * u;
          }
          store32<false>(p, row, col, v);
        }
      }
    }
  }
}

inline int vec_ok(const void* y, int64_t ldy, bool f32) {
  return (reinterpret_cast<uintptr_t>(y) & 15) == 0 && (ldy * (f32 ? 4 : 2)) % 16 == 0;
}

}  // namespace fp4
}  // namespace aex
