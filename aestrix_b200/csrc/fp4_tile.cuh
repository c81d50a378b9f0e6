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
  int vec;  // vec_ok
};

// One cluster's share of an output tile: records [r0, r1) along K of tile
// (mt, nt); slot >= 0: a piece of a split tile, -1: the whole of it.
struct TilePiece {
  int mt, nt, r0, r1, slot;
};

// The output tiles and who computes them. Tiles are numbered with the rows'
// tiles fastest. The first `whole` go to the clusters in turn, one cluster
// each; the records of the `split` others are dealt out evenly, in order, over
// the first `parts` clusters (at least one record each), so that a cluster gets
// at most the end of one tile and the start of the next. The piece of split
// tile r that cluster c computes has slot c + r (from one piece to the next,
// either c or r goes up by one).
struct TileWork {
  int m_tiles, whole, split, parts, recs;
  int rows;  // rows of a slot (stored in bands of 32)
  float* pieces;

  // First record of cluster c's share; split * recs * (parts + 1) < 2^31 (plan_tiles), since 64-bit divisions at the
  // start of every role cost over a microsecond.
  __device__ int start(int c) const { return split * recs * c / parts; }
  // The i-th piece of cluster c; false past the last.
  __device__ bool piece(int c, int clusters, int i, TilePiece* t) const {
    int n = 0;
    t->r0 = 0;
    t->r1 = recs;
    t->slot = -1;
    if (c < parts) {
      const int u0 = start(c), u1 = start(c + 1);
      const int first = u0 / recs, last = (u1 - 1) / recs;
      n = last - first + 1;
      if (i < n) {
        const int r = first + i;
        if (i == 0) t->r0 = u0 - r * recs;
        if (r == last) t->r1 = u1 - r * recs;
        t->slot = c + r;
        t->mt = (whole + r) % m_tiles;
        t->nt = (whole + r) / m_tiles;
        return true;
      }
    }
    const int at = c + (i - n) * clusters;
    if (at >= whole) return false;
    t->mt = at % m_tiles;
    t->nt = at / m_tiles;
    return true;
  }
};

// kN pairs of bf16 to an address of which only the type's alignment is known. A
// store takes a request of its own whatever its size, so sixteen values are
// turned to the 16-byte vector that lies whole within them and what is left
// before and behind: 356 x 288 -> 599 12.5 us, in words 17.7, one by one 41.8;
// 3412 x 1344 -> 225 gated 18.9, 21.0 and 32. (Through shared memory, 32 rows at
// a time: 13.3, but the warp barriers that takes in the epilogue cost the
// block-scaled GEMM's aligned rows 40 of 130 us.)
template <int kN>
__device__ __forceinline__ void store_words(uint16_t* y, const uint32_t* pk) {
  const bool odd = reinterpret_cast<uintptr_t>(y) & 2;
  uint32_t* w = reinterpret_cast<uint32_t*>(y - (odd ? 1 : 0));
  if (kN != 8) {
    if (odd)
      y[0] = static_cast<uint16_t>(pk[0] & 0xFFFFu);
    else
      w[0] = pk[0];
#pragma unroll
    for (int e = 1; e < kN; ++e) w[e] = odd ? pk[e - 1] >> 16 | pk[e] << 16 : pk[e];
    if (odd) y[2 * kN - 1] = static_cast<uint16_t>(pk[kN - 1] >> 16);
    return;
  }
  // r[q ..): the words from w on, w being word q of its vector; the first and the last are halves where y is odd
  const uint32_t q = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(w) >> 2) & 3;
  uint32_t r[12];
#pragma unroll
  for (int e = 0; e < 9; ++e) {
    const uint32_t lo = e ? pk[e - 1] : 0u, hi = e < 8 ? pk[e] : 0u;
    r[e] = odd ? __funnelshift_r(lo, hi, 16) : hi;
  }
  r[9] = r[10] = r[11] = 0;
#pragma unroll
  for (int e = 9; e > 0; --e) r[e] = q & 1 ? r[e - 1] : r[e];
#pragma unroll
  for (int e = 11; e > 1; --e) r[e] = q & 2 ? r[e - 2] : r[e];
  uint32_t* v = w - q;
  const uint32_t first = q + (odd ? 1 : 0);  // the first whole word
  if (first == 0) {
    *reinterpret_cast<uint4*>(v) = make_uint4(r[0], r[1], r[2], r[3]);
  } else {
    if (first == 1) v[1] = r[1];
    if (first <= 2) *reinterpret_cast<uint2*>(v + 2) = make_uint2(r[2], r[3]);
    if (first == 3) v[3] = r[3];
  }
  *reinterpret_cast<uint4*>(v + 4) = make_uint4(r[4], r[5], r[6], r[7]);
  if (q >= 2) *reinterpret_cast<uint2*>(v + 8) = make_uint2(r[8], r[9]);
  if (q == 1) v[8] = r[8];
  if (q == 3) v[10] = r[10];
  if (odd) {
    y[0] = static_cast<uint16_t>(pk[0] & 0xFFFFu);
    y[15] = static_cast<uint16_t>(pk[7] >> 16);
  }
}

// kN (8 or 16) columns [c, c + kN) of a tile's row from their f32 sums (gated:
// v of the gate, u of the up projection), columns 256 nt + c (gated: 128 nt + c)
// of y. Each lane writes a row of its own: whole 32-byte sectors where y allows.
template <bool kGated, int kN>
__device__ __forceinline__ void finish(const TileOut& p, int64_t row, int nt, int c, const float* v, const float* u) {
  const int col = nt * (kGated ? 128 : 256) + c;
  const int have = columns_within(col, kN, p.cols);
  if (have <= 0) return;
  const bool all = have == kN;
  float o[kN];
  if (!kGated) {
#pragma unroll
    for (int e = 0; e < kN; ++e) o[e] = v[e] * p.alpha0;
  } else if (p.y_f32) {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float g = v[e] * p.alpha0;
      o[e] = g * sigmoid<false>(sigmoid_arg(g, p.activation)) * (u[e] * p.alpha1);
    }
  } else if (p.activation == AEX_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float g = v[e] * p.alpha0;
      o[e] = g * sigmoid<true>(g) * (u[e] * p.alpha1);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float g = v[e] * p.alpha0;
      o[e] = g * sigmoid<true>(sigmoid_arg(g, AEX_ACT_GELU_TANH)) * (u[e] * p.alpha1);
    }
  }
  if (p.y_f32) {
    float* y = static_cast<float*>(p.y) + row * p.ldy + col;
    if (p.vec && all) {
#pragma unroll
      for (int e = 0; e < kN; e += 4) *reinterpret_cast<float4*>(y + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (e < have) y[e] = o[e];
    }
  } else {
    uint16_t* y = static_cast<uint16_t*>(p.y) + row * p.ldy + col;
    uint32_t pk[kN / 2];
#pragma unroll
    for (int e = 0; e < kN / 2; ++e) pk[e] = pack_bf16x2(o[2 * e], o[2 * e + 1]);
    if (kN == 16 && p.vec == 2 && all) {
      st_global_32(y, pk);
    } else if (p.vec && all) {
#pragma unroll
      for (int e = 0; e < kN / 2; e += 4)
        *reinterpret_cast<uint4*>(y + 2 * e) = make_uint4(pk[e], pk[e + 1], pk[e + 2], pk[e + 3]);
    } else if (all) {
      store_words<kN / 2>(y, pk);
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (e < have) y[e] = static_cast<uint16_t>((e & 1) ? pk[e >> 1] >> 16 : pk[e >> 1] & 0xFFFFu);
    }
  }
}

// Reads kN accumulator columns (16 at a time) from tensor memory.
template <int kN>
__device__ __forceinline__ void tmem_read(uint32_t taddr, float* v) {
  uint32_t r[kN];
#pragma unroll
  for (int e = 0; e < kN; e += 16) tmem_ld16(taddr + e, r + e);
  tmem_wait_ld();
#pragma unroll
  for (int e = 0; e < kN; ++e) v[e] = __uint_as_float(r[e]);
}

// Half of a row's 256 accumulator columns starting at tensor-memory address
// tbase: columns [128 half, ..) or (gated) outputs [64 half, ..).
template <bool kGated>
__device__ __forceinline__ void tile_half(const TileOut& p, int64_t row, int nt, int half, uint32_t tbase) {
  if (!kGated) {
#pragma unroll 1
    for (int c = 128 * half; c < 128 * half + 128; c += 32) {
      float v[32];
      tmem_read<32>(tbase + c, v);
      if (row < p.m) {
        finish<false, 16>(p, row, nt, c, v, nullptr);
        finish<false, 16>(p, row, nt, c + 16, v + 16, nullptr);
      }
    }
  } else {
#pragma unroll 1
    for (int c = 64 * half; c < 64 * half + 64; c += 16) {
      uint32_t g[16], u[16];
      tmem_ld16(tbase + c, g);
      tmem_ld16(tbase + 128 + c, u);
      tmem_wait_ld();
      if (row < p.m) finish<true, 16>(p, row, nt, c, reinterpret_cast<float*>(g), reinterpret_cast<float*>(u));
    }
  }
}

// ------------------------------------------------------------- split tiles
// A slot holds a piece's raw accumulators as [32 rows' band][8 columns'
// group][row][8 columns]: a warp's rows of a group are one kilobyte, written
// and read 32 bytes a lane.
__device__ __forceinline__ float* piece_at(const TileWork& w, int slot, int in_tile, int group) {
  const int bands = (w.rows + 31) >> 5;
  return w.pieces + ((((static_cast<size_t>(slot) * bands + (in_tile >> 5)) * 32 + group) * 32) + (in_tile & 31)) * 8;
}

// Columns [c, c + 16) of a row.
__device__ __forceinline__ void store_piece16(const TileWork& w, int slot, int in_tile, int c, const float* v) {
  st_global_32(piece_at(w, slot, in_tile, c >> 3), reinterpret_cast<const uint32_t*>(v));
  st_global_32(piece_at(w, slot, in_tile, (c >> 3) + 1), reinterpret_cast<const uint32_t*>(v + 8));
}

// Half of a piece's row.
__device__ __forceinline__ void store_piece(const TileWork& w, int slot, int in_tile, bool live, int half,
                                            uint32_t tbase) {
#pragma unroll 1
  for (int c = 128 * half; c < 128 * half + 128; c += 16) {
    float v[16];
    tmem_read<16>(tbase + c, v);
    if (live) store_piece16(w, slot, in_tile, c, v);
  }
}

// Adds the pieces of the split tiles in the order of the clusters that wrote
// them and hands eight columns of a row at a time to `emit(row, nt, c, v, u)`
// (gated: v of columns [c, c + 8), u of [128 + c, ..)). One thread each, a warp
// for 32 rows, four pieces in flight.
constexpr int kJoinThreads = 256;
inline int join_blocks(const TileWork& w, bool gated) {
  return (w.split * ((w.rows + 31) / 32) * (gated ? 16 : 32) + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
}

template <bool kGated, typename F>
__device__ __forceinline__ void join_tile(const TileWork& w, int m, F emit) {
  constexpr int kGroups = kGated ? 16 : 32, kSums = kGated ? 2 : 1, kAhead = 4;
  launch_dependents();
  const int wid = static_cast<int>(blockIdx.x) * (kJoinThreads / 32) + (threadIdx.x >> 5);
  const int bands = (w.rows + 31) / 32;
  const int group = wid % kGroups, band = wid / kGroups % bands, r = wid / (kGroups * bands);
  if (r >= w.split) return;
  const int t = w.whole + r;
  const int in_tile = band * 32 + (threadIdx.x & 31);
  const int64_t row = static_cast<int64_t>(t % w.m_tiles) * 256 + in_tile;
  if (in_tile >= w.rows || row >= m) return;
  // Clusters c with records of tile r: start(c + 1) > r * recs and start(c) < (r + 1) * recs.
  const int total = w.split * w.recs;
  int c = ((r * w.recs + 1) * w.parts + total - 1) / total - 1;
  const int end = ((r + 1) * w.parts + w.split - 1) / w.split;
  wait_dependency();  // the pieces are written
  float v[kSums][8];
#pragma unroll
  for (int q = 0; q < kSums; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[q][e] = 0.f;
  for (; c < end; c += kAhead) {
    float4 x[kAhead][kSums][2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int q = 0; q < kSums; ++q) {
        x[i][q][0] = x[i][q][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c + i < end) {
          const float4* src = reinterpret_cast<const float4*>(piece_at(w, c + i + r, in_tile, group + 16 * q));
          x[i][q][0] = src[0];
          x[i][q][1] = src[1];
        }
      }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int q = 0; q < kSums; ++q) {
        v[q][0] += x[i][q][0].x, v[q][1] += x[i][q][0].y, v[q][2] += x[i][q][0].z, v[q][3] += x[i][q][0].w;
        v[q][4] += x[i][q][1].x, v[q][5] += x[i][q][1].y, v[q][6] += x[i][q][1].z, v[q][7] += x[i][q][1].w;
      }
  }
  emit(row, t / w.m_tiles, group * 8, v[0], v[kSums - 1]);
}

inline TileWork tile_work(const TilePlan& plan, void* pieces) {
  return TileWork{plan.m_tiles, plan.whole, plan.split, plan.parts, plan.recs, plan.rows, static_cast<float*>(pieces)};
}

// 2: rows of whole 32-byte sectors, 1: of 16-byte vectors, 0: neither.
inline int vec_ok(const void* y, int64_t ldy, bool f32) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(y) | static_cast<uint64_t>(ldy * (f32 ? 4 : 2));
  return bits % 32 == 0 ? 2 : bits % 16 == 0 ? 1 : 0;
}

}  // namespace fp4
}  // namespace aex
