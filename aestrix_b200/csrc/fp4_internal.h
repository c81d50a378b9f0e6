// fp4_internal.h — host-side pieces shared by the translation units of the
// microscaled 4-bit operators.
#pragma once
#ifdef __CUDACC__
#define AEX_HD __host__ __device__
#else
#define AEX_HD
#endif
#include <algorithm>
#include <atomic>

#include "internal.h"

struct aex_fp4weight {
  int device = 0;
  int n = 0, k = 0;
  int format = AEX_FP4_NV;
  float tensor_scale = 1.f;
  int n_tiles = 0;           // ceil(n / 128)
  int k_blocks = 0;          // ceil(k / 256)
  int clusters = 0;          // CTA pairs of the GEMMs that the device holds at once (one CTA per SM)
  uint8_t* records = nullptr;
  size_t bytes = 0;
};

namespace aex {

// Makes the context's device current and puts the caller's back on leaving.
struct DeviceGuard {
  int prev = -1, rc = AEX_OK;
  bool switched = false;
  explicit DeviceGuard(aex_ctx* ctx) {
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != ctx->device) {
      e = cudaSetDevice(ctx->device);
      switched = e == cudaSuccess;
    }
    if (e != cudaSuccess) rc = cuda_error(ctx, e, "selecting the context's device");
  }
  ~DeviceGuard() {
    if (switched) cudaSetDevice(prev);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
};

// cudaFuncSetAttribute(maximum dynamic shared memory), once per kernel and device: it costs a good part of a launch.
struct SmemOptIn {
  std::atomic<uint64_t> done{0};
  int operator()(aex_ctx* ctx, const void* kernel, int bytes) {
    const uint64_t bit = uint64_t{1} << (ctx->device & 63);
    if (ctx->device < 64 && (done.load(std::memory_order_acquire) & bit)) return AEX_OK;
    AEX_CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_release);
    return AEX_OK;
  }
};

namespace fp4 {

constexpr int kRecRows = 128;
constexpr int kRecK = 256;
constexpr int kRecCodes = kRecRows * kRecK / 2;  // 16384

AEX_HD constexpr int block_of(int format) { return format == AEX_FP4_MX ? 32 : 16; }
AEX_HD constexpr int rec_scales(int format) { return kRecRows * kRecK / block_of(format); }
AEX_HD constexpr int rec_bytes(int format) { return kRecCodes + rec_scales(format); }

// Byte offset of row r's scale group g (4 consecutive scales) inside a record.
AEX_HD constexpr int scale_off(int r, int g) {
  return kRecCodes + g * 512 + (r & 31) * 16 + (r >> 5) * 4;
}

// How many of the columns [col, col + count) a matrix of `cols` has (col + count may leave 32 bits).
AEX_HD constexpr int columns_within(int col, int count, int cols) { return cols - col < count ? cols - col : count; }
// Records along k columns (k + 255 may leave 32 bits).
constexpr int records_along(int k) { return (k - 1) / kRecK + 1; }

// The conversions count their units of 16 columns (`upr` a row) in 32 bits and
// find a unit's row by a division that is exact below 2^31.
struct FastDiv {  // u / div = umulhi(u, mul) >> shift for u < 2^31
  uint32_t mul, shift, div;
};
inline FastDiv fast_div(uint32_t d) {
  if (d == 1) return FastDiv{0, 0, 1};
  uint32_t l = 1;
  while ((uint64_t{1} << l) < d) ++l;
  return FastDiv{static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + d - 1) / d), l - 1, d};
}
// Rows of one launch: at most 2^30 units, in whole tiles of 128 rows, or (rows of more than 2^23 units) a power of two
// of rows, so that a slice lies within one tile. A row has at most 2^27 units, k being below 2^31.
inline int64_t slice_rows(uint32_t upr) {
  const int64_t most = (int64_t{1} << 30) / upr;
  if (most >= kRecRows) return most / kRecRows * kRecRows;
  int64_t rows = 1;
  while (2 * rows <= most) rows *= 2;
  return rows;
}

// Whether two matrices of `rows` rows at a and b, of so many bytes a row and from one row to the next, share memory.
// Rows of one pitch may lie beside one another (columns of one buffer); of two pitches they are taken to share what
// their ranges share.
inline bool overlap(uintptr_t a, int64_t a_row, int64_t a_pitch, uintptr_t b, int64_t b_row, int64_t b_pitch, int rows) {
  const uintptr_t a_end = a + static_cast<uintptr_t>((rows - 1) * a_pitch + a_row);
  const uintptr_t b_end = b + static_cast<uintptr_t>((rows - 1) * b_pitch + b_row);
  if (a >= b_end || b >= a_end) return false;
  if (rows == 1 || a_pitch != b_pitch) return true;
  const auto pitch = static_cast<uintptr_t>(a_pitch);
  const auto d = static_cast<int64_t>(b >= a ? (b - a) % pitch : (pitch - (a - b) % pitch) % pitch);  // b's first column
  return d < a_row || d + b_row > a_pitch;
}

int check_format(aex_ctx* ctx, int format, float tensor_scale);
// A row-major matrix that is read or written in 16-byte vectors.
int check_matrix(aex_ctx* ctx, const char* name, const void* p, int dtype, int64_t ld, int rows, int cols);

// x [m, k] -> records (columns padded to whole records with zeros; rows past m left as they are).
int quantize_records(aex_ctx* ctx, const void* x, bool f32, int64_t ldx, int m, int k, int format, float ts,
                     uint8_t* records, cudaStream_t s);

// One product (w1 NULL) or gated projection act(x w0^T) * (x w1^T).
struct Job {
  const aex_fp4weight* w0;
  const aex_fp4weight* w1;
  int activation;
  const void* x;
  bool x_f32;
  int64_t ldx;
  int m;
  bool quantize;
  float x_scale;
  void* y;
  bool y_f32;
  int64_t ldy;
  uint8_t* x_records;  // workspace: the quantized x, and the pieces of split tiles
  void* pieces;
};

// How a GEMM's 256 x 256 output tiles go to `clusters` CTA pairs (TileWork).
struct TilePlan {
  int clusters = 0;  // of the launch
  int m_tiles = 0, whole = 0, split = 0, parts = 0, recs = 0;
  int rows = 0;       // of a piece
  size_t bytes = 0;   // of all pieces
};

// `recs` records along K per tile, `rec_us` microseconds each in the main loop. Tiles that do not fill a last wave of
// the clusters are split when that wave's records, dealt out over the clusters (32 pieces a tile at most), and the
// join take less than the wave. The join: 2.5 us, 1 us for every eight pieces of a tile, and the pieces written and
// read (B200, measured: 4 us for 6 MB, 8 us for 20 MB; 77 rows through 7680 -> 4096 51 us whole, 22 us split; 512
// rows back through 4096 -> 7680 30.8 us whole, 32.0 us split).
inline TilePlan plan_tiles(int clusters, int m, int64_t col_tiles, int recs, double rec_us) {
  TilePlan p;
  p.m_tiles = (m - 1) / 256 + 1;
  p.rows = m < 256 ? m : 256;
  p.recs = recs;
  const int64_t tiles = p.m_tiles * col_tiles;
  if (tiles > 0x3FFFFFFF) return p;  // refused by the caller
  const int64_t left = tiles % clusters;
  p.whole = static_cast<int>(tiles);
  if (left && left * recs < 0x7FFFFFFF / (clusters + 1)) {
    const int64_t parts = std::min<int64_t>(clusters, left * std::min(recs, 32));
    const int64_t share = (left * recs + parts - 1) / parts;
    const size_t bytes = static_cast<size_t>(parts + left) * ((p.rows + 31) / 32 * 32) * 256 * sizeof(float);
    const double join = 2.5 + 1.0 * static_cast<double>(parts / left / 8 + 1) + 2.0 * static_cast<double>(bytes) / 6.5e6;
    if (rec_us * static_cast<double>(recs - share) > join) {
      p.split = static_cast<int>(left);
      p.parts = static_cast<int>(parts);
      p.whole -= p.split;
      p.bytes = bytes;
    }
  }
  p.clusters = std::max(p.parts, std::min(p.whole, clusters));
  return p;
}
TilePlan plan_gemm(const aex_fp4weight* w, bool gated, int m);
TilePlan plan_dgrad(const aex_fp4weight* w, bool two, int m);
TilePlan plan_block(const aex_fp4weight* w, bool gated, int m);
int gemm_clusters(aex_ctx* ctx, int* out);

// One launch of CTA pairs; `after`: set up while the stream's previous kernel runs (the kernel waits for it itself).
template <typename... Args>
int launch_pairs(aex_ctx* ctx, const void* kernel, int clusters, int threads, int smem, bool after, cudaStream_t s,
                 Args*... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * clusters, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after ? 2 : 1;
  void* argv[] = {args...};
  AEX_CUDA_TRY(ctx, cudaLaunchKernelExC(&cfg, kernel, argv));
  return check_launch(ctx, "fp4 GEMM");
}
// A plain grid that is set up while the stream's previous kernel runs and waits for it itself.
template <typename... Args>
int launch_after(aex_ctx* ctx, const void* kernel, int blocks, int threads, cudaStream_t s, Args*... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* argv[] = {args...};
  AEX_CUDA_TRY(ctx, cudaLaunchKernelExC(&cfg, kernel, argv));
  return check_launch(ctx, "fp4 join");
}

// The few-rows kernel takes a row as one column of its 8-column operand where it is bf16 or quantized, f32 rows as
// two columns each. No workspace. More rows go to the GEMMs: 19 rows, 7520 -> 5376, take 37 us as four times 8
// columns and 24 us there.
constexpr int kSmallRows = 16;
int run_small(aex_ctx* ctx, const Job& j, cudaStream_t s);
// Any number of bf16 rows: dequantizing GEMM.
int run_gemm(aex_ctx* ctx, const Job& j, cudaStream_t s);
// Quantized rows (x_records): block-scaled GEMM.
int run_block(aex_ctx* ctx, const Job& j, cudaStream_t s);
// dst [rows, cols] (16-byte aligned, pitch ldd a multiple of 8) = src, bf16, at any pitch and element-aligned start;
// columns [cols, ldd) become zeros.
int pad_rows(aex_ctx* ctx, const void* src, int64_t ld, int rows, int cols, void* dst, int64_t ldd, cudaStream_t s);
// dx = alpha (d0 . W0 + d1 . W1) (w1, d1 NULL: one product), d bf16 [m, n].
int run_dgrad(aex_ctx* ctx, const aex_fp4weight* w0, const aex_fp4weight* w1, const void* d0, int64_t ld0,
              const void* d1, int64_t ld1, int m, float alpha, void* dx, bool dx_f32, int64_t lddx, void* pieces,
              cudaStream_t s);
// dg = ts_g dh u act'(g), du = ts_u dh act(g), bf16 [m, n] at row pitch ld, g and u from x.
int run_gated_grad(aex_ctx* ctx, const aex_fp4weight* wg, const aex_fp4weight* wu, int activation, const void* x,
                   int64_t ldx, int m, const void* dh, int64_t lddh, uint16_t* dg, uint16_t* du, int64_t ld,
                   void* pieces, cudaStream_t s);

}  // namespace fp4
}  // namespace aex
