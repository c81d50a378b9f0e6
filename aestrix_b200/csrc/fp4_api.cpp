// fp4_api.cpp — argument checks and dispatch of the products with microscaled
// 4-bit weights.
#include <cmath>

#include "fp4_internal.h"

namespace aex {
namespace {

int check_weight(aex_ctx* ctx, const aex_fp4weight* w, const char* name) {
  if (!w) return set_error(ctx, AEX_ERR_INVALID_ARG, "%s is NULL", name);
  if (w->device != ctx->device) return set_error(ctx, AEX_ERR_INVALID_ARG, "%s lives on another device", name);
  return AEX_OK;
}

int check_pair(aex_ctx* ctx, const aex_fp4weight* g, const aex_fp4weight* u, int activation) {
  if (int r = check_weight(ctx, g, "w_gate")) return r;
  if (int r = check_weight(ctx, u, "w_up")) return r;
  if (g->n != u->n || g->k != u->k || g->format != u->format)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "w_gate and w_up must have one shape and format");
  if (activation != AEX_ACT_SILU && activation != AEX_ACT_GELU_TANH)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "activation must be AEX_ACT_SILU or AEX_ACT_GELU_TANH");
  return AEX_OK;
}

int check_out(aex_ctx* ctx, const char* name, const void* y, int dtype, int64_t ld, int cols) {
  if (!y) return set_error(ctx, AEX_ERR_INVALID_ARG, "%s is NULL", name);
  if (dtype != AEX_DTYPE_BF16 && dtype != AEX_DTYPE_F32)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "%s: dtype must be AEX_DTYPE_BF16 or AEX_DTYPE_F32", name);
  if ((reinterpret_cast<uintptr_t>(y) & (dtype == AEX_DTYPE_F32 ? 3 : 1)) || ld < cols)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "%s must be aligned to its element with a row pitch of at least %d", name,
                     cols);
  return AEX_OK;
}

// Other CTAs may still read the input when the first results are written.
int check_apart(aex_ctx* ctx, const char* out, const void* y, int y_dtype, int64_t ldy, int cols, const char* in,
                const void* x, int x_dtype, int64_t ldx, int x_cols, int rows) {
  const int64_t sy = y_dtype == AEX_DTYPE_F32 ? 4 : 2, sx = x_dtype == AEX_DTYPE_F32 ? 4 : 2;
  if (fp4::overlap(reinterpret_cast<uintptr_t>(y), cols * sy, ldy * sy, reinterpret_cast<uintptr_t>(x), x_cols * sx,
                   ldx * sx, rows))
    return set_error(ctx, AEX_ERR_INVALID_ARG, "%s must not overlap %s", out, in);
  return AEX_OK;
}

int check_workspace(aex_ctx* ctx, const void* p, size_t have, size_t need) {
  if (need && (!p || have < need || (reinterpret_cast<uintptr_t>(p) & 255)))
    return set_error(ctx, AEX_ERR_INVALID_ARG, "workspace: %zu bytes, 256-byte aligned, are needed", need);
  return AEX_OK;
}

size_t round256(size_t v) { return (v + 255) & ~size_t{255}; }

size_t records_bytes(const aex_fp4weight* w, int m) {
  const size_t tiles = (static_cast<size_t>(m) + fp4::kRecRows - 1) / fp4::kRecRows;
  return round256(tiles * w->k_blocks * fp4::rec_bytes(w->format));
}

// The workspace of a product: records of the quantized x, then the pieces of split tiles.
size_t mm_workspace(const aex_fp4weight* w, bool gated, int m, bool quantize) {
  if (m <= fp4::kSmallRows) return 0;
  return quantize ? records_bytes(w, m) + fp4::plan_block(w, gated, m).bytes : fp4::plan_gemm(w, gated, m).bytes;
}

// The gradients read dy and dh in 16-byte vectors. Where n is no multiple of 8, rows that do not stand so (those of a
// contiguous result, say) are copied into the workspace first.
int64_t padded(int n) { return (static_cast<int64_t>(n) + 7) / 8 * 8; }
size_t grad_bytes(int m, int n) { return round256(static_cast<size_t>(m) * padded(n) * 2); }
size_t copy_bytes(int m, int n) { return n % 8 ? grad_bytes(m, n) : 0; }

int check_grad(aex_ctx* ctx, const char* name, const void* p, int64_t ld, int m, int n) {
  if (n % 8 == 0) return fp4::check_matrix(ctx, name, p, AEX_DTYPE_BF16, ld, m, n);
  if (m <= 0) return set_error(ctx, AEX_ERR_INVALID_ARG, "%s: the number of rows must be positive", name);
  return check_out(ctx, name, p, AEX_DTYPE_BF16, ld, n);
}

bool whole_rows(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

int check_tiles(aex_ctx* ctx, const fp4::TilePlan& p) {
  return p.clusters ? AEX_OK : set_error(ctx, AEX_ERR_UNSUPPORTED, "the product has too many output tiles");
}

int run(aex_ctx* ctx, const aex_fp4weight* w0, const aex_fp4weight* w1, int activation, const aex_fp4_mm_args* a,
        aex_stream stream) {
  if (!a) return set_error(ctx, AEX_ERR_INVALID_ARG, "args is NULL");
  if (a->m <= 0) return set_error(ctx, AEX_ERR_INVALID_ARG, "m must be positive");
  if (int r = fp4::check_matrix(ctx, "x", a->x, a->x_dtype, a->ldx, a->m, w0->k)) return r;
  if (int r = check_out(ctx, "y", a->y, a->y_dtype, a->ldy, w0->n)) return r;
  if (int r = check_apart(ctx, "y", a->y, a->y_dtype, a->ldy, w0->n, "x", a->x, a->x_dtype, a->ldx, w0->k, a->m))
    return r;
  const bool f32 = a->x_dtype == AEX_DTYPE_F32;
  if (a->quantize_x != 0 && a->quantize_x != 1)
    return set_error(ctx, AEX_ERR_INVALID_ARG, "quantize_x must be 0 or 1");
  if (a->quantize_x)
    if (int r = fp4::check_format(ctx, w0->format, a->x_scale)) return r;
  // The sums are multiplied by both tensor scales at once.
  for (const aex_fp4weight* w : {w0, w1})
    if (a->quantize_x && w && !std::isnormal(a->x_scale * w->tensor_scale))
      return set_error(ctx, AEX_ERR_INVALID_ARG, "x_scale times the weight's tensor scale must be a normal f32");
  if (f32 && !a->quantize_x && a->m > fp4::kSmallRows)
    return set_error(ctx, AEX_ERR_UNSUPPORTED, "f32 activations without quantize_x are supported for m <= %d",
                     fp4::kSmallRows);
  const bool gated = w1 != nullptr;
  if (a->m > fp4::kSmallRows)
    if (int r = check_tiles(ctx, a->quantize_x ? fp4::plan_block(w0, gated, a->m) : fp4::plan_gemm(w0, gated, a->m)))
      return r;
  if (int r = check_workspace(ctx, a->workspace, a->workspace_bytes, mm_workspace(w0, gated, a->m, a->quantize_x)))
    return r;
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  fp4::Job j{};
  j.w0 = w0;
  j.w1 = w1;
  j.activation = activation;
  j.x = a->x;
  j.x_f32 = f32;
  j.ldx = a->ldx;
  j.m = a->m;
  j.quantize = a->quantize_x != 0;
  j.x_scale = j.quantize ? a->x_scale : 1.f;
  j.y = a->y;
  j.y_f32 = a->y_dtype == AEX_DTYPE_F32;
  j.ldy = a->ldy;
  auto s = static_cast<cudaStream_t>(stream);
  if (j.m <= fp4::kSmallRows) return fp4::run_small(ctx, j, s);
  if (j.quantize) {
    j.x_records = static_cast<uint8_t*>(a->workspace);
    j.pieces = j.x_records + records_bytes(w0, j.m);
    if (int r = fp4::quantize_records(ctx, j.x, j.x_f32, j.ldx, j.m, w0->k, w0->format, j.x_scale, j.x_records, s))
      return r;
    return fp4::run_block(ctx, j, s);
  }
  j.pieces = a->workspace;
  return fp4::run_gemm(ctx, j, s);
}

}  // namespace
}  // namespace aex

extern "C" {

size_t aex_fp4_mm_workspace_bytes(const aex_fp4weight* w, int m, int quantize_x) {
  return w && m > 0 ? aex::mm_workspace(w, false, m, quantize_x != 0) : 0;
}

size_t aex_fp4_gated_mm_workspace_bytes(const aex_fp4weight* w_gate, int m, int quantize_x) {
  return w_gate && m > 0 ? aex::mm_workspace(w_gate, true, m, quantize_x != 0) : 0;
}

int aex_fp4_mm(aex_ctx* ctx, const aex_fp4weight* w, const aex_fp4_mm_args* args, aex_stream stream) {
  using namespace aex;
  if (!ctx) return set_error(ctx, AEX_ERR_INVALID_ARG, "NULL ctx");
  if (int r = check_weight(ctx, w, "w")) return r;
  return run(ctx, w, nullptr, AEX_ACT_SILU, args, stream);
}

int aex_fp4_gated_mm(aex_ctx* ctx, const aex_fp4weight* w_gate, const aex_fp4weight* w_up, int activation,
                     const aex_fp4_mm_args* args, aex_stream stream) {
  using namespace aex;
  if (!ctx) return set_error(ctx, AEX_ERR_INVALID_ARG, "NULL ctx");
  if (int r = check_pair(ctx, w_gate, w_up, activation)) return r;
  return run(ctx, w_gate, w_up, activation, args, stream);
}

size_t aex_fp4_mm_dgrad_workspace_bytes(const aex_fp4weight* w, int m) {
  return w && m > 0 ? aex::copy_bytes(m, w->n) + aex::fp4::plan_dgrad(w, false, m).bytes : 0;
}

int aex_fp4_mm_dgrad(aex_ctx* ctx, const aex_fp4weight* w, const void* dy, int64_t lddy, int m, void* dx,
                     int dx_dtype, int64_t lddx, void* workspace, size_t workspace_bytes, aex_stream stream) {
  using namespace aex;
  if (!ctx) return set_error(ctx, AEX_ERR_INVALID_ARG, "NULL ctx");
  if (int r = check_weight(ctx, w, "w")) return r;
  if (int r = check_grad(ctx, "dy", dy, lddy, m, w->n)) return r;
  if (int r = check_out(ctx, "dx", dx, dx_dtype, lddx, w->k)) return r;
  if (int r = check_apart(ctx, "dx", dx, dx_dtype, lddx, w->k, "dy", dy, AEX_DTYPE_BF16, lddy, w->n, m)) return r;
  const fp4::TilePlan plan = fp4::plan_dgrad(w, false, m);
  if (int r = check_tiles(ctx, plan)) return r;
  const size_t copy = whole_rows(dy, lddy) ? 0 : copy_bytes(m, w->n);
  if (int r = check_workspace(ctx, workspace, workspace_bytes, copy + plan.bytes)) return r;
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  auto s = static_cast<cudaStream_t>(stream);
  if (copy) {
    if (int r = fp4::pad_rows(ctx, dy, lddy, m, w->n, workspace, padded(w->n), s)) return r;
    dy = workspace;
    lddy = padded(w->n);
  }
  return fp4::run_dgrad(ctx, w, nullptr, dy, lddy, nullptr, 0, m, w->tensor_scale, dx, dx_dtype == AEX_DTYPE_F32, lddx,
                        static_cast<uint8_t*>(workspace) + copy, s);
}

// dg and du, bf16, rows padded to 16 bytes, the copy of dh, then the pieces of whichever of the two products has more.
size_t aex_fp4_gated_mm_dgrad_workspace_bytes(const aex_fp4weight* w_gate, int m) {
  if (!w_gate || m <= 0) return 0;
  const size_t d = aex::grad_bytes(m, w_gate->n);
  const size_t p0 = aex::fp4::plan_gemm(w_gate, true, m).bytes, p1 = aex::fp4::plan_dgrad(w_gate, true, m).bytes;
  return 2 * d + aex::copy_bytes(m, w_gate->n) + (p0 > p1 ? p0 : p1);
}

int aex_fp4_gated_mm_dgrad(aex_ctx* ctx, const aex_fp4weight* w_gate, const aex_fp4weight* w_up, int activation,
                           const void* x, int64_t ldx, const void* dh, int64_t lddh, int m, void* dx, int64_t lddx,
                           void* workspace, size_t workspace_bytes, aex_stream stream) {
  using namespace aex;
  if (!ctx) return set_error(ctx, AEX_ERR_INVALID_ARG, "NULL ctx");
  if (int r = check_pair(ctx, w_gate, w_up, activation)) return r;
  if (int r = fp4::check_matrix(ctx, "x", x, AEX_DTYPE_BF16, ldx, m, w_gate->k)) return r;
  if (int r = check_grad(ctx, "dh", dh, lddh, m, w_gate->n)) return r;
  if (int r = check_out(ctx, "dx", dx, AEX_DTYPE_BF16, lddx, w_gate->k)) return r;
  if (int r = check_tiles(ctx, fp4::plan_gemm(w_gate, true, m))) return r;
  if (int r = check_tiles(ctx, fp4::plan_dgrad(w_gate, true, m))) return r;
  const size_t copy = whole_rows(dh, lddh) ? 0 : copy_bytes(m, w_gate->n);
  const size_t need = aex_fp4_gated_mm_dgrad_workspace_bytes(w_gate, m) - (copy_bytes(m, w_gate->n) - copy);
  if (int r = check_workspace(ctx, workspace, workspace_bytes, need)) return r;
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  auto s = static_cast<cudaStream_t>(stream);
  // The tensor scales go into dg and du, so that one accumulator takes both products.
  const int64_t ld = padded(w_gate->n);
  const size_t d = grad_bytes(m, w_gate->n);
  auto* ws = static_cast<uint8_t*>(workspace);
  auto* dg = reinterpret_cast<uint16_t*>(ws);
  auto* du = reinterpret_cast<uint16_t*>(ws + d);
  if (copy) {
    if (int r = fp4::pad_rows(ctx, dh, lddh, m, w_gate->n, ws + 2 * d, ld, s)) return r;
    dh = ws + 2 * d;
    lddh = ld;
  }
  void* pieces = ws + 2 * d + copy;
  if (int r = fp4::run_gated_grad(ctx, w_gate, w_up, activation, x, ldx, m, dh, lddh, dg, du, ld, pieces, s)) return r;
  return fp4::run_dgrad(ctx, w_gate, w_up, dg, ld, du, ld, m, 1.f, dx, false, lddx, pieces, s);
}

}  // extern "C"
