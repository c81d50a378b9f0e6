"""Microscaled 4-bit floating-point linears over libaestrix_cuda (ctypes binding), beside the affine
ones of :mod:`aestrix_b200.qmm`.

A matrix is held as e2m1 codes (two to a byte, the even column in the low nibble; the uint32 words
of an MLX pack of mode "mxfp4" or "nvfp4", unchanged) and one scale byte per block of columns:

* ``"mxfp4"``: blocks of 32, scale 2^(byte - 127);
* ``"nvfp4"``: blocks of 16, scale an e4m3 number, times one f32 for the whole tensor.

* :func:`quantize`, :func:`dequantize` — to this form and back;
* :class:`FP4Weight` — a weight laid out on the device for the products;
* :func:`fp4_mm` — ``y = x . W^T``, activations as they are or quantized within the call;
* :func:`fp4_gated_mm` — ``act(x . Wg^T) * (x . Wu^T)`` in one kernel (linear_in -> silu(g) * u,
  Sources/ImarelloDiT/FeedForward.swift:11-24);
* :func:`fp4_mm_dgrad`, :func:`fp4_gated_mm_dgrad` — their gradients with respect to ``x`` (a 4-bit
  weight is frozen).

Tensors are 2-D CUDA tensors with contiguous rows whose pitch is a multiple of 16 bytes. Every call
runs on ``stream`` (default: the current stream of the tensors' device); scratch comes from torch's
allocator, so calls on different streams and captured graphs do not share any.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

MODES = {"mxfp4": _lib.AEX_FP4_MX, "nvfp4": _lib.AEX_FP4_NV}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
ACTIVATIONS = {"silu": _lib.AEX_ACT_SILU, "gelu_tanh": _lib.AEX_ACT_GELU_TANH}
_DTYPES = {torch.bfloat16: _lib.AEX_DTYPE_BF16, torch.float32: _lib.AEX_DTYPE_F32}


def _mode(mode):
    if mode not in MODES:
        raise ValueError(f"mode must be one of {sorted(MODES)}")
    return MODES[mode]


def _matrix(name, t, dtypes=(torch.bfloat16, torch.float32), cols=None):
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.dim() != 2:
        raise TypeError(f"{name} must be a 2-D tensor of {' or '.join(str(d) for d in dtypes)}")
    if not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if cols is not None and t.shape[1] != cols:
        raise ValueError(f"{name} must have {cols} columns, has {t.shape[1]}")
    if t.shape[0] < 1:
        raise ValueError(f"{name} has no rows")
    if t.stride(1) != 1 and t.shape[1] != 1:
        raise ValueError(f"{name} must have contiguous rows")
    return t


def _pitch(t):
    # the stride of a single row says nothing: torch leaves any value there
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


def _empty(shape, dtype, device, stream):
    """A tensor that belongs to the stream its kernels run on, as one made under torch.cuda.stream(stream)."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _out(out, rows, cols, dtype, like, stream):
    if out is None:
        if dtype not in _DTYPES:
            raise TypeError("out_dtype must be torch.bfloat16 or torch.float32")
        return _empty((rows, cols), dtype, like.device, stream)
    _matrix("out", out)
    if tuple(out.shape) != (rows, cols) or out.device != like.device:
        raise ValueError(f"out must be [{rows}, {cols}] on {like.device}")
    return out


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _stream(stream, device):
    return (stream or torch.cuda.current_stream(device)).cuda_stream


def _check_codes(codes, scales, mode):
    for name, t in (("codes", codes), ("scales", scales)):
        _matrix(name, t, (torch.uint8,))
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    _same_device(codes.device, scales=scales)
    rows, k = codes.shape[0], codes.shape[1] * 2
    if tuple(scales.shape) != (rows, k // BLOCK[mode]) or k % 32:
        raise ValueError(f"codes [rows, k/2] and scales [rows, k/{BLOCK[mode]}] with k a multiple of 32")
    return rows, k


def quantize(x, mode="nvfp4", tensor_scale=1.0, ctx=None, stream=None):
    """codes uint8 [rows, k/2], scales uint8 [rows, k/block] of x [rows, k] (bf16 or f32, k a multiple
    of 32). nvfp4: the usual tensor_scale is amax(|x|) / (448 * 6); mxfp4 has none. A block's scale
    and codes are those of the exact quotients, ties to even; a block that holds an infinity or NaN
    gets a NaN scale."""
    fmt = _mode(mode)
    _matrix("x", x)
    rows, k = x.shape
    if k % 32 or k == 0:
        raise ValueError("the number of columns must be a positive multiple of 32")
    ctx = ctx or _lib.context(x.device.index or 0)
    codes = _empty((rows, k // 2), torch.uint8, x.device, stream)
    scales = _empty((rows, k // BLOCK[mode]), torch.uint8, x.device, stream)
    ctx.check(_lib.lib().aex_fp4_quantize(ctx.handle, x.data_ptr(), _DTYPES[x.dtype], _pitch(x), rows, k, fmt,
                                          tensor_scale, codes.data_ptr(), scales.data_ptr(),
                                          _stream(stream, x.device)))
    return codes, scales


def dequantize(codes, scales, mode="nvfp4", tensor_scale=1.0, out_dtype=torch.bfloat16, out=None, ctx=None,
               stream=None):
    """[rows, k] code * scale * tensor_scale, rounded once to bf16 or f32."""
    fmt = _mode(mode)
    rows, k = _check_codes(codes, scales, mode)
    out = _out(out, rows, k, out_dtype, codes, stream)
    ctx = ctx or _lib.context(codes.device.index or 0)
    ctx.check(_lib.lib().aex_fp4_dequantize(ctx.handle, codes.data_ptr(), scales.data_ptr(), rows, k, fmt,
                                            tensor_scale, out.data_ptr(), _DTYPES[out.dtype], _pitch(out),
                                            _stream(stream, codes.device)))
    return out


class FP4Weight:
    """Device-resident microscaled 4-bit weight [n, k] (owns an aex_fp4weight handle). codes and scales
    as :func:`quantize` returns them, or as they stand in a pack (uint32 words viewed as uint8)."""

    def __init__(self, codes, scales, mode="nvfp4", tensor_scale=1.0, ctx=None, stream=None):
        fmt = _mode(mode)
        self.n, self.k = _check_codes(codes, scales, mode)
        self.mode = mode
        self.tensor_scale = tensor_scale
        self.device = codes.device
        self.ctx = ctx or _lib.context(codes.device.index or 0)
        h = C.c_void_p()
        self.ctx.check(_lib.lib().aex_fp4weight_create(self.ctx.handle, codes.data_ptr(), scales.data_ptr(), self.n,
                                                       self.k, fmt, tensor_scale, C.byref(h),
                                                       _stream(stream, codes.device)))
        self.handle = h

    def close(self):
        if getattr(self, "handle", None):
            _lib.lib().aex_fp4weight_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def dequantize(self, out_dtype=torch.bfloat16, stream=None):
        if out_dtype not in _DTYPES:
            raise TypeError("out_dtype must be torch.bfloat16 or torch.float32")
        out = _empty((self.n, self.k), out_dtype, self.device, stream)
        self.ctx.check(_lib.lib().aex_fp4weight_dequantize(self.ctx.handle, self.handle, out.data_ptr(),
                                                           _DTYPES[out_dtype], self.k, _stream(stream, self.device)))
        return out

    def __call__(self, x, **kw):
        return fp4_mm(x, self, **kw)


def _open(*weights):
    for w in weights:
        if not isinstance(w, FP4Weight):
            raise TypeError("weights must be FP4Weight")
        if not w.handle:
            raise ValueError("the weight is closed")


def _args(x, w, quantize_x, x_scale, out, stream):
    a = _lib.aex_fp4_mm_args()
    a.x, a.x_dtype, a.ldx, a.m = x.data_ptr(), _DTYPES[x.dtype], _pitch(x), x.shape[0]
    a.quantize_x, a.x_scale = int(bool(quantize_x)), x_scale
    a.y, a.y_dtype, a.ldy = out.data_ptr(), _DTYPES[out.dtype], out.stride(0) if a.m > 1 else w.n
    a.workspace_bytes = _lib.lib().aex_fp4_mm_workspace_bytes(w.handle, a.m, a.quantize_x)
    ws = _empty((a.workspace_bytes,), torch.uint8, x.device, stream) if a.workspace_bytes else None
    a.workspace = None if ws is None else ws.data_ptr()
    return a, ws


def fp4_mm(x, w: FP4Weight, quantize_x=False, x_scale=1.0, out_dtype=torch.bfloat16, out=None, stream=None):
    """y[m, n] = x[m, k] . W[n, k]^T, f32 sums, rounded once to bf16 or f32. x is bf16, or f32 for m <= 16.
    With quantize_x, x (bf16 or f32, any m) goes through :func:`quantize`'s rounding in the weight's
    mode first, with x_scale as its tensor scale, and both operands are multiplied in 4 bits. f32
    results of more than 16 rows carry the tensor core's truncating f32 sums (about 1e-5 of their
    size at k = 9216, as the affine linears' do)."""
    _open(w)
    _matrix("x", x, cols=w.k)
    _same_device(w.device, x=x)
    out = _out(out, x.shape[0], w.n, out_dtype, x, stream)
    a, ws = _args(x, w, quantize_x, x_scale, out, stream)
    w.ctx.check(_lib.lib().aex_fp4_mm(w.ctx.handle, w.handle, C.byref(a), _stream(stream, w.device)))
    del ws
    return out


def fp4_gated_mm(x, w_gate: FP4Weight, w_up: FP4Weight, activation="silu", quantize_x=False, x_scale=1.0,
                 out_dtype=torch.bfloat16, out=None, stream=None):
    """h[m, n] = act(x . Wg^T) * (x . Wu^T): both projections, the activation ("silu" or "gelu_tanh") and
    the product in one kernel, rounded once. x, quantize_x and x_scale as :func:`fp4_mm`."""
    _open(w_gate, w_up)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    _matrix("x", x, cols=w_gate.k)
    _same_device(w_gate.device, x=x)
    out = _out(out, x.shape[0], w_gate.n, out_dtype, x, stream)
    a, ws = _args(x, w_gate, quantize_x, x_scale, out, stream)
    w_gate.ctx.check(_lib.lib().aex_fp4_gated_mm(w_gate.ctx.handle, w_gate.handle, w_up.handle,
                                                 ACTIVATIONS[activation], C.byref(a),
                                                 _stream(stream, w_gate.device)))
    del ws
    return out


def fp4_mm_dgrad(dy, w: FP4Weight, out_dtype=torch.bfloat16, out=None, stream=None):
    """dx[m, k] = dy[m, n] . W[n, k], the gradient of :func:`fp4_mm` (without quantize_x); dy bf16."""
    _open(w)
    _matrix("dy", dy, (torch.bfloat16,), cols=w.n)
    _same_device(w.device, dy=dy)
    out = _out(out, dy.shape[0], w.k, out_dtype, dy, stream)
    w.ctx.check(_lib.lib().aex_fp4_mm_dgrad(w.ctx.handle, w.handle, dy.data_ptr(), _pitch(dy), dy.shape[0],
                                            out.data_ptr(), _DTYPES[out.dtype], _pitch(out),
                                            _stream(stream, w.device)))
    return out


def fp4_gated_mm_dgrad(dh, x, w_gate: FP4Weight, w_up: FP4Weight, activation="silu", out_dtype=torch.bfloat16,
                       out=None, stream=None):
    """dx[m, k] of :func:`fp4_gated_mm` (without quantize_x) from dh[m, n] and the forward pass's x; both
    bf16, dx bf16. The projections are computed again; nothing need be kept from the forward pass."""
    _open(w_gate, w_up)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    _matrix("x", x, (torch.bfloat16,), cols=w_gate.k)
    _matrix("dh", dh, (torch.bfloat16,), cols=w_gate.n)
    _same_device(w_gate.device, x=x, dh=dh)
    if dh.shape[0] != x.shape[0]:
        raise ValueError("dh and x must have the same number of rows")
    out = _out(out, x.shape[0], w_gate.k, out_dtype, x, stream)
    if out.dtype != torch.bfloat16:
        raise TypeError("the gradient is bfloat16")
    n = _lib.lib().aex_fp4_gated_mm_dgrad_workspace_bytes(w_gate.handle, x.shape[0])
    ws = _empty((n,), torch.uint8, x.device, stream)
    w_gate.ctx.check(_lib.lib().aex_fp4_gated_mm_dgrad(
        w_gate.ctx.handle, w_gate.handle, w_up.handle, ACTIVATIONS[activation], x.data_ptr(), _pitch(x),
        dh.data_ptr(), _pitch(dh), x.shape[0], out.data_ptr(), _pitch(out), ws.data_ptr(), n,
        _stream(stream, w_gate.device)))
    del ws
    return out
