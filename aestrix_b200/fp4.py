"""Microscaled 4-bit floating-point linears over libaestrix_cuda (ctypes binding), beside the affine
ones of :mod:`aestrix_b200.qmm`.

A matrix is held as e2m1 codes (two to a byte, the even column in the low nibble; the uint32 words
of an MLX pack of mode "mxfp4" or "nvfp4", unchanged) and one scale byte per block of columns:

* ``"mxfp4"``: blocks of 32, scale 2^(byte - 127);
* ``"nvfp4"``: blocks of 16, scale an e4m3 number, times one f32 for the whole tensor.

* :func:`quantize`, :func:`dequantize` — to this form and back;
* :class:`FP4Weight` — a weight laid out on the device for the products;
* :func:`fp4_mm` — ``y = x . W^T``, activations as they are or quantized within the call;
* :func:`fp4_gated_mm` — ``act(x . Wg^T) * (x . Wu^T)``, neither projection stored (linear_in ->
  silu(g) * u, Sources/ImarelloDiT/FeedForward.swift:11-24);
* :func:`fp4_mm_dgrad`, :func:`fp4_gated_mm_dgrad` — their gradients with respect to ``x`` (a 4-bit
  weight is frozen). Autograd does not record the products: a result has no history, whatever x
  requires, and a backward pass calls these.

Tensors are 2-D CUDA tensors with contiguous rows; inputs start on 16 bytes and have a pitch of a
multiple of that (an incoming gradient of n columns, n no multiple of 8, may have any: it is copied
first). Results may have any pitch and start, and may not overlap an input. Every call runs on ``stream`` (default: the current
stream of the tensors' device); scratch comes from torch's allocator, so calls on different streams
and captured graphs do not share any. Tensors handed to a call with a ``stream`` of its own are
recorded on it, so they may be dropped at once; to order that stream behind whatever wrote them is
the caller's.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

MODES = {"mxfp4": _lib.AEX_FP4_MX, "nvfp4": _lib.AEX_FP4_NV}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
ACTIVATIONS = {"silu": _lib.AEX_ACT_SILU, "gelu_tanh": _lib.AEX_ACT_GELU_TANH}
_MAX = 2**31 - 1  # the C calls count rows and columns in 32 bits
_DTYPES = {torch.bfloat16: _lib.AEX_DTYPE_BF16, torch.float32: _lib.AEX_DTYPE_F32}


def _mode(mode):
    fmt = MODES.get(mode)
    if fmt is None:
        raise ValueError(f"mode must be one of {sorted(MODES)}")
    return fmt


# A few-rows product takes some microseconds on the device, so the checks before it count: they go
# by get_device() and plain integers, not by torch.device objects.

def _matrix(name, t, dtypes, cols=None, device=None):
    """The checks of a 2-D input with contiguous rows; its device's index."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.dim() != 2:
        raise TypeError(f"{name} must be a 2-D tensor of {' or '.join(str(d) for d in dtypes)}")
    at = t.get_device()
    if at < 0:
        raise TypeError(f"{name} must be a CUDA tensor")
    if device is not None and at != device:
        raise ValueError(f"{name} is on cuda:{at}, not on cuda:{device}")
    rows, have = t.shape
    if cols is not None and have != cols:
        raise ValueError(f"{name} must have {cols} columns, has {have}")
    if not 0 < rows <= _MAX or have > _MAX:
        raise ValueError(f"{name} has more than {_MAX} rows or columns" if rows else f"{name} has no rows")
    if have != 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have contiguous rows")
    return at


def _pitch(t):
    # the stride of a single row says nothing: torch leaves any value there
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


def _empty(shape, dtype, like, stream):
    """A tensor on like's device that belongs to the stream its kernels run on, as one made under
    torch.cuda.stream(stream)."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _used(stream, *tensors):
    """Tells torch's allocator of tensors that the given stream uses, so that their memory is handed to nobody
    before it has passed the call."""
    for t in tensors:
        t.record_stream(stream)


def _out(out, rows, cols, dtype, like, device, stream):
    if out is None:
        if dtype not in _DTYPES:
            raise TypeError("out_dtype must be torch.bfloat16 or torch.float32")
        return _empty((rows, cols), dtype, like, stream)
    _matrix("out", out, _DTYPES, cols, device)
    if out.shape[0] != rows:
        raise ValueError(f"out must have {rows} rows, has {out.shape[0]}")
    return out


_OPEN = {}  # device index -> (library, default context), looked up without the binding's locks


def _handles(ctx, device):
    if ctx is not None:
        if ctx.device != device:
            raise ValueError(f"the tensors are on cuda:{device}, the context on cuda:{ctx.device}")
        return _lib.lib(), ctx
    got = _OPEN.get(device)
    if got is None:
        got = _OPEN[device] = (_lib.lib(), _lib.context(device))
    return got


def _stream(stream, device):
    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(device)


_UINT8 = (torch.uint8,)
_BF16 = (torch.bfloat16,)


def _check_codes(codes, scales, mode):
    device = _matrix("codes", codes, _UINT8)
    _matrix("scales", scales, _UINT8, device=device)
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError("codes and scales must be contiguous")
    rows, k = codes.shape
    k *= 2
    if k > _MAX:
        raise ValueError(f"codes has more than {_MAX} columns")
    if k % 32 or scales.shape != (rows, k // BLOCK[mode]):
        raise ValueError(f"codes [rows, k/2] and scales [rows, k/{BLOCK[mode]}] with k a multiple of 32")
    return rows, k, device


def quantize(x, mode="nvfp4", tensor_scale=1.0, ctx=None, stream=None):
    """codes uint8 [rows, k/2], scales uint8 [rows, k/block] of x [rows, k] (bf16 or f32, k a multiple
    of 32). nvfp4: the usual tensor_scale is amax(|x|) / (448 * 6); mxfp4 has none. A block's scale
    and codes are those of the exact quotients, ties to even; a block that holds an infinity or NaN
    gets a NaN scale."""
    fmt = _mode(mode)
    device = _matrix("x", x, _DTYPES)
    rows, k = x.shape
    if k % 32 or k == 0:
        raise ValueError("the number of columns must be a positive multiple of 32")
    lib, ctx = _handles(ctx, device)
    codes = _empty((rows, k // 2), torch.uint8, x, stream)
    scales = _empty((rows, k // BLOCK[mode]), torch.uint8, x, stream)
    rc = lib.aex_fp4_quantize(ctx.handle, x.data_ptr(), _DTYPES[x.dtype], x.stride(0) if rows > 1 else k, rows, k, fmt,
                              tensor_scale, codes.data_ptr(), scales.data_ptr(), _stream(stream, device))
    if stream is not None:
        _used(stream, x)
    if rc:
        ctx.check(rc)
    return codes, scales


def dequantize(codes, scales, mode="nvfp4", tensor_scale=1.0, out_dtype=torch.bfloat16, out=None, ctx=None,
               stream=None):
    """[rows, k] code * scale * tensor_scale, rounded once to bf16 or f32."""
    fmt = _mode(mode)
    rows, k, device = _check_codes(codes, scales, mode)
    out = _out(out, rows, k, out_dtype, codes, device, stream)
    lib, ctx = _handles(ctx, device)
    rc = lib.aex_fp4_dequantize(ctx.handle, codes.data_ptr(), scales.data_ptr(), rows, k, fmt, tensor_scale,
                                out.data_ptr(), _DTYPES[out.dtype], out.stride(0) if rows > 1 else k,
                                _stream(stream, device))
    if stream is not None:
        _used(stream, codes, scales, out)
    if rc:
        ctx.check(rc)
    return out


class FP4Weight:
    """Device-resident microscaled 4-bit weight [n, k] (owns an aex_fp4weight handle). codes and scales
    as :func:`quantize` returns them, or as they stand in a pack (uint32 words viewed as uint8). Laid
    out on ``stream``; products on other streams are the caller's to order behind it. Not while a
    stream is being captured."""

    def __init__(self, codes, scales, mode="nvfp4", tensor_scale=1.0, ctx=None, stream=None):
        fmt = _mode(mode)
        self.n, self.k, self.index = _check_codes(codes, scales, mode)
        self.mode = mode
        self.tensor_scale = tensor_scale
        self.device = codes.device
        self.lib, self.ctx = _handles(ctx, self.index)
        h = C.c_void_p()
        self.ctx.check(self.lib.aex_fp4weight_create(self.ctx.handle, codes.data_ptr(), scales.data_ptr(), self.n,
                                                     self.k, fmt, tensor_scale, C.byref(h),
                                                     _stream(stream, self.index)))
        self.handle = h
        if stream is not None:
            _used(stream, codes, scales)

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
        _open(self)
        if out_dtype not in _DTYPES:
            raise TypeError("out_dtype must be torch.bfloat16 or torch.float32")
        if stream is None:
            out = torch.empty(self.n, self.k, dtype=out_dtype, device=self.device)
        else:
            with torch.cuda.stream(stream):
                out = torch.empty(self.n, self.k, dtype=out_dtype, device=self.device)
        self.ctx.check(self.lib.aex_fp4weight_dequantize(self.ctx.handle, self.handle, out.data_ptr(),
                                                         _DTYPES[out_dtype], self.k, _stream(stream, self.index)))
        return out

    def __call__(self, x, **kw):
        return fp4_mm(x, self, **kw)


def _open(*weights):
    for w in weights:
        if not isinstance(w, FP4Weight):
            raise TypeError("weights must be FP4Weight")
        if not w.handle:
            raise ValueError("the weight is closed")


_SMALL_ROWS = 16  # up to here a product needs no workspace, and the library need not be asked


def _product(x, w, w_up, activation, quantize_x, x_scale, out_dtype, out, stream):
    device = w.index
    _matrix("x", x, _DTYPES, w.k, device)
    m = x.shape[0]
    out = _out(out, m, w.n, out_dtype, x, device, stream)
    q = 1 if quantize_x else 0
    n_ws = 0
    if m > _SMALL_ROWS:
        need = w.lib.aex_fp4_mm_workspace_bytes if w_up is None else w.lib.aex_fp4_gated_mm_workspace_bytes
        n_ws = need(w.handle, m, q)
    ws = _empty((n_ws,), torch.uint8, x, stream) if n_ws else None
    a = _lib.aex_fp4_mm_args(x.data_ptr(), _DTYPES[x.dtype], x.stride(0) if m > 1 else w.k, m, q, x_scale, out.data_ptr(),
                             _DTYPES[out.dtype], out.stride(0) if m > 1 else w.n, ws.data_ptr() if n_ws else None,
                             n_ws)
    if w_up is None:
        rc = w.lib.aex_fp4_mm(w.ctx.handle, w.handle, a, _stream(stream, device))
    else:
        rc = w.lib.aex_fp4_gated_mm(w.ctx.handle, w.handle, w_up.handle, activation, a, _stream(stream, device))
    if stream is not None:
        _used(stream, x, out)
    if rc:
        w.ctx.check(rc)
    return out


def fp4_mm(x, w: FP4Weight, quantize_x=False, x_scale=1.0, out_dtype=torch.bfloat16, out=None, stream=None):
    """y[m, n] = x[m, k] . W[n, k]^T, f32 sums, rounded once to bf16 or f32. x is bf16, or f32 for m <= 16
    (each value held to within 2^-23 of itself).
    With quantize_x, x (bf16 or f32, any m) goes through :func:`quantize`'s rounding in the weight's
    mode first, with x_scale as its tensor scale, and both operands are multiplied in 4 bits. f32
    results of more than 16 rows carry the tensor core's truncating f32 sums (about 1e-5 of their
    size at k = 9216, as the affine linears' do)."""
    _open(w)
    return _product(x, w, None, 0, quantize_x, x_scale, out_dtype, out, stream)


def fp4_gated_mm(x, w_gate: FP4Weight, w_up: FP4Weight, activation="silu", quantize_x=False, x_scale=1.0,
                 out_dtype=torch.bfloat16, out=None, stream=None):
    """h[m, n] = act(x . Wg^T) * (x . Wu^T): both projections, the activation ("silu" or "gelu_tanh") and
    their product fused, rounded once. x, quantize_x and x_scale as :func:`fp4_mm`."""
    _open(w_gate, w_up)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    return _product(x, w_gate, w_up, act, quantize_x, x_scale, out_dtype, out, stream)


def fp4_mm_dgrad(dy, w: FP4Weight, out_dtype=torch.bfloat16, out=None, stream=None):
    """dx[m, k] = dy[m, n] . W[n, k], the gradient of :func:`fp4_mm` (without quantize_x); dy bf16, of any
    pitch where n is no multiple of 8 (:func:`fp4_mm`'s own results, say)."""
    _open(w)
    _matrix("dy", dy, _BF16, w.n, w.index)
    m = dy.shape[0]
    out = _out(out, m, w.k, out_dtype, dy, w.index, stream)
    n_ws = w.lib.aex_fp4_mm_dgrad_workspace_bytes(w.handle, m)
    ws = _empty((n_ws,), torch.uint8, dy, stream) if n_ws else None
    rc = w.lib.aex_fp4_mm_dgrad(w.ctx.handle, w.handle, dy.data_ptr(), _pitch(dy), m, out.data_ptr(),
                                _DTYPES[out.dtype], out.stride(0) if m > 1 else w.k, ws.data_ptr() if n_ws else None,
                                n_ws, _stream(stream, w.index))
    if stream is not None:
        _used(stream, dy, out)
    if rc:
        w.ctx.check(rc)
    return out


def fp4_gated_mm_dgrad(dh, x, w_gate: FP4Weight, w_up: FP4Weight, activation="silu", out_dtype=torch.bfloat16,
                       out=None, stream=None):
    """dx[m, k] of :func:`fp4_gated_mm` (without quantize_x) from dh[m, n] and the forward pass's x; both
    bf16, dx bf16. The projections are computed again; nothing need be kept from the forward pass."""
    _open(w_gate, w_up)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}")
    w = w_gate
    _matrix("x", x, _BF16, w.k, w.index)
    _matrix("dh", dh, _BF16, w.n, w.index)
    m = x.shape[0]
    if dh.shape[0] != m:
        raise ValueError("dh and x must have the same number of rows")
    if (out.dtype if out is not None else out_dtype) != torch.bfloat16:
        raise TypeError("the gradient is bfloat16")
    out = _out(out, m, w.k, out_dtype, x, w.index, stream)
    n_ws = w.lib.aex_fp4_gated_mm_dgrad_workspace_bytes(w.handle, m)
    ws = _empty((n_ws,), torch.uint8, x, stream)
    rc = w.lib.aex_fp4_gated_mm_dgrad(w.ctx.handle, w.handle, w_up.handle, act, x.data_ptr(), _pitch(x),
                                      dh.data_ptr(), _pitch(dh), m, out.data_ptr(),
                                      out.stride(0) if m > 1 else w.k, ws.data_ptr(), n_ws,
                                      _stream(stream, w.index))
    if stream is not None:
        _used(stream, x, dh, out)
    if rc:
        w.ctx.check(rc)
    return out
