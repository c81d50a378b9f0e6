"""The microscaled 4-bit operators against float64 (oracle/fp4_ref.py).

Tolerances. A rounding to bf16 is off by at most 2^-8 of the value, to f32 by 2^-24. A product's
f32 sums on the tensor cores truncate: every one of the accumulation steps (K/16, or K/64 for two
4-bit operands; 16 for each 256 columns in the few-rows kernel, which adds those in f32) can lose
a unit of the last place of a partial sum, which no partial sum's terms' magnitudes S = sum |x w|
exceed, and aligning the terms of a step the same again: at most (steps + 8) 2^-22 S."""
import ctypes as C

import numpy as np
import pytest
import torch

from aestrix_b200 import _lib, fp4
from oracle import fp4_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
MODES = ["mxfp4", "nvfp4"]


def f64(t):
    return t.detach().double().cpu().numpy()


def activations(m, k, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * (1.0 + 7.0 * (torch.rand(k, generator=g) < 0.02))
    return x.to(dtype).cuda()


def make_weight(n, k, mode, seed, tensor_scale=None):
    """(FP4Weight, float64 values): random codes and scales, as a pack may hold them."""
    g = np.random.default_rng(seed)
    codes = g.integers(0, 16, (n, k)).astype(np.uint8)
    if mode == "mxfp4":
        scales, ts = g.integers(115, 124, (n, k // 32)).astype(np.uint8), 1.0
    else:
        scales, ts = g.integers(8, 126, (n, k // 16)).astype(np.uint8), np.float32(tensor_scale or 0.0007)
    w = fp4.FP4Weight(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), mode,
                      tensor_scale=float(ts))
    return w, R.values(codes, scales, mode, ts)


def close(got, ref, bound, what=""):
    got = f64(got) if isinstance(got, torch.Tensor) else got
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - ref) - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"{what} at {at}: got {got[at]!r}, exact {ref[at]!r}, allowed {bound[at]:.3e}"


def sum_bound(x, w, steps):
    return (steps + 8) * 2.0**-22 * (np.abs(x) @ np.abs(w).T)


def steps_of(m, k, quantized):
    if m <= 16:
        return 16 + -(-k // 256) + 3
    return -(-k // 256) * (4 if quantized else 16)


# --------------------------------------------------------------------------- quantize, dequantize

@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k", [(1, 32), (1, 4096), (3, 96), (77, 1120), (130, 256), (257, 544)])
def test_quantize_codes_and_scales_are_exact(cuda_ctx, mode, dtype, m, k):
    x = activations(m, k, m * 1000 + k, DT[dtype])
    ts = float(np.float32(f64(x.abs().max()) / (448 * 6) * 1.1)) if mode == "nvfp4" else 1.0
    codes, scales = fp4.quantize(x, mode, tensor_scale=ts)
    ref_codes, ref_scales = R.quantize(f64(x), mode, ts)
    assert np.array_equal(scales.cpu().numpy(), ref_scales)
    assert np.array_equal(codes.cpu().numpy(), R.pack(ref_codes))
    ref = R.values(ref_codes, ref_scales, mode, ts)
    for out in (torch.bfloat16, torch.float32):
        close(fp4.dequantize(codes, scales, mode, tensor_scale=ts, out_dtype=out), ref, HALF[out] * np.abs(ref))


def border_rows(mode, ts, n):
    """f32 blocks whose elements lie on the borders of codes, one step to either side, and beyond 6."""
    g = np.random.default_rng(7)
    rows = []
    for _ in range(n):
        if mode == "mxfp4":
            unit = 2.0 ** g.integers(-120, 120)
        else:
            unit = R.E4M3[g.integers(1, 127)] * ts
        borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
        v = np.float32(np.concatenate([borders, borders]) * unit)
        v[g.random(16) < 0.3] *= -1
        way = g.integers(-1, 2, 16)
        v = np.where(way > 0, np.nextafter(v, np.float32(np.inf)), np.where(way < 0, np.nextafter(v, np.float32(0)), v))
        v[7] = np.float32(6.0 * unit)
        rows.append(np.concatenate([v] * (R.BLOCK[mode] // 16)))
    return np.stack(rows).astype(np.float32)


@pytest.mark.parametrize("mode,ts", [("mxfp4", 1.0), ("nvfp4", 1.0), ("nvfp4", 0.000731), ("nvfp4", 1.9e-20)])
def test_quantize_on_the_borders(cuda_ctx, mode, ts):
    """Values on a border go to the even code, their neighbours to their own side, whatever the
    quotient rounds to in f32."""
    ts = float(np.float32(ts))
    x = np.concatenate([border_rows(mode, ts, 512)] * (32 // R.BLOCK[mode]), 1)
    codes, scales = fp4.quantize(torch.from_numpy(x).cuda(), mode, tensor_scale=ts)
    ref_codes, ref_scales = R.quantize(x, mode, ts)
    assert np.array_equal(scales.cpu().numpy(), ref_scales)
    assert np.array_equal(codes.cpu().numpy(), R.pack(ref_codes))


@pytest.mark.parametrize("ts", [1.0, 0.00137])
def test_quantize_scale_borders(cuda_ctx, ts):
    """Largest magnitudes half-way between two e4m3 scales (and one f32 step beside it), below the
    smallest scale and above the largest."""
    ts = float(np.float32(ts))
    mids = (R.E4M3[:-1] + R.E4M3[1:]) / 2
    top = np.concatenate([mids, R.E4M3, [480.0, 1e4, 1e-4, 2.0**-10, 2.0**-11]]) * 6.0 * ts
    top = np.float32(top)
    top = np.concatenate([top, np.nextafter(top, np.float32(np.inf)), np.nextafter(top, np.float32(0))])
    x = np.zeros((len(top), 32), np.float32)
    x[:, 5] = top
    x[:, 21] = -top
    x[:, 9] = top / 3
    codes, scales = fp4.quantize(torch.from_numpy(x).cuda(), "nvfp4", tensor_scale=ts)
    ref_codes, ref_scales = R.quantize(x, "nvfp4", ts)
    assert np.array_equal(scales.cpu().numpy(), ref_scales)
    assert np.array_equal(codes.cpu().numpy(), R.pack(ref_codes))


@pytest.mark.parametrize("mode", MODES)
def test_quantize_extreme_values(cuda_ctx, mode):
    """Zero blocks, subnormals, the largest f32, and blocks that hold an infinity or NaN: a NaN scale,
    and only theirs."""
    x = np.zeros((8, 64), np.float32)
    x[1, 3] = 1e-45
    x[2, 40] = -3e-39
    x[3, :] = np.finfo(np.float32).max
    x[4, 33] = np.inf
    x[5, 2] = np.nan
    x[6, 10], x[6, 11] = 1e-30, 1e30
    x[7, :] = np.linspace(-6, 6, 64)
    codes, scales = fp4.quantize(torch.from_numpy(x).cuda(), mode)
    ref_codes, ref_scales = R.quantize(x, mode)
    assert np.array_equal(scales.cpu().numpy(), ref_scales)
    fine = np.isfinite(x).reshape(8, -1, R.BLOCK[mode]).all(-1).repeat(R.BLOCK[mode], 1)
    assert np.array_equal(R.unpack(codes.cpu().numpy())[fine], ref_codes[fine])
    back = f64(fp4.dequantize(codes, scales, mode, out_dtype=torch.float32))
    assert np.isnan(back[~fine]).all()
    assert np.array_equal(back[fine], R.values(ref_codes, ref_scales, mode)[fine])


def test_dequantize_rounds_once(cuda_ctx):
    """Every code and scale byte with a tensor scale of a full significand: bf16 is the nearest to
    the exact product, not to its f32."""
    codes = np.tile(np.arange(16, dtype=np.uint8), (127, 2))
    scales = np.repeat(np.arange(127, dtype=np.uint8)[:, None], 2, 1)
    for ts in (1.0, float(np.float32(0.1)), float(np.float32(1.0000001)), float(np.float32(7.3e-11))):
        got = fp4.dequantize(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), "nvfp4",
                             tensor_scale=ts)
        ref = R.values(codes, scales, "nvfp4", ts)
        # round to nearest even on the bf16 grid, in integers of 2^(e - 7)
        _, e = np.frexp(ref)
        step = np.ldexp(1.0, e - 8)
        assert np.array_equal(f64(got), np.where(ref == 0, 0.0, np.round(ref / step) * step))


def test_quantize_strided_rows(cuda_ctx):
    base = activations(40, 512, 3)
    view = base[::2, 64:320]
    a, b = fp4.quantize(view, "mxfp4"), fp4.quantize(view.contiguous(), "mxfp4")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("n,k", [(1, 32), (128, 256), (129, 288), (300, 1120)])
def test_weight_layout_round_trip(cuda_ctx, mode, n, k):
    w, ref = make_weight(n, k, mode, n + k)
    got = w.dequantize(torch.float32)
    close(got, ref, 2.0**-24 * np.abs(ref))


# ------------------------------------------------------------------------------------- products

SHAPES = [(1, 256, 512), (1, 40, 32), (2, 129, 96), (8, 1000, 1120), (9, 128, 4096), (16, 257, 2080),
          (17, 256, 256), (77, 384, 544), (128, 129, 512), (129, 1000, 768), (257, 513, 1120), (600, 40, 4096)]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_mm(cuda_ctx, mode, out, m, n, k):
    x = activations(m, k, m + n + k)
    w, ref_w = make_weight(n, k, mode, n * 3 + k)
    ref = f64(x) @ ref_w.T
    y = fp4.fp4_mm(x, w, out_dtype=DT[out])
    cuda_ctx.sync()
    close(y, ref, HALF[DT[out]] * np.abs(ref) + sum_bound(f64(x), ref_w, steps_of(m, k, False)))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m", [1, 2, 3, 5, 6, 16])
def test_mm_f32_rows(cuda_ctx, mode, m):
    """f32 activations count to within 2^-23 of themselves."""
    n, k = 300, 4512
    x = activations(m, k, m, torch.float32) * 1.000123
    w, ref_w = make_weight(n, k, mode, m)
    ref = f64(x) @ ref_w.T
    y = fp4.fp4_mm(x, w, out_dtype=torch.float32)
    close(y, ref, 2.0**-24 * np.abs(ref) + sum_bound(f64(x), ref_w, steps_of(m, k, False)))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_mm_quantized(cuda_ctx, mode, dtype, m, n, k):
    x = activations(m, k, m + n + k, DT[dtype])
    ts = float(np.float32(f64(x.abs().max()) / (448 * 6))) if mode == "nvfp4" else 1.0
    w, ref_w = make_weight(n, k, mode, n * 3 + k)
    xq = R.values(*R.quantize(f64(x), mode, ts), mode, ts)
    ref = xq @ ref_w.T
    y = fp4.fp4_mm(x, w, quantize_x=True, x_scale=ts)
    cuda_ctx.sync()
    close(y, ref, 2.0**-8 * np.abs(ref) + sum_bound(xq, ref_w, steps_of(m, k, True)))


def gated_bound(x, wg, wu, act, steps, half):
    """|h - exact|: the sums' errors through act (slope at most 1.2) and the product, the fast
    exponential's (2 + 1.2 |z|) 2^-23, the rounding."""
    g, u = x @ wg.T, x @ wu.T
    a, _ = R.act(g, act)
    h = a * u
    eg, eu = sum_bound(x, wg, steps), sum_bound(x, wu, steps)
    z = np.minimum(np.abs(g) if act == "silu" else 1.6 * np.abs(g + 0.045 * g**3), 90.0)
    bound = 1.2 * np.abs(u) * eg + np.abs(a) * eu + 1.2 * eg * eu
    return h, bound + ((6 + 1.2 * z) * 2.0**-23 + half) * np.abs(h) + 2.0**-126


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("quantize_x", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (3, 129, 96), (16, 300, 2080), (17, 128, 256), (130, 257, 544),
                                   (300, 40, 1120)])
def test_gated(cuda_ctx, mode, act, quantize_x, m, n, k):
    x = activations(m, k, m + n + k)
    ts = float(np.float32(f64(x.abs().max()) / (448 * 6))) if mode == "nvfp4" else 1.0
    wg, rg = make_weight(n, k, mode, 1, 0.00011)
    wu, ru = make_weight(n, k, mode, 2, 0.00037)
    xr = R.values(*R.quantize(f64(x), mode, ts), mode, ts) if quantize_x else f64(x)
    for out in (torch.bfloat16, torch.float32):
        y = fp4.fp4_gated_mm(x, wg, wu, activation=act, quantize_x=quantize_x, x_scale=ts, out_dtype=out)
        cuda_ctx.sync()
        ref, bound = gated_bound(xr, rg, ru, act, steps_of(m, k, quantize_x), HALF[out])
        close(y, ref, bound, f"{out}")


def test_gated_f32_rows(cuda_ctx):
    m, n, k = 5, 200, 1120
    x = activations(m, k, 5, torch.float32) * 0.999871
    wg, rg = make_weight(n, k, "nvfp4", 1, 0.00011)
    wu, ru = make_weight(n, k, "nvfp4", 2, 0.00037)
    y = fp4.fp4_gated_mm(x, wg, wu, out_dtype=torch.float32)
    ref, bound = gated_bound(f64(x), rg, ru, "silu", steps_of(m, k, False), 2.0**-24)
    close(y, ref, bound)


# ------------------------------------------------------------------------------------- gradients

@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (1, 256, 512), (16, 136, 288), (77, 384, 544), (257, 520, 1120),
                                   (130, 1000, 256)])
def test_mm_dgrad(cuda_ctx, mode, out, m, n, k):
    dy = activations(m, n, m + n)
    w, ref_w = make_weight(n, k, mode, n + k)
    ref = f64(dy) @ ref_w
    dx = fp4.fp4_mm_dgrad(dy, w, out_dtype=DT[out])
    cuda_ctx.sync()
    close(dx, ref, HALF[DT[out]] * np.abs(ref) + sum_bound(f64(dy), ref_w.T, -(-n // 128) * 8))


def gated_grad_ref(x, dh, rg, ru, act):
    g, u = x @ rg.T, x @ ru.T
    a, slope = R.act(g, act)
    return dh * u * slope, dh * a, g, u, a, slope


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (5, 256, 512), (77, 264, 544), (130, 1000, 288), (300, 128, 1120)])
def test_gated_dgrad(cuda_ctx, mode, act, m, n, k):
    x, dh = activations(m, k, m + k), activations(m, n, m + n + 1)
    wg, rg = make_weight(n, k, mode, 1, 0.00011)
    wu, ru = make_weight(n, k, mode, 2, 0.00037)
    X, D = f64(x), f64(dh)
    dg, du, g, u, a, slope = gated_grad_ref(X, D, rg, ru, act)
    steps = -(-k // 256) * 16
    eg, eu = sum_bound(X, rg, steps), sum_bound(X, ru, steps)
    # act'' is at most 1.2 in magnitude; 2^-18 covers the fast exponential; dg and du are rounded to bf16
    e_dg = (2.0**-8 + 2.0**-18) * np.abs(dg) + np.abs(D) * (np.abs(slope) * eu + 1.2 * np.abs(u) * eg) * 1.01 \
        + 2.0**-18 * np.abs(D * u)
    e_du = (2.0**-8 + 2.0**-18) * np.abs(du) + 1.2 * np.abs(D) * eg * 1.01
    ref = dg @ rg + du @ ru
    n_steps = 2 * -(-n // 128) * 8
    bound = e_dg @ np.abs(rg) + e_du @ np.abs(ru) + 2.0**-8 * np.abs(ref) \
        + (n_steps + 8) * 2.0**-22 * 1.01 * (np.abs(dg) @ np.abs(rg) + np.abs(du) @ np.abs(ru))
    dx = fp4.fp4_gated_mm_dgrad(dh, x, wg, wu, activation=act)
    cuda_ctx.sync()
    close(dx, ref, bound)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gated_dgrad_against_differences(cuda_ctx, act):
    """The gradient along directions against central differences of the float64 forward pass: the
    formula itself, not only its evaluation."""
    m, n, k = 6, 64, 96
    x, dh = activations(m, k, 1), activations(m, n, 2)
    wg, rg = make_weight(n, k, "nvfp4", 1, 0.00011)
    wu, ru = make_weight(n, k, "nvfp4", 2, 0.00037)
    X, D = f64(x), f64(dh)

    def loss(v):
        return (R.act(v @ rg.T, act)[0] * (v @ ru.T) * D).sum(1)

    dx = f64(fp4.fp4_gated_mm_dgrad(dh, x, wg, wu, activation=act))
    rng = np.random.default_rng(0)
    dg, du, *_ = gated_grad_ref(X, D, rg, ru, act)
    size = np.abs(dg) @ np.abs(rg) + np.abs(du) @ np.abs(ru)
    for _ in range(4):
        d = rng.standard_normal(k)
        h = 1e-4
        slope = (loss(X + h * d) - loss(X - h * d)) / (2 * h)
        # dg, du and dx are rounded to bf16 (2^-8 each of what they sum); the difference is good to h^2
        assert (np.abs(dx @ d - slope) <= 2.1 * 2.0**-8 * (size @ np.abs(d)) + 1e-6).all()


# ---------------------------------------------------------------------------------- repeatability

@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", [(1, 2048, 7680), (16, 1000, 4096), (257, 2048, 7680), (1024, 1024, 4096)])
def test_same_bits_every_time(cuda_ctx, mode, m, n, k):
    """No sum depends on which warp or CTA is first, and no slot of a ring is filled again before it is
    read: every one of many calls in a row, queued without a gap, gives the same bits."""
    x, dh = activations(m, k, 1), activations(m, n, 2)
    wg, _ = make_weight(n, k, mode, 1, 0.00011)
    wu, _ = make_weight(n, k, mode, 2, 0.00037)
    calls = {
        "mm": lambda: fp4.fp4_mm(x, wg),
        "gated": lambda: fp4.fp4_gated_mm(x, wg, wu),
        "quantized": lambda: fp4.fp4_mm(x, wg, quantize_x=True),
        "gated quantized": lambda: fp4.fp4_gated_mm(x, wg, wu, quantize_x=True),
        "dgrad": lambda: fp4.fp4_mm_dgrad(dh, wg),
        "gated dgrad": lambda: fp4.fp4_gated_mm_dgrad(dh, x, wg, wu),
    }
    for name, call in calls.items():
        first = call()
        differ = torch.zeros((), dtype=torch.int64, device="cuda")
        for _ in range(100):
            differ += (call() != first).sum()
        assert differ.item() == 0, name


# ------------------------------------------------------------- values that need care

def wide_rows(m, k, seed):
    """f32 rows whose 256-column stretches span more binades than f16 holds: huge and tiny values side by
    side, the huge ones where it matters next to zeros."""
    g = np.random.default_rng(seed)
    x = g.standard_normal((m, k)) * np.ldexp(1.0, g.integers(-60, 60, (m, k)))
    x[:, ::5] = 0.0
    return torch.from_numpy(x.astype(np.float32))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k", [(1, 512), (3, 1120), (7, 2048), (16, 544)])
def test_few_rows_wide_range(cuda_ctx, mode, dtype, m, k):
    """The few-rows kernel's f16 staging does not hold these; every element still counts in full: the
    tolerance is that of the f32 sums, and a row whose large values meet zero weights keeps its small
    ones."""
    x = wide_rows(m, k, m + k).to(DT[dtype]).cuda()
    w, ref_w = make_weight(136, k, mode, k)
    y = fp4.fp4_mm(x, w, out_dtype=torch.float32)
    close(y, f64(x) @ ref_w.T, 2.0**-24 * np.abs(f64(x) @ ref_w.T) + sum_bound(f64(x), ref_w, steps_of(m, k, False)))
    # one huge value against a weight column of zeros, tiny ones elsewhere
    codes = np.ones((130, k), np.uint8)  # 0.5
    codes[:, 7] = 0
    scales = np.full((130, k // R.BLOCK[mode]), 127 if mode == "mxfp4" else 56, np.uint8)  # 1.0
    w = fp4.FP4Weight(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), mode)
    x = torch.full((m, k), 2.0**-40, dtype=DT[dtype], device="cuda")
    x[:, 7] = 2.0**100
    y = fp4.fp4_mm(x, w, out_dtype=torch.float32)
    ref = (k - 1) * 2.0**-41
    assert np.abs(f64(y) - ref).max() <= ref * (steps_of(m, k, False) + 8) * 2.0**-22


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m", [2, 20, 40, 300])
@pytest.mark.parametrize("quantize_x", [False, True])
def test_infinities_and_nan_stay_where_they_are(cuda_ctx, mode, m, quantize_x):
    """A row that holds an infinity or NaN, and a weight row with a NaN scale, spoil their own outputs
    only. Without quantization an infinity gives infinities of the right sign."""
    k, n = 544, 264
    x = activations(m, k, 3)
    g = np.random.default_rng(5)
    codes = g.integers(1, 8, (n, k)).astype(np.uint8)  # positive, none zero
    scales = np.full((n, k // R.BLOCK[mode]), 120 if mode == "mxfp4" else 40, np.uint8)
    scales[100, 3] = 255 if mode == "mxfp4" else 127
    w = fp4.FP4Weight(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), mode)
    clean = fp4.fp4_mm(x, w, quantize_x=quantize_x, x_scale=1.0)
    assert torch.isnan(clean[:, 100]).all() and torch.isfinite(clean[:, :100]).all()
    assert torch.isfinite(clean[:, 101:]).all()
    y = x.clone()
    y[0, 17] = float("-inf")
    y[m - 1, 300] = float("nan")
    got = fp4.fp4_mm(y, w, quantize_x=quantize_x, x_scale=1.0)
    keep = [c for c in range(n) if c != 100]
    assert torch.equal(got[1:m - 1, keep], clean[1:m - 1, keep])
    assert torch.isnan(got[m - 1]).all()
    if quantize_x:
        assert torch.isnan(got[0]).all()
    else:
        assert (got[0, keep] == float("-inf")).all()


def test_mx_scale_extremes(cuda_ctx):
    """mxfp4 scale bytes from 0 (2^-127) to 250, in every kernel: the value is code * 2^(byte - 127)."""
    n, k = 272, 256
    g = np.random.default_rng(9)
    codes = g.integers(0, 16, (n, k)).astype(np.uint8)
    scales = np.repeat(np.linspace(0, 250, n).astype(np.uint8)[:, None], k // 32, 1)
    w = fp4.FP4Weight(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), "mxfp4")
    ref_w = R.values(codes, scales, "mxfp4")
    for m in (3, 20, 50):
        x = (activations(m, k, m).float() * 2.0**-10).to(torch.bfloat16)
        y = fp4.fp4_mm(x, w, out_dtype=torch.float32)
        ref = f64(x) @ ref_w.T
        fits = np.abs(ref) < 1e38
        # products below the smallest normal f32 may be flushed by the tensor cores: k of them a sum
        bound = 2.0**-24 * np.abs(ref) + sum_bound(f64(x), ref_w, steps_of(m, k, False)) + k * 2.0**-125
        assert (np.abs(f64(y) - ref)[fits] <= bound[fits]).all()


def test_zero_rows_and_zero_weights(cuda_ctx):
    for m in (1, 9, 40, 200):
        x = activations(m, 544, 1)
        x[0] = 0
        codes, scales = np.zeros((136, 544), np.uint8), np.zeros((136, 34), np.uint8)
        w = fp4.FP4Weight(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), "nvfp4")
        assert not fp4.fp4_mm(x, w).any()
        w, _ = make_weight(136, 544, "nvfp4", 1)
        for q in (False, True):
            assert not fp4.fp4_mm(x, w, quantize_x=q, x_scale=0.01)[0].any()


# -------------------------------------------------------- layouts, streams, graphs, long inputs

@pytest.mark.parametrize("m", [5, 20, 150])
@pytest.mark.parametrize("offset,pitch", [(0, 264), (1, 263), (3, 257), (8, 304), (16, 272)])
def test_output_pitch_and_surroundings(cuda_ctx, m, offset, pitch):
    """Any pitch and element-aligned start of the result; what lies around it is left as it was."""
    n, k = 257, 288
    x = activations(m, k, 2)
    w, _ = make_weight(n, k, "nvfp4", 3)
    for dtype in (torch.bfloat16, torch.float32):
        for q in (False, True):
            want = fp4.fp4_mm(x, w, quantize_x=q, x_scale=0.02, out_dtype=dtype)
            buf = torch.full(((m + 2) * pitch + offset + n,), 7.0, dtype=dtype, device="cuda")
            out = buf[offset:].as_strided((m, n), (pitch, 1))
            fp4.fp4_mm(x, w, quantize_x=q, x_scale=0.02, out=out)
            assert torch.equal(out, want)
            mask = torch.ones_like(buf, dtype=torch.bool)
            mask[offset:].as_strided((m, n), (pitch, 1)).fill_(False)
            assert (buf[mask] == 7.0).all()
            want = fp4.fp4_gated_mm(x, w, w, quantize_x=q, x_scale=0.02, out_dtype=dtype)
            fp4.fp4_gated_mm(x, w, w, quantize_x=q, x_scale=0.02, out=out)
            assert torch.equal(out, want) and (buf[mask] == 7.0).all()


@pytest.mark.parametrize("m", [4, 24, 140])
def test_input_pitch_and_start(cuda_ctx, m):
    """Rows of a wider tensor, starting 16 (not 32) bytes into it."""
    n, k = 136, 288
    base = activations(m, 512, 4)
    x = base[:, 8:8 + k]
    w, _ = make_weight(n, k, "mxfp4", 3)
    for q in (False, True):
        assert torch.equal(fp4.fp4_mm(x, w, quantize_x=q), fp4.fp4_mm(x.contiguous(), w, quantize_x=q))
    dy = base[:, 8:8 + n]
    assert torch.equal(fp4.fp4_mm_dgrad(dy, w), fp4.fp4_mm_dgrad(dy.contiguous(), w))
    a = fp4.fp4_gated_mm_dgrad(dy, x, w, w)
    assert torch.equal(a, fp4.fp4_gated_mm_dgrad(dy.contiguous(), x.contiguous(), w, w))


@pytest.mark.parametrize("m,n,k,dtype", [(2, 20000, 9216, "bf16"), (16, 130, 24576, "f32"), (32, 1000, 9216, "bf16"),
                                         (13, 5000, 7680, "f32")])
def test_few_rows_long_columns(cuda_ctx, m, n, k, dtype):
    """More columns than a CTA stages at once."""
    x = activations(m, k, 6, DT[dtype])
    w, ref_w = make_weight(n, k, "nvfp4", 8)
    y = fp4.fp4_mm(x, w, out_dtype=torch.float32)
    ref = f64(x) @ ref_w.T
    close(y, ref, 2.0**-24 * np.abs(ref) + sum_bound(f64(x), ref_w, 19 + k // 256))


def test_more_than_2_to_31_elements(cuda_ctx):
    """Offsets past 32 bits: the last rows of a matrix of 2.2 billion elements, against the same rows alone."""
    m, k = 270000, 8192
    x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    x.normal_()
    codes, scales = fp4.quantize(x, "nvfp4", tensor_scale=0.002)
    tail = x[-300:].clone()
    c, s = fp4.quantize(tail, "nvfp4", tensor_scale=0.002)
    assert torch.equal(codes[-300:], c) and torch.equal(scales[-300:], s)
    back = fp4.dequantize(codes, scales, "nvfp4", tensor_scale=0.002)
    assert torch.equal(back[-300:], fp4.dequantize(c, s, "nvfp4", tensor_scale=0.002))
    del back, codes, scales
    w, _ = make_weight(40, k, "nvfp4", 1)
    # tiles are summed whole or in pieces by their number: the f32 sums may differ by their rounding
    for q in (False, True):
        a = fp4.fp4_mm(x, w, quantize_x=q, x_scale=0.002)[-300:].float()
        b = fp4.fp4_mm(tail, w, quantize_x=q, x_scale=0.002).float()
        assert (a - b).abs().max() <= 2.0**-7 * b.abs().max()
    dx = fp4.fp4_mm_dgrad(x[:, :40], w)[-300:].float()
    ref = fp4.fp4_mm_dgrad(tail[:, :40], w).float()
    assert (dx - ref).abs().max() <= 2.0**-7 * ref.abs().max()


def feed_forward(x, ws, quantize_x, scale):
    """The block as a transformer runs it: gated projection, then down."""
    h = fp4.fp4_gated_mm(x, ws["gate"], ws["up"], quantize_x=quantize_x, x_scale=scale)
    return h, fp4.fp4_mm(h, ws["down"], quantize_x=quantize_x, x_scale=scale)


def feed_forward_weights(hidden, width, mode):
    out, ref = {}, {}
    for i, (name, n, k) in enumerate((("gate", width, hidden), ("up", width, hidden), ("down", hidden, width))):
        out[name], ref[name] = make_weight(n, k, mode, 11 + i, 0.0002)
    return out, ref


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m", [1, 20, 150])
def test_feed_forward_and_its_gradient(cuda_ctx, mode, m):
    """The operators as they are used together: forward through the gated block and down, the gradient
    back through both, against float64 with h rounded to bf16 between (as it is handed over)."""
    hidden, width = 512, 1120
    ws, ref = feed_forward_weights(hidden, width, mode)
    x, dy = activations(m, hidden, 1), activations(m, hidden, 2)
    h, y = feed_forward(x, ws, False, 1.0)
    want_h, bound_h = gated_bound(f64(x), ref["gate"], ref["up"], "silu", steps_of(m, hidden, False), 2.0**-8)
    close(h, want_h, bound_h)
    H = f64(h)
    want = H @ ref["down"].T
    close(y, want, 2.0**-8 * np.abs(want) + sum_bound(H, ref["down"], steps_of(m, width, False)))
    dh = fp4.fp4_mm_dgrad(dy, ws["down"])
    want = f64(dy) @ ref["down"]
    close(dh, want, 2.0**-8 * np.abs(want) + sum_bound(f64(dy), ref["down"].T, -(-hidden // 128) * 8))
    dx = fp4.fp4_gated_mm_dgrad(dh, x, ws["gate"], ws["up"])
    dg, du, *_ = gated_grad_ref(f64(x), f64(dh), ref["gate"], ref["up"], "silu")
    want = dg @ ref["gate"] + du @ ref["up"]
    size = np.abs(dg) @ np.abs(ref["gate"]) + np.abs(du) @ np.abs(ref["up"])
    close(dx, want, 2.0**-8 * np.abs(want) + 1.1 * 2.0**-8 * size)


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("quantize_x", [False, True])
def test_captured_and_replayed(cuda_ctx, m, quantize_x):
    """Two graphs of the block, replayed in turn and at once on two streams with new inputs: each has its
    own workspaces, and each replay reads what its input holds then."""
    hidden, width = 512, 2048
    ws, _ = feed_forward_weights(hidden, width, "nvfp4")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for s in (s1, s2):
        x = activations(m, hidden, 1)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            feed_forward(x, ws, quantize_x, 0.02)
            fp4.fp4_gated_mm_dgrad(torch.zeros(m, width, dtype=torch.bfloat16, device="cuda"), x, ws["gate"], ws["up"])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            h, y = feed_forward(x, ws, quantize_x, 0.02)
            dx = fp4.fp4_gated_mm_dgrad(h, x, ws["gate"], ws["up"])
        graphs.append((g, x, y, dx))
    for r in range(3):
        ins = [activations(m, hidden, 10 + 2 * r + i) for i in range(2)]
        want = []
        for x in ins:
            h, y = feed_forward(x, ws, quantize_x, 0.02)
            want.append((y, fp4.fp4_gated_mm_dgrad(h, x, ws["gate"], ws["up"])))
        for (g, x, _, _), new in zip(graphs, ins):
            x.copy_(new)
        torch.cuda.synchronize()
        for s, (g, *_rest) in zip((s1, s2), graphs):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for (g, x, y, dx), (wy, wdx) in zip(graphs, want):
            assert torch.equal(y, wy) and torch.equal(dx, wdx)
    assert cuda_ctx.device_status() == 0


@pytest.mark.parametrize("m", [3, 60, 260])
def test_given_stream_and_two_streams_at_once(cuda_ctx, m):
    """The stream argument is the one the kernels run on; calls on two streams that share a weight do not
    touch one another's scratch."""
    n, k = 1000, 2080
    w, _ = make_weight(n, k, "mxfp4", 1)
    xs = [activations(m, k, i) for i in range(2)]
    want = [[fp4.fp4_mm(x, w), fp4.fp4_mm(x, w, quantize_x=True), fp4.quantize(x, "mxfp4")[0]] for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            got[i].append([fp4.fp4_mm(xs[i], w, stream=s), fp4.fp4_mm(xs[i], w, quantize_x=True, stream=s),
                           fp4.quantize(xs[i], "mxfp4", stream=s)[0]])
    torch.cuda.synchronize()
    for i in range(2):
        for row in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(row, want[i]))


def test_current_device_is_left_alone(cuda_ctx):
    before = torch.cuda.current_device()
    w, _ = make_weight(40, 64, "mxfp4", 1)
    fp4.fp4_mm(activations(2, 64, 1), w)
    assert torch.cuda.current_device() == before


# ------------------------------------------------------------------------------------- refusals

def test_refusals(cuda_ctx):
    x = activations(40, 288, 1)
    w, _ = make_weight(136, 288, "mxfp4", 1)
    v, _ = make_weight(136, 288, "nvfp4", 1)
    t, _ = make_weight(128, 288, "mxfp4", 1)
    E = _lib.AexError
    with pytest.raises(ValueError, match="columns"):
        fp4.fp4_mm(x[:, :256], w)
    with pytest.raises(E, match="multiple of 16 bytes"):
        fp4.fp4_mm(torch.empty(40, 292, dtype=torch.bfloat16, device="cuda")[:, :288], w)
    with pytest.raises(E, match="16-byte aligned"):
        fp4.fp4_mm(torch.empty(40, 296, dtype=torch.bfloat16, device="cuda")[:, 4:292], w)
    with pytest.raises(ValueError, match="contiguous rows"):
        fp4.fp4_mm(torch.empty(288, 40, dtype=torch.bfloat16, device="cuda").t(), w)
    with pytest.raises(TypeError):
        fp4.fp4_mm(x.half(), w)
    with pytest.raises(E, match="m <= 16"):
        fp4.fp4_mm(x.float(), w)
    with pytest.raises(E, match="no tensor scale"):
        fp4.fp4_mm(x, w, quantize_x=True, x_scale=0.5)
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-35):
        with pytest.raises(E, match="tensor_scale"):
            fp4.fp4_mm(x, v, quantize_x=True, x_scale=bad)
        with pytest.raises(E, match="tensor_scale"):
            fp4.quantize(x, "nvfp4", tensor_scale=bad)
    with pytest.raises(ValueError, match="multiple of 32"):
        fp4.quantize(x[:, :48], "mxfp4")
    with pytest.raises(ValueError, match="no rows"):
        fp4.fp4_mm(x[:0], w)
    with pytest.raises(TypeError, match="out_dtype"):
        fp4.fp4_mm(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="rows"):
        fp4.fp4_mm(x, w, out=torch.empty(39, 136, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(E, match="row pitch"):
        fp4.fp4_mm(x, w, out=torch.empty(1, 136, dtype=torch.bfloat16, device="cuda").expand(40, 136))
    for other in (v, t):
        with pytest.raises(E, match="one shape and format"):
            fp4.fp4_gated_mm(x, w, other)
    with pytest.raises(ValueError, match="activation"):
        fp4.fp4_gated_mm(x, w, w, activation="relu")
    with pytest.raises(TypeError):
        fp4.fp4_mm_dgrad(x.float()[:, :136], w)
    with pytest.raises(ValueError, match="same number of rows"):
        fp4.fp4_gated_mm_dgrad(x[:39, :136].contiguous(), x, w, w)
    with pytest.raises(TypeError, match="bfloat16"):
        fp4.fp4_gated_mm_dgrad(x[:, :136].contiguous(), x, w, w, out_dtype=torch.float32)
    codes, scales = fp4.quantize(x, "mxfp4")
    with pytest.raises(ValueError, match="scales"):
        fp4.FP4Weight(codes, scales, "nvfp4")
    with pytest.raises(ValueError, match="contiguous"):
        fp4.FP4Weight(codes.t().contiguous().t(), scales, "mxfp4")
    w.close()
    with pytest.raises(ValueError, match="closed"):
        fp4.fp4_mm(x, w)
    # the workspace of the C call: too small, misaligned, missing
    a = _lib.aex_fp4_mm_args()
    y = torch.empty(40, 136, dtype=torch.bfloat16, device="cuda")
    a.x, a.x_dtype, a.ldx, a.m = x.data_ptr(), _lib.AEX_DTYPE_BF16, 288, 40
    a.quantize_x, a.x_scale, a.y, a.y_dtype, a.ldy = 1, 1.0, y.data_ptr(), _lib.AEX_DTYPE_BF16, 136
    L = _lib.lib()
    need = L.aex_fp4_mm_workspace_bytes(v.handle, 40, 1)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    for p, n in ((None, 0), (ws.data_ptr(), need - 1), (ws.data_ptr() + 16, need)):
        a.workspace, a.workspace_bytes = p, n
        assert L.aex_fp4_mm(cuda_ctx.handle, v.handle, a, None) == _lib.AEX_ERR_INVALID_ARG
        assert b"workspace" in L.aex_last_error_string(cuda_ctx.handle)
    for field, value in (("quantize_x", 2), ("m", 0), ("y_dtype", 5), ("x_dtype", -1)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert L.aex_fp4_mm(cuda_ctx.handle, v.handle, a, None) == _lib.AEX_ERR_INVALID_ARG
        setattr(a, field, old)
    assert cuda_ctx.device_status() == 0


def test_refuses_what_32_bits_do_not_count(cuda_ctx):
    w, _ = make_weight(128, 288, "mxfp4", 1)
    row = torch.zeros(1, 288, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="2147483647"):
        fp4.fp4_mm(row.expand(2**32 + 1, 288), w)
    with pytest.raises(ValueError, match="2147483647"):
        fp4.quantize(row.expand(2**31, 288), "mxfp4")
    codes = torch.zeros(1, 16, dtype=torch.uint8, device="cuda").expand(2**32 + 128, 16)
    scales = torch.zeros(1, 1, dtype=torch.uint8, device="cuda").expand(2**32 + 128, 1)
    with pytest.raises(ValueError, match="2147483647"):
        fp4.FP4Weight(codes, scales, "mxfp4")


def test_refuses_another_devices_context(cuda_ctx):
    class Other:
        device = 1

    x = activations(3, 64, 1)
    with pytest.raises(ValueError, match="context on cuda:1"):
        fp4.quantize(x, "mxfp4", ctx=Other())
    codes, scales = fp4.quantize(x, "mxfp4")
    with pytest.raises(ValueError, match="context on cuda:1"):
        fp4.FP4Weight(codes, scales, "mxfp4", ctx=Other())


@pytest.mark.parametrize("m", [2, 40])
def test_refuses_tensor_scales_whose_product_leaves_f32(cuda_ctx, m):
    x = activations(m, 288, 1)
    for ts, xs in ((2.0**90, 2.0**90), (2.0**-90, 2.0**-90)):
        w, _ = make_weight(128, 288, "nvfp4", 1, ts)
        v, _ = make_weight(128, 288, "nvfp4", 1, 1.0)
        for call in (lambda: fp4.fp4_mm(x, w, quantize_x=True, x_scale=xs),
                     lambda: fp4.fp4_gated_mm(x, v, w, quantize_x=True, x_scale=xs)):
            with pytest.raises(_lib.AexError, match="normal f32"):
                call()
        fp4.fp4_mm(x, v, quantize_x=True, x_scale=xs)
    cuda_ctx.sync()


def test_a_weight_is_not_created_under_capture(cuda_ctx):
    x = activations(5, 288, 1)
    codes, scales = fp4.quantize(activations(64, 288, 2), "mxfp4")
    w = fp4.FP4Weight(codes, scales, "mxfp4")
    s = torch.cuda.Stream()
    fp4.fp4_mm(x, w, stream=s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        with pytest.raises(_lib.AexError, match="captured"):
            fp4.FP4Weight(codes, scales, "mxfp4")
        y = fp4.fp4_mm(x, w)  # the capture goes on
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, fp4.fp4_mm(x, w))


# ------------------------------------------------------------------- gates far out, tiles of many pieces

@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gated_dgrad_of_gates_far_out(cuda_ctx, mode, act):
    """Gates of 1e20 and more, whose squares leave f32: the slope is 1 on one side and 0 on the other.
    All terms have one sign, so the roundings bound the result relative to itself: dg and du (2^-8, and
    2^-18 for what they are computed from), dx (2^-8), the sums."""
    m, n, k = 4, 136, 96
    g = np.random.default_rng(3)
    pair = []
    for _ in range(2):
        codes = g.integers(1, 8, (n, k)).astype(np.uint8)  # positive, none zero
        scales = np.full((n, k // R.BLOCK[mode]), 124 if mode == "mxfp4" else 40, np.uint8)
        pair.append((fp4.FP4Weight(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), mode),
                     R.values(codes, scales, mode, 1.0)))
    (wg, rg), (wu, ru) = pair
    x = (torch.rand(m, k, generator=torch.Generator().manual_seed(1)) + 0.5).bfloat16().cuda() * 2.0**70
    x[m // 2:] *= -1
    dh = (torch.rand(m, n, generator=torch.Generator().manual_seed(2)) + 0.5).bfloat16().cuda() * 2.0**-40
    dx = f64(fp4.fp4_gated_mm_dgrad(dh, x, wg, wu, activation=act))
    X, D = f64(x)[:m // 2], f64(dh)[:m // 2]
    ref = (D * (X @ ru.T)) @ rg + (D * (X @ rg.T)) @ ru
    steps = 16 + 2 * 2 * 8 + 16
    assert (np.abs(dx[:m // 2] - ref) <= ref * (2.0**-8 + 1.01 * (2.0**-8 + 2.0**-18 + steps * 2.0**-22))).all()
    assert (dx[m // 2:] == 0).all()


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", [(95, 128, 2336), (33, 256, 8256), (300, 100, 1056)])
def test_few_tiles_of_many_pieces(cuda_ctx, mode, m, n, k):
    """One or two output tiles, split along a long axis over more clusters than they have records."""
    x = activations(m, k, m)
    w, ref_w = make_weight(n, k, mode, n)
    close(fp4.fp4_mm(x, w), f64(x) @ ref_w.T,
          HALF[torch.bfloat16] * np.abs(f64(x) @ ref_w.T) + sum_bound(f64(x), ref_w, steps_of(m, k, False)))
    dy = activations(m, k, m + 1)  # the same lengths, summed over the weight's rows
    v, ref_v = make_weight(k, n // 32 * 32, mode, k)
    ref = f64(dy) @ ref_v
    close(fp4.fp4_mm_dgrad(dy, v), ref,
          HALF[torch.bfloat16] * np.abs(ref) + sum_bound(f64(dy), ref_v.T, -(-k // 128) * 8))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("m", [1, 4, 7, 16])
def test_f32_rows_to_the_last_bits(cuda_ctx, mode, wide, m):
    """One value a row, so that nothing but its own rounding (2^-23) and that of the sums counts: the
    products of its two parts (or three, in a record that also holds a huge value against zero weights)
    are exact, added in f32 and scaled (at most six roundings or truncations, 2^-23 each)."""
    k, n = 544, 130
    g = np.random.default_rng(m)
    codes = g.integers(1, 8, (n, k)).astype(np.uint8)  # positive, none zero
    codes[:, 7] = 0
    scales = np.full((n, k // R.BLOCK[mode]), 127 if mode == "mxfp4" else 56, np.uint8)  # 1.0
    w = fp4.FP4Weight(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), mode)
    x = np.zeros((m, k), np.float32)
    x[np.arange(m), g.integers(8, 256, m)] = g.uniform(1, 2, m).astype(np.float32) * np.float32(2.0**-40)
    if wide:
        x[:, 7] = 2.0**50
    ref = x.astype(np.float64) @ R.values(codes, scales, mode, 1.0).T
    y = f64(fp4.fp4_mm(torch.from_numpy(x).cuda(), w, out_dtype=torch.float32))
    assert (np.abs(y - ref) <= 7 * 2.0**-23 * ref).all()


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("quantize_x", [False, True])
@pytest.mark.parametrize("m", [1, 9, 40, 300])
def test_chain_over_the_same_buffers(cuda_ctx, mode, quantize_x, m):
    """Calls that read what the call before wrote, over and over the same buffers, against the same
    calls one at a time: a kernel that is set up while the one before it runs must not see old rows."""
    n = 768
    w, _ = make_weight(n, n, mode, 1, 0.00011)
    v, _ = make_weight(n, n, mode, 2, 0.00011)
    x0 = activations(m, n, 1)

    def chain(each):
        a, b, c, rows = x0.clone(), torch.empty_like(x0), torch.empty_like(x0), []
        for i in range(12):
            fp4.fp4_mm(a, w, quantize_x=quantize_x, out=b)
            each()
            fp4.fp4_gated_mm_dgrad(b, a, w, v, out=c)
            each()
            fp4.fp4_mm_dgrad(c, v, out=b)
            each()
            rows.append(b.clone())
            fp4.fp4_gated_mm(b.clamp_(-4, 4), v, w, quantize_x=quantize_x, out=a)
            each()
            a.copy_(x0 * (1 + i % 3)) if i % 2 else a.clamp_(-4, 4)
        return rows

    one_by_one = chain(torch.cuda.synchronize)
    assert all(torch.isfinite(r).all() and r.any() for r in one_by_one)
    for _ in range(5):
        for got, ref in zip(chain(lambda: None), one_by_one):
            assert torch.equal(got.view(torch.int16), ref.view(torch.int16))


# ------------------------------------------------------------------------------- errors of a call

def test_a_failed_call_leaves_no_error_for_the_next(cuda_ctx):
    """The runtime keeps a call's error until it is read: a weight that does not fit (309 GB) is refused,
    and the launch after it, which looks whether it failed itself, has no part in that."""
    x = activations(3, 64, 1)
    want = fp4.quantize(x, "nvfp4")
    codes, scales = want
    h = C.c_void_p()
    rc = _lib.lib().aex_fp4weight_create(cuda_ctx.handle, codes.data_ptr(), scales.data_ptr(), 2**30, 512,
                                         _lib.AEX_FP4_NV, 1.0, C.byref(h), None)
    assert rc == _lib.AEX_ERR_OOM and not h.value
    got = fp4.quantize(x, "nvfp4")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------- several tiles to a pair of CTAs

def on_gpu(ref):
    return torch.from_numpy(ref).cuda()


def near(got, ref, bound, what):
    """close(), for float64 tensors on the GPU (all of a large result)."""
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - ref).abs() - bound).flatten()
    at = int(over.argmax())
    assert over[at] <= 0, (f"{what} at {divmod(at, ref.shape[1])}: got {got.flatten()[at].item()!r}, exact "
                           f"{ref.flatten()[at].item()!r}, allowed {bound.flatten()[at].item():.3e}")


def gpu_sum_bound(x, w, steps):
    return (steps + 8) * 2.0**-22 * (x.abs() @ w.abs().T)


def gpu_act(g, name):
    """R.act on the GPU."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1.0 + g * (1.0 - s))
    c = (2.0 / np.pi) ** 0.5
    t = torch.tanh(c * (g + 0.044715 * g**3))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g**2)


# Of 2309 rows (ten tiles) and 128 (gated) or 256 columns a tile: 270 tiles, three to four for each of 74 pairs; 150,
# two each and two more, which are split along their 9 or 33 records over many pairs that then take whole ones.
MANY = [(2309, 27 * 128 - 116, 96), (2309, 27 * 128 - 116, 544), (2309, 15 * 128 - 72, 2080),
        (2309, 15 * 128 - 72, 8256)]
X_SCALE = 2.0**-8  # a power of two: the 4-bit form of x is exact in f32


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("quantize_x", [False, True])
@pytest.mark.parametrize("m,n,k", MANY)
def test_gated_of_many_tiles(cuda_ctx, mode, quantize_x, m, n, k):
    """Pairs that go from tile to tile: both accumulators, again and again, and whole tiles after a piece
    of a split one. Every element against float64."""
    ts = X_SCALE if mode == "nvfp4" else 1.0
    x = activations(m, k, m + k)
    wg, rg = make_weight(n, k, mode, 1, 0.00011)
    wu, ru = make_weight(n, k, mode, 2, 0.00037)
    rg, ru = on_gpu(rg), on_gpu(ru)
    if quantize_x:
        X = fp4.dequantize(*fp4.quantize(x, mode, tensor_scale=ts), mode, tensor_scale=ts,
                           out_dtype=torch.float32).double()
    else:
        X = x.double()
    steps = steps_of(m, k, quantize_x)
    g, u = X @ rg.T, X @ ru.T
    eg, eu = gpu_sum_bound(X, rg, steps), gpu_sum_bound(X, ru, steps)
    for act in ("silu", "gelu_tanh"):
        a, _ = gpu_act(g, act)
        z = (g.abs() if act == "silu" else 1.6 * (g + 0.045 * g**3).abs()).clamp(max=90.0)
        bound = 1.2 * u.abs() * eg + a.abs() * eu + 1.2 * eg * eu  # as gated_bound
        bound += ((6 + 1.2 * z) * 2.0**-23 + 2.0**-8) * (a * u).abs() + 2.0**-126
        near(fp4.fp4_gated_mm(x, wg, wu, activation=act, quantize_x=quantize_x, x_scale=ts), a * u, bound, act)
    cuda_ctx.sync()


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("quantize_x", [False, True])
@pytest.mark.parametrize("m,n,k", [(m, 2 * n + 1, k) for m, n, k in MANY])
def test_mm_of_many_tiles(cuda_ctx, mode, quantize_x, m, n, k):
    ts = X_SCALE if mode == "nvfp4" else 1.0
    x = activations(m, k, m + k)
    w, ref_w = make_weight(n, k, mode, 1)
    ref_w = on_gpu(ref_w)
    X = x.double()
    if quantize_x:
        X = fp4.dequantize(*fp4.quantize(x, mode, tensor_scale=ts), mode, tensor_scale=ts,
                           out_dtype=torch.float32).double()
    ref, bound = X @ ref_w.T, gpu_sum_bound(X, ref_w, steps_of(m, k, quantize_x))
    for out in (torch.bfloat16, torch.float32):
        near(fp4.fp4_mm(x, w, quantize_x=quantize_x, x_scale=ts, out_dtype=out), ref, HALF[out] * ref.abs() + bound,
             str(out))
    cuda_ctx.sync()


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", [(m, n // 8 * 8, k) for m, n, k in MANY])
def test_gated_dgrad_of_many_tiles(cuda_ctx, mode, act, m, n, k):
    x, dh = activations(m, k, m + k), activations(m, n, m + n + 1)
    wg, rg = make_weight(n, k, mode, 1, 0.00011)
    wu, ru = make_weight(n, k, mode, 2, 0.00037)
    rg, ru, X, D = on_gpu(rg), on_gpu(ru), x.double(), dh.double()
    g, u = X @ rg.T, X @ ru.T
    a, slope = gpu_act(g, act)
    dg, du = D * u * slope, D * a
    steps = -(-k // 256) * 16
    eg, eu = gpu_sum_bound(X, rg, steps), gpu_sum_bound(X, ru, steps)
    # as test_gated_dgrad
    e_dg = (2.0**-8 + 2.0**-18) * dg.abs() + D.abs() * (slope.abs() * eu + 1.2 * u.abs() * eg) * 1.01 \
        + 2.0**-18 * (D * u).abs()
    e_du = (2.0**-8 + 2.0**-18) * du.abs() + 1.2 * D.abs() * eg * 1.01
    ref = dg @ rg + du @ ru
    bound = e_dg @ rg.abs() + e_du @ ru.abs() + 2.0**-8 * ref.abs() \
        + (2 * -(-n // 128) * 8 + 8) * 2.0**-22 * 1.01 * (dg.abs() @ rg.abs() + du.abs() @ ru.abs())
    near(fp4.fp4_gated_mm_dgrad(dh, x, wg, wu, activation=act), ref, bound, act)
    cuda_ctx.sync()


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", [(2309, 96, 27 * 256 - 96), (2309, 2080, 15 * 256 - 160),
                                   (2309, 8256, 15 * 256 - 160)])
def test_mm_dgrad_of_many_tiles(cuda_ctx, mode, m, n, k):
    dy = activations(m, n, m + n)
    w, ref_w = make_weight(n, k, mode, n + k)
    ref_w, D = on_gpu(ref_w), dy.double()
    ref, bound = D @ ref_w, gpu_sum_bound(D, ref_w.T, -(-n // 128) * 8)
    for out in (torch.bfloat16, torch.float32):
        near(fp4.fp4_mm_dgrad(dy, w, out_dtype=out), ref, HALF[out] * ref.abs() + bound, str(out))
    cuda_ctx.sync()


# ------------------------------------------------------------------------------ rows on their own

@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("quantize_x", [False, True])
@pytest.mark.parametrize("m", [3, 8, 9, 16])
def test_few_rows_beside_a_row_of_infinities(cuda_ctx, mode, dtype, quantize_x, m):
    """A row that holds an infinity or NaN sends its 256 columns of every row through the other staging:
    the clean rows' results, in one and in two 8-column operands, are those of the formula all the same."""
    k, n = 544, 264
    g = np.random.default_rng(5)
    codes = g.integers(1, 8, (n, k)).astype(np.uint8)  # positive, none zero
    scales = np.full((n, k // R.BLOCK[mode]), 120 if mode == "mxfp4" else 40, np.uint8)
    w = fp4.FP4Weight(torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda(), mode)
    ref_w = R.values(codes, scales, mode)
    x = activations(m, k, 3, DT[dtype])
    x[0, 17] = float("-inf")
    x[m - 1, 300] = float("nan")
    ts = 2.0**-6 if mode == "nvfp4" else 1.0
    X = f64(x)[1:m - 1]
    if quantize_x:
        X = R.values(*R.quantize(X, mode, ts), mode, ts)
    ref = X @ ref_w.T
    for out in (torch.bfloat16, torch.float32):
        y = fp4.fp4_mm(x, w, quantize_x=quantize_x, x_scale=ts, out_dtype=out)
        close(y[1:m - 1], ref, HALF[out] * np.abs(ref) + sum_bound(X, ref_w, steps_of(m, k, quantize_x)))
        assert torch.isnan(y[m - 1]).all()
        assert (torch.isnan(y[0]) if quantize_x else y[0] == float("-inf")).all()


# --------------------------------------------------------------- tensors dropped after a call

def test_tensors_given_to_another_stream_may_be_dropped(cuda_ctx, monkeypatch):
    """A call's tensors are recorded on a stream of its own, and while that is behind they are not handed
    to new work on the stream they came from (a pack's arrays are usually dropped as soon as the weight
    is made; making it allocates, which may wait for the device, so there only the recording is seen)."""
    m, n, k = 200, 520, 544
    s = torch.cuda.Stream()
    wg, _ = make_weight(n, k, "nvfp4", 1)
    wu, _ = make_weight(n, k, "nvfp4", 2)
    x0, dh0 = activations(m, k, 1), activations(m, n, 2)
    c0, s0 = fp4.quantize(activations(n, k, 3), "nvfp4")
    calls = {
        "weight": ([c0, s0], lambda c, sc: fp4.FP4Weight(c, sc, "nvfp4", stream=s)),
        "quantize": ([x0], lambda x: fp4.quantize(x, "nvfp4", stream=s)),
        "dequantize": ([c0, s0], lambda c, sc: fp4.dequantize(c, sc, "nvfp4", stream=s)),
        "mm": ([x0, dh0], lambda x, out: fp4.fp4_mm(x, wg, out=out, stream=s)),
        "gated": ([x0], lambda x: fp4.fp4_gated_mm(x, wg, wu, quantize_x=True, stream=s)),
        "dgrad": ([dh0], lambda dh: fp4.fp4_mm_dgrad(dh, wg, stream=s)),
        "gated dgrad": ([dh0, x0], lambda dh, x: fp4.fp4_gated_mm_dgrad(dh, x, wg, wu, stream=s)),
    }
    seen, record = set(), torch.Tensor.record_stream

    def spy(t, stream):
        seen.add((t.data_ptr(), stream.cuda_stream))
        record(t, stream)

    monkeypatch.setattr(torch.Tensor, "record_stream", spy)
    for name, (given, call) in calls.items():
        call(*[t.clone() for t in given])  # whatever a first call sets up
        torch.cuda.synchronize()
        mine = [t.clone() for t in given]
        at = {t.data_ptr() for t in mine}
        torch.cuda.synchronize()
        seen.clear()
        with torch.cuda.stream(s):
            torch.cuda._sleep(200_000_000)  # some 0.1 s
        got = call(*mine)
        assert {(p, s.cuda_stream) for p in at} <= seen, name
        del mine
        new = [torch.full_like(t, 1) for t in given for _ in range(4)]
        if name != "weight":
            assert not at & {t.data_ptr() for t in new}, name
        torch.cuda.synchronize()
        if name == "weight":
            assert torch.equal(got.dequantize(), fp4.dequantize(c0, s0, "nvfp4"))
        del got, new


# ------------------------------------------------------------------- gradients of odd widths

def placed(t, how):
    """t's values as a contiguous tensor, in rows of whole vectors with NaN behind them, or anywhere."""
    m, n = t.shape
    if how == "contiguous":
        return t.contiguous()
    pitch, start = (-(-n // 8) * 8 + 8, 0) if how == "padded" else (n + 3, 5)
    buf = torch.full((m * pitch + start,), float("nan"), dtype=t.dtype, device=t.device)
    out = buf[start:].as_strided((m, n), (pitch, 1))
    out.copy_(t)
    return out


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("how", ["contiguous", "padded", "anywhere"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (5, 1, 544), (1, 257, 96), (3, 129, 288), (77, 257, 544),
                                   (300, 1003, 1120), (33, 8251, 256)])
def test_dgrads_of_odd_widths(cuda_ctx, mode, how, m, n, k):
    """Incoming gradients as the products return them (contiguous rows of n), in rows of whole vectors
    whose rest holds NaN, and at any start and pitch; several tiles, and tiles in pieces."""
    x, d = activations(m, k, m + k), placed(activations(m, n, m + n + 1), how)
    wg, rg = make_weight(n, k, mode, 1, 0.00011)
    wu, ru = make_weight(n, k, mode, 2, 0.00037)
    X, D = f64(x), f64(d)
    ref, bound = D @ rg, sum_bound(D, rg.T, -(-n // 128) * 8)
    for out in (torch.bfloat16, torch.float32):
        close(fp4.fp4_mm_dgrad(d, wg, out_dtype=out), ref, HALF[out] * np.abs(ref) + bound)
    dg, du, g, u, a, slope = gated_grad_ref(X, D, rg, ru, "silu")
    eg, eu = (sum_bound(X, w, -(-k // 256) * 16) for w in (rg, ru))
    # as test_gated_dgrad
    e_dg = (2.0**-8 + 2.0**-18) * np.abs(dg) + np.abs(D) * (np.abs(slope) * eu + 1.2 * np.abs(u) * eg) * 1.01 \
        + 2.0**-18 * np.abs(D * u)
    e_du = (2.0**-8 + 2.0**-18) * np.abs(du) + 1.2 * np.abs(D) * eg * 1.01
    ref = dg @ rg + du @ ru
    bound = e_dg @ np.abs(rg) + e_du @ np.abs(ru) + 2.0**-8 * np.abs(ref) \
        + (2 * -(-n // 128) * 8 + 8) * 2.0**-22 * 1.01 * (np.abs(dg) @ np.abs(rg) + np.abs(du) @ np.abs(ru))
    close(fp4.fp4_gated_mm_dgrad(d, x, wg, wu), ref, bound)
    cuda_ctx.sync()


def test_a_products_own_result_goes_back(cuda_ctx):
    """What fp4_mm and fp4_gated_mm return is a gradient that their gradients take, whatever the width."""
    for n in (256, 257, 1003):
        w, _ = make_weight(n, 288, "nvfp4", 1)
        x = activations(20, 288, 1)
        for y in (fp4.fp4_mm(x, w), fp4.fp4_gated_mm(x, w, w)):
            whole = placed(y, "padded") if n % 8 else y
            assert torch.equal(fp4.fp4_mm_dgrad(y, w), fp4.fp4_mm_dgrad(whole, w))
            assert torch.equal(fp4.fp4_gated_mm_dgrad(y, x, w, w), fp4.fp4_gated_mm_dgrad(whole, x, w, w))


def test_odd_gradient_rows_refusals(cuda_ctx):
    E = _lib.AexError
    w, _ = make_weight(264, 288, "nvfp4", 1)
    dy = torch.zeros(5, 267, dtype=torch.bfloat16, device="cuda")[:, :264]
    with pytest.raises(E, match="multiple of 16 bytes"):  # a width of whole vectors has them
        fp4.fp4_mm_dgrad(dy, w)
    v, _ = make_weight(257, 288, "nvfp4", 1)
    with pytest.raises(E, match="row pitch of at least 257"):
        fp4.fp4_mm_dgrad(torch.zeros(1, 257, dtype=torch.bfloat16, device="cuda").expand(5, 257), v)
    dx = torch.empty(5, 288, dtype=torch.bfloat16, device="cuda")
    d = torch.zeros(5, 257, dtype=torch.bfloat16, device="cuda")
    L, h = _lib.lib(), cuda_ctx.handle
    need = L.aex_fp4_mm_dgrad_workspace_bytes(v.handle, 5)
    assert need >= 5 * 264 * 2
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for p, n in ((None, 0), (ws.data_ptr(), need - 1)):
        assert L.aex_fp4_mm_dgrad(h, v.handle, d.data_ptr(), 257, 5, dx.data_ptr(), 0, 288, p, n,
                                  None) == _lib.AEX_ERR_INVALID_ARG
        assert b"workspace" in L.aex_last_error_string(h)
    for ptr, ld, m in ((d.data_ptr() + 1, 257, 5), (d.data_ptr(), 256, 5), (d.data_ptr(), 257, 0), (None, 257, 5)):
        assert L.aex_fp4_mm_dgrad(h, v.handle, ptr, ld, m, dx.data_ptr(), 0, 288, ws.data_ptr(), need,
                                  None) == _lib.AEX_ERR_INVALID_ARG
    assert cuda_ctx.device_status() == 0


# ------------------------------------------------------------------------ results over inputs

@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_a_result_may_not_lie_over_an_input(cuda_ctx, m):
    """It would be read by one CTA while another writes it. Columns of one buffer, and rows behind one
    another, are apart."""
    n = k = 256
    w, _ = make_weight(n, k, "nvfp4", 1)
    buf = torch.zeros(2 * m * 3 * k, dtype=torch.bfloat16, device="cuda")
    wide = buf.view(2 * m, 3 * k)
    x = wide[:m, :k]
    x.copy_(activations(m, k, 1))
    before = buf.clone()
    for out in (x, wide[:m, k // 2:k // 2 + n], wide[m - 1:2 * m - 1, :n], buf[k - 8:].as_strided((m, n), (n, 1))):
        for call in (lambda: fp4.fp4_mm(x, w, out=out), lambda: fp4.fp4_mm(x, w, quantize_x=True, out=out),
                     lambda: fp4.fp4_gated_mm(x, w, w, out=out), lambda: fp4.fp4_mm_dgrad(x, w, out=out)):
            with pytest.raises(_lib.AexError, match="must not overlap"):
                call()
    assert torch.equal(buf, before)
    for out in (wide[:m, k:k + n], wide[:m, 2 * k:2 * k + n], wide[m:, :n]):
        assert torch.equal(fp4.fp4_mm(x, w, out=out), fp4.fp4_mm(x, w))
        assert torch.equal(fp4.fp4_mm_dgrad(x, w, out=out), fp4.fp4_mm_dgrad(x, w))
        assert torch.equal(fp4.fp4_gated_mm(x, w, w, out=out), fp4.fp4_gated_mm(x, w, w))


def test_whole_rows_of_an_odd_width_need_no_copy(cuda_ctx):
    """A C caller whose rows are of whole vectors needs the copy's part of the workspace neither."""
    w, _ = make_weight(257, 288, "nvfp4", 1)
    d = placed(activations(5, 257, 1), "padded")
    dx, L = torch.empty(5, 288, dtype=torch.bfloat16, device="cuda"), _lib.lib()
    assert L.aex_fp4_mm_dgrad_workspace_bytes(w.handle, 5) == -(-5 * 264 * 2 // 256) * 256
    rc = L.aex_fp4_mm_dgrad(cuda_ctx.handle, w.handle, d.data_ptr(), d.stride(0), 5, dx.data_ptr(),
                            _lib.AEX_DTYPE_BF16, 288, None, 0, None)
    assert rc == _lib.AEX_OK
    torch.cuda.synchronize()
    assert torch.equal(dx, fp4.fp4_mm_dgrad(d, w))


@pytest.mark.parametrize("m", [3, 70])
def test_captured_with_streams_and_odd_widths(cuda_ctx, m):
    """Calls given the capturing stream, over tensors that are dropped, and gradients that are copied
    first: the graph replays what the calls compute, next to other work of the same pool."""
    n, k = 257, 544
    w, _ = make_weight(n, k, "mxfp4", 1)
    x = activations(m, k, 1)

    def calls(stream):
        y = fp4.fp4_mm(x, w, quantize_x=True, stream=stream)
        dx = fp4.fp4_mm_dgrad(y, w, stream=stream)
        return fp4.fp4_gated_mm_dgrad(y, dx, w, w, stream=stream)  # y and dx are dropped here

    s = torch.cuda.Stream()
    want = calls(None)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        calls(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = calls(s)
    for seed in (1, 2):
        x.copy_(activations(m, k, seed))
        want = calls(None)
        torch.cuda.synchronize()
        g.replay()
        junk = [torch.full_like(x, 3.0) for _ in range(8)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del junk


# ------------------------------------------------------------------------ rows beyond 2^27 columns

@pytest.mark.parametrize("mode", MODES)
def test_rows_of_more_units_than_a_launch_holds_128_of(cuda_ctx, mode):
    """2^27 and 32 columns: 64 rows a launch, so that the second starts inside a tile of 128. x is zero
    but for forty columns, whose blocks say all there is to say."""
    if torch.cuda.mem_get_info()[0] < 100e9:
        pytest.skip("needs 100 GB of device memory")
    m, k, block = 70, 2**27 + 32, R.BLOCK[mode]
    g = np.random.default_rng(1)
    blocks = np.unique(np.concatenate([[0, k // block - 1], g.integers(0, k // block, 38)]))
    some = np.zeros((m, len(blocks), block), np.float32)
    some[:, np.arange(len(blocks)), g.integers(0, block, len(blocks))] = g.choice([-3.0, -1.0, 0.5, 2.0, 6.0],
                                                                                  (m, len(blocks)))
    some = some.reshape(m, -1)
    cols = torch.from_numpy((blocks[:, None] * block + np.arange(block)).reshape(-1)).cuda()
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[:, cols] = torch.from_numpy(some).bfloat16().cuda()
    ref_codes, ref_scales = R.quantize(some, mode)
    ref = R.values(ref_codes, ref_scales, mode)
    codes, scales = fp4.quantize(x, mode)
    at = torch.from_numpy(blocks).cuda()
    assert np.array_equal(scales[:, at].cpu().numpy(), ref_scales)
    assert int(scales.count_nonzero()) == int((ref_scales != 0).sum())
    assert np.array_equal(codes[:, cols[::2] // 2].cpu().numpy(), R.pack(ref_codes))
    assert int(codes.count_nonzero()) == int((R.pack(ref_codes) != 0).sum())
    y = torch.empty(m, 40, device="cuda")
    w = fp4.FP4Weight(codes[:40], scales[:40], mode)
    fp4.fp4_mm(x, w, quantize_x=True, out=y)
    want = ref @ ref[:40].T
    # the sums have at most forty terms, in as many steps
    close(y, want, 2.0**-24 * np.abs(want) + (len(blocks) + 8) * 2.0**-22 * (np.abs(ref) @ np.abs(ref[:40]).T))
    del w, x
    torch.cuda.empty_cache()
    back = fp4.dequantize(codes, scales, mode)
    assert np.array_equal(f64(back[:, cols]), ref)
    assert int(back.count_nonzero()) == int((ref != 0).sum())
    w = fp4.FP4Weight(codes, scales, mode)
    got = w.dequantize()
    assert all(torch.equal(got[r], back[r]) for r in range(m))
    del w, got, back, codes, scales
    torch.cuda.empty_cache()


def test_dequantize_rounds_once_next_to_ties(cuda_ctx):
    """Tensor scales amax * 1.25 / 2688 = amax * 5 / (21 * 2^9) of bf16 amax, rounded to f32: a scale of 1.75 times a
    code of 1.5 has the factor 21, so those products lie within 2^-24 of numbers of 11 bits, ties of bf16 among
    them. Rounding them to f32 on the way would take some to the wrong side."""
    codes = np.tile(np.arange(16, dtype=np.uint8), (127, 2))
    scales = np.repeat(np.arange(127, dtype=np.uint8)[:, None], 2, 1)
    c, s = torch.from_numpy(R.pack(codes)).cuda(), torch.from_numpy(scales).cuda()
    twice = 0
    for a in range(128):
        ts = float(np.float32((1 + a / 128) * 1.25 / 2688))
        ref = R.values(codes, scales, "nvfp4", ts)  # exact: 6 by 24 bits
        _, e = np.frexp(ref)
        step = np.ldexp(1.0, e - 8)
        once = np.where(ref == 0, 0.0, np.round(ref / step) * step)
        assert np.array_equal(f64(fp4.dequantize(c, s, "nvfp4", tensor_scale=ts)), once)
        twice += (np.round(np.float32(ref).astype(np.float64) / step) * step != once).sum()
    assert twice  # these scales do hold such products
