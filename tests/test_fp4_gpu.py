"""The microscaled 4-bit operators against float64 (oracle/fp4_ref.py).

Tolerances. A rounding to bf16 is off by at most 2^-8 of the value, to f32 by 2^-24. A product's
f32 sums on the tensor cores truncate: every one of the accumulation steps (K/16, or K/64 for two
4-bit operands; 16 for each 256 columns in the few-rows kernel, which adds those in f32) can lose
a unit of the last place of a partial sum, which no partial sum's terms' magnitudes S = sum |x w|
exceed, and aligning the terms of a step the same again: at most (steps + 8) 2^-22 S."""
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
    """f32 activations keep all 24 bits."""
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
