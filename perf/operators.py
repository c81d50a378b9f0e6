"""What is measured of the microscaled 4-bit floating-point operators.

A matrix in this form holds e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, two to a
byte, the even column in the low nibble) and one 8-bit scale for every block of columns:

* ``mxfp4``: blocks of 32, the scale an exponent byte, 2^(byte - 127);
* ``nvfp4``: blocks of 16, the scale an e4m3 number, and one f32 scale for the whole tensor.

Operators: quantisation (and the values back), the product with such a weight (activations as
they are, or brought to 4 bits within the call), the gated feed-forward projection
act(x Wg^T) * (x Wu^T), and both products' gradients with respect to their inputs (a 4-bit weight
is frozen and has none).
"""
import math

import torch

own = False

BLOCK = {"mxfp4": 32, "nvfp4": 16}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------ cases

def listed():
    """Rows are tokens: 1 to 16 in a decoding or conditioning step, some dozens to hundreds for a
    prompt, thousands for an image's latents. Widths are those of a 4-billion-parameter
    transformer's feed-forward blocks, or odd ones near them."""
    return [
        # A prompt's embeddings brought to 4 bits, as they leave a text encoder in f32: latency.
        dict(name="quantize_prompt", op="quantize", mode="mxfp4", m=77, k=7680, dtype="f32", out="f32"),
        # The hidden activations of an image's feed-forward block: bandwidth.
        dict(name="quantize_latents", op="quantize", mode="nvfp4", m=4608, k=9216, dtype="bf16", out="bf16"),
        # One token through a projection: the weight is read once, nothing else counts.
        dict(name="mm_token", op="mm", mode="nvfp4", m=1, n=9216, k=4096, dtype="bf16", out="bf16", quant=False),
        # A conditioning vector's modulation heads in f32, an odd number of outputs.
        dict(name="mm_conditioning", op="mm", mode="mxfp4", m=3, n=18431, k=4096, dtype="f32", out="f32",
             quant=False),
        # A prompt's context projection: some dozens of rows, so the weight still dominates.
        dict(name="mm_prompt", op="mm", mode="mxfp4", m=77, n=4096, k=7680, dtype="bf16", out="bf16", quant=False),
        # A part of an image (an odd number of rows) down from the hidden width, activations kept.
        dict(name="mm_rows", op="mm", mode="nvfp4", m=1111, n=4104, k=9216, dtype="bf16", out="bf16", quant=False),
        # A whole image's projection with both operands in 4 bits.
        dict(name="mm_latents", op="mm", mode="nvfp4", m=4608, n=12288, k=4096, dtype="bf16", out="bf16",
             quant=True),
        # The gradient that reaches a prompt's embeddings through a frozen projection.
        dict(name="mm_dgrad_prompt", op="mm_dgrad", mode="nvfp4", m=512, n=4096, k=7680, dtype="bf16", out="bf16"),
        # One token through the gated block, activations brought to 4 bits on the way.
        dict(name="gated_token", op="gated", mode="nvfp4", m=1, n=9216, k=4096, dtype="bf16", out="bf16",
             quant=True, act="silu"),
        # The text stream's gated block, activations kept.
        dict(name="gated_text", op="gated", mode="mxfp4", m=512, n=9216, k=4096, dtype="bf16", out="bf16",
             quant=False, act="silu"),
        # The image stream's gated block with both operands in 4 bits: the largest.
        dict(name="gated_latents", op="gated", mode="mxfp4", m=4608, n=9216, k=4096, dtype="bf16", out="bf16",
             quant=True, act="gelu_tanh"),
        # Tuning what comes before a frozen gated block.
        dict(name="gated_dgrad_text", op="gated_dgrad", mode="nvfp4", m=1024, n=9216, k=4096, dtype="bf16",
             out="bf16", act="silu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: any operator, form, type and number of rows; widths from
    a few dozen to the largest listed, odd numbers of outputs among them."""
    op = rng.choice(["quantize", "mm", "mm", "mm_dgrad", "gated", "gated", "gated_dgrad"])
    case = dict(op=op, mode=rng.choice(["mxfp4", "nvfp4"]), m=_log(rng, 1, 4608), k=32 * _log(rng, 4, 288))
    if op == "quantize":
        case["dtype"] = rng.choice(["bf16", "f32"])
        case["out"] = rng.choice(["bf16", "f32"])
        return case
    n = _log(rng, 40, 12288)
    case["n"] = n if rng.random() < 0.3 else max(8, n // 8 * 8)  # most are whole vectors, some are odd
    while case["m"] * case["n"] * case["k"] * (2 if op.startswith("gated") else 1) > 2 * 4608 * 9216 * 4096 // (
            2 if op == "gated_dgrad" else 1):
        case["m"] = (case["m"] + 1) // 2
    case["dtype"] = "bf16"
    case["out"] = "bf16"
    if op in ("mm", "gated"):
        case["quant"] = rng.random() < 0.5
        # f32 activations are taken as they are for up to 16 rows, and for any number when quantised
        if (case["quant"] or case["m"] <= 16) and rng.random() < 0.4:
            case["dtype"] = "f32"
        # few rows: conditioning vectors, which stay in f32
        if case["m"] <= 16 and rng.random() < 0.4:
            case["out"] = "f32"
    if op.startswith("gated"):
        case["act"] = rng.choice(["silu", "gelu_tanh"])
    if op in ("mm_dgrad", "gated_dgrad"):
        case["n"] = max(8, case["n"] // 8 * 8)  # the incoming gradient's rows are whole 16-byte vectors
    return case


def work(case):
    """Inputs read once, outputs written once; a product's multiplications and additions."""
    m, k, op = case["m"], case["k"], case["op"]
    four = 0.5 + 1.0 / BLOCK[case["mode"]]  # bytes of a code and its share of the scale
    if op == "quantize":
        # x in, the 4-bit form out and in again, the values out
        return {"bytes": m * k * (SIZE[case["dtype"]] + 2 * four + SIZE[case["out"]]), "flops": 4 * m * k}
    n = case["n"]
    mats = 2 if op.startswith("gated") else 1
    weights = mats * n * k * four
    if op in ("mm", "gated"):
        return {"bytes": weights + m * k * SIZE[case["dtype"]] + m * n * SIZE[case["out"]],
                "flops": 2 * mats * m * n * k}
    if op == "mm_dgrad":
        return {"bytes": weights + m * n * 2 + m * k * SIZE[case["out"]], "flops": 2 * m * n * k}
    # the projections again (they are not kept), then both gradients
    return {"bytes": weights + m * n * 2 + m * k * 2 + m * k * SIZE[case["out"]], "flops": 8 * m * n * k}


# ----------------------------------------------------------------------------------------- inputs

def _activations(g, m, k, dtype):
    """Rows of unit variance with a few wide channels, as a transformer's activations have."""
    x = torch.randn(m, k, generator=g, device="cuda")
    wide = 1.0 + 7.0 * (torch.rand(k, generator=g, device="cuda") < 0.01).float()
    return (x * wide).to(dtype)


def _tensor_scale(amax, mode):
    """The usual choice: the largest value takes the largest block scale and code."""
    return amax / (448.0 * 6.0) if mode == "nvfp4" else 1.0


def _weight(g, n, k, mode):
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    scale = torch.tensor(_tensor_scale(w.abs().max().item(), mode), dtype=torch.float32).item()
    codes, scales = _quantize(w, mode, scale)
    return {"codes": _pack(codes), "scales": scales, "scale": scale}


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m, k, mode = case["m"], case["k"], case["mode"]
    s = {}
    if case["op"] == "mm_dgrad":
        s["dy"] = torch.randn(m, case["n"], generator=g, device="cuda").to(torch.bfloat16)
    else:
        s["x"] = _activations(g, m, k, TYPES[case["dtype"]])
        # a calibrated scale: somewhat above what these rows need
        s["x_scale"] = torch.tensor(_tensor_scale(1.25 * s["x"].float().abs().max().item(), mode),
                                    dtype=torch.float32).item()
    if case["op"] == "gated_dgrad":
        s["dh"] = torch.randn(m, case["n"], generator=g, device="cuda").to(torch.bfloat16)
    if case["op"] != "quantize":
        names = ("gate", "up") if case["op"].startswith("gated") else ("w",)
        for name in names:
            s[name] = _weight(g, case["n"], k, mode)
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        from aestrix_b200 import fp4

        for name in ("w", "gate", "up"):
            if name in state:
                w = state[name]
                state[name] = fp4.FP4Weight(w["codes"], w["scales"], case["mode"], tensor_scale=w["scale"])
    return state


# ------------------------------------------------------------------------------------ plain forms

def _e4m3(v):
    """Round to the nearest e4m3 number (ties to the even mantissa, at most 448), 64-bit in and out."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(v / step) * step).clamp(max=448.0)


def _e2m1(q):
    """Codes 0..7 of magnitudes, nearest value, ties to the even code, at most 6."""
    c = (q > 0.25).to(torch.uint8)
    for border, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (q >= border) if up else (q > border)
    return c


def _quantize(x, mode, tensor_scale):
    """Codes (one a byte) and scale bytes; in 64 bits, since values lie on the borders of codes."""
    m, k = x.shape
    v = x.double().view(m, k // BLOCK[mode], BLOCK[mode])
    mag = v.abs()
    amax = mag.amax(-1)
    if mode == "mxfp4":
        _, e = torch.frexp(amax)
        byte = torch.where(amax > 0, (e - 1 - 2 + 127).clamp(0, 254), torch.zeros_like(e))
        scales = byte.to(torch.uint8)
        unit = torch.exp2(byte.double() - 127)
    else:
        s = _e4m3(amax / (6.0 * tensor_scale))
        scales = s.to(torch.float8_e4m3fn).view(torch.uint8)
        unit = s * tensor_scale
    unit = unit.unsqueeze(-1)
    q = torch.where(unit > 0, mag / unit, torch.zeros_like(mag))
    codes = _e2m1(q) | ((v < 0).to(torch.uint8) << 3)
    return codes.view(m, k), scales


def _pack(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def _values(codes, scales, mode):
    """f32 values of codes (one a byte) and scale bytes, before the tensor's scale: exact."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=codes.device)
    if mode == "mxfp4":
        unit = torch.exp2(scales.float() - 127)
    else:
        unit = scales.view(torch.float8_e4m3fn).float()
    m, k = codes.shape
    return (table[codes.int()].view(m, -1, BLOCK[mode]) * unit.unsqueeze(-1)).view(m, k)


def _unpacked(w, mode):
    codes = torch.stack((w["codes"] & 15, w["codes"] >> 4), -1).view(w["codes"].shape[0], -1)
    return _values(codes, w["scales"], mode)


def _sigmoid_arg(g, act):
    if act == "silu":
        return g
    return math.sqrt(8.0 / math.pi) * (g + 0.044715 * g * g * g)  # gelu's tanh form is g * sigmoid(2 u)


def _sigmoid_arg_slope(g, act):
    if act == "silu":
        return torch.ones_like(g)
    return math.sqrt(8.0 / math.pi) * (1.0 + 3 * 0.044715 * g * g)


def _plain(state):
    case = state["case"]
    op, mode = case["op"], case["mode"]
    out = TYPES[case["out"]]
    if op == "quantize":
        codes, scales = _quantize(state["x"], mode, state["x_scale"])
        return (_values(codes, scales, mode).double() * state["x_scale"]).to(out)
    if op == "mm_dgrad":
        return (state["dy"].float() @ _unpacked(state["w"], mode) * state["w"]["scale"]).to(out)
    x, unit = state["x"].float(), 1.0
    if case.get("quant"):
        codes, scales = _quantize(state["x"], mode, state["x_scale"])
        x, unit = _values(codes, scales, mode), state["x_scale"]
    if op == "mm":
        return (x @ _unpacked(state["w"], mode).t() * (unit * state["w"]["scale"])).to(out)
    wg, wu = _unpacked(state["gate"], mode), _unpacked(state["up"], mode)
    g = x @ wg.t() * (unit * state["gate"]["scale"])
    u = x @ wu.t() * (unit * state["up"]["scale"])
    sig = 1.0 / (1.0 + torch.exp(-_sigmoid_arg(g, case["act"])))
    if op == "gated":
        return (g * sig * u).to(out)
    dh = state["dh"].float()
    dg = dh * u * (sig + g * sig * (1.0 - sig) * _sigmoid_arg_slope(g, case["act"]))
    du = dh * g * sig
    return (dg @ wg * state["gate"]["scale"] + du @ wu * state["up"]["scale"]).to(out)


def _framework(state):
    from aestrix_b200 import fp4

    case = state["case"]
    op, out = case["op"], TYPES[case["out"]]
    if op == "quantize":
        codes, scales = fp4.quantize(state["x"], case["mode"], tensor_scale=state["x_scale"])
        return fp4.dequantize(codes, scales, case["mode"], tensor_scale=state["x_scale"], out_dtype=out)
    if op == "mm":
        return fp4.fp4_mm(state["x"], state["w"], quantize_x=case["quant"], x_scale=state["x_scale"], out_dtype=out)
    if op == "mm_dgrad":
        return fp4.fp4_mm_dgrad(state["dy"], state["w"], out_dtype=out)
    if op == "gated":
        return fp4.fp4_gated_mm(state["x"], state["gate"], state["up"], activation=case["act"],
                                quantize_x=case["quant"], x_scale=state["x_scale"], out_dtype=out)
    return fp4.fp4_gated_mm_dgrad(state["dh"], state["x"], state["gate"], state["up"], activation=case["act"],
                                  out_dtype=out)


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------ exact

def _nearest(v, grid):
    """Index of the nearest entry of an ascending 64-bit grid, ties to the even index, ends clamped."""
    hi = torch.searchsorted(grid, v.contiguous()).clamp(1, grid.numel() - 1)
    lo = hi - 1
    below, above = v - grid[lo], grid[hi] - v
    take_hi = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(take_hi, hi, lo)


def _exact_values(x, mode, tensor_scale):
    """What the 4-bit form of x stands for, over the tensor's scale, in 64 bits."""
    e2m1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    blocks = x.double().reshape(-1, BLOCK[mode])
    top = blocks.abs().max(dim=1).values
    if mode == "mxfp4":
        # the power of two that puts the largest magnitude into [4, 8)
        powers = torch.tensor([2.0 ** (i - 127) for i in range(255)], dtype=torch.float64, device=x.device)
        i = torch.searchsorted(powers * 4.0, top, right=True) - 1
        unit = powers[i.clamp(0, 254)]
        real = unit
    else:
        positive = [(1 + f / 8) * 2.0 ** (e - 7) if e else f * 2.0 ** -9 for e in range(16) for f in range(8)][:127]
        grid = torch.tensor(positive, dtype=torch.float64, device=x.device)
        unit = grid[_nearest(top / (tensor_scale * 6.0), grid)]
        real = unit * tensor_scale
    safe = torch.where(real > 0, real, torch.ones_like(real))[:, None]
    mag = e2m1[_nearest(blocks.abs() / safe, e2m1)] * (real > 0)[:, None]
    return (torch.sign(blocks) * mag * unit[:, None]).reshape(x.shape)


def _exact_weight(w, mode):
    """The weight's values in 64 bits, the tensor's scale among them, byte by byte from their definition."""
    magnitudes = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    low = torch.tensor([magnitudes[b & 7] * (-1.0 if b & 8 else 1.0) for b in range(256)], dtype=torch.float64)
    high = torch.tensor([magnitudes[(b >> 4) & 7] * (-1.0 if b & 128 else 1.0) for b in range(256)],
                        dtype=torch.float64)
    if mode == "mxfp4":
        unit = torch.tensor([2.0 ** (b - 127) for b in range(256)], dtype=torch.float64)
    else:
        unit = torch.tensor([(1 + (b & 7) / 8) * 2.0 ** ((b >> 3 & 15) - 7) if b >> 3 & 15 else (b & 7) * 2.0 ** -9
                             for b in range(256)], dtype=torch.float64)
    byte = w["codes"].long()
    n, half = byte.shape
    out = torch.empty(n, 2 * half, dtype=torch.float64, device=byte.device)
    out[:, 0::2] = low.to(byte.device)[byte]
    out[:, 1::2] = high.to(byte.device)[byte]
    out *= unit.to(byte.device)[w["scales"].long()].repeat_interleave(BLOCK[mode], dim=1)
    return out * w["scale"]


def exact(case, seed):
    s = _inputs(case, seed)
    op, mode = case["op"], case["mode"]
    if op == "quantize":
        return _exact_values(s["x"], mode, s["x_scale"]) * s["x_scale"]
    if op == "mm_dgrad":
        return s["dy"].double() @ _exact_weight(s["w"], mode)
    x = s["x"].double()
    if case.get("quant"):
        x = _exact_values(s["x"], mode, s["x_scale"]) * s["x_scale"]
    if op == "mm":
        return x @ _exact_weight(s["w"], mode).T
    gate, up = _exact_weight(s["gate"], mode), _exact_weight(s["up"], mode)
    g, u = x @ gate.T, x @ up.T
    if case["act"] == "silu":
        value = g * torch.sigmoid(g)
        slope = torch.sigmoid(g) * (1.0 + g * torch.sigmoid(-g))
    else:
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g ** 3))
        value = 0.5 * g * (1.0 + t)
        slope = 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 0.134145 * g ** 2)
    if op == "gated":
        return value * u
    dh = s["dh"].double()
    return (dh * u * slope) @ gate + (dh * value) @ up
