"""Microscaled 4-bit floating point in float64 (numpy), from the definitions: the checker of the
fp4 operators' tests. Arrays stand for real numbers; quotients that decide a rounding are formed in
float64, where bf16 and f32 inputs, e4m3 scales and an f32 tensor scale leave no doubt about a
border (a quotient of 24- by 28-bit significands is never within 2^-53 of a short one it differs
from)."""
import numpy as np

BLOCK = {"mxfp4": 32, "nvfp4": 16}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([(1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) if b >> 3 else (b & 7) * 2.0**-9 for b in range(127)])


def nearest(v, grid):
    """Index of the nearest of an ascending grid, ties to the even index, ends clamped (v >= 0)."""
    hi = np.clip(np.searchsorted(grid, v), 1, len(grid) - 1)
    below, above = v - grid[hi - 1], grid[hi] - v
    return np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, hi - 1)


def scale_values(scales, mode):
    """float64 values of scale bytes (NaN bytes: NaN)."""
    s = np.asarray(scales).astype(np.int64)
    if mode == "mxfp4":
        return np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return np.append(E4M3, np.nan)[s & 127]


def quantize(x, mode, tensor_scale=1.0):
    """codes (one a byte) [rows, k] and scales [rows, k/block] of float64 x."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    v = x.reshape(rows, k // BLOCK[mode], BLOCK[mode])
    bad = ~np.isfinite(v).all(-1)
    mag = np.abs(np.where(bad[..., None], 0.0, v))
    amax = mag.max(-1)
    if mode == "mxfp4":
        e = np.frexp(amax)[1] - 1  # floor(log2)
        byte = np.where(amax > 0, np.clip(e - 2 + 127, 0, 254), 0)
        unit = np.ldexp(1.0, byte - 127)
        scales = np.where(bad, 255, byte)
    else:
        byte = nearest(amax / (6.0 * float(tensor_scale)), E4M3)
        unit = E4M3[byte] * float(tensor_scale)
        scales = np.where(bad, 127, byte)
    unit = unit[..., None]
    q = np.divide(mag, unit, out=np.zeros_like(mag), where=unit > 0)
    codes = nearest(q, E2M1) | (np.signbit(v).astype(np.int64) << 3)
    return codes.reshape(rows, k).astype(np.uint8), scales.astype(np.uint8)


def pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    packed = np.asarray(packed)
    return np.stack((packed & 15, packed >> 4), -1).reshape(packed.shape[0], -1)


def values(codes, scales, mode, tensor_scale=1.0):
    """float64 [rows, k] that codes (one a byte) and scales stand for."""
    codes = np.asarray(codes).astype(np.int64)
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = scale_values(scales, mode)[..., None]
    return (v.reshape(codes.shape[0], -1, BLOCK[mode]) * s).reshape(codes.shape) * float(tensor_scale)


def act(g, name):
    """act(g) and its derivative."""
    if name == "silu":
        s = 1.0 / (1.0 + np.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    c = np.sqrt(2.0 / np.pi)
    t = np.tanh(c * (g + 0.044715 * g**3))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g**2)
