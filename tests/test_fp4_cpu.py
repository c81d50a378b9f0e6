"""CPU side of the microscaled 4-bit operators: the float64 checker against values worked out by
hand, and the refusals that need no device."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from aestrix_b200 import _lib, fp4
from oracle import fp4_ref as R


def test_checker_known_values():
    # mxfp4: amax 5 -> 2^(2 - 2) = 1; codes to nearest, ties to the even code
    x = np.zeros((1, 32))
    x[0, :9] = [5.0, 0.25, 0.26, 0.75, -1.25, 1.75, 2.5, 3.5, -0.1]
    codes, scales = R.quantize(x, "mxfp4")
    assert scales[0, 0] == 127
    assert list(codes[0, :9]) == [6, 0, 1, 2, 8 | 2, 4, 4, 6, 8]
    # nvfp4: amax 6 * 448 -> the largest scale; a block of zeros -> scale 0
    x = np.zeros((1, 32))
    x[0, 0] = 6 * 448.0
    x[0, 1] = 448.0 * 0.75
    codes, scales = R.quantize(x, "nvfp4")
    assert list(scales[0]) == [0x7E, 0] and list(codes[0, :2]) == [7, 2]
    assert R.values(codes, scales, "nvfp4")[0, 1] == 448.0
    # rounding of the scale to e4m3: 17 lies half-way between 16 and 18 and goes to the even mantissa
    x[0, 0], x[0, 1] = 6 * 17.0, 0.0
    assert R.scale_values(R.quantize(x, "nvfp4")[1], "nvfp4")[0, 0] == 16.0
    # the tensor's scale divides out
    a, b = R.quantize(x, "nvfp4"), R.quantize(x * 0.125, "nvfp4", 0.125)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_checker_e4m3_and_packing():
    assert R.E4M3[1] == 2.0**-9 and R.E4M3[8] == 2.0**-6 and R.E4M3[126] == 448.0
    assert (np.diff(R.E4M3) > 0).all()
    t = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, R.E4M3)
    codes = np.arange(32, dtype=np.uint8).reshape(1, 32) % 16
    assert R.pack(codes)[0, 0] == 0x10
    assert np.array_equal(R.unpack(R.pack(codes)), codes)


def test_checker_keeps_a_nan_to_its_block():
    x = np.ones((1, 64))
    x[0, 40] = np.nan
    for mode in ("mxfp4", "nvfp4"):
        v = R.values(*R.quantize(x, mode), mode)
        bad = np.isnan(v[0])
        lo = 40 // R.BLOCK[mode] * R.BLOCK[mode]
        assert bad[lo:lo + R.BLOCK[mode]].all() and bad.sum() == R.BLOCK[mode]


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_checker_activation_slope(act):
    g = np.linspace(-9, 9, 181)
    h = 1e-6
    slope = (R.act(g + h, act)[0] - R.act(g - h, act)[0]) / (2 * h)
    assert np.abs(slope - R.act(g, act)[1]).max() < 1e-8
    assert np.abs(R.act(g, act)[1]).max() < 1.2  # the bound the gated tests use


def test_refusals_without_a_device():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="mode"):
        fp4.quantize(x, "int4")
    with pytest.raises(TypeError, match="CUDA"):
        fp4.quantize(x)
    with pytest.raises(TypeError):
        fp4.quantize(x.to(torch.float16))
    with pytest.raises(TypeError):
        fp4.quantize(x.view(2, 2, 64))
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8)
    with pytest.raises(TypeError, match="CUDA"):
        fp4.dequantize(codes, scales, "nvfp4")
    with pytest.raises(TypeError, match="CUDA"):
        fp4.FP4Weight(codes, scales, "nvfp4")
    with pytest.raises(TypeError, match="FP4Weight"):
        fp4.fp4_mm(x, codes)
    with pytest.raises(TypeError, match="FP4Weight"):
        fp4.fp4_gated_mm(x, None, None)
    with pytest.raises(TypeError, match="FP4Weight"):
        fp4.fp4_mm_dgrad(x, codes)
    with pytest.raises(TypeError, match="FP4Weight"):
        fp4.fp4_gated_mm_dgrad(x, x, None, None)


def test_c_entry_points_refuse_null():
    L, bad = _lib.lib(), _lib.AEX_ERR_INVALID_ARG
    a = _lib.aex_fp4_mm_args()
    h = C.c_void_p()
    assert L.aex_fp4_quantize(None, None, 0, 32, 1, 32, 0, 1.0, None, None, None) == bad
    assert L.aex_fp4_dequantize(None, None, None, 1, 32, 0, 1.0, None, 0, 32, None) == bad
    assert L.aex_fp4weight_create(None, None, None, 1, 32, 0, 1.0, C.byref(h), None) == bad and not h.value
    assert L.aex_fp4weight_dequantize(None, None, None, 0, 32, None) == bad
    assert L.aex_fp4weight_shape(None, None, None) == bad
    assert L.aex_fp4_mm(None, None, C.byref(a), None) == bad
    assert L.aex_fp4_gated_mm(None, None, None, 0, C.byref(a), None) == bad
    assert L.aex_fp4_mm_dgrad(None, None, None, 8, 1, None, 0, 32, None, 0, None) == bad
    assert L.aex_fp4_gated_mm_dgrad(None, None, None, 0, None, 32, None, 8, 1, None, 32, None, 0, None) == bad
    assert L.aex_fp4_mm_workspace_bytes(None, 100, 1) == 0
    assert L.aex_fp4_gated_mm_workspace_bytes(None, 100, 1) == 0
    assert L.aex_fp4_mm_dgrad_workspace_bytes(None, 100) == 0
    assert L.aex_fp4_gated_mm_dgrad_workspace_bytes(None, 100) == 0
    L.aex_fp4weight_destroy(None)


def test_args_struct_matches_the_header():
    """The ctypes structure has the C structure's layout (offsets worked out from the header's types)."""
    f = _lib.aex_fp4_mm_args
    assert [getattr(f, n).offset for n, _ in f._fields_] == [0, 8, 16, 24, 28, 32, 40, 48, 56, 64, 72]
    assert C.sizeof(f) == 80


# ---------------------------------------------------------------- host arithmetic of the library

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def compiled(tmp_path, body):
    """What a program prints that includes the fp4 operators' host header."""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text('#include <cstdio>\n#include "fp4_internal.h"\nusing namespace aex::fp4;\n'
                   "int main() {\n" + body + "\nreturn 0; }\n")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    include = [os.path.join(ROOT, "aestrix_b200", "csrc"), os.path.join(cuda, "include")]
    subprocess.run(["g++", "-std=c++17", "-O1", str(src), "-o", str(exe)] + ["-I" + d for d in include], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()


LONGEST = 2**31 - 32  # columns: the largest multiple of 32 that an int holds


@pytest.mark.parametrize("k", [32, 8192, 2**27 - 32, 2**27, 2**28, 406039616, 2**30 + 32, LONGEST])
def test_conversions_count_their_units_in_range(tmp_path, k):
    """The conversions' kernels find a unit's row by a division that is exact below 2^31: every launch's
    units have to stay below that (124 rows of 406,039,616 columns in one launch left their last
    columns unwritten), a launch lies in whole tiles of 128 rows or within one, and the division is
    exact at either end of every row of a launch."""
    uprs = {k // 16, ((k - 1) // 256 + 1) * 16}  # of a plain matrix and of records
    got = compiled(tmp_path, f"""
        std::printf("%d\\n", records_along({k}));
        for (uint32_t upr : {{{", ".join(f"{u}u" for u in sorted(uprs))}}}) {{
          const FastDiv f = fast_div(upr);
          std::printf("%u %lld %u %u\\n", upr, (long long)slice_rows(upr), f.mul, f.shift);
        }}""")
    assert int(got[0]) == -(-k // 256)
    for i in range(1, len(got), 4):
        upr, rows, mul, shift = map(int, got[i:i + 4])
        assert rows >= 1 and rows * upr + 256 < 2**31
        assert rows % 128 == 0 or 128 % rows == 0
        for row in {0, 1, rows // 2, rows - 1} & set(range(rows)):
            for u in (row * upr, row * upr + upr - 1):
                assert (u if upr == 1 else (u * mul >> 32) >> shift) == row


def test_last_columns_of_the_widest_results(tmp_path):
    """A tile's columns past the last are told without leaving 32 bits: the end of the group that the
    last columns of a result of nearly 2^31 are in does (col + 16 > cols has no meaning there)."""
    cases = [(0, 16, 40), (32, 16, 40), (48, 16, 40), (LONGEST - 16, 16, LONGEST), (LONGEST, 16, LONGEST),
             (LONGEST + 16, 16, LONGEST), (2**31 - 16, 16, 2**31 - 1), (2**31 - 8, 8, 2**31 - 3)]
    got = compiled(tmp_path, "\n".join(f'std::printf("%d\\n", columns_within({a}, {b}, {c}));' for a, b, c in cases))
    assert [max(0, int(g)) for g in got] == [max(0, min(b, c - a)) for a, b, c in cases]


def test_overlap_of_two_matrices(tmp_path):
    """Byte by byte over small ones: never false where they share a byte, and true without one only
    where the pitches differ."""
    got = iter(compiled(tmp_path, """
        for (int rows = 1; rows < 4; ++rows)
          for (int aw = 1; aw < 5; ++aw) for (int ap = aw; ap < 7; ++ap)
            for (int bw = 1; bw < 5; ++bw) for (int bp = bw; bp < 7; ++bp)
              for (int b = 60; b < 120; ++b) std::putchar(overlap(80, aw, ap, b, bw, bp, rows) ? '1' : '0');""")[0])
    for rows in range(1, 4):
        for aw in range(1, 5):
            for ap in range(aw, 7):
                mine = {80 + r * ap + c for r in range(rows) for c in range(aw)}
                for bw in range(1, 5):
                    for bp in range(bw, 7):
                        for b in range(60, 120):
                            share = any(b + r * bp + c in mine for r in range(rows) for c in range(bw))
                            said = next(got) == "1"
                            assert said == share or (said and ap != bp), (rows, aw, ap, bw, bp, b)
