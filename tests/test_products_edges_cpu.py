"""Refusals of pointers that are no addresses of their type: a kernel's access to one would be a misaligned address."""
import ctypes

import pytest

from test_products_cpu import BACK, CHECK, FFN, INT8, QUANT, refused


def at(address):
    return ctypes.c_void_p(address)  # never dereferenced: each call fails its checks first


WORK = 1 << 20  # bytes, enough for any copy of these sizes


@pytest.mark.parametrize("kind,place,address", [
    (0, 0, 258), (0, 0, 257), (1, 0, 257), (2, 0, 257), (2, 7, 258), (2, 7, 257),
])
def test_quantize_rows_refuses(kind, place, address, abft):
    args = list(QUANT)
    args[2] = kind
    args[place] = at(address)
    assert refused(abft, "abft_quantize_rows", *args)


@pytest.mark.parametrize("checksum,expect", [(258, 256), (257, 256), (256, 260), (256, 257)])
def test_quantize_rows_refuses_places_of_expected_sums(checksum, expect, abft):
    args = list(QUANT)
    args[8], args[9] = at(checksum), at(expect)
    assert refused(abft, "abft_quantize_rows", *args)


@pytest.mark.parametrize("address", [257, 258])
def test_column_checksum_refuses(address, abft):
    args = list(CHECK)
    args[4] = at(address)
    assert refused(abft, "abft_column_checksum", *args)


@pytest.mark.parametrize("kind,place,address", [(2, 2, 258), (2, 5, 257), (0, 9, 258), (1, 9, 257), (2, 9, 257)])
def test_int8_matmul_refuses(kind, place, address, abft):
    args = list(INT8)
    args[11] = kind
    args[place] = at(address)
    assert refused(abft, "abft_int8_matmul", *args)


@pytest.mark.parametrize("expect,rowdiff", [(260, 256), (256, 260), (256, 257)])
def test_int8_matmul_refuses_places_of_row_sums(expect, rowdiff, abft):
    args = list(INT8)
    args[12], args[13] = at(expect), at(rowdiff)
    assert refused(abft, "abft_int8_matmul", *args)


@pytest.mark.parametrize("place", [0, 2, 4, 11, 13, 15])
@pytest.mark.parametrize("kind", [1, 2])
def test_gated_ffn_refuses(place, kind, abft):
    args = list(FFN)
    args[9] = kind
    args[13], args[14], args[15], args[16] = at(256), 8, at(256), 8
    args[17], args[18] = at(256), WORK
    args[place] = at(257)
    assert refused(abft, "abft_gated_ffn", *args)


@pytest.mark.parametrize("place", [0, 2, 4, 6, 8, 10, 17, 19, 21])
@pytest.mark.parametrize("kind", [1, 2])
def test_gated_ffn_backward_refuses(place, kind, abft):
    args = list(BACK)
    args[15] = kind
    args[place] = at(257)
    assert refused(abft, "abft_gated_ffn_backward", *args)


def test_normal_distribution_fit_from_its_argument():
    """The fitted tail of the normal distribution, its coefficients read from the kernel's source, against erfc. In 64 bits
    it is off by 1.29e-7 at most (z = 0.057). Restated in float32 from g on: nine multiply-adds and the reciprocal lose at
    most 2^-24 of terms below 1.6 each, the exponent half a step of its size; z = g / sqrt2 is off by 1.5 * 2^-24 (constant
    and product), times |d ln erfc / d ln z| < z (z + sqrt(z^2 + 2))."""
    import math
    import os
    import re
    import numpy as np
    from conftest import PKG_NAME, ROOT
    src = open(os.path.join(ROOT, PKG_NAME, "csrc", "abft_products.cu")).read()
    body = src[src.index("float normal(float g)"):]
    body = body[:body.index("\n}\n")]
    f = np.float32
    c = [f(v) for v in re.findall(r"float f = (-?[\d.]+)f;|fmaf\(f, t, (-?[\d.]+)f\)", body) for v in v if v]
    assert len(c) == 9

    def erfc(z):
        return np.array([math.erfc(float(v)) for v in z])
    z = np.linspace(0, 9.2, 60001)
    t = 1 / (0.4 * z + 1)
    fit = t * np.exp(np.polyval([float(v) for v in c], t) - z * z)
    assert np.abs(fit / erfc(z) - 1).max() <= 1.3e-7
    g = np.linspace(0, 13, 60001).astype(f)
    z = (g * f(0.70710678118654752)).astype(f)
    t = (1 / (f(0.4).astype(np.float64) * z + 1).astype(f)).astype(f)
    p = np.full_like(t, c[0])
    for v in c[1:]:
        p = (p.astype(np.float64) * t + float(v)).astype(f)
    arg = (p.astype(np.float64) - z.astype(np.float64) ** 2).astype(f)
    got = t.astype(np.float64) * np.exp(arg.astype(np.float64))
    off = np.abs(got / erfc(g.astype(np.float64) * math.sqrt(0.5)) - 1)
    z = z.astype(np.float64)
    tol = 1.3e-7 + (10 * 1.6 + np.abs(arg) + 1.5 * z * (z + np.sqrt(z * z + 2))) * 2.0 ** -24
    assert (off <= tol).all()
