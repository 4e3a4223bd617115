"""Refusals of the language-model products: every bad argument is an error before any CUDA call."""
import ctypes
import inspect
import math

import pytest
import torch

ERR = -1
FAKE = ctypes.c_void_p(256)  # never dereferenced: each call fails its checks first


def refused(abft, name, *args):
    rc = getattr(abft.lib, name)(*args)
    return rc == ERR and abft._lib.last_error().startswith(name)


# argument lists that pass every check but need a device; each case spoils one place
QUANT = [FAKE, 64, 2, 4, 64, FAKE, 64, FAKE, None, None, None]
CHECK = [FAKE, 64, 8, 64, FAKE, None]
INT8 = [FAKE, 64, FAKE, FAKE, 64, FAKE, 4, 8, 64, FAKE, 8, 2, None, None, None, 0, None]
FFN = [FAKE, 64, FAKE, 64, FAKE, 64, 4, 8, 64, 2, 0, FAKE, 8, None, 0, None, 0, None, 0, None]
BACK = [FAKE, 8, FAKE, 64, FAKE, 64, FAKE, 64, FAKE, 8, FAKE, 8, 4, 8, 64, 2, 0, FAKE, 64, FAKE, 64, FAKE, 64, FAKE,
        1 << 20, None]


@pytest.mark.parametrize("place,value", [
    (0, None), (1, 63), (2, 3), (2, -1), (3, -1), (3, (1 << 30) + 1), (4, 0), (4, (1 << 30) + 1), (5, None), (6, 63),
    (7, None),
    (8, FAKE),  # a checksum without a place for the expected sums
    (9, FAKE),  # and the other way round
])
def test_quantize_rows_refuses(abft, place, value):
    args = list(QUANT)
    args[place] = value
    assert refused(abft, "abft_quantize_rows", *args)


@pytest.mark.parametrize("place,value", [(0, None), (1, 63), (2, 0), (2, 16777217), (3, 0), (4, None)])
def test_column_checksum_refuses(abft, place, value):
    args = list(CHECK)
    args[place] = value
    assert refused(abft, "abft_column_checksum", *args)


@pytest.mark.parametrize("place,value", [
    (0, None), (1, 63), (2, None), (3, None), (4, 63), (5, None), (6, -1), (7, 0), (8, 0), (8, 131072), (9, None),
    (10, 7), (11, 3), (12, FAKE), (13, FAKE), (6, (1 << 30) + 1), (7, (1 << 30) + 1),
    (1, 65), (4, 65), (0, ctypes.c_void_p(264)), (3, ctypes.c_void_p(258)),  # operands to be copied, but no workspace
])
def test_int8_matmul_refuses(abft, place, value):
    args = list(INT8)
    args[place] = value
    assert refused(abft, "abft_int8_matmul", *args)


@pytest.mark.parametrize("place,value", [
    (0, None), (1, 63), (2, None), (3, 63), (4, None), (5, 63), (6, -1), (7, 0), (8, 0), (9, 0), (9, 3), (10, 3),
    (10, -1), (11, None), (12, 7), (13, FAKE), (15, FAKE), (6, (1 << 30) + 1), (7, (1 << 30) + 1), (8, (1 << 30) + 1),
    (1, 65), (3, 65), (5, 65), (2, ctypes.c_void_p(258)),  # operands to be copied, but no workspace
])
def test_gated_ffn_refuses(abft, place, value):
    args = list(FFN)
    args[place] = value
    assert refused(abft, "abft_gated_ffn", *args)


@pytest.mark.parametrize("place,value", [
    (0, None), (1, 7), (2, None), (3, 63), (4, None), (5, 63), (6, None), (7, 63), (8, None), (9, 7), (10, None),
    (11, 7), (12, -1), (13, 0), (14, 0), (15, 0), (16, 3), (17, None), (18, 63), (19, None), (20, 63), (21, None),
    (22, 63), (23, None), (23, ctypes.c_void_p(264)), (24, 1), (12, (1 << 30) + 1), (13, (1 << 30) + 1),
    (14, (1 << 30) + 1),
])
def test_gated_ffn_backward_refuses(abft, place, value):
    args = list(BACK)
    args[place] = value
    assert refused(abft, "abft_gated_ffn_backward", *args)


def test_no_tokens_is_no_work(abft):
    assert abft.lib.abft_quantize_rows(None, 64, 2, 0, 64, None, 64, None, None, None, None) == 0
    assert abft.lib.abft_int8_matmul(None, 64, None, FAKE, 64, FAKE, 0, 8, 64, None, 8, 2, None, None, None, 0,
                                     None) == 0
    assert abft.lib.abft_gated_ffn(None, 64, FAKE, 64, FAKE, 64, 0, 8, 64, 2, 0, None, 8, None, 0, None, 0, None, 0,
                                   None) == 0


def test_python_wrappers_refuse_host_tensors(abft):
    p = abft.products
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="x must be"):
        p.quantize_rows(x)
    with pytest.raises(ValueError, match="w must be"):
        p.column_checksum(x.to(torch.int8))
    with pytest.raises(ValueError, match="q must be"):
        p.int8_matmul(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0])
    with pytest.raises(ValueError, match="x must be"):
        p.gated_ffn(x.half(), x.half(), x.half())
    with pytest.raises(ValueError, match="x must be"):
        p.gated_ffn_backward(x, x, x, x, x, x)


def test_products_are_reachable_from_the_package(abft):
    names = {"quantize_rows", "column_checksum", "int8_matmul", "gated_ffn", "gated_ffn_backward"}
    assert names <= {n for n, f in vars(abft.products).items() if inspect.isfunction(f)}


def test_rounding_rule_on_ties():
    """The kernel's rule (guess, exact remainder, one step) restated in float32:
    it equals the real quotient rounded to even, next to every half."""
    import numpy as np
    f = np.float32
    rng = np.random.default_rng(3)
    for scale in rng.uniform(0.5, 1.0, 200).astype(f):
        halves = (np.arange(-127, 127) + f(0.5)) * np.float64(scale)
        x = halves.astype(f)
        x = np.concatenate([x, np.nextafter(x, f(0)), np.nextafter(x, f(1000)) , np.nextafter(x, f(-1000))])
        q = np.rint(x * (f(1) / scale)).astype(f)
        # x - q * scale, exact: at most 24 bits, so the 64-bit value is a float32 too
        r64 = x.astype(np.float64) - q.astype(np.float64) * np.float64(scale)
        r = r64.astype(f)
        assert (r.astype(np.float64) == r64).all()
        over = np.abs(f(2) * r) - scale
        step = (over > 0) | ((over == 0) & (q.astype(np.int32) % 2 != 0))
        q = np.clip(q + np.where(step, np.copysign(f(1), r), f(0)), -127, 127)
        # the real quotient in integers of 2^-60: nearest, ties to even
        from fractions import Fraction
        for xi, qi in zip(x[::17], q[::17]):
            want = max(-127, min(127, round(Fraction(float(xi)) / Fraction(float(scale)))))
            assert int(qi) == want, (float(xi), float(scale))


def test_normal_distribution_fit():
    """The fitted tail of the normal distribution, restated in float32 from the kernel's source, against erfc: the fit is
    off by 1.1e-7, nine multiply-adds and the reciprocal lose at most 2^-24 of terms below 1.6 each, and the exponent
    (z^2 + f, rounded once) half a step of its size."""
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
    z = np.linspace(0, 9.2, 40001).astype(f)
    t = (f(1) / (f(0.4) * z + f(1))).astype(f)
    p = np.full_like(t, c[0])
    for v in c[1:]:
        p = (p.astype(np.float64) * t + v).astype(f)
    arg = (p.astype(np.float64) - z.astype(np.float64) ** 2).astype(f)
    got = t.astype(np.float64) * np.exp(arg.astype(np.float64))
    want = np.array([math.erfc(float(v)) for v in z])
    tol = 1.1e-7 + 10 * 1.6 * 2.0 ** -24 + np.abs(arg) * 2.0 ** -24
    assert (np.abs(got / want - 1) <= tol).all()
