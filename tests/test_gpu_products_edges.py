"""The language-model products where calls meet limits: of shared memory, of views, of streams and threads, of a type's range.

Tolerances as in test_gpu_products: half a step for every rounding.
"""
import math
import os
import subprocess
import sys

import pytest
import torch

from conftest import PKG_NAME, ROOT
from test_gpu_products import HALF, assert_near, backward_def, block, gen, half_step, int_product, quantize_def, randn

pytestmark = pytest.mark.gpu


# ------------------------------------- checksums that fill shared memory ---

def expected_sums(q, c):
    return (q.cpu().to(torch.int64) * c.cpu().to(torch.int64)).sum(1).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("K", [8193, 12192, 12193, 12288, 12289, 16384, 16385])
@pytest.mark.parametrize("T", [1, 149, 400])
def test_wide_rows_with_a_checksum(T, K, dtype, abft):
    g = gen(T + K)
    x = randn(g, T, K).to(dtype)
    c = torch.randint(-2 ** 31, 2 ** 31 - 1, (K,), generator=g, device="cuda", dtype=torch.int32)
    q, scale, expect = abft.products.quantize_rows(x, checksum=c)
    want_q, want_s = quantize_def(x)
    assert torch.equal(q, want_q) and torch.equal(scale, want_s)
    assert torch.equal(expect, expected_sums(want_q, c))


FIRST = """
import importlib, sys, torch
sys.path.insert(0, {root!r})
p = importlib.import_module({pkg!r}).products
for dtype in (torch.float32, torch.float16, torch.bfloat16):
    x = torch.randn({T}, 12288, device="cuda").to(dtype)
    c = torch.randint(-20000, 20000, (12288,), device="cuda", dtype=torch.int32)
    q, scale, expect = p.quantize_rows(x, checksum=c)
    assert torch.equal(expect.cpu(), (q.cpu().long() * c.cpu().long()).sum(1))
    assert torch.equal(q, p.quantize_rows(x)[0])
"""


@pytest.mark.parametrize("T", [1, 400])
def test_wide_rows_with_a_checksum_come_first(T):
    """A process whose first rows have checksums of just 48 KB: no wider call has raised the kernel's limit before."""
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=ROOT, pkg=PKG_NAME, T=T)], capture_output=True, text=True,
                       timeout=300, env=dict(os.environ))
    assert r.returncode == 0, r.stderr[-2000:]


# ------------------------------------------------------ views of one buffer ---

@pytest.mark.parametrize("T", [4, 40, 200, 1000])
@pytest.mark.parametrize("order", [0, 1])
def test_weights_that_start_at_one_place(T, order, abft):
    """Two weights with the same first row and different pitches (every row and every second one of a buffer)."""
    N, K = 264, 136
    g = gen(T)
    rows = (randn(g, 2 * N, K) / math.sqrt(K)).bfloat16()
    views = rows[:N], rows[::2]
    wg, wu = views[order], views[1 - order]
    x, dh = randn(g, T, K).bfloat16(), randn(g, T, N).bfloat16()
    p = abft.products
    got = p.gated_ffn(x, wg, wu, save=True)
    want = p.gated_ffn(x, wg.contiguous(), wu.contiguous(), save=True)
    got += p.gated_ffn_backward(dh, x, wg, wu, *want[1:])
    want += p.gated_ffn_backward(dh, x, wg.contiguous(), wu.contiguous(), *want[1:])
    for a, b, name in zip(got, want, ("h", "g", "u", "dx", "dw_gate", "dw_up")):
        assert torch.equal(a, b), name


# ------------------------------------------------- the status of the waits ---

def run_out(abft, call):
    """Makes every wait of the kernels that `call` launches give up at once."""
    before = abft.lib.abft_set_wait_limit(0)
    try:
        call()
    finally:
        abft.lib.abft_set_wait_limit(before)


def test_status_waits_for_other_streams(abft):
    """A check right after a call on a side stream, whose kernel has not begun by then."""
    p = abft.products
    _, x, wg, wu = block(31, 200, 300, 128, torch.bfloat16)
    want = p.gated_ffn(x, wg, wu)
    p.check_waits()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # 0.2 s
    run_out(abft, lambda: p.gated_ffn(x, wg, wu, stream=side))
    with pytest.raises(abft.AbftError, match="wait"):
        p.check_waits()
    p.check_waits()
    h = p.gated_ffn(x, wg, wu, stream=side)
    p.check_waits()
    assert torch.equal(h, want)


def test_a_thread_is_told_of_a_fault_that_another_has_seen(abft):
    from concurrent.futures import ThreadPoolExecutor
    p = abft.products
    _, x, wg, wu = block(32, 200, 300, 128, torch.bfloat16)

    def told():
        try:
            p.check_waits(x.device)
        except abft.AbftError:
            return True
        return False
    with ThreadPoolExecutor(1) as other:
        told(), other.submit(told).result()
        assert not told() and not other.submit(told).result()
        run_out(abft, lambda: p.gated_ffn(x, wg, wu))
        assert other.submit(told).result() and told()
        assert not other.submit(told).result() and not told()
        run_out(abft, lambda: p.gated_ffn(x, wg, wu))
        assert told() and other.submit(told).result()
        assert not told() and not other.submit(told).result()


# --------------------------------------------------- after a call that failed ---

def test_a_refused_call_does_not_fail_the_next(abft):
    """An error that the CUDA runtime answers (a workspace larger than the GPU) is told once, by the call it belongs to."""
    import ctypes
    p, lib = abft.products, abft.lib
    w = torch.randint(-128, 128, (40, 64), generator=gen(2), device="cuda", dtype=torch.int8)
    want = p.column_checksum(w)
    most = 1 << 30
    one, zero, ws = (ctypes.c_int * 1)(most), (ctypes.c_int * 1)(0), ctypes.c_void_p()
    assert lib.abft_ws_bytes(most, most, most, 1, one, most) > torch.cuda.get_device_properties(0).total_memory
    assert lib.abft_ws_create(most, most, most, 1, one, zero, most, None, 0, ctypes.byref(ws)) == -2
    assert torch.equal(p.column_checksum(w), want)
    p.check_waits()


# ------------------------------------------------------ the types' ranges ---

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,N,K", [(3, 40, 520), (30, 72, 4096), (40, 72, 4096), (300, 300, 256), (1100, 2100, 128)])
def test_scales_over_the_whole_range(T, N, K, dtype, abft):
    """Row and channel scales from the smallest subnormal number to the largest: a result is right wherever it is a number
    of the type, however large the sum times the row's scale is."""
    g = gen(T + N + K)
    q = torch.randint(-127, 128, (T, K), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    sizes = torch.tensor([3e38, 2.6e36, 1e33, 3e29, 1.9e19, 1.7e19, 1.0, 1e-12, 1e-30, 2e-38, 1e-41, 1.5e-45], device="cuda")
    qs, ws = sizes[torch.arange(T, device="cuda") % 12], sizes.flip(0)[torch.arange(N, device="cuda") % 12]
    y = abft.products.int8_matmul(q, qs, w, ws, dtype=dtype)
    want = int_product(q, w) * qs.double()[:, None] * ws.double()
    most = torch.finfo(dtype).max
    inside, beyond = want.abs() < 0.99 * most, want.abs() > 1.01 * most
    # the sum to 32 bits and two products with scales, the last one down to the smallest numbers: half a step each
    tol = half_step(want, dtype) + want.abs() * (3 * 2.0 ** -24) * 1.01 + 2.0 ** -150
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    assert_near(torch.where(inside, y.double(), zero), torch.where(inside, want, zero), tol)
    assert torch.equal(y[beyond].double(), torch.sign(want[beyond]) * math.inf)
    assert inside.any() and beyond.any()


@pytest.mark.parametrize("T", [3, 40, 200])
def test_scales_of_either_sign(T, abft):
    """A caller's own scales may be negative."""
    g = gen(T)
    q = torch.randint(-127, 128, (T, 2000), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (70, 2000), generator=g, device="cuda", dtype=torch.int8)
    sign = 1 - 2 * (torch.arange(200, device="cuda") % 2)
    qs, ws = 2e37 * sign[:T], 1e-33 * sign[:70]
    want = int_product(q, w) * qs.double()[:, None] * ws.double()
    y = abft.products.int8_matmul(q, qs, w, ws, dtype=torch.float32)
    assert_near(y, want, half_step(want, torch.float32) + want.abs() * (3 * 2.0 ** -24) * 1.01)


def test_wide_range_rows_are_quantised_and_multiplied(abft):
    """Rows near the largest numbers through a weight of small ones: the results are ordinary numbers."""
    p, g = abft.products, gen(7)
    for T in (2, 100):
        x, w = (randn(g, T, 1000) * 1e37).bfloat16(), randn(g, 96, 1000) * 1e-35
        wq, ws = p.quantize_rows(w)
        q, s, e = p.quantize_rows(x, checksum=p.column_checksum(wq))
        y, diff = p.int8_matmul(q, s, wq, ws, dtype=torch.float32, expect=e)
        want = int_product(q, wq) * s.double()[:, None] * ws.double()
        assert_near(y, want, half_step(want, torch.float32) + want.abs() * (3 * 2.0 ** -24) * 1.01)
        assert (diff == 0).all() and want.abs().max() < 1e7


@pytest.mark.parametrize("dtype", HALF)
def test_quantize_every_value(dtype, abft):
    """Every finite value of the type, under row maxima over its whole range, in rows held in registers and in wider ones."""
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)].cuda()
    f = torch.finfo(dtype)
    tops = [f.max, f.max * 0.7, f.smallest_normal, f.smallest_normal * f.eps, f.smallest_normal * f.eps * 5]
    tops += [1.37 * 2.0 ** e for e in range(int(math.log2(f.smallest_normal)), int(math.log2(f.max)), 5)]
    tops = torch.tensor(tops, dtype=torch.float64, device="cuda").to(dtype)
    wide = torch.where(v.double().abs() <= tops.double()[:, None], v, torch.zeros_like(v))
    short = torch.nn.functional.pad(wide, (0, -len(v) % 4095)).view(-1, 4095)
    short = torch.cat([tops.repeat_interleave(short.shape[0] // len(tops))[:, None], short], 1)
    for x in (wide, short, short[:, :200]):
        q, scale = abft.products.quantize_rows(x)
        want_q, want_s = quantize_def(x)
        assert torch.equal(scale, want_s) and torch.equal(q, want_q)


@pytest.mark.parametrize("T", [6, 200, 600])
def test_float16_gradients_at_their_limit(T, abft):
    """dgate is an operand of the products in the tensors' type: below 65504 the gradients are as ever; above, it is
    infinite there, in the token's row of dx and the channel's row of dw_gate alone."""
    dtype, N, K = torch.float16, 136, 72
    r, x, wg, wu = block(T, T, N, K, dtype)
    g, u, dh = (randn(r, T, N).to(dtype) for _ in range(3))
    t, n = T // 2, 77
    g[t, n], u[t, n] = 0.5, 2.0
    slope = torch.sigmoid(torch.tensor(0.5)) * (1 + 0.5 * (1 - torch.sigmoid(torch.tensor(0.5))))
    p = abft.products
    dh[t, n] = 65000 / 2 / float(slope)
    clean = p.gated_ffn_backward(dh, x, wg, wu, g, u)
    # dgate = 65000 here, so that results pass the type's largest number where |x[t]| > 1.01: infinite by their own rounding
    for grad, (want, tol) in zip(clean, backward_def(dh, x, wg, wu, g, u, "silu", dtype)):
        most = torch.finfo(dtype).max
        inside, beyond = want.abs() + tol < most, want.abs() - tol > most * (1 + torch.finfo(dtype).eps)
        zero = torch.zeros((), dtype=torch.float64, device="cuda")
        assert_near(torch.where(inside, grad.double(), zero), torch.where(inside, want, zero), tol)
        assert torch.equal(grad[beyond].double(), torch.sign(want[beyond]) * math.inf)
    dh[t, n] = 60000
    dx, dwg, dwu = p.gated_ffn_backward(dh, x, wg, wu, g, u)
    rows = torch.arange(T, device="cuda") != t
    channels = torch.arange(N, device="cuda") != n
    assert torch.equal(dx[rows], clean[0][rows]) and not dx[t].isfinite().any()
    assert torch.equal(dwg[channels], clean[1][channels]) and not dwg[n].isfinite().any()
    assert torch.equal(dwu[channels], clean[2][channels])


def test_threads_at_once(abft):
    """Four threads with streams of their own, calls of every size among one another: each gets its own bits."""
    from concurrent.futures import ThreadPoolExecutor
    p = abft.products
    shapes = [(1, 300, 264), (40, 1000, 1032), (200, 264, 136), (1100, 1300, 96)]

    def inputs(i):
        T, N, K = shapes[i]
        r, x, wg, wu = block(40 + i, T, N, K, torch.bfloat16)
        return x, wg, wu, randn(r, T, N).bfloat16()

    def run(x, wg, wu, dh):
        h, g, u = p.gated_ffn(x, wg, wu, save=True)
        w, ws = p.quantize_rows(wg)
        q, s, e = p.quantize_rows(x, checksum=p.column_checksum(w))
        return (h, *p.gated_ffn_backward(dh, x, wg, wu, g, u), *p.int8_matmul(q, s, w, ws, expect=e))
    sets = [inputs(i) for i in range(4)]
    wants = [run(*s) for s in sets]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = run(*sets[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, wants[i])):
                    return False
        return True
    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))


# -------------------------------------------------------------- other views ---

def test_views_with_a_pending_sign_are_refused(abft):
    """The imaginary part of a conjugate holds the numbers with the other sign; resolved, it is a tensor like any other."""
    p, g = abft.products, gen(8)
    column = torch.randn(5, 1, dtype=torch.complex64, generator=g, device="cuda").conj().imag
    one = torch.randn(1, dtype=torch.complex64, generator=g, device="cuda").conj().imag
    assert column.is_neg() and one.is_neg()
    q, s = p.quantize_rows(column.resolve_neg())
    assert torch.equal(q.float(), 127 * column.resolve_neg().sign())
    for bad in (lambda: p.quantize_rows(column), lambda: p.quantize_rows(column[:, 0].unsqueeze(1)),
                lambda: p.quantize_rows(column[:1]), lambda: p.int8_matmul(q, s, q[:1], one),
                lambda: p.int8_matmul(q[:1], one, q, s)):
        with pytest.raises(ValueError):
            bad()
