"""The language-model products against their definitions in 64 bits.

Tolerances are sums of what each step may lose: half a step of every rounding
(finfo.eps / 2 relative), and for a sum of n products in 32 bits n steps of
2^-23 of the sum of magnitudes (a tensor core may cut instead of round).
"""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
ACTS = ["silu", "gelu", "gelu_tanh"]

# T, N, K: one token to several tiles, edges of tiles, odd and even widths
SHAPES = [
    (1, 1, 1), (1, 256, 512), (2, 40, 24), (3, 7, 1001), (8, 129, 64), (9, 33, 65), (16, 300, 136), (17, 64, 2048),
    (31, 8, 8), (33, 257, 200), (64, 1531, 40), (65, 128, 128), (128, 96, 777), (129, 130, 264), (200, 520, 72),
    (257, 513, 1000), (1000, 640, 320), (515, 1280, 136),
]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def half_step(want, dtype):
    """Half a step of rounding `want` to dtype, the smallest numbers' included."""
    f = torch.finfo(dtype)
    return want.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def sum_loss(a, b, n):
    """What n additions in 32 bits may lose of a b^T."""
    return (a.abs().double() @ b.abs().double().t()) * (n + 8) * 2.0 ** -23


def assert_near(got, want, tol, what=""):
    off = (got.double() - want).abs() - tol
    bad = ~(off <= 0)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by {float(off.max()):.3g}, " \
                          f"first at {bad.nonzero()[0].tolist()}"


def pitched(t, pad=8, shift=0):
    """The same matrix as a view into a wider buffer of a filling that must not matter."""
    wide = torch.full((t.shape[0], t.shape[1] + pad + shift), 99, dtype=t.dtype, device=t.device)
    if t.is_floating_point():
        wide.fill_(float("nan"))
    view = wide[:, shift:shift + t.shape[1]]
    view.copy_(t)
    return view


# ------------------------------------------------------------ definitions ---

def quantize_def(x):
    x = x.double()
    scale = (x.abs().amax(1) / 127).float()
    scale = torch.where(x.isfinite().all(1), scale, math.nan)
    s = scale.double()[:, None]
    q = torch.where(s > 0, torch.round(x / s), torch.zeros_like(x)).clamp(-127, 127)
    return q.to(torch.int8), scale


def same(a, b):
    """Equal values, NaN at the same places."""
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def int_product(q, w):
    return q.double() @ w.double().t()  # whole numbers below 2^53


def act_def(g, kind):
    # forms without 1 + (something near -1), which would lose the tails in 64 bits too
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return g * 0.5 * torch.erfc(-g * math.sqrt(0.5))
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))  # (1 + tanh z) / 2 = sigmoid(2 z)


def slope_def(g, kind):
    g = g.clone().requires_grad_()
    return torch.autograd.grad(act_def(g, kind).sum(), g)[0]


# ----------------------------------------------------------- quantisation ---

@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 4096), (3, 7), (2, 16), (5, 129), (300, 1001), (70, 8192), (2, 50000),
                                 (66000, 24), (4, 17), (1, 131071)])
def test_quantize_rows(T, K, dtype, abft):
    g = gen(T * 7 + K)
    x = (randn(g, T, K) * torch.exp(3 * randn(g, T, 1))).to(dtype)
    c = torch.randint(-2 ** 31, 2 ** 31 - 1, (K,), generator=g, device="cuda", dtype=torch.int32)
    for xi in (x, pitched(x, 8), pitched(x, 3, 1)):
        q, scale, expect = abft.products.quantize_rows(xi, checksum=c)
        want_q, want_s = quantize_def(x)
        assert same(scale, want_s)
        assert torch.equal(q, want_q)
        assert q.stride(0) % 16 == 0 or T == 1
        assert torch.equal(expect, (want_q.cpu().to(torch.int64) * c.cpu().to(torch.int64)).sum(1).cuda())
    q2, s2 = abft.products.quantize_rows(x)
    assert torch.equal(q2, q) and same(s2, scale)


def test_quantize_ties_and_extremes(abft):
    """Quotients at and next to a half, subnormal rows, the largest numbers, zeros of both signs."""
    rows = []
    base = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    for s in (1.0, 2.0 ** -40, 2.0 ** 100, 0.7310585975646973, 2.0 ** -126, 2.0 ** -133, 1.1e-38, 3e-39):
        h = (base * s).float()
        rows += [h, torch.nextafter(h, torch.zeros_like(h)), torch.nextafter(h, torch.full_like(h, 3e38))]
        for r in rows[-3:]:
            r[0] = 127 * torch.tensor(s).float()  # the scale
    for v in (3.4028234e38, 1e-45, 1.4e-43, 9e-44, 8.8e-44, 1.18e-38):
        r = torch.zeros(254)
        r[3], r[5], r[7] = v, -v / 2, v / 3
        rows.append(r)
    rows.append(torch.zeros(254))
    rows.append(-torch.zeros(254))
    x = torch.stack(rows).cuda()
    q, scale = abft.products.quantize_rows(x)
    want_q, want_s = quantize_def(x)
    assert same(scale, want_s)
    assert torch.equal(q, want_q)


def test_quantize_every_bf16(abft):
    """Every finite bfloat16, in rows whose largest value differs by one step."""
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    v = v[torch.isfinite(v)].cuda()
    v = v[v.abs() <= 200]
    x = torch.stack([torch.cat([v[v.abs() <= m], torch.zeros(int((v.abs() > m).sum()), device="cuda").bfloat16()])
                     for m in (200, 100.5, 3.0, 1.0, 0.0077, 1e-30, 1e-38)])
    q, scale = abft.products.quantize_rows(x)
    want_q, want_s = quantize_def(x)
    assert torch.equal(scale, want_s) and torch.equal(q, want_q)


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_rows_that_are_not_finite(value, dtype, abft):
    """Their scale is NaN and their integers 0, so the product's row is NaN; the other rows are as before."""
    g = gen(5)
    x = randn(g, 6, 300).to(dtype)
    w, ws = abft.products.quantize_rows(randn(g, 40, 300))
    c = abft.products.column_checksum(w)
    clean_q, clean_s, clean_e = abft.products.quantize_rows(x, checksum=c)
    x[2, 299] = value
    x[4, 0] = value
    q, s, e = abft.products.quantize_rows(x, checksum=c)
    keep = torch.tensor([0, 1, 3, 5], device="cuda")
    assert torch.equal(q[keep], clean_q[keep]) and torch.equal(s[keep], clean_s[keep])
    assert torch.equal(e[keep], clean_e[keep])
    assert (q[2] == 0).all() and (q[4] == 0).all() and s[2].isnan() and s[4].isnan() and e[2] == 0 and e[4] == 0
    y, diff = abft.products.int8_matmul(q, s, w, ws, dtype=dtype, expect=e)
    assert y[2].isnan().all() and y[4].isnan().all() and y[keep].isfinite().all() and (diff == 0).all()


@pytest.mark.parametrize("N,K", [(1, 1), (5, 33), (1000, 1001), (4097, 64), (16384, 520), (3, 5000)])
def test_column_checksum(N, K, abft):
    w = torch.randint(-128, 128, (N, K), generator=gen(N + K), device="cuda", dtype=torch.int8)
    for wi in (w, pitched(w, 16), pitched(w, 2, 3)):
        assert torch.equal(abft.products.column_checksum(wi), w.sum(0, dtype=torch.int32))


# ---------------------------------------------------------- 8-bit product ---

@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("T,N,K", SHAPES + [(40, 4096, 4096), (1, 5000, 8192), (1500, 2050, 96),
                                            # pairs of SMs; K split over 8 and over 5 or 6 CTAs
                                            (1000, 4096, 2060), (48, 520, 16000), (330, 500, 9000)])
def test_int8_matmul(T, N, K, dtype, abft):
    g = gen(T + 3 * N + 5 * K)
    q = torch.randint(-128, 128, (T, K), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    # scales that keep every result inside float16
    qs = torch.exp(randn(g, T)).clamp(0.1, 8) / 128
    ws = torch.exp(randn(g, N)).clamp(0.1, 8) / 128 / math.sqrt(K) / 8
    acc = int_product(q, w)
    want = acc * qs.double()[:, None] * ws.double()
    expect = torch.randint(-2 ** 40, 2 ** 40, (T,), generator=g, device="cuda", dtype=torch.int64)
    # the sum to 32 bits and two products with scales: half a step each
    tol = half_step(want, dtype) + want.abs() * (3 * 2.0 ** -24) * 1.01
    for qi, wi in ((q, w), (pitched(q, 16 + (-K) % 16), pitched(w, 32 + (-K) % 16)), (pitched(q, 1), pitched(w, 2, 5))):
        y, diff = abft.products.int8_matmul(qi, qs, wi, ws, dtype=dtype, expect=expect)
        assert_near(y, want, tol, "y")
        assert torch.equal(diff, acc.sum(1).to(torch.int64) - expect)
    assert torch.equal(abft.products.int8_matmul(q, qs, w, ws, dtype=dtype), y)


@pytest.mark.parametrize("T,N", [(1, 24), (40, 24), (130, 260)])
def test_int8_sums_at_their_limit(T, N, abft):
    """K = 131071 of -128 * -128 is the largest 32-bit sum; -128 * 127 the lowest."""
    K = abft.products.INT8_MAX_K
    q = torch.full((T, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((N, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    w[1::2] = 127
    one_t, one_n = torch.ones(T, device="cuda"), torch.ones(N, device="cuda")
    expect = torch.zeros(T, dtype=torch.int64, device="cuda")
    y, diff = abft.products.int8_matmul(q, one_t, w, one_n, dtype=torch.float32, expect=expect)
    assert (y[:, 0::2].double() == torch.tensor(16384.0 * K).float().double().item()).all()
    assert (y[:, 1::2].double() == torch.tensor(-16256.0 * K).float().double().item()).all()
    assert (diff == (N - N // 2) * 16384 * K - (N // 2) * 16256 * K).all()


@pytest.mark.parametrize("T,N,K", [(1, 300, 512), (7, 4096, 256), (50, 300, 1001), (300, 520, 264)])
def test_checksum_finds_what_changed(T, N, K, abft):
    """A bit that flips in the weight or in the tokens after they were encoded shows in the rows it reaches, and only there."""
    g = gen(T + N)
    p = abft.products
    w, ws = p.quantize_rows(randn(g, N, K))
    c = p.column_checksum(w)
    q, qs, e = p.quantize_rows(randn(g, T, K).bfloat16(), checksum=c)
    y, diff = p.int8_matmul(q, qs, w, ws, expect=e)
    assert (diff == 0).all()
    q[:, K // 2] = torch.arange(T, device="cuda").remainder(3).to(torch.int8)  # rows that meet the weight with 0, 1, 2
    q, qs, e = p.quantize_rows(q.float() * 127, checksum=c)
    bad = torch.empty_strided(w.shape, w.stride(), dtype=w.dtype, device="cuda").copy_(w)
    bad[N - 1, K // 2] ^= 64
    change = int(bad[N - 1, K // 2]) - int(w[N - 1, K // 2])
    _, diff = p.int8_matmul(q, qs, bad, ws, expect=e)
    assert torch.equal(diff, q[:, K // 2].to(torch.int64) * change)
    _, diff = p.int8_matmul(q, qs, w, ws, expect=e)
    assert (diff == 0).all()
    row = T - 1
    q[row, 0] ^= 1
    _, diff = p.int8_matmul(q, qs, w, ws, expect=e)
    step = 1 if int(q[row, 0]) & 1 else -1
    assert int(diff[row]) == step * int(c[0]) and (diff[:row] == 0).all()


# ------------------------------------------------------ gated feed-forward ---

def block(seed, T, N, K, dtype):
    g = gen(seed)
    x = randn(g, T, K).to(dtype)
    wg, wu = ((randn(g, N, K) * (1.5 / math.sqrt(K))).to(dtype) for _ in range(2))
    return g, x, wg, wu


def forward_def(x, wg, wu, kind, dtype):
    """(h, g, u) in 64 bits and what each may be off."""
    K = x.shape[1]
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    lg, lu = sum_loss(x, wg, K), sum_loss(x, wu, K)
    a = act_def(g, kind)
    # |act'| < 1.13; the exponential and the division lose a few steps of 2^-23 each, and act() near its zero is
    # as exact as its argument (absolute, below |g| 2^-19)
    la = 1.13 * lg + g.abs() * 2.0 ** -19
    h = a * u
    lh = la * u.abs() + a.abs() * lu + la * lu
    return (h, half_step(h, dtype) + 1.01 * lh), (g, half_step(g, dtype) + 1.01 * lg), (u, half_step(u, dtype) + 1.01 * lu)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T,N,K", SHAPES + [(1, 4096, 4096), (24, 2048, 4096), (1100, 1300, 96),
                                            # pairs of SMs; K split over the CTAs of a cluster
                                            (1000, 2050, 1100), (48, 1000, 4100), (333, 500, 9000)])
def test_gated_ffn(T, N, K, dtype, abft):
    kind = ACTS[(T + N) % 3]
    _, x, wg, wu = block(T + 2 * N + K, T, N, K, dtype)
    wants = forward_def(x, wg, wu, kind, dtype)
    p = abft.products
    for xi, gi, ui in ((x, wg, wu), (pitched(x, 8 + (-K) % 8), pitched(wg, 16 + (-K) % 8), pitched(wu, 8 + (-K) % 8)),
                       (pitched(x, 1, 1), pitched(wg, 2), wu)):
        got = p.gated_ffn(xi, gi, ui, activation=kind, save=True)
        for y, (want, tol), name in zip(got, wants, "hgu"):
            assert_near(y, want, tol, name)
        assert torch.equal(p.gated_ffn(xi, gi, ui, activation=kind), got[0])


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("T", [1, 20, 200])
def test_activation_over_its_range(T, kind, dtype, abft):
    """K = 1 makes g any chosen number: tails where exp overflows, zeros, the largest numbers."""
    vals = torch.cat([torch.linspace(-30, 30, 400), torch.tensor([-60000., -3000., -100., -89., -1e-6, 0., 1e-6, 88., 100.,
                                                                  3000., 60000.])])
    wg = vals.cuda().to(dtype)[:, None]
    wu = torch.ones_like(wg)
    x = torch.ones(T, 1, dtype=dtype, device="cuda")
    (h, tol), _, _ = forward_def(x, wg, wu, kind, dtype)
    assert_near(abft.products.gated_ffn(x, wg, wu, activation=kind), h, tol, kind)


def backward_def(dh, x, wg, wu, g, u, kind, dtype):
    dh, xd, wgd, wud, g, u = (t.double() for t in (dh, x, wg, wu, g, u))
    a, s = act_def(g, kind), slope_def(g, kind)
    dg, du = dh * u * s, dh * a
    # the slope is below 1.13 and off by a few steps of 2^-21 in its terms; dg and du are rounded once to the type
    ldg = half_step(dg, dtype) + (dh * u).abs() * (2.0 ** -19) * (1 + g.abs().clamp(max=16))
    ldu = half_step(du, dtype) + (dh * g).abs() * 2.0 ** -19
    T, N = dh.shape

    def product(a, la, b, n):  # a b^T with a off by la
        return a @ b.t(), la @ b.abs().t() + ((a.abs() + la) @ b.abs().t()) * (n + 8) * 2.0 ** -23
    d1, l1 = product(dg, ldg, wgd.t(), 2 * N)
    d2, l2 = product(du, ldu, wud.t(), 2 * N)
    g1, k1 = product(dg.t(), ldg.t(), xd.t(), T)
    g2, k2 = product(du.t(), ldu.t(), xd.t(), T)
    return [(w, half_step(w, dtype) + 1.01 * l) for w, l in ((d1 + d2, l1 + l2), (g1, k1), (g2, k2))]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T,N,K", SHAPES + [(4096, 136, 64), (700, 1000, 1300),
                                            # pairs of SMs; N split; T split
                                            (1000, 1100, 4100), (333, 4096, 1000), (9000, 130, 200)])
def test_gated_ffn_backward(T, N, K, dtype, abft):
    kind = ACTS[(T + K) % 3]
    r, x, wg, wu = block(2 * T + N + K, T, N, K, dtype)
    g, u, dh = (randn(r, T, N).to(dtype) for _ in range(3))
    wants = backward_def(dh, x, wg, wu, g, u, kind, dtype)
    p = abft.products
    even = (-K) % 8
    for args in ((dh, x, wg, wu, g, u),
                 (pitched(dh, 8 + (-N) % 8), pitched(x, 8 + even), pitched(wg, 8 + even), pitched(wu, 24 + even),
                  pitched(g, 16 + (-N) % 8), pitched(u, 8 + (-N) % 8)),
                 (pitched(dh, 1), pitched(x, 1, 1), pitched(wg, 2), wu, pitched(g, 3, 2), u)):
        for y, (want, tol), name in zip(p.gated_ffn_backward(*args, activation=kind), wants, ("dx", "dw_gate", "dw_up")):
            assert_near(y, want, tol, name)


@pytest.mark.parametrize("kind", ACTS)
def test_slope_over_its_range(kind, abft):
    """One token and K = 1: dw_gate is the slope itself, tails and the largest numbers included."""
    dtype = torch.bfloat16
    vals = torch.cat([torch.linspace(-20, 20, 500), torch.tensor([-1e30, -3e4, -200., 0., 200., 3e4, 1e30])])
    g = vals.cuda().to(dtype)[None]
    N = g.shape[1]
    one = torch.ones(1, N, device="cuda", dtype=dtype)
    w, x = torch.zeros(N, 1, device="cuda", dtype=dtype), torch.ones(1, 1, device="cuda", dtype=dtype)
    _, dw_gate, dw_up = abft.products.gated_ffn_backward(one, x, w, w, g, one, activation=kind)
    want = slope_def(g.double().clamp(-1e4, 1e4), kind)[0]
    assert_near(dw_gate[:, 0], want, half_step(want, dtype) * 2.1 + 2.0 ** -19 * (1 + g.double().abs()[0].clamp(max=16)))
    want = act_def(g.double(), kind)[0]
    # the sigmoid is 1 / (1 + e^-z) by __fdividef, which is 0 for a divisor above 2^126: the value lost is below 2^-126,
    # times g
    tail = g.double().abs()[0].clamp(max=16) * 2.0 ** -126
    assert_near(dw_up[:, 0], want, half_step(want, dtype) * 2.1 + want.abs() * 2.0 ** -19 + tail)


@pytest.mark.parametrize("kind", ACTS)
def test_gradients_against_differences(kind, abft):
    """The gradients along a random direction against central differences of the 64-bit definition."""
    dtype, (T, N, K) = torch.bfloat16, (40, 72, 56)
    r, x, wg, wu = block(9, T, N, K, dtype)
    dh = randn(r, T, N).to(dtype)
    _, g, u = abft.products.gated_ffn(x, wg, wu, activation=kind, save=True)
    got = abft.products.gated_ffn_backward(dh, x, wg, wu, g, u, activation=kind)

    def loss(x, wg, wu):
        return (dh.double() * act_def(x @ wg.t(), kind) * (x @ wu.t())).sum()
    leaves = [t.double() for t in (x, wg, wu)]
    # g and u are kept in the type: half a step each in both factors, then dg / du and the result: 4 half steps of the
    # magnitudes that meet in the sum (act' < 1.13, |act(g)| <= |g|), and 2 more for the second derivative's (< 1.6 |g| step)
    gd, ud = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    size = dh.double().abs() * (gd.abs() * (1 + ud.abs()) + 2 * ud.abs())
    for i, grad in enumerate(got):
        d = randn(r, *leaves[i].shape).double()
        eps = 1e-5
        hi, lo = (loss(*[t + s * eps * d if j == i else t for j, t in enumerate(leaves)]) for s in (1, -1))
        want = (hi - lo) / (2 * eps)
        if i == 0:
            reach = d.abs() @ (wg.double().abs() + wu.double().abs()).t()
        else:
            reach = x.double().abs() @ d.abs().t()
        tol = 6 * torch.finfo(dtype).eps / 2 * (size * reach).sum() + (grad.double() * d).abs().sum() * torch.finfo(dtype).eps / 2
        assert abs(float((grad.double() * d).sum() - want)) <= float(tol)


def test_values_that_are_not_finite_stay_in_their_rows(abft):
    """A token's NaN or infinity reaches its own row of h and no other; a channel's its own column."""
    for T in (4, 40, 300):
        _, x, wg, wu = block(3, T, 200, 96, torch.bfloat16)
        clean = abft.products.gated_ffn(x, wg, wu)
        x[1, 5] = math.nan
        wg[7, 3] = math.inf
        got = abft.products.gated_ffn(x, wg, wu)
        assert got[1].isnan().all()
        rows = torch.ones(T, dtype=torch.bool, device="cuda")
        rows[1] = False
        cols = torch.ones(200, dtype=torch.bool, device="cuda")
        cols[7] = False
        assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
        assert not got[rows][:, 7].isfinite().all()


# ------------------------------------------------- how a user's program calls ---

def test_no_tokens(abft):
    p = abft.products
    for dtype in HALF:
        x = torch.empty(0, 48, dtype=dtype, device="cuda")
        w = torch.ones(32, 48, dtype=dtype, device="cuda")
        q, s = p.quantize_rows(x)
        assert q.shape == (0, 48) and s.shape == (0,)
        wq, ws = p.quantize_rows(w)
        c = p.column_checksum(wq)
        q, s, e = p.quantize_rows(x, checksum=c)
        y, diff = p.int8_matmul(q, s, wq, ws, expect=e)
        assert y.shape == (0, 32) and diff.shape == (0,)
        h, g, u = p.gated_ffn(x, w, w, save=True)
        assert h.shape == g.shape == u.shape == (0, 32)
        dx, dwg, dwu = p.gated_ffn_backward(h, x, w, w, g, u)
        torch.cuda.synchronize()
        assert dx.shape == (0, 48) and (dwg == 0).all() and (dwu == 0).all() and dwg.shape == dwu.shape == (32, 48)


def test_refusals_of_device_tensors(abft):
    p = abft.products
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    q, s = p.quantize_rows(x)
    wq, ws = p.quantize_rows(w)
    e = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (lambda: p.quantize_rows(x.double()), lambda: p.quantize_rows(x.t()), lambda: p.quantize_rows(x[0]),
                lambda: p.quantize_rows(x[:1].expand(4, 64)), lambda: p.quantize_rows(x[:, :0]),
                lambda: p.quantize_rows(x, checksum=torch.zeros(63, dtype=torch.int32, device="cuda")),
                lambda: p.quantize_rows(x, checksum=torch.zeros(64, dtype=torch.int64, device="cuda")),
                lambda: p.column_checksum(wq[:0]), lambda: p.column_checksum(w),
                lambda: p.int8_matmul(q, s, wq[:, :63], ws), lambda: p.int8_matmul(q, s[:3], wq, ws),
                lambda: p.int8_matmul(q, s, wq, ws.double()), lambda: p.int8_matmul(q, s, wq, ws.cpu()),
                lambda: p.int8_matmul(q, s, wq, ws, dtype=torch.int32),
                lambda: p.int8_matmul(q, s, wq, ws, expect=e[:2]), lambda: p.int8_matmul(q, s, wq[:0], ws[:0]),
                lambda: p.gated_ffn(x, w, w.half()), lambda: p.gated_ffn(x, w, w[:7]),
                lambda: p.gated_ffn(x.float(), w.float(), w.float()),
                lambda: p.gated_ffn(x, w, w, activation="relu"), lambda: p.gated_ffn(x, w[:, ::2], w),
                lambda: p.gated_ffn_backward(x, x, w, w, x, x),
                lambda: p.gated_ffn_backward(x[:, :8], x, w, w, x[:, :8], x[:3, :8])):
        with pytest.raises(ValueError):
            bad()


def everything(p, x, w, wg, wu, dh):
    """One run of all the operators together: a trained block's weight served in 8 bits."""
    h, g, u = p.gated_ffn(x, wg, wu, save=True)
    grads = p.gated_ffn_backward(dh, x, wg, wu, g, u)
    wq, ws = p.quantize_rows(w)
    c = p.column_checksum(wq)
    q, s, e = p.quantize_rows(h, checksum=c)
    y, diff = p.int8_matmul(q, s, wq, ws, dtype=x.dtype, expect=e)
    return (h, g, u, *grads, q, s, y, diff)


@pytest.mark.parametrize("T", [1, 5, 33, 200])
def test_streams_and_graphs(T, abft):
    """The same bits eagerly, on another stream, from two captured graphs replayed in turn and side by side."""
    dtype, N, K = torch.bfloat16, 260, 136
    p = abft.products
    sets = []
    for seed in (1, 2):
        r, x, wg, wu = block(seed, T, N, K, dtype)
        sets.append((x, (randn(r, 70, N) / 16).to(dtype), wg, wu, randn(r, T, N).to(dtype)))
    wants = [[t.clone() for t in everything(p, *s)] for s in sets]
    for s, want in zip(sets, wants):
        assert (want[-1] == 0).all()
        for a, b in zip(everything(p, *s), want):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    h = p.gated_ffn(*(sets[0][i] for i in (0, 2, 3)), stream=side)
    q, sc = p.quantize_rows(h, stream=side)
    side.synchronize()
    assert torch.equal(h, wants[0][0]) and torch.equal(q, wants[0][6]) and torch.equal(sc, wants[0][7])
    with torch.cuda.stream(side):
        for s in sets:
            everything(p, *s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(everything(p, *s))
        graphs.append(gr)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for o, want in zip(outs, wants):
            for a, b in zip(o, want):
                assert torch.equal(a, b)


def test_outputs_keep_to_their_rows_and_columns(abft):
    """Through the C ABI, into views of wider and longer buffers: nothing around them is written."""
    lib = abft.lib

    def framed(rows, cols, dtype, pad):
        t = torch.full((rows + 2, cols + pad), 77, dtype=dtype, device="cuda")
        return t, t[1:rows + 1, :cols]

    def untouched(t, rows, cols):
        t = t.clone()
        t[1:rows + 1, :cols] = 77
        return bool((t == 77).all())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for T, N, K in ((1, 37, 64), (20, 37, 72), (40, 130, 64), (150, 261, 104)):
        for pad in (3, 8, 11):
            _, x, wg, wu = block(T, T, N, K, torch.bfloat16)
            H, h = framed(T, N, torch.bfloat16, pad)
            G, g = framed(T, N, torch.bfloat16, pad)
            U, u = framed(T, N, torch.bfloat16, pad)
            args = (x.data_ptr(), K, wg.data_ptr(), K, wu.data_ptr(), K, T, N, K)
            nb = lib.abft_gated_ffn_ws_bytes(*args)
            work = torch.empty(max(nb, 16), dtype=torch.uint8, device="cuda")
            assert lib.abft_gated_ffn(*args, 2, 0, h.data_ptr(), N + pad, g.data_ptr(), N + pad, u.data_ptr(), N + pad,
                                      work.data_ptr(), nb, stream) == 0
            for got, want in zip((h, g, u), abft.products.gated_ffn(x, wg, wu, save=True)):
                assert torch.equal(got, want)
            assert untouched(H, T, N) and untouched(G, T, N) and untouched(U, T, N)
            dh = torch.randn(T, N, device="cuda", dtype=torch.bfloat16)
            DX, dx = framed(T, K, torch.bfloat16, pad)
            DG, dg = framed(N, K, torch.bfloat16, pad)
            DU, du = framed(N, K, torch.bfloat16, pad)
            nb = lib.abft_gated_ffn_backward_ws_bytes(*args)
            work = torch.full((nb + 64,), 55, dtype=torch.uint8, device="cuda")
            assert lib.abft_gated_ffn_backward(dh.data_ptr(), N, *args[:6], g.data_ptr(), N + pad, u.data_ptr(), N + pad,
                                               T, N, K, 2, 0, dx.data_ptr(), K + pad, dg.data_ptr(), K + pad,
                                               du.data_ptr(), K + pad, work.data_ptr(), nb, stream) == 0
            for got, want in zip((dx, dg, du), abft.products.gated_ffn_backward(dh, x, wg, wu, g, u)):
                assert torch.equal(got, want)
            assert untouched(DX, T, K) and untouched(DG, N, K) and untouched(DU, N, K) and (work[nb:] == 55).all()
            wq, ws = abft.products.quantize_rows(wg)
            Q, q = framed(T, K, torch.int8, pad)
            s = torch.full((T + 1,), 77.0, device="cuda")
            assert lib.abft_quantize_rows(x.data_ptr(), K, 2, T, K, q.data_ptr(), K + pad, s.data_ptr(), None, None,
                                          stream) == 0
            want = abft.products.quantize_rows(x)
            assert torch.equal(q, want[0]) and torch.equal(s[:T], want[1]) and s[T] == 77 and untouched(Q, T, K)
            for code, dtype in enumerate((torch.float32, torch.float16, torch.bfloat16)):
                Y, y = framed(T, N, dtype, pad)
                args = (q.data_ptr(), K + pad, wq.data_ptr(), wq.stride(0))
                nb = lib.abft_int8_matmul_ws_bytes(*args, T, N, K)
                work = torch.empty(max(nb, 16), dtype=torch.uint8, device="cuda")
                assert lib.abft_int8_matmul(args[0], args[1], s.data_ptr(), args[2], args[3], ws.data_ptr(), T, N, K,
                                            y.data_ptr(), N + pad, code, None, None, work.data_ptr(), nb, stream) == 0
                assert torch.equal(y, abft.products.int8_matmul(want[0], want[1], wq, ws, dtype=dtype))
                assert untouched(Y, T, N)
                nb and refuse_small_workspace(abft, args, s, ws, T, N, K, y, pad, code, work, nb, stream)


FRESH = """
import importlib, sys, torch
sys.path.insert(0, {root!r})
p = importlib.import_module({pkg!r}).products
T, N, K = {shape}
gen = torch.Generator(device="cuda").manual_seed(1)
x, wg, wu, dh = (torch.randn(*s, generator=gen, device="cuda").bfloat16() for s in ((T, K), (N, K), (N, K), (T, N)))
def run():
    h, g, u = p.gated_ffn(x, wg, wu, save=True)
    grads = p.gated_ffn_backward(dh, x, wg, wu, g, u)
    wq, ws = p.quantize_rows(wg)
    c = p.column_checksum(wq)
    q, s, e = p.quantize_rows(x, checksum=c)
    return (h, *grads, *p.int8_matmul(q, s, wq, ws, expect=e))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = run()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(captured, run()):
    assert torch.equal(a, b)
assert (captured[-1] == 0).all()
p.check_waits()
"""


@pytest.mark.parametrize("shape", [(1, 300, 256), (40, 300, 256), (300, 2000, 256), (2100, 2560, 130)])
def test_first_call_is_captured(shape):
    """A process whose first call of every kernel is recorded into a graph."""
    import os
    import subprocess
    import sys
    from conftest import PKG_NAME, ROOT
    r = subprocess.run([sys.executable, "-c", FRESH.format(root=ROOT, pkg=PKG_NAME, shape=shape)], capture_output=True,
                       text=True, timeout=300, env=dict(os.environ))
    assert r.returncode == 0, r.stderr[-2000:]


def test_offsets_past_32_bits(abft):
    """Operands and results of more than 2^31 elements: the last rows as well as the first."""
    p, g = abft.products, gen(4)
    T, N, K = 70000, 40000, 32
    q = torch.randint(-128, 128, (T, K), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    one_t, one_n = torch.ones(T, device="cuda"), torch.ones(N, device="cuda")
    e = (q.double() @ w.sum(0, dtype=torch.int32).double()).to(torch.int64)
    y, diff = p.int8_matmul(q, one_t, w, one_n, dtype=torch.bfloat16, expect=e)
    assert (diff == 0).all() and T * N > 2 ** 31
    for rows in (slice(0, 200), slice(T - 200, T)):
        assert torch.equal(y[rows], int_product(q[rows], w).bfloat16())
    q8, s8, e8 = p.quantize_rows(y, checksum=torch.ones(N, dtype=torch.int32, device="cuda"))
    for rows in (slice(0, 3), slice(T - 3, T)):
        want_q, want_s = quantize_def(y[rows])
        assert torch.equal(q8[rows], want_q) and torch.equal(s8[rows], want_s)
        assert torch.equal(e8[rows], want_q.to(torch.int64).sum(1))
    del y, q8
    # few tokens and many channels on a wide pitch
    wide = torch.empty(33000, 70000, dtype=torch.bfloat16, device="cuda")
    wg, wu = wide[:, :64], wide[:, 64:128]
    wg.normal_(generator=g)
    wu.normal_(generator=g)
    x = randn(g, 3, 64).bfloat16()
    want = p.gated_ffn(x, wg.contiguous(), wu.contiguous(), save=True)
    for a, b in zip(p.gated_ffn(x, wg, wu, save=True), want):
        assert torch.equal(a, b)
    x = randn(g, 140, 64).bfloat16()
    h, gs, us = p.gated_ffn(x, wg, wu, save=True)
    dh = randn(g, *h.shape).bfloat16()
    for a, b in zip(p.gated_ffn_backward(dh, x, wg, wu, gs, us),
                    p.gated_ffn_backward(dh, x, wg.contiguous(), wu.contiguous(), gs, us)):
        assert torch.equal(a, b)


def test_many_tokens_and_channels(abft):
    """More rows than a grid's second dimension, in each place a row can stand."""
    p = abft.products
    for T, N, K in ((70000, 16, 24), (40, 140000, 16)):
        r, x, wg, wu = block(5, T, N, K, torch.bfloat16)
        wants = forward_def(x, wg, wu, "silu", torch.bfloat16)
        got = p.gated_ffn(x, wg, wu, save=True)
        for y, (want, tol) in zip(got, wants):
            assert_near(y, want, tol)
        dh = randn(r, T, N).bfloat16()
        for y, (want, tol) in zip(p.gated_ffn_backward(dh, x, wg, wu, *got[1:]),
                                  backward_def(dh, x, wg, wu, *got[1:], "silu", torch.bfloat16)):
            assert_near(y, want, tol)
    w = torch.full((1 << 24, 3), -128, dtype=torch.int8, device="cuda")
    w[:, 1] = 127
    assert p.column_checksum(w).tolist() == [-2 ** 31, 127 << 24, -2 ** 31]


def test_streams_by_handle_and_freed_inputs(abft):
    """A raw stream handle works like the stream; inputs dropped right after a call on another stream stay until it ran."""
    p = abft.products
    _, x, wg, wu = block(8, 600, 520, 264, torch.float16)
    want = p.gated_ffn(x, wg, wu)
    assert torch.equal(p.gated_ffn(x, wg, wu, stream=torch.cuda.current_stream().cuda_stream), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    h = p.gated_ffn(x, wg, wu, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(h, want)
    got = []
    for _ in range(20):
        a, b, c = x.clone(), wg.clone(), wu.clone()
        side.wait_stream(torch.cuda.current_stream())
        got.append(p.gated_ffn(a, b, c, stream=side))
        del a, b, c
        torch.empty_like(x).fill_(7), torch.empty_like(wg).fill_(7), torch.empty_like(wu).fill_(7)
    torch.cuda.synchronize()
    for h in got:
        assert torch.equal(h, want)
    with pytest.raises(ValueError):
        p.gated_ffn(x, wg.cpu(), wu)


def test_many_launches_in_a_row(abft):
    """Thousands of launches that follow each other without a pause, kernels of pairs of SMs among them: each starts up
    while the one before it ends, and every result is the first one's. The host watches the time."""
    import time
    p, (T, N, K) = abft.products, (1024, 2048, 1024)
    r, x, wg, wu = block(13, T, N, K, torch.bfloat16)
    h, g, u = p.gated_ffn(x, wg, wu, save=True)
    dh = randn(r, T, N).bfloat16()
    w, ws = p.quantize_rows(wg)
    q, s, e = p.quantize_rows(x, checksum=p.column_checksum(w))
    want = [h, *p.gated_ffn_backward(dh, x, wg, wu, g, u), *p.int8_matmul(q, s, w, ws, expect=e)]
    for _ in range(10):
        for _ in range(200):
            got = [p.gated_ffn(x, wg, wu), *p.gated_ffn_backward(dh, x, wg, wu, g, u),
                   *p.int8_matmul(q, s, w, ws, expect=e)]
        done, began = torch.cuda.Event(), time.monotonic()
        done.record()
        while not done.query():
            assert time.monotonic() - began < 20
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    p.check_waits()


@pytest.mark.parametrize("T,N,K", [(40, 1024, 4096), (200, 300, 128), (3000, 4096, 64)])
def test_waits_that_run_out(T, N, K, abft):
    """With a limit of 0 every wait inside the kernels gives up at once: they
    return, the status says so once, and the next calls are right again."""
    p = abft.products
    _, x, wg, wu = block(11, T, N, K, torch.bfloat16)
    q, s = p.quantize_rows(x)
    w, ws = p.quantize_rows(wg)
    h, g, u = p.gated_ffn(x, wg, wu, save=True)
    want = [t.clone() for t in (h, *p.gated_ffn_backward(h, x, wg, wu, g, u), p.int8_matmul(q, s, w, ws))]
    p.check_waits()
    before = abft.lib.abft_set_wait_limit(0)
    try:
        for call in (lambda: p.gated_ffn(x, wg, wu), lambda: p.gated_ffn_backward(h, x, wg, wu, g, u),
                     lambda: p.int8_matmul(q, s, w, ws)):
            call()
            with pytest.raises(abft.AbftError, match="wait"):
                p.check_waits()
            p.check_waits()
    finally:
        abft.lib.abft_set_wait_limit(before)
    for a, b in zip((p.gated_ffn(x, wg, wu), *p.gated_ffn_backward(h, x, wg, wu, g, u), p.int8_matmul(q, s, w, ws)), want):
        assert torch.equal(a, b)
    p.check_waits()


def refuse_small_workspace(abft, args, s, ws, T, N, K, y, pad, code, work, nb, stream):
    rc = abft.lib.abft_int8_matmul(args[0], args[1], s.data_ptr(), args[2], args[3], ws.data_ptr(), T, N, K, y.data_ptr(),
                                   N + pad, code, None, None, work.data_ptr(), nb - 1, stream)
    assert rc == -1 and "workspace" in abft._lib.last_error()


@pytest.mark.parametrize("T", [3, 160])
def test_a_block_is_trained_and_served(T, abft):
    """A feed-forward layer as a program uses the operators together: a training step (the second product's
    gradients by plain products), then all three weights quantised and the layer served in 8 bits, verified."""
    p, dtype, N, K = abft.products, torch.bfloat16, 264, 120
    r, x, wg, wu = block(17, T, N, K, dtype)
    wd = (randn(r, K, N) / math.sqrt(N)).to(dtype)
    h, g, u = p.gated_ffn(x, wg, wu, save=True)
    dy = randn(r, T, K).to(dtype)
    dh = (dy.float() @ wd.float()).to(dtype)
    dx, dwg, dwu = p.gated_ffn_backward(dh, x, wg, wu, g, u)
    for got, (want, tol) in zip((dx, dwg, dwu), backward_def(dh, x, wg, wu, g, u, "silu", dtype)):
        assert_near(got, want, tol)
    wg, wu = wg - (0.01 * dwg).to(dtype), wu - (0.01 * dwu).to(dtype)
    served = {}
    for name, w in (("gate", wg), ("up", wu), ("down", wd)):
        q, s = p.quantize_rows(w)
        served[name] = (q, s, p.column_checksum(q))

    def linear(x, name, dt):
        wq, ws, c = served[name]
        q, s, e = p.quantize_rows(x, checksum=c)
        y, diff = p.int8_matmul(q, s, wq, ws, dtype=dt, expect=e)
        assert (diff == 0).all()
        want = int_product(q, wq) * s.double()[:, None] * ws.double()
        assert_near(y, want, half_step(want, dt) + want.abs() * 4 * 2.0 ** -24)
        return y
    gate, up = linear(x, "gate", torch.float32), linear(x, "up", torch.float32)
    y = linear(act_def(gate, "silu") * up, "down", dtype)
    assert y.shape == (T, K)
