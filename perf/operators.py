"""Plain forms, cases and exact values of the framework's language-model products.

Operators: rows quantised to 8-bit integers, the 8-bit product with a scale for each token and channel and its exact
checksum test, and the gated feed-forward block with its backward pass. Matrices are row-major; weights are [N, K].
"""
import functools
import importlib
import math

import torch

own = False

PKG = "asynchronous_abft_for_mpi-cuda_architectures_b200"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one token's activations before a projection in decoding: latency alone
        {"name": "quantize_token", "op": "quantize", "T": 1, "K": 4096, "type": "bf16", "check": False},
        # a long prompt's (or a training batch's) activations, with the expected row sums of the product that follows
        {"name": "quantize_prompt", "op": "quantize", "T": 16384, "K": 4096, "type": "bf16", "check": True},
        # one decoded token through an 8-bit projection: quantise, multiply, verify
        {"name": "linear_token", "op": "linear", "T": 1, "K": 4096, "N": 16384, "type": "bf16", "check": True},
        # a batch of decoded tokens through an 8-bit projection
        {"name": "linear_batch", "op": "linear", "T": 48, "K": 8192, "N": 8192, "type": "f16", "check": False},
        # sizes that no tile divides and rows that no vector divides, unrounded results
        {"name": "product_odd", "op": "product", "T": 777, "K": 1001, "N": 1531, "type": "f32", "check": True},
        # the largest 8-bit product of a long prompt, verified
        {"name": "product_prompt", "op": "product", "T": 16384, "K": 4096, "N": 16384, "type": "bf16", "check": True},
        # one decoded token through the gated block
        {"name": "ffn_token", "op": "ffn", "T": 1, "K": 4096, "N": 16384, "type": "bf16", "act": "silu", "save": False},
        # a few drafted tokens at once, a smaller block
        {"name": "ffn_draft", "op": "ffn", "T": 13, "K": 2048, "N": 8192, "type": "f16", "act": "gelu", "save": False},
        # a ragged batch, odd widths, values kept for the backward pass
        {"name": "ffn_odd", "op": "ffn", "T": 1000, "K": 1001, "N": 1531, "type": "bf16", "act": "gelu_tanh", "save": True},
        # the forward half of a training step
        {"name": "ffn_train", "op": "ffn", "T": 8192, "K": 4096, "N": 16384, "type": "bf16", "act": "silu", "save": True},
        # gradients of a short batch
        {"name": "ffn_back_short", "op": "back", "T": 333, "K": 1024, "N": 4096, "type": "f16", "act": "gelu"},
        # the backward half of a training step
        {"name": "ffn_back_train", "op": "back", "T": 8192, "K": 4096, "N": 16384, "type": "bf16", "act": "silu"},
    ]


def draw(rng):
    def size(low, high):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        # half of the widths are multiples of 64, as models' are; the others fall anywhere
        return n if rng.random() < 0.5 else max(64, n // 64 * 64)

    while True:
        op = rng.choice(["quantize", "linear", "product", "ffn", "back"])
        T = int(round(math.exp(rng.uniform(0.0, math.log(16384)))))
        case = {"op": op, "T": T, "K": size(64, 16384), "type": rng.choice(["bf16", "f16"])}
        if op != "quantize":
            case["N"] = size(64, 16384)
        if op in ("ffn", "back"):
            case["act"] = rng.choice(["silu", "gelu", "gelu_tanh"])
            if op == "ffn":
                case["save"] = rng.random() < 0.5
        else:
            case["type"] = rng.choice(["bf16", "f16", "f32"])
            case["check"] = rng.random() < 0.5
        top = 2 * 16384 * 4096 * 16384
        if work(case)["flops"] <= (2 * top if op == "back" else top) and work(case)["bytes"] <= 3 << 30:
            return case


def work(case):
    T, K, e = case["T"], case["K"], SIZE[case["type"]]
    op = case["op"]
    if op == "quantize":
        more = 4 * K + 8 * T if case["check"] else 0
        return {"bytes": T * K * (e + 1) + 4 * T + more, "flops": 2 * T * K}
    N = case["N"]
    if op == "linear":
        more = 4 * K + 8 * T if case["check"] else 0
        return {"bytes": T * K * e + N * K + 4 * N + T * N * e + more, "flops": 2 * T * N * K}
    if op == "product":
        more = 16 * T if case["check"] else 0
        return {"bytes": T * K + N * K + 4 * (T + N) + T * N * e + more, "flops": 2 * T * N * K}
    if op == "ffn":
        return {"bytes": e * (T * K + 2 * N * K + T * N * (3 if case["save"] else 1)), "flops": 4 * T * N * K}
    return {"bytes": e * (3 * T * N + 2 * T * K + 4 * N * K), "flops": 8 * T * N * K}


def _activations(gen, T, K, dtype):
    """Rows as a layer sees them: their sizes differ, and a few channels are much larger than the others."""
    x = torch.randn(T, K, generator=gen, device="cuda")
    channel = 1.0 + 15.0 * (torch.rand(K, generator=gen, device="cuda") < 0.01)
    row = torch.exp(0.5 * torch.randn(T, 1, generator=gen, device="cuda"))
    return (x * channel * row).to(dtype)


def _int8(gen, rows, K):
    """8-bit rows on a pitch of 16 bytes, and their scales."""
    pitch = (K + 15) // 16 * 16
    q = torch.randn(rows, pitch, generator=gen, device="cuda").mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
    scale = torch.exp(0.3 * torch.randn(rows, generator=gen, device="cuda")) / 32.0
    return q[:, :K], scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, K, dtype = case["T"], case["K"], TYPES[case["type"]]
    op = case["op"]
    state = {"case": case}
    if op in ("quantize", "linear"):
        state["x"] = _activations(gen, T, K, dtype)
    if op in ("linear", "product"):
        # the weight is quantised and its column checksum taken once, when it is loaded
        state["w"], scale = _int8(gen, case["N"], K)
        state["w_scale"] = scale / math.sqrt(K)
    if op == "product":
        state["q"], state["q_scale"] = _int8(gen, T, K)
    if op in ("quantize", "linear", "product") and case["check"]:
        if op == "quantize":
            state["checksum"] = torch.randint(-20000, 20000, (K,), generator=gen, device="cuda", dtype=torch.int32)
        else:
            state["checksum"] = state["w"].sum(0, dtype=torch.int32)
        if op == "product":
            state["expect"] = (state["q"].double() @ state["checksum"].double()).to(torch.int64)
    if op in ("ffn", "back"):
        N = case["N"]
        state["x"] = torch.randn(T, K, generator=gen, device="cuda").to(dtype)
        for name in ("w_gate", "w_up"):
            state[name] = (torch.randn(N, K, generator=gen, device="cuda") / math.sqrt(K)).to(dtype)
        if op == "back":
            # what the forward pass kept, and the gradient that comes back through the block's second product
            for name in ("g", "u", "dh"):
                state[name] = torch.randn(T, N, generator=gen, device="cuda").to(dtype)
    return state


@functools.lru_cache(None)
def _products():
    return importlib.import_module(PKG).products


def _quantize(x, checksum):
    # in 64 bits: a quotient next to a half would be rounded to the wrong side in 32
    scale = (x.abs().amax(1).double() / 127.0).float()
    q = torch.round(x.double() / scale.double()[:, None]).nan_to_num_(0.0).clamp_(-127, 127)
    expect = None if checksum is None else (q @ checksum.double()).to(torch.int64)
    return q.to(torch.int8), scale, expect


def _product(q, q_scale, w, w_scale, expect, dtype):
    # 64 bits hold the integer sums exactly
    acc = q.double() @ w.double().t()
    rowdiff = None if expect is None else acc.sum(1).to(torch.int64) - expect
    return (acc * q_scale.double()[:, None] * w_scale.double()).to(dtype), rowdiff


def _act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if kind == "gelu":
        p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)


def run(state):
    case = state["case"]
    op, dtype = case["op"], TYPES[case["type"]]
    if op == "quantize":
        if own:
            return _products().quantize_rows(state["x"], checksum=state.get("checksum"))
        got = _quantize(state["x"], state.get("checksum"))
        return got if case["check"] else got[:2]
    if op == "linear":
        if own:
            p = _products()
            got = p.quantize_rows(state["x"], checksum=state.get("checksum"))
            return p.int8_matmul(got[0], got[1], state["w"], state["w_scale"], dtype=dtype,
                                 expect=got[2] if case["check"] else None)
        q, scale, expect = _quantize(state["x"], state.get("checksum"))
        got = _product(q, scale, state["w"], state["w_scale"], expect, dtype)
        return got if case["check"] else got[0]
    if op == "product":
        if own:
            return _products().int8_matmul(state["q"], state["q_scale"], state["w"], state["w_scale"], dtype=dtype,
                                           expect=state.get("expect"))
        got = _product(state["q"], state["q_scale"], state["w"], state["w_scale"], state.get("expect"), dtype)
        return got if case["check"] else got[0]
    x, w_gate, w_up = state["x"], state["w_gate"], state["w_up"]
    if op == "ffn":
        if own:
            return _products().gated_ffn(x, w_gate, w_up, activation=case["act"], save=case["save"])
        xf = x.float()
        g, u = xf @ w_gate.float().t(), xf @ w_up.float().t()
        h = _act(g, case["act"])[0] * u
        return (h.to(dtype), g.to(dtype), u.to(dtype)) if case["save"] else h.to(dtype)
    if own:
        return _products().gated_ffn_backward(state["dh"], x, w_gate, w_up, state["g"], state["u"],
                                              activation=case["act"])
    dh, u = state["dh"].float(), state["u"].float()
    a, slope = _act(state["g"].float(), case["act"])
    dg, du = dh * u * slope, dh * a
    xf = x.float()
    return ((dg @ w_gate.float() + du @ w_up.float()).to(dtype), (dg.t() @ xf).to(dtype), (du.t() @ xf).to(dtype))


def _exact_integers(a, b):
    """Integer sums of 8-bit rows; they stay far below 2^53, where float64 holds every integer."""
    return torch.einsum("nk,tk->tn", b.double(), a.double())


def _exact_quantize(x):
    """Nearest integers of x / scale found from the remainder, ties to even."""
    x = x.double()
    scale = (x.abs().max(1).values / 127.0).float().double()
    safe = torch.where(scale > 0, scale, 1.0)[:, None]
    low = torch.floor(x / safe)
    rest = x - low * safe
    up = (2 * rest > safe) | ((2 * rest == safe) & (low.remainder(2) == 1))
    q = torch.where(scale[:, None] > 0, (low + up.double()).clamp(-127, 127), 0.0)
    return q, scale


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        q, scale = _exact_quantize(state["x"])
        if not case["check"]:
            return q.to(torch.int8), scale
        return q.to(torch.int8), scale, (q.to(torch.int64) * state["checksum"].to(torch.int64)).sum(1)
    if op in ("linear", "product"):
        if op == "linear":
            q, q_scale = _exact_quantize(state["x"])
        else:
            q, q_scale = state["q"], state["q_scale"].double()
        acc = _exact_integers(q, state["w"])
        y = acc * (q_scale[:, None] * state["w_scale"].double()[None, :])
        if not case["check"]:
            return y
        # the checksum is that of the weight itself: a sound product leaves no difference
        return y, torch.zeros(case["T"], dtype=torch.int64, device="cuda")
    x, wg, wu = (state[n].double() for n in ("x", "w_gate", "w_up"))
    g = torch.einsum("tk,nk->tn", x, wg) if op == "ffn" else state["g"].double()
    u = torch.einsum("tk,nk->tn", x, wu) if op == "ffn" else state["u"].double()
    g.requires_grad_(op == "back")
    if case["act"] == "silu":
        a = torch.sigmoid(g) * g
    elif case["act"] == "gelu":
        a = g * 0.5 * torch.erfc(-g / math.sqrt(2.0))
    else:
        a = g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
    if op == "ffn":
        return (a * u, g, u) if case["save"] else a * u
    dh = state["dh"].double()
    (dg,) = torch.autograd.grad(a, g, dh * u)
    du = dh * a.detach()
    return (torch.einsum("tn,nk->tk", dg, wg) + torch.einsum("tn,nk->tk", du, wu), torch.einsum("tn,tk->nk", dg, x),
            torch.einsum("tn,tk->nk", du, x))
