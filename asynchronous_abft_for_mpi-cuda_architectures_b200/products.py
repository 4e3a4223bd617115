"""Products of language models: 8-bit matrix product with exact checksums, gated feed-forward block.

Each function enqueues on a CUDA stream (default: the inputs' device's current
stream) and returns immediately; matrices are row-major torch CUDA tensors
(views with a row pitch are fine), weights are N x K. Outputs and scratch are
allocated on that stream; the rows of an output whose width is not a multiple of
8 (of q: 16) lie on a pitch that is; inputs handed to a stream that is not the current
one are kept from reuse until its work is done. Nothing is kept between calls,
so they can be captured into CUDA graphs and issued on several streams. No
autograd graph is recorded: gated_ffn_backward gives the gradients.
"""
import contextlib
import ctypes

import torch

from ._lib import ABFT_ERR_CUDA, AbftError, check, lib

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}

MAX_EXTENT = 1 << 30         # rows and columns of any matrix
INT8_MAX_K = 131071          # 128 * 128 * K fits a 32-bit sum
INT8_MAX_ROWS = 1 << 24      # 127 * N fits a 32-bit checksum


def _matrix(t, name, dtypes, rows=None, cols=None, device=None):
    """Checks a row-major CUDA matrix and returns its row pitch in elements."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.ndim == 2):
        raise ValueError(f"{name} must be a 2-d CUDA tensor of {' or '.join(str(d)[6:] for d in dtypes)}")
    r, c = t.shape
    if (rows is not None and r != rows) or (cols is not None and c != cols):
        raise ValueError(f"{name} is {r} x {c}, need {'any' if rows is None else rows} x "
                         f"{'any' if cols is None else cols}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if c < 1 or r > MAX_EXTENT or c > MAX_EXTENT:
        raise ValueError(f"{name} is {r} x {c}: rows of at least one element and extents up to 2^30 are supported")
    pitch, step = t.stride()
    if step != 1 and c > 1:
        raise ValueError(f"{name} must be row-major (stride 1 along a row)")
    # the imaginary part of a conjugate, whose memory holds the other sign; longer rows of it have a stride of 2
    if c == 1 and t.is_neg():
        raise ValueError(f"{name} is a view with a pending negation: resolve_neg() it first")
    if r <= 1:
        return (c + 15) & ~15  # one row has no pitch: any that keeps it aligned
    if pitch < c:
        raise ValueError(f"{name}'s rows overlap (row stride {pitch} < {c})")
    return pitch


def _vector(t, name, dtype, n, device):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype and t.shape == (n,)
            and (t.is_contiguous() or n <= 1)):
        raise ValueError(f"{name} must be a contiguous CUDA vector of {n} {str(dtype)[6:]}")
    if n == 1 and t.is_neg():  # see _matrix; longer ones are not contiguous
        raise ValueError(f"{name} is a view with a pending negation: resolve_neg() it first")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, not {name!r}")
    return ACTIVATIONS[name]


_HERE = contextlib.nullcontext()
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _on(device, stream, inputs):
    """(raw stream, context to allocate and launch in) of one call."""
    if stream is None:
        # the raw forms: torch.cuda.current_stream() alone is 2 us, as long as a launch
        index = device.index
        return _raw_stream(index), _HERE if index == _current_device() else torch.cuda.device(device)
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    if stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    if stream != torch.cuda.current_stream(device):
        for t in inputs:
            if t is not None:
                t.record_stream(stream)
    return stream.cuda_stream, torch.cuda.stream(stream)


def _work(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _empty(rows, cols, pitch, dtype, device):
    return torch.empty_strided((rows, cols), (pitch, 1), dtype=dtype, device=device)


def check_waits(device=None):
    """Synchronous: waits for all work on the device, its other streams' too, and
    raises AbftError if a wait inside a product kernel has run out since this host
    thread's last check (its first: since the library was loaded). The kernels wait
    for their own copies and matrix instructions, each wait with a limit; after one
    that ran out, the results of the calls since the last check are void. Not to be
    called while a stream is being captured."""
    fault = ctypes.c_int()
    with torch.cuda.device(device):
        check(lib.abft_products_status(ctypes.byref(fault)), "abft_products_status")
    if fault.value:
        raise AbftError("products", ABFT_ERR_CUDA, "a wait inside a kernel did not end within the wait limit; the "
                                                   "results since the last check are void")


def quantize_rows(x, checksum=None, stream=None):
    """8-bit rows of x (T x K; float32, float16 or bfloat16): (q, scale) or, with
    checksum, (q, scale, expect).

    scale[t] = float32(max |x[t]| / 127); q[t] = x[t] / scale[t] rounded once to
    the nearest integer, ties to even (0 where the scale is 0). A row with an
    infinity or NaN has scale NaN and q = 0. For activations the scales are per
    token; for a weight (N x K) per channel. q lies on a pitch of 16 bytes.

    checksum: column_checksum() of the weight the rows will be multiplied with;
    expect[t] = sum_k q[t, k] * checksum[k] (int64) is what int8_matmul's rows
    have to sum to.
    """
    ldx = _matrix(x, "x", TYPES)
    T, K = x.shape
    dev = x.device
    if checksum is not None:
        _vector(checksum, "checksum", torch.int32, K, dev)
    s, where = _on(dev, stream, (x, checksum))
    with where:
        q = _empty(T, K, (K + 15) & ~15, torch.int8, dev)
        scale = torch.empty(T, dtype=torch.float32, device=dev)
        expect = None if checksum is None else torch.empty(T, dtype=torch.int64, device=dev)
        rc = lib.abft_quantize_rows(x.data_ptr(), ldx, TYPES[x.dtype], T, K, q.data_ptr(), (K + 15) & ~15,
             scale.data_ptr(), _ptr(checksum), _ptr(expect), s)
        if rc:
            check(rc, "abft_quantize_rows")
    return (q, scale) if checksum is None else (q, scale, expect)


def column_checksum(w, stream=None):
    """sum_n w[n, k] of an 8-bit weight (N x K), exact (int32 vector of K)."""
    ldw = _matrix(w, "w", (torch.int8,))
    N, K = w.shape
    if N < 1 or N > INT8_MAX_ROWS:
        raise ValueError(f"w has {N} rows: 1 to {INT8_MAX_ROWS} are supported")
    s, where = _on(w.device, stream, (w,))
    with where:
        out = torch.empty(K, dtype=torch.int32, device=w.device)
        rc = lib.abft_column_checksum(w.data_ptr(), ldw, N, K, out.data_ptr(), s)
        if rc:
            check(rc, "abft_column_checksum")
    return out


def int8_matmul(q, q_scale, w, w_scale, dtype=torch.bfloat16, expect=None, stream=None):
    """y[t, n] = (sum_k q[t, k] * w[n, k]) * q_scale[t] * w_scale[n].

    q (T x K) and w (N x K) are int8 (K <= 131071), the scales float32; the sums
    are exact and scaled in 32 bits, in this order (three roundings, and no overflow
    unless the result does), y has the given dtype (float32, float16, bfloat16).

    expect (from quantize_rows) verifies the product while it is computed:
    returns (y, rowdiff) with rowdiff[t] = sum_n sum_k q[t, k] * w[n, k] -
    expect[t] in exact integers, 0 for every sound row. A bit that flipped in q
    or w since they were encoded, or in a sum, leaves a difference in the rows it
    reached, unless its effects on a row's sum cancel (a flip in q[t, k] where the
    weight's column k sums to 0); the scaling after the sums is not covered.
    """
    ldq = _matrix(q, "q", (torch.int8,))
    T, K = q.shape
    dev = q.device
    ldw = _matrix(w, "w", (torch.int8,), cols=K, device=dev)
    N = w.shape[0]
    if N < 1 or K > INT8_MAX_K:
        raise ValueError(f"w is {tuple(w.shape)}: at least one row of at most {INT8_MAX_K} elements is supported")
    if dtype not in TYPES:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    _vector(q_scale, "q_scale", torch.float32, T, dev)
    _vector(w_scale, "w_scale", torch.float32, N, dev)
    if expect is not None:
        _vector(expect, "expect", torch.int64, T, dev)
    s, where = _on(dev, stream, (q, q_scale, w, w_scale, expect))
    with where:
        ld = (N + 7) & ~7
        y = _empty(T, N, ld, dtype, dev)
        rowdiff = None if expect is None else torch.empty(T, dtype=torch.int64, device=dev)
        qp, wp = q.data_ptr(), w.data_ptr()
        aligned = not ((qp | wp | ldq | ldw) & 15)  # then there is nothing to copy
        nbytes = 0 if aligned else lib.abft_int8_matmul_ws_bytes(qp, ldq, wp, ldw, T, N, K)
        work = _work(nbytes, dev)
        rc = lib.abft_int8_matmul(qp, ldq, q_scale.data_ptr(), wp, ldw, w_scale.data_ptr(), T, N, K, y.data_ptr(),
             ld, TYPES[dtype], _ptr(expect), _ptr(rowdiff), _ptr(work), nbytes, s)
        if rc:
            check(rc, "abft_int8_matmul")
    return y if expect is None else (y, rowdiff)


_HALF = (torch.float16, torch.bfloat16)


def _block(x, w_gate, w_up):
    ldx = _matrix(x, "x", _HALF)
    K, dev, same = x.shape[1], x.device, (x.dtype,)
    ldwg = _matrix(w_gate, "w_gate", same, cols=K, device=dev)
    N = w_gate.shape[0]
    ldwu = _matrix(w_up, "w_up", same, rows=N, cols=K, device=dev)
    if N < 1:
        raise ValueError("the weights have no rows")
    return ldx, ldwg, ldwu, x.shape[0], N, K


def gated_ffn(x, w_gate, w_up, activation="silu", save=False, stream=None):
    """h = act(x w_gate^T) * (x w_up^T); x is T x K, the weights N x K, float16 or bfloat16.

    activation: "silu", "gelu" or "gelu_tanh". Sums and activation are in 32
    bits, h is rounded once. save=True returns (h, g, u) with g = x w_gate^T and
    u = x w_up^T for gated_ffn_backward.
    """
    ldx, ldwg, ldwu, T, N, K = _block(x, w_gate, w_up)
    act = _activation(activation)
    dev = x.device
    s, where = _on(dev, stream, (x, w_gate, w_up))
    with where:
        ld = (N + 7) & ~7
        h = _empty(T, N, ld, x.dtype, dev)
        g = _empty(T, N, ld, x.dtype, dev) if save else None
        u = _empty(T, N, ld, x.dtype, dev) if save else None
        xp, gp, up = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr()
        aligned = not ((xp | gp | up) & 15 or (ldx | ldwg | ldwu) & 7)  # then there is nothing to copy
        nbytes = 0 if aligned else lib.abft_gated_ffn_ws_bytes(xp, ldx, gp, ldwg, up, ldwu, T, N, K)
        work = _work(nbytes, dev)
        rc = lib.abft_gated_ffn(xp, ldx, gp, ldwg, up, ldwu, T, N, K, TYPES[x.dtype], act, h.data_ptr(), ld,
             _ptr(g), ld, _ptr(u), ld, _ptr(work), nbytes, s)
        if rc:
            check(rc, "abft_gated_ffn")
    return (h, g, u) if save else h


def gated_ffn_backward(dh, x, w_gate, w_up, g, u, activation="silu", stream=None):
    """Gradients (dx, dw_gate, dw_up) of gated_ffn from dh (T x N) and the kept g, u.

    dgate = dh * u * act'(g) and dup = dh * act(g) are rounded to the tensors'
    type (they are operands of the products): in float16 one above 65504 is
    infinite, and with it its token's row of dx and its channel's row of the
    weight's gradient. Sums are in 32 bits and each gradient is rounded once.
    """
    ldx, ldwg, ldwu, T, N, K = _block(x, w_gate, w_up)
    act = _activation(activation)
    dev, same = x.device, (x.dtype,)
    ldd = _matrix(dh, "dh", same, T, N, dev)
    ldg = _matrix(g, "g", same, T, N, dev)
    ldu = _matrix(u, "u", same, T, N, dev)
    s, where = _on(dev, stream, (dh, x, w_gate, w_up, g, u))
    with where:
        ld = (K + 7) & ~7
        dx = _empty(T, K, ld, x.dtype, dev)
        dw_gate = _empty(N, K, ld, x.dtype, dev)
        dw_up = _empty(N, K, ld, x.dtype, dev)
        xp, gp, up = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr()
        nbytes = lib.abft_gated_ffn_backward_ws_bytes(xp, ldx, gp, ldwg, up, ldwu, T, N, K)
        work = _work(nbytes, dev)
        rc = lib.abft_gated_ffn_backward(dh.data_ptr(), ldd, xp, ldx, gp, ldwg, up, ldwu, g.data_ptr(), ldg,
             u.data_ptr(), ldu, T, N, K, TYPES[x.dtype], act, dx.data_ptr(), ld, dw_gate.data_ptr(), ld,
             dw_up.data_ptr(), ld, _ptr(work), nbytes, s)
        if rc:
            check(rc, "abft_gated_ffn_backward")
    return dx, dw_gate, dw_up
