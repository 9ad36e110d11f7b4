"""Operators over a user's logits for the whole catalogue, on the device.

``quantize_blocks`` / ``matmul_blocks``  logits as a product of 8-bit operands with a scale for each
                                        block of 128 values (GMF models: user factors x item factors)
``sample_items``                        items drawn from the logits: temperature, top-k, top-p, min-p
``distill_loss`` / ``distill_grad`` / ``distill_loss_grad``
                                        a student's logits against a teacher's list of best items

Every tensor lives on one HIP device and the work is enqueued on that device's current stream; no
call synchronises, and what a call needs beside its outputs it allocates from torch's caching
allocator, so calls on several streams and captured graphs share nothing.  Matrices may be strided
over their rows; their last dimension is dense.  A wrong argument raises ``ValueError``.

The reference scores a list of items for one user and keeps the best (movierec/trt_client.py:43-57).
"""

import ctypes
import math
import numbers

import torch

from . import _native as N

BLOCK = 128   # values that share a scale
_DTYPES = {torch.float32: N.NCF_F32, torch.bfloat16: N.NCF_BF16, torch.float16: N.NCF_F16}
_FP8 = torch.float8_e4m3fn


def _dtype_code(name, dtype):
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError("%s must be float32, bfloat16 or float16, got %s" % (name, dtype))
    return code


def _matrix(name, t, device=None):
    """Checks a 2-D device tensor with a dense last dimension; returns its row distance."""
    if not torch.is_tensor(t) or t.dim() != 2:
        raise ValueError("%s must be a 2-D tensor" % name)
    _on_device(name, t, device)
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError("%s: the last dimension must be dense (stride 1), got stride %d" % (name, t.stride(1)))
    return t.stride(0)


def _on_device(name, t, device=None):
    if not t.is_cuda:
        raise ValueError("%s must be on a HIP device (got %s); there is no CPU path" % (name, t.device))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, the other tensors on %s" % (name, t.device, device))


def _dense(name, t, shape, dtype, device):
    """Checks a contiguous tensor of this shape and type."""
    if not torch.is_tensor(t) or tuple(t.shape) != tuple(shape):
        raise ValueError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(getattr(t, "shape", ()))))
    _on_device(name, t, device)
    if t.dtype != dtype:
        raise ValueError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t


def _call(fn, device, *args):
    """The library call on ``device``'s current stream (its last argument), on that device."""
    idx = device.index
    if idx == torch.cuda.current_device():
        N.check(fn(*args, N.stream_handle(idx)))
    else:
        with torch.cuda.device(idx):
            N.check(fn(*args, N.stream_handle(idx)))


def _workspace(size_fn, d, device):
    """Scratch for the call that struct ``d`` describes (None where it needs none)."""
    nbytes = ctypes.c_size_t()
    N.check(size_fn(ctypes.byref(d), ctypes.byref(nbytes)))
    return torch.empty(nbytes.value, dtype=torch.uint8, device=device) if nbytes.value else None


def quantize_blocks(x, tile=False):
    """``x`` (rows, cols; float32, bfloat16 or float16) as 8-bit values with block scales: ``(q, scale)``
    with ``q`` float8_e4m3fn (rows, cols) and ``scale`` float32, one per 128 consecutive values of a
    row, (rows, ceil(cols / 128)); ``tile=True``: one per 128 x 128 tile, (ceil(rows / 128),
    ceil(cols / 128)) — for weights.  scale = max(max|x| / 448, 2^-126), q = e4m3(x / scale).
    Rows of ``q`` start at multiples of 16 bytes."""
    ld = _matrix("x", x)
    code = _dtype_code("x", x.dtype)
    rows, cols = x.shape
    if cols < 1:
        raise ValueError("x has no columns")
    kb = (cols + BLOCK - 1) // BLOCK
    q = torch.empty(rows, (cols + 15) // 16 * 16, dtype=_FP8, device=x.device)
    scale = torch.empty((rows + BLOCK - 1) // BLOCK if tile else rows, kb, dtype=torch.float32, device=x.device)
    if rows:
        _call(N.lib().ncf_quantize_blocks, x.device, x.data_ptr(), code, rows, cols, ld, 1 if tile else 0,
              q.data_ptr(), q.stride(0), scale.data_ptr())
    return q[:, :cols], scale


def matmul_blocks(a, a_scale, b, b_scale, bias=None, out_dtype=torch.float32):
    """``y = dequantized(a) @ dequantized(b).T + bias`` of operands held by ``quantize_blocks``: a (m, k)
    with a_scale (m, ceil(k / 128)); b (n, k) with b_scale (n, ceil(k / 128)) or, per tile,
    (ceil(n / 128), ceil(k / 128)); bias (n,) float32.  Sums are float32, rounded once to
    ``out_dtype``.  Operands may start at any byte, but products of long rows are two to seven times as fast
    where both operands' rows start at multiples of 16 bytes, as ``quantize_blocks`` lays them out
    (``.contiguous()`` on its result undoes that)."""
    lda, ldb = _matrix("a", a), _matrix("b", b, a.device)
    if a.dtype != _FP8 or b.dtype != _FP8:
        raise ValueError("a and b must be float8_e4m3fn, got %s and %s" % (a.dtype, b.dtype))
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k or k < 1:
        raise ValueError("a is %s and b is %s: their rows must have the same, positive length"
                         % (tuple(a.shape), tuple(b.shape)))
    kb = (k + BLOCK - 1) // BLOCK
    _dense("a_scale", a_scale, (m, kb), torch.float32, a.device)
    tile = not (torch.is_tensor(b_scale) and tuple(b_scale.shape) == (n, kb))
    _dense("b_scale", b_scale, ((n + BLOCK - 1) // BLOCK if tile else n, kb), torch.float32, a.device)
    if bias is not None:
        _dense("bias", bias, (n,), torch.float32, a.device)
    code = _dtype_code("out_dtype", out_dtype)
    y = torch.empty(m, n, dtype=out_dtype, device=a.device)
    if m and n:
        _call(N.lib().ncf_matmul_blocks, a.device, a.data_ptr(), lda, a_scale.data_ptr(), b.data_ptr(), ldb,
              b_scale.data_ptr(), 1 if tile else 0, N.ptr(bias), m, n, k, code, y.data_ptr(), n)
    return y


def _number(name, value, whole=False):
    if type(value) is not int and (whole or type(value) is not float):
        if not isinstance(value, numbers.Integral if whole else numbers.Real):
            raise ValueError("%s must be %s, got %r" % (name, "an integer" if whole else "a number", value))
    return value


def _setting(name, value, rows, dtype, device, low, high):
    """One number for all rows, or a tensor with one per row: (number, address or None)."""
    if torch.is_tensor(value):
        return 0, _dense(name, value, (rows,), dtype, device).data_ptr()
    if not low <= _number(name, value, dtype is torch.int32) <= high:   # (a NaN fails too)
        raise ValueError("%s must be in [%g, %g], got %r" % (name, low, high, value))
    return value, None


def check_draw(rows, n, device, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """Checks the settings and the mask of a draw from (rows, n) logits on ``device``; returns
    :func:`sample_items`' argument struct with them filled in."""
    d = N.NcfDraw()
    d.temperature, d.temperature_rows = _setting("temperature", temperature, rows, torch.float32, device, 0, math.inf)
    d.top_k, d.top_k_rows = _setting("top_k", top_k, rows, torch.int32, device, 0, 2 ** 62)
    d.top_p, d.top_p_rows = _setting("top_p", top_p, rows, torch.float32, device, 0, 1)
    d.min_p, d.min_p_rows = _setting("min_p", min_p, rows, torch.float32, device, 0, 1)
    if mask is not None:
        if not torch.is_tensor(mask) or mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError("mask must be a bool or uint8 tensor")
        if tuple(mask.shape) == (n,):
            mask = mask.expand(rows, n)
        if tuple(mask.shape) != (rows, n):
            raise ValueError("mask must have shape (%d, %d) or (%d,), got %s" % (rows, n, n, tuple(mask.shape)))
        d.mask_ld = _matrix("mask", mask, device)
        d.mask = mask.data_ptr()
    return d


def sample_items(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """Draws items from ``logits`` (rows, n; float32, bfloat16 or float16) by the given uniform numbers
    ``u`` (rows,) or (rows, draws), float32 or float64 in [0, 1): ``(items, probs)`` of u's shape, int32
    and float32.  A row keeps its ``top_k`` best items (0: all), of them the shortest leading list with
    at least ``top_p`` of the weight exp(logit / temperature), of it the items with at least ``min_p``
    of the best one's weight; equals rank by the lower id.  A draw takes the first kept item, in the
    order of the ids, at which the running sum of the weights passes u times their total; its
    probability is its share.  Draws of a row are independent (with replacement).  temperature 0 is
    the best item alone.

    ``mask`` (rows, n) or (n,) for every row, bool or uint8: False/0 items are never drawn, whatever
    their logits; neither are NaN and -inf.  A row with nothing to draw gives item -1, probability 0.
    Each setting is a number or a tensor with one per row (float32; top_k int32), where values outside
    the range act as its nearest end."""
    ld = _matrix("logits", logits)
    dev = logits.device
    rows, n = logits.shape
    code = _dtype_code("logits", logits.dtype)
    if n < 1:
        raise ValueError("logits has no columns")
    if not torch.is_tensor(u) or u.dim() not in (1, 2) or u.shape[0] != rows:
        raise ValueError("u must have shape (%d,) or (%d, draws)" % (rows, rows))
    if u.dtype not in (torch.float32, torch.float64):
        raise ValueError("u must be float32 or float64, got %s" % u.dtype)
    _dense("u", u, u.shape, u.dtype, dev)
    d = check_draw(rows, n, dev, temperature, top_k, top_p, min_p, mask)
    d.dtype = code
    items = torch.empty(u.shape, dtype=torch.int32, device=dev)
    probs = torch.empty(u.shape, dtype=torch.float32, device=dev)
    d.draws = 1 if u.dim() == 1 else u.shape[1]
    if rows and d.draws:
        d.logits, d.rows, d.n, d.ld = logits.data_ptr(), rows, n, ld
        d.u, d.u64 = u.data_ptr(), 1 if u.dtype == torch.float64 else 0
        d.items, d.probs = items.data_ptr(), probs.data_ptr()
        ws = _workspace(N.lib().ncf_draw_workspace, d, dev)
        if ws is not None:
            d.ws, d.ws_bytes = ws.data_ptr(), ws.numel()
        _call(N.lib().ncf_draw_items, dev, ctypes.byref(d))
    return items, probs


def _distill(logits, teacher_items, teacher_logits, temperature, teacher_lse):
    """Checks what every distillation call takes; the filled argument struct."""
    d = N.NcfDistill()
    d.ld = _matrix("logits", logits)
    dev = logits.device
    d.dtype = _dtype_code("logits", logits.dtype)
    d.rows, d.v = logits.shape
    if d.v < 1:
        raise ValueError("logits has no columns")
    d.items_ld = _matrix("teacher_items", teacher_items, dev)
    if teacher_items.dtype not in (torch.int32, torch.int64):
        raise ValueError("teacher_items must be int32 or int64, got %s" % teacher_items.dtype)
    d.k = teacher_items.shape[1]
    if teacher_items.shape[0] != d.rows or not 1 <= d.k <= N.NCF_DISTILL_MAX_K:
        raise ValueError("teacher_items must have shape (%d, 1..%d), got %s"
                         % (d.rows, N.NCF_DISTILL_MAX_K, tuple(teacher_items.shape)))
    d.teacher_ld = _matrix("teacher_logits", teacher_logits, dev)
    if teacher_logits.shape != teacher_items.shape or teacher_logits.dtype != torch.float32:
        raise ValueError("teacher_logits must be float32 of shape %s, got %s of %s"
                         % (tuple(teacher_items.shape), teacher_logits.dtype, tuple(teacher_logits.shape)))
    if teacher_lse is not None:
        d.teacher_lse = _dense("teacher_lse", teacher_lse, (d.rows,), torch.float32, dev).data_ptr()
    if not 2.0 ** -100 <= _number("temperature", temperature) <= 2.0 ** 100:
        raise ValueError("temperature must be in [2^-100, 2^100], got %r" % (temperature,))
    d.temperature = temperature
    d.logits, d.teacher_items, d.teacher_logits = logits.data_ptr(), teacher_items.data_ptr(), teacher_logits.data_ptr()
    d.items64 = 1 if teacher_items.dtype == torch.int64 else 0
    return d


def _distill_outputs(d, logits, grad_loss):
    if torch.is_tensor(grad_loss):
        d.grad_loss = _dense("grad_loss", grad_loss, (d.rows,), torch.float32, logits.device).data_ptr()
    else:
        d.grad_loss_value = _number("grad_loss", grad_loss)
    grad = torch.empty(d.rows, d.v, dtype=logits.dtype, device=logits.device)
    d.grad, d.grad_ld = grad.data_ptr(), d.v
    return grad


def distill_loss(logits, teacher_items, teacher_logits, temperature=1.0, teacher_lse=None):
    """Per row, the divergence of a student's softmax over the catalogue from a teacher's list of its
    best items: ``(loss, state)``, loss float32 (rows,), state for :func:`distill_grad`.

    ``logits`` (rows, v; float32, bfloat16 or float16) are the student's; ``teacher_items`` (rows, k;
    int32 or int64, k <= 1024) and ``teacher_logits`` (rows, k; float32) the teacher's list, as
    ``NCFEngine.score_topk`` gives items (ids outside [0, v), such as -1, are padding).  With
    p = softmax(logits / temperature) and q = softmax(teacher_logits / temperature) over the list,
    loss = sum q (log q - log p[items]).  ``teacher_lse`` (rows,) float32, the teacher's
    logsumexp(logits / temperature) over its whole catalogue, makes q the teacher's probabilities
    and adds the mass outside the list as one more class.  A row without an entry, or whose logits
    are all -inf, has loss 0.  ``temperature`` is in [2^-100, 2^100].  (Gradients by soft targets usually carry a factor temperature ** 2:
    pass it in ``grad_loss``.)"""
    d = _distill(logits, teacher_items, teacher_logits, temperature, teacher_lse)
    dev = logits.device
    loss = torch.empty(d.rows, dtype=torch.float32, device=dev)
    state = torch.empty(d.rows, N.NCF_DISTILL_STATE, dtype=torch.float64, device=dev)
    ws = _workspace(N.lib().ncf_distill_workspace, d, dev)
    d.loss, d.state = loss.data_ptr(), state.data_ptr()
    if d.rows:
        _call(N.lib().ncf_distill_loss, dev, ctypes.byref(d), N.ptr(ws), ws.numel() if ws is not None else 0)
    return loss, state


def distill_grad(logits, teacher_items, teacher_logits, state, grad_loss=1.0, temperature=1.0, teacher_lse=None):
    """d sum(grad_loss * loss) / d logits, of logits' type and shape, from the ``state`` that
    :func:`distill_loss` gave for the same inputs.  ``grad_loss``: a number or float32 (rows,)."""
    d = _distill(logits, teacher_items, teacher_logits, temperature, teacher_lse)
    dev = logits.device
    _dense("state", state, (d.rows, N.NCF_DISTILL_STATE), torch.float64, dev)
    grad = _distill_outputs(d, logits, grad_loss)
    d.state = state.data_ptr()
    if d.rows:
        _call(N.lib().ncf_distill_grad, dev, ctypes.byref(d))
    return grad


def distill_loss_grad(logits, teacher_items, teacher_logits, grad_loss=1.0, temperature=1.0, teacher_lse=None):
    """:func:`distill_loss` and :func:`distill_grad` in one call: ``(loss, grad)``."""
    d = _distill(logits, teacher_items, teacher_logits, temperature, teacher_lse)
    dev = logits.device
    loss = torch.empty(d.rows, dtype=torch.float32, device=dev)
    grad = _distill_outputs(d, logits, grad_loss)
    ws = _workspace(N.lib().ncf_distill_workspace, d, dev)
    d.loss = loss.data_ptr()
    if d.rows:
        _call(N.lib().ncf_distill_loss_grad, dev, ctypes.byref(d), N.ptr(ws), ws.numel() if ws is not None else 0)
    return loss, grad
