"""Operators over a user's logits for the whole catalogue, on the device.

``quantize_blocks`` / ``matmul_blocks``  logits as a product of 8-bit operands with a scale for each
                                        block of 128 values (GMF models: user factors x item factors)

Every tensor lives on one HIP device and the work is enqueued on that device's current stream; no
call synchronises, and what a call needs beside its outputs it allocates from torch's caching
allocator, so calls on several streams and captured graphs share nothing.  Matrices may be strided
over their rows; their last dimension is dense.  A wrong argument raises ``ValueError``.

The reference scores a list of items for one user and keeps the best (movierec/trt_client.py:43-57).
"""

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
    with torch.cuda.device(x.device):
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
    ``out_dtype``."""
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
    with torch.cuda.device(a.device):
        y = torch.empty(m, n, dtype=out_dtype, device=a.device)
    if m and n:
        _call(N.lib().ncf_matmul_blocks, a.device, a.data_ptr(), lda, a_scale.data_ptr(), b.data_ptr(), ldb,
              b_scale.data_ptr(), 1 if tile else 0, N.ptr(bias), m, n, k, code, y.data_ptr(), n)
    return y
