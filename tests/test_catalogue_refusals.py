"""Refusals of the catalogue operators that need no device: the C ABI checks its arguments before it
launches anything, and the Python layer refuses host tensors."""

import ctypes

import pytest
import torch

from movierec import _native as N
from movierec import catalogue as C

P = ctypes.c_void_p(0x1000)   # never read: every call below is refused or empty


def refused(rc):
    with pytest.raises(ValueError):
        N.check(rc)


def test_quantize_arguments():
    L = N.lib()
    refused(L.ncf_quantize_blocks(P, 7, 4, 8, 8, 0, P, 16, P, None))      # element type
    refused(L.ncf_quantize_blocks(None, 0, 4, 8, 8, 0, P, 16, P, None))
    refused(L.ncf_quantize_blocks(P, 0, 4, 8, 8, 0, P, 7, P, None))       # q's rows would overlap
    refused(L.ncf_quantize_blocks(P, 0, 4, 0, 8, 0, P, 16, P, None))
    refused(L.ncf_quantize_blocks(P, 0, -1, 8, 8, 0, P, 16, P, None))
    refused(L.ncf_quantize_blocks(P, 0, 4, 8, 8, 0, P, 16, None, None))
    refused(L.ncf_quantize_blocks(P, 0, 4, 1 << 31, 8, 0, P, 1 << 31, P, None))
    refused(L.ncf_quantize_blocks(P, 0, 1 << 40, 1 << 30, 1 << 30, 1, P, 1 << 30, P, None))
    assert L.ncf_quantize_blocks(None, 0, 0, 8, 8, 0, None, 8, None, None) == 0   # nothing to do


def test_matmul_arguments():
    L = N.lib()

    def mm(a=P, lda=64, sa=P, b=P, ldb=64, sb=P, m=4, n=8, k=64, dt=0, y=P, ldy=8):
        return L.ncf_matmul_blocks(a, lda, sa, b, ldb, sb, 0, None, m, n, k, dt, y, ldy, None)

    for kw in (dict(a=None), dict(b=None), dict(sa=None), dict(sb=None), dict(y=None), dict(k=0), dict(k=-5),
               dict(m=-1), dict(n=-1), dict(dt=3), dict(ldy=7), dict(lda=-64), dict(ldb=-1), dict(k=1 << 31),
               dict(m=1 << 30, n=1 << 30, ldy=1 << 30)):
        refused(mm(**kw))
    assert mm(m=0, a=None) == 0 and mm(n=0, y=None) == 0


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        C.quantize_blocks(torch.zeros(2, 4))
    q = torch.zeros(2, 16, dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        C.matmul_blocks(q, torch.ones(2, 1), q, torch.ones(2, 1))


def draw(**kw):
    d = N.NcfDraw()
    d.logits = d.u = d.items = d.probs = 0x1000
    d.rows, d.n, d.ld, d.draws, d.temperature, d.top_p = 4, 8, 8, 2, 1.0, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return N.lib().ncf_draw_items(ctypes.byref(d), None)


def test_draw_arguments():
    refused(N.lib().ncf_draw_items(None, None))
    for kw in (dict(dtype=9), dict(logits=None), dict(u=None), dict(items=None), dict(probs=None), dict(n=0),
               dict(n=1 << 31), dict(rows=-1), dict(draws=-1), dict(ld=-8), dict(mask=0x1000, mask_ld=-1),
               dict(rows=1 << 32), dict(draws=1 << 30)):
        refused(draw(**kw))
    assert draw(rows=0, logits=None) == 0 and draw(draws=0, u=None) == 0


def distill(call, ws=0x1000, ws_bytes=1 << 20, **kw):
    d = N.NcfDistill()
    d.logits = d.teacher_items = d.teacher_logits = d.loss = d.state = d.grad = 0x1000
    d.rows, d.v, d.ld, d.k, d.items_ld, d.teacher_ld, d.grad_ld, d.temperature = 4, 100, 100, 8, 8, 8, 100, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    L = N.lib()
    if call == "grad":
        return L.ncf_distill_grad(ctypes.byref(d), None)
    fn = L.ncf_distill_loss if call == "loss" else L.ncf_distill_loss_grad
    return fn(ctypes.byref(d), ws, ws_bytes, None)


@pytest.mark.parametrize("call", ["loss", "grad", "both"])
def test_distill_arguments(call):
    for kw in (dict(dtype=9), dict(logits=None), dict(teacher_items=None), dict(teacher_logits=None),
               dict(v=0), dict(v=1 << 31), dict(k=0), dict(k=1025), dict(rows=-1),
               dict(rows=1 << 31), dict(temperature=0.0), dict(temperature=float("nan")),
               dict(temperature=float("inf")), dict(ld=-1), dict(items_ld=-1)):
        refused(distill(call, **kw))
    if call != "grad":
        refused(distill(call, loss=None))
        long = dict(v=60000, ld=60000, grad_ld=60000)   # longer than a workgroup holds
        refused(distill(call, ws=None, **long))
        refused(distill(call, ws_bytes=8, **long))
    if call != "both":
        refused(distill(call, state=None))
    if call != "loss":
        refused(distill(call, grad=None))
        refused(distill(call, grad_ld=99))
    assert distill(call, rows=0, logits=None) == 0


def test_distill_workspace_size():
    L = N.lib()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    N.check(L.ncf_distill_workspace_size(4, 100, ctypes.byref(a)))
    N.check(L.ncf_distill_workspace_size(64, 1000000, ctypes.byref(b)))
    assert b.value > 0 and a.value == 0   # short rows need none
    refused(L.ncf_distill_workspace_size(4, 0, ctypes.byref(a)))
    refused(L.ncf_distill_workspace_size(1 << 40, 1000000, ctypes.byref(a)))
    refused(L.ncf_distill_workspace_size(4, 100, None))


def test_host_tensors_are_refused_by_draw_and_distill():
    x = torch.zeros(2, 4)
    with pytest.raises(ValueError):
        C.sample_items(x, torch.zeros(2))
    with pytest.raises(ValueError):
        C.distill_loss(x, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1))
