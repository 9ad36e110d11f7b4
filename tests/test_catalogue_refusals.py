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
