"""Limits of the catalogue operators that need no device: the C ABI checks its arguments before it launches anything."""

import ctypes

import pytest

from movierec import _native as N
from test_catalogue_refusals import P, distill, refused


@pytest.mark.parametrize("call", ["loss", "grad", "both"])
def test_temperatures_without_a_float32_factor(call):
    """log2(e) / t scales float32 differences: outside [2^-100, 2^100] it would overflow, or vanish under a -inf."""
    for t in (1e-39, 5e-324, 2.0 ** -101, 2.0 ** 101, 1e39, 1e300, -1.0):
        refused(distill(call, temperature=t))


def test_more_tiles_than_a_launch_takes():
    """2^24 workgroups of 256 threads are 2^32 threads, which a launch does not count: refused before it."""
    refused(N.lib().ncf_quantize_blocks(P, 0, 1 << 31, 128, 128, 1, P, 128, P, None))


def workspace(fn, struct, **fields):
    for name, value in fields.items():
        setattr(struct, name, value)
    size = ctypes.c_size_t(77)
    N.check(fn(ctypes.byref(struct), ctypes.byref(size)))
    return size.value


def test_no_workspace_for_rows_that_a_workgroup_holds():
    L = N.lib()

    def draw(n, dtype):
        return workspace(L.ncf_draw_workspace, N.NcfDraw(), rows=8192, n=n, dtype=dtype)

    def any_type(n):
        size = ctypes.c_size_t(77)
        N.check(L.ncf_draw_workspace_size(8192, n, ctypes.byref(size)))
        return size.value

    assert draw(40960, N.NCF_F32) == 0 < draw(40961, N.NCF_F32) == any_type(40961)
    for half in (N.NCF_BF16, N.NCF_F16):
        assert draw(32768, half) == 0 < draw(32769, half) == any_type(32769)
    assert any_type(32768) == 0 and draw(32769, N.NCF_F32) == 0

    def distill(v, k):
        return workspace(L.ncf_distill_workspace, N.NcfDistill(), rows=8192, v=v, k=k)

    def any_list(v):
        size = ctypes.c_size_t(77)
        N.check(L.ncf_distill_workspace_size(8192, v, ctypes.byref(size)))
        return size.value

    assert distill(57344, 64) == 0 < distill(57344, 65) == any_list(57344)
    assert distill(28672, 65) == 0 == any_list(28672)
    assert 0 < distill(57345, 1) == any_list(57345)
    refused(L.ncf_draw_workspace(None, ctypes.byref(ctypes.c_size_t())))
    refused(L.ncf_distill_workspace(None, ctypes.byref(ctypes.c_size_t())))
    refused(L.ncf_draw_workspace(ctypes.byref(N.NcfDraw(rows=1, n=8)), None))
    refused(L.ncf_distill_workspace(ctypes.byref(N.NcfDistill(rows=1, v=8)), None))
