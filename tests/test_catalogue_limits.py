"""Limits of the catalogue operators that need no device: the C ABI checks its arguments before it launches anything."""

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
