"""How far a draw may be from real arithmetic, derived for the row's length.

A weight w in (0, 1] is held as round(w 2^S), S = min(51, 62 - ceil(log2 n)): off by at most 2^-(S + 1); w itself is a
64-bit exponential, relative 2^-50 with all its roundings.  A running sum of up to n weights, and the total (at least
1: the best item's weight), are each off by at most n 2^-(S + 1) + 2^-50 of the total, so their quotient by twice that;
the reference's own running sums of n float64 add n 2^-53.  (2^-22 at 1,000,003 items, where S = 42.)"""

import math

import pytest

from conftest import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    import test_catalogue_sample_gpu as S


@pytest.mark.parametrize("n", [1000, 70001, 300000, 1000003])
def test_draws_within_the_derived_distance_of_a_border(n, monkeypatch):
    s = min(51, 62 - math.ceil(math.log2(n)))
    monkeypatch.setattr(S, "NEAR", 2 * (n * 2.0 ** -(s + 1) + 2.0 ** -50) + n * 2.0 ** -53)
    x = S.logits(2, n, "float32", n)
    x[1] = 4 * x[1]                                   # many items of less than half a unit
    u = torch.rand(2, 64, generator=S.gen(n + 1), dtype=torch.float64)
    for kw in (dict(), dict(t=3.0), dict(p=0.9), dict(k=n // 2, t=0.7)):
        S.check(x, u, *S.call(x, u, **kw), **kw)
