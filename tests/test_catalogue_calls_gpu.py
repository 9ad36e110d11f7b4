"""Calls of the catalogue operators at the edge of what they take: every one is served or refused by a ValueError."""

import pytest

from conftest import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec import catalogue as C
    from test_catalogue_distill_gpu import both, problem


@pytest.mark.parametrize("v", [60, 9000, 40000])
def test_distillation_at_extreme_temperatures(v):
    """Masked logits and equals of the best stay numbers over the whole range of temperatures; outside it: refused."""
    for t in (2.0 ** -100, 1e-30, 1e-12, 1e30, 2.0 ** 100):
        x, items, y, _ = problem(3, v, 5, seed=v)
        x[0, ::2] = -float("inf")
        x[0, items[0]] = 1.0
        x[1, items[1]] = x[1].max()
        for r in both(x, items, y, t):
            assert torch.isfinite(r).all()
    x, items, y = (a.cuda() for a in problem(3, v, 5, seed=v)[:3])
    for t in (1e-39, 5e-324, 1e39, 1e300):
        with pytest.raises(ValueError):
            C.distill_loss(x, items, y, temperature=t)
