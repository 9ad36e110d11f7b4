"""Distillation where the listed items and the rest lie far apart.

The listed items lead the others (or trail them) by more than a float32 weight relative to the row's best logit can
hold.  Tolerances: those of test_catalogue_distill_gpu.py, whose |z| (at most 42 with weight that counts) is within
each of the two classes: a class's weights and sum are relative to its own best logit, and the way between the two
is 64 bits."""

import pytest

from conftest import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from test_catalogue_distill_gpu import both

SIZES = [(500, 5), (9000, 65), (20000, 5), (20000, 65), (40000, 5), (40000, 65), (60000, 5)]


def problem(rows, v, k, lead, t, dtype, seed, mass=0.5):
    """Teacher's list of k items that lead the student's other logits by lead * t; the teacher gives it `mass`."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g)
    items = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(rows)])
    x.scatter_add_(1, items, torch.full((rows, k), lead * t))
    y = torch.randn(rows, k, generator=g)
    lse = torch.logsumexp(y.double() / t, 1) - torch.log(torch.tensor(mass, dtype=torch.float64))
    return x.to(getattr(torch, dtype)), items, y, lse.float()


@pytest.mark.parametrize("lead", [-300, -110, -95, -80, 80, 95, 110, 300])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_list_and_rest_far_apart(size, lead):
    for t, dtype in ((0.5, "float32"), (1.0, "bfloat16")):
        x, items, y, lse = problem(3, *size, lead, t, dtype, seed=size[0] + lead)
        both(x, items, y, t, lse)
        both(x, items, y, t, lse, torch.full((3,), 4096.0))
