"""Distillation where the listed items and the rest lie far apart, and where a list's probabilities are no fractions of one.

The listed items lead the others (or trail them) by more than a float32 weight relative to the row's best logit can
hold.  Tolerances: those of test_catalogue_distill_gpu.py, whose |z| (at most 42 with weight that counts) is within
each of the two classes: a class's weights and sum are relative to its own best logit, and the way between the two
is 64 bits."""

import pytest

from conftest import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec import catalogue as C
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


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_more_than_one_mass_in_the_list(size):
    """A teacher_lse below the list's own log-sum-exp: single q above 2, the same formula in every kernel."""
    x, items, y, lse = problem(3, *size, 0.0, 1.0, "float32", seed=size[0], mass=6.0 * size[1])
    items[1, 1] = items[1, 0]
    loss, grad = both(x, items, y, 1.0, lse)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all()


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_little_mass_in_the_list(size):
    """q far below 2^-51 of one, of items the student gives nothing: the gradient there is -q.  The other tests'
    reference forms c outside as a difference of numbers near one, 2^-53 of rounding where c is 2^-60 here; below it
    is sum q - q0 r, the same by algebra.  Their tolerance, for each item: 2 e + 2^-21 of p c, and 2^-22 of q."""
    x, items, y, lse = problem(3, *size, -110.0, 1.0, "float32", seed=size[0], mass=2.0 ** -60)
    items[2, 1] = items[2, 0]
    q = torch.zeros(x.shape, dtype=torch.float64).scatter_add_(1, items, torch.exp(y.double() - lse.double()[:, None]))
    listed = torch.zeros(x.shape, dtype=torch.bool).scatter_(1, items, True)
    z = x.double()
    out, inside = (torch.logsumexp(z.masked_fill(m, -float("inf")), 1, keepdim=True) for m in (listed, ~listed))
    r, mass = torch.exp(inside - out), q.sum(1, keepdim=True)
    c = torch.where(listed, torch.exp(z - inside) * r, torch.exp(z - out) * (mass - (1 - mass) * r)) / (1 + r)
    tol = c.abs() * (2 * 2.0 ** -23 * (1.5 * 42 / 0.6931 + 1) + 2.0 ** -21) + q * 2.0 ** -22 + 1.5e-45
    a = [t.cuda() for t in (x, items, y)]
    loss, state = C.distill_loss(*a, teacher_lse=lse.cuda())
    for grad in (C.distill_grad(*a, state, teacher_lse=lse.cuda()), C.distill_loss_grad(*a, teacher_lse=lse.cuda())[1]):
        assert torch.all((grad.cpu().double() - (c - q)).abs() <= tol)
        assert (grad.cpu().gather(1, items) < 0).all()
