"""Distillation from a teacher's list against the formula in 64 bits, and its gradient against differences.

Tolerances.  A weight exp2((x - m) c) in float32: the difference is off by half a step, the product by
another and c by a third, so the exponent by |z| 1.5 * 2^-23 (z = (x - m) / t, at most Z = max |z| with
weight that counts; weights below 2^-60 do not) and the exp2 itself by one step: relative
e = 2^-23 (1.5 Z / ln 2 + 1).  Sums are 64 bits, so log p is off by at most e in absolute terms, the loss
by sum(q) e, plus its own rounding; with ``teacher_lse`` q0 e more for log p0 and (sum q + q0)
2^-23 for the float32 logarithm that lse is (an input, equal in both).  The gradient is
(p c - q) g / t: p relative 2 e, q and the factors one step each, then the output type's half step."""

import numpy as np
import pytest

from conftest import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec import catalogue as C


def reference(x, items, y, t, lse, gl):
    """Loss and gradient in float64, row by row: (loss, grad, p c, q, sum q + q0, p q0 in / out)."""
    x, y = x.double().numpy(), y.double().numpy()
    items = items.numpy()
    rows, v = x.shape
    loss, grad = np.zeros(rows), np.zeros((rows, v))
    pc, qv, mass, part = np.zeros((rows, v)), np.zeros((rows, v)), np.zeros(rows), np.zeros((rows, v))
    with np.errstate(all="ignore"):
        for r in range(rows):
            m = x[r].max()
            if m == -np.inf:
                continue
            z = (x[r] - m) / t
            w = np.exp(z)
            s = w.sum()
            ok = (items[r] >= 0) & (items[r] < v)
            it, yy = items[r][ok], y[r][ok] / t
            listed = np.zeros(v, bool)
            listed[it] = True
            if lse is not None:
                ref = float(lse[r])
            elif yy.size and yy.max() > -np.inf:
                ref = yy.max() + np.log(np.exp(yy - yy.max()).sum())
            else:
                ref = np.inf
            lq = yy - ref
            q = np.exp(lq)
            on = q > 0
            loss[r] = (q[on] * (lq[on] - (z[it][on] - np.log(s)))).sum()
            cin = cout = q.sum()
            if lse is not None:
                q0, out = 1 - q.sum(), w[~listed].sum()
                if q0 > 0 and out > 0:
                    loss[r] += q0 * (np.log(q0) + np.log1p(w[listed].sum() / out))
                    cin = q.sum() + q0
                    cout = cin - q0 * s / out
                    part[r] = np.where(listed, 0, w / s * q0 * w[listed].sum() / out)
            np.add.at(qv[r], it, q)
            pc[r] = w / s * np.where(listed, cin, cout)
            mass[r] = abs(cin) + q.sum()
            grad[r] = (pc[r] - qv[r]) * gl[r] / t
    return loss, grad, pc, qv, mass, part


def check(x, items, y, t=1.0, lse=None, gl=None, got=None):
    rows = x.shape[0]
    g = np.ones(rows) if gl is None else gl.double().numpy()
    loss, grad, pc, qv, mass, part = reference(x, items, y, t, None if lse is None else lse.double().numpy(), g)
    xd = x.double().numpy()
    with np.errstate(all="ignore"):
        z = np.abs(np.where(np.isfinite(xd), xd - xd.max(1, keepdims=True), 0) / t)
    zmax = np.minimum(z, 42.0).max(1)
    e = 2.0 ** -23 * (1.5 * zmax / np.log(2) + 1)
    assert np.all(np.abs(got[0].double().cpu().numpy() - loss) <= 2 * mass * e + np.abs(loss) * 2.0 ** -23 + 1e-30)
    if len(got) > 1:
        fi = torch.finfo(x.dtype)
        # c outside = sum q - q0 in / out is a difference of the two: in and out are each off by e, so the second
        # term by 2 e of itself, which is more than 2 e of a c that cancels (k = 1, q = 0.0208, q0 in / out = 0.0210)
        tol = (np.abs(pc) * (2 * e[:, None] + 2.0 ** -21) + qv * 2.0 ** -22 + part * 2 * e[:, None]) * np.abs(g)[:, None] / t
        tol = tol + np.maximum((np.abs(grad) + tol) * fi.eps / 2, fi.smallest_normal * fi.eps)
        assert got[1].dtype == x.dtype
        err = np.abs(got[1].double().cpu().numpy() - grad)
        assert np.all(err <= tol), (err - tol).max()


def problem(rows, v, k, dtype="float32", seed=0, lse_t=None, index="int64"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g) * 2
    z = x + torch.randn(rows, v, generator=g)
    y, items = torch.topk(z, k, 1)
    lse = torch.logsumexp(z / lse_t, 1) if lse_t else None
    return x.to(getattr(torch, dtype)), items.to(getattr(torch, index)), y.contiguous(), lse


def both(x, items, y, t=1.0, lse=None, gl=None):
    """The three calls, each against the reference; the one-call form's outputs."""
    dev = lambda a: None if a is None else a.cuda()   # noqa: E731
    g = 1.0 if gl is None else gl.cuda()
    loss, state = C.distill_loss(dev(x), dev(items), dev(y), temperature=t, teacher_lse=dev(lse))
    grad = C.distill_grad(dev(x), dev(items), dev(y), state, g, temperature=t, teacher_lse=dev(lse))
    check(x, items, y, t, lse, gl, (loss, grad))
    one = C.distill_loss_grad(dev(x), dev(items), dev(y), g, temperature=t, teacher_lse=dev(lse))
    check(x, items, y, t, lse, gl, one)
    return one


SIZES = [(1, 1, 1), (3, 2, 2), (5, 10, 3), (7, 100, 10), (2, 257, 257), (4, 2047, 32), (3, 4100, 1), (2, 8192, 100),
         (3, 8193, 32), (2, 27278, 32), (2, 32769, 300), (1, 100003, 1024)]


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_fp32(size, lse):
    t = 1.7
    x, items, y, ls = problem(*size, seed=sum(size), lse_t=t if lse else None)
    gl = torch.rand(size[0], generator=torch.Generator().manual_seed(1)) + 0.1
    both(x, items, y, t, ls, gl)


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("size", [(300, 20000, 32, "float32"), (130, 28672, 9, "bfloat16"), (200, 8193, 700, "float16")],
                         ids=str)
def test_many_rows(size, lse):
    x, items, y, ls = problem(*size, seed=2, lse_t=1.0 if lse else None)
    both(x, items, y, 1.0, ls, torch.rand(size[0], generator=torch.Generator().manual_seed(1)))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("size", [(3, 100, 10), (2, 2048, 32), (2, 8200, 5), (2, 27278, 32), (1, 70001, 64)], ids=str)
def test_half(size, dtype):
    x, items, y, ls = problem(*size, dtype=dtype, seed=3, lse_t=0.8, index="int32")
    both(x, items, y, 0.8, None)
    both(x, items, y, 0.8, ls)


@pytest.mark.parametrize("v", [40, 9000, 40000])
def test_padding_duplicates_and_empty_lists(v):
    x, items, y, lse = problem(7, v, 12, seed=4, lse_t=1.0)
    items[0, 5:] = -1                       # a shorter list
    items[1] = -1                           # none
    items[2, 3] = v                         # just past the end
    items[2, 4] = 2 ** 40                   # beyond 32 bits
    items[3, 1] = items[3, 0]               # one item twice
    items[3, 7] = items[3, 0]
    items[4] = items[4, 0]                  # twelve times
    y[5, 2:] = -float("inf")                # entries of no mass
    y[6] = -float("inf")
    both(x, items, y)
    both(x, items, y, 1.0, lse + 0.3)
    loss, grad = C.distill_loss_grad(x.cuda(), items.cuda(), y.cuda())
    assert loss[1] == 0 and loss[6] == 0 and not grad[1].any() and not grad[6].any()


@pytest.mark.parametrize("v", [30, 5000, 20000])
def test_masked_logits(v):
    x, items, y, lse = problem(5, v, 4, seed=5, lse_t=1.0)
    hide = torch.ones(v, dtype=torch.bool)
    hide[items[0]] = False
    x[0, hide] = -float("inf")              # nothing outside the list: no last class
    x[1] = -float("inf")                    # nothing at all
    x[2, v // 2:] = torch.finfo(torch.float32).min
    x[2, items[2]] = 1.0
    x[3, :] = -float("inf")
    x[3, items[3, 0]] = 0.0                 # the other entries have no probability: an infinite loss
    for ls in (None, lse):
        loss, grad = C.distill_loss_grad(x.cuda(), items.cuda(), y.cuda(), temperature=1.0,
                                         teacher_lse=None if ls is None else ls.cuda())
        assert loss[1] == 0 and not grad[1].any()
        assert loss[3] == float("inf") and torch.isfinite(grad[3]).all()
        keep = [0, 2, 4]
        check(x[keep], items[keep], y[keep], 1.0, None if ls is None else ls[keep], None, (loss[keep], grad[keep]))
        assert not grad[0].cpu()[hide].any()


def test_nan_stays_in_its_row():
    x, items, y, lse = problem(6, 3000, 8, seed=6, lse_t=1.0)
    x[1, 77] = float("nan")
    y[3, 2] = float("nan")
    x[4, 5] = float("inf")
    loss, grad = C.distill_loss_grad(x.cuda(), items.cuda(), y.cuda())
    assert torch.isnan(loss).cpu().tolist() == [False, True, False, True, True, False]
    assert torch.isnan(grad).any(1).cpu().tolist() == [False, True, False, True, True, False]
    keep = [0, 2, 5]
    check(x[keep], items[keep], y[keep], got=(loss[keep], grad[keep]))


def test_gradient_against_differences():
    """Central differences of the library's own loss, summed in float64 over the rows.  The loss is
    off by E = 2 * 2 * 2^-23 (1.5 * 12 / ln 2 + 1) <= 1.3e-5 (|z| < 12 here) a row, so a difference over
    2 h = 0.5 by 2 E / 0.5; the third derivative of the loss is at most 1 / t^3, its term h^2 / 6."""
    t, h = 1.0, 0.25
    x, items, y, lse = problem(2, 60, 6, seed=7, lse_t=t)
    x = x.clamp(-5, 5)
    for ls in (None, lse.cuda()):
        _, grad = C.distill_loss_grad(x.cuda(), items.cuda(), y.cuda(), temperature=t, teacher_lse=ls)
        pick = list(range(0, 60, 7)) + items[0, :3].tolist()
        for j in pick:
            up, dn = x.clone(), x.clone()
            up[:, j] += h
            dn[:, j] -= h
            a, _ = C.distill_loss(up.cuda(), items.cuda(), y.cuda(), temperature=t, teacher_lse=ls)
            b, _ = C.distill_loss(dn.cuda(), items.cuda(), y.cuda(), temperature=t, teacher_lse=ls)
            step = (up[:, j] - dn[:, j]).double()
            diff = (a.double().cpu() - b.double().cpu()) / step
            assert torch.all((diff - grad[:, j].double().cpu()).abs() <= 2 * 1.3e-5 / 0.5 + h * h / 6)


def test_strides_and_alignment():
    base, items, y, lse = problem(4, 9000, 20, seed=8, lse_t=1.0)
    for at, v in ((0, 4097), (1, 4096), (3, 8191)):
        x = base[:, at:at + v]
        it = (items - at).clamp_min(-1)
        got = C.distill_loss_grad(base.cuda()[:, at:at + v], it.cuda(), y.cuda())
        check(x, it, y, got=got)
    # a list that is part of a wider one, one shared by all rows, one user's logits for all lists
    got = C.distill_loss_grad(base.cuda(), items.cuda()[:, :7], y.cuda()[:, :7])
    check(base, items[:, :7], y[:, :7], got=got)
    got = C.distill_loss_grad(base.cuda(), items.cuda()[:1].expand(4, 20), y.cuda()[:1].expand(4, 20))
    check(base, items[:1].expand(4, 20), y[:1].expand(4, 20), got=got)
    got = C.distill_loss_grad(base.cuda()[:1].expand(4, 9000), items.cuda(), y.cuda())
    check(base[:1].expand(4, 9000), items, y, got=got)


def test_repeatable_on_streams_and_in_graphs():
    x, items, y, lse = (a.cuda() for a in problem(3, 20000, 32, dtype="bfloat16", seed=9, lse_t=1.0))
    items[:, 5] = items[:, 4]
    want = C.distill_loss_grad(x, items, y, 0.5, teacher_lse=lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = C.distill_loss_grad(x, items, y, 0.5, teacher_lse=lse)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, state = C.distill_loss(x, items, y, teacher_lse=lse)
            out = loss, C.distill_grad(x, items, y, state, 0.5, teacher_lse=lse)
        graphs.append((g, out))
    for seed in range(3):
        x.copy_(torch.randn(3, 20000, generator=torch.Generator().manual_seed(seed)))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        loss, state = C.distill_loss(x, items, y, teacher_lse=lse)
        grad = C.distill_grad(x, items, y, state, 0.5, teacher_lse=lse)
        for _, out in graphs:
            assert torch.equal(out[0], loss) and torch.equal(out[1], grad)


def test_empty_and_refusals():
    x, items, y, lse = (a.cuda() for a in problem(3, 50, 4, lse_t=1.0))
    loss, state = C.distill_loss(x[:0], items[:0], y[:0])
    assert loss.shape == (0,) and C.distill_grad(x[:0], items[:0], y[:0], state).shape == (0, 50)
    loss, state = C.distill_loss(x, items, y)
    bad = [lambda: C.distill_loss(x.double(), items, y), lambda: C.distill_loss(x[0], items, y),
           lambda: C.distill_loss(x, items.short(), y), lambda: C.distill_loss(x, items[:2], y[:2]),
           lambda: C.distill_loss(x, items, y[:, :3]), lambda: C.distill_loss(x, items, y.half()),
           lambda: C.distill_loss(x, items[:, :0], y[:, :0]), lambda: C.distill_loss(x, items.cpu(), y),
           lambda: C.distill_loss(x, items, y, temperature=0), lambda: C.distill_loss(x, items, y, teacher_lse=lse[:2]),
           lambda: C.distill_loss(x, items, y, temperature=float("inf")),
           lambda: C.distill_loss(x, items.t().contiguous().t(), y),
           lambda: C.distill_loss(x, items.repeat(1, 300), y.repeat(1, 300)),
           lambda: C.distill_grad(x, items, y, state[:2]), lambda: C.distill_grad(x, items, y, state.float()),
           lambda: C.distill_loss_grad(x, items, y, torch.ones(2, device="cuda")),
           lambda: C.distill_loss_grad(x, items, y, torch.ones(3, device="cuda", dtype=torch.float64))]
    for f in bad:
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("k", [1, 63, 64, 65])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_long_rows_with_padding_and_duplicates(dtype, k):
    """Rows that a workgroup of several waves holds, lists on both sides of a wave's 64 entries."""
    x, items, y, lse = problem(130, 9001, k, dtype=dtype, seed=k, lse_t=1.0)
    items[0] = -1
    items[1] = items[1, 0]
    items[2, k // 2:] = 9001 + 2 ** 33
    items[3] = 9000                          # the last item, in the row's last, partial vector
    y[4] = -float("inf")
    x[5] = -float("inf")
    x[6, items[6, 0]] = -float("inf")        # a listed item whose logit is masked: the loss is infinite
    y[6, 0] = -float("inf")                  # (but not when it has no mass)
    both(x, items, y)
    both(x, items, y, 1.0, lse + 0.2, torch.rand(130, generator=torch.Generator().manual_seed(2)))


@pytest.mark.parametrize("k", [5, 64, 65])
@pytest.mark.parametrize("v", [28673, 40001, 57344, 57345])
def test_rows_around_the_longest_that_a_workgroup_holds(v, k):
    x, items, y, lse = problem(3, v, k, dtype="bfloat16" if v % 2 else "float32", seed=v + k, lse_t=1.2)
    items[1, 1] = items[1, 0]
    both(x, items, y, 1.2)
    both(x, items, y, 1.2, lse, torch.rand(3, generator=torch.Generator().manual_seed(2)))
