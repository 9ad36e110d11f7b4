"""Drawing items from logits against the definition in 64 bits.

The reference below keeps each row's items by an explicit sort and draws with numpy's cumulative sums
in float64.  A draw may differ from it only where u lies within the weights' resolution of a border:
n items of weight round(w 2^S), S = min(51, 62 - ceil(log2 n)), and a 64-bit exp (2 units in the last
place), so a running sum relative to the total is off by at most n (2^-S + 2^-51) <= 2^-30 for the sizes
here.  ``check`` accepts another item only if u is that close to the border between the two; the
probability is one float32 rounding of a quotient off by as much."""

import numpy as np
import pytest

from conftest import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec import catalogue as C

NEAR = 2.0 ** -30


def kept_weights(x, mask, t, k, p, min_p):
    """Weights (0 for what is not kept) of one row in the order of the ids."""
    x = np.where(mask & ~np.isnan(x) & (x > -np.inf), x, -np.inf)
    order = np.lexsort((np.arange(x.size), -x))
    order = order[x[order] > -np.inf]
    w = np.zeros(x.size)
    if order.size == 0:
        return w
    if not t > 0 or p <= 0:
        k = 1
    if k > 0:
        order = order[:k]
    with np.errstate(all="ignore"):
        v = np.exp((x[order] - x[order[0]]) / (t if t > 0 else 1.0))
    v = np.where(x[order] == x[order[0]], 1.0, np.nan_to_num(v))
    if 0 < p < 1:
        c = np.cumsum(v)
        m = 1 + np.searchsorted(c, p * c[-1], side="left")
        order, v = order[:m], v[:m]
    keep = v >= min(min_p, 1.0)
    w[order[keep]] = v[keep]
    return w


def check(x, u, items, probs, mask=None, t=1.0, k=0, p=1.0, min_p=0.0):
    """x, u: CPU tensors; settings: numbers or per-row arrays."""
    xs, us = x.double().numpy(), u.double().numpy().reshape(x.shape[0], -1)
    it, pr = items.cpu().numpy().reshape(us.shape), probs.cpu().numpy().reshape(us.shape)
    rows = x.shape[0]
    ms = np.ones(xs.shape, bool) if mask is None else np.broadcast_to(mask.numpy().astype(bool), xs.shape)
    t, k, p, min_p = (np.broadcast_to(np.asarray(s, np.float64), (rows,)) for s in (t, k, p, min_p))
    for r in range(rows):
        w = kept_weights(xs[r], ms[r], t[r], int(k[r]), p[r], min_p[r])
        c = np.cumsum(w)
        for d in range(us.shape[1]):
            if c[-1] == 0:
                assert it[r, d] == -1 and pr[r, d] == 0
                continue
            uu = min(max(us[r, d], 0.0), np.nextafter(1.0, 0.0))
            want = int(np.searchsorted(c, uu * c[-1], side="right"))
            got = int(it[r, d])
            assert 0 <= got < xs.shape[1] and w[got] > 0, (r, d, got, want)
            if got != want:
                lo, hi = min(got, want), max(got, want)
                assert abs(c[hi - 1] / c[-1] - uu) <= NEAR and abs(c[lo] / c[-1] - uu) <= NEAR, (r, d, got, want)
            share = w[got] / c[-1]
            assert abs(pr[r, d] - share) <= share * (2.0 ** -24) + NEAR


def gen(seed):
    return torch.Generator().manual_seed(seed)


def logits(rows, n, dtype, seed, scale=2.0):
    return (torch.randn(rows, n, generator=gen(seed)) * scale).to(getattr(torch, dtype))


SETTINGS = [dict(), dict(t=0.5), dict(k=1), dict(k=7), dict(k=50, t=2.0), dict(p=0.3), dict(p=0.9, t=0.7),
            dict(min_p=0.1), dict(k=40, p=0.8, min_p=0.05, t=1.3), dict(t=0.0), dict(p=0.0), dict(min_p=1.0)]


def call(x, u, mask=None, t=1.0, k=0, p=1.0, min_p=0.0):
    return C.sample_items(x.cuda(), u.cuda(), temperature=t, top_k=k, top_p=p, min_p=min_p,
                          mask=None if mask is None else mask.cuda())


@pytest.mark.parametrize("n", [1, 2, 31, 64, 100, 1000, 2049, 4097, 27278, 33000, 70001])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_sizes_and_types(n, dtype):
    rows = 3
    x = logits(rows, n, dtype, n)
    u = torch.rand(rows, 5, generator=gen(n + 1))
    for s in SETTINGS:
        check(x, u, *call(x, u, **s), **s)


def test_large_catalogue():
    x = logits(2, 1000003, "float32", 3)
    u = torch.rand(2, 4, generator=gen(4), dtype=torch.float64)
    for s in (dict(), dict(k=1000, p=0.9), dict(p=0.6), dict(min_p=0.01, k=200000)):
        check(x, u, *call(x, u, **s), **s)


@pytest.mark.parametrize("n", [10, 700, 5000, 40000])
def test_equal_logits_rank_by_the_lower_id(n):
    x = torch.zeros(4, n)
    x[1, ::2] = 1.0
    x[2, : n // 2] = -3.0
    x[3] = torch.tensor([0.0, -0.0]).repeat(n)[:n]      # equal logits of either sign
    u = torch.rand(4, 9, generator=gen(1))
    for s in (dict(), dict(k=3), dict(k=n - 1), dict(p=0.5), dict(p=0.25, k=n // 2), dict(min_p=0.5),
              dict(k=n // 3, p=0.7)):
        check(x, u, *call(x, u, **s), **s)


def test_more_equal_logits_than_a_long_row_lists():
    n = 150001
    x = torch.zeros(3, n)
    x[1, ::3] = 2.0
    x[2] = torch.randint(0, 3, (n,), generator=gen(2)).float()
    u = torch.rand(3, 5, generator=gen(3))
    for s in (dict(), dict(k=70000), dict(k=n - 1), dict(p=0.5), dict(p=0.9, k=120000), dict(p=0.3, min_p=0.5)):
        check(x, u, *call(x, u, **s), **s)


@pytest.mark.parametrize("n", [5, 300, 9000, 50000])
def test_masks_infinities_and_nan(n):
    x = logits(8, n, "float32", 5)
    mask = torch.rand(8, n, generator=gen(6)) < 0.5
    mask[0] = False                        # nothing left
    mask[1] = False
    mask[1, n // 2] = True                 # one item
    x[2, mask[2]] = -float("inf")          # nothing left by the logits
    x[3, ~mask[3]] = float("nan")          # what the mask hides may hold anything
    x[4, ~mask[4]] = float("inf")
    x[5] = torch.finfo(torch.float32).min  # the lowest value is a logit like any other
    x[6, : n // 2] = float("inf")          # infinities share the mass
    x[7, ::3] = float("nan")               # a NaN is never drawn, mask or not
    u = torch.rand(8, 6, generator=gen(7))
    for s in (dict(), dict(k=3), dict(p=0.7), dict(k=2, p=0.9, min_p=0.1), dict(t=0.3)):
        check(x, u, *call(x, u, mask=mask, **s), mask=mask, **s)
    none = torch.full((2, n), -float("inf"))
    items, probs = call(none, torch.rand(2, 3))
    assert (items == -1).all() and (probs == 0).all()


def test_mask_shared_by_all_rows_and_uint8():
    x = logits(5, 777, "bfloat16", 8)
    mask = torch.rand(777, generator=gen(9)) < 0.3
    u = torch.rand(5, generator=gen(10))
    check(x, u, *call(x, u, mask=mask, k=20), mask=mask, k=20)
    m8 = mask.to(torch.uint8) * 4
    check(x, u, *call(x, u, mask=m8.view(1, -1).expand(5, 777), k=20), mask=mask, k=20)


@pytest.mark.parametrize("n", [50, 3000, 35000])
def test_settings_of_their_own_for_every_row(n):
    rows = 9
    x = logits(rows, n, "float32", 11)
    u = torch.rand(rows, 4, generator=gen(12))
    t = torch.tensor([1.0, 0.0, 0.5, 2.0, -1.0, 1.0, float("nan"), float("inf"), 1e-30])
    k = torch.tensor([0, 5, 3, -2, 9, 10 ** 9, 4, 2, 8], dtype=torch.int32)
    p = torch.tensor([0.5, 0.9, 1.0, 0.3, 0.2, 2.0, 0.9, 0.0, 0.6])
    mp = torch.tensor([0.0, 0.1, 0.5, 0.0, 0.0, 0.2, 0.0, 0.0, 7.0])
    items, probs = C.sample_items(x.cuda(), u.cuda(), temperature=t.cuda(), top_k=k.cuda(), top_p=p.cuda(),
                                  min_p=mp.cuda())
    tt = np.nan_to_num(t.double().numpy(), nan=0.0, posinf=np.inf)
    check(x, u, items, probs, t=tt, k=np.maximum(k.numpy(), 0), p=p.double().numpy(), min_p=mp.double().numpy())


def test_u_at_the_ends_and_on_borders():
    x = torch.zeros(1, 8).expand(1, 8)
    u = torch.tensor([[0.0, 0.125, 0.25, 0.875, 0.9999999, 1.0, 3.0, -1.0, float("nan"), float("inf")]])
    items, probs = call(x, u)
    assert items.tolist()[0] == [0, 1, 2, 7, 7, 7, 7, 0, 0, 7]
    assert torch.allclose(probs.cpu(), torch.full((1, 10), 0.125))


def test_strided_rows_alignment_and_order():
    base = logits(6, 2 * 1500 + 9, "float32", 13)
    u = torch.rand(6, 3, generator=gen(14))
    for at in (0, 1, 5):
        x = base[:, at:at + 1500]
        got = C.sample_items(base.cuda()[:, at:at + 1500], u.cuda(), top_k=30, top_p=0.9)
        check(x, u, *got, k=30, p=0.9)
    one = base[:1, :1500]
    got = C.sample_items(one.cuda().expand(6, 1500), u.cuda(), top_p=0.9)
    check(one.expand(6, 1500), u, *got, p=0.9)
    # 16-bit rows that start at odd elements, rows one element longer than a vector
    b16 = logits(5, 20001, "bfloat16", 15)
    got = C.sample_items(b16.cuda()[:, 3:18004], u[:5].cuda(), top_k=100)
    check(b16[:, 3:18004], u[:5], *got, k=100)


def test_many_draws_follow_the_distribution_of_their_numbers():
    x = logits(1, 300, "float32", 16)
    u = ((torch.arange(5000, dtype=torch.float64) + 0.5) / 5000).view(1, -1)
    check(x, u, *call(x, u, p=0.95), p=0.95)


def test_repeatable_on_streams_and_in_graphs():
    x = logits(4, 40000, "float32", 17).cuda()
    u = torch.rand(4, 3, generator=gen(18)).cuda()
    want = C.sample_items(x, u, top_k=500, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = C.sample_items(x, u, top_k=500, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for _ in range(2):      # two graphs over the same inputs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = C.sample_items(x, u, top_k=500, top_p=0.9)
        graphs.append((g, out))
    for seed in range(3):
        x.copy_(logits(4, 40000, "float32", 30 + seed))
        u.copy_(torch.rand(4, 3, generator=gen(40 + seed)))
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = C.sample_items(x, u, top_k=500, top_p=0.9)
        for g, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_empty_and_refusals():
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    assert C.sample_items(x[:0], u[:0])[0].shape == (0,)
    assert C.sample_items(x, torch.zeros(3, 0, device="cuda"))[0].shape == (3, 0)
    bad = [lambda: C.sample_items(x[:, :0], u), lambda: C.sample_items(x.double(), u),
           lambda: C.sample_items(x, u[:2]), lambda: C.sample_items(x, u.half()),
           lambda: C.sample_items(x, u.cpu()), lambda: C.sample_items(x.cpu(), u),
           lambda: C.sample_items(x.t(), torch.zeros(10, device="cuda")),
           lambda: C.sample_items(x, u, temperature=-1), lambda: C.sample_items(x, u, temperature=float("nan")),
           lambda: C.sample_items(x, u, top_k=-1), lambda: C.sample_items(x, u, top_p=1.5),
           lambda: C.sample_items(x, u, min_p=-0.1), lambda: C.sample_items(x, u, mask=x),
           lambda: C.sample_items(x, u, mask=(x == 0)[:2]), lambda: C.sample_items(x, u, mask=(x == 0).cpu()),
           lambda: C.sample_items(x, u, top_k=torch.zeros(3, device="cuda")),
           lambda: C.sample_items(x, u, temperature=torch.ones(2, device="cuda"))]
    for f in bad:
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("shift", [-20.0, 20.0])
@pytest.mark.parametrize("n", [300, 5000, 20000, 60000])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_sixteen_bit_logits_of_either_sign_with_many_equals(dtype, n, shift):
    """Few distinct values, all of one sign: the bound is found digit by digit of a 16-bit logit."""
    x = (torch.randint(0, 24, (3, n), generator=gen(n)) / 16 + shift).to(getattr(torch, dtype))
    x[1, ::2] = -x[1, ::2]
    u = torch.rand(3, 6, generator=gen(n + 2))
    for s in (dict(k=n // 2), dict(k=n - 1, p=0.8), dict(p=0.35), dict(p=0.9, t=3.0), dict(k=n // 3, min_p=0.4)):
        check(x, u, *call(x, u, **s), **s)


@pytest.mark.parametrize("n", [64, 3000, 27278, 40000])
def test_min_p_and_infinite_temperature(n):
    """Every item weighs the same in an infinite temperature, infinite logits included; min_p = 1 keeps what
    equals the best."""
    x = logits(3, n, "float32", 12)
    x[1, : n // 4] = float("inf")
    x[2, 5] = x[2].max()
    u = torch.rand(3, 4, generator=gen(13))
    hot = torch.full((3,), float("inf"))
    it, pr = C.sample_items(x.cuda()[:1], u.cuda()[:1], temperature=hot.cuda()[:1])
    check(x[:1], u[:1], it, pr, t=np.inf)
    check(x, u, *call(x, u, min_p=1.0), min_p=1.0)
    check(x, u, *call(x, u, min_p=1e-30), min_p=1e-30)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [28672, 28673, 32768, 32769, 40960, 40961])
def test_rows_around_the_longest_that_a_workgroup_holds(n, dtype):
    x = logits(4, n, dtype, n)
    x[3] = (x[3] * 2).round()                # many equals
    mask = torch.rand(4, n, generator=gen(5)) < 0.8
    mask[2] = False
    u = torch.rand(4, 7, generator=gen(n + 1))
    for s in (dict(), dict(k=5000, p=0.9), dict(k=n // 2, t=3.0), dict(p=0.4, min_p=0.01), dict(k=100)):
        check(x, u, *call(x, u, mask=mask, **s), mask=mask, **s)
