"""Calls of the catalogue operators at the edge of what they take: every one is served or refused by a ValueError."""

import numpy as np
import pytest

from conftest import gpu_available
from oracle import ncf_oracle as O

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec import catalogue as C
    from movierec import engine as engine_module
    from test_catalogue_distill_gpu import both, problem
    from test_catalogue_model_gpu import gmf_weights, model
    from test_score_gpu import _engine, _weights


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


def test_draws_rank_by_the_logits_that_the_ranking_uses(tmp_path):
    """Models without the MFMA scorer draw from fp32 logits unless the caller asks for fewer bits."""
    shape = O.NCFShape(50, 2000, [], 64)
    eng = _engine(shape, gmf_weights(shape, 5))
    users, u = np.arange(50, dtype=np.int32), torch.zeros(50, device="cuda")
    best = eng.score_topk(users, k=1, precision="fp32")[0].view(-1)
    assert torch.equal(eng.sample_items(users, u, temperature=0.0)[0], best)
    eight = eng.score_logits(users, precision="fp8").argmax(1)
    assert not torch.equal(eight.int(), best)         # (8 bits name another for some users)
    assert torch.equal(eng.sample_items(users, u, temperature=0.0, precision="fp8")[0], eight.int())
    m = model(tmp_path, "g", layers=(), gmf=64, seed=4)
    np.testing.assert_array_equal(m.recommend_sampled(np.arange(50), temperature=0.0)[0],
                                  m.recommend(np.arange(50), k=1, precision="fp32")[0])


def test_masks_and_settings_belong_to_the_users_asked_for(monkeypatch):
    shape = O.NCFShape(64, 700, [64, 32, 16, 8], 8)
    eng = _engine(shape, _weights(shape, 8))
    users, u = np.arange(20, dtype=np.int32), torch.rand(20, 4, device="cuda")
    mask = torch.ones(64, 700, dtype=torch.bool, device="cuda")
    t = torch.ones(64, device="cuda")
    for part in (20, 7, 1):                           # users at a time
        monkeypatch.setattr(engine_module, "SAMPLE_LOGITS", part * 700)
        bad = [dict(mask=mask), dict(mask=mask[:21]), dict(mask=mask[:19]), dict(mask=mask[:1]), dict(mask=mask[:7]),
               dict(mask=mask[:20, :699]), dict(mask=mask[0, :20]), dict(mask=mask[:20].float()),
               dict(temperature=t), dict(temperature=t[:7]), dict(temperature=t[:6]), dict(temperature=t[:1]),
               dict(temperature=t[0]), dict(top_k=t[:7].int()), dict(top_p=t[:21]), dict(min_p=t[:20].view(20, 1))]
        for kw in bad:
            with pytest.raises(ValueError):
                eng.sample_items(users, u, **kw)
        items, probs = eng.sample_items(users, u, mask=mask[:20], temperature=t[:20])
        assert (items >= 0).all() and items.shape == (20, 4)
    for kw in (dict(mask=mask[:1]), dict(temperature=t[:1]), dict(top_p=2.0)):   # (no user: still checked)
        with pytest.raises(ValueError):
            eng.sample_items(users[:0], u[:0], **kw)


def test_settings_that_are_no_numbers():
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    it, y = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.zeros(3, 1, device="cuda")
    bad = [lambda: C.sample_items(x, u, top_k=2.5), lambda: C.sample_items(x, u, top_k="2"),
           lambda: C.sample_items(x, u, top_k=None), lambda: C.sample_items(x, u, temperature="1"),
           lambda: C.sample_items(x, u, temperature=None), lambda: C.sample_items(x, u, top_p=[0.5, 0.5, 0.5]),
           lambda: C.sample_items(x, u, min_p=1j), lambda: C.sample_items(x, u, temperature=np.ones(3)),
           lambda: C.distill_loss(x, it, y, temperature="1"), lambda: C.distill_loss(x, it, y, temperature=None),
           lambda: C.distill_loss(x, it, y, temperature=torch.ones(3, device="cuda")),
           lambda: C.distill_loss_grad(x, it, y, "1"), lambda: C.distill_loss_grad(x, it, y, None),
           lambda: C.distill_loss_grad(x, it, y, [1.0, 1.0, 1.0])]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    # numbers of numpy are numbers
    a = C.sample_items(x, u, temperature=np.float32(0.5), top_k=np.int64(3), top_p=np.float64(0.9))
    b = C.sample_items(x, u, temperature=0.5, top_k=3, top_p=0.9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(C.distill_loss_grad(x, it, y, np.float32(2))[1], C.distill_loss_grad(x, it, y, 2)[1])


def test_more_draws_than_workgroups_of_one_launch():
    """5,000,000 draws of one row of 41,000 items: what a draw gives does not depend on the others."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 41000, generator=g).cuda()
    u = torch.rand(1, 5000000, generator=g).cuda()
    items, probs = C.sample_items(x, u, top_k=300, top_p=0.9)
    pick = torch.cat([torch.arange(0, 5000000, 4999), torch.arange(4999000, 5000000)]).cuda()
    few = C.sample_items(x, u[:, pick].contiguous(), top_k=300, top_p=0.9)
    assert torch.equal(items[:, pick], few[0]) and torch.equal(probs[:, pick], few[1])
    assert int(items.min()) >= 0 and float(probs.min()) > 0


def test_more_rows_than_workgroups_of_one_launch():
    """70,000,000 rows of two items: the same as those rows by themselves, on both sides of every 2^21st."""
    rows = 70000000
    x = torch.randn(rows, 2, device="cuda", dtype=torch.bfloat16)
    u = torch.rand(rows, device="cuda")
    k = torch.randint(0, 3, (rows,), device="cuda", dtype=torch.int32)
    at = torch.cat([torch.arange(0, rows, 2 ** 21)[:, None] + torch.arange(-3, 4), torch.arange(rows - 7, rows)[None]])
    at = at[(at >= 0) & (at < rows)].cuda()
    items, probs = C.sample_items(x, u, top_k=k)
    few = C.sample_items(x[at], u[at], top_k=k[at])
    assert torch.equal(items[at], few[0]) and torch.equal(probs[at], few[1])
    assert int(items.min()) == 0 and int(items.max()) == 1
    del items, probs
    it = torch.randint(-1, 2, (rows, 1), device="cuda", dtype=torch.int32)
    y = torch.randn(rows, 1, device="cuda")
    lse = y.view(-1) + 0.5
    loss, grad = C.distill_loss_grad(x, it, y, teacher_lse=lse)
    few = C.distill_loss_grad(x[at], it[at], y[at], teacher_lse=lse[at])
    assert torch.equal(loss[at], few[0]) and torch.equal(grad[at], few[1])
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all()
    del loss, grad
    loss, state = C.distill_loss(x, it, y, teacher_lse=lse)
    few = C.distill_loss(x[at], it[at], y[at], teacher_lse=lse[at])
    assert torch.equal(loss[at], few[0])
    grad = C.distill_grad(x, it, y, state, teacher_lse=lse)
    assert torch.equal(grad[at], C.distill_grad(x[at], it[at], y[at], few[1], teacher_lse=lse[at]))


def test_product_of_more_columns_than_one_launch_takes():
    """One row by 1,100,000,000 columns of one value: every output is its column's value, exactly."""
    n = 1100000000
    b = (torch.arange(n, device="cuda", dtype=torch.int32) % 127).to(torch.uint8).view(n, 1)
    q = torch.ones(1, 1, device="cuda").to(torch.float8_e4m3fn)
    scale = torch.ones((n + 127) // 128, 1, device="cuda")
    scale[-1] = 2.0
    y = C.matmul_blocks(q, torch.ones(1, 1, device="cuda"), b.view(torch.float8_e4m3fn), scale,
                        out_dtype=torch.bfloat16).view(-1)
    value = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().bfloat16().cuda()
    for at in range(0, n, 1 << 27):
        part = slice(at, min(n, at + (1 << 27)))
        want = value[b.view(-1)[part].long()]
        if part.stop == n:
            want[-(n % 128 or 128):] *= 2
        assert torch.equal(y[part], want), at


def test_scratch_is_what_the_rows_need():
    """Rows that a workgroup holds ask for no scratch: beside its outputs a call allocates next to nothing."""
    def grown(call):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        out = call()
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - before - sum(o.numel() * o.element_size() for o in out)

    u = torch.rand(500, device="cuda")
    for n, dtype in ((32768, torch.bfloat16), (40960, torch.float32)):
        x = torch.randn(500, n, device="cuda").to(dtype)
        assert grown(lambda: C.sample_items(x, u, top_k=50)) < 1 << 16
    x = torch.randn(500, 50000, device="cuda")
    it, y = torch.zeros(500, 64, dtype=torch.int32, device="cuda"), torch.zeros(500, 64, device="cuda")
    assert grown(lambda: C.distill_loss(x, it, y)) < 1 << 12      # (outputs are rounded up to 512 bytes)


@pytest.mark.parametrize("dims", [(70, 130, [], 12), (200, 1, [], 64), (3, 2111, [], 130), (129, 64, [], 16),
                                  (65, 65, [], 1)], ids=str)
def test_fp32_logits_of_gmf_models_are_the_forwards(dims):
    """Every item's logit in fp32 has the bits of the pair's own forward (the same roundings in the same order)."""
    shape = O.NCFShape(*dims)
    eng = _engine(shape, gmf_weights(shape, 9))
    users = torch.from_numpy(np.random.RandomState(3).permutation(dims[0] + 2).astype(np.int32) - 1).cuda()
    z = eng.score_logits(users, precision="fp32")
    pairs = eng.predict_logits(users.view(-1, 1).expand(-1, dims[1]), torch.arange(dims[1]).repeat(users.numel()))
    assert torch.equal(torch.nan_to_num(z.view(-1), nan=77.0), torch.nan_to_num(pairs, nan=77.0))
    known = (users >= 0) & (users < dims[0])
    assert torch.equal(torch.isnan(z).all(1), ~known) and torch.equal(torch.isnan(z).any(1), ~known)


def test_teacher_lists_of_no_length_are_refused(tmp_path):
    m = model(tmp_path, "t")
    x = [np.arange(3), np.arange(12).reshape(3, 4)]
    for top in (0, -1):
        with pytest.raises(ValueError):
            m.distill_on_batch(x, m, top=top)
    assert np.isfinite(m.distill_on_batch(x, m, top=9))      # (more than there are candidates: all)
