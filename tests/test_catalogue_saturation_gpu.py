"""Distillation of models whose output sigmoid is 0 or 1 in float32: the step is taken on the logits.

Tolerances.  A logit of a GMF-only model is a float32 sum of g products of three factors and a bias: off by at most
e = (2 g + 4) 2^-24 (sum of magnitudes).  That changes a loss by at most 2 e / t of the list's mass and a probability
by 2 e / t of itself; beside it stand the kernel's own errors (test_catalogue_distill_gpu.py).  The step sees the
gradient dz of a pair as (p - y) / (b c) with y = p - b c dz: the two p are off from each other by 2^-22 + p (1 - p)
2 e, y is one rounding more.  A weight's gradient sums dz times what multiplies it, n terms with n + 5 roundings, and
is read off an SGD step of lr 1 (the weight's own rounding).  Logits of layered models: 1e-5 for |z| up to 5
(test_score_gpu.py), in proportion beyond."""

import numpy as np
import pytest

from conftest import gpu_available
from oracle import ncf_oracle as O

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec.engine import NCFEngine
    from test_catalogue_distill_gpu import reference
    from test_catalogue_model_gpu import gmf_weights, model, softmax_target
    from test_score_gpu import _engine, _weights


def reach(shape, w, users, items, z):
    """Item factors such that pair (users[j], items[j]) has the logit z[j]; every item of the list stands once."""
    for u, i, want in zip(users, items, z):
        a = w["user_gmf_embedding"][u] * w["output/kernel"][:shape.gmf_dim, 0]
        w["item_gmf_embedding"][i] = 0
        w["item_gmf_embedding"] = w["item_gmf_embedding"].astype(np.float32).astype(np.float64)
        now = float(np.log(1 / (1 / O.forward(shape, w, np.array([u]), np.array([i]))[0][0] - 1)))
        w["item_gmf_embedding"][i] = (want - now) * a / (a @ a)
    return {k: v.astype(np.float32).astype(np.float64) for k, v in w.items()}


def logits(shape, w, users, items):
    z = O.score_all_items(shape, w, users)
    return np.take_along_axis(z, items.astype(np.int64), 1)


@pytest.mark.parametrize("lse", [False, True])
def test_step_of_a_saturated_student(lse):
    shape = O.NCFShape(40, 60, [], 12)
    rng = np.random.RandomState(3)
    b, c, top, t = 8, 20, 5, 1.5
    w = gmf_weights(shape, 11)
    users = rng.permutation(40)[:b].astype(np.int32)
    items = np.stack([rng.permutation(50)[:c] for _ in range(b)]).astype(np.int32)
    want = [20.0, 40.0, -20.0, 15.0, 13.0, 120.0, 16.7, -120.0]
    items[:, 4] = 50 + np.arange(b)                   # an item of each user's own
    w = reach(shape, w, users, items[:, 4], want)
    z = logits(shape, w, users, items)
    assert np.max(np.abs(z[:, 4] - want)) < 1e-3
    zt = np.clip(z, -12, 12) + rng.randn(b, c)
    places = np.argsort(-zt, 1)[:, :top].copy()
    places[2, 0] = places[7, 0] = 4                   # teachers that like what the student has at nearly 0
    y = np.take_along_axis(zt, places, 1).astype(np.float32)
    ls = np.log(np.exp(zt / t).sum(1)).astype(np.float32) + np.float32(0.3) if lse else None
    ref = reference(torch.from_numpy(z), torch.from_numpy(places), torch.from_numpy(y), t, ls, np.full(b, t * t / b))
    loss, dz, pc, qv, mass, part = ref
    eng = NCFEngine(40, 60, [], 12, max_batch=1024, optimizer="sgd", lr=1.0)
    eng.set_keras_weights(w)
    got = eng.distill_step(users, items, torch.from_numpy(places).cuda(), torch.from_numpy(y).cuda(), temperature=t,
                           teacher_lse=None if ls is None else torch.from_numpy(ls).cuda()).cpu().numpy()
    g = 12
    gu, gi = w["user_gmf_embedding"][users], w["item_gmf_embedding"][items]
    wo = w["output/kernel"][:, 0]
    e = (2 * g + 4) * 2.0 ** -24 * ((np.abs(gu)[:, None] * np.abs(gi)) @ np.abs(wo) + abs(w["output/bias"][0]))
    e = e.max(1)
    ek = 2.0 ** -23 * (1.5 * 42 / np.log(2) + 1)
    assert np.all(np.abs(got - loss) <= mass * (2 * e / t + 2 * ek) + np.abs(loss) * 2.0 ** -23)
    # pairs whose p lies outside Keras' clip have no gradient
    with np.errstate(over="ignore"):
        p = 1 / (1 + np.exp(-z))
    lo, hi = O.clip_bounds()
    inside = (p >= lo) & (p <= hi)
    assert (~inside).sum() == 6 and not inside[[0, 1, 2, 5, 6, 7], 4].any()
    e_dz = (np.abs(pc) * (2 * e[:, None] / t + 2 * ek + 2.0 ** -21) + qv * 2.0 ** -22 + part * (4 * e[:, None] / t + 2 * ek)) * t / b
    e_dz += (2.0 ** -22 + p * (1 - p) * 2 * e[:, None] + 2.0 ** -23 * (p + b * c * np.abs(dz))) / (b * c)
    dz, e_dz = np.where(inside, dz, 0), np.where(inside, e_dz, 0)
    now = eng.keras_weights()

    def check(name, at, terms, errors):
        """terms: (pairs, what they go to, factor); the step's gradient of weight `at` against their sum"""
        have = w[name][at] - now[name][at]
        tol = errors + (terms[1] + 5) * 2.0 ** -24 * terms[2] + 2.0 ** -23 * (np.abs(w[name][at]) + np.abs(have))
        assert np.all(np.abs(have - terms[0]) <= tol), (name, np.max(np.abs(have - terms[0]) - tol))

    for r, u in enumerate(users):
        f = wo * gi[r]                                # c x g
        check("user_gmf_embedding", u, (dz[r] @ f, c, np.abs(dz[r]) @ np.abs(f)), e_dz[r] @ np.abs(f))
    for i in range(60):
        r, j = np.nonzero(items == i)
        f = wo * gu[r]
        check("item_gmf_embedding", i, (dz[r, j] @ f, len(r), np.abs(dz[r, j]) @ np.abs(f)), e_dz[r, j] @ np.abs(f))
    f = (gu[:, None] * gi).reshape(-1, g)
    check("output/kernel", (slice(None), 0), (dz.reshape(-1) @ f, b * c, np.abs(dz.reshape(-1)) @ np.abs(f)),
          e_dz.reshape(-1) @ np.abs(f))
    assert any(np.abs(now[k] - w[k]).max() > 1e-3 for k in w)


@pytest.mark.parametrize("layers", [(64, 32, 16, 8), (6, 4)], ids=str)
def test_saturated_teacher_and_student(tmp_path, layers):
    """Logits of 15 and more on both sides: the teacher's order and the loss are those of the logits."""
    teacher, student = model(tmp_path, "t", layers=layers, seed=2), model(tmp_path, "s", layers=layers, seed=3)
    rng = np.random.RandomState(1)
    b, c, top, t = 6, 12, 4, 2.0
    users = rng.permutation(50)[:b].astype(np.int32)
    items = np.stack([rng.permutation(100)[:c] for _ in range(b)]).astype(np.int32)
    items[:, 1:4] = 100 + np.arange(3 * b).reshape(b, 3)
    shape = O.NCFShape(50, 120, list(layers), 8)
    z = {}
    for m, want in ((teacher, [30.0, 15.0, 15.4]), (student, [17.0, 14.6, -25.0])):
        w = _weights(shape, 5 if m is teacher else 6)
        w = reach(shape, w, np.repeat(users, 3), items[:, 1:4].reshape(-1), want * b)
        m.model.engine.set_keras_weights(w)
        z[m] = logits(shape, w, users, items)
    zt = z[teacher]
    places = np.argsort(-zt, 1)[:, :top]
    assert (places[:, :3] == [1, 3, 2]).all()
    want = softmax_target(z[student], places, np.take_along_axis(zt, places, 1), t, np.log(np.exp(zt / t).sum(1)))[0]
    loss = student.distill_on_batch([users, items], teacher, top=top, temperature=t)
    e, ek = 1e-5 * 30 / 5, 2.0 ** -23 * (1.5 * 42 / np.log(2) + 1)     # (masses c and sum q: at most 1 each)
    assert abs(loss - want.mean()) <= 2 * (2 * e / t + 2 * ek) + want.mean() * 2.0 ** -23
    after = student.model.engine.keras_weights()
    assert all(np.isfinite(v).all() for v in after.values())


@pytest.mark.parametrize("dims", [(40, 60, [64, 32, 16, 8], 8), (40, 60, [128, 64, 32, 16], 64), (40, 60, [], 12),
                                  (30, 40, [7, 5], 3), (40, 60, [256, 128, 64, 32], 128)], ids=str)
def test_logits_of_pairs(dims):
    """NCFEngine.predict_logits in each of the forward kernels, and where the sigmoid has no digits left."""
    shape = O.NCFShape(*dims)
    w = gmf_weights(shape, 21) if not dims[2] else _weights(shape, 21)
    users = np.repeat(np.arange(20), 30).astype(np.int32)
    items = np.tile(np.arange(30), 20).astype(np.int32)
    w = reach(shape, w, [0, 1, 2, 3], [0, 1, 2, 3], [25.0, -40.0, 16.0, 9.0])
    eng = _engine(shape, w)
    want = O.score_all_items(shape, w, np.arange(20))[:, :30].reshape(-1)
    z = eng.predict_logits(users, items)
    assert z.shape == (600,) and z.dtype == torch.float32
    assert np.all(np.abs(z.double().cpu().numpy() - want) <= 1e-5 * np.maximum(np.abs(want), 40) / 5)
    p = eng.predict(users, items)
    assert torch.all((torch.sigmoid(z) - p).abs() <= p * 2.0 ** -22)
    assert p[0] == 1                                  # (25: the sigmoid has lost it)
    ids = torch.tensor([3, dims[0], -1, 7], dtype=torch.int32, device="cuda")
    assert torch.isnan(eng.predict_logits(ids, ids)).cpu().tolist() == [False, True, True, False]
    assert eng.predict_logits(users[:0], items[:0]).shape == (0,)
    with pytest.raises(ValueError):
        eng.predict_logits(users, items[:5])
