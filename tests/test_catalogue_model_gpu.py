"""The catalogue operators as the model uses them: logits of every item, items drawn from them, and a
training step towards a teacher, against the numpy oracle.

Tolerances.  fp32 logits: that of the top-k scorer (test_score_gpu.py).  fp16 logits: ``half_error``, the
scorer's roundings carried through its layers (a tolerance for the best items' logits, as the top-k tests
have it, does not bound all of them: 5.007e-3 was seen where it says 5e-3).  8-bit logits: a factor
a is off by at most max(2^-4 |a|, 2^-10 s) (half a step of e4m3: 3 bits after the point, steps of 2^-9 s
below 2^-6 s, s = max|a| / 448 its block's scale), so a product of factors by ea |b| + |a| eb + ea eb, and
float32 sums by (f + 3) 2^-24 of the sum of magnitudes, f values.  A distillation step: see there."""

import numpy as np
import pytest

from conftest import gpu_available
from oracle import ncf_oracle as O

pytestmark = pytest.mark.gpu

if gpu_available():
    import torch
    from movierec import catalogue as C
    from movierec.engine import NCFEngine
    from test_catalogue_sample_gpu import check as check_draws
    from test_score_gpu import TOL_Z, _engine, _weights


def gmf_weights(shape, seed):
    rng = np.random.RandomState(seed)
    w = O.init_weights(shape, seed=seed)
    w = {k: rng.uniform(-0.8, 0.8, size=v.shape) for k, v in w.items()}
    return {k: v.astype(np.float32).astype(np.float64) for k, v in w.items()}


def block_error(x):
    """What e4m3 with a scale for each 128 values of a row can be off (x: rows x values)."""
    s = np.repeat(np.stack([np.abs(x[:, j:j + 128]).max(1) / 448 for j in range(0, x.shape[1], 128)], 1),
                  128, axis=1)[:, :x.shape[1]]
    return np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s) * (1 + 2.0 ** -20)


def half_error(shape, w, users):
    """What the fp16 scorer's logits of all items can be off.  With h = 2^-11 (half a step of fp16, and what
    each rounded operand is relatively off): layer 2 takes max(c, -a) of the rounded item term c and user term a
    (off by h max(|c|, |a|)) times rounded weights, so its sums are off by 2 h |W2|' max(|c|, |a|); a relu keeps
    an error; layer 3 rounds the activations and its weights again, and so does the output layer; the GMF term
    is a product of two rounded factors.  The sums are fp32 over at most 128 values of each (2^-17 of their
    magnitude covers them); 1.01 covers products of errors; values below fp16's normal range are off by half a
    step of 2^-24 at most, 2^-25 a value."""
    h, tiny = 2.0 ** -11 + 2.0 ** -17, 2.0 ** -25
    L = shape.layers
    du = L[0] // 2
    w1, w2, w3 = (w["hidden_%d/kernel" % i] for i in (1, 2, 3))
    a = w["user_embedding"][users] @ w1[:du] + w["hidden_1/bias"]
    c = w["item_embedding"] @ w1[du:]
    big = np.maximum(np.abs(a)[:, None, :], np.abs(c)[None])
    s1 = np.maximum(a[:, None] + c[None], 0)
    e2 = (2 * h * big + tiny) @ np.abs(w2) + tiny * (big.sum(-1, keepdims=True))
    h2 = np.maximum(s1 @ w2 + w["hidden_2/bias"], 0)
    e3 = (e2 + 2 * h * h2 + tiny) @ np.abs(w3) + tiny * h2.sum(-1, keepdims=True)
    h3 = np.maximum(h2 @ w3 + w["hidden_3/bias"], 0)
    out = np.abs(w["output/kernel"][:, 0])
    g = shape.gmf_dim
    e = (e3 + 2 * h * h3 + tiny) @ out[g:] + tiny * h3.sum(-1)
    if g:
        u = np.abs(w["user_gmf_embedding"][users]) * out[:g]
        i = np.abs(w["item_gmf_embedding"])
        e = e + 2 * h * u @ i.T + tiny * (u.sum(1)[:, None] + i.sum(1)[None])
    return 1.01 * e + 2.0 ** -20


@pytest.mark.parametrize("dims", [(943, 1682, [], 8), (200, 301, [], 64), (50, 4000, [], 130)], ids=str)
def test_logits_of_gmf_models_in_8_bits(dims):
    shape = O.NCFShape(*dims)
    w = gmf_weights(shape, 1)
    eng = _engine(shape, w)
    users = np.random.RandomState(2).randint(0, dims[0], 37).astype(np.int32)
    z = eng.score_logits(users).double().cpu().numpy()     # (8 bits are these models' first choice)
    ref = O.score_all_items(shape, w, users)
    g = dims[3]
    a = w["user_gmf_embedding"][users] * w["output/kernel"][:, 0]
    b = w["item_gmf_embedding"]
    a32 = a.astype(np.float32).astype(np.float64)
    ea, eb = block_error(a32) + np.abs(a - a32), block_error(b)
    tol = ea @ np.abs(b).T + np.abs(a) @ eb.T + ea @ eb.T
    tol += (g + 3) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T + np.abs(w["output/bias"][0]))
    assert np.all(np.abs(z - ref) <= tol)
    np.testing.assert_array_equal(z, eng.score_logits(users, precision="fp8").double().cpu().numpy())
    z32 = eng.score_logits(users, precision="fp32").double().cpu().numpy()
    assert np.max(np.abs(z32 - ref)) <= TOL_Z["fp32"]
    with pytest.raises(ValueError):
        eng.score_logits(users, precision="fp16")


@pytest.mark.parametrize("dims", [(200, 999, [128, 64, 32, 16], 64), (150, 640, [128, 64, 32, 16], 0),
                                  (100, 333, [64, 32, 16, 8], 8), (90, 2111, [64, 32, 16, 8], 0)], ids=str)
def test_logits_of_scorer_models(dims):
    shape = O.NCFShape(*dims)
    w = _weights(shape, 3)
    eng = _engine(shape, w)
    users = np.random.RandomState(4).randint(0, dims[0], 77).astype(np.int32)
    ref = O.score_all_items(shape, w, users)
    for precision in ("fp16", "fp32"):
        z = eng.score_logits(users, precision=precision).double().cpu().numpy()
        assert z.shape == ref.shape
        tol = TOL_Z["fp32"] if precision == "fp32" else half_error(shape, w, users)
        assert np.all(np.abs(z - ref) <= tol)
    with pytest.raises(ValueError):
        eng.score_logits(users, precision="fp8")
    with pytest.raises(ValueError):
        eng.score_logits(users, precision="fp4")
    assert eng.score_logits(users[:0]).shape == (0, dims[1])


def test_logits_of_any_shape():
    shape = O.NCFShape(31, 17, [7, 5], 3)
    w = _weights(shape, 6)
    z = _engine(shape, w).score_logits(np.arange(31, dtype=np.int32)).double().cpu().numpy()
    assert np.max(np.abs(z - O.score_all_items(shape, w, np.arange(31)))) <= TOL_Z["fp32"]


@pytest.mark.parametrize("dims", [(40, 90, [], 16), (40, 90, [64, 32, 16, 8], 8), (40, 90, [6, 4], 0)], ids=str)
def test_users_outside_the_table(dims):
    shape = O.NCFShape(*dims)
    eng = _engine(shape, gmf_weights(shape, 7) if not dims[2] else _weights(shape, 7))
    ids = torch.tensor([3, 40, -1, 7], dtype=torch.int32, device="cuda")
    z = eng.score_logits(ids)
    assert torch.isnan(z).all(1).tolist() == [False, True, True, False] and not torch.isnan(z[[0, 3]]).any()
    items, probs = eng.sample_items(ids, torch.rand(4, 3, device="cuda"), top_k=5)
    assert (items[1:3] == -1).all() and (probs[1:3] == 0).all() and (items[[0, 3]] >= 0).all()


def test_engine_draws_are_those_of_its_logits(monkeypatch):
    shape = O.NCFShape(64, 700, [64, 32, 16, 8], 8)
    eng = _engine(shape, _weights(shape, 8))
    users = np.arange(50, dtype=np.int32)
    u = torch.rand(50, 4, device="cuda")
    mask = torch.rand(50, 700, device="cuda") < 0.7
    t = torch.rand(50, device="cuda") + 0.5
    z = eng.score_logits(users)
    items, probs = eng.sample_items(users, u, temperature=t, top_k=40, top_p=0.9, mask=mask)
    check_draws(z.cpu(), u.cpu(), items, probs, mask=mask.cpu(), t=t.double().cpu().numpy(), k=40, p=0.9)
    # the same in several parts of the users: 7 at a time
    from movierec import engine
    monkeypatch.setattr(engine, "SAMPLE_LOGITS", 7 * 700)
    parts = eng.sample_items(users, u, temperature=t, top_k=40, top_p=0.9, mask=mask)
    assert torch.equal(parts[0], items) and torch.equal(parts[1], probs)
    with pytest.raises(ValueError):
        eng.sample_items(users, u[:49])
    with pytest.raises(ValueError):
        eng.sample_items(users, u, mask=mask.cpu().numpy())


def model(tmp_path, name, layers=(64, 32, 16, 8), gmf=8, seed=1, l2=0.0):
    from movierec.model import MovierecModel
    params = dict(num_users=50, num_items=120, layers_sizes=list(layers), layers_l2reg=[l2] * len(layers),
                  optimizer="adam", lr=0.001, batch_size=100, num_negs_per_pos=9, batch_size_eval=200,
                  num_negs_per_pos_eval=99, k=5, seed=seed, gmf_dim=gmf)
    return MovierecModel(params, name, str(tmp_path), verbose=0)


def test_model_recommends_by_draws(tmp_path):
    m = model(tmp_path, "a")
    seen = np.ones((3, 120), bool)
    seen[0, ::2] = False
    seen[1] = False                       # nothing left for this user
    a = m.recommend_sampled([0, 7, 49], draws=6, top_k=30, top_p=0.9, mask=seen, seed=5)
    b = m.recommend_sampled([0, 7, 49], draws=6, top_k=30, top_p=0.9, mask=seen, seed=5)
    np.testing.assert_array_equal(a[0], b[0])
    np.testing.assert_array_equal(a[1], b[1])
    assert a[0].shape == (3, 6) and a[0].dtype == np.int32
    assert np.all(a[0][0] % 2 == 1) and np.all(a[0][1] == -1) and np.all(a[1][1] == 0)
    best = m.recommend([0, 7, 49], k=1)[0]
    greedy = m.recommend_sampled([0, 7, 49], temperature=0.0)[0]
    np.testing.assert_array_equal(greedy, best)
    with pytest.raises(ValueError):
        m.recommend_sampled([50])
    with pytest.raises(ValueError):
        m.recommend_sampled([1], draws=0)
    assert m.recommend_sampled([], draws=2)[0].shape == (0, 2)


def softmax_target(z, places, y, t, lse):
    """Loss per user and dz = t^2 / b d loss / dz of the mean divergence, in float64."""
    b, c = z.shape
    p = np.exp(z / t - np.log(np.exp(z / t).sum(1, keepdims=True)))
    loss, dz = np.zeros(b), np.zeros((b, c))
    for r in range(b):
        ref = np.log(np.exp(y[r] / t).sum()) if lse is None else lse[r]
        q = np.exp(y[r] / t - ref)
        loss[r] = (q * (np.log(q) - np.log(p[r, places[r]]))).sum()
        cin = cout = q.sum()
        if lse is not None:
            out = np.ones(c, bool)
            out[places[r]] = False
            q0, p0 = 1 - q.sum(), p[r, out].sum()
            if q0 > 0 and p0 > 0:
                loss[r] += q0 * np.log(q0 / p0)
                cin, cout = q.sum() + q0, q.sum() + q0 - q0 / p0
        coef = np.full(c, cout)
        coef[places[r]] = cin
        d = p[r] * coef
        np.add.at(d, places[r], -q)
        dz[r] = d * t * t / t / b
    return loss, dz


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("dims", [(40, 60, [64, 32, 16, 8], 8), (40, 60, [], 12), (30, 40, [6, 4], 0)], ids=str)
def test_distillation_step_matches_the_oracle(dims, lse):
    """The step against the oracle's training step on the float64 labels p - b c dz: the same comparison
    as a training step's on labels (weights to 1e-5 after one Adam step of 1e-3, whose direction is the
    gradient's sign where its size passes the fp32 error; the output bias is left out, whose gradient is 0:
    a softmax does not see it), and the losses: p is off by 2e-6 relative to p (1 - p) at the |z| < 6 here
    (the forward's own test), so a logit by 2e-6 / (p (1 - p)) <= 2e-6 * 410, and a loss by twice that."""
    shape = O.NCFShape(*dims)
    w = gmf_weights(shape, 11) if not dims[2] else _weights(shape, 11)
    eng = _engine(shape, w)
    rng = np.random.RandomState(12)
    b, c, top, t = 8, 20, 5, 1.5
    users = rng.randint(0, dims[0], b).astype(np.int32)
    items = np.stack([rng.permutation(dims[1])[:c] for _ in range(b)]).astype(np.int32)
    pairs = np.repeat(users, c), items.reshape(-1)
    p, cache = O.forward(shape, w, *pairs)
    z = np.log(p / (1 - p)).reshape(b, c)
    assert np.abs(z).max() < 6
    zt = z + rng.randn(b, c)
    places = np.argsort(-zt, 1)[:, :top].copy()
    y = np.take_along_axis(zt, places, 1).astype(np.float32)
    ls = np.log(np.exp(zt / t).sum(1)).astype(np.float32) if lse else None
    loss, dz = softmax_target(z, places, y.astype(np.float64), t, None if ls is None else ls.astype(np.float64))
    got = eng.distill_step(users, items, torch.from_numpy(places).cuda(), torch.from_numpy(y).cuda(), temperature=t,
                           teacher_lse=None if ls is None else torch.from_numpy(ls).cuda())
    assert np.max(np.abs(got.cpu().numpy() - loss)) <= 2 * 2e-6 * 410
    labels = (p.reshape(b, c) - b * c * dz).reshape(-1)
    ref = {k: v.copy() for k, v in w.items()}
    st = O.new_opt_state(ref)
    O.train_step(shape, ref, st, pairs[0], pairs[1], labels,
                 dict(optimizer="adam", lr=0.001, beta_1=0.9, beta_2=0.999, layers_l2reg=[0] * max(len(dims[2]), 1)))
    grad = O.loss_and_grads(shape, w, pairs[0], pairs[1], labels, [0] * max(len(dims[2]), 1))[1]
    now = eng.keras_weights()
    for name in sorted(set(ref) - {"output/bias"}):
        clear = np.abs(grad[name]) > 1e-4     # the sign of a gradient this large is certain
        assert clear.any(), name
        assert np.max(np.abs(now[name] - ref[name])[clear]) <= 1e-5, name
    assert int(eng.step.item()) == 1


def test_distillation_step_gradient_is_the_labels(tmp_path):
    """The gradient itself, before the optimizer: forward_backward on the same labels gives the dense
    layers' gradient of the divergence, checked against central differences of the divergence over the
    output bias and two output weights (float64 oracle, h = 1e-4: the third derivative times h^2 is below
    1e-6 of these sizes)."""
    shape = O.NCFShape(30, 50, [16, 8], 4)
    w = _weights(shape, 13)
    rng = np.random.RandomState(14)
    b, c, t = 6, 10, 2.0
    users = rng.randint(0, 30, b).astype(np.int32)
    items = np.stack([rng.permutation(50)[:c] for _ in range(b)]).astype(np.int32)
    pairs = np.repeat(users, c), items.reshape(-1)
    zt = rng.randn(b, c) * 2
    places = np.argsort(-zt, 1)[:, :3].copy()
    y = np.take_along_axis(zt, places, 1).astype(np.float32)

    def total(weights):
        p = O.forward(shape, weights, *pairs)[0]
        z = np.log(p / (1 - p)).reshape(b, c)
        return softmax_target(z, places, y.astype(np.float64), t, None)[0].mean() * t * t

    eng = _engine(shape, w)
    p = eng.predict(*pairs)
    _, dz = C.distill_loss_grad(torch.logit(p).view(b, c), torch.from_numpy(places).cuda(),
                                torch.from_numpy(y).cuda(), grad_loss=t * t / b, temperature=t)
    grads = eng.alloc_grads()
    eng.forward_backward(pairs[0], pairs[1], torch.sub(p, dz.view(-1), alpha=float(b * c)), group=c, k=1,
                         inv_batch=1.0 / (b * c), grads=grads)
    got = eng.layout.from_device(grads[0][:eng.num_rows].cpu().numpy(), grads[1].cpu().numpy())
    for name, at in (("output/bias", 0), ("output/kernel", 1), ("output/kernel", 5)):
        up, dn = ({k: v.copy() for k, v in w.items()} for _ in range(2))
        up[name].reshape(-1)[at] += 1e-4
        dn[name].reshape(-1)[at] -= 1e-4
        diff = (total(up) - total(dn)) / 2e-4
        assert abs(got[name].reshape(-1)[at] - diff) <= 1e-4 * max(1.0, abs(diff)), (name, at)


def test_models_distil_and_sample_together(tmp_path):
    """A teacher's ranking taught to a smaller model, then items drawn from the student: the calls as a
    program makes them, the loss of the first step against the oracle's logits."""
    teacher, student = model(tmp_path, "t", seed=2), model(tmp_path, "s", layers=(16, 8), gmf=4, seed=3)
    rng = np.random.RandomState(1)
    users = rng.randint(0, 50, 12).astype(np.int32)
    items = np.stack([rng.permutation(120)[:25] for _ in range(12)]).astype(np.int32)
    zs = {}
    for m, shape in ((teacher, O.NCFShape(50, 120, [64, 32, 16, 8], 8)), (student, O.NCFShape(50, 120, [16, 8], 4))):
        p = O.forward(shape, {k: v.astype(np.float64) for k, v in m.model.get_weights().items()},
                      np.repeat(users, 25), items.reshape(-1))[0]
        zs[m] = np.log(p / (1 - p)).reshape(12, 25)
    zt = zs[teacher]
    places = np.argsort(-zt, 1)[:, :6]
    want = softmax_target(zs[student], places, np.take_along_axis(zt, places, 1), 2.0,
                          np.log(np.exp(zt / 2.0).sum(1)))[0].mean()
    before = {k: v.copy() for k, v in student.model.get_weights().items()}
    loss = student.distill_on_batch([users, items], teacher, top=6, temperature=2.0)
    assert abs(loss - want) <= 1e-5
    after = student.model.get_weights()
    assert any(np.any(before[k] != after[k]) for k in before)
    for _ in range(3):
        assert np.isfinite(student.distill_on_batch([users, items], teacher, top=6, temperature=2.0))
    drawn, probs = student.recommend_sampled(users, draws=4, top_k=20, seed=0)
    assert drawn.shape == (12, 4) and np.all(drawn >= 0) and np.all(probs > 0)
    student.model.engine.check_errors()
    for bad in ([users, items.reshape(-1)], [users[:3], items], [users, items[:, :0]]):
        with pytest.raises(ValueError):
            student.distill_on_batch(bad, teacher)
    with pytest.raises(ValueError):
        student.distill_on_batch([users, items + 120], teacher)
    with pytest.raises(ValueError):
        student.distill_on_batch([users, items], teacher, temperature=0)


def test_distillation_leaves_out_users_with_unknown_ids():
    shape = O.NCFShape(30, 40, [64, 32, 16, 8], 8)
    w = _weights(shape, 15)
    a, b = _engine(shape, w), _engine(shape, w)
    rng = np.random.RandomState(16)
    users = torch.from_numpy(rng.randint(0, 30, 4).astype(np.int32)).cuda()
    items = torch.from_numpy(np.stack([rng.permutation(40)[:8] for _ in range(4)]).astype(np.int32)).cuda()
    places = torch.arange(3, device="cuda").expand(4, 3)
    y = torch.randn(4, 3, device="cuda")
    items[2, 5] = 40
    loss = a.distill_step(users, items, places, y)
    assert torch.isnan(loss).cpu().tolist() == [False, False, True, False]
    assert all(np.isfinite(v).all() for v in a.keras_weights().values())
    with pytest.raises(ValueError):
        a.check_errors()                   # the id is reported, as a training step's
    b.distill_step(users, items[:, :5], places, y)
    with pytest.raises(ValueError):
        b.distill_step(users, items[0], places, y)
    with pytest.raises(ValueError):
        b.distill_step(users[:3], items, places, y)


def test_distillation_refuses_bf16_operands():
    eng = NCFEngine(50, 40, [64, 32, 16, 8], 8, max_batch=64, precision="bf16")
    with pytest.raises(ValueError):
        eng.distill_step(np.zeros(2, np.int32), np.zeros((2, 4), np.int32), torch.zeros(2, 1, dtype=torch.int32,
                         device="cuda"), torch.zeros(2, 1, device="cuda"))
