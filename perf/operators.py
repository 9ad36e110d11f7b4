"""Cases of the catalogue operators (``movierec.catalogue``): the block-scaled 8-bit product that
scores users against a catalogue and the quantiser that feeds it, drawing items from the logits,
and distillation from a teacher's best items.

``own`` chooses what ``run`` computes: False, the operators' plain forms in torch; True, the calls
a user makes of the library.  ``exact`` is the definition of each operator in 64 bits.

Sizes: catalogues of 1,682 (ml-100k), 3,952 (ml-1m), 27,278 (ml-20m) and 1,000,000 items; factor
widths 8 to 128 of the GMF models; 100 candidates per user is the evaluation protocol (one positive
and 99 negatives); lists of 10 and 32 are the scorer's default and its largest.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 128          # values of a row that share a scale
E4M3_MAX = 448.0     # largest finite e4m3 value
MIN_SCALE = 2.0 ** -126

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def _catalogue():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "movierecommender-tf-trt_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from movierec import catalogue
    return catalogue


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one request: one user's vector against the ml-20m catalogue (GMF width 64)
        dict(name="product_one_user", op="product", m=1, n=27278, k=64, wide=False, bias=True, out="fp32"),
        # a ragged batch over the ml-100k catalogue, a width that ends inside a block
        dict(name="product_ragged", op="product", m=333, n=1682, k=200, wide=False, bias=True, out="fp16"),
        # bulk scoring: 8,192 users against the ml-20m catalogue
        dict(name="product_users", op="product", m=8192, n=27278, k=64, wide=False, bias=True, out="fp32"),
        # a wide dense layer with one scale per 128 x 128 tile of its weights
        dict(name="product_dense", op="product", m=8192, n=4096, k=4096, wide=True, bias=False, out="bf16"),
        # user vectors of a small batch, an odd width, held in bf16
        dict(name="quantize_users", op="quantize", r=943, k=100, wide=False, dtype="bf16"),
        # the item table of a 1,000,000-item catalogue, width 128
        dict(name="quantize_items", op="quantize", r=1000000, k=128, wide=False, dtype="fp32"),
        # one request: one draw for one user over the ml-20m catalogue, all filters on
        dict(name="sample_one_user", op="sample", r=1, n=27278, draws=1, dtype="fp32", temperature=0.8, top_k=50,
             top_p=0.9, min_p=0.0, rows=False, seen=0.0),
        # a batch of users, ten draws each, their seen items masked out
        dict(name="sample_users", op="sample", r=2048, n=27278, draws=10, dtype="fp32", temperature=1.0, top_k=1000,
             top_p=0.95, min_p=0.01, rows=False, seen=0.005),
        # a large catalogue in bf16, every user with settings of their own, no bound on the list
        dict(name="sample_large", op="sample", r=16, n=1000000, draws=4, dtype="bf16", temperature=1.3, top_k=0,
             top_p=0.8, min_p=0.0, rows=True, seen=0.0),
        # the evaluation protocol's 100 candidates per user: loss and gradient in two calls
        dict(name="distill_candidates", op="distill", r=512, v=100, k=10, dtype="fp32", temperature=2.0, lse=False,
             direction="two", item="int64"),
        # a training step over the ml-20m catalogue, bf16 logits, the scorer's largest list
        dict(name="distill_users", op="distill", r=2048, v=27278, k=32, dtype="bf16", temperature=1.0, lse=False,
             direction="both", item="int32"),
        # a large catalogue, the teacher's mass outside its list kept as one more class
        dict(name="distill_large", op="distill", r=64, v=1000000, k=32, dtype="fp32", temperature=1.5, lse=True,
             direction="both", item="int32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["product", "product", "quantize", "sample", "sample", "distill", "distill"])
    if op == "product":
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 100, 1000000), _log(rng, 8, 4096)
            if m * n * k <= 8192 * 4096 * 4096 and m * n <= 8192 * 27278 and n * k <= 1000000 * 128:
                break
        return dict(op=op, m=m, n=n, k=k, wide=rng.random() < 0.4, bias=rng.random() < 0.5,
                    out=rng.choice(["fp32", "bf16", "fp16"]))
    if op == "quantize":
        k = _log(rng, 8, 4096)
        r = _log(rng, 1, max(2, min(1000000, 1000000 * 128 // k)))
        return dict(op=op, r=r, k=k, wide=rng.random() < 0.4, dtype=rng.choice(["fp32", "bf16", "fp16"]))
    if op == "sample":
        n = _log(rng, 1, 1000000)
        r = _log(rng, 1, max(2, min(8192, 2048 * 27278 // (2 * n))))
        return dict(op=op, r=r, n=n, draws=rng.choice([1, 1, 2, 5, 10, 33]),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), temperature=round(rng.uniform(0.3, 2.0), 3),
                    top_k=rng.choice([0, 1, 10, 50, _log(rng, 1, 5000)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]),
                    min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), rows=rng.random() < 0.4,
                    seen=rng.choice([0.0, 0.01, 0.3]))
    v = _log(rng, 2, 1000000)
    r = _log(rng, 1, max(2, min(8192, 2048 * 27278 // (2 * v))))
    return dict(op=op, r=r, v=v, k=min(v, rng.choice([1, 5, 10, 32, 32, 100, 257])),
                dtype=rng.choice(["fp32", "bf16", "fp16"]), temperature=round(rng.uniform(0.5, 4.0), 3),
                lse=rng.random() < 0.4, direction=rng.choice(["loss", "two", "both"]),
                item=rng.choice(["int32", "int64"]))


# ------------------------------------------------------------------------------------- inputs

def _blocks(k):
    return (k + BLOCK - 1) // BLOCK


def _held_in_8_bits(x, wide):
    """x (rows x k, fp32) as e4m3 values and scales, rows 16-byte aligned."""
    r, k = x.shape
    kb = _blocks(k)
    pad = torch.zeros(r, kb * BLOCK, device=x.device)
    pad[:, :k] = x
    a = pad.view(r, kb, BLOCK).abs().amax(2)
    if wide:
        rb = (r + BLOCK - 1) // BLOCK
        t = torch.zeros(rb * BLOCK, kb, device=x.device)
        t[:r] = a
        a = t.view(rb, BLOCK, kb).amax(1)
    scale = (a / torch.full_like(a, E4M3_MAX)).clamp_min(MIN_SCALE)
    full = (scale.repeat_interleave(BLOCK, 0)[:r] if wide else scale).repeat_interleave(BLOCK, 1)[:, :k]
    store = torch.zeros(r, (k + 15) // 16 * 16, device=x.device, dtype=torch.float8_e4m3fn)
    store[:, :k] = (x / full).to(torch.float8_e4m3fn)
    return store[:, :k], scale


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    s = dict(case)
    if own:
        s["lib"] = _catalogue()
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        # rows of different length, as trained factors have
        a = normal(m, k) * (0.5 + uniform(m, 1))
        b = normal(n, k) * (0.2 + uniform(n, 1)) / math.sqrt(k)
        s["a"], s["a_scale"] = _held_in_8_bits(a, False)
        s["b"], s["b_scale"] = _held_in_8_bits(b, case["wide"])
        s["bias"] = normal(n) * 0.1 if case["bias"] else None
    elif case["op"] == "quantize":
        x = normal(case["r"], case["k"]) * torch.exp(normal(case["r"], 1))
        s["x"] = x.to(DTYPES[case["dtype"]])
    elif case["op"] == "sample":
        r, n = case["r"], case["n"]
        # popularity over the catalogue plus the user's own taste
        x = normal(1, n) * 1.5 + normal(r, n) * 1.2
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["u"] = uniform(r, case["draws"])
        s["mask"] = uniform(r, n) >= case["seen"] if case["seen"] > 0 else None
        for name, spread in (("temperature", 0.5), ("top_k", 0.9), ("top_p", 0.2), ("min_p", 0.5)):
            v = case[name]
            if case["rows"]:
                if name == "top_k":
                    v = (torch.full((r,), float(v), device=dev) * (1 - spread * uniform(r))).ceil().to(torch.int32)
                else:
                    v = torch.full((r,), float(v), device=dev) * (1 - spread * uniform(r))
            s[name] = v
    else:
        r, v, k = case["r"], case["v"], case["k"]
        x = normal(1, v) * 1.5 + normal(r, v) * 1.2
        # the teacher's best items: mostly the student's own better ones, in the teacher's order
        items = torch.empty(r, k, device=dev, dtype=torch.int64)
        t = torch.empty(r, k, device=dev)
        lse = torch.empty(r, device=dev)
        step = max(1, (1 << 26) // v)
        for i in range(0, r, step):
            z = x[i:i + step] + normal(min(step, r - i), v) * 0.8
            t[i:i + step], items[i:i + step] = torch.topk(z, k, 1)
            lse[i:i + step] = torch.logsumexp(z / case["temperature"], 1)
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["teacher_items"] = items.to(getattr(torch, case["item"]))
        s["teacher_logits"] = t
        s["teacher_lse"] = lse if case["lse"] else None
        # the step's mean over its rows, with a weight for each user; in fp16 times a loss scale
        s["grad_loss"] = (0.5 + uniform(r)) * ((4096.0 if case["dtype"] == "fp16" else 1.0) / r)
    return s


# ------------------------------------------------------------------------------------- one pass

def run(state):
    return {"product": _product, "quantize": _quantize, "sample": _sample, "distill": _distill}[state["op"]](state)


def _product(s):
    if own:
        return s["lib"].matmul_blocks(s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"],
                                      out_dtype=DTYPES[s["out"]])
    k = s["k"]
    a = s["a"].float() * s["a_scale"].repeat_interleave(BLOCK, 1)[:, :k]
    w = s["b_scale"].repeat_interleave(BLOCK, 1)[:, :k]
    if s["wide"]:
        w = w.repeat_interleave(BLOCK, 0)[:s["n"]]
    b = s["b"].float() * w
    y = a @ b.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(DTYPES[s["out"]])


def _quantize(s):
    if own:
        q, scale = s["lib"].quantize_blocks(s["x"], tile=s["wide"])
        return q.float(), scale
    x = s["x"].float()
    r, k = x.shape
    kb = _blocks(k)
    pad = torch.nn.functional.pad(x.abs(), (0, kb * BLOCK - k))
    a = pad.view(r, kb, BLOCK).amax(2)
    if s["wide"]:
        rb = (r + BLOCK - 1) // BLOCK
        a = torch.nn.functional.pad(a, (0, 0, 0, rb * BLOCK - r)).view(rb, BLOCK, kb).amax(1)
    # (a tensor as the divisor: a quotient, not a product with the reciprocal)
    scale = (a / torch.full_like(a, E4M3_MAX)).clamp_min(MIN_SCALE)
    w = scale.repeat_interleave(BLOCK, 1)[:, :k]
    if s["wide"]:
        w = w.repeat_interleave(BLOCK, 0)[:r]
    return (x / w).to(torch.float8_e4m3fn).float(), scale


def _sample(s):
    if own:
        return s["lib"].sample_items(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                     top_p=s["top_p"], min_p=s["min_p"], mask=s["mask"])
    x = s["logits"].double()
    dev, (r, n) = x.device, x.shape

    def setting(v):
        v = v.double() if torch.is_tensor(v) else torch.full((r,), float(v), device=dev, dtype=torch.float64)
        return v.view(r, 1)

    temperature, top_k, top_p, min_p = (setting(s[c]) for c in ("temperature", "top_k", "top_p", "min_p"))
    if s["mask"] is not None:
        x = x.masked_fill(~s["mask"], -math.inf)
    value, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((value - value[:, :1]) / temperature)
    rank = torch.arange(n, device=dev).view(1, n)
    w = torch.where((value > -math.inf) & ((top_k <= 0) | (rank < top_k)), w, torch.zeros_like(w))
    mass = torch.cumsum(w, 1)
    before = torch.nn.functional.pad(mass[:, :-1], (1, 0))
    keep = (top_p >= 1) | (before < top_p * mass[:, -1:]) | (rank == 0)
    w = torch.where(keep & (w >= min_p), w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, order, w)   # back in the catalogue's order
    mass = torch.cumsum(w, 1)
    total = mass[:, -1:]
    item = torch.searchsorted(mass, s["u"].double() * total, right=True).clamp_max(n - 1)
    prob = torch.where(total > 0, w.gather(1, item) / total, torch.zeros_like(total))
    item = torch.where(total > 0, item, torch.full_like(item, -1))
    return item.to(torch.int32), prob.float()


def _distill(s):
    x, items, t, lse = s["logits"], s["teacher_items"], s["teacher_logits"], s["teacher_lse"]
    temperature = s["temperature"]
    if own:
        lib = s["lib"]
        args = dict(temperature=temperature, teacher_lse=lse)
        if s["direction"] == "both":
            return lib.distill_loss_grad(x, items, t, s["grad_loss"], **args)
        loss, saved = lib.distill_loss(x, items, t, **args)
        if s["direction"] == "loss":
            return (loss,)
        return loss, lib.distill_grad(x, items, t, saved, s["grad_loss"], **args)
    items = items.long()
    z = x.float() / temperature
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    # what depends on the row's sums alone in 64 bits: the loss is a small difference of large logs
    mass = e.sum(1, keepdim=True, dtype=torch.float64)
    log_p = z.gather(1, items).double() - top.double() - torch.log(mass)
    t = t.double() / temperature
    if lse is None:
        log_q = t - torch.logsumexp(t, 1, keepdim=True)
    else:
        log_q = t - lse.double().view(-1, 1)
    q = torch.exp(log_q)
    loss = (q * (log_q - log_p)).sum(1)
    inside, outside = q.sum(1, keepdim=True), q.sum(1, keepdim=True)
    if lse is not None:
        q0 = (1 - inside).clamp_min(0)
        in_list = e.gather(1, items).sum(1, keepdim=True, dtype=torch.float64)
        e0 = e.scatter(1, items, 0.0).sum(1, keepdim=True, dtype=torch.float64)
        p0 = e0 / mass
        on = (q0 > 0) & (p0 > 0)
        q0 = torch.where(on, q0, torch.zeros_like(q0))
        loss = loss + torch.where(on, q0 * (torch.log1p(-inside) + torch.log1p(in_list / e0)), q0).view(-1)
        inside = inside + q0
        outside = inside - torch.where(on, q0 / p0, q0)
    loss = loss.float()
    if s["direction"] == "loss":
        return (loss,)
    p = e / mass.float()
    grad = p * outside.float()
    grad.scatter_(1, items, p.gather(1, items) * inside.float())
    grad.scatter_add_(1, items, -q.float())
    return loss, (grad * (s["grad_loss"] / temperature).view(-1, 1)).to(x.dtype)


# ------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"product": _product_64, "quantize": _quantize_64, "sample": _sample_64,
            "distill": _distill_64}[case["op"]](s)


def _product_64(s):
    """y = sum over the blocks of (a_scale b_scale) times the block's product, plus the bias."""
    y = torch.zeros(s["m"], s["n"], dtype=torch.float64, device=s["a"].device)
    a, b = s["a"].to(torch.float32).double(), s["b"].to(torch.float32).double()
    for j in range(_blocks(s["k"])):
        cut = slice(j * BLOCK, min(s["k"], (j + 1) * BLOCK))
        sb = s["b_scale"][:, j].double()
        if s["wide"]:
            sb = sb[torch.arange(s["n"], device=sb.device) // BLOCK]
        y += (a[:, cut] * s["a_scale"][:, j:j + 1].double()) @ (b[:, cut] * sb.view(-1, 1)).t().contiguous()
    if s["bias"] is not None:
        y += s["bias"].double()
    return y


def _quantize_64(s):
    """scale = max(largest magnitude / 448, 2^-126) held in 32 bits; value = the quotient, held in 32
    bits, to the nearest e4m3 number (3 bits after the point from 2^-6 up, steps of 2^-9 below)."""
    x = s["x"].double().cpu().numpy()
    r, k = x.shape
    kb = _blocks(k)
    top = np.zeros((r, kb))
    for j in range(kb):
        top[:, j] = np.abs(x[:, j * BLOCK:(j + 1) * BLOCK]).max(1)
    if s["wide"]:
        top = np.stack([top[i:i + BLOCK].max(0) for i in range(0, r, BLOCK)])
    scale = np.maximum((top / 448.0).astype(np.float32), np.float32(2.0 ** -126))
    row = np.arange(r) // BLOCK if s["wide"] else np.arange(r)
    out = np.empty((r, k), np.float32)
    for j in range(kb):
        cut = slice(j * BLOCK, min(k, (j + 1) * BLOCK))
        v = (x[:, cut] / scale[row, j].astype(np.float64)[:, None]).astype(np.float32).astype(np.float64)
        _, e = np.frexp(v)
        step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
        out[:, cut] = np.rint(v / step) * step
    return out, scale


def _sample_64(s):
    """Row by row: the best top_k items, of them the shortest leading list that holds top_p of the
    mass, of it what weighs at least min_p of the best; then the first item, in the catalogue's
    order, whose running sum passes u times the total."""
    x = s["logits"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()
    mask = None if s["mask"] is None else s["mask"].cpu().numpy()
    r, n = x.shape

    def setting(v):
        return v.double().cpu().numpy() if torch.is_tensor(v) else np.full(r, float(v))

    temperature, top_k, top_p, min_p = (setting(s[c]) for c in ("temperature", "top_k", "top_p", "min_p"))
    items = np.full(u.shape, -1, np.int32)
    probs = np.zeros(u.shape)
    for i in range(r):
        ids = np.flatnonzero(x[i] > -np.inf) if mask is None else np.flatnonzero(mask[i] & (x[i] > -np.inf))
        if ids.size == 0:
            continue
        v = x[i, ids]
        k = ids.size if top_k[i] <= 0 else min(ids.size, int(top_k[i]))
        if k < ids.size:
            # all above the k-th largest value, then the lowest ids among its equals
            bound = np.partition(v, ids.size - k)[ids.size - k]
            above = v > bound
            equal = np.flatnonzero(v == bound)[:k - int(above.sum())]
            above[equal] = True
            ids, v = ids[above], v[above]
        w = np.exp((v - v.max()) / temperature[i])
        if top_p[i] < 1:
            order = np.lexsort((ids, -v))
            c = np.cumsum(w[order])
            m = 1 + int(np.searchsorted(c, top_p[i] * c[-1], side="left"))
            chosen = np.sort(order[:m])
            ids, w = ids[chosen], w[chosen]
        chosen = w >= min_p[i]
        ids, w = ids[chosen], w[chosen]
        c = np.cumsum(w)
        at = np.minimum(np.searchsorted(c, u[i] * c[-1], side="right"), ids.size - 1)
        items[i] = ids[at]
        probs[i] = w[at] / c[-1]
    return items, probs


def _distill_64(s):
    """The loss as a function of the logits, and its derivative by automatic differentiation."""
    z = s["logits"].double().requires_grad_(True)
    items, t = s["teacher_items"].long(), s["teacher_logits"].double() / s["temperature"]
    log_p = torch.log_softmax(z / s["temperature"], 1)
    if s["teacher_lse"] is None:
        q = torch.softmax(t, 1)
        loss = (q * (torch.log_softmax(t, 1) - log_p.gather(1, items))).sum(1)
    else:
        log_q = t - s["teacher_lse"].double()[:, None]
        q = torch.exp(log_q)
        loss = (q * (log_q - log_p.gather(1, items))).sum(1)
        rest = (1 - q.sum(1)).clamp_min(0)
        listed_ = torch.zeros_like(z, dtype=torch.bool).scatter_(1, items, True)
        log_rest = torch.logsumexp(log_p.masked_fill(listed_, -math.inf), 1)
        # no item outside the list: the mass left over is rounding alone
        on = (rest > 0) & torch.isfinite(log_rest)
        log_rest = torch.where(on, log_rest, torch.zeros_like(log_rest))
        loss = loss + torch.where(on, rest * (torch.log(rest.clamp_min(1e-300)) - log_rest), 0 * rest)
    if s["direction"] == "loss":
        return (loss.detach(),)
    grad, = torch.autograd.grad((loss * s["grad_loss"].double()).sum(), z)
    return loss.detach(), grad


# ------------------------------------------------------------------------------------- work

def work(case):
    """Bytes and operations of one pass: every input read once, every output written once."""
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        kb = _blocks(k)
        nb = (n + BLOCK - 1) // BLOCK if case["wide"] else n
        byte = (m + n) * k + 4 * kb * (m + nb) + (4 * n if case["bias"] else 0) + m * n * SIZE[case["out"]]
        return {"bytes": byte, "flops": 2 * m * n * k}
    if case["op"] == "quantize":
        r, k = case["r"], case["k"]
        rb = (r + BLOCK - 1) // BLOCK if case["wide"] else r
        return {"bytes": r * k * (SIZE[case["dtype"]] + 1) + 4 * rb * _blocks(k), "flops": 3 * r * k}
    if case["op"] == "sample":
        r, n = case["r"], case["n"]
        byte = r * n * (SIZE[case["dtype"]] + (1 if case["seen"] > 0 else 0)) + r * case["draws"] * 12
        return {"bytes": byte, "flops": 8 * r * n}
    r, v, k = case["r"], case["v"], case["k"]
    index = 8 if case["item"] == "int64" else 4
    writes = 0 if case["direction"] == "loss" else r * v * SIZE[case["dtype"]]
    byte = r * v * SIZE[case["dtype"]] + writes + r * k * (4 + index) + 8 * r
    return {"bytes": byte, "flops": (4 if case["direction"] == "loss" else 7) * r * v}
