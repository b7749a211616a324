"""The losses of the framework's classifiers as performance cases: ``linear_cross_entropy`` and ``distillation_loss``.

Every case is a dict of plain values with an ``op``:

  ce        softmax cross entropy of a linear classifier, ``x @ weight`` against labels, the mean over the rows that
            have a label; ``train`` with the gradients of ``x`` and ``weight``, otherwise the rows' losses alone
  distill   divergence of a student's class scores from a teacher's best scores per row; ``train`` with the gradient
            of the scores, otherwise the rows' losses alone

``own`` selects the framework's operators; without it the same values are computed with elementary tensor
operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}
IGNORED = -100
MOST_SCORES = 16384 * 100003            # scores of the largest distillation case
MOST_PRODUCTS = 16384 * 1024 * 65536    # products of the largest classifier


def listed():
    return [
        # the training rows of a small citation graph, seven classes behind a hidden width of 16 (neighbours and self): latency
        dict(name="ce_small_f32", op="ce", rows=140, width=32, classes=7, dtype="f32", order="dv", train=True, scale=1.0, ignored=0.0),
        # the default storage type, many classes, row and class counts that fit no tile
        dict(name="ce_odd_f32", op="ce", rows=2001, width=256, classes=10007, dtype="f32", order="dv", train=True, scale=1.0, ignored=0.03),
        # a mini-batch of 1,024 seeds, hidden width 256 (neighbours and self)
        dict(name="ce_seeds_bf16", op="ce", rows=1024, width=512, classes=32768, dtype="bf16", order="dv", train=True, scale=1.0,
             ignored=0.0),
        # all training rows of the mid-size graph, 172 classes: the long axis is the rows'
        dict(name="ce_rows_bf16", op="ce", rows=90941, width=512, classes=172, dtype="bf16", order="dv", train=True, scale=1.0, ignored=0.0),
        # nothing divides by eight; half precision with a loss scale
        dict(name="ce_ragged_f16", op="ce", rows=5003, width=301, classes=49999, dtype="f16", order="dv", train=True, scale=1024.0,
             ignored=0.1),
        # the largest training step, the weight of a linear layer (one row per class)
        dict(name="ce_large_bf16", op="ce", rows=16384, width=1024, classes=65536, dtype="bf16", order="vd", train=True, scale=1.0,
             ignored=0.05),
        # the rows' losses of an evaluation pass
        dict(name="ce_eval_bf16", op="ce", rows=8192, width=512, classes=131072, dtype="bf16", order="dv", train=False, scale=1.0,
             ignored=0.0),
        # a small student: latency
        dict(name="distill_small_f32", op="distill", rows=64, classes=172, kept=8, dtype="f32", pad=0, train=True, scale=1.0, temperature=2.0,
             empty=0.0),
        # every node of the mid-size graph, 47 classes cut from rows of 48, as the last layer returns them
        dict(name="distill_nodes_bf16", op="distill", rows=169343, classes=47, kept=5, dtype="bf16", pad=1, train=True, scale=1.0,
             temperature=2.0, empty=0.02),
        # rows that start at odd addresses, half precision with a loss scale
        dict(name="distill_ragged_f16", op="distill", rows=30011, classes=4999, kept=20, dtype="f16", pad=0, train=True, scale=1024.0,
             temperature=1.5, empty=0.02),
        # the largest student
        dict(name="distill_large_bf16", op="distill", rows=16384, classes=100003, kept=32, dtype="bf16", pad=5, train=True, scale=1.0,
             temperature=1.0, empty=0.0),
        # the losses of three rows over a long class axis
        dict(name="distill_few_f32", op="distill", rows=3, classes=262144, kept=64, dtype="f32", pad=0, train=False, scale=1.0,
             temperature=4.0, empty=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _near(rng, v):
    """``v``, or the next multiple of 8, or a size beside it."""
    return max(1, rng.choice([v, -(-v // 8) * 8, -(-v // 64) * 64, v + 1]))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    train = rng.random() < 0.75
    scale = 1024.0 if dtype == "f16" else 1.0
    if rng.random() < 0.55:
        while True:
            rows, width, classes = _near(rng, _log(rng, 1, 60000)), _near(rng, _log(rng, 8, 1440)), 1 + _near(rng, _log(rng, 2, 131000))
            if rows * width * classes <= MOST_PRODUCTS // (4 if dtype == "f32" else 1) and rows * classes <= MOST_SCORES:
                break
        return dict(op="ce", rows=rows, width=width, classes=classes, dtype=dtype, order=rng.choice(["dv", "vd"]), train=train, scale=scale,
                    ignored=rng.choice([0.0, 0.0, 0.05, 0.3]))
    while True:
        rows, classes = _near(rng, _log(rng, 1, 170000)), 1 + _near(rng, _log(rng, 2, 262000))
        if rows * classes * ESIZE[dtype] <= MOST_SCORES:
            break
    return dict(op="distill", rows=rows, classes=classes, kept=min(classes, _log(rng, 1, 100)), dtype=dtype, pad=rng.choice([0, 0, 0, 1, 8]),
                train=train, scale=scale, temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), empty=rng.choice([0.0, 0.02, 0.2]))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _labels(case, gen):
    n, dev = case["rows"], "cuda"
    labels = torch.randint(0, case["classes"], (n,), generator=gen, device=dev)
    if case["ignored"]:
        labels[torch.rand(n, generator=gen, device=dev) < case["ignored"]] = IGNORED
        labels[n // 2] = case["classes"] // 2           # one row that counts, whatever was drawn
    return labels


def prepare(case, seed):
    gen, dev, dtype = _generator(seed), "cuda", DTYPES[case["dtype"]]
    n, v = case["rows"], case["classes"]
    s = dict(case=case, grad=torch.tensor(float(case["scale"]), device=dev))
    if case["op"] == "ce":
        d = case["width"]
        # normalised activations and weights of a trained head: scores spread over a few units
        x = torch.randn(n, d, generator=gen, device=dev).to(dtype)
        w = (torch.randn((d, v) if case["order"] == "dv" else (v, d), generator=gen, device=dev) * (2.5 / math.sqrt(d))).to(dtype)
        w = w if case["order"] == "dv" else w.t()
        s.update(x=x.requires_grad_(case["train"]), weight=w.requires_grad_(case["train"]), labels=_labels(case, gen))
        return s
    k = case["kept"]
    z = torch.empty(n, v + case["pad"], dtype=dtype, device=dev)
    for lo in range(0, n, 4096):
        z[lo:lo + 4096] = (2.5 * torch.randn(min(4096, n - lo), v + case["pad"], generator=gen, device=dev)).to(dtype)
    z = z[:, :v]
    # K different classes per row, the best first; the last entries of some rows are missing, some rows have none
    first = torch.randint(0, v, (n, 1), generator=gen, device=dev)
    step = torch.randint(1, max(2, v // k + 1), (n, 1), generator=gen, device=dev)
    step = torch.where(step * k > v, torch.ones_like(step), step)
    ids = (first + step * torch.arange(k, device=dev)) % v
    kept = torch.where(torch.rand(n, generator=gen, device=dev) < 0.1, torch.randint(1, k + 1, (n,), generator=gen, device=dev), k)
    if case["empty"]:
        kept = torch.where(torch.rand(n, generator=gen, device=dev) < case["empty"], 0, kept)
        kept[n // 2] = k
    ids = torch.where(torch.arange(k, device=dev) < kept[:, None], ids, -1).to(torch.int32)
    t = (9.0 + torch.randn(n, 1, generator=gen, device=dev) - 3.0 * torch.rand(n, k, generator=gen, device=dev).cumsum(1) / math.sqrt(k)).to(dtype)
    s.update(logits=z.requires_grad_(case["train"]), teacher=t, ids=ids)
    return s


def _plain_ce(s):
    case = s["case"]
    x, w, y = s["x"].detach().float(), s["weight"].detach().float(), s["labels"]
    valid = y != IGNORED
    at = torch.where(valid, y, 0)[:, None]
    e = x @ w
    top = e.amax(1, keepdim=True)
    label_score = e.gather(1, at) - top
    e.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(valid, (total.log() - label_score)[:, 0], 0.0)
    if not case["train"]:
        return {"loss": loss}
    count = valid.sum()
    g = e.div_(total).scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float32))
    g *= torch.where(valid, s["grad"] / count, 0.0)[:, None]
    dtype = s["x"].dtype
    return {"loss": loss.sum() / count, "dx": (g @ w.t()).to(dtype), "dweight": (x.t() @ g).to(dtype)}


def _plain_distill(s):
    case, T = s["case"], s["case"]["temperature"]
    z, ids = s["logits"].detach().float() / T, s["ids"].long()
    there = ids >= 0
    t = torch.where(there, s["teacher"].float() / T, -math.inf)
    any_ = there.any(1)
    top = torch.where(any_, t.amax(1), 0.0)[:, None]
    p = torch.exp(t - top)
    p_total = torch.where(any_, p.sum(1), 1.0)[:, None]
    log_p = t - top - p_total.log()
    p = p / p_total
    at = torch.where(there, ids, 0)
    z_top = z.amax(1, keepdim=True)
    e = z.sub_(z_top)
    picked = e.gather(1, at)
    e.exp_()
    total = e.sum(1, keepdim=True)
    rows = T * T * torch.where(there & (p > 0), p * (log_p - picked + total.log()), 0.0).sum(1)
    if not case["train"]:
        return {"loss": rows}
    count = any_.sum()
    e.div_(total).scatter_add_(1, at, torch.where(there, -p, 0.0))
    e *= torch.where(any_, s["grad"] * T / count, 0.0)[:, None]
    return {"loss": rows.sum() / count, "dlogits": e.to(s["logits"].dtype)}


def _own_ce(s):
    from graph_rws_b200.layers import linear_cross_entropy
    if not s["case"]["train"]:
        return {"loss": linear_cross_entropy(s["x"], s["weight"], s["labels"], ignore_index=IGNORED, reduction="none")}
    loss = linear_cross_entropy(s["x"], s["weight"], s["labels"], ignore_index=IGNORED)
    dx, dw = torch.autograd.grad(loss, (s["x"], s["weight"]), s["grad"])
    return {"loss": loss.detach(), "dx": dx, "dweight": dw}


def _own_distill(s):
    from graph_rws_b200.layers import distillation_loss
    T = s["case"]["temperature"]
    if not s["case"]["train"]:
        return {"loss": distillation_loss(s["logits"], s["teacher"], s["ids"], temperature=T, reduction="none")}
    loss = distillation_loss(s["logits"], s["teacher"], s["ids"], temperature=T)
    dz, = torch.autograd.grad(loss, (s["logits"],), s["grad"])
    return {"loss": loss.detach(), "dlogits": dz}


def run(state):
    if state["case"]["op"] == "ce":
        return _own_ce(state) if own else _plain_ce(state)
    return _own_distill(state) if own else _plain_distill(state)


def work(case):
    n, v, e = case["rows"], case["classes"], ESIZE[case["dtype"]]
    if case["op"] == "ce":
        d = case["width"]
        once = n * d * e + d * v * e
        if not case["train"]:
            return {"bytes": once + 8 * n + 4 * n, "flops": 2 * n * d * v}
        return {"bytes": 2 * once + 8 * n, "flops": 6 * n * d * v}
    teacher = n * case["kept"] * (e + 4)
    if not case["train"]:
        return {"bytes": n * v * e + teacher + 4 * n, "flops": 3 * n * v}
    return {"bytes": 2 * n * v * e + teacher, "flops": 6 * n * v}


def exact(case, seed):
    s = prepare(case, seed)
    n, step = case["rows"], max(1, (1 << 29) // case["classes"])
    if case["op"] == "ce":
        w = s["weight"].detach().double()
        y, counted = s["labels"], float((s["labels"] >= 0).sum())
        losses, dx, dw = [], [], torch.zeros_like(w) if case["train"] else None
        for lo in range(0, n, step):
            x, lab = s["x"][lo:lo + step].detach().double(), y[lo:lo + step]
            log_q = torch.log_softmax(x @ w, 1)
            has = (lab >= 0).double()
            onehot = lab.clamp(min=0)
            losses.append(-has * log_q[torch.arange(lab.numel(), device=lab.device), onehot])
            if case["train"]:
                g = log_q.exp_()
                g[torch.arange(lab.numel(), device=lab.device), onehot] -= 1.0
                g *= (has * (case["scale"] / counted))[:, None]
                dx.append(g @ w.t())
                dw += x.t() @ g
        losses = torch.cat(losses)
        return {"loss": losses.sum() / counted, "dx": torch.cat(dx), "dweight": dw} if case["train"] else {"loss": losses}
    T, ids = case["temperature"], s["ids"].long()
    held = (ids >= 0).sum(1)
    counted = float((held > 0).sum())
    losses, grads = [], []
    for lo in range(0, n, step):
        log_q = torch.log_softmax(s["logits"][lo:lo + step].detach().double() / T, 1)
        i, t = ids[lo:lo + step], s["teacher"][lo:lo + step].double() / T
        has = held[lo:lo + step] > 0
        log_p = torch.log_softmax(t.masked_fill((i < 0) & has[:, None], -math.inf), 1)
        p = torch.where(i >= 0, log_p.exp(), 0.0)
        terms = p * (log_p.masked_fill(i < 0, 0.0) - log_q.gather(1, i.clamp(min=0)))
        losses.append(T * T * terms.sum(1))
        if case["train"]:
            q = log_q.exp_()
            at = torch.arange(q.shape[0], device=q.device)[:, None].expand_as(i)
            q.index_put_((at, i.clamp(min=0)), -p, accumulate=True)
            grads.append((q * (has.double() * (T * case["scale"] / counted))[:, None]).to(torch.float32 if q.numel() > 1 << 27 else q.dtype))
    losses = torch.cat(losses)
    return {"loss": losses.sum() / counted, "dlogits": torch.cat(grads)} if case["train"] else {"loss": losses}
