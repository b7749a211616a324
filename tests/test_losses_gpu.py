"""linear_cross_entropy and distillation_loss (csrc/linear_ce.cu, csrc/distill.cu) against the operators' definition in
64 bits.  Bounds are worst cases of the arithmetic, element by element: u is half a step of a type, fp32 sums of k terms
are off by at most k u of the sum of the terms' sizes, an exponential by 2^-21 of itself (exp2's 2^-22 and its argument's
rounding) plus the error of its argument."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}        # half the smallest step
FLUSHED = 2.0 ** -126       # an exponential below fp32's smallest normal number is 0
U32 = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def within(got, want, bound, what):
    # half a step past the type's largest number rounding gives infinity: 65,520 and above in fp16
    most = torch.finfo(got.dtype).max * (1 + U[got.dtype])
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= bound) & ~((want.abs() + bound >= most) & torch.isinf(got) & (got.sign() == want.sign()))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / bound).max()):.3g} times the bound, "
                           f"first at {bad.nonzero()[0].tolist()}: {float(got[bad][0])!r}, expected {float(want[bad][0])!r} +- {float(bound[bad][0]):.3g}")


# ---------------------------------------------------------------------------------------------
# linear cross entropy
# ---------------------------------------------------------------------------------------------
def ce_inputs(n, d, V, dtype, class_major=False, ignored=0.0, seed=0, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * n + d + V)
    x = torch.randn(n, d, generator=g, device="cuda").to(dtype)
    w = (torch.randn(d, V, generator=g, device="cuda") * (spread / math.sqrt(d))).to(dtype)
    w = w.t().contiguous().t() if class_major else w
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    if ignored:
        y[torch.rand(n, generator=g, device="cuda") < ignored] = -100
        y[0] = V - 1
    return x, w, y


def ce_reference(x, w, y, r, ignore=-100):
    """Rows' losses, dx and dw for row factors r, in 64 bits, and the error bounds of each."""
    x64, w64 = x.double(), w.double()
    s = x64 @ w64
    lse = torch.logsumexp(s, 1, keepdim=True)
    keep = y != ignore
    at = torch.where(keep, y, 0).long()[:, None]
    rows = torch.where(keep, (lse - s.gather(1, at))[:, 0], 0.0)
    r = torch.where(keep, r.double(), 0.0)[:, None]
    q = torch.exp(s - lse)
    e = torch.zeros_like(q).scatter_(1, at, 1.0)
    G = r * (q - e)
    d, V = w.shape
    n = x.shape[0]
    ds = (d + 8) * U32 * (x64.abs() @ w64.abs())                    # a score's error
    dlse = ds.amax(1, keepdim=True) + (V + 16) * U32 + 2.0 ** -21   # the log of its row's sum
    rows_bound = ds.gather(1, at)[:, 0] + dlse[:, 0] + 8 * U32 * (rows.abs() + s.abs().amax(1))
    # G: q relative to its argument's error; the subtraction of the label; its storage
    u_g = 4 * U32 if x.dtype == torch.float32 else U[x.dtype]
    dG = r.abs() * (q * (ds + dlse + 2.0 ** -21 + 8 * U32 * (s - lse).abs()) * 1.01 + 4 * U32 * (q + e) + FLUSHED)
    dG = dG + u_g * (G.abs() + dG) + r.abs() * TINY[x.dtype]
    dx, dw = G @ w64.t(), x64.t() @ G
    gx, gw = G.abs() @ w64.abs().t(), x64.abs().t() @ G.abs()
    dx_bound = dG @ w64.abs().t() + (V + 64) * U32 * gx
    dw_bound = x64.abs().t() @ dG + (n + 64) * U32 * gw
    out = lambda v, b: b + U[x.dtype] * (v.abs() + b) + TINY[x.dtype]    # noqa: E731  rounded once more at the end
    return rows, rows_bound, dx, out(dx, dx_bound), dw, out(dw, dw_bound)


def run_ce(x, w, y, reduction, grad=None, ignore=-100):
    from graph_rws_b200.layers import linear_cross_entropy
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, y, ignore_index=ignore, reduction=reduction)
    assert loss.dtype == torch.float32
    dx, dw = torch.autograd.grad(loss, (x, w), grad if grad is not None else torch.ones_like(loss))
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dx.shape == x.shape and dw.shape == w.shape
    return loss.detach(), dx, dw


def check_ce(x, w, y, reduction="mean", grad=None, ignore=-100):
    n = x.shape[0]
    counted = int((y != ignore).sum())
    loss, dx, dw = run_ce(x, w, y, reduction, grad, ignore)
    g = torch.ones((), device="cuda") if grad is None else grad
    r = torch.broadcast_to(g / counted if reduction == "mean" else g, (n,))
    rows, rb, dx64, dxb, dw64, dwb = ce_reference(x, w, y, r, ignore)
    if reduction == "none":
        within(loss, rows, rb, "loss")
    else:
        total, bound = rows.sum(), rb.sum() + (n + 64) * U32 * rows.abs().sum()
        within(loss, total / counted if reduction == "mean" else total, bound / counted if reduction == "mean" else bound, "loss")
    scale = 1 + 4 * U32                                              # the factor itself is rounded
    within(dx, dx64, dxb * scale + 4 * U32 * dx64.abs(), "dx")
    within(dw, dw64, dwb * scale + 4 * U32 * dw64.abs(), "dweight")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("class_major", [False, True])
@pytest.mark.parametrize("n,d,V", [(1, 1, 1), (1, 8, 2), (3, 5, 7), (64, 64, 64), (140, 32, 7), (65, 129, 1003), (200, 301, 517), (1000, 24, 47),
                                   (2, 72, 20011), (129, 256, 264), (300, 520, 2056)])
def test_cross_entropy_matches_the_definition(n, d, V, dtype, class_major):
    check_ce(*ce_inputs(n, d, V, dtype, class_major))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,d,V", [(97, 40, 171), (513, 136, 1030)])
def test_cross_entropy_reductions_and_ignored_rows(n, d, V, dtype, reduction):
    x, w, y = ce_inputs(n, d, V, dtype, ignored=0.3)
    g = torch.rand(n, device="cuda") * 3 - 1 if reduction == "none" else torch.tensor(0.37, device="cuda")
    check_ce(x, w, y, reduction, g)
    check_ce(x, w, y.int(), reduction, g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("class_major", [False, True])
@pytest.mark.parametrize("V", [16376, 16384, 16391])
def test_cross_entropy_rows_that_are_no_whole_lines(V, dtype, class_major):
    """Rows of 208 bytes (416 in fp32) within wider ones of NaN, on both sides of the number of classes from which they are copied."""
    x, w, y = ce_inputs(261, 104, V, dtype, class_major)
    wide = torch.full((261, 120), float("nan"), dtype=dtype, device="cuda")
    wide[:, 8:112] = x
    check_ce(wide[:, 8:112], w, y)


def test_cross_entropy_against_differences():
    """The gradient of an fp32 loss against central differences in 64 bits along random directions."""
    x, w, y = ce_inputs(33, 20, 50, torch.float32, ignored=0.2)
    _, dx, dw = run_ce(x, w, y, "mean")
    f = lambda a, b: torch.nn.functional.cross_entropy(a @ b, y)      # noqa: E731
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        u = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64)
        v = torch.randn(w.shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        slope = (f(x.double() + h * u, w.double() + h * v) - f(x.double() - h * u, w.double() - h * v)) / (2 * h)
        got = (dx.double() * u).sum() + (dw.double() * v).sum()
        assert abs(float(slope - got)) <= 1e-5 * float((dx.double() * u).abs().sum() + (dw.double() * v).abs().sum())


@pytest.mark.parametrize("dtype,class_major", [(torch.float32, False), (torch.float16, True), (torch.bfloat16, False)])
def test_cross_entropy_in_pieces_of_the_classes(dtype, class_major):
    """So many rows that the workspace of the backward pass holds a part of the classes at a time."""
    check_ce(*ce_inputs(70001, 24, 4501, dtype, class_major, ignored=0.2))


@pytest.mark.parametrize("d", [40, 301])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_cross_entropy_narrow_weights_in_pieces(d, dtype):
    """Gradients of [d, classes] weights whose few rows fill no tile, from several pieces of the classes."""
    check_ce(*ce_inputs(9001, d, 33001, dtype, ignored=0.1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,V", [(700, 96, 11003), (700, 97, 11008), (400, 161, 16391), (3001, 301, 9001)])
def test_cross_entropy_narrow_weights(n, d, V, dtype):
    """The same from all classes at once, with odd and even rows, columns behind the last whole 32 and a cut of the weight."""
    x, w, y = ce_inputs(n, d, V, dtype, ignored=0.1)
    check_ce(x, w, y)
    wide = torch.full((d, V + 9), float("nan"), dtype=dtype, device="cuda")
    wide[:, 3:V + 3] = w
    check_ce(x, wide[:, 3:V + 3], y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_strides(dtype):
    """Operands cut from wider ones, at odd offsets, and orders that need a copy."""
    x, w, y = ce_inputs(70, 48, 90, dtype)
    wide = torch.zeros(70, 61, dtype=dtype, device="cuda")
    wide[:, 5:53] = x
    want = run_ce(x, w, y, "mean")
    tall = torch.zeros(48, 101, dtype=dtype, device="cuda")
    tall[:, 3:93] = w
    for a, b in ((wide[:, 5:53], w), (x, tall[:, 3:93]), (x.t().contiguous().t(), w), (x, tall[:, 3:93].t().contiguous().t()),
                 (torch.stack([x, x], 2)[:, :, 0], torch.stack([w, w], 2)[:, :, 1])):
        got = run_ce(a, b, y, "mean")
        check_ce(a, b, y)
        within(got[0], want[0], 1e-5, "loss")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,V", [(40, 16, 30), (300, 128, 1000)])
def test_cross_entropy_rows_without_labels(n, d, V, dtype):
    x, w, y = ce_inputs(n, d, V, dtype)
    none = torch.full_like(y, -100)
    loss, dx, dw = run_ce(x, w, none, "mean")
    assert torch.isnan(loss) and not dx.any() and not dw.any()
    loss, dx, dw = run_ce(x, w, none, "sum")
    assert loss == 0 and not dx.any() and not dw.any()
    # an ignored label that is a class number, and one past the classes
    y2 = y.clone()
    y2[3] = V // 2
    check_ce(x, w, y2, ignore=V // 2)
    y2[5] = V
    loss, dx, dw = run_ce(x, w, y2, "none")
    assert torch.isnan(loss[5]) and torch.isfinite(loss[torch.arange(n, device="cuda") != 5]).all()
    assert torch.isnan(dx[5]).all() and torch.isnan(dw).all()
    y2[5] = -1
    assert torch.isnan(run_ce(x, w, y2, "mean")[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_empty_and_partial_gradients(dtype):
    from graph_rws_b200.layers import linear_cross_entropy
    x, w, y = ce_inputs(0, 16, 24, dtype)
    loss, dx, dw = run_ce(x, w, y, "sum")
    assert loss == 0 and dx.shape == (0, 16) and not dw.any()
    assert torch.isnan(run_ce(x, w, y, "mean")[0]) and run_ce(x, w, y, "none")[0].shape == (0,)
    x, w, y = ce_inputs(80, 40, 100, dtype)
    _, dx, dw = run_ce(x, w, y, "mean")
    for only in (0, 1):
        a, b = x.detach().requires_grad_(only == 0), w.detach().requires_grad_(only == 1)
        got, = torch.autograd.grad(linear_cross_entropy(a, b, y), (a, b)[only])
        assert torch.equal(got, (dx, dw)[only])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,V", [(50, 32, 70), (260, 256, 1500)])
def test_cross_entropy_extreme_scores(n, d, V, dtype):
    """Scores far apart (one class takes all), and rows whose scores are all equal."""
    x, w, y = ce_inputs(n, d, V, dtype, spread=60.0)
    x[1] = 0
    check_ce(x, w, y)


def test_cross_entropy_half_gradients_do_not_underflow():
    """Mean over many rows in fp16: a row's factor is far below fp16's smallest number and comes in at the end."""
    x, w, y = ce_inputs(600, 64, 900, torch.float16)
    check_ce(x, w, y, grad=torch.tensor(1024.0, device="cuda"))
    check_ce(x, w, y, "none", torch.full((600,), 1e-9, device="cuda"))
    check_ce(x, w, y, "none", torch.linspace(0, 7e4, 600, device="cuda"))


# ---------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------
def distill_inputs(n, V, K, dtype, pad=0, seed=0, t_dtype=None, missing=0.1, empty=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed + 5 * n + V + 3 * K)
    z = (2.5 * torch.randn(n, V + pad, generator=g, device="cuda")).to(dtype)[:, :V]
    ids = torch.rand(n, V, generator=g, device="cuda").argsort(1)[:, :K]
    if K > V:
        ids = torch.randint(0, V, (n, K), generator=g, device="cuda")
    t = (3 * torch.randn(n, K, generator=g, device="cuda")).to(t_dtype or dtype)
    ids = torch.where(torch.rand(n, K, generator=g, device="cuda") < missing, -1, ids)
    ids = torch.where(torch.rand(n, 1, generator=g, device="cuda") < empty, -1, ids)
    ids[n // 2, 0] = V - 1
    return z, t, ids


def distill_reference(z, t, ids, T, r):
    z64, n, V = z.double() / T, z.shape[0], z.shape[1]
    there = (ids >= 0) & (t != -math.inf)
    has = there.any(1)
    t64 = torch.where(there, t.double() / T, -math.inf)
    lt = torch.where(has, torch.logsumexp(t64, 1), 0.0)[:, None]
    lp = t64 - lt
    p = torch.where(there, lp.exp(), 0.0)
    lse = torch.logsumexp(z64, 1, keepdim=True)
    at = torch.where(there, ids, 0).long()
    lq = (z64 - lse).gather(1, at)
    rows = T * T * torch.where(p > 0, p * (lp - lq), 0.0).sum(1)
    # errors: an argument (z - max) / T log2(e) is off by 4 u of itself, a sum of V terms by V u
    # (where q or p is 0 in 64 bits it is 0 in 32)
    far = torch.where((z64 - lse).exp() > 0, z64.amax(1, keepdim=True) - z64, 0.0)
    far_p = torch.where(there, torch.where(has[:, None], t64, 0.0).amax(1, keepdim=True) - t64, 0.0)
    K = ids.shape[1]
    rel_q = 4 * U32 * far + 2 * 2.0 ** -21 + (V + 32) * U32
    rel_p = 4 * U32 * far_p + 2 * 2.0 ** -21 + (K + 32) * U32
    size = torch.where(p > 0, lp.abs() + lq.abs(), 0.0)
    term = p * (rel_p * size + (rel_p + rel_q.gather(1, at)) + 8 * U32 * size)
    rows_bound = 1.01 * T * T * (term.sum(1) + (K + 32) * U32 * (p * size).sum(1)) + 1e-30
    q = (z64 - lse).exp()
    taken = torch.zeros_like(q).scatter_add_(1, at, p)
    taken_err = torch.zeros_like(q).scatter_add_(1, at, p * rel_p)
    f = torch.where(has, r.double() * T, 0.0)[:, None]
    dz = f * (q - taken)
    b = f.abs() * (1.01 * (q * rel_q + taken_err) + 8 * U32 * (q + taken) + FLUSHED)
    return rows, rows_bound, dz, b + U[z.dtype] * (dz.abs() + b) + TINY[z.dtype], has


def run_distill(z, t, ids, T, reduction, grad=None):
    from graph_rws_b200.layers import distillation_loss
    z = z.detach().requires_grad_(True)
    loss = distillation_loss(z, t, ids, temperature=T, reduction=reduction)
    assert loss.dtype == torch.float32
    dz, = torch.autograd.grad(loss, z, grad if grad is not None else torch.ones_like(loss))
    assert dz.dtype == z.dtype and dz.shape == z.shape
    return loss.detach(), dz


def check_distill(z, t, ids, T=2.0, reduction="mean", grad=None):
    n = z.shape[0]
    loss, dz = run_distill(z, t, ids, T, reduction, grad)
    g = torch.ones((), device="cuda") if grad is None else grad
    has = ((ids >= 0) & (t != -math.inf)).any(1)
    counted = int(has.sum())
    r = torch.broadcast_to(g / counted if reduction == "mean" else g, (n,))
    rows, rb, dz64, dzb, _ = distill_reference(z, t, ids, T, r)
    if reduction == "none":
        within(loss, rows, rb, "loss")
    else:
        total, bound = rows.sum(), rb.sum() + (n + 64) * U32 * rows.abs().sum()
        within(loss, total / counted if reduction == "mean" else total, bound / counted if reduction == "mean" else bound, "loss")
    within(dz, dz64, dzb + 4 * U32 * dz64.abs(), "dlogits")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,K", [(1, 1, 1), (1, 2, 2), (5, 3, 7), (64, 172, 8), (257, 47, 5), (33, 1024, 64), (33, 1024, 65), (20, 1025, 20),
                                   (7, 4999, 33), (3, 70001, 64), (1, 262144, 1024), (1300, 8192, 16), (300, 130, 1)])
def test_distillation_matches_the_definition(n, V, K, dtype):
    check_distill(*distill_inputs(n, V, K, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,V,K", [(90, 41, 6), (40, 3001, 12), (2, 50000, 9)])
def test_distillation_reductions(n, V, K, dtype, reduction):
    z, t, ids = distill_inputs(n, V, K, dtype, pad=7, t_dtype=torch.float32)
    g = torch.rand(n, device="cuda") * 3 - 1 if reduction == "none" else torch.tensor(0.37, device="cuda")
    check_distill(z, t, ids, 1.0, reduction, g)
    check_distill(z, t.bfloat16(), ids.int(), 4.0, reduction, g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [47, 1500, 20000])
def test_distillation_same_class_twice(V, dtype):
    z, t, ids = distill_inputs(30, V, 12, dtype)
    ids[:, 3] = ids[:, 1]
    ids[:, 7] = ids[:, 1]
    ids[4] = 11
    check_distill(z, t, ids)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [60, 2000, 30000])
def test_distillation_rows_without_entries_and_infinities(V, dtype):
    z, t, ids = distill_inputs(20, V, 6, dtype, missing=0.0, empty=0.0)
    ids[0], ids[19] = -1, -7
    t[1] = -math.inf                      # entries of weight zero are none
    t[2, 1:] = -math.inf                  # a single entry
    z[3, :] = torch.finfo(dtype).min      # a mask of the type's lowest value, the teacher's classes left
    z[3, ids[3]] = 1.0
    z[4, :] = -math.inf
    z[4, ids[4]] = 2.0
    z[5] = 0.5                            # all classes alike
    check_distill(z, t, ids)
    check_distill(z, t, ids, reduction="none")
    # a class the student excludes: infinite loss, finite gradient
    z2 = z.clone()
    z2[6, ids[6, 0]] = -math.inf
    loss, dz = run_distill(z2, t, ids, 2.0, "none")
    assert torch.isinf(loss[6]) and torch.isfinite(dz).all() and torch.isfinite(loss[7:]).all()
    # an id past the classes, a NaN
    ids2, z3 = ids.clone(), z.clone()
    ids2[8, 2] = V
    z3[9, V // 2] = math.nan
    loss, dz = run_distill(z3, t, ids2, 2.0, "none")
    for row in (8, 9):
        assert torch.isnan(loss[row]) and torch.isnan(dz[row]).all()
    assert torch.isfinite(loss[10:]).all() and torch.isfinite(dz[10:]).all()
    none = torch.full_like(ids, -1)
    loss, dz = run_distill(z, t, none, 2.0, "mean")
    assert torch.isnan(loss) and not dz.any()
    loss, dz = run_distill(z, t, none, 2.0, "sum")
    assert loss == 0 and not dz.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 45, 1400, 9001])
def test_distillation_offsets_and_strides(V, dtype):
    """Every alignment of the rows, a narrow cut of a wide matrix, transposed orders."""
    z, t, ids = distill_inputs(12, V, min(V, 5), dtype)
    want = run_distill(z, t, ids, 2.0, "mean")
    for off, width in ((1, V + 1), (3, V + 8), (7, V + 9), (0, V + 100)):
        wide = torch.full((12, off + width), 77.0, dtype=dtype, device="cuda")
        wide[:, off:off + V] = z
        got = run_distill(wide[:, off:off + V], t, ids, 2.0, "mean")
        assert torch.allclose(got[0], want[0], rtol=1e-5) and torch.allclose(got[1].float(), want[1].float(), rtol=3 * U[dtype], atol=1e-7)
    check_distill(z.t().contiguous().t(), t.t().contiguous().t(), ids.t().contiguous().t())


def test_distillation_empty_batch():
    z, t, ids = (torch.zeros(0, k, device="cuda") for k in (9, 3, 3))
    ids = ids.long()
    assert run_distill(z, t, ids, 1.0, "sum")[0] == 0 and torch.isnan(run_distill(z, t, ids, 1.0, "mean")[0])
    assert run_distill(z, t, ids, 1.0, "none")[1].shape == (0, 9)


def test_distillation_offsets_past_31_bits():
    """Rows behind the 2^31st element of a matrix."""
    n, V = 33000, 65536
    z = torch.zeros(n, V, dtype=torch.bfloat16, device="cuda")
    z[-3:] = torch.randn(3, V, device="cuda").bfloat16()
    ids = torch.full((n, 4), -1, dtype=torch.int32, device="cuda")
    ids[-3:] = torch.tensor([5, 65535, 40000, 77], dtype=torch.int32, device="cuda")
    t = torch.randn(n, 4, device="cuda")
    loss, dz = run_distill(z, t, ids, 1.0, "none")
    assert not loss[:-3].any() and not dz[:-3].any()
    rows, rb, dz64, dzb, _ = distill_reference(z[-3:], t[-3:], ids[-3:], 1.0, torch.ones(3, device="cuda"))
    within(loss[-3:], rows, rb, "loss")
    within(dz[-3:], dz64, dzb, "dlogits")


# ---------------------------------------------------------------------------------------------
# both, as a program uses them
# ---------------------------------------------------------------------------------------------
def _both(x, w, y, t, ids):
    from graph_rws_b200.layers import distillation_loss, linear_cross_entropy
    return linear_cross_entropy(x, w, y) + 0.5 * distillation_loss(x @ w, t, ids, temperature=2.0)


def _case(dtype=torch.bfloat16):
    x, w, y = ce_inputs(200, 96, 700, dtype)
    _, t, ids = distill_inputs(200, 700, 8, dtype)
    return x, w, y, t, ids


def test_repeat_bit_by_bit():
    x, w, y, t, ids = _case()
    first = run_ce(x, w, y, "mean") + run_distill(x @ w, t, ids, 2.0, "mean")
    for _ in range(3):
        again = run_ce(x, w, y, "mean") + run_distill(x @ w, t, ids, 2.0, "mean")
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_two_streams_at_once():
    cases = [ce_inputs(n, 160, 1200, torch.bfloat16, seed=n) for n in (300, 301)]
    want = [run_ce(*c, "mean") for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(run_ce(*c, "mean"))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_another_stream_than_the_operands_and_another_device():
    x, w, y = ce_inputs(130, 64, 500, torch.bfloat16)
    want = run_ce(x, w, y, "mean")
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = run_ce(x, w, y, "mean")
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if torch.cuda.device_count() > 1:
        from graph_rws_b200.layers import linear_cross_entropy
        a, b = (t.to("cuda:1").requires_grad_(True) for t in (x, w))
        assert torch.cuda.current_device() == 0
        loss = linear_cross_entropy(a, b, y.to("cuda:1"))
        grads = torch.autograd.grad(loss, (a, b))
        assert loss.device.index == 1 and torch.equal(grads[0].cpu(), want[1].cpu()) and torch.equal(grads[1].cpu(), want[2].cpu())


def test_broadcast_inputs_and_shared_weights():
    """Gradients of a row used by all rows, and of a weight used twice, are sums."""
    from graph_rws_b200.layers import distillation_loss, linear_cross_entropy
    x, w, y = ce_inputs(60, 32, 90, torch.float32)
    row = x[:1].detach().requires_grad_(True)
    w1 = w.detach().requires_grad_(True)
    loss = linear_cross_entropy(row.expand(60, 32), w1, y) + linear_cross_entropy(x, w1, y)
    got = torch.autograd.grad(loss, (row, w1))
    rd, wd = row.detach().double().requires_grad_(True), w.double().requires_grad_(True)
    ref = torch.nn.functional.cross_entropy(rd.expand(60, 32) @ wd, y) + torch.nn.functional.cross_entropy(x.double() @ wd, y)
    for a, b in zip(got, torch.autograd.grad(ref, (rd, wd))):
        assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
    z, t, ids = distill_inputs(40, 77, 5, torch.float32)
    zr = z[:1].detach().clone().requires_grad_(True)
    dz, = torch.autograd.grad(distillation_loss(zr.expand(40, 77), t, ids, temperature=2.0, reduction="sum"), zr)
    _, _, dz64, _, _ = distill_reference(z[:1].expand(40, 77), t, ids, 2.0, torch.ones(40, device="cuda"))
    assert dz.shape == (1, 77) and float((dz.double() - dz64.sum(0)).abs().max()) <= 1e-5 * float(dz64.sum(0).abs().max())


def test_captured_step_replays_on_new_inputs():
    x, w, y, t, ids = _case()
    bufs = [v.clone() for v in (x, w, y, t, ids)]
    xs, ws = bufs[0].requires_grad_(True), bufs[1].requires_grad_(True)

    def body():
        return (lambda loss: (loss.detach(),) + torch.autograd.grad(loss, (xs, ws)))(_both(xs, ws, *bufs[2:]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    for seed in (1, 2):
        x2, w2, y2 = ce_inputs(200, 96, 700, torch.bfloat16, seed=seed)
        with torch.no_grad():
            xs.copy_(x2)
            ws.copy_(w2)
        bufs[2].copy_(y2)
        graph.replay()
        got = [v.clone() for v in out]
        a, b = x2.requires_grad_(True), w2.requires_grad_(True)
        loss = _both(a, b, y2, t, ids)
        want = (loss.detach(),) + torch.autograd.grad(loss, (a, b))
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_backward_twice_on_one_graph():
    from graph_rws_b200.layers import distillation_loss, linear_cross_entropy
    x, w, y, t, ids = _case()
    x.requires_grad_(True)
    for loss in (linear_cross_entropy(x, w, y), distillation_loss(x @ w, t, ids)):
        a, = torch.autograd.grad(loss, x, retain_graph=True)
        b, = torch.autograd.grad(loss, x)
        assert torch.equal(a, b)


def test_refusals():
    from graph_rws_b200.layers import distillation_loss, linear_cross_entropy
    x, w, y, t, ids = _case()
    z = (x @ w).detach()
    bad = [
        lambda: linear_cross_entropy(x.cpu(), w, y), lambda: linear_cross_entropy(x, w.float(), y), lambda: linear_cross_entropy(x, w.t(), y),
        lambda: linear_cross_entropy(x, w, y[:-1]), lambda: linear_cross_entropy(x, w, y.float()), lambda: linear_cross_entropy(x, w, y.cpu()),
        lambda: linear_cross_entropy(x[0], w, y), lambda: linear_cross_entropy(x.double(), w.double(), y),
        lambda: linear_cross_entropy(x[:, :0], w[:0], y), lambda: linear_cross_entropy(x, w[:, :0], y),
        lambda: distillation_loss(z, t, ids[:, :-1]), lambda: distillation_loss(z[:-1], t, ids), lambda: distillation_loss(z, t, ids.float()),
        lambda: distillation_loss(z, t.cpu(), ids), lambda: distillation_loss(z.double(), t, ids),
        lambda: distillation_loss(z, t.detach().requires_grad_(True), ids), lambda: distillation_loss(z, t[:, :0], ids[:, :0]),
        lambda: distillation_loss(z, t.repeat(1, 129), ids.repeat(1, 129)),
    ]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: linear_cross_entropy(x, w, y, reduction="average"), lambda: distillation_loss(z, t, ids, temperature=0.0),
                 lambda: distillation_loss(z, t, ids, temperature=math.nan), lambda: distillation_loss(z, t, ids, reduction="batchmean")):
        with pytest.raises(ValueError):
            call()
    xg = x.detach().requires_grad_(True)
    g, = torch.autograd.grad(linear_cross_entropy(xg, w, y), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
