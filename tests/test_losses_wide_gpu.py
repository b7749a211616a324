"""linear_cross_entropy of wide 16-bit rows: scores as near to 64 bits as those of narrow ones."""
import math

import pytest
import torch

from test_losses_gpu import TINY, U, U32, check_ce, ce_inputs

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("class_major", [False, True])
@pytest.mark.parametrize("n,V", [(5, 2), (300, 300), (600, 129)])
def test_sums_of_one_sign(n, V, class_major, dtype):
    """Scores s > 0 of one class, all products positive, 0 of the others, the label one of those: the loss is log(exp(s) + V - 1), so
    what the sum over 65,536 elements loses is seen as it is.

    The tensor cores cut a sum off, 16 products and what is there at a time, each of the 17 by a unit of 2^-24 of the result at most.  In a chain of 256
    elements, which grows evenly, that is 17 * (1 + .. + 16) / 16 units = 145; the 256 chains are added with half a unit of a sum that grows
    evenly each, 64 in all; 32 more for the softmax.  A single chain would lose 17 * 4,096 / 2 at worst."""
    d = 65536
    g = torch.Generator(device="cuda").manual_seed(n)
    x = (1 + torch.rand(n, d, generator=g, device="cuda")).to(dtype)
    w = torch.zeros(d, V, device="cuda")
    w[:, 0] = (1 + torch.rand(d, generator=g, device="cuda")) * (8.0 / d)
    w = w.to(dtype)
    w = w.t().contiguous().t() if class_major else w
    from graph_rws_b200.layers import linear_cross_entropy
    loss = linear_cross_entropy(x, w, torch.full((n,), V - 1, device="cuda"), reduction="none").double()
    want = torch.log(torch.exp(x.double() @ w[:, 0].double()) + (V - 1))
    assert ((loss - want).abs() <= (145 + 64 + 32) * U32 * want).all(), float(((loss - want) / want).abs().max())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("class_major", [False, True])
@pytest.mark.parametrize("n,V", [(5, 2), (300, 300)])
def test_gradients_of_sums_of_one_sign(n, V, class_major, dtype):
    """The same scores with the label's class masked by a weight of 0: dx_ik = g (q_i w_k0) with q_i = 1 / (1 + (V - 1) exp(-s_i)).  G and dx are
    rounded, the softmax is off by twice what a score is: the test above."""
    d = 65536
    g = torch.Generator(device="cuda").manual_seed(n)
    x = (1 + torch.rand(n, d, generator=g, device="cuda")).to(dtype)
    w = torch.zeros(d, V, device="cuda")
    w[:, 0] = (1 + torch.rand(d, generator=g, device="cuda")) * (8.0 / d)
    w = w.to(dtype)
    w = (w.t().contiguous().t() if class_major else w).requires_grad_(True)
    x.requires_grad_(True)
    from graph_rws_b200.layers import linear_cross_entropy
    loss = linear_cross_entropy(x, w, torch.full((n,), V - 1, device="cuda"), reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w), torch.tensor(64.0, device="cuda"))
    s = x.detach().double() @ w[:, 0].detach().double()
    q = 1 / (1 + (V - 1) * torch.exp(-s))
    want = 64 * q[:, None] * w[:, 0].detach().double()
    bound = 2 * U[dtype] + 2 * float(s.max()) * (145 + 64 + 32) * U32 + 64 * U32
    assert ((dx.double() - want).abs() <= bound * want + TINY[dtype]).all(), float(((dx.double() - want) / want).abs().max())
    want = 64 * x.detach().double().t() @ q
    assert ((dw[:, 0].double() - want).abs() <= (bound + n * U32) * want).all(), float(((dw[:, 0].double() - want) / want).abs().max())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("class_major", [False, True])
@pytest.mark.parametrize("n,d,V", [(100, 769, 7), (100, 768, 128), (300, 832, 128), (300, 776, 129), (70, 1024, 300), (300, 1032, 129), (3, 1440, 2001), (513, 1441, 640),
                                   (1, 2500, 1), (260, 4096, 70), (70, 4097, 300), (300, 4200, 129)])
def test_wide_rows(n, d, V, class_major, dtype):
    """Both sides of the widths from which sums are taken in chains, and classes that end in every part of a tile."""
    check_ce(*ce_inputs(n, d, V, dtype, class_major, ignored=0.1))


@pytest.mark.parametrize("dtype", HALVES)
def test_wide_rows_with_infinities(dtype):
    x, w, y = ce_inputs(200, 1300, 257, dtype)
    x[:, 5] = 1.0
    w[5, 200:] = torch.finfo(dtype).min
    y = y % 200
    from graph_rws_b200.layers import linear_cross_entropy
    loss = linear_cross_entropy(x, w, y, reduction="none").double()
    s = x.double() @ w[:, :200].double()
    bound = 2 * (1308 * U32 * (x.double().abs() @ w[:, :200].double().abs()).amax(1) + 300 * U32 + 2.0 ** -21)
    assert ((loss - torch.nn.functional.cross_entropy(s, y, reduction="none")).abs() <= bound).all()
    x[3, 7], x[4, 8] = math.inf, math.nan
    got = linear_cross_entropy(x, w, y, reduction="none").double()
    others = torch.ones(200, dtype=torch.bool, device="cuda")
    others[3:5] = False
    assert torch.equal(got[others], loss[others]) and torch.isnan(got[3:5]).all()
