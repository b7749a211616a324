"""distillation_loss with as many classes as 31 bits hold: the last part of the row ends at the row's end."""
import math

import pytest
import torch

from test_losses_gpu import U32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [2 ** 31 - 1, 2 ** 31 - 4096, 2 ** 31 - 2 ** 23])
def test_distillation_of_the_longest_rows(V):
    """All scores 0 but 20 of 20.0 near the end.  Rounding: the 2^31 ones are summed by 2^17 threads and joined, each sum of at
    most 2^15 terms, so the sum of exponentials is off by 2^-9 of itself at most and far less in earnest: 2^-12 is allowed."""
    from graph_rws_b200.layers import distillation_loss
    z = torch.zeros(1, V, dtype=torch.bfloat16, device="cuda")
    high = V - 1 - 1000 * torch.arange(20, device="cuda")
    z[0, high] = 20.0
    ids = torch.tensor([[V - 1, 7, V - 1001, V - 3]], device="cuda")
    t = torch.tensor([[1.0, 0.5, -0.5, 0.0]], device="cuda")
    lse = math.log(20 * math.exp(20.0) + V - 20)
    p = torch.softmax(t.double(), 1)[0].cpu()
    lq = torch.tensor([20.0, 0.0, 20.0, 0.0], dtype=torch.float64) - lse
    want = float((p * (p.log() - lq)).sum())
    z.requires_grad_(True)
    loss = distillation_loss(z, t, ids, reduction="none")
    assert abs(float(loss.detach()) - want) <= 2.0 ** -12 + 64 * U32 * abs(want)
    dz, = torch.autograd.grad(loss, z, torch.ones_like(loss))
    q0, q1 = math.exp(-lse), math.exp(20.0 - lse)
    step = 2.0 ** -8 + 2.0 ** -12 + 64 * U32
    got = dz[0, ids[0]].double().cpu()
    expected = lq.exp() - p
    assert ((got - expected).abs() <= step * (expected.abs() + lq.exp())).all()
    got = dz[0, high[2:]].double()
    assert ((got - q1).abs() <= step * q1).all()
    with torch.no_grad():
        dz[0, ids[0]] = q0
        dz[0, high] = q0
    least, most = torch.aminmax(dz)
    assert q0 * (1 - step) <= float(least) and float(most) <= q0 * (1 + step)
