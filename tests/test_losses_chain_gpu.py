"""Calls of the losses that follow each other without anything between them, each on what the one before has just written:
the same as with the GPU waited for after every call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _chain(step, first, times, wait):
    out, value = [], first
    for _ in range(times):
        loss, value = step(value)
        if wait:
            torch.cuda.synchronize()
        out += [loss, value]
    return out


def _same(step, first, times=6):
    want = _chain(step, first, times, True)
    for _ in range(5):
        torch.cuda.synchronize()
        got = _chain(step, first, times, False)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("n,d,V", [(70, 24, 50), (1500, 96, 4000), (20000, 40, 170)])
def test_cross_entropy_of_the_gradients_just_written(n, d, V, dtype, reduction):
    from graph_rws_b200.layers import linear_cross_entropy
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, d, generator=g, device="cuda").to(dtype)
    w = torch.randn(d, V, generator=g, device="cuda").to(dtype)
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    grad = torch.full((n,) if reduction == "none" else (), 1.0 if reduction == "none" else float(n), device="cuda")

    def step(x):
        x = x.detach().requires_grad_(True)
        loss = linear_cross_entropy(x, w, y, reduction=reduction)
        return loss.detach(), torch.autograd.grad(loss, x, grad)[0]
    _same(step, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("n,V,K", [(3000, 47, 5), (700, 5000, 20), (3, 60000, 9)])
def test_distillation_of_the_gradients_just_written(n, V, K, dtype, reduction):
    from graph_rws_b200.layers import distillation_loss
    g = torch.Generator(device="cuda").manual_seed(n)
    z = torch.randn(n, V, generator=g, device="cuda").to(dtype)
    t = torch.randn(n, K, generator=g, device="cuda")
    ids = torch.randint(0, V, (n, K), generator=g, device="cuda")
    grad = torch.full((n,) if reduction == "none" else (), 4.0 if reduction == "none" else 4.0 * n, device="cuda")

    def step(z):
        z = z.detach().requires_grad_(True)
        loss = distillation_loss(z, t, ids, temperature=1.5, reduction=reduction)
        return loss.detach(), torch.autograd.grad(loss, z, grad)[0]
    _same(step, z)
