"""linear_cross_entropy without a reduction, with row gradients of very different sizes: every row's dx is checked relative to its
own size, and an ignored row's gradient, whatever it is, changes nothing."""
import pytest
import torch

from test_losses_gpu import DTYPES, check_ce, ce_inputs, run_ce

pytestmark = pytest.mark.gpu

SIZES = [(64, 40, 90), (300, 96, 2000), (500, 64, 20011)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("class_major", [False, True])
@pytest.mark.parametrize("n,d,V", SIZES)
def test_row_gradients_over_many_decades(n, d, V, class_major, dtype):
    x, w, y = ce_inputs(n, d, V, dtype, class_major)
    g = torch.logspace(4, -5, n, device="cuda")
    g[::3] *= -1
    check_ce(x, w, y, "none", g[torch.randperm(n, generator=torch.Generator().manual_seed(1)).cuda()])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,V", SIZES)
def test_ignored_rows_with_large_gradients(n, d, V, dtype):
    x, w, y = ce_inputs(n, d, V, dtype, ignored=0.2)
    g = torch.rand(n, device="cuda") + 0.5
    want = run_ce(x, w, y, "none", g)
    g2 = torch.where(y == -100, 1e37, g)
    check_ce(x, w, y, "none", g2)
    got = run_ce(x, w, y, "none", g2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g2 = torch.where(y == -100, torch.inf, g)
    got = run_ce(x, w, y, "none", g2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_only_small_gradients_reach(dtype):
    """Columns of x that are 0 where the gradients are large: their rows of dweight come from the small ones alone."""
    n, d, V = 200, 64, 400
    x, w, y = ce_inputs(n, d, V, dtype)
    x[:100, 32:] = 0
    g = torch.full((n,), 1e4, device="cuda")
    g[100:] = 1e-3
    check_ce(x, w, y, "none", g)
