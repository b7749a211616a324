"""linear_cross_entropy without a reduction: an ignored row's gradient, whatever it is, changes nothing."""
import pytest
import torch

from test_losses_gpu import DTYPES, check_ce, ce_inputs, run_ce

pytestmark = pytest.mark.gpu

SIZES = [(64, 40, 90), (300, 96, 2000), (500, 64, 20011)]


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
