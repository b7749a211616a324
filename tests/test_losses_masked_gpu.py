"""linear_cross_entropy where classes are masked in the weight: the row of a constant input column holds the type's lowest
value, or -inf.  Such a class has probability 0, so everything is as without it, and its column of dweight is 0."""
import pytest
import torch

from test_losses_gpu import DTYPES, U32, ce_inputs, ce_reference, run_ce, within

pytestmark = pytest.mark.gpu


def masked(n, d, V, dtype, class_major, value):
    """Inputs with a column of ones, `value` in its weight row for two classes of three, labels among the others, and which these are."""
    x, w, y = ce_inputs(n, d, V, dtype, class_major)
    x[:, d // 2] = 1.0
    open_ = torch.arange(0, V, 3, device="cuda")
    mask = torch.ones(V, dtype=torch.bool, device="cuda")
    mask[open_] = False
    w[d // 2, mask] = value
    y = open_[y % open_.numel()]
    return x, w, y, open_, mask


# on both sides of 2^21 products, from which fp32 goes to the tensor cores; one and two CTAs a tile; classes in pieces
SIZES = [(50, 32, 70), (200, 128, 200), (100, 260, 1003), (600, 72, 5000), (70001, 24, 4501)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("class_major", [False, True])
@pytest.mark.parametrize("value", ["lowest", "-inf"])
@pytest.mark.parametrize("n,d,V", SIZES)
def test_masked_classes(n, d, V, value, class_major, dtype):
    x, w, y, open_, mask = masked(n, d, V, dtype, class_major, torch.finfo(dtype).min if value == "lowest" else float("-inf"))
    r = torch.full((n,), 1.0, device="cuda")
    rows, rb, dx64, dxb, dw64, dwb = ce_reference(x, w[:, open_], y // 3, r)
    loss, dx, dw = run_ce(x, w, y, "sum")
    within(loss, rows.sum(), rb.sum() + (n + 64) * U32 * rows.abs().sum(), "loss")
    within(dw[:, open_], dw64, dwb * (1 + 4 * U32), "dweight")
    assert not dw[:, mask].any()
    if value == "-inf":
        # 0 * -inf: NaN in the definition as well, in the masking column alone
        assert torch.isnan(dx[:, d // 2]).all()
        keep = torch.arange(d, device="cuda") != d // 2
        dx, dx64, dxb = dx[:, keep], dx64[:, keep], dxb[:, keep]
    within(dx, dx64, dxb * (1 + 4 * U32), "dx")


@pytest.mark.parametrize("value", [3.4028234e38, -3.4028234e38, 3.3961775e38, 3.39e38])
@pytest.mark.parametrize("n,d,V", [(50, 32, 70), (200, 128, 200)])
def test_values_past_the_largest_bf16_number(n, d, V, value):
    """fp32's largest values, times numbers that bring them back, in x and in the weight."""
    x, w, y = ce_inputs(n, d, V, torch.float32)
    x[:, 3] = value
    w[3] *= 2.0 ** -126 * 8           # products of up to some 60, the weight's lower planes still normal numbers in part
    got = run_ce(x, w, y, "none")[0]
    s = x.double() @ w.double()
    want = torch.nn.functional.cross_entropy(s, y, reduction="none")
    # the planes below 2^-133 of w are lost: 2^-9 of the smallest normal number's 2^-126 at worst
    lost = abs(value) * 2.0 ** -133
    bound = 4 * lost + 2 * (d + V + 32) * U32 * (x.double().abs() @ w.double().abs()).amax(1) + 2.0 ** -20
    within(got, want, bound, "loss")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("n,d,V", [(50, 32, 70), (200, 128, 200)])
def test_infinities_and_nans_stay_in_their_rows(n, d, V, what, dtype):
    x, w, y = ce_inputs(n, d, V, dtype)
    want, dxw, _ = run_ce(x, w, y, "none")
    x[7, 3] = what
    loss, dx, _ = run_ce(x, w, y, "none")
    others = torch.arange(n, device="cuda") != 7
    assert torch.isnan(loss[7]) and torch.isnan(dx[7]).all()
    assert torch.equal(loss[others], want[others]) and torch.equal(dx[others], dxw[others])
