"""gated_residual_norm on rows that do not fit the registers: the sums' error does not grow with the row.

A row's sum: squares and pairwise sums of eight (4 roundings), a compensated sum (2) and a tree over the CTA (10), 16 * 2^-24 relative in the
mean square with the mean's scale (2), half of that after the square root; rsqrt 2^-22, two more roundings in y.  9 * 2^-24 + 4 * 2^-24 + 2 * 2^-24 < 2^-20 of
the value.  Layer norm: the mean is off by at most 13 * 2^-24 of mean |x| and x - mean by one rounding, so 2^-19 of the row's largest
(|x| + mean |x|) / std covers it with the above."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


@pytest.mark.parametrize("first", [0, 1], ids=["aligned", "odd address"])
@pytest.mark.parametrize("n", [20000, 131072 * 8, 131072 * 8 + 40])
@pytest.mark.parametrize("value", [1.1015625, 0.7001953125])
def test_rms_of_equal_values(ab, n, first, value):
    """Equal squares: every addition of a plain sum rounds the same way over long stretches."""
    x = torch.full((2, n + first), value, dtype=torch.float32, device="cuda")[:, first:]
    y, _ = ab.gated_residual_norm(x, eps=0.0)
    assert (y.double() - 1).abs().max().item() <= 2.0**-20


@pytest.mark.parametrize("first", [0, 1], ids=["aligned", "odd address"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("n", [16392, 300000, 131072 * 8])
def test_against_64_bits(ab, n, norm, first):
    g = torch.Generator().manual_seed(n)
    x = (torch.rand(3, n + first, generator=g) + 0.5).cuda()[:, first:]  # a mean that is not zero
    y, _ = ab.gated_residual_norm(x, norm=norm, eps=0.0)
    v = x.double()
    mean = v.mean(1, keepdim=True) if norm == "layer" else torch.zeros(3, 1, dtype=torch.float64, device="cuda")
    std = ((v - mean) ** 2).mean(1, keepdim=True).sqrt()
    want = (v - mean) / std
    tol = 2.0**-20 * want.abs() if norm == "rms" else 2.0**-20 * want.abs() + 2.0**-19 * ((v.abs() + v.abs().mean(1, keepdim=True)) / std).amax(1, keepdim=True)
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("first", [0, 1], ids=["aligned", "odd address"])
def test_infinities(ab, first):
    """One infinity, and squares whose sum passes the largest float: the mean square is infinite, the finite values become 0."""
    n = 20000
    x = torch.ones(3, n + first, dtype=torch.float32, device="cuda")[:, first:]
    x[0, 777] = float("inf")
    x[1, 5] = float("nan")
    x[2, :] = 1e19  # (squares of 1e38)
    y, _ = ab.gated_residual_norm(x)
    keep = torch.arange(n, device="cuda") != 777
    assert (y[0][keep] == 0).all() and torch.isnan(y[0, 777])
    assert torch.isnan(y[1]).all()
    assert (y[2] == 0).all()
