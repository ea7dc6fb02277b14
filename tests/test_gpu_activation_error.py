"""The activations over their whole range, tails included, relative to the value in 64 bits.

Bounds (steps of 2^-24, with rcp.approx good to 2 steps and ex2.approx to 4): silu x / (1 + e), e = 2^(-x log2 e): the argument and the constant
are rounded once each, so e is off by |x| * 1.5 steps + 4, and 1 + e, its reciprocal and the product add 4: 2^-21 + |x| 2^-23.  gelu_tanh: the
argument -2u log2 e takes four roundings of its largest term: |2u| * 4 steps, and 8 more: 2^-21 + |2u| 2^-22.  gelu: x^2 and its product with the
constant, x^2 / 2 * 3 steps, t off by 3 steps, which the polynomial passes on with a factor below 2, its eight steps with a condition of at most
two, 2 of the fit, 4 of the power, 4 products: 32 steps = 2^-19, + x^2 2^-23.  The gated product rounds once more (2^-24).
Magnitudes below 2^-119 may come out as 0 (the reciprocal and the power flush)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FLUSH = 2.0**-119


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


def want_and_tol(x, act):
    x = x.double()
    if act == "silu":
        return x * torch.sigmoid(x), 2.0**-21 + x.abs() * 2.0**-23
    if act == "gelu":
        return 0.5 * x * torch.erfc(-x / math.sqrt(2)), 2.0**-19 + x * x * 2.0**-23
    if act == "gelu_tanh":
        u2 = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)
        return x * torch.sigmoid(u2), 2.0**-21 + u2.abs() * 2.0**-22
    return x.clamp(min=0), torch.zeros_like(x)


def check(got, x, act, what):
    want, rel = want_and_tol(x, act)
    off = (got.double() - want).abs()
    bad = off > (rel + 2.0**-23) * want.abs() + FLUSH
    assert torch.isfinite(got).all() and not bad.any(), f"{what}: {int(bad.sum())} off, first at x = {x[bad][0].item()!r}"


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_gated_activation(ab, act):
    n = 1 << 20
    parts = [torch.linspace(-lim, lim, n, dtype=torch.float64) for lim in (0.01, 1.0, 16.0, 120.0)]
    parts.append(torch.logspace(-36, 36, n // 2, dtype=torch.float64))
    parts.append(-torch.logspace(-36, 36, n // 2, dtype=torch.float64))
    x = torch.stack([p for p in parts[:4]] + [torch.cat(parts[4:])]).float().cuda()
    ones = torch.ones_like(x)
    check(ab.act_and_mul(torch.cat([x, ones], 1), act), x, act, "rows on 16-byte boundaries")
    odd = x[:, : n - 3]
    check(ab.act_and_mul(torch.cat([odd, ones[:, : n - 3]], 1), act), odd, act, "rows on odd addresses")


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m", [1, 20, 600], ids=["one row", "few rows", "tiles"])
def test_fused_gemm(ab, m, act):
    """A selects one column of B, so the accumulator is the bf16 value itself."""
    n, k = 8192, 64
    g = torch.Generator().manual_seed(m)
    x = torch.cat([(torch.rand(n // 2, generator=g) - 0.5) * 32, (torch.rand(n // 2, generator=g) - 0.5) * 220]).bfloat16().cuda()
    a, b = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    a[:, 5] = 1
    b[:, 5] = x
    y = ab.gemm_a16w16_fused(a, b, activation=act, otype=torch.float32)
    check(y, x.float().expand(m, n), act, f"{m} rows")
