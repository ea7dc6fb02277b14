"""MX GEMMs with a fused epilogue whose output or residual rows allow no tile copies: odd pitches, shifted bases, one broadcast residual
row.  More than 256 rows take CTA pairs with the weights on the 128-row slot."""
import pytest
import torch

from tests.test_gpu_gemm_fused import Problem, check, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


@pytest.mark.parametrize("m", [65, 200, 257, 300, 1024, 4100])
@pytest.mark.parametrize("n", [16, 528, 1040])
@pytest.mark.parametrize("kind", ["mxfp8", "mxfp4"])
def test_rows_without_tile_copies(ab, kind, n, m):
    k = 256
    p = Problem(ab, kind, m, n, k)
    residual, bias = randn(m, m, n), randn(n, n)
    for pitch, first in ((n + 5, 3), (n + 16, 1), (n + 1, 0)):
        buf = torch.full((m + 2, pitch), 7.0, dtype=torch.bfloat16, device="cuda")
        view = buf[1 : m + 1, first : first + n]
        view.copy_(residual)
        p.check(p.run(activation="gelu", bias=bias, residual=view, out=view), bias=bias, activation="gelu", residual=residual, what=f"in place, pitch {pitch}, first {first}")
        view.fill_(7.0)
        assert (buf == 7).all(), "something around the output was written"
        wide = torch.full((m, pitch), 3.0, dtype=torch.float32, device="cuda")[:, first : first + n]
        wide.copy_(residual)
        p.check(p.run(activation="silu", residual=wide, otype=torch.float32), activation="silu", residual=residual, what=f"fp32 residual, pitch {pitch}, first {first}")
    row = randn(5, 1, n, dtype=torch.float16)
    p.check(p.run(residual=row.expand(m, n), otype=torch.float16), residual=row.expand(m, n), what="one row for all")
    p.check(p.run(activation="relu", bias=bias, residual=row[0, :1].expand(m, n).contiguous(), out=torch.empty(m, n + 1, dtype=torch.bfloat16, device="cuda")[:, :n]), bias=bias,
            activation="relu", residual=row[0, :1].expand(m, n), what="odd output rows")
    assert ab.device_status(0) == (0, 0, 0, 0)


@pytest.mark.parametrize("m,n", [(1024, 528), (4100, 1040), (4096, 16)])
def test_mxfp4_with_and_without_a_workspace(ab, m, n):
    k = 4096
    p = Problem(ab, "mxfp4", m, n, k)
    A, B, SA, SB = p.args
    assert ab._ffi._lib.aiter_b200_gemm_a4w4_fused_workspace(m, n, k) > 0
    residual = randn(m, m, n)
    for pitch in (n, n + 3):
        with_ws, without = (torch.full((m, pitch), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        p.run(activation="silu", residual=residual, out=with_ws[:, :n])
        ab._ffi.call("aiter_b200_gemm_a4w4_fused", A, B, SA, SB, None, residual, without[:, :n], None, 2, 1, None)
        for what, got in (("with", with_ws), ("without", without)):
            check(got[:, :n], p.a, p.b, p.steps, None, "silu", residual, f"{what} a workspace, pitch {pitch}")
            assert (got[:, n:] == 7).all()
    assert ab.device_status(0) == (0, 0, 0, 0)
