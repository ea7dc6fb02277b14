"""The fused GEMMs, the norm and the gated activation need no call before a capture: each is captured as the first call of a process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys

import torch

import aiter_b200 as ab


def randn(*shape):
    return torch.randn(*shape, device="cuda").bfloat16()


def mxfp4(rows, k):
    # any codes, scales of 2^-2 .. 2^2
    codes = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda").view(ab.dtypes.fp4x2)
    scales = torch.randint(125, 130, ((rows + 255) // 256 * 256, k // 32), dtype=torch.uint8, device="cuda").view(ab.dtypes.fp8_e8m0)
    return codes, scales


what = sys.argv[1]
torch.manual_seed(0)
if what == "gemm, one row":
    a, b, bias = randn(1, 1024), randn(512, 1024), randn(512)
    call = lambda: ab.gemm_a16w16_fused(a, b, bias, "silu")
elif what == "gemm, few rows":
    a, b, r = randn(48, 1024), randn(512, 1024), randn(48, 512)
    call = lambda: ab.gemm_a16w16_fused(a, b, None, "gelu", r)
elif what == "gemm, many rows":
    a, b, bias = randn(1300, 256), randn(1040, 256), randn(1040)
    call = lambda: ab.gemm_a16w16_fused(a, b, bias, "relu")
elif what == "mxfp4 gemm with a workspace":
    (a, sa), (b, sb) = mxfp4(1024, 4096), mxfp4(1024, 4096)
    call = lambda: ab.gemm_a4w4_fused(a, b, sa, sb)
elif what == "norm, one row":
    x, w = randn(1, 4096), randn(4096)
    call = lambda: ab.gated_residual_norm(x, x, w)[0]
elif what == "norm, many rows":
    x, w = randn(2000, 4096), randn(4096)
    call = lambda: ab.gated_residual_norm(x, x, w)[0]
elif what == "gated activation":
    x = randn(100, 512)
    call = lambda: ab.act_and_mul(x)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
got.fill_(float("nan"))
graph.replay()
torch.cuda.synchronize()
assert torch.equal(got, call()), "replayed and eager outputs differ"
assert ab.device_status(0) == (0, 0, 0, 0)
print("captured first")
"""


@pytest.mark.parametrize("what", ["gemm, one row", "gemm, few rows", "gemm, many rows", "mxfp4 gemm with a workspace", "norm, one row", "norm, many rows", "gated activation"])
def test_first_call_of_a_process_inside_a_capture(what):
    p = subprocess.run([sys.executable, "-c", PROGRAM, what], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "captured first" in p.stdout, p.stdout[-2000:] + p.stderr[-3000:]
