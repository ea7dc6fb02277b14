"""Output tiles that leave through shared memory, with a last column tile that is partly outside the output: the steps that store
nothing must not let a later step write memory that an earlier tile store still reads.  Short K (the epilogue follows on the heels of
the next tile's operands), no activation and no residual (the shortest steps), many repeats, every one compared bit for bit."""
import pytest
import torch

from tests.test_gpu_gemm_fused import Problem

pytestmark = pytest.mark.gpu

REPEATS = 40


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


def repeats_agree(run, what):
    want = run()
    outs = [run() for _ in range(REPEATS)]
    bad = [i for i, o in enumerate(outs) if not torch.equal(o, want)]
    assert not bad, f"{what}: repeats {bad} differ from the first call"
    return want


@pytest.mark.parametrize("otype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("name", ["tc5_256x192_n_s0", "tc5_256x256_n_s0", "tc5_128x192_n_s0", "tc5_128x96_n_s0", ""])
@pytest.mark.parametrize("n", [4096, 4096 + 64, 4096 + 16])
@pytest.mark.parametrize("kind", ["bf16", "mxfp8", "mxfp4"])
def test_fused_epilogue_without_a_residual(ab, kind, n, name, otype):
    p = Problem(ab, kind, 1280, n, 256)
    got = repeats_agree(lambda: p.run(otype=otype, kernelName=name), f"{kind} {n} {name}")
    p.check(got, what=f"{kind} {n} {name}")
    assert ab.device_status(0) == (0, 0, 0, 0)


@pytest.mark.parametrize("name", ["tc5_256x192_n_s3", "tc5_256x256_n_s3", "tc5_128x192_n_s3", "tc5_128x96_n_s3", "tc5_128x224_n_s2", "tc5_128x128_t_s3", ""])
@pytest.mark.parametrize("m,n", [(1280, 4096), (1280, 4096 + 64), (1296, 4096 + 16)])
@pytest.mark.parametrize("kind", ["bf16", "mxfp8", "mxfp4"])
def test_plain_epilogue(ab, kind, m, n, name):
    p = Problem(ab, kind, m, n, 256)

    def run():
        if kind == "mxfp8":
            return ab.gemm_a8w8_mxfp8(*p.args, a_preshuffle=False, kernelName=name)
        out = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
        return ab.gemm_a16w16_asm(*p.args, out, kernelName=name) if kind == "bf16" else ab.gemm_a4w4_asm(*p.args, out, kernelName=name)

    got = repeats_agree(run, f"{kind} {m} {n} {name}")
    p.check(got, what=f"{kind} {m} {n} {name}")
    assert ab.device_status(0) == (0, 0, 0, 0)
