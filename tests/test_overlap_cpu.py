"""Whatever a call writes must not share memory with what it reads: the refusals, without a GPU."""
import pytest
import torch

from tests.test_block_ops_cpu import BASE, fake, refuse

MB = 1 << 20
M, N, K = 4, 256, 128


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


def mxfp8(ab, **over):
    q, u8, far = torch.float8_e4m3fn, torch.uint8, BASE + 32 * MB
    a = dict(A=fake(ab, (M, K), q, ptr=far), B=fake(ab, (N, K), q, ptr=far + MB), ScaleA=fake(ab, (32, K // 32), u8, ptr=far + 2 * MB),
             ScaleB=fake(ab, (N, K // 32), u8, ptr=far + 3 * MB), bias=fake(ab, (N,), ptr=far + 4 * MB), residual=fake(ab, (M, N), ptr=far + 5 * MB),
             out=fake(ab, (M, N), ptr=BASE), activation=0, a_preshuffle=0, name=None)
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def mxfp4(ab, **over):
    u8, far = torch.uint8, BASE + 32 * MB
    a = dict(A=fake(ab, (M, K // 2), u8, ptr=far), B=fake(ab, (N, K // 2), u8, ptr=far + MB), A_scale=fake(ab, (256, 8), u8, ptr=far + 2 * MB),
             B_scale=fake(ab, (N, 8), u8, ptr=far + 3 * MB), bias=fake(ab, (N,), ptr=far + 4 * MB), residual=fake(ab, (M, N), ptr=far + 5 * MB),
             out=fake(ab, (M, N), ptr=BASE), workspace=fake(ab, (4096,), u8, ptr=far + 6 * MB), activation=0, bpreshuffle=1, name=None)
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def test_fused_gemms_refuse_scales_and_workspaces_that_overlap(ab):
    u8, f = torch.uint8, lambda *a, **k: fake(ab, *a, **k)
    out_bytes = M * N * 2
    for at in (BASE, BASE + out_bytes - 16, BASE - 16):  # the first, the last and the bytes around out's beginning
        refuse(ab, "aiter_b200_gemm_a8w8_mxfp8_fused", mxfp8(ab, ScaleA=f((32, K // 32), u8, ptr=at)), "out overlaps the block scales")
        refuse(ab, "aiter_b200_gemm_a8w8_mxfp8_fused", mxfp8(ab, ScaleB=f((N, K // 32), u8, ptr=at)), "out overlaps the block scales")
        refuse(ab, "aiter_b200_gemm_a4w4_fused", mxfp4(ab, A_scale=f((256, 8), u8, ptr=at)), "out overlaps the block scales")
        refuse(ab, "aiter_b200_gemm_a4w4_fused", mxfp4(ab, B_scale=f((N, 8), u8, ptr=at)), "out overlaps the block scales")
        refuse(ab, "aiter_b200_gemm_a4w4_fused", mxfp4(ab, workspace=f((4096,), u8, ptr=at)), "workspace overlaps out")
    far = BASE + 32 * MB
    for at, match in [(far + 16, "workspace overlaps an operand"), (far + MB + N * K // 2 - 16, "workspace overlaps an operand"),
                      (far + 2 * MB + 256 * 8 - 16, "workspace overlaps the block scales"), (far + 3 * MB - 4080, "workspace overlaps the block scales"),
                      (far + 4 * MB, "workspace overlaps bias or residual"), (far + 5 * MB + out_bytes - 16, "workspace overlaps bias or residual")]:
        refuse(ab, "aiter_b200_gemm_a4w4_fused", mxfp4(ab, workspace=f((4096,), u8, ptr=at)), match)


def test_norm_refuses_scales_over_a_parameter(ab):
    f, far = lambda *a, **k: fake(ab, *a, **k), BASE + 32 * MB
    at = far + 8 * MB
    base = dict(out=f((M, N), torch.float8_e4m3fn, ptr=BASE), scales=f((M, N // 32), torch.uint8, ptr=at), residual_out=f((M, N), ptr=far), x=f((M, N), ptr=far + MB),
                residual=f((M, N), ptr=far + 2 * MB), weight=None, bias=None, gate=None, post_weight=None, post_bias=None, residual_scale=1.0, weight_offset=0.0,
                eps=1e-6, norm=1, post_norm=1, shuffle=0)
    for name in ("weight", "bias", "gate", "post_weight", "post_bias"):
        for p in (f((N,), ptr=at), f((N,), torch.float32, ptr=at - N * 4 + 16), f((2, N), ptr=at - 2 * N * 2 + 16)):
            refuse(ab, "aiter_b200_gated_residual_norm", list({**base, name: p}.values()), "scales overlap a parameter")
