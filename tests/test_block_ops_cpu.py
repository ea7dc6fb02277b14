"""Refusals of the operators between two GEMMs, without a GPU: descriptors that claim device memory are checked, and refused,
before anything is launched."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


BASE = 1 << 40  # an address that nothing dereferences


def fake(ab, shape, dtype=torch.bfloat16, strides=None, ptr=BASE, device=0):
    t = ab._ffi.aiter_tensor_t()
    if strides is None:
        strides, acc = [], 1
        for s in reversed(shape):
            strides.insert(0, acc)
            acc *= s
    t.ptr, t.ndim, t.dtype_, t.device_id = ptr, len(shape), ab.dtypes.aiter_dtype_id(dtype), device
    t.numel_ = 1
    for i, s in enumerate(shape):
        t.shape[i], t.strides[i] = s, strides[i]
        t.numel_ *= s
    return t


def refuse(ab, name, args, match):
    lib = ab._ffi._lib
    cargs = []
    for a in args:
        if isinstance(a, float):
            cargs.append(ctypes.c_float(a))
        elif isinstance(a, int):
            cargs.append(ctypes.c_int(a))
        else:
            cargs.append(None if a is None else ctypes.byref(a))
    assert getattr(lib, name)(*cargs, None) == -1
    msg = lib.aiter_get_last_error().decode()
    assert match in msg, msg


M, N = 4, 256


def norm_args(ab, **over):
    a = {"out": fake(ab, (M, N), ptr=BASE), "scales": None, "residual_out": fake(ab, (M, N), ptr=BASE + (1 << 20)), "x": fake(ab, (M, N), ptr=BASE + (2 << 20)),
         "residual": fake(ab, (M, N), ptr=BASE + (3 << 20)), "weight": fake(ab, (N,), ptr=BASE + (4 << 20)), "bias": None, "gate": None, "post_weight": None,
         "post_bias": None, "residual_scale": 1.0, "weight_offset": 0.0, "eps": 1e-6, "norm": 0, "post_norm": 0, "shuffle": 0}
    assert set(over) <= set(a)
    a.update(over)
    return list(a.values())


def test_norm_refusals(ab):
    name, f = "aiter_b200_gated_residual_norm", lambda *a, **k: fake(ab, *a, **k)
    far = BASE + (9 << 20)
    cases = [
        ({"norm": 2}, "norm must be 0"),
        ({"x": f((M, N), torch.int32, ptr=far)}, "x must be bf16, fp16 or fp32"),
        ({"x": f((M, N), ptr=far, device=-1)}, "must live on a GPU"),
        ({"residual": f((M, N + 1), ptr=far)}, "residual must be [4, 256]"),
        ({"residual": f((M, N), ptr=far, device=1)}, "lives on device 1"),
        ({"residual": f((M, N), strides=(1, M), ptr=far)}, "contiguous along its last dimension"),
        ({"weight": f((N - 1,), ptr=far)}, "weight must have 256 columns"),
        ({"weight": f((3, N), ptr=far)}, "3 entries, which do not divide 4 rows"),
        ({"weight": f((2, 1), ptr=far)}, "weight must have 256 columns"),
        ({"gate": f((3, 1), ptr=far)}, "3 entries, which do not divide 4 rows"),
        ({"gate": f((2, 2, N), ptr=far)}, "gate must be 2-D"),
        ({"post_weight": f((N,), ptr=far)}, "go with the first norm only"),
        ({"scales": f((M, N // 32), torch.uint8, ptr=far)}, "scales go with an MX output only"),
        ({"out": f((M, N), torch.float8_e4m3fn)}, "scales is required"),
        ({"out": f((M, N), torch.float8_e4m3fn), "scales": f((M, N // 32), torch.uint8, ptr=far), "shuffle": 3}, "shuffle_scale must be 0"),
        ({"out": f((M, N), torch.float8_e4m3fn), "scales": f((M, N // 32), torch.uint8, ptr=far), "shuffle": 1}, "pad32(M), pad8(n/32)"),
        ({"out": f((M, N), torch.float8_e4m3fn), "scales": f((M, N // 32), torch.uint8, ptr=far), "shuffle": 2}, "pad32(M), n/32"),
        ({"out": f((M, N), torch.float8_e4m3fn), "scales": f((M, N // 32), torch.float32, ptr=far)}, "scales must be e8m0"),
        ({"out": f((M, N), torch.float8_e4m3fn), "scales": f((M, N // 32), torch.uint8, ptr=far), "x": f((M, N), ptr=far + 2 + (1 << 20))}, "16-byte boundary"),
        ({"out": f((M, N // 2 + 1), torch.uint8), "scales": f((M, N // 32), torch.uint8, ptr=far)}, "out must be [M, n/2]"),
        ({"out": f((M, N), ptr=BASE + (1 << 20) + 64)}, "residual_out overlaps out"),
        ({"out": f((M, N), ptr=BASE + (2 << 20) + 64)}, "out overlaps x"),
        ({"out": f((M, N), ptr=BASE + (3 << 20) + 64)}, "out overlaps residual"),
        ({"residual_out": f((M, N), ptr=BASE + (3 << 20) - 16)}, "residual_out overlaps residual"),
        ({"residual_out": f((M, N), torch.float16, ptr=BASE + (3 << 20))}, "residual_out overlaps residual"),
        ({"residual_out": f((M, N), strides=(0, 1), ptr=far)}, "rows of residual_out overlap"),
        ({"out": f((M, N), strides=(N - 8, 1))}, "rows of out overlap"),
        ({"residual": f((M, N), ptr=far + 1)}, "residual does not start on an element's boundary"),
        ({"residual": f((M, N), strides=(-N, 1), ptr=far)}, "negative stride"),
        ({"weight": f((N,), torch.float32, ptr=far + 2)}, "weight does not start on an element's boundary"),
        ({"weight": f((N,), ptr=BASE + 64)}, "overlaps a parameter"),
    ]
    for over, match in cases:
        refuse(ab, name, norm_args(ab, **over), match)
    # (the zero-width row of x)
    refuse(ab, name, norm_args(ab, x=f((M, 0), ptr=far)), "at least one column")


def test_act_refusals(ab):
    name, f = "aiter_b200_act_and_mul", lambda *a, **k: fake(ab, *a, **k)
    far = BASE + (9 << 20)
    x = f((M, 2 * N), ptr=far)
    for args, match in [
        ([f((M, N)), None, f((M, 2 * N + 1), ptr=far), 2, 0], "even number of columns"),
        ([f((M, N)), None, x, 0, 0], "activation must be 1"),
        ([f((M, N)), None, x, 5, 0], "activation must be 1"),
        ([f((M, N + 8)), None, x, 2, 0], "out must be [4, 256]"),
        ([f((M, N), torch.int8), None, x, 2, 0], "out must be bf16, fp16 or fp32"),
        ([f((M, N), device=1), None, x, 2, 0], "lives on device 1"),
        ([f((M, N), strides=(2 * N, 1), ptr=far + 2 * N), None, x, 2, 0], "overlaps the input"),
        ([f((M, N), torch.float8_e4m3fn), None, x, 2, 0], "scales is required"),
        ([f((M, 48), torch.float8_e4m3fn), f((M, 2), torch.uint8, ptr=far + (1 << 20)), f((M, 96), ptr=far), 2, 0], "multiple of 32 columns"),
        ([f((M, N), torch.float8_e4m3fn), f((M, N // 32), torch.uint8, ptr=far + (1 << 20)), f((M, 2 * N), strides=(2 * N + 4, 1), ptr=far), 2, 0], "16-byte boundaries"),
    ]:
        refuse(ab, name, args, match)


def test_fused_gemm_refusals(ab):
    K, far = 128, BASE + (9 << 20)
    f = lambda *a, **k: fake(ab, *a, **k)  # noqa: E731
    A, B, out, bias, res = (f((M, K), ptr=BASE), f((N, K), ptr=BASE + (1 << 20)), f((M, N), ptr=BASE + (2 << 20)), f((N,), ptr=BASE + (3 << 20)), f((M, N), ptr=BASE + (4 << 20)))
    base = dict(A=A, B=B, bias=bias, residual=res, out=out, activation=2, bpreshuffle=0, name=None)
    for over, match in [
        (dict(activation=5), "activation must be 0"),
        (dict(activation=-1), "activation must be 0"),
        (dict(out=f((M, N + 1), ptr=far)), "out must be [M, N]"),
        (dict(out=f((M, N), torch.int32, ptr=far)), "unsupported output dtype"),
        (dict(out=f((M, N), strides=(N // 2, 1), ptr=far)), "rows of out overlap"),
        (dict(bias=f((N + 1,), ptr=far)), "bias must be [256]"),
        (dict(bias=f((1, N), ptr=far)), "bias must be 1-D"),
        (dict(bias=f((N,), strides=(2,), ptr=far)), "contiguous along its last dimension"),
        (dict(bias=f((N,), torch.int8, ptr=far)), "bias must be bf16, fp16 or fp32"),
        (dict(residual=f((M + 1, N), ptr=far)), "residual must be [4, 256]"),
        (dict(residual=f((M, N), strides=(1, M), ptr=far)), "contiguous along its last dimension"),
        (dict(residual=f((M, N), ptr=BASE + (2 << 20) + 2 * N)), "out overlaps residual"),
        (dict(residual=f((M, N), torch.float16, ptr=BASE + (2 << 20))), "out overlaps residual"),
        (dict(residual=f((M, N), ptr=far, device=2)), "lives on device 2"),
        (dict(B=f((N, K + 8), ptr=far)), "disagree on K"),
        (dict(out=f((M, N), ptr=BASE + 256)), "out overlaps an operand"),
        (dict(out=f((M, N), ptr=BASE + (1 << 20))), "out overlaps an operand"),
        (dict(bias=f((N,), ptr=BASE + (2 << 20) + 32)), "out overlaps bias"),
        (dict(out=f((M, N), torch.float32, ptr=far + 2)), "out does not start on an element's boundary"),
        (dict(B=f((N, K), ptr=far, device=1)), "lives on device 1"),
        (dict(A=f((M, K), torch.float16, ptr=far)), "only bf16 inputs"),
        (dict(A=f((M, K), ptr=far, device=-1)), "must live on a GPU"),
        (dict(bpreshuffle=1, B=f((N, K), strides=(K + 8, 1), ptr=far)), "shuffled weight must be contiguous"),
    ]:
        args = {**base, **over}
        refuse(ab, "aiter_b200_gemm_a16w16_fused", list(args.values()), match)
    q, s32 = torch.float8_e4m3fn, f((32, K // 32), torch.uint8, ptr=BASE + (5 << 20))
    sb = f((N, K // 32), torch.uint8, ptr=BASE + (6 << 20))
    for args, match in [
        ([f((M, K), q), f((N, K), q, ptr=far), s32, sb, f((N, 1), ptr=far), None, out, 0, 0, None], "bias must be 1-D"),
        ([f((M, K), q), f((N, K), q, ptr=far), s32, f((N, K // 32), torch.uint8, ptr=far, device=1), None, None, out, 0, 0, None], "lives on device 1"),
        ([f((M, K), q), f((N, K), q, ptr=far), s32, sb, None, None, out, 7, 0, None], "activation must be 0"),
        ([f((M, 96), q), f((N, 96), q, ptr=far), s32, sb, None, None, out, 0, 0, None], "K must be divisible by 128"),
    ]:
        refuse(ab, "aiter_b200_gemm_a8w8_mxfp8_fused", args, match)
    a4, b4 = f((M, K // 2), torch.uint8), f((N, K // 2), torch.uint8, ptr=far)
    s4 = f((256, 8), torch.uint8, ptr=BASE + (7 << 20))
    for ws, match in [(f((16,), torch.float32, ptr=far + (1 << 20)), "workspace must be a uint8"), (f((4, 4), torch.uint8, ptr=far + (1 << 20)), "workspace must be 1-D"),
                      (f((16,), torch.uint8, ptr=far + 8), "workspace must be 16-byte aligned"), (f((16,), torch.uint8, ptr=far, device=3), "lives on device 3")]:
        refuse(ab, "aiter_b200_gemm_a4w4_fused", [a4, b4, s4, s4, None, None, out, ws, 0, 1, None], match)
    # workspace is asked for where the scales are re-laid: tall problems with a long K
    workspace = ab._ffi._lib.aiter_b200_gemm_a4w4_fused_workspace
    assert workspace(64, 4096, 4096) == 0 and workspace(4096, 4096, 4096) == (128 + 128) * 32 * 128
    with pytest.raises(ValueError, match="unknown activation"):
        ab.gemm_a16w16_fused(torch.zeros(4, 64), torch.zeros(8, 64), activation="swish")
    with pytest.raises(ValueError, match="residual must be"):
        ab.gemm_a16w16_fused(torch.zeros(4, 64), torch.zeros(8, 64), residual=torch.zeros(4, 9))
    with pytest.raises(ValueError, match="out must be"):
        ab.gemm_a16w16_fused(torch.zeros(4, 64), torch.zeros(8, 64), out=torch.zeros(5, 8))
    with pytest.raises(RuntimeError, match="must live on a GPU"):
        ab.gemm_a16w16_fused(torch.zeros(4, 64).bfloat16(), torch.zeros(8, 64).bfloat16())


def test_python_refusals(ab):
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="unknown norm"):
        ab.gated_residual_norm(x, norm="batch")
    with pytest.raises(ValueError, match="multiple of 32"):
        ab.gated_residual_norm(x[:, :40], quant_dtype=ab.dtypes.fp8)
    with pytest.raises(ValueError, match="exclude one another"):
        ab.gated_residual_norm(x, quant_dtype=ab.dtypes.fp8, otype=torch.bfloat16)
    with pytest.raises(ValueError, match="residual_out must have x's shape"):
        ab.gated_residual_norm(x, x, residual_out=x[:2])
    with pytest.raises(ValueError, match="unsupported quant_dtype"):
        ab.act_and_mul(x, quant_dtype=torch.int8)
    with pytest.raises(ValueError, match="unknown activation"):
        ab.act_and_mul(x, "swish")
    with pytest.raises(ValueError, match="an activation is required"):
        ab.act_and_mul(x, "none")
    with pytest.raises(ValueError, match="must be even"):
        ab.act_and_mul(x[:, :63])
    with pytest.raises(RuntimeError, match="must live on a GPU"):
        ab.gated_residual_norm(x, x)


def test_fused_gemms_trace_on_the_meta_device(ab):
    e = lambda *s, t=torch.bfloat16: torch.empty(*s, dtype=t, device="meta")  # noqa: E731
    o = torch.ops.aiter.gemm_a16w16_fused(e(2, 7, 32), e(48, 32), e(48), "gelu", e(2, 7, 48))
    assert o.shape == (2, 7, 48) and o.dtype == torch.bfloat16
    assert torch.ops.aiter.gemm_a16w16_fused(e(7, 32), e(48, 32), otype=torch.float32).dtype == torch.float32
    q, s = e(64, 128, t=torch.float8_e4m3fn), e(64, 4, t=torch.uint8)
    assert torch.ops.aiter.gemm_a8w8_mxfp8_fused(q, q, s, s, None, "silu", None, torch.float16).dtype == torch.float16
    p = e(64, 64, t=torch.uint8)
    assert torch.ops.aiter.gemm_a4w4_fused(p, p, s, s).shape == (64, 64)
