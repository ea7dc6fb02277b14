"""gated_residual_norm and act_and_mul against their formulas in 64 bits; MX outputs bit for bit against the oracle's quantiser
applied to the operator's own fp32 output.

Tolerance of a value stored in type t: half a step of t relative to the value (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) plus what the
fp32 arithmetic may lose.  A row's sum of up to n squares is a chain of at most 32 additions per thread and a tree of 10, so a
relative error of at most 42 * 2^-24 in the mean square, half of that after the square root; the other steps are about ten
roundings of 2^-24 of the largest intermediate.  Two norms in a row at most double it: 2^-17 of the row's largest intermediate
covers all of it."""
import math

import numpy as np
import pytest
import torch

from oracle import mx_oracle as ox

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25, torch.float32: 2.0**-149}  # half of the smallest step


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


def randn(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def spread(p, m):
    p = p.double()
    return p if p.dim() == 1 else p.repeat_interleave(m // p.shape[0], dim=0)


def norm64(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def ref64(x, residual=None, weight=None, bias=None, gate=None, residual_scale=1.0, post_weight=None, post_bias=None, norm="rms", eps=1e-6,
          weight_offset=0.0, post_norm=False):
    """-> (y, h, magnitude of the largest intermediate per row of y, the same of h)"""
    m = x.shape[0]
    h = x.double()
    big = h.abs()
    if post_norm or post_weight is not None or post_bias is not None:
        h = norm64(h, norm, eps)
        if post_weight is not None:
            h = h * post_weight.double() if post_weight.dim() == 1 else h * spread(post_weight, m)
        big = h.abs()
        if post_bias is not None:
            h = h + spread(post_bias, m)
            big = big + spread(post_bias, m).abs()
    if gate is not None:
        h = h * spread(gate, m)
        big = big * spread(gate, m).abs()
    if residual is not None:
        h = residual_scale * residual.double() + h
        big = big + (residual_scale * residual.double()).abs()
    big_h = big.amax(-1, keepdim=True)
    rms = torch.sqrt(((h - h.mean(-1, keepdim=True) if norm == "layer" else h) ** 2).mean(-1, keepdim=True) + eps)
    y = norm64(h, norm, eps)
    big_y = big_h / rms
    if weight is not None:
        w = weight_offset + spread(weight, m)
        y, big_y = y * w, big_y * w.abs().amax(-1, keepdim=True)
    if bias is not None:
        y, big_y = y + spread(bias, m), big_y + spread(bias, m).abs().amax(-1, keepdim=True)
    return y, h, big_y, big_h


def check(got, want, big, what):
    tol = HALF_STEP[got.dtype] * want.abs() + TINY[got.dtype] + 2.0**-17 * big
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = off > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst by {float((off / tol).max()):.3g} of the tolerance, first at {bad.nonzero()[0].tolist()}"


CASES = [
    # m, n, x, residual, options
    (1, 4096, "bf16", "bf16", {}),
    (5, 8, "bf16", None, {}),
    (3, 1, "fp32", "fp32", {"gate": "channel"}),
    (37, 33, "fp16", "fp32", {"norm": "layer", "bias": True}),
    (130, 1155, "bf16", "fp32", {"norm": "layer", "bias": True, "gate": "sample2", "affine": "sample2", "offset": 1.0}),
    (64, 1000, "fp32", "bf16", {"post": True, "gate": "channel"}),
    (6, 2048, "bf16", "bf16", {"post": True, "post_bias": True, "norm": "layer", "gate": "token", "scale": 0.5}),
    (700, 7168, "bf16", "bf16", {"scale": 1.25}),
    (300, 8192, "fp16", "fp16", {"post": True, "gate": "sample3"}),
    (2, 16384, "fp32", "fp32", {"post": True}),
    (310, 12288, "bf16", "fp32", {"gate": "token"}),
    (3, 16392, "bf16", "bf16", {"post": True, "norm": "layer", "bias": True, "gate": "channel"}),
    (2, 20001, "fp16", "fp32", {"post": True, "norm": "layer", "post_bias": True}),
    (4, 2051, "bf16", None, {"gate": "channel"}),
    (9, 16383, "bf16", "bf16", {"norm": "layer"}),
    # rows on any element's address, types that differ
    (29, 9371, "bf16", "fp32", {"post": True, "gate": "token"}),
    (6, 3075, "bf16", "fp32", {"affine": "sample3", "bias": True}),
    (400, 5287, "fp32", "bf16", {"gate": "token", "affine": "sample2", "bias": True, "norm": "layer"}),
    (600, 1571, "fp32", "fp16", {"norm": "layer", "gate": "channel16", "scale": 1.25, "post": True, "post_bias": True}),
    (350, 8203, "bf16", "fp16", {"norm": "layer", "post": True}),
    (2, 16377, "fp32", "bf16", {"gate": "channel"}),
    (5, 7, "fp16", "bf16", {"norm": "layer", "bias": True}),
    (2001, 37, "bf16", "fp32", {"norm": "layer", "bias": True, "post": True}),
    (1003, 99, "fp32", "bf16", {"post": True, "post_bias": True, "gate": "token"}),
    (4800, 1155, "bf16", "fp32", {"norm": "layer", "affine": "sample4", "offset": 1.0, "bias": True, "gate": "sample4", "post": True}),
    (700, 8000, "bf16", "bf16", {"post": True, "norm": "layer"}),
    (3, 8190, "bf16", "bf16", {"post": True, "post_bias": True}),
    # many rows: the streaming kernels, aligned and not, every width class
    (1200, 64, "bf16", "bf16", {"post": True, "gate": "channel16"}),
    (999, 40, "fp16", "fp32", {"norm": "layer", "bias": True, "gate": "token"}),
    (3001, 128, "bf16", "fp32", {"norm": "layer", "bias": True, "post": True, "post_bias": True}),
    (640, 256, "fp32", "fp32", {"gate": "sample4", "affine": "sample4", "offset": 1.0, "bias": True}),
    (600, 200, "bf16", None, {"gate": "channel16", "scale": 0.5}),
    (500, 328, "bf16", "bf16", {"post": True, "gate": "token16"}),
    (444, 1152, "bf16", "fp32", {"norm": "layer", "affine": "sample4", "offset": 1.0, "bias": True, "gate": "sample4", "post": True}),
    (400, 1155, "bf16", "fp32", {"norm": "layer", "affine": "sample4", "offset": 1.0, "bias": True, "gate": "sample4", "post": True, "post_bias": True}),
    (500, 101, "fp16", "fp16", {"post": True, "norm": "layer", "post_bias": True}),
    (350, 8191, "bf16", "bf16", {"post": True, "norm": "layer"}),
    (333, 4098, "fp32", "fp32", {}),
    (300, 16384, "fp16", "fp32", {"post": True, "gate": "token"}),
    (299, 12296, "bf16", "bf16", {"norm": "layer", "bias": True, "post": True}),
    (450, 8192, "bf16", "bf16", {"post": True, "gate": "channel16", "scale": 0.5, "post_bias": True}),
    (310, 9001, "bf16", "bf16", {"post": True}),
    (400, 512, "bf16", "fp16", {"gate": "channel"}),
    (700, 4096, "fp32", "bf16", {"post": True, "gate": "channel16"}),
    (5000, 128, "fp32", "fp16", {"norm": "layer", "bias": True}),
    (444, 1152, "fp32", "fp16", {"gate": "token", "scale": 0.5}),
    (6400, 1001, "fp32", "bf16", {"norm": "layer", "affine": "sample4", "offset": 1.0, "gate": "sample4", "bias": True}),
    (320, 12288, "fp32", "bf16", {"post": True, "post_bias": True}),
    (1300, 7001, "fp16", "fp32", {"post": True, "norm": "layer", "post_bias": True, "bias": True}),
    (6400, 1001, "fp32", "fp32", {"gate": "token", "affine": "sample4", "offset": 1.0}),
    (10000, 513, "bf16", "bf16", {"norm": "layer", "gate": "sample4", "post": True, "scale": 0.5}),
    (16400, 257, "bf16", None, {"gate": "channel", "bias": True}),
    (1300, 7999, "bf16", "bf16", {"post": True, "gate": "channel16"}),
]
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(case, seed=0):
    m, n, x, residual, o = case
    g = torch.Generator().manual_seed(seed + m * 131 + n)

    def param(kind):
        if kind == "channel":
            return randn(g, n, dtype=torch.float32, scale=0.5)
        if kind == "channel16":  # of x's own type, like the other parameters
            return randn(g, n, dtype=DT[x], scale=0.5)
        if kind.startswith("token"):
            return randn(g, m, 1, dtype=torch.bfloat16)
        return randn(g, int(kind[6:]), n, dtype=torch.float16 if m < 296 else DT[x], scale=0.5)

    args = {"x": randn(g, m, n, dtype=DT[x], scale=2.0) + 0.25, "norm": o.get("norm", "rms"), "eps": 1e-5,
            "residual_scale": o.get("scale", 1.0), "weight_offset": o.get("offset", 0.0)}
    if residual:
        args["residual"] = randn(g, m, n, dtype=DT[residual], scale=3.0)
    few = m < 296  # few rows: parameters of several types; many: of x's, as the streaming kernels want them
    args["weight"] = param(o["affine"]) if "affine" in o else randn(g, n, dtype=torch.bfloat16 if few else DT[x])
    if o.get("bias"):
        args["bias"] = param(o["affine"]) if "affine" in o else randn(g, n, dtype=torch.float32 if few else DT[x])
    if "gate" in o:
        args["gate"] = param(o["gate"])
    if o.get("post"):
        args["post_weight"] = randn(g, n, dtype=torch.bfloat16 if few else DT[x])
        if o.get("post_bias"):
            args["post_bias"] = randn(g, n, dtype=torch.bfloat16 if few else DT[x])
    return args


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}-{c[2]}")
@pytest.mark.parametrize("otype", ["bf16", "fp16", "fp32"])
def test_norm_against_64_bits(ab, case, otype):
    args = make(case)
    y, h = ab.gated_residual_norm(**args, otype=DT[otype])
    ry, rh, big_y, big_h = ref64(**args)
    assert y.dtype == DT[otype] and h.dtype == (args["residual"] if "residual" in args else args["x"]).dtype
    check(y, ry, big_y, "y")
    check(h, rh, big_h, "h")


def test_norm_without_anything_returns_x(ab):
    x = randn(torch.Generator().manual_seed(1), 4, 256)
    y, h = ab.gated_residual_norm(x)
    assert h is x
    ry, _, big, _ = ref64(x)
    check(y, ry, big, "y")
    y2, h2 = ab.gated_residual_norm(x, post_norm=True)
    ry2, rh2, b1, b2 = ref64(x, post_norm=True)
    check(y2, ry2, b1, "y"), check(h2, rh2, b2, "h")


def test_norm_strides_leading_dimensions_and_in_place(ab):
    g = torch.Generator().manual_seed(2)
    wide = randn(g, 3, 5, 3 * 264)
    x, residual, spare = wide[..., :264], wide[..., 264:528], wide[..., 528:].clone()
    mod = randn(g, 3, 2 * 264)  # a strided modulation tensor: one entry per sample, rows of 528
    w = randn(g, 264)
    want = ref64(x.reshape(15, 264), residual.reshape(15, 264), w, gate=mod[:, 264:].contiguous())
    y, h = ab.gated_residual_norm(x, residual, w, gate=mod[:, 264:])
    assert y.shape == x.shape and h.shape == x.shape
    check(y.view(15, 264), want[0], want[2], "y"), check(h.view(15, 264), want[1], want[3], "h")
    # updated in place, inside a wider tensor whose other columns stay as they were
    x2, r2 = x.reshape(15, 264), torch.empty(15, 400, dtype=torch.bfloat16, device="cuda").fill_(7.0)
    r2[:, 8:272] = residual.reshape(15, 264)
    y2, h2 = ab.gated_residual_norm(x2, r2[:, 8:272], w, gate=mod[:, 264:], residual_out=r2[:, 8:272])
    assert torch.equal(y2, y.view(15, 264)) and torch.equal(h2, h.view(15, 264)) and torch.equal(r2[:, 8:272], h2)
    assert (r2[:, :8] == 7).all() and (r2[:, 272:] == 7).all()
    assert torch.equal(wide[..., 528:], spare)
    # rows that start on no 16-byte boundary (shifted groups): same values up to the order of the sums
    x3 = torch.empty(15, 271, dtype=torch.bfloat16, device="cuda")[:, 3:267]
    x3.copy_(x2)
    y3, _ = ab.gated_residual_norm(x3, residual.reshape(15, 264), w, gate=mod[:, 264:])
    check(y3, want[0], want[2], "y unaligned")


@pytest.mark.parametrize("m,n", [(1, 32), (33, 320), (300, 1024), (65, 7168), (700, 2176), (2, 20480), (1001, 32), (777, 128), (545, 224), (301, 416), (333, 8192), (297, 9216)])
@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("layout", [False, True, 2])
def test_norm_mx_output_is_the_quantised_fp32_output(ab, m, n, fp4, layout):
    if layout == 2 and n % 128:
        pytest.skip("the (m/32,k/4,32,4) order needs a multiple of 128 columns")
    g = torch.Generator().manual_seed(m + n)
    x = randn(g, m, n) * torch.exp2(torch.randint(-8, 8, (m, 1), generator=g).float()).cuda().bfloat16()
    x[0, :32] = 0  # a block of zeros
    r, w = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda"), randn(g, n)
    y32, h0 = ab.gated_residual_norm(x, r, w, otype=torch.float32)
    y, s, h = ab.gated_residual_norm(x, r, w, quant_dtype=ab.dtypes.fp4x2 if fp4 else ab.dtypes.fp8, shuffle=layout)
    assert torch.equal(h, h0)
    check_mx(ab, y, s, y32, m, n, fp4, layout)


def check_mx(ab, y, s, y32, m, n, fp4, layout):
    q, b = (ox.quant_mxfp4 if fp4 else ox.quant_mxfp8)(y32.cpu().numpy())
    assert np.array_equal(y.view(torch.uint8).cpu().numpy(), q)
    got = s.view(torch.uint8).cpu().numpy()
    if layout is False:
        assert got.shape == b.shape and np.array_equal(got, b)
    elif layout == 2:
        assert np.array_equal(got.reshape(-1), np.asarray(ox.shuffle_mxfp8fp4_scale(b)).reshape(-1))
    else:
        rows = (m + 31) // 32 * 32  # the last group of 32 rows is filled up; rows behind it belong to nobody
        want = np.asarray(ox.e8m0_shuffle(b)).reshape(-1)
        assert got.shape == ((m + 255) // 256 * 256, (n // 32 + 7) // 8 * 8)
        assert np.array_equal(got.reshape(-1)[: rows * got.shape[1]], want[: rows * got.shape[1]])


def test_norm_nan_and_infinity_stay_in_their_rows(ab):
    g = torch.Generator().manual_seed(3)
    x = randn(g, 6, 512)
    clean = ab.gated_residual_norm(x, x)[0]
    x2 = x.clone()
    x2[1, 7], x2[3, 100], x2[4] = float("nan"), float("inf"), 0
    y, h = ab.gated_residual_norm(x2, x2)
    for r in (0, 2, 5):
        assert torch.equal(y[r], clean[r])
    assert torch.isnan(y[1]).all() and (y[4] == 0).all()
    assert torch.isinf(h[3, 100])
    q, s, _ = ab.gated_residual_norm(x2, x2, quant_dtype=ab.dtypes.fp8)
    assert (s.view(torch.uint8)[1] == 255).all() and (s.view(torch.uint8)[4] == 0).all() and (s.view(torch.uint8)[0] < 255).all()


@pytest.mark.parametrize("m,n", [(1, 1), (16, 9216), (333, 1001), (7, 8), (2050, 264), (1, 40001)])
@pytest.mark.parametrize("x", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_act_and_mul_against_64_bits(ab, m, n, x, act):
    g = torch.Generator().manual_seed(m + n)
    v = randn(g, m, 2 * n, dtype=DT[x], scale=3.0)
    a = act64(v[:, :n].double(), act)
    want = a * v[:, n:].double()
    for otype in (DT[x], torch.float32):
        y = ab.act_and_mul(v, act, otype=otype)
        # e^x carries |x| 2^-24 from its scaled argument: 2^-18 of the product covers |x| up to 30 and the other roundings;
        # the gelus add an absolute 2^-22 |x| from 1 + erf, 1 + tanh
        tol = HALF_STEP[otype] * want.abs() + TINY[otype] + 2.0**-18 * want.abs() + 2.0**-22 * (v[:, :n].double() * v[:, n:].double()).abs()
        assert ((y.double() - want).abs() <= tol).all()


def act64(x, act):
    if act == "relu":
        return x.clamp(min=0)
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu":
        return 0.5 * x * torch.erfc(-x / math.sqrt(2))
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)))


@pytest.mark.parametrize("m,n", [(1, 32), (33, 320), (300, 1024), (65, 2176)])
@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("layout", [False, True, 2])
@pytest.mark.parametrize("x", ["bf16", "fp32"])
def test_act_mx_output_is_the_quantised_fp32_output(ab, m, n, fp4, layout, x):
    if layout == 2 and n % 128:
        pytest.skip("the (m/32,k/4,32,4) order needs a multiple of 128 columns")
    g = torch.Generator().manual_seed(m + n)
    v = randn(g, m, 2 * n, dtype=DT[x], scale=2.0)
    v[0, :32] = 0
    y32 = ab.act_and_mul(v, "silu", otype=torch.float32)
    y, s = ab.act_and_mul(v, "silu", quant_dtype=ab.dtypes.fp4x2 if fp4 else ab.dtypes.fp8, shuffle=layout)
    check_mx(ab, y, s, y32, m, n, fp4, layout)


def test_act_extremes_in_place_and_out_forms(ab):
    x = torch.tensor([[-1e4, -90.0, -0.0, 0.0, 30.0, 1e4, float("inf"), float("nan"), 2.0, 2.0, 2.0, 2.0, 2.0, 2.0, 2.0, 2.0]], device="cuda")
    for act in ("silu", "gelu", "gelu_tanh", "relu"):
        y = ab.act_and_mul(x, act)[0]
        assert y[0] == 0 and y[2] == 0 and y[3] == 0 and y[4] == 60 and y[5] == 2e4 and torch.isinf(y[6]) and torch.isnan(y[7]), (act, y)
        assert abs(float(y[1])) < 1e-30
    v = randn(torch.Generator().manual_seed(4), 9, 2 * 136)
    want = ab.act_and_mul(v, "gelu_tanh")
    out = torch.empty(9, 136, dtype=torch.bfloat16, device="cuda")
    ab.gelu_tanh_and_mul(out, v)
    assert torch.equal(out, want)
    ab.gelu_and_mul(out, v)
    assert torch.equal(out, ab.act_and_mul(v, "gelu"))
    keep = v.clone()
    ab.silu_and_mul(v[:, :136], v)  # over its own gate half
    assert torch.equal(v[:, :136], ab.act_and_mul(keep)) and torch.equal(v[:, 136:], keep[:, 136:])


def test_empty_batches(ab):
    x = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
    y, h = ab.gated_residual_norm(x, x)
    assert y.shape == h.shape == (0, 256)
    y, s, _ = ab.gated_residual_norm(x, x, quant_dtype=ab.dtypes.fp8, shuffle=2)
    assert y.shape == (0, 256)
    assert ab.act_and_mul(x).shape == (0, 128)


def test_other_stream_and_captured_graphs(ab):
    g = torch.Generator().manual_seed(5)
    x, r, w = randn(g, 64, 1024), randn(g, 64, 1024), randn(g, 1024)
    want = ab.gated_residual_norm(x, r, w)
    want_a = ab.act_and_mul(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_a = ab.gated_residual_norm(x, r, w), ab.act_and_mul(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got_a, want_a)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append((*ab.gated_residual_norm(x, r, w), ab.act_and_mul(x)))
        graphs.append(gr)
    x.copy_(randn(g, 64, 1024))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
    torch.cuda.synchronize()
    want = (*ab.gated_residual_norm(x, r, w), ab.act_and_mul(x))
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.parametrize("fp4", [False, True])
def test_mx_scale_of_every_magnitude(ab, fp4):
    """Blocks whose largest value runs through every exponent and the significands around the step of the scale, denormals, zero,
    infinity and NaN among them: bytes and elements as the oracle's division gives them."""
    tops = []
    for e in range(-149, 128):
        for mant in (1.0, 1.5 - 2.0**-23, 1.5, 1.5 + 2.0**-23, 1.75 - 2.0**-23, 1.75, 1.75 + 2.0**-23, 2.0 - 2.0**-23):
            tops.append(math.ldexp(mant, e))
    tops += [0.0, float("inf"), float("nan")]
    top = np.array(tops, dtype=np.float64)
    top = top[~(np.abs(top) > 3.4028234663852886e38) | np.isinf(top)].astype(np.float32)
    rows = len(top)
    # (the factor half is ones: the product is relu of the gate half, x < 0 ? 0 : x, which keeps the sign of a zero)
    x = np.concatenate([np.tile(top[:, None] * np.float32(1), (1, 32)) * np.linspace(1.0, -0.9, 32, dtype=np.float32)[None, :], np.ones((rows, 32), np.float32)], axis=1)
    x[:, 0] = top
    with np.errstate(all="ignore"):
        want_q, want_s = (ox.quant_mxfp4 if fp4 else ox.quant_mxfp8)(np.where(x[:, :32] < 0, np.float32(0), x[:, :32]))
    y, s = ab.act_and_mul(torch.from_numpy(x).cuda(), "relu", quant_dtype=ab.dtypes.fp4x2 if fp4 else ab.dtypes.fp8)
    assert np.array_equal(s.view(torch.uint8).cpu().numpy(), want_s)
    finite = np.isfinite(top)
    assert np.array_equal(y.view(torch.uint8).cpu().numpy()[finite], want_q[finite])
