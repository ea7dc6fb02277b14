"""GEMMs with a fused epilogue, act(A B^T + bias) + residual, against the formula in 64 bits.

Tolerance: half a step of the output type relative to the value, plus what the fp32 accumulation may lose before the epilogue.  The
tensor core adds one product group of K bytes = 32 (16 bf16, 32 e4m3, 64 e2m1 elements) per step and may truncate: at most
2^-23 of the running sum per step, which |A||B|^T bounds.  An activation passes an error on with a factor of at most 1.13 (the
gelus' steepest slope; relu 1, silu 1.1) and adds 2^-18 of the value and 2^-22 of its argument (e^x of a rounded argument)."""
import math

import pytest
import torch

from oracle import mx_oracle as ox
from tests.helpers import quant_fp4, quant_fp8, randn_bf16, to_cuda_u8

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25, torch.float32: 2.0**-149}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


def act64(x, act):
    if act == "relu":
        return x.clamp(min=0)
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu":
        return 0.5 * x * torch.erfc(-x / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)))
    return x


def check(got, a, b, steps, bias, act, residual, what=""):
    """a, b: the operands' values in 64 bits"""
    x = a @ b.t()
    lost = (a.abs() @ b.abs().t()) * (2.0**-23 * (steps + 2))
    if bias is not None:
        x = x + bias.double()
    want = act64(x, act)
    tol = 1.13 * lost + (2.0**-18 * want.abs() + 2.0**-22 * x.abs() if act not in (None, "none", "relu") else 0)
    if residual is not None:
        want = want + residual.double()
    tol = tol + (HALF_STEP[got.dtype] + 2.0**-23) * want.abs() + TINY[got.dtype] + 2.0**-23 * x.abs()
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = off > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off / tol).max()):.3g} of the tolerance, first at {bad.nonzero()[0].tolist()}"


class Problem:
    def __init__(self, ab, kind, m, n, k, seed=0):
        x, w = randn_bf16(m, k, seed + m + n + k), randn_bf16(n, k, seed + 1 + m + n + k, scale=1 / math.sqrt(k))
        self.ab, self.kind = ab, kind
        if kind == "bf16":
            self.args, self.a, self.b, self.steps = (x.cuda(), w.cuda()), x.cuda().double(), w.cuda().double(), k / 16
            self.fn, self.more = ab.gemm_a16w16_fused, {}
        elif kind == "mxfp8":
            (xq, xs), (wq, ws) = quant_fp8(x), quant_fp8(w)
            self.a, self.b = (torch.from_numpy(ox.dequant_mxfp8(q, s)).cuda().double() for q, s in ((xq, xs), (wq, ws)))
            self.args = (to_cuda_u8(xq, torch.float8_e4m3fn), ab.shuffle_mxfp8fp4_b(to_cuda_u8(wq, torch.float8_e4m3fn)), ab.shuffle_mxfp8fp4_scale(to_cuda_u8(xs)),
                         ab.shuffle_mxfp8fp4_scale(to_cuda_u8(ws)))
            self.fn, self.more, self.steps = ab.gemm_a8w8_mxfp8_fused, {"a_preshuffle": False}, k / 32
        else:
            (xq, xs), (wq, ws) = quant_fp4(x), quant_fp4(w)
            self.a, self.b = (torch.from_numpy(ox.dequant_mxfp4(q, s)).cuda().double() for q, s in ((xq, xs), (wq, ws)))
            self.args = (to_cuda_u8(xq, ab.dtypes.fp4x2), ab.shuffle_weight(to_cuda_u8(wq), layout=(16, 16)), ab.fp4_utils.e8m0_shuffle(to_cuda_u8(xs)),
                         ab.fp4_utils.e8m0_shuffle(to_cuda_u8(ws)))
            self.fn, self.more, self.steps = ab.gemm_a4w4_fused, {}, k / 64

    def run(self, **kw):
        return self.fn(*self.args, **self.more, **kw)

    def check(self, got, bias=None, activation=None, residual=None, what=""):
        check(got, self.a, self.b, self.steps, bias, activation, residual, what)


def randn(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


# every kernel variant that the library's own choice reaches: few rows (one tile, several, K split), one-CTA tiles, pairs, odd sizes
SHAPES = {
    "bf16": [(1, 128, 64), (1, 4096, 4096), (7, 40, 8), (16, 1001, 520), (33, 256, 1032), (64, 1024, 1024), (100, 512, 2048), (200, 1001, 72), (256, 4096, 512),
             (257, 64, 1024), (333, 1001, 1160), (700, 24, 128), (600, 520, 4096), (1024, 4096, 256), (4096, 1160, 192), (2100, 2056, 64),
             (1, 76, 856), (2, 4096, 1032), (3, 1001, 520), (4, 333, 8), (4, 130, 16384), (2, 5, 24), (1, 1, 8), (3, 9000, 264), (4, 2048, 2048), (5, 1024, 4096)],
    "mxfp8": [(1, 256, 128), (16, 4096, 1024), (64, 528, 512), (130, 4096, 256), (300, 1040, 384), (1024, 2048, 512), (4100, 1152, 256)],
    "mxfp4": [(1, 256, 64), (32, 7168, 512), (64, 528, 320), (200, 1024, 1024), (300, 1040, 384), (1024, 2048, 512), (4100, 1152, 4096)],
}
EPILOGUES = [
    {"activation": "silu", "bias": "bf16"},
    {"residual": "bf16"},
    {"activation": "gelu", "bias": "fp32", "residual": "fp32", "otype": "fp32"},
    {"activation": "gelu_tanh", "bias": "fp16", "residual": "fp16", "otype": "fp16"},
    {"activation": "relu", "residual": "fp32"},
    {"bias": "bf16", "residual": "bf16", "otype": "fp32"},
    {"otype": "fp32"},
]


@pytest.mark.parametrize("kind,shape", [(k, s) for k, v in SHAPES.items() for s in v], ids=lambda v: v if isinstance(v, str) else "x".join(map(str, v)))
def test_against_64_bits(ab, kind, shape):
    m, n, k = shape
    p = Problem(ab, kind, m, n, k)
    for i, e in enumerate(EPILOGUES):
        args = {"activation": e.get("activation"), "bias": randn(i, n, dtype=DT[e["bias"]]) if "bias" in e else None,
                "residual": randn(i + 9, m, n, dtype=DT[e["residual"]]) if "residual" in e else None}
        got = p.run(**args, otype=DT[e.get("otype", "bf16")])
        assert got.dtype == DT[e.get("otype", "bf16")]
        p.check(got, **args, what=f"{kind} {shape} {e}")
    assert ab.device_status(0) == (0, 0, 0, 0)


@pytest.mark.parametrize("name", ["tc5_128x64_n_s0", "tc5_128x128_n_s0", "tc5_128x192_n_s3", "tc5_128x256_n_s0", "tc5_128x96_n_s0", "tc5_128x32_n_s0", "tc5_256x128_n_s0",
                                  "tc5_256x192_n_s0", "tc5_256x256_n_s0", "tc5_128x16_t_s0_k2", "tc5_128x64_t_s0_k1", "tc5_128x128_t_s0_k2", "tc5_128x128_t_s8_k3", "tc5_128x256_t_s0",
                                  "tc5_128x128_n_s0_k4", "tc5_256x256_t_s0", "tc5_256x128_t_s0", "tc5_256x192_t_s0"])
def test_named_tiles(ab, name):
    m, n, k = (14, 1160, 1024) if "x16_t" in name else (240, 1160, 1024) if "_t_" in name else (700, 1160, 1024)
    p = Problem(ab, "bf16", m, n, k)
    for i, e in enumerate(EPILOGUES):
        args = {"activation": e.get("activation"), "bias": randn(i, n, dtype=DT[e["bias"]]) if "bias" in e else None,
                "residual": randn(i + 9, m, n, dtype=DT[e["residual"]]) if "residual" in e else None}
        p.check(p.run(**args, otype=DT[e.get("otype", "bf16")], kernelName=name), **args, what=f"{name} {e}")
    assert ab.device_status(0) == (0, 0, 0, 0)


@pytest.mark.parametrize("m", [1, 3, 5, 64, 300, 1024])
def test_strides_in_place_and_neighbours(ab, m):
    """Outputs and residuals inside wider tensors, at pitches that do and do not allow tile copies; what lies around stays as it was."""
    n, k = 528, 256
    p = Problem(ab, "bf16", m, n, k)
    for pitch, first in ((544, 8), (533, 3), (536, 4)):
        buf = torch.full((m + 2, pitch), 7.0, dtype=torch.bfloat16, device="cuda")
        view = buf[1 : m + 1, first : first + n]
        residual = randn(m, m, n)
        view.copy_(residual)
        got = p.run(activation="silu", residual=view, out=view)
        assert got is view
        p.check(got, activation="silu", residual=residual, what=f"in place, pitch {pitch}")
        view.fill_(7.0)
        assert (buf == 7).all(), "something around the output was written"
        wide = torch.full((m, pitch), 3.0, dtype=torch.float32, device="cuda")[:, first : first + n]
        wide.copy_(residual)
        p.check(p.run(residual=wide, otype=torch.float16), residual=residual, what=f"fp32 residual, pitch {pitch}")
    a3 = p.args[0].view(1, m, k)
    got = ab.gemm_a16w16_fused(a3, p.args[1], residual=residual.view(1, m, n))
    assert got.shape == (1, m, n) and torch.equal(got[0], p.run(residual=residual))


def test_torch_ops_namespace(ab):
    for kind in ("bf16", "mxfp8", "mxfp4"):
        p = Problem(ab, kind, 70, 512, 256)
        r, more = randn(1, 70, 512), [False] if kind == "mxfp8" else []
        name = {"bf16": "gemm_a16w16_fused", "mxfp8": "gemm_a8w8_mxfp8_fused", "mxfp4": "gemm_a4w4_fused"}[kind]
        got = getattr(torch.ops.aiter, name)(*p.args, None, "gelu", r, torch.float16, *more)
        assert got.dtype == torch.float16 and torch.equal(got, p.run(activation="gelu", residual=r, otype=torch.float16))


def test_shuffled_weight_and_empty_batch(ab):
    p = Problem(ab, "bf16", 40, 512, 256)
    bias = randn(1, 512)
    w = ab.shuffle_weight(p.args[1], layout=(16, 16))
    p.check(ab.gemm_a16w16_fused(p.args[0], w, bias, "relu"), bias=bias, activation="relu")
    assert ab.gemm_a16w16_fused(p.args[0][:0], p.args[1], bias, "relu").shape == (0, 512)


def test_infinities_and_nan(ab):
    m, n, k = 20, 256, 64
    for rows in (m, 300):
        a, b = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
        a[:, 0] = 1
        b[:, 0] = torch.linspace(-120, 120, n, device="cuda").bfloat16()
        r = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
        r[2, 3], r[4, 5] = float("nan"), float("-inf")
        for act in ("relu", "silu", "gelu", "gelu_tanh"):
            y = ab.gemm_a16w16_fused(a, b, activation=act, residual=r, otype=torch.float32)
            want = act64(b[:, 0].double(), act)
            assert torch.isnan(y[2, 3]) and y[4, 5] == float("-inf")
            keep = torch.ones_like(y, dtype=torch.bool)
            keep[2, 3] = keep[4, 5] = False
            off = (y.double() - want).abs()[keep]
            assert (off <= (2.0**-16 * want.abs() + 1e-30 + 2.0**-21 * b[:, 0].double().abs()).expand(rows, n)[keep]).all(), act


def test_other_stream_and_two_captured_graphs_at_once(ab):
    """Two graphs captured one after the other and replayed at the same time on two streams: they share no workspace."""
    cases = [(Problem(ab, "bf16", 4, 1024, 4096), randn(1, 4, 1024)), (Problem(ab, "bf16", 5, 1024, 4096), randn(4, 5, 1024)), (Problem(ab, "bf16", 300, 512, 8192), randn(2, 300, 512)),
             (Problem(ab, "mxfp4", 1024, 1024, 4096), randn(3, 1024, 1024))]
    for p, r in cases:
        want = p.run(activation="gelu", residual=r)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = p.run(activation="gelu", residual=r)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        graphs, outs = [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append([p.run(activation="gelu", residual=r) for _ in range(3)])
            graphs.append(g)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(4):
            with torch.cuda.stream(s1):
                graphs[0].replay()
            with torch.cuda.stream(s2):
                graphs[1].replay()
        torch.cuda.synchronize()
        for o in outs:
            for t in o:
                p.check(t, activation="gelu", residual=r, what="replayed")
        # (the captured form of a tall MXFP4 problem may take another order of additions than the eager one)
    assert ab.device_status(0) == (0, 0, 0, 0)
