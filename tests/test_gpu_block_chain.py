"""The operators of a block in a row, as a layer runs them: norm with gate and residual sum -> GEMM -> gated activation -> GEMM with the
residual in its epilogue -> the next norm.  Every step is checked against its formula in 64 bits on what the step before it left (the
tolerances of the single operators); an MX operand goes from the operator that makes it to the GEMM untouched."""
import math

import pytest
import torch

from oracle import mx_oracle as ox
from tests.helpers import quant_fp4, quant_fp8, randn_bf16, to_cuda_u8
from tests.test_gpu_block_ops import check as check_values, randn, ref64
from tests.test_gpu_gemm_fused import act64, check as check_gemm

pytestmark = pytest.mark.gpu

D, HIDDEN = 512, 384
STEP = {"bf16": 16, "mxfp8": 32, "mxfp4": 64}  # elements of one product group of the tensor core


@pytest.fixture(scope="module")
def ab():
    import aiter_b200

    return aiter_b200


class Weight:
    def __init__(self, ab, kind, n, k, seed):
        self.ab, self.kind = ab, kind
        w = randn_bf16(n, k, seed, scale=1 / math.sqrt(k))
        if kind == "bf16":
            self.w, self.value = w.cuda(), w.cuda().double()
        elif kind == "mxfp8":
            q, s = quant_fp8(w)
            self.value = torch.from_numpy(ox.dequant_mxfp8(q, s)).cuda().double()
            self.w, self.s = ab.shuffle_mxfp8fp4_b(to_cuda_u8(q, torch.float8_e4m3fn)), ab.shuffle_mxfp8fp4_scale(to_cuda_u8(s))
        else:
            q, s = quant_fp4(w)
            self.value = torch.from_numpy(ox.dequant_mxfp4(q, s)).cuda().double()
            self.w, self.s = ab.shuffle_weight(to_cuda_u8(q), layout=(16, 16)), ab.fp4_utils.e8m0_shuffle(to_cuda_u8(s))

    def __call__(self, a, **kw):
        if self.kind == "bf16":
            return self.ab.gemm_a16w16_fused(a[0], self.w, **kw)
        if self.kind == "mxfp8":
            return self.ab.gemm_a8w8_mxfp8_fused(a[0], self.w, a[1], self.s, a_preshuffle=False, **kw)
        return self.ab.gemm_a4w4_fused(a[0], self.w, a[1], self.s, **kw)


class Layer:
    def __init__(self, ab, kind, m):
        g = torch.Generator().manual_seed(m)
        self.ab, self.kind = ab, kind
        self.up, self.down = Weight(ab, kind, 2 * HIDDEN, D, 1), Weight(ab, kind, D, HIDDEN, 2)
        self.w1, self.w2, self.post, self.gate = (randn(g, D) for _ in range(4))
        self.bias = randn(g, D, dtype=torch.float32)
        self.x, self.r = randn(g, m, D), randn(g, m, D)
        self.mx = {} if kind == "bf16" else {"quant_dtype": ab.dtypes.fp8, "shuffle": 2} if kind == "mxfp8" else {"quant_dtype": ab.dtypes.fp4x2, "shuffle": True}

    def run(self):
        ab = self.ab
        *a, h = ab.gated_residual_norm(self.x, self.r, self.w1, **self.mx)
        both = self.up(a)
        c = ab.act_and_mul(both, "silu", **self.mx)
        c = c if isinstance(c, tuple) else (c,)
        h1 = self.down(c, bias=self.bias, residual=h)
        y, h2 = ab.gated_residual_norm(h1, h, self.w2, post_weight=self.post, gate=self.gate, otype=torch.float16)
        return a, h, both, c, h1, y, h2

    def values(self, a, plain):
        """The operand's values in 64 bits; `plain`: the same call with its scales in plain order"""
        if self.kind == "bf16":
            return a[0].double()
        assert torch.equal(a[0].view(torch.uint8), plain[0].view(torch.uint8))
        q, s = (t.view(torch.uint8).cpu().numpy() for t in plain[:2])
        return torch.from_numpy((ox.dequant_mxfp8 if self.kind == "mxfp8" else ox.dequant_mxfp4)(q, s)).cuda().double()

    def check(self, a, h, both, c, h1, y, h2):
        ab, step = self.ab, STEP[self.kind]
        plain = {**self.mx, "shuffle": False} if self.mx else {}
        want_y, want_h, big_y, big_h = ref64(self.x, self.r, self.w1)
        check_values(h, want_h, big_h, "h")
        if self.kind == "bf16":
            check_values(a[0], want_y, big_y, "normalised")
        # (MX operands are compared bit for bit with the oracle in the operators' own tests)
        check_gemm(both, self.values(a, ab.gated_residual_norm(self.x, self.r, self.w1, **plain)), self.up.value, D / step, None, None, None, "up")
        u, v = both.double().chunk(2, dim=1)
        if self.kind == "bf16":
            want = act64(u, "silu") * v
            check_values(c[0], want, want.abs(), "activation")
        check_gemm(h1, self.values(c, ab.act_and_mul(both, "silu", **plain)), self.down.value, HIDDEN / step, self.bias, None, h, "down")
        want_y, want_h, big_y, big_h = ref64(h1, h, self.w2, post_weight=self.post, gate=self.gate)
        check_values(h2, want_h, big_h, "second h")
        check_values(y, want_y, big_y, "second y")


@pytest.mark.parametrize("m", [1, 33, 300, 1100])
@pytest.mark.parametrize("kind", ["bf16", "mxfp8", "mxfp4"])
def test_layer(ab, kind, m):
    layer = Layer(ab, kind, m)
    layer.check(*layer.run())
    # captured, and replayed on other values: the same bits as the eager run of those
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.run()
    g = torch.Generator().manual_seed(7)
    layer.x.copy_(randn(g, m, D))
    layer.r.copy_(randn(g, m, D))
    graph.replay()
    torch.cuda.synchronize()
    layer.check(*out)
    want = layer.run()
    for i in (1, 2, 4, 5, 6):
        assert torch.equal(out[i], want[i]), f"step {i}: the replayed graph differs from the eager run"
    assert ab.device_status(0) == (0, 0, 0, 0)


def test_broadcast_rows(ab):
    """Residuals that are one row for all (stride 0), x that is one row for all, columns cut out of wider tensors."""
    g = torch.Generator().manual_seed(3)
    a, b, row = randn(g, 300, 256), randn(g, 512, 256), randn(g, 1, 512)
    for m in (5, 300):
        got = ab.gemm_a16w16_fused(a[:m], b, residual=row.expand(m, 512))
        assert torch.equal(got, ab.gemm_a16w16_fused(a[:m], b, residual=row.repeat(m, 1)))
    x = randn(g, 700, 512)
    for m in (3, 700):
        for xs, rs in ((x[:m], row.expand(m, 512)), (row.expand(m, 512), x[:m])):
            got, want = ab.gated_residual_norm(xs, rs, b[0].repeat(2)), ab.gated_residual_norm(xs.contiguous(), rs.contiguous(), b[0].repeat(2))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(ab.act_and_mul(row.expand(m, 512)), ab.act_and_mul(row.repeat(m, 1)))


def test_offsets_beyond_32_bits(ab):
    """Rows so far apart that an element's offset does not fit 32 bits: every kernel of the norm and of the gated activation."""
    g = torch.Generator().manual_seed(11)
    buf = torch.empty(700 * (2**22 + 9), dtype=torch.bfloat16, device="cuda")
    assert buf.numel() > 2**31
    for m, n, pitch in ((700, 8192, 2**22 + 8), (700, 7001, 2**22 + 9), (700, 128, 2**22 + 8), (250, 8192, 2**23), (250, 1003, 2**23 + 1)):
        view = torch.as_strided(buf, (m, n), (pitch, 1))
        x, r, w = randn(g, m, n), randn(g, m, n), randn(g, n)
        want_y, want_h, big_y, big_h = ref64(x, r, w)
        view.copy_(x)
        y, h = ab.gated_residual_norm(view, r, w)
        check_values(y, want_y, big_y, "x far apart"), check_values(h, want_h, big_h, "x far apart")
        view.copy_(r)
        y, h = ab.gated_residual_norm(x, view, w, residual_out=view)
        check_values(y, want_y, big_y, "residual far apart"), check_values(h, want_h, big_h, "residual far apart")
        assert h is view
        two = torch.as_strided(buf, (m, n // 2 * 2), (pitch, 1))
        u, v = x[:, : n // 2].double(), x[:, n // 2 : n // 2 * 2].double()
        two.copy_(x[:, : n // 2 * 2])
        want = act64(u, "silu") * v
        check_values(ab.act_and_mul(two), want, want.abs(), "input far apart")
        out = torch.as_strided(buf, (m, n // 2), (pitch, 1), n)
        ab.silu_and_mul(out, x[:, : n // 2 * 2])
        check_values(out, want, want.abs(), "output far apart")


def test_several_threads_at_once(ab):
    """Four host threads, each on a stream of its own, run layers of different sizes at the same time."""
    import threading

    layers = [Layer(ab, kind, m) for kind, m in (("bf16", 40), ("mxfp8", 300), ("mxfp4", 1100), ("bf16", 1))]
    want = [layer.run() for layer in layers]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    out = layers[i].run()
                torch.cuda.current_stream().synchronize()
            for k in (1, 2, 4, 5, 6):
                assert torch.equal(out[k], want[i][k]), f"layer {i}, step {k}"
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(layers))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert ab.device_status(0) == (0, 0, 0, 0)
