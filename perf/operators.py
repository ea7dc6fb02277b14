"""The operators of a transformer block around the matrix products, as cases that can be timed and compared.

  linear  out = act(A B^T + bias) + residual, A and B in bf16, MXFP8 or MXFP4
  norm    h = residual_scale * residual + gate * post(x),  y = norm(h) * (weight_offset + weight) + bias, y in 16 / 32 bits or as MXFP8
  act     y = act(gate half) * up half of [rows, 2 n], y in 16 bits or as MXFP8 / MXFP4

With `own` false run() computes them from elementary torch operations, with `own` true through the package's operators.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ------------------------------------------------------------------------------------------------ cases
def _linear(name, fmt, m, n, k, bias="none", act="none", residual="none", out="bf16"):
    return {"name": name, "op": "linear", "fmt": fmt, "m": m, "n": n, "k": k, "bias": bias, "act": act, "residual": residual, "out": out}


def _norm(name, m, n, kind="rms", x="bf16", residual="bf16", post=False, gate="none", samples=1, scale=1.0, affine="channel", out="bf16"):
    return {"name": name, "op": "norm", "m": m, "n": n, "kind": kind, "x": x, "residual": residual, "post": post, "gate": gate,
            "samples": samples, "scale": scale, "affine": affine, "out": out}


def _act(name, m, n, act="silu", x="bf16", out="bf16"):
    return {"name": name, "op": "act", "m": m, "n": n, "act": act, "x": x, "out": out}


def listed():
    return [
        # one generated token through a hidden layer: latency
        _linear("linear token", "bf16", 1, 4096, 4096, bias="bf16", act="silu"),
        # a decode batch through an output projection with a packed 4-bit weight, added to the residual stream
        _linear("linear mxfp4 batch", "mxfp4", 32, 7168, 2048, residual="bf16"),
        # a short prompt, sizes that fill no tile and rows that start on no 16-byte boundary
        _linear("linear ragged", "bf16", 333, 1001, 1160, bias="fp32", act="gelu_tanh", residual="fp16", out="fp16"),
        # prompts of a batch through an 8-bit hidden layer
        _linear("linear mxfp8 prompts", "mxfp8", 4096, 7168, 2048, bias="bf16", act="gelu"),
        # long prompts into a residual stream kept in 32 bits
        _linear("linear long", "bf16", 16384, 7168, 2048, bias="bf16", residual="fp32", out="fp32"),
        # one token between two blocks: latency
        _norm("norm token", 1, 4096),
        # long prompts, norms on both sides of a block, a learned gate per channel and a scaled residual
        _norm("norm sandwich", 16384, 8192, post=True, gate="channel", scale=0.5),
        # images of a batch, modulated per sample; an odd width and a residual stream in 32 bits
        _norm("norm samples", 8200, 1155, kind="layer", residual="fp32", gate="sample", samples=8, affine="sample"),
        # prompts in front of an 8-bit product: the norm leaves the product's operand and its block scales
        _norm("norm mxfp8", 4096, 7168, out="mxfp8"),
        # a decode batch between the two products of a gated layer
        _act("act batch", 16, 9216),
        # a short prompt in front of a 4-bit product
        _act("act mxfp4", 512, 4096, out="mxfp4"),
        # long prompts
        _act("act long", 16384, 12288, act="gelu_tanh", x="fp16", out="fp16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "norm", "act"])
    if op == "linear":
        fmt = rng.choice(["bf16", "bf16", "mxfp8", "mxfp4"])
        out = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        m, n, k = _log(rng, 1, 16384), _log(rng, 64, 8192), _log(rng, 64, 2048 if out == "fp32" else 8192)
        if fmt == "bf16":
            k = (k + 7) // 8 * 8
        else:
            n, k = (n + 15) // 16 * 16, (k + 127) // 128 * 128
        m = max(1, min(m, 16384 * 7168 * 2048 // (n * k)))
        c = _linear("", fmt, m, n, k, bias=rng.choice(["none", "bf16", "fp32"]), act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    residual=rng.choice(["none", "bf16", "fp16", "fp32"]), out=out)
    elif op == "norm":
        out = rng.choice(["bf16", "fp16", "fp32", "mxfp8"])
        n, samples = _log(rng, 33, 16384), rng.choice([1, 2, 3, 8])
        if out == "mxfp8":
            n = (n + 127) // 128 * 128
        m = max(1, min(_log(rng, 1, 16384), 16384 * 8192 // n))
        m = (m + samples - 1) // samples * samples
        c = _norm("", m, n, kind=rng.choice(["rms", "layer"]), x=rng.choice(["bf16", "fp16", "fp32"]),
                  residual=rng.choice(["none", "bf16", "fp16", "fp32"]), post=rng.random() < 0.4,
                  gate=rng.choice(["none", "channel", "sample", "token"]), samples=samples, scale=rng.choice([1.0, 0.5, 1.25]),
                  affine=rng.choice(["none", "channel", "sample"]), out=out)
    else:
        out = rng.choice(["bf16", "fp16", "mxfp8", "mxfp4"])
        n = _log(rng, 33, 24576)
        if out in ("mxfp8", "mxfp4"):
            n = (n + 127) // 128 * 128
        m = max(1, min(_log(rng, 1, 16384), (1 << 21 if out == "mxfp4" else 16384 * 12288) // n))
        c = _act("", m, n, act=rng.choice(["silu", "gelu", "gelu_tanh"]), x=rng.choice(["bf16", "fp16"]), out=out)
    del c["name"]
    return c


def work(case):
    c, size = case, {"bf16": 2, "fp16": 2, "fp32": 4, "none": 0, "mxfp8": 1 + 1 / 32, "mxfp4": 0.5 + 1 / 32}
    m, n = c["m"], c["n"]
    if c["op"] == "linear":
        return {"bytes": (m + n) * c["k"] * size[c["fmt"]] + n * size[c["bias"]] + m * n * (size[c["residual"]] + size[c["out"]]), "flops": 2 * m * n * c["k"]}
    if c["op"] == "norm":
        residual = c["residual"] if c["residual"] != "none" else c["x"]
        return {"bytes": m * n * (size[c["x"]] + size[c["residual"]] + size[residual] + size[c["out"]]), "flops": 12 * m * n}
    return {"bytes": m * n * (2 * size[c["x"]] + size[c["out"]]), "flops": 12 * m * n}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _codes(g, rows, k, fmt, std):
    """Elements as their byte codes [rows, k] (e4m3, or e2m1 in the low nibble) and scale bytes [rows, k / 32], as a 1x32 quantiser leaves them."""
    v = _randn(g, rows, k // 32, 32)
    top = v.abs().amax(dim=2, keepdim=True) * (std / (448.0 if fmt == "mxfp8" else 6.0))
    _, e = torch.frexp(top)
    scaled = v * std / torch.exp2(e.float())
    byte = (e + 127).to(torch.uint8).view(rows, k // 32)
    if fmt == "mxfp8":
        return scaled.to(E4M3).view(torch.uint8).view(rows, k), byte
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    code = torch.bucketize(scaled.abs(), edges).to(torch.uint8) | ((scaled < 0).to(torch.uint8) << 3)
    return code.view(rows, k), byte


def _inputs(case, seed):
    """What the case is about, before any layout: operands as values or codes."""
    c, g = case, _gen(seed)
    m, n = c["m"], c["n"]
    if c["op"] == "linear":
        k = c["k"]
        if c["fmt"] == "bf16":
            s = {"a": _randn(g, m, k).bfloat16(), "b": (_randn(g, n, k) / math.sqrt(k)).bfloat16()}
        else:
            s = {}
            s["a"], s["a_scale"] = _codes(g, m, k, c["fmt"], 1.0)
            s["b"], s["b_scale"] = _codes(g, n, k, c["fmt"], 1 / math.sqrt(k))
        s["bias"] = None if c["bias"] == "none" else (0.5 * _randn(g, n)).to(DT[c["bias"]])
        s["residual"] = None if c["residual"] == "none" else _randn(g, m, n).to(DT[c["residual"]])
        return s
    if c["op"] == "norm":
        b = c["samples"]
        s = {"x": (_randn(g, m, n) * torch.exp2(2 * _randn(g, m, 1))).to(DT[c["x"]])}
        s["residual"] = None if c["residual"] == "none" else (3 * _randn(g, m, n) + 0.5).to(DT[c["residual"]])
        s["post"] = (1 + 0.2 * _randn(g, n)).bfloat16() if c["post"] else None
        s["gate"] = {"none": None, "channel": (0.3 * _randn(g, n)).bfloat16(), "sample": (0.5 * _randn(g, b, n)).bfloat16(), "token": torch.sigmoid(_randn(g, m, 1))}[c["gate"]]
        if c["affine"] == "none":
            s["weight"], s["bias"] = None, None
        elif c["affine"] == "channel":
            s["weight"], s["bias"] = (1 + 0.2 * _randn(g, n)).bfloat16(), (0.1 * _randn(g, n)).bfloat16() if c["kind"] == "layer" else None
        else:
            s["weight"], s["bias"] = (0.2 * _randn(g, b, n)).bfloat16(), (0.3 * _randn(g, b, n)).bfloat16()
        return s
    return {"x": (2 * _randn(g, m, 2 * n)).to(DT[c["x"]])}


def _tiles(t, rows, cols):
    """[R, C] bytes -> tiles of rows x cols, row-major inside and among the tiles; R padded to whole tiles by the caller."""
    r, c = t.shape
    return t.view(r // rows, rows, c // cols, cols).transpose(1, 2).contiguous().view(r, c)


def _untiles(t, rows, cols):
    r, c = t.shape
    return t.view(r // rows, c // cols, rows, cols).transpose(1, 2).reshape(r, c)


def _pad_rows(t, to, value):
    more = -t.shape[0] % to
    return t if not more else torch.cat([t, t.new_full((more, t.shape[1]), value)])


def _interleave(byte, rows_to, fill_rows):
    """Scale bytes [R, C] -> the interleaved order of the 4-bit product: 32 rows by 8 columns as [4][16][2][2]; columns padded by `fill_rows` too."""
    t = _pad_rows(byte, rows_to, fill_rows)
    more = -t.shape[1] % 8
    t = t if not more else torch.cat([t, t.new_full((t.shape[0], more), fill_rows)], dim=1)
    r, c = t.shape
    return t.view(r // 32, 2, 16, c // 8, 2, 4).permute(0, 3, 5, 2, 4, 1).contiguous().view(r, c)


def _uninterleave(t):
    r, c = t.shape
    return t.view(r // 32, c // 8, 4, 16, 2, 2).permute(0, 5, 3, 1, 4, 2).reshape(r, c)


def _pack(code):
    return code[:, 0::2] | (code[:, 1::2] << 4)


def prepare(case, seed):
    """The tensors a program holds: weights and block scales in the layouts the products read."""
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "linear" and case["fmt"] == "mxfp8":
        s["a"], s["b"] = s["a"].view(E4M3), _tiles(s["b"], 16, 16).view(E4M3)
        for name in ("a_scale", "b_scale"):
            s[name] = _tiles(_pad_rows(s[name], 32, 127), 32, 4).view(E8M0)
    elif case["op"] == "linear" and case["fmt"] == "mxfp4":
        s["a"], s["b"] = _pack(s["a"]), _tiles(_pack(s["b"]), 16, 16)
        for name in ("a_scale", "b_scale"):
            s[name] = _interleave(s[name], 256, 127).view(E8M0)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _activate(x, act):
    if act == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _e2m1():
    return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")


def _widen(s, name, fmt, rows):
    """An operand of a block-scaled product as 32-bit values [rows, k]."""
    tiled = name == "b"
    if fmt == "mxfp8":
        v, sc = s[name], _untiles(s[name + "_scale"].view(torch.uint8), 32, 4)
        v = (_untiles(v.view(torch.uint8), 16, 16).view(E4M3) if tiled else v).float()
    else:
        q, sc = s[name], _uninterleave(s[name + "_scale"].view(torch.uint8))
        q = _untiles(q, 16, 16) if tiled else q
        v = _e2m1()[torch.stack([q & 15, q >> 4], dim=2).view(rows, -1).int()]
    k = v.shape[1]
    return (v.view(rows, k // 32, 32) * torch.exp2(sc[:rows, : k // 32].float() - 127)[:, :, None]).view(rows, k)


def _plain_linear(c, s):
    if c["fmt"] == "bf16":
        a, b = s["a"].float(), s["b"].float()
    else:
        a, b = _widen(s, "a", c["fmt"], c["m"]), _widen(s, "b", c["fmt"], c["n"])
    y = a @ b.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _activate(y, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DT[c["out"]])


def _rows(p, m):
    """A parameter [n], [samples, n] or [m, 1] as something that broadcasts over [m, n]."""
    return p if p.dim() == 1 or p.shape[0] == m else p.repeat_interleave(m // p.shape[0], dim=0)


def _normed(v, kind, eps=1e-6):
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    return v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps)


def _round_blocks(y, fmt):
    """Values [m, n] (64 bits: a scale or an element next to a border of its type) -> element values and scale bytes per 32."""
    m, n = y.shape
    v = y.view(m, n // 32, 32)
    top = v.abs().amax(dim=2) / (448.0 if fmt == "mxfp8" else 6.0)
    mant, e = torch.frexp(top)
    e = torch.where(mant == 0.5, e - 1, e)  # the power of two at or above
    e = torch.where(top == 0, torch.full_like(e, -127), e).clamp(-127, 127)
    z = v * torch.exp2(-e.double())[:, :, None]
    if fmt == "mxfp8":
        # round at the step of the binade in 64 bits; what is left fits e4m3 exactly
        _, b = torch.frexp(z)
        step = torch.exp2((b - 4).clamp(min=-9).double())
        q = (torch.round(z / step) * step).clamp(-448, 448)
    else:
        a = z.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(a.dtype)
        q = torch.copysign((torch.round(a / step) * step).clamp(max=6), z)
    return q.view(m, n).float().to(E4M3), (e + 127).to(torch.uint8)


def _plain_quantised(y, fmt):
    """As the operators leave it: elements, and scales in the order that the products read, the last group of 32 rows filled up."""
    q, byte = _round_blocks(y, fmt)
    if fmt == "mxfp8":
        return q, _tiles(_pad_rows(byte, 32, 127), 32, 4).view(E8M0)
    return q, _interleave(byte, 32, 0).view(E8M0)


def _plain_norm(c, s):
    m, wide = c["m"], torch.float64 if c["out"] == "mxfp8" else torch.float32
    h = s["x"].to(wide)
    if s["post"] is not None:
        h = _normed(h, c["kind"]) * s["post"].to(wide)
    if s["gate"] is not None:
        h = h * _rows(s["gate"], m).to(wide)
    if s["residual"] is not None:
        h = h + c["scale"] * s["residual"].to(wide)
    y = _normed(h, c["kind"])
    if s["weight"] is not None:
        y = y * (_rows(s["weight"], m).to(wide) + (1 if c["affine"] == "sample" else 0))
    if s["bias"] is not None:
        y = y + _rows(s["bias"], m).to(wide)
    h = h.to((s["residual"] if s["residual"] is not None else s["x"]).dtype)
    return [*_plain_quantised(y, "mxfp8"), h] if c["out"] == "mxfp8" else [y.to(DT[c["out"]]), h]


def _plain_act(c, s):
    n = c["n"]
    x = s["x"].to(torch.float64 if c["out"] in ("mxfp8", "mxfp4") else torch.float32)
    y = _activate(x[:, :n], c["act"]) * x[:, n:]
    return list(_plain_quantised(y, c["out"])) if c["out"] in ("mxfp8", "mxfp4") else [y.to(DT[c["out"]])]


# ------------------------------------------------------------------------------------------------ the operators
def _own(c, s):
    import aiter_b200 as ab

    if c["op"] == "linear":
        more = {"bias": s["bias"], "activation": c["act"], "residual": s["residual"], "otype": DT[c["out"]]}
        if c["fmt"] == "bf16":
            return ab.gemm_a16w16_fused(s["a"], s["b"], **more)
        if c["fmt"] == "mxfp8":
            return ab.gemm_a8w8_mxfp8_fused(s["a"], s["b"], s["a_scale"], s["b_scale"], a_preshuffle=False, **more)
        return ab.gemm_a4w4_fused(s["a"], s["b"], s["a_scale"], s["b_scale"], **more)
    if c["op"] == "norm":
        more = {"weight": s["weight"], "bias": s["bias"], "gate": s["gate"], "residual_scale": c["scale"], "post_weight": s["post"], "norm": c["kind"],
                "eps": 1e-6, "weight_offset": 1.0 if c["affine"] == "sample" else 0.0}
        if c["out"] == "mxfp8":
            y, scale, h = ab.gated_residual_norm(s["x"], s["residual"], quant_dtype=ab.dtypes.fp8, shuffle=2, **more)
            return [y, scale, h]
        return list(ab.gated_residual_norm(s["x"], s["residual"], otype=DT[c["out"]], **more))
    if c["out"] == "mxfp8":
        return list(ab.act_and_mul(s["x"], c["act"], quant_dtype=ab.dtypes.fp8, shuffle=2))
    if c["out"] == "mxfp4":
        y, scale = ab.act_and_mul(s["x"], c["act"], quant_dtype=ab.dtypes.fp4x2, shuffle=True)
        # two elements a byte: as the values they stand for
        if "pairs" not in s:
            both = torch.arange(256, device="cuda")
            s["pairs"] = _e2m1()[torch.stack([both & 15, both >> 4], dim=1)].to(E4M3).view(torch.int16).view(-1)
        q = s["pairs"][y.view(torch.uint8).int()].view(E4M3)
        return [q, scale.view(torch.uint8)[: (c["m"] + 31) // 32 * 32].view(E8M0)]
    return [ab.act_and_mul(s["x"], c["act"], otype=DT[c["out"]])]


def run(state):
    c = state["case"]
    if own:
        return _own(c, state)
    return {"linear": _plain_linear, "norm": _plain_norm, "act": _plain_act}[c["op"]](c, state)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_operand(v, byte, fmt):
    if fmt == "bf16":
        return v.double()
    if fmt == "mxfp8":
        sign, e, f = (v >> 7).double(), ((v >> 3) & 15).double(), (v & 7).double()
        mag = torch.where(e == 0, f * 2.0**-9, (1 + f / 8) * 2 ** (e - 7))
    else:
        sign, e, f = (v >> 3).double(), ((v >> 1) & 3).double(), (v & 1).double()
        mag = torch.where(e == 0, f * 0.5, (1 + f / 2) * 2 ** (e - 1))
    return (1 - 2 * sign) * mag * (2 ** (byte.double() - 127)).repeat_interleave(32, dim=1)


def _exact_activation(x, act):
    if act == "relu":
        return x.clamp(min=0)
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu":
        return x * 0.5 * torch.erfc(-x / math.sqrt(2))
    if act == "gelu_tanh":  # (1 + tanh u) / 2 is the logistic function of 2 u
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x**3))
    return x


def _exact_quantised(y, fmt):
    m, n = y.shape
    blocks = y.reshape(-1, 32)
    e = torch.ceil(torch.log2(blocks.abs().amax(dim=1) / (448 if fmt == "mxfp8" else 6))).clamp(-127, 127)
    z = blocks / 2 ** e[:, None]
    if fmt == "mxfp8":
        unit = 2 ** (torch.floor(torch.log2(z.abs().clamp(min=2.0**-6))) - 3)
    else:
        unit = 2 ** (torch.floor(torch.log2(z.abs().clamp(min=1.0))) - 1)
    z = (torch.round(z / unit) * unit).reshape(m, n)
    top = 448 if fmt == "mxfp8" else 6
    return z.clamp(-top, top), 2**e.reshape(m, n // 32)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    m, n = c["m"], c["n"]
    if c["op"] == "linear":
        y = _exact_operand(s["a"], s.get("a_scale"), c["fmt"]) @ _exact_operand(s["b"], s.get("b_scale"), c["fmt"]).T
        if s["bias"] is not None:
            y += s["bias"].double()
        y = _exact_activation(y, c["act"])
        return y if s["residual"] is None else y + s["residual"].double()
    if c["op"] == "act":
        y = _exact_activation(s["x"][:, :n].double(), c["act"]) * s["x"][:, n:].double()
        if c["out"] not in ("mxfp8", "mxfp4"):
            return [y]
        return [_exact_quantised(y, c["out"])[0], None]
    per = torch.arange(m, device="cuda") * c["samples"] // m  # each row's sample

    def spread(p):
        return p.double() if p.dim() == 1 or p.shape[1] == 1 else p.double()[per]

    def norm(v):
        if c["kind"] == "layer":
            var, mean = torch.var_mean(v, dim=1, keepdim=True, correction=0)
            return (v - mean) * torch.rsqrt(var + 1e-6)
        return v * torch.rsqrt(v.square().sum(dim=1, keepdim=True) / n + 1e-6)

    h = s["x"].double()
    if s["post"] is not None:
        h = norm(h) * s["post"].double()
    if s["gate"] is not None:
        h = spread(s["gate"]) * h
    if s["residual"] is not None:
        h = torch.add(h, s["residual"].double(), alpha=c["scale"])
    y = norm(h)
    if s["weight"] is not None:
        w = spread(s["weight"])
        y = y * (1 + w if c["affine"] == "sample" else w)
    if s["bias"] is not None:
        y = y + spread(s["bias"])
    if c["out"] == "mxfp8":
        return [_exact_quantised(y, "mxfp8")[0], None, h]
    return [y, h]
