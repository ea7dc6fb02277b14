"""What stands between two GEMMs of a transformer block, one kernel launch each: the norms around a block with its gate and
residual sum, and the gated activation.  Both can leave the operand of an MX GEMM (data and block scales in the GEMM's layout)
instead of 16-bit values.  The reference's closest forms: aiter/ops/rmsnorm.py, aiter/ops/norm.py, aiter/ops/activation.py."""
from __future__ import annotations

import torch
from torch import Tensor

from . import dtypes
from ._ffi import call_host, current_stream, host

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_NORMS = {"rms": 0, "layer": 1}


def activation_id(activation: str | None, fn: str) -> int:
    try:
        return ACTIVATIONS["none" if activation is None else activation]
    except KeyError:
        raise ValueError(f"{fn}: unknown activation {activation!r}, expected one of {', '.join(ACTIVATIONS)}") from None


def _mx_bits(fn: str, n: int, quant_dtype, otype) -> int:
    if otype is not None:
        raise ValueError(f"{fn}: otype and quant_dtype exclude one another")
    if n % 32 != 0:
        raise ValueError(f"{fn}: an MX output needs a multiple of 32 columns, got {n}")
    if quant_dtype == dtypes.fp4x2:
        return 4
    if quant_dtype == dtypes.fp8:
        return 8
    raise ValueError(f"{fn}: unsupported quant_dtype {quant_dtype}, expected one of (dtypes.fp4x2, dtypes.fp8)")


def gated_residual_norm(x: Tensor, residual: Tensor | None = None, weight: Tensor | None = None, bias: Tensor | None = None,
                        gate: Tensor | None = None, residual_scale: float = 1.0, post_weight: Tensor | None = None,
                        post_bias: Tensor | None = None, norm: str = "rms", eps: float = 1e-6, weight_offset: float = 0.0,
                        post_norm: bool | None = None, otype: torch.dtype | None = None, quant_dtype: torch.dtype | None = None,
                        shuffle=False, residual_out: Tensor | None = None):
    """The end of one block and the beginning of the next in one launch:

        u = norm(x) * post_weight + post_bias   (with a post_weight / post_bias, or post_norm=True; else u = x)
        h = residual_scale * residual + gate * u
        y = norm(h) * (weight_offset + weight) + bias

    norm "rms": v / sqrt(mean v^2 + eps), "layer": (v - mean v) / sqrt(var v + eps), over the last dimension.  Sums, statistics and h
    are fp32; y comes from h before h is rounded to its own type.  x and residual [.., n] in bf16 / fp16 / fp32.  Parameters are [n]
    (every row), or [groups, n] with groups dividing the rows (modulation per sample: consecutive rows share an entry); the gate may
    also be [groups, 1] (one value per entry: per token with groups = rows).

    Returns (y, h), or (y, y_scale, h) with quant_dtype fp4x2 / fp8: y then is an MX operand, its e8m0 scales laid out by `shuffle` as
    per_1x32_mx_quant_hip does (True: what gemm_a4w4 reads; 2: what the MXFP8 GEMMs read).  otype: type of y (default x's).  h has the
    residual's type and goes to `residual_out` where that is given (it may be `residual` itself).  Without a residual, gate and first
    norm h is x, which is returned as it is."""
    fn = "gated_residual_norm"
    if norm not in _NORMS:
        raise ValueError(f"{fn}: unknown norm {norm!r}, expected 'rms' or 'layer'")
    post = (post_weight is not None or post_bias is not None) if post_norm is None else bool(post_norm)
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, x.shape[-1])
    r2 = residual if residual is None or residual.dim() == 2 else residual.reshape(-1, residual.shape[-1])
    o2 = residual_out
    if o2 is not None:
        if o2.shape != x.shape:
            raise ValueError(f"{fn}: residual_out must have x's shape {tuple(x.shape)}, got {tuple(o2.shape)}")
        o2 = o2 if flat else o2.view(-1, x.shape[-1])
    bits, layout = (0, 0) if quant_dtype is None else (_mx_bits(fn, x2.shape[1], quant_dtype, otype), int(shuffle))
    y, scale, h = call_host("aiter_b200_gated_residual_norm", host.norm, x2, r2, weight, bias, gate, post_weight, post_bias, o2, bits, otype,
                     residual_scale, weight_offset, eps, _NORMS[norm], post, layout, current_stream(x.get_device()))
    if not flat:
        y = y.view(*x.shape[:-1], y.shape[-1])
        h = h if h is None else h.view(x.shape)
    if residual_out is not None:
        h = residual_out
    elif h is None:
        h = x
    return (y, h) if scale is None else (y, scale, h)


def act_and_mul(x: Tensor, activation: str = "silu", otype: torch.dtype | None = None, quant_dtype: torch.dtype | None = None,
                shuffle=False):
    """y[.., j] = act(x[.., j]) * x[.., n + j] for x [.., 2n] (gate half first): the step between the two GEMMs of a gated layer.
    activation: silu, gelu (erf), gelu_tanh or relu, computed in fp32 (csrc/activation.cuh states the error; magnitudes of the activation
    below 2^-119 may come out as 0).  Returns y, or (y, y_scale) with quant_dtype fp4x2 / fp8: an MX operand, its
    scales laid out by `shuffle` as per_1x32_mx_quant_hip does."""
    fn = "act_and_mul"
    act = activation_id(activation, fn)
    if act == 0:
        raise ValueError(f"{fn}: an activation is required")
    if x.shape[-1] % 2 != 0:
        raise ValueError(f"{fn}: the last dimension must be even, got {x.shape[-1]}")
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, x.shape[-1])
    bits, layout = (0, 0) if quant_dtype is None else (_mx_bits(fn, x2.shape[1] // 2, quant_dtype, otype), int(shuffle))
    y, scale = call_host("aiter_b200_act_and_mul", host.act, x2, None, bits, otype, act, layout, current_stream(x.get_device()))
    if not flat:
        y = y.view(*x.shape[:-1], y.shape[-1])
    return y if scale is None else (y, scale)


def silu_and_mul(out: Tensor, input: Tensor) -> None:
    """out = silu(input[.., :n]) * input[.., n:] (aiter/ops/activation.py)."""
    _act_and_mul_into(out, input, "silu")


def gelu_and_mul(out: Tensor, input: Tensor) -> None:
    _act_and_mul_into(out, input, "gelu")


def gelu_tanh_and_mul(out: Tensor, input: Tensor) -> None:
    _act_and_mul_into(out, input, "gelu_tanh")


def _act_and_mul_into(out: Tensor, input: Tensor, activation: str) -> None:
    x2 = input if input.dim() == 2 else input.reshape(-1, input.shape[-1])
    o2 = out if out.dim() == 2 else out.view(-1, out.shape[-1])
    call_host("aiter_b200_act_and_mul", host.act, x2, o2, 0, None, ACTIVATIONS[activation], 0, current_stream(input.get_device()))
