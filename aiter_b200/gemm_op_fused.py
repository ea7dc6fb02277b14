"""GEMMs with a fused epilogue: out = act(A @ B^T + bias) + residual in one launch, computed in fp32 from the accumulator and rounded
once.  Operands as for gemm_a16w16, gemm_a8w8_mxfp8 and gemm_a4w4."""
from __future__ import annotations

import torch
from torch import Tensor

from . import dtypes
from ._ffi import call_host, current_stream, host
from .block_ops import ACTIVATIONS, activation_id


def _fused(bits: int, fn: str, A: Tensor, B: Tensor, k: int, A_scale, B_scale, bias, activation, residual, otype, out, flag, kernelName: str) -> Tensor:
    act = ACTIVATIONS.get(activation, 0)
    if act == 0:
        act = activation_id(activation, fn)
    n = B.shape[0]
    flat = A.dim() == 2
    if residual is not None and residual.shape != (*A.shape[:-1], n):
        raise ValueError(f"{fn}: residual must be {(*A.shape[:-1], n)}, got {tuple(residual.shape)}")
    if out is not None and (out.shape != (*A.shape[:-1], n) or (otype is not None and out.dtype != otype)):
        raise ValueError(f"{fn}: out must be {otype} {(*A.shape[:-1], n)}, got {out.dtype} {tuple(out.shape)}")
    a2, r2, o2 = A, residual, out
    if not flat:
        a2 = A.reshape(-1, k)
        r2 = None if residual is None else residual.reshape(-1, n)
        o2 = None if out is None else out.view(-1, n)
    result = call_host("aiter_b200_" + fn, host.gemm, bits, a2, B, A_scale, B_scale, bias, r2, o2, otype, act, flag,
                       kernelName.encode() if kernelName else None, current_stream(A.get_device()))
    if out is not None:
        return out
    return result if flat else result.view(*A.shape[:-1], n)


def gemm_a16w16_fused(A: Tensor, B: Tensor, bias: Tensor | None = None, activation: str | None = None, residual: Tensor | None = None,
                      otype: torch.dtype | None = None, out: Tensor | None = None, kernelName: str = "") -> Tensor:
    """act(A[.., K] @ B[N, K]^T + bias[N]) + residual[.., N] in bf16 operands.  activation: none, relu, silu, gelu (erf) or gelu_tanh.
    bias and residual in bf16, fp16 or fp32; otype (default A's type) bf16, fp16 or fp32.  `out` may be `residual` itself.  A weight
    produced by shuffle_weight (tagged `.is_shuffled`) is consumed in its shuffled form.  K % 8 == 0."""
    if otype is None and out is None:
        otype = A.dtype
    return _fused(16, "gemm_a16w16_fused", A, B, B.shape[1], None, None, bias, activation, residual, otype, out, getattr(B, "is_shuffled", False), kernelName)


def gemm_a8w8_mxfp8_fused(A: Tensor, B: Tensor, ScaleA: Tensor, ScaleB: Tensor, bias: Tensor | None = None, activation: str | None = None,
                          residual: Tensor | None = None, otype: torch.dtype = dtypes.bf16, a_preshuffle: bool = True,
                          out: Tensor | None = None, kernelName: str = "") -> Tensor:
    """The same epilogue behind gemm_a8w8_mxfp8: A [M, K] e4m3, B [N, K] e4m3 as 16x16-byte tiles, scales in the (m/32,k/4,32,4) order."""
    return _fused(8, "gemm_a8w8_mxfp8_fused", A, B, B.shape[1], ScaleA, ScaleB, bias, activation, residual, otype, out, a_preshuffle, kernelName)


def gemm_a4w4_fused(A: Tensor, B: Tensor, A_scale: Tensor, B_scale: Tensor, bias: Tensor | None = None, activation: str | None = None,
                    residual: Tensor | None = None, otype: torch.dtype = dtypes.bf16, bpreshuffle: bool = True, out: Tensor | None = None,
                    kernelName: str = "") -> Tensor:
    """The same epilogue behind gemm_a4w4: A [.., K/2] and B [N, K/2] packed e2m1 (B (16,16)-shuffled when bpreshuffle), scales e8m0 in
    the e8m0_shuffle layout."""
    return _fused(4, "gemm_a4w4_fused", A, B, B.shape[1], A_scale, B_scale, bias, activation, residual, otype, out, bpreshuffle, kernelName)
