"""GEMMs with a fused epilogue: out = act(A @ B^T + bias) + residual in one launch, computed in fp32 from the accumulator and rounded
once.  Operands as for gemm_a16w16, gemm_a8w8_mxfp8 and gemm_a4w4."""
from __future__ import annotations

import torch
from torch import Tensor, empty

from . import _ffi, dtypes
from .block_ops import activation_id


def _rows(t: Tensor | None, n: int):
    return t if t is None or t.dim() == 2 else t.reshape(-1, n)


def _out(fn: str, A: Tensor, m: int, n: int, otype, out):
    """-> (the [m, n] matrix the kernel writes, what the caller gets)"""
    if out is None:
        o = empty(m, n, dtype=otype, device=A.device)
        return o, (o if A.dim() == 2 else o.view(*A.shape[:-1], n))
    if out.shape != (*A.shape[:-1], n) or (otype is not None and out.dtype != otype):
        raise ValueError(f"{fn}: out must be {otype} {(*A.shape[:-1], n)}, got {out.dtype} {tuple(out.shape)}")
    return (out if out.dim() == 2 else out.view(m, n)), out


def _check_residual(fn: str, A: Tensor, n: int, residual: Tensor | None):
    if residual is not None and residual.shape != (*A.shape[:-1], n):
        raise ValueError(f"{fn}: residual must be {(*A.shape[:-1], n)}, got {tuple(residual.shape)}")


def gemm_a16w16_fused(A: Tensor, B: Tensor, bias: Tensor | None = None, activation: str | None = None, residual: Tensor | None = None,
                      otype: torch.dtype | None = None, out: Tensor | None = None, kernelName: str = "") -> Tensor:
    """act(A[.., K] @ B[N, K]^T + bias[N]) + residual[.., N] in bf16 operands.  activation: none, relu, silu, gelu (erf) or gelu_tanh.
    bias and residual in bf16, fp16 or fp32; otype (default A's type) bf16, fp16 or fp32.  `out` may be `residual` itself.  A weight
    produced by shuffle_weight (tagged `.is_shuffled`) is consumed in its shuffled form.  K % 8 == 0."""
    fn = "gemm_a16w16_fused"
    act = activation_id(activation, fn)
    n, k = B.shape
    a2 = A if A.dim() == 2 else A.reshape(-1, k)
    _check_residual(fn, A, n, residual)
    o2, result = _out(fn, A, a2.shape[0], n, otype if otype is not None else (A.dtype if out is None else None), out)
    _ffi.call("aiter_b200_gemm_a16w16_fused", a2, B, bias, _rows(residual, n), o2, act, getattr(B, "is_shuffled", False), kernelName or None)
    return result


def gemm_a8w8_mxfp8_fused(A: Tensor, B: Tensor, ScaleA: Tensor, ScaleB: Tensor, bias: Tensor | None = None, activation: str | None = None,
                          residual: Tensor | None = None, otype: torch.dtype = dtypes.bf16, a_preshuffle: bool = True,
                          out: Tensor | None = None, kernelName: str = "") -> Tensor:
    """The same epilogue behind gemm_a8w8_mxfp8: A [M, K] e4m3, B [N, K] e4m3 as 16x16-byte tiles, scales in the (m/32,k/4,32,4) order."""
    fn = "gemm_a8w8_mxfp8_fused"
    act = activation_id(activation, fn)
    n = B.shape[0]
    _check_residual(fn, A, n, residual)
    a2 = A if A.dim() == 2 else A.reshape(-1, A.shape[-1])
    o2, result = _out(fn, A, a2.shape[0], n, otype, out)
    _ffi.call("aiter_b200_gemm_a8w8_mxfp8_fused", a2, B, ScaleA, ScaleB, bias, _rows(residual, n), o2, act, bool(a_preshuffle), kernelName or None)
    return result


def gemm_a4w4_fused(A: Tensor, B: Tensor, A_scale: Tensor, B_scale: Tensor, bias: Tensor | None = None, activation: str | None = None,
                    residual: Tensor | None = None, otype: torch.dtype = dtypes.bf16, bpreshuffle: bool = True, out: Tensor | None = None,
                    kernelName: str = "") -> Tensor:
    """The same epilogue behind gemm_a4w4: A [.., K/2] and B [N, K/2] packed e2m1 (B (16,16)-shuffled when bpreshuffle), scales e8m0 in
    the e8m0_shuffle layout."""
    fn = "gemm_a4w4_fused"
    act = activation_id(activation, fn)
    n = B.shape[0]
    _check_residual(fn, A, n, residual)
    a2 = A if A.dim() == 2 else A.reshape(-1, A.shape[-1])
    m = a2.shape[0]
    o2, result = _out(fn, A, m, n, otype, out)
    # tall problems re-lay the block scales once per call, in memory of this call's own (two captured graphs share none)
    nbytes = _ffi.fused_workspace_bytes(m, n, 2 * a2.shape[1]) if m >= 1024 else 0
    workspace = empty(nbytes, dtype=torch.uint8, device=A.device) if nbytes else None
    _ffi.call("aiter_b200_gemm_a4w4_fused", a2, B, A_scale, B_scale, bias, _rows(residual, n), o2, workspace, act, bool(bpreshuffle),
              kernelName or None)
    return result
