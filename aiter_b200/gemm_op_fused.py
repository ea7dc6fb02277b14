"""GEMMs with a fused epilogue: out = act(A @ B^T + bias) + residual in one launch, computed in fp32 from the accumulator and rounded
once.  Operands as for gemm_a16w16, gemm_a8w8_mxfp8 and gemm_a4w4."""
from __future__ import annotations

import torch
from torch import Tensor, empty

from . import _ffi, dtypes
from ._ffi import _pack_tensor as pack, call_packed, pack_rows
from .block_ops import ACTIVATIONS, activation_id


def _prepare(fn: str, A: Tensor, k: int, n: int, activation, residual: Tensor | None, otype, out: Tensor | None):
    """Checks, the allocation of the output -> (rows, activation id, packed A, packed residual, packed out, result)"""
    act = ACTIVATIONS.get(activation, 0)
    if act == 0:
        act = activation_id(activation, fn)
    flat = A.dim() == 2
    a2 = A if flat else A.reshape(-1, k)
    m = a2.shape[0]
    if residual is not None and residual.shape != ((m, n) if flat else (*A.shape[:-1], n)):
        raise ValueError(f"{fn}: residual must be {(*A.shape[:-1], n)}, got {tuple(residual.shape)}")
    if out is None:
        o2 = empty(m, n, dtype=otype, device=A.device)
        result = o2 if flat else o2.view(*A.shape[:-1], n)
        packed = pack_rows(o2, m, n, A.get_device())
    else:
        if out.shape != (*A.shape[:-1], n) or (otype is not None and out.dtype != otype):
            raise ValueError(f"{fn}: out must be {otype} {(*A.shape[:-1], n)}, got {out.dtype} {tuple(out.shape)}")
        result, packed = out, pack(out if flat else out.view(m, n))
    r2 = residual if residual is None or flat else residual.reshape(m, n)
    return m, act, pack(a2), pack(r2), packed, result


def gemm_a16w16_fused(A: Tensor, B: Tensor, bias: Tensor | None = None, activation: str | None = None, residual: Tensor | None = None,
                      otype: torch.dtype | None = None, out: Tensor | None = None, kernelName: str = "") -> Tensor:
    """act(A[.., K] @ B[N, K]^T + bias[N]) + residual[.., N] in bf16 operands.  activation: none, relu, silu, gelu (erf) or gelu_tanh.
    bias and residual in bf16, fp16 or fp32; otype (default A's type) bf16, fp16 or fp32.  `out` may be `residual` itself.  A weight
    produced by shuffle_weight (tagged `.is_shuffled`) is consumed in its shuffled form.  K % 8 == 0."""
    n, k = B.shape
    if otype is None and out is None:
        otype = A.dtype
    _, act, a, r, o, result = _prepare("gemm_a16w16_fused", A, k, n, activation, residual, otype, out)
    call_packed("aiter_b200_gemm_a16w16_fused", A.get_device(), a, pack(B), pack(bias), r, o, act, getattr(B, "is_shuffled", False),
                kernelName.encode() if kernelName else None)
    return result


def gemm_a8w8_mxfp8_fused(A: Tensor, B: Tensor, ScaleA: Tensor, ScaleB: Tensor, bias: Tensor | None = None, activation: str | None = None,
                          residual: Tensor | None = None, otype: torch.dtype = dtypes.bf16, a_preshuffle: bool = True,
                          out: Tensor | None = None, kernelName: str = "") -> Tensor:
    """The same epilogue behind gemm_a8w8_mxfp8: A [M, K] e4m3, B [N, K] e4m3 as 16x16-byte tiles, scales in the (m/32,k/4,32,4) order."""
    n, k = B.shape
    _, act, a, r, o, result = _prepare("gemm_a8w8_mxfp8_fused", A, k, n, activation, residual, otype, out)
    call_packed("aiter_b200_gemm_a8w8_mxfp8_fused", A.get_device(), a, pack(B), pack(ScaleA), pack(ScaleB), pack(bias), r, o, act,
                bool(a_preshuffle), kernelName.encode() if kernelName else None)
    return result


def gemm_a4w4_fused(A: Tensor, B: Tensor, A_scale: Tensor, B_scale: Tensor, bias: Tensor | None = None, activation: str | None = None,
                    residual: Tensor | None = None, otype: torch.dtype = dtypes.bf16, bpreshuffle: bool = True, out: Tensor | None = None,
                    kernelName: str = "") -> Tensor:
    """The same epilogue behind gemm_a4w4: A [.., K/2] and B [N, K/2] packed e2m1 (B (16,16)-shuffled when bpreshuffle), scales e8m0 in
    the e8m0_shuffle layout."""
    n, k2 = B.shape
    m, act, a, r, o, result = _prepare("gemm_a4w4_fused", A, k2, n, activation, residual, otype, out)
    # tall problems re-lay the block scales once per call, in memory of this call's own (two captured graphs share none)
    nbytes = _ffi.fused_workspace_bytes(m, n, 2 * k2) if m >= 1024 else 0
    workspace = empty(nbytes, dtype=torch.uint8, device=A.device) if nbytes else None
    call_packed("aiter_b200_gemm_a4w4_fused", A.get_device(), a, pack(B), pack(A_scale), pack(B_scale), pack(bias), r, o, pack(workspace), act,
                bool(bpreshuffle), kernelName.encode() if kernelName else None)
    return result
