"""Operators of a layer that sends every token to several experts, on torch ROCm tensors.

Thin calls of the C ABI (include/infmoe.h has the definitions and limits): torch gives device memory and the current stream
of the tensors' device, libinfmoe.so computes.  Outputs are new tensors unless `out` is given; workspaces come from torch's
allocator per call, so concurrent streams and captured graphs never share one.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import capi

_DTYPES = {torch.float32: capi.DTYPE_F32, torch.float16: capi.DTYPE_F16, torch.bfloat16: capi.DTYPE_BF16}


def _need(cond: bool, message: str) -> None:
    if not cond:
        raise capi.InfMoEError(capi.ERR_INVALID_ARGUMENT, message)


def _dtype(name: str, t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    _need(code is not None, f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def _rows(name: str, t: torch.Tensor, cols: Optional[int] = None) -> int:
    """Checks a matrix of rows whose elements lie side by side; returns its row stride."""
    _need(t.dim() == 2 and (cols is None or t.shape[1] == cols), f"{name} must be [rows, {cols if cols is not None else 'columns'}]")
    _need(t.shape[1] <= 1 or t.stride(1) == 1, f"{name}: the elements of a row must lie side by side")
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _same_device(first: torch.Tensor, **tensors: Optional[torch.Tensor]) -> None:
    _need(first.is_cuda, "tensors must be on the GPU")
    for name, t in tensors.items():
        _need(t is None or t.device == first.device, f"{name} is on {None if t is None else t.device}, not on {first.device}")


def _on(device: torch.device, call, *args) -> None:
    """call(*args, stream) with the tensors' device current and its current stream."""
    if device.index == torch.cuda.current_device():
        capi.check(call(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            capi.check(call(*args, torch.cuda.current_stream(device).cuda_stream))


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def route_topk(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
               top_groups: int = 1, group_top: int = 1, renormalize: bool = True, scale: float = 1.0,
               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The k best experts of every row of `logits` [T, E] and their weights: int32 [T, k], float32 [T, k].

    score: "softmax" or "sigmoid"; bias: float32 [E], added to the scores for the choice only; groups > 1: only the
    top_groups groups with the largest sums of their group_top best experts stay.  See infmoe_route_topk."""
    _same_device(logits, bias=bias)
    dtype, stride = _dtype("logits", logits), _rows("logits", logits)
    T, E = logits.shape
    _need(score in capi.SCORE_KINDS, f"unknown score {score!r}")
    _need(bias is None or (bias.dtype == torch.float32 and bias.shape == (E,) and bias.is_contiguous()), "bias must be float32 [E]")
    if out is None:
        _need(0 < k <= E, "k must be 1 to the number of experts")
        ids = torch.empty((T, k), dtype=torch.int32, device=logits.device)
        weights = torch.empty((T, k), dtype=torch.float32, device=logits.device)
    else:
        ids, weights = out
        _same_device(logits, ids=ids, weights=weights)
        _need(ids.dtype == torch.int32 and ids.shape == (T, k) and ids.is_contiguous(), "ids must be a contiguous int32 [T, k]")
        _need(weights.dtype == torch.float32 and weights.shape == (T, k) and weights.is_contiguous(), "weights must be a contiguous float32 [T, k]")
    _on(logits.device, capi.load().infmoe_route_topk, T, E, k, dtype, logits.data_ptr(), stride, capi.SCORE_KINDS[score], _ptr(bias),
        groups, top_groups, group_top, int(renormalize), scale, ids.data_ptr(), weights.data_ptr())
    return ids, weights
