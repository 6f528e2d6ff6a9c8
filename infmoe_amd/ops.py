"""Operators of a layer that sends every token to several experts, on torch ROCm tensors.

Thin calls of the C ABI (include/infmoe.h has the definitions and limits): torch gives device memory and the current stream
of the tensors' device, libinfmoe.so computes.  Outputs are new tensors unless `out` is given; workspaces come from torch's
allocator per call, so concurrent streams and captured graphs never share one.  There is no backward pass: tensors that require a
gradient are refused unless gradients are off (torch.no_grad(), torch.inference_mode()).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import capi

_DTYPES = {torch.float32: capi.DTYPE_F32, torch.float16: capi.DTYPE_F16, torch.bfloat16: capi.DTYPE_BF16}
_F32, _I32 = torch.float32, torch.int32
_lib = None


def _load():
    global _lib
    _lib = capi.load()
    return _lib


def _refuse(message: str) -> None:
    raise capi.InfMoEError(capi.ERR_INVALID_ARGUMENT, message)


def _forward_only(*tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _refuse("an input requires a gradient, which these operators do not give: detach it or call under torch.no_grad()")


def _start(name: str, t: torch.Tensor) -> Tuple[int, int, int, int]:
    """Checks the operator's matrix of rows; returns (rows, columns, row stride, dtype code)."""
    code = _DTYPES.get(t.dtype)
    if code is None:
        _refuse(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    if not t.is_cuda:
        _refuse("tensors must be on the GPU")
    if t.dim() != 2:
        _refuse(f"{name} must be [rows, columns]")
    (rows, cols), (stride, step) = t.shape, t.stride()
    if step != 1 and cols > 1:
        _refuse(f"{name}: the elements of a row must lie side by side")
    return rows, cols, stride if rows > 1 else max(cols, 1), code


def _check(name: str, t: torch.Tensor, dtype: torch.dtype, shape: Tuple[int, ...], device: torch.device) -> None:
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        _refuse(f"{name} must be contiguous {dtype} {list(shape)} on {device}, not {t.dtype} {list(t.shape)} on {t.device}")


def _call(device: torch.device, function, *args) -> None:
    """function(*args, stream) with the tensors' device current and its current stream."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        status = function(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = function(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        capi.check(status)


def route_topk(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
               top_groups: int = 1, group_top: int = 1, renormalize: bool = True, scale: float = 1.0,
               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The k best experts of every row of `logits` [T, E] and their weights: int32 [T, k], float32 [T, k].

    score: "softmax" or "sigmoid"; bias: float32 [E], added to the scores for the choice only; groups > 1: only the
    top_groups groups with the largest sums of their group_top best experts stay.  See infmoe_route_topk."""
    _forward_only(logits, bias, *(out or ()))
    T, E, stride, dtype = _start("logits", logits)
    device = logits.device
    kind = capi.SCORE_KINDS.get(score)
    if kind is None:
        _refuse(f"unknown score {score!r}")
    if bias is not None:
        _check("bias", bias, _F32, (E,), device)
    if out is None:
        if not 0 < k <= E:
            _refuse("k must be 1 to the number of experts")
        ids = torch.empty((T, k), dtype=_I32, device=device)
        weights = torch.empty((T, k), dtype=_F32, device=device)
    else:
        ids, weights = out
        _check("ids", ids, _I32, (T, k), device)
        _check("weights", weights, _F32, (T, k), device)
    _call(device, (_lib or _load()).infmoe_route_topk, T, E, k, dtype, logits.data_ptr(), stride, kind, None if bias is None else bias.data_ptr(),
          groups, top_groups, group_top, renormalize, scale, ids.data_ptr(), weights.data_ptr())
    return ids, weights


def _matrices(name: str, t: torch.Tensor, dtype: torch.dtype, shape: Tuple[int, int, int], device: torch.device) -> int:
    """Checks [E, rows, columns] of contiguous matrices; returns the elements from one matrix to the next."""
    E, rows, cols = shape
    if t.dtype is not dtype or t.shape != shape or t.device != device:
        _refuse(f"{name} must be {dtype} {list(shape)} on {device}, not {t.dtype} {list(t.shape)} on {t.device}")
    each, row, step = t.stride()
    if (cols > 1 and step != 1) or (rows > 1 and row != cols):
        _refuse(f"{name}: each matrix must be contiguous")
    return each if E > 1 else rows * cols


def _out(out: Optional[torch.Tensor], x: torch.Tensor, rows: int, cols: int) -> Tuple[torch.Tensor, int]:
    if out is None:
        return torch.empty((rows, cols), dtype=x.dtype, device=x.device), cols
    if out.dtype is not x.dtype or out.device != x.device or out.shape != (rows, cols):
        _refuse(f"out must be {x.dtype} [{rows}, {cols}] on {x.device}")
    return out, _start("out", out)[2]


def experts_topk(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, wi: torch.Tensor, wo: torch.Tensor,
                 wi_1: Optional[torch.Tensor] = None, *, ffn: str = "relu", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = sum over j of weights[t, j] * wo[e] act(wi[e] x[t] [, wi_1[e] x[t]]) with e = ids[t, j]: x [T, d], ids int32 and
    weights float32 [T, k] as route_topk gives them, wi, wi_1 [E, h, d], wo [E, d, h] -> [T, d].

    ffn: "relu", "gated_gelu" or "gated_silu" (the gated ones take wi_1).  An id that is no expert adds nothing.  Hidden rows are
    held in x's type: in float16 values beyond 65504 become infinite.  See infmoe_experts_topk."""
    _forward_only(x, weights, wi, wo, wi_1, out)
    T, d, x_stride, dtype = _start("x", x)
    device, kind = x.device, capi.TOPK_FFN_KINDS.get(ffn)
    if kind is None:
        _refuse(f"unknown ffn {ffn!r}")
    if (wi_1 is None) != (ffn == "relu"):
        _refuse("wi_1 goes with the gated kinds")
    if wi.dim() != 3 or ids.dim() != 2:
        _refuse("wi must be [E, h, d] and ids [T, k]")
    E, h, k = wi.shape[0], wi.shape[1], ids.shape[1]
    _check("ids", ids, _I32, (T, k), device)
    _check("weights", weights, _F32, (T, k), device)
    wi_stride, wo_stride = _matrices("wi", wi, x.dtype, (E, h, d), device), _matrices("wo", wo, x.dtype, (E, d, h), device)
    if wi_1 is not None and _matrices("wi_1", wi_1, x.dtype, (E, h, d), device) != wi_stride:
        _refuse("wi and wi_1 must be strided alike")
    y, y_stride = _out(out, x, T, d)
    lib = _lib or _load()
    ws = torch.empty(lib.infmoe_experts_topk_workspace_bytes(T, k, E, d, h, dtype), dtype=torch.uint8, device=device)
    _call(device, lib.infmoe_experts_topk, T, k, E, d, h, kind, dtype, x.data_ptr(), x_stride, ids.data_ptr(), weights.data_ptr(), wi.data_ptr(),
          None if wi_1 is None else wi_1.data_ptr(), wo.data_ptr(), wi_stride, wo_stride, y.data_ptr(), y_stride, ws.data_ptr())
    return y


def lora_project(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter: torch.Tensor,
                 scale: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = w x[t] + scale[i] * b[i] (a[i] x[t]) with i = adapter[t]: x [T, d], w [n, d], a [L, r, d], b [L, n, r], adapter int32
    [T], scale float32 [L] -> [T, n].  A row whose adapter is none of the L gets w x[t].  See infmoe_lora_project."""
    _forward_only(x, w, a, b, scale, out)
    T, d, x_stride, dtype = _start("x", x)
    device = x.device
    if w.dim() != 2 or a.dim() != 3:
        _refuse("w must be [n, d] and a [L, r, d]")
    n, (L, r) = w.shape[0], a.shape[:2]
    _check("w", w, x.dtype, (n, d), device)
    _check("a", a, x.dtype, (L, r, d), device)
    _check("b", b, x.dtype, (L, n, r), device)
    _check("adapter", adapter, _I32, (T,), device)
    if scale is not None:
        _check("scale", scale, _F32, (L,), device)
    y, y_stride = _out(out, x, T, n)
    lib = _lib or _load()
    ws = torch.empty(lib.infmoe_lora_project_workspace_bytes(T, d, n, r, dtype), dtype=torch.uint8, device=device)
    _call(device, lib.infmoe_lora_project, T, d, n, r, L, dtype, x.data_ptr(), x_stride, w.data_ptr(), a.data_ptr(), b.data_ptr(), adapter.data_ptr(),
          None if scale is None else scale.data_ptr(), y.data_ptr(), y_stride, ws.data_ptr())
    return y
