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


def _matrices(name: str, t: torch.Tensor, like: torch.Tensor, shape: Tuple[int, ...]) -> int:
    """Checks [E, rows, columns] of contiguous matrices; returns the elements from one matrix to the next."""
    _need(t.dtype == like.dtype, f"{name} must be {like.dtype} as x is, not {t.dtype}")
    _need(t.dim() == 3 and tuple(t.shape) == shape, f"{name} must be {list(shape)}, not {list(t.shape)}")
    _need((shape[2] == 1 or t.stride(2) == 1) and (shape[1] == 1 or t.stride(1) == shape[2]), f"{name}: each matrix must be contiguous")
    return t.stride(0) if shape[0] > 1 else shape[1] * shape[2]


def _out(name: str, out: Optional[torch.Tensor], x: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    if out is None:
        return torch.empty((rows, cols), dtype=x.dtype, device=x.device)
    _need(out.dtype == x.dtype and out.device == x.device and tuple(out.shape) == (rows, cols), f"{name} must be {x.dtype} [{rows}, {cols}] on {x.device}")
    return out


def experts_topk(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, wi: torch.Tensor, wo: torch.Tensor,
                 wi_1: Optional[torch.Tensor] = None, *, ffn: str = "relu", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = sum over j of weights[t, j] * wo[e] act(wi[e] x[t] [, wi_1[e] x[t]]) with e = ids[t, j]: x [T, d], ids int32 and
    weights float32 [T, k] as route_topk gives them, wi, wi_1 [E, h, d], wo [E, d, h] -> [T, d].

    ffn: "relu", "gated_gelu" or "gated_silu" (the gated ones take wi_1).  An id that is no expert adds nothing.  See
    infmoe_experts_topk."""
    _same_device(x, ids=ids, weights=weights, wi=wi, wo=wo, wi_1=wi_1)
    dtype, x_stride = _dtype("x", x), _rows("x", x)
    _need(ffn in capi.TOPK_FFN_KINDS, f"unknown ffn {ffn!r}")
    _need((wi_1 is None) == (ffn == "relu"), "wi_1 goes with the gated kinds")
    T, d = x.shape
    _need(wi.dim() == 3, "wi must be [E, h, d]")
    E, h = wi.shape[:2]
    _need(ids.dim() == 2 and ids.shape[0] == T, "ids must be [T, k]")
    k = ids.shape[1]
    _need(ids.dtype == torch.int32 and ids.is_contiguous(), "ids must be contiguous int32 [T, k]")
    _need(weights.dtype == torch.float32 and weights.shape == ids.shape and weights.is_contiguous(), "weights must be contiguous float32 [T, k]")
    wi_stride, wo_stride = _matrices("wi", wi, x, (E, h, d)), _matrices("wo", wo, x, (E, d, h))
    _need(wi_1 is None or _matrices("wi_1", wi_1, x, (E, h, d)) == wi_stride, "wi and wi_1 must be strided alike")
    y = _out("out", out, x, T, d)
    y_stride = _rows("out", y)
    lib = capi.load()
    ws = torch.empty(lib.infmoe_experts_topk_workspace_bytes(T, k, E, d, h, dtype), dtype=torch.uint8, device=x.device)
    _on(x.device, lib.infmoe_experts_topk, T, k, E, d, h, capi.TOPK_FFN_KINDS[ffn], dtype, x.data_ptr(), x_stride, ids.data_ptr(),
        weights.data_ptr(), wi.data_ptr(), _ptr(wi_1), wo.data_ptr(), wi_stride, wo_stride, y.data_ptr(), y_stride, ws.data_ptr())
    return y


def lora_project(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter: torch.Tensor,
                 scale: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = w x[t] + scale[i] * b[i] (a[i] x[t]) with i = adapter[t]: x [T, d], w [n, d], a [L, r, d], b [L, n, r], adapter int32
    [T], scale float32 [L] -> [T, n].  A row whose adapter is none of the L gets w x[t].  See infmoe_lora_project."""
    _same_device(x, w=w, a=a, b=b, adapter=adapter, scale=scale)
    dtype, x_stride = _dtype("x", x), _rows("x", x)
    T, d = x.shape
    _need(w.dtype == x.dtype and w.dim() == 2 and w.shape[1] == d and w.is_contiguous(), f"w must be contiguous {x.dtype} [n, {d}]")
    n = w.shape[0]
    _need(a.dim() == 3 and a.is_contiguous() and b.is_contiguous(), "a and b must be contiguous [L, r, d] and [L, n, r]")
    L, r = a.shape[:2]
    _matrices("a", a, x, (L, r, d)), _matrices("b", b, x, (L, n, r))
    _need(adapter.dtype == torch.int32 and adapter.shape == (T,) and adapter.is_contiguous(), "adapter must be contiguous int32 [T]")
    _need(scale is None or (scale.dtype == torch.float32 and scale.shape == (L,) and scale.is_contiguous()), "scale must be float32 [L]")
    y = _out("out", out, x, T, n)
    y_stride = _rows("out", y)
    lib = capi.load()
    ws = torch.empty(lib.infmoe_lora_project_workspace_bytes(T, d, n, r, dtype), dtype=torch.uint8, device=x.device)
    _on(x.device, lib.infmoe_lora_project, T, d, n, r, L, dtype, x.data_ptr(), x_stride, w.data_ptr(), a.data_ptr(), b.data_ptr(),
        adapter.data_ptr(), _ptr(scale), y.data_ptr(), y_stride, ws.data_ptr())
    return y
