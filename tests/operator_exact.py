"""The oracles of oracle/topk_oracle.py for whole batches on the GPU: the same definitions and bounds, in 64 bits, by torch's
matrix product."""
import numpy as np

from oracle import topk_oracle as O


def _mm(a, b):  # a [m, k], b [n, k] -> a b^T
    return a.double() @ b.double().t().contiguous()


def _mm_abs(a, b):
    return _mm(a.double().abs(), b.double().abs())


def lora_project(torch, x, w, a, b, adapter, scale, dtype):
    L, r, d = a.shape
    rel, tiny = O.half_step(dtype)
    y, bound = _mm(x, w), (d + r + 2) * O.U * _mm_abs(x, w)
    for i in range(L):
        t = (adapter == i).nonzero()[:, 0]
        if t.numel() == 0:
            continue
        s = float(scale[i])
        u = s * _mm(x[t], a[i])
        off = abs(s) * (d + 2) * O.U * _mm_abs(x[t], a[i]) + rel * u.abs() * 1.01 + tiny
        y[t] += _mm(u, b[i])
        bound[t] += _mm_abs(off, b[i]) + (d + r + 2) * O.U * _mm_abs(u, b[i])
    return y, bound * 1.01 + rel * y.abs() * 1.01 + tiny


def _activate(torch, ffn, u, v):
    if ffn == "relu":
        return u.clamp_min(0)
    if ffn == "gated_gelu":
        return 0.5 * u * (1 + torch.tanh(np.sqrt(2 / np.pi) * (u + 0.044715 * u ** 3))) * v
    return u / (1 + torch.exp(-u)) * v


def experts_topk(torch, x, ids, weights, wi, wo, wi_1, ffn, dtype):
    E, h, d = wi.shape
    T, k = ids.shape
    rel, tiny = O.half_step(dtype)
    y = torch.zeros(T, d, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        rows = x[t]
        u, P = _mm(rows, wi[e]), _mm_abs(rows, wi[e])
        v = one = None
        if wi_1 is not None:
            v, Q, one = _mm(rows, wi_1[e]), _mm_abs(rows, wi_1[e]), torch.ones_like(u)
        hid = _activate(torch, ffn, u, v)
        off = 1.13 * (v.abs() if v is not None else 1.0) * (d + 1) * O.U * P
        if v is not None:
            off = off + _activate(torch, ffn, u, one).abs() * (d + 1) * O.U * Q
        off = off + hid.abs() * (32 * O.U + rel) + tiny
        g = weights[t, j].double()[:, None]
        y.index_add_(0, t, g * _mm(hid, wo[e]))
        bound.index_add_(0, t, g.abs() * (_mm_abs(off * 1.01, wo[e]) + (h + k + 2) * O.U * _mm_abs(hid, wo[e])))
    return y, bound * 1.01 + rel * y.abs() * 1.01 + tiny


def assert_within(got, want, bound, what=""):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: {int((off > bound).sum())} of {off.numel()} beyond their bound, worst {float((off / bound).max()):.3g} times, first at {(off > bound).nonzero()[0].tolist()}"
