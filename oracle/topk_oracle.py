"""Float64 oracles of the operators for several experts per token: routing, the experts' products, adapters."""
import numpy as np


def route_topk(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0):
    """(ids int32 [T, k], weights float64 [T, k]); row by row, as include/infmoe.h defines it."""
    x = np.asarray(logits, np.float64)
    T, E = x.shape
    ids = np.full((T, k), -1, np.int32)
    w = np.zeros((T, k))
    per = E // groups
    b = None if bias is None else np.asarray(bias, np.float64)
    with np.errstate(all="ignore"):
        for t in range(T):
            row = x[t]
            masked = row == -np.inf
            if score == "softmax":
                p = np.where(masked, 0.0, np.exp(row - row.max())) if not masked.all() else np.zeros(E)
                p = p / p.sum() if p.sum() > 0 else p
            else:
                p = 1.0 / (1.0 + np.exp(-row))
            scored = b is not None or group_top == 2
            c = np.where(masked, -np.inf, p + (0.0 if b is None else b)) if scored else row.copy()
            if np.isnan(row).any() or np.isnan(c).any() or (score == "softmax" and (row == np.inf).any()) or (scored and (c == np.inf).any()):
                w[t] = np.nan
                continue
            if groups > 1:
                best = -np.sort(-c.reshape(groups, per), axis=1)[:, :group_top].sum(axis=1)
                keep = np.argsort(-best, kind="stable")[:top_groups]
                for g in range(groups):
                    if g not in keep:
                        c[g * per:(g + 1) * per] = -np.inf
            order = np.argsort(-c, kind="stable")[:k]
            order = order[c[order] > -np.inf]
            ids[t, :len(order)] = order
            if len(order) == 0:
                continue
            if renormalize:  # in logarithms: ratios of scores far below float64's range are ratios all the same
                logs = row[order] if score == "softmax" else -np.logaddexp(0.0, -row[order])
                q = np.exp(logs - logs.max())
                w[t, :len(order)] = scale * q / q.sum()
            else:
                w[t, :len(order)] = scale * p[order]
    return ids, w


U = 2.0 ** -24  # FP32's largest relative rounding error


def half_step(dtype):
    """(largest relative rounding error, largest absolute one near zero) of a type."""
    return {"float32": (2.0 ** -24, 2.0 ** -150), "bfloat16": (2.0 ** -8, 2.0 ** -134), "float16": (2.0 ** -11, 2.0 ** -25)}[dtype]


def activate(ffn, u, v):
    with np.errstate(over="ignore", invalid="ignore"):
        if ffn == "relu":
            return np.where(u < 0, 0.0, u)
        if ffn == "gated_gelu":
            return 0.5 * u * (1 + np.tanh(np.sqrt(2 / np.pi) * (u + 0.044715 * u ** 3))) * v
        return u / (1 + np.exp(-u)) * v


def experts_topk(x, ids, weights, wi, wo, wi_1=None, ffn="relu", dtype="float32"):
    """(y float64 [T, d], bound [T, d]): bound is what |computed - y| cannot exceed when sums are FP32 in any order, the hidden
    rows and y are rounded to dtype, and the activation is good to 32 u (its exponential to (1.45 |x| + 2) u, |x| < 16 here).

    With P = |wi| |x|, Q = |wi_1| |x| a first product is off by d u P (Q), the hidden value by 1.13 |v| d u P + |act| d u Q (1.13:
    the steepest slope of the activations) and by its rounding; the second product adds h u per term, the weighted sum k."""
    x, weights, wi, wo = (np.asarray(a, np.float64) for a in (x, weights, wi, wo))
    E, h, d = wi.shape
    T, k = ids.shape
    rel, tiny = half_step(dtype)
    y, bound = np.zeros((T, d)), np.zeros((T, d))
    for e in range(E):
        t, j = np.nonzero(ids == e)
        if len(t) == 0:
            continue
        rows = x[t]
        u, P = rows @ wi[e].T, np.abs(rows) @ np.abs(wi[e]).T
        v = Q = None
        if wi_1 is not None:
            w1 = np.asarray(wi_1[e], np.float64)
            v, Q = rows @ w1.T, np.abs(rows) @ np.abs(w1).T
        hid = activate(ffn, u, v)
        off = 1.13 * (np.abs(v) if v is not None else 1.0) * (d + 1) * U * P
        if v is not None:
            off = off + np.abs(activate(ffn, u, 1.0)) * (d + 1) * U * Q
        off = off + np.abs(hid) * (32 * U + rel) + tiny
        w = weights[t, j][:, None]
        np.add.at(y, t, w * (hid @ wo[e].T))
        size = np.abs(wo[e])
        np.add.at(bound, t, np.abs(w) * ((off * 1.01) @ size.T + (h + k + 2) * U * (np.abs(hid) @ size.T)))
    none = ~((ids >= 0) & (ids < E))
    y += np.where(none, 0.0 * weights, 0.0).sum(axis=1)[:, None]
    return y, bound * 1.01 + rel * np.abs(y) * 1.01 + tiny


def lora_project(x, w, a, b, adapter, scale=None, dtype="float32"):
    """(y float64 [T, n], bound [T, n]): sums in FP32 in any order, scale a x and y rounded to dtype."""
    x, w, a, b = (np.asarray(v, np.float64) for v in (x, w, a, b))
    L, r, d = a.shape
    rel, tiny = half_step(dtype)
    scale = np.ones(L) if scale is None else np.asarray(scale, np.float64)
    y, bound = x @ w.T, (d + r + 2) * U * (np.abs(x) @ np.abs(w).T)
    for i in range(L):
        t = np.nonzero(adapter == i)[0]
        if len(t) == 0:
            continue
        u = scale[i] * (x[t] @ a[i].T)
        off = np.abs(scale[i]) * (d + 2) * U * (np.abs(x[t]) @ np.abs(a[i]).T) + rel * np.abs(u) * 1.01 + tiny
        y[t] += u @ b[i].T
        bound[t] += off @ np.abs(b[i]).T + (d + r + 2) * U * (np.abs(u) @ np.abs(b[i]).T)
    return y, bound * 1.01 + rel * np.abs(y) * 1.01 + tiny
