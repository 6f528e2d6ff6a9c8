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
