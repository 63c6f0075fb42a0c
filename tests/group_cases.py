"""Oracle of routing by scores, a bias and groups in float64, from its definition."""
from __future__ import annotations

import numpy as np


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=2, norm=True, scale=1.0, mask=None):
    l = np.asarray(logits, np.float64)
    T, E = l.shape
    live = (np.ones(T, bool) if mask is None else np.asarray(mask, bool)) & (l > -np.inf).any(1)
    ids, w = np.full((T, k), -1), np.zeros((T, k))
    soft, p, s, lse = np.zeros_like(l), np.zeros_like(l), np.zeros_like(l), np.zeros(T)
    gs = E // groups
    for t in np.flatnonzero(live):
        m = l[t].max()
        ex = np.exp(l[t] - m)
        soft[t], lse[t] = ex / ex.sum(), m + np.log(ex.sum())
        with np.errstate(over="ignore"):
            s[t] = 1 / (1 + np.exp(-l[t])) if score == "sigmoid" else soft[t]
        p[t] = s[t] / s[t].sum() if s[t].sum() > 0 else soft[t]
        c = s[t] + (0 if bias is None else bias)
        can = (l[t] > -np.inf) & (c > -np.inf)
        c = np.where(can, c, -np.inf)
        if groups > 1:
            best = []
            for g in range(groups):
                top = np.sort(c[g * gs:(g + 1) * gs])[::-1][:group_top]
                best.append(top[top > -np.inf].sum() if (top > -np.inf).any() else -np.inf)
            kept = np.argsort(-np.array(best), kind="stable")[:top_groups]
            can &= np.isin(np.arange(E) // gs, kept)
        order = np.argsort(-np.where(can, c if bias is not None else l[t], -np.inf), kind="stable")
        order = [e for e in order if can[e]][:k]
        ids[t, :len(order)] = order
        # relative weights by logarithms, which do not vanish
        ls = -np.logaddexp(0, -l[t, order]) if score == "sigmoid" else l[t, order] - lse[t]
        if norm and order:
            r = np.exp(ls - ls.max())
            w[t, :len(order)] = scale * r / r.sum()
        else:
            w[t, :len(order)] = scale * np.exp(ls)
    counts = np.bincount(ids[ids >= 0], minlength=E)
    n = int(live.sum())
    balance = E * (counts / (n * k) * p.sum(0) / n).sum() if n else 0.0
    z = (lse[live] ** 2).sum() / n if n else 0.0
    return dict(ids=ids, w=w, counts=counts, balance=balance, z=z, n=n, p=p, s=s, soft=soft, lse=lse, live=live, l=l)


def grad(r, k, score, norm, scale, dw, gb, gz):
    """The formula's gradient of the logits, and the size of its terms (for a bar)."""
    n, E = max(r["n"], 1), r["p"].shape[1]
    f = gb * E * r["counts"] / (n * n * k)
    p, soft = r["p"], r["soft"]
    q = 1 / (1 + np.exp(r["l"])) if score == "sigmoid" else np.ones_like(p)
    u = p * (f - (p * f).sum(1, keepdims=True))
    size = p * (np.abs(f) + (p * np.abs(f)).sum(1, keepdims=True))
    wdw = r["w"] * dw
    sw, aw = wdw.sum(1), np.abs(wdw).sum(1)
    for t in np.flatnonzero(r["live"]):
        for j, e in enumerate(r["ids"][t]):
            if e >= 0:
                u[t, e] += wdw[t, j] - (r["w"][t, j] / scale * sw[t] if norm else 0.0)
                size[t, e] += abs(wdw[t, j]) + (r["w"][t, j] / scale * aw[t] if norm else 0.0)
    d, size = u * q, size * q
    if score == "softmax" and not norm:
        d = d - soft * sw[:, None]
        size = size + soft * aw[:, None]
    d = d + 2 * gz / n * r["lse"][:, None] * soft
    size = size + abs(2 * gz / n) * (np.abs(r["lse"][:, None]) + 1) * soft
    d[~r["live"]], size[~r["live"]] = 0, 0
    return d, size
