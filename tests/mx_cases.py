"""MXFP4 and router oracles in float64, from the formats' definitions, and seeded inputs."""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# half a step of rounding to nearest, relative to the value
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def quantize(x):
    """x [R, C] (any float) -> codes uint8 [R, 16 B], scales uint8 [R, B]."""
    x = np.asarray(x, np.float64)
    R, C = x.shape
    B = -(-C // 32)
    b = np.zeros((R, B * 32))
    b[:, :C] = x
    b = b.reshape(R, B, 32)
    codes = np.zeros((R, B, 32), np.uint8)
    scales = np.zeros((R, B), np.uint8)
    for r in range(R):
        for i in range(B):
            blk = b[r, i]
            if not np.isfinite(blk).all():
                scales[r, i] = 255
                continue
            top = np.abs(blk).max()
            e = max(int(np.floor(np.log2(top))) - 2, -127) if top > 0 else -127
            if top > 0:                                    # log2 may round up to the next power
                while e > -127 and 2.0 ** (e + 2) > top:
                    e -= 1
                while 2.0 ** (e + 3) <= top:
                    e += 1
            q = np.abs(blk) / 2.0 ** e
            d = np.abs(q[:, None] - GRID[None])            # exact: few bits, powers of two
            near = d.min(1, keepdims=True)
            tie = d == near
            # of two nearest codes the even one
            code = np.where(tie.sum(1) > 1, [2 * (np.flatnonzero(t)[0] // 2 + np.flatnonzero(t)[0] % 2)
                                             for t in tie], tie.argmax(1))
            codes[r, i] = code + 8 * np.signbit(blk)
            scales[r, i] = e + 127
    c = codes.reshape(R, -1)
    return c[:, 0::2] | (c[:, 1::2] << 4), scales


def values(codes, scales, C):
    """The float64 values [..., C] of packed codes and scales."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v.reshape(*scales.shape, 32) * s[..., None]).reshape(*codes.shape[:-1], -1)[..., :C]


def weight(rng, *shape, spread=3):
    """Random codes [..., 16 B] and scales [..., B] of rows of shape[-1] values, about
    1 / sqrt(columns) large, scales over `spread` powers of two; codes past the row are zero."""
    C = shape[-1]
    B = -(-C // 32)
    c = rng.integers(0, 16, (*shape[:-1], 32 * B)).astype(np.uint8)
    c[..., C:] = 0
    base = 127 - 2 - int(np.round(np.log2(np.sqrt(C))))
    scales = rng.integers(base - spread + 1, base + 1, (*shape[:-1], B)).astype(np.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), scales


def torch_dtype(name):
    import torch
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


def acts(rng, dtype, *shape):
    """N(0, 1) activations of a dtype on the GPU, and their float64 values."""
    import torch
    x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch_dtype(dtype))
    return x.cuda(), x.double().numpy()


def product_bar(x, w, dtype, more=0.0):
    """Bar of y = x . w^T: the sum of n exact products in any order of fp32 additions is off by at
    most n * 2^-24 * sum |x w| (each of n additions rounds by half a step of a partial sum, which
    sum |x w| bounds), then one rounding into dtype. `more` adds to |y|'s error before it."""
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    acc = x.shape[1] * 2.0 ** -24 * mag + more
    return y, acc + HALF_STEP[dtype] * (np.abs(y) + acc)


def assert_within(got, ref, bar, what=""):
    got = got.detach().double().cpu().numpy() if hasattr(got, "cpu") else np.asarray(got, np.float64)
    assert got.shape == ref.shape, (got.shape, ref.shape)
    bad = ~(np.abs(got - ref) <= bar)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside the bar, first at {i}: "
                             f"{got[i]} for {ref[i]} +- {bar[i]}")


def route(logits, k, norm=True, mask=None):
    """float64 routing: ids, weights, counts, balance, z, n, probabilities."""
    l = np.asarray(logits, np.float64)
    T, E = l.shape
    live = (np.ones(T, bool) if mask is None else np.asarray(mask, bool)) & (l > -np.inf).any(1)
    p = np.zeros_like(l)
    lse = np.zeros(T)
    ids = np.full((T, k), -1)
    w = np.zeros((T, k))
    for t in np.flatnonzero(live):
        m = l[t].max()
        ex = np.exp(l[t] - m)
        p[t] = ex / ex.sum()
        lse[t] = m + np.log(ex.sum())
        order = [e for e in np.argsort(-l[t], kind="stable")[:k] if l[t, e] > -np.inf]
        ids[t, :len(order)] = order
        w[t, :len(order)] = p[t, order] / (p[t, order].sum() if norm else 1.0)
    counts = np.bincount(ids[ids >= 0], minlength=E)
    n = int(live.sum())
    balance = E * (counts / (n * k) * p.sum(0) / n).sum() if n else 0.0
    z = (lse[live] ** 2).sum() / n if n else 0.0
    return dict(ids=ids, w=w, counts=counts, balance=balance, z=z, n=n, p=p, lse=lse, live=live)


def route_grad(r, k, norm, dw, gb, gz):
    """The formula's gradient of the logits, float64."""
    p, n = r["p"], max(r["n"], 1)
    E = p.shape[1]
    f = gb * E * r["counts"] / (n * n * k)
    d = p * (f - (p * f).sum(1, keepdims=True)) + 2 * gz / n * r["lse"][:, None] * p
    s = (r["w"] * dw).sum(1)
    for t in np.flatnonzero(r["live"]):
        for j, e in enumerate(r["ids"][t]):
            if e >= 0:
                d[t, e] += r["w"][t, j] * (dw[t, j] - (s[t] if norm else 0.0))
        if not norm:
            d[t] -= p[t] * s[t]
    d[~r["live"]] = 0
    return d


def experts(x, ids, w, gate, up, down, h_round):
    """y [T, H] of float64 weights [E, ., .], and a bar for its error: gate and up are off by
    their fp32 sums, the SwiGLU row by that and by h_round, down and the weighted sum by fp32."""
    T, H = x.shape
    y, bar = np.zeros((T, H)), np.zeros((T, H))
    I = gate.shape[1]
    eps = 2.0 ** -24
    for t in range(T):
        for j, e in enumerate(ids[t]):
            if not 0 <= e < gate.shape[0]:
                continue
            g, u = x[t] @ gate[e].T, x[t] @ up[e].T
            dg = H * eps * (np.abs(x[t]) @ np.abs(gate[e]).T)
            du = H * eps * (np.abs(x[t]) @ np.abs(up[e]).T)
            sg = g / (1 + np.exp(-g))
            h = sg * u
            # |silu'| < 1.1; silu itself in fp32 to a few units in the last place
            dh = (1.1 * dg + 16 * eps * np.abs(sg)) * np.abs(u) + np.abs(sg) * du + 1.1 * dg * du
            dh = dh + h_round * (np.abs(h) + dh)
            yj, mag = h @ down[e].T, (np.abs(h) + dh) @ np.abs(down[e]).T
            dy = dh @ np.abs(down[e]).T + I * eps * mag
            y[t] += w[t, j] * yj
            bar[t] += abs(w[t, j]) * (dy + (ids.shape[1] + 2) * eps * np.abs(mag))
    return y, bar
