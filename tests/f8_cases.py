"""Oracles of 8-bit rows, weights and norms in float64 (and the 32-bit steps of the quantiser), from
the definitions, and seeded inputs."""
from __future__ import annotations

import numpy as np

BLOCK = 128
MIN_SCALE = np.float32(2.0 ** -126)


def grid(q):
    """q (float64) rounded to e4m3: three bits after the first, multiples of 2^-9, ties to even."""
    mag = np.maximum(np.abs(q), 2.0 ** -6)
    e = np.floor(np.log2(mag))
    e = np.where(2.0 ** e > mag, e - 1, e)
    e = np.where(2.0 ** (e + 1) <= mag, e + 1, e)
    step = 2.0 ** (e - 3)
    return np.copysign(np.minimum(np.round(np.abs(q) / step) * step, 448.0), q)


def _scale(top):
    """fp32 scale of blocks whose largest magnitude is `top` (fp32); NaN where that is not finite."""
    with np.errstate(all="ignore"):
        s = np.maximum((top.astype(np.float64) / 448).astype(np.float32), MIN_SCALE)
    return np.where(np.isfinite(top), s, np.float32(np.nan))


def _code_values(b, s):
    """b (fp32) under scales s: the codes as values (0 where the scale is NaN)."""
    with np.errstate(all="ignore"):
        inv = (1.0 / s.astype(np.float64)).astype(np.float32)
        q = (b.astype(np.float64) * inv.astype(np.float64)).astype(np.float32).astype(np.float64)
        return np.where(np.isnan(s), 0.0, grid(np.where(np.isnan(s), 0.0, q)))


def quantize(x):
    """x [R, C] -> code values float64 [R, C], scales fp32 [R, ceil(C / 128)]."""
    x = np.asarray(x, np.float32)
    R, C = x.shape
    B = -(-C // BLOCK)
    b = np.zeros((R, B, BLOCK), np.float32)
    b.reshape(R, -1)[:, :C] = x
    s = _scale(np.abs(b).max(-1))
    return _code_values(b, s[..., None]).reshape(R, -1)[:, :C], s


def quantize_weight(w):
    """w [O, I] -> code values float64, scales fp32 of 128 x 128."""
    w = np.asarray(w, np.float32)
    O, I = w.shape
    p = np.zeros((-(-O // BLOCK) * BLOCK, -(-I // BLOCK) * BLOCK), np.float32)
    p[:O, :I] = w
    b = p.reshape(p.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    s = _scale(np.abs(b).max((1, 3)))
    return _code_values(b, s[:, None, :, None]).reshape(p.shape)[:O, :I], s


def row_values(q, s):
    return q * np.repeat(s.astype(np.float64), BLOCK, 1)[:, :q.shape[1]]


def weight_values(q, s):
    s = np.repeat(np.repeat(s.astype(np.float64), BLOCK, 0)[:q.shape[0]], BLOCK, 1)
    return q * s[:, :q.shape[1]]


def weight(rng, O, I, spread=4):
    """Random codes (uint8, every finite one) [O, I], scales fp32 over `spread` powers of two, and the
    float64 values they stand for; about 1 / sqrt(I) large."""
    codes = rng.integers(0, 256, (O, I)).astype(np.uint8)
    codes[(codes & 127) == 127] -= 1                       # 0x7f, 0xff: NaN
    s = (2.0 ** rng.uniform(-spread, 0, (-(-O // BLOCK), -(-I // BLOCK))) / 150 / np.sqrt(I)).astype(np.float32)
    return codes, s, weight_values(decode(codes), s)


def decode(codes):
    """e4m3 codes (uint8) as float64 values."""
    c = np.asarray(codes, np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


def product_bar(x, w, dtype):
    """Bar of y = x . w^T: n exact products summed in fp32 in any order are off by at most n * 2^-24 *
    sum |x w|; each block's sum is multiplied by its scale (the product of two, rounded once: 2^-24)
    in a fused multiply-add (one of the n additions) and K slices add up to 16 more; one rounding into
    dtype, which below fp16's smallest normal number 2^-14 is off by half of the fixed step 2^-24."""
    from mx_cases import HALF_STEP
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    acc = (x.shape[1] + 20) * 2.0 ** -24 * mag
    step = HALF_STEP[dtype] * (np.abs(y) + acc)
    return y, acc + (np.maximum(step, 2.0 ** -25) if dtype == "fp16" else step)


def norm(x, res, w, eps, round_to):
    """h, r, y in float64; round_to: numpy rounding of the sum into x's type."""
    h = x if res is None else round_to(x + res)
    r = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return h, r, h * r * w


def norm_grad(h, r, w, dy, dh):
    xh, g = h * r, dy * w
    dx = r * (g - xh * (g * xh).mean(1, keepdims=True)) + (0 if dh is None else dh)
    return dx, (dy * xh).sum(0)


def instruction_bar(q, sx, w8, sw):
    """What the 8-bit matrix instructions may drop: of eight neighbouring products (columns 8 i .. 8 i + 7
    of a row) each is cut towards zero at 2^-13 of the power of two of the largest, which that product
    is at least; the largest itself loses nothing. q, w8: code values; sx [N, B], sw [O / 128, B]."""
    N, C = q.shape
    pad = lambda a: np.pad(np.abs(a), ((0, 0), (0, -C % BLOCK))).reshape(a.shape[0], -1, BLOCK // 8, 8)
    a, b = pad(q), pad(w8)
    swo = np.repeat(sw.astype(np.float64), BLOCK, 0)[:w8.shape[0]]
    bar = np.zeros((N, w8.shape[0]))
    for n in range(N):
        top = (a[n][None] * b).max(-1).sum(-1)             # [O, B]
        bar[n] = 7 * 2.0 ** -13 * (top * swo * sx[n].astype(np.float64)).sum(-1)
    return bar
