"""MXFP4 modules at the ends of their number ranges, against float64."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mx_cases as mc

pytestmark = pytest.mark.gpu

# A SwiGLU row in two bf16 parts: the first leaves at most half its step, 2^(e - 8) of a value in
# [2^e, 2^(e + 1)); what it leaves is below that, so the second part's half step is at most
# 2^(e - 17).
H_ROUND = {"bf16": 2.0 ** -17, "fp16": 2.0 ** -17, "fp32": 2.0 ** -24}


def _dev(*arrays):
    return tuple(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays)


def _switch(rng, E, OUT, IN, shift=0):
    """Experts whose weights are about 2^shift / sqrt(IN) large, and their values."""
    from vqlab_amd import mx
    codes, scales = mc.weight(rng, E, OUT, IN)
    scales = (scales.astype(np.int64) + shift).astype(np.uint8)
    return mx.MXSwitchLinear(*_dev(codes, scales), IN), mc.values(codes, scales, IN)


def _glu(rng, E, H, I, shifts=(0, 0, 0)):
    from vqlab_amd import mx
    (g, gw), (u, uw) = _switch(rng, E, I, H, shifts[0]), _switch(rng, E, I, H, shifts[1])
    d, dw = _switch(rng, E, H, I, shifts[2])
    return mx.MXSwitchGLU(g, u, d), (gw, uw, dw)


# ------------------------------------------------------------- SwiGLU rows
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,k,E,H,I", [(3, 2, 5, 96, 64), (60, 2, 5, 96, 64), (300, 4, 6, 64, 200), (40, 4, 64, 128, 160)])
def test_swiglu_rows_keep_more_than_the_type(dtype, T, k, E, H, I):
    """Few pairs and sorted ones alike: what is rounded to x's type is the output."""
    rng = np.random.default_rng(T + I)
    glu, ws = _glu(rng, E, H, I)
    x, xv = mc.acts(rng, dtype, T, H)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)])
    w = rng.random((T, k)).astype(np.float32)
    ref, bar = mc.experts(xv, ids, w.astype(np.float64), *ws, H_ROUND[dtype])
    bar = bar + mc.HALF_STEP[dtype] * (np.abs(ref) + bar) + (2.0 ** -25 if dtype == "fp16" else 0.0)
    mc.assert_within(glu(x, *_dev(ids, w)), ref, bar, "experts")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [3, 60, 300])
def test_swiglu_rows_beyond_fp16(dtype, T):
    """silu(g) * u of 1e5 and more, brought back by small down weights: a batch's rows are those of
    a token alone."""
    rng = np.random.default_rng(T)
    E, H, I, k = 5, 96, 64, 2
    glu, ws = _glu(rng, E, H, I, (9, 9, -16))
    assert glu.down_proj._w.f16_exact
    x, xv = mc.acts(rng, dtype, T, H)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)])
    w = rng.random((T, k)).astype(np.float32)
    g = np.einsum("th,eih->tei", xv, ws[0])
    u = np.einsum("th,eih->tei", xv, ws[1])
    assert np.abs(g * u / (1 + np.exp(-np.clip(g, -500, None)))).max() > 1e5
    ref, bar = mc.experts(xv, ids, w.astype(np.float64), *ws, H_ROUND[dtype])
    bar = bar + mc.HALF_STEP[dtype] * (np.abs(ref) + bar) + (2.0 ** -25 if dtype == "fp16" else 0.0)
    mc.assert_within(glu(x, *_dev(ids, w)), ref, bar, "experts")


# ----------------------------------------------------- x beyond bf16's range
@pytest.mark.parametrize("N", [1, 20, 70, 200])
def test_fp32_x_above_the_largest_bf16(N):
    """Every finite fp32 x is finite in the product, forward and backward."""
    from vqlab_amd import mx
    rng = np.random.default_rng(N)
    codes, scales = mc.weight(rng, 48, 96)
    lin, w = mx.MXLinear(*_dev(codes, scales - 8), 96), mc.values(codes, scales - 8, 96)
    big = float(np.finfo(np.float32).max)
    for cols, rows, call in ((96, w, lin), (48, w.T, lin._dx)):
        x, _ = mc.acts(rng, "fp32", N, cols)
        x[0, 3], x[N // 2, 17], x[N - 1, cols - 1] = big, -big, big * (1 - 2.0 ** -10)
        y, bar = mc.product_bar(x.double().cpu().numpy(), rows, "fp32")
        assert np.abs(y).max() < big
        mc.assert_within(call(x), y, bar, "large x")
