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


# ------------------------------------------- weights of 2^128 and beyond
def _huge(rng, E, OUT, IN):
    """Experts of ordinary weights, but for expert 0: 6 * 2^127 throughout."""
    codes, scales = mc.weight(rng, E, OUT, IN)
    codes[0], scales[0] = 0x77, 254
    return codes, scales


def test_values_past_fp32_read_as_infinite():
    from vqlab_amd import mx
    codes = np.tile(np.arange(16, dtype=np.uint8) * 17, (4, 1))           # each code twice
    scales = np.array([[252], [253], [254], [255]], np.uint8)
    ref = mc.values(codes, scales, 32)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = mx.mx_dequantize(*_dev(codes, scales), 32, dtype).double().cpu().numpy()
        top = float(torch.finfo(dtype).max)
        want = np.where(np.abs(ref) > top, np.copysign(np.inf, ref), ref)
        assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("T,k", [(1, 3), (7, 2), (40, 2)])
@pytest.mark.parametrize("IN", [96, 640, 1664])
def test_pairs_without_an_expert_are_zero_beside_an_expert_of_infinities(T, k, IN):
    from vqlab_amd import mx
    rng = np.random.default_rng(T + IN)
    codes, scales = _huge(rng, 6, 48, IN)
    sw, w = mx.MXSwitchLinear(*_dev(codes, scales), IN), mc.values(codes, scales, IN)
    x, xv = mc.acts(rng, "bf16", T, 1, 1, IN)
    ids = rng.integers(1, 6, (T, k))
    ids[rng.random((T, k)) < 0.4] = -1
    ids[0, 0], ids[T - 1, k - 1] = -1, 6
    y = sw(x, *_dev(ids))
    for t in range(T):
        for j in range(k):
            if 1 <= ids[t, j] < 6:
                ref, bar = mc.product_bar(xv[t, 0], w[ids[t, j]], "bf16")
                mc.assert_within(y[t, j], ref, bar, f"pair {t}, {j}")
            else:
                assert (y[t, j] == 0).all()


@pytest.mark.parametrize("T", [1, 5, 40])
def test_an_expert_that_nobody_chose_changes_nothing(T):
    from vqlab_amd import mx
    rng = np.random.default_rng(T)
    E, H, I, k = 6, 160, 96, 3
    mods, ws = [], []
    for OUT, IN in ((I, H), (I, H), (H, I)):
        codes, scales = _huge(rng, E, OUT, IN)
        mods.append(mx.MXSwitchLinear(*_dev(codes, scales), IN))
        ws.append(mc.values(codes, scales, IN))
    glu = mx.MXSwitchGLU(*mods)
    x, xv = mc.acts(rng, "bf16", T, H)
    ids = np.stack([1 + rng.permutation(E - 1)[:k] for _ in range(T)])
    ids[0, 1] = -1
    w = rng.random((T, k)).astype(np.float32)
    ref, bar = mc.experts(xv, ids, w.astype(np.float64), *ws, mc.HALF_STEP["bf16"])
    mc.assert_within(glu(x, *_dev(ids, w)), ref, bar + mc.HALF_STEP["bf16"] * (np.abs(ref) + bar), "experts")


@pytest.mark.parametrize("N", [1, 2, 9, 20, 70])
@pytest.mark.parametrize("IN", [640, 1152, 5248])
def test_an_infinite_weight_in_the_last_chunk(N, IN):
    """Products of positive x with a weight of 2^128 or more are infinite, not NaN."""
    from vqlab_amd import mx
    rng = np.random.default_rng(N + IN)
    codes, scales = mc.weight(rng, 40, IN)
    codes[7, -16:], scales[7, -1] = 0x77, 254
    codes[20, -16:], scales[20, -1] = 0xff, 253
    lin = mx.MXLinear(*_dev(codes, scales), IN)
    x = (mc.acts(rng, "bf16", N, IN)[0].abs() + 0.5)
    y = lin(x).float().cpu().numpy()
    assert (y[:, 7] == np.inf).all() and (y[:, 20] == -np.inf).all()
    rest = np.delete(np.arange(40), [7, 20])
    ref, bar = mc.product_bar(x.double().cpu().numpy(), mc.values(codes, scales, IN)[rest], "bf16")
    mc.assert_within(y[:, rest], ref, bar, "other rows")


@pytest.mark.parametrize("N", [20, 70, 200])
def test_4_bit_products_of_huge_weights(N):
    """From 65 rows on the matrix instruction takes both scales as they are: a product that fits is
    finite. Fewer rows multiply by the values, which are infinite."""
    from vqlab_amd import mx
    rng = np.random.default_rng(N)
    codes, scales = mc.weight(rng, 40, 96)
    codes[7], scales[7] = 0x77, 254
    lin = mx.MXLinear(*_dev(codes, scales), 96, act="mxfp4")
    x = ((mc.acts(rng, "fp32", N, 96)[0].abs() + 0.5) * 2.0 ** -100)
    y = lin(x)
    q = mc.values(*mc.quantize(x.double().cpu().numpy()), 96)
    ref, bar = mc.product_bar(q, mc.values(codes, scales, 96), "fp32")
    if N < 65:
        assert (y[:, 7] == float("inf")).all()
        ref, bar, y = np.delete(ref, 7, 1), np.delete(bar, 7, 1), y[:, [i for i in range(40) if i != 7]]
    mc.assert_within(y, ref, bar, "huge weights")


# ------------------------------------------------ tiles, planes, many experts
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("exact", [True, False])
@pytest.mark.parametrize("counts", [(5, 16, 17, 32), (10, 30, 40, 60), (20, 50, 90, 120), (1, 64, 65, 300)])
def test_every_way_a_tile_holds_its_planes(dtype, exact, counts):
    """Experts with 1..4 groups of 32 rows in tiles of 32, 64 and 128, x and SwiGLU rows in one, two
    and three planes (exact: whether the weights are fp16 numbers)."""
    rng = np.random.default_rng(sum(counts))
    E, H, I = len(counts), 160, 288
    glu, ws = _glu(rng, E, H, I)
    if not exact:
        from vqlab_amd import mx
        mods = []
        for i, (m, w) in enumerate(zip((glu.gate_proj, glu.up_proj, glu.down_proj), ws)):
            scales = m.scales.cpu().numpy()
            scales[:, ::5] = 90
            codes = m.codes.cpu().numpy()
            mods.append(mx.MXSwitchLinear(*_dev(codes, scales), m.input_dims))
            assert not mods[-1]._w.f16_exact
            ws = (*ws[:i], mc.values(codes, scales, m.input_dims), *ws[i + 1:])
        glu = mx.MXSwitchGLU(*mods)
    ids = rng.permutation(np.repeat(np.arange(E), counts))[:, None]
    x, xv = mc.acts(rng, dtype, len(ids), H)
    w = rng.random((len(ids), 1)).astype(np.float32)
    ref, bar = mc.experts(xv, ids, w.astype(np.float64), *ws, H_ROUND[dtype])
    bar = bar + mc.HALF_STEP[dtype] * (np.abs(ref) + bar) + (2.0 ** -25 if dtype == "fp16" else 0.0)
    mc.assert_within(glu(x, *_dev(ids, w)), ref, bar, "experts")


@pytest.mark.parametrize("T,k", [(3, 4), (1000, 4), (2100, 4)])
def test_the_most_experts(T, k):
    rng = np.random.default_rng(T)
    E, H, I = 4096, 33, 16
    glu, ws = _glu(rng, E, H, I)
    x, xv = mc.acts(rng, "bf16", T, H)
    ids = rng.integers(0, E, (T, k))
    ids[0] = [0, E - 1, E, -1]
    w = rng.random((T, k)).astype(np.float32)
    ref, bar = mc.experts(xv, ids, w.astype(np.float64), *ws, H_ROUND["bf16"])
    mc.assert_within(glu(x, *_dev(ids, w)), ref, bar + mc.HALF_STEP["bf16"] * (np.abs(ref) + bar), "experts")


def test_a_block_of_the_most_experts_and_choices_it_routes():
    from vqlab_amd import mx
    rng = np.random.default_rng(11)
    E, H, I = 2048, 32, 16
    glu, ws = _glu(rng, E, H, I)
    for T, k in ((2, 64), (90, 64)):
        x, xv = mc.acts(rng, "bf16", T, H)
        lg = rng.standard_normal((T, E)).astype(np.float32)
        r = mc.route(lg, k)
        ref, bar = mc.experts(xv, r["ids"], r["w"], *ws, H_ROUND["bf16"])
        # weights, which sum to 1: exp of a difference rounded once (2 max |l| of it), sums of k terms;
        # so many parts of the largest expert's output
        g, u = (np.einsum("th,eih->tei", xv, m) for m in ws[:2])
        most = np.abs(np.einsum("tei,ehi->teh", g / (1 + np.exp(-g)) * u, ws[2])).max(1)
        bar = bar + (2 * np.abs(lg).max() + 8 + k) * 2.0 ** -24 * most
        bar = bar + mc.HALF_STEP["bf16"] * (np.abs(ref) + bar)
        mc.assert_within(mx.MXSparseMoeBlock(glu, k)(x, *_dev(lg)), ref, bar, "block")
    with pytest.raises(NotImplementedError):
        mx.MXSparseMoeBlock(glu, 65)(x, *_dev(lg))
