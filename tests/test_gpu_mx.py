"""MXFP4 quantisation, linears and experts on the GPU against float64 oracles: every type, odd
sizes, special blocks, strides, streams and captured graphs."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mx_cases as mc

pytestmark = pytest.mark.gpu

TYPES = ["bf16", "fp16", "fp32"]


def _dev(*arrays):
    return tuple(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays)


def _linear(rng, OUT, IN, act=None, spread=3):
    from vqlab_amd import mx
    codes, scales = mc.weight(rng, OUT, IN, spread=spread)
    return mx.MXLinear(*_dev(codes, scales), IN, act), mc.values(codes, scales, IN)


# ------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 64), (7, 100), (1, 4096),
                                       (17, 992), (4, 2055)])
def test_quantize_matches_the_format(dtype, rows, cols):
    from vqlab_amd import mx
    rng = np.random.default_rng(rows * 7919 + cols)
    x, xv = mc.acts(rng, dtype, rows, cols)
    x *= torch.exp2(torch.randint(-6, 7, (rows, 1), device="cuda")).to(x.dtype)
    xv = x.double().cpu().numpy()
    codes, scales = mx.mx_quantize(x)
    rc, rs = mc.quantize(xv)
    assert np.array_equal(scales.cpu().numpy(), rs)
    assert np.array_equal(codes.cpu().numpy(), rc)
    back = mx.mx_dequantize(codes, scales, cols, x.dtype)
    assert back.shape == x.shape and back.dtype == x.dtype
    assert np.array_equal(back.double().cpu().numpy(), mc.values(rc, rs, cols))


def test_quantize_every_bf16_magnitude_under_every_scale():
    """Each finite bf16 magnitude as the largest of its block, beside fractions of it that fall on
    and next to every rounding border of the 4-bit grid."""
    from vqlab_amd import mx
    top = torch.arange(0, 0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    f = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5]) / 8
    f = torch.cat([f, f * (1 + 2.0 ** -7), f * (1 - 2.0 ** -7)])
    # powers of two carry the borders exactly; other magnitudes put the fractions anywhere
    lead = torch.exp2(torch.floor(torch.log2(top.double().clamp(min=2.0 ** -133))))
    x = torch.zeros(top.numel(), 32, dtype=torch.bfloat16)
    x[:, 0] = top
    x[:, 1:25] = (lead[:, None] * 2 * f.double()).to(torch.bfloat16)
    x[:, 1:25] = torch.minimum(x[:, 1:25], top[:, None])
    x[:, 25:] = -x[:, 1:8]
    codes, scales = mx.mx_quantize(x.cuda())
    rc, rs = mc.quantize(x.double().numpy())
    assert np.array_equal(scales.cpu().numpy(), rs)
    assert np.array_equal(codes.cpu().numpy(), rc)
    back = mx.mx_dequantize(codes, scales, 32, torch.float32).double().cpu().numpy()
    assert np.array_equal(back, mc.values(rc, rs, 32))


def test_quantize_special_blocks():
    """Zeros, signed zeros, subnormals, the largest numbers, infinities and NaN."""
    from vqlab_amd import mx
    tiny, big = np.float32(1e-45), np.finfo(np.float32).max
    x = np.zeros((8, 64), np.float32)
    x[1] = -0.0
    x[2, 3], x[2, 40] = tiny, -np.float32(2.0 ** -126)
    x[3, 0], x[3, 33] = big, -big
    x[4, 5] = np.inf
    x[5, 6] = np.nan
    x[6, 7] = -np.inf
    x[6, 40] = 1.0
    x[7] = np.linspace(-3, 3, 64)
    codes, scales = mx.mx_quantize(torch.from_numpy(x).cuda())
    rc, rs = mc.quantize(x)
    assert np.array_equal(scales.cpu().numpy(), rs) and np.array_equal(codes.cpu().numpy(), rc)
    back = mx.mx_dequantize(codes, scales, 64, torch.float32).double().cpu().numpy()
    ref = mc.values(rc, rs, 64)
    assert np.array_equal(back, ref, equal_nan=True)
    assert np.isnan(back[4, :32]).all() and not np.isnan(back[4, 32:]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided_rows_and_lead_dimensions(dtype):
    from vqlab_amd import mx
    rng = np.random.default_rng(5)
    x, _ = mc.acts(rng, dtype, 6, 3, 101)
    for view in (x[:, 1], x[:, 1, 4:97], x.transpose(0, 1), x[::2, :, ::3]):
        codes, scales = mx.mx_quantize(view)
        rc, rs = mc.quantize(view.double().cpu().numpy().reshape(-1, view.shape[-1]))
        assert codes.shape[:-1] == view.shape[:-1]
        assert np.array_equal(codes.cpu().numpy().reshape(rc.shape), rc)
        assert np.array_equal(scales.cpu().numpy().reshape(rs.shape), rs)


def test_quantize_empty():
    from vqlab_amd import mx
    for shape in ((0, 64), (3, 0), (0, 0)):
        codes, scales = mx.mx_quantize(torch.empty(shape, device="cuda"))
        assert codes.shape == (shape[0], -(-shape[1] // 32) * 16)
        assert mx.mx_dequantize(codes, scales, shape[1]).shape == shape


# ------------------------------------------------------------------- linear
SHAPES = [(1, 16, 32), (1, 64, 4096), (2, 33, 1), (3, 17, 95), (16, 48, 160), (17, 100, 257), (31, 130, 512),
          (33, 64, 1056), (64, 80, 128), (65, 40, 224), (130, 272, 640), (300, 129, 1000),
          # every split of k over the waves, rows too long for them, and x through LDS to its last chunk
          (1, 32, 8192), (3, 32, 8192), (9, 48, 6144), (16, 16, 5120), (20, 33, 8200), (2, 40, 17408), (5, 24, 768),
          (12, 20, 1536), (18, 40, 2048), (30, 40, 3000), (32, 16, 4096), (1, 70000, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,OUT,IN", SHAPES)
def test_linear(dtype, N, OUT, IN):
    rng = np.random.default_rng(N * 1009 + OUT * 31 + IN)
    lin, w = _linear(rng, OUT, IN)
    x, xv = mc.acts(rng, dtype, N, IN)
    y, bar = mc.product_bar(xv, w, dtype)
    mc.assert_within(lin(x), y, bar, "linear")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,OUT,IN", [(1, 64, 512), (5, 33, 96), (16, 40, 70), (70, 64, 256), (130, 272, 640),
                                      (257, 130, 1000), (300, 520, 1152), (65, 33, 128), (129, 257, 384),
                                      (200, 16, 4096)])
def test_linear_4_bit_activations(dtype, N, OUT, IN):
    rng = np.random.default_rng(N * 11 + OUT + IN)
    lin, w = _linear(rng, OUT, IN, act="mxfp4")
    x, xv = mc.acts(rng, dtype, N, IN)
    q = mc.values(*mc.quantize(xv), IN)
    y, bar = mc.product_bar(q, w, dtype)
    mc.assert_within(lin(x), y, bar, "a4 linear")


@pytest.mark.parametrize("act", [None, "mxfp4"])
@pytest.mark.parametrize("N", [1, 20, 70, 200])
@pytest.mark.parametrize("IN", [320, 384])
def test_linear_scales_far_apart(N, act, IN):
    """Scales over 200 powers of two, 0 (a subnormal 2^-127) among them: every weight is exact."""
    rng = np.random.default_rng(N)
    from vqlab_amd import mx
    codes, _ = mc.weight(rng, 48, IN)
    scales = rng.integers(0, 200, (48, IN // 32)).astype(np.uint8)
    lin, w = mx.MXLinear(*_dev(codes, scales), IN, act), mc.values(codes, scales, IN)
    x, xv = mc.acts(rng, "fp32", N, IN)
    if act:
        xv = mc.values(*mc.quantize(xv), IN)
    y, bar = mc.product_bar(xv, w, "fp32")
    # sums of values below fp32's normal range may be flushed: IN terms of up to 2^-126 each
    mc.assert_within(lin(x), y, bar + IN * 2.0 ** -126, "far scales")


@pytest.mark.parametrize("N", [1, 20, 70, 200])
@pytest.mark.parametrize("lo,hi", [(104, 120), (80, 120)])
def test_linear_fp16_x_and_weights_beyond_fp16(N, lo, hi):
    """Weights that are fp16 numbers down to the last subnormal, and weights that are not, among
    blocks of zeros under the smallest scale: exact either way."""
    from vqlab_amd import mx
    rng = np.random.default_rng(N + lo)
    codes, _ = mc.weight(rng, 48, 320)
    scales = rng.integers(lo, hi + 1, (48, 10)).astype(np.uint8)
    scales[0] = lo
    codes[3, :16], scales[3, 0] = 0, 0
    lin, w = mx.MXLinear(*_dev(codes, scales), 320), mc.values(codes, scales, 320)
    assert bool(lin._w.f16_exact) == (lo >= 104)
    x, xv = mc.acts(rng, "fp16", N, 320)
    y, bar = mc.product_bar(xv, w, "fp16")
    mc.assert_within(lin(x), y, bar + 2.0 ** -25, "fp16")     # half a step of fp16's subnormals


@pytest.mark.parametrize("act", [None, "mxfp4"])
@pytest.mark.parametrize("N", [1, 20, 70, 200])
@pytest.mark.parametrize("IN", [384, 416])
def test_linear_nan_blocks_stay_in_their_column(N, act, IN):
    from vqlab_amd import mx
    rng = np.random.default_rng(N + 50)
    codes, scales = mc.weight(rng, 70, IN)
    scales[5, 3] = 255
    scales[33, 0] = scales[69, 11] = 255
    lin = mx.MXLinear(*_dev(codes, scales), IN, act)
    x, _ = mc.acts(rng, "bf16", N, IN)
    x[0] = 0
    y = lin(x).float().cpu().numpy()
    assert np.isnan(y[:, [5, 33, 69]]).all()
    assert np.isfinite(np.delete(y, [5, 33, 69], 1)).all()


@pytest.mark.parametrize("act", [None, "mxfp4"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 20, 70, 200])
@pytest.mark.parametrize("IN", [200, 256])
def test_linear_not_finite_x_stays_in_its_row(dtype, N, act, IN):
    rng = np.random.default_rng(N)
    lin, _ = _linear(rng, 40, IN, act)
    x, _ = mc.acts(rng, dtype, N, IN)
    x[N // 2, 7] = float("nan")
    x[N - 1, IN - 1] = float("inf")
    bad = {N // 2, N - 1}
    y = lin(x).float().cpu().numpy()
    for r in range(N):
        assert not np.isfinite(y[r]).any() if r in bad and act else True
        assert np.isfinite(y[r]).all() if r not in bad else not np.isfinite(y[r]).all()


def test_linear_views_of_x_and_raw_codes():
    """Strided x, an x and codes that start off 16 bytes, lead dimensions, empty x."""
    from vqlab_amd import mx
    rng = np.random.default_rng(8)
    codes, scales = mc.weight(rng, 24, 96)
    raw = torch.zeros(codes.size + 3, dtype=torch.uint8, device="cuda")
    raw[3:] = torch.from_numpy(codes.reshape(-1)).cuda()
    lin = mx.MXLinear(raw[3:].reshape(24, 48), *_dev(scales), 96)
    w = mc.values(codes, scales, 96)
    x, _ = mc.acts(rng, "bf16", 4, 6, 97)
    for view in (x[..., 1:], x[:, ::2, :96], x[1, :, 1:97], x[0, 0, :96], x.reshape(-1)[5:5 + 96]):
        y, bar = mc.product_bar(view.double().cpu().numpy().reshape(-1, 96), w, "bf16")
        got = lin(view)
        assert got.shape == (*view.shape[:-1], 24)
        mc.assert_within(got.reshape(-1, 24), y, bar, "view")
    assert lin(x[:0, :, :96]).shape == (0, 6, 24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,OUT,IN", [(1, 32, 64), (3, 33, 95), (65, 100, 257), (300, 192, 640), (130, 520, 1000)])
def test_linear_gradient(dtype, N, OUT, IN):
    rng = np.random.default_rng(N + OUT + IN)
    lin, w = _linear(rng, OUT, IN)
    x, _ = mc.acts(rng, dtype, N, IN)
    dy, dv = mc.acts(rng, dtype, N, OUT)
    x.requires_grad_(True)
    dx = torch.autograd.grad(lin(x), x, dy)[0]
    ref, bar = mc.product_bar(dv, w.T, dtype)
    mc.assert_within(dx, ref, bar, "dx")


def test_linear_gradient_against_differences():
    """A linear map's difference quotient is its derivative, whatever the step."""
    rng = np.random.default_rng(3)
    lin, w = _linear(rng, 20, 70)
    x, xv = mc.acts(rng, "fp32", 2, 70)
    dy, dv = mc.acts(rng, "fp32", 2, 20)
    x.requires_grad_(True)
    dx = torch.autograd.grad(lin(x), x, dy)[0].double().cpu().numpy()
    for r, c in ((0, 0), (1, 33), (0, 69)):
        hi, lo = x.detach().clone(), x.detach().clone()
        hi[r, c] += 4
        lo[r, c] -= 4
        diff = ((lin(hi).double() - lin(lo).double()) * dy.double()).sum().item()
        step = float(hi[r, c]) - float(lo[r, c])
        # each y is off by its bar, twice, over the step
        _, bar = mc.product_bar(np.abs(xv) + 4, np.abs(w), "fp32")
        _, own = mc.product_bar(dv, w.T, "fp32")
        assert abs(diff / step - dx[r, c]) <= 2 * (np.abs(dv) * bar).sum() / step + own[r, c]


def test_linear_backward_twice_and_other_leaves():
    """The gradient reaches a leaf behind another operation and adds up over two uses."""
    rng = np.random.default_rng(4)
    lin, w = _linear(rng, 32, 64)
    x, xv = mc.acts(rng, "fp32", 5, 64)
    x.requires_grad_(True)
    (lin(2 * x).sum() + lin(x).sum()).backward()
    ref, bar = mc.product_bar(np.full((5, 32), 3.0), w.T, "fp32")
    mc.assert_within(x.grad, ref, 2 * bar, "sum of uses")


# ------------------------------------------------------------------ experts
def _switch(rng, E, OUT, IN):
    from vqlab_amd import mx
    codes, scales = mc.weight(rng, E, OUT, IN)
    return mx.MXSwitchLinear(*_dev(codes, scales), IN), mc.values(codes, scales, IN)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,E,OUT,IN", [(1, 1, 1, 16, 32), (1, 4, 8, 33, 95), (9, 3, 5, 64, 160),
                                          (40, 6, 16, 48, 256), (200, 2, 3, 40, 70), (150, 8, 9, 144, 288)])
def test_switch_linear(dtype, T, k, E, OUT, IN):
    rng = np.random.default_rng(T + k + E)
    sw, w = _switch(rng, E, OUT, IN)
    x, xv = mc.acts(rng, dtype, T, 1, 1, IN)
    idx = rng.integers(-1, E + 1, (T, k))                   # ids outside [0, E) among them
    y = sw(x, torch.from_numpy(idx).cuda())
    assert y.shape == (T, k, 1, OUT)
    for t in range(T):
        for j in range(k):
            e = idx[t, j]
            if 0 <= e < E:
                ref, bar = mc.product_bar(xv[t, 0], w[e], dtype)
                mc.assert_within(y[t, j], ref, bar, f"pair {t}, {j}")
            else:
                assert (y[t, j] == 0).all()
    xk, xkv = mc.acts(rng, dtype, T, k, 1, IN)               # a row for each pair
    y = sw(xk, torch.from_numpy(idx.astype(np.int32)).cuda())
    for t in range(0, T, 7):
        for j in range(k):
            if 0 <= idx[t, j] < E:
                ref, bar = mc.product_bar(xkv[t, j], w[idx[t, j]], dtype)
                mc.assert_within(y[t, j], ref, bar, f"row {t}, {j}")


def _glu(rng, E, H, I):
    from vqlab_amd import mx
    (g, gw), (u, uw), (d, dw) = _switch(rng, E, I, H), _switch(rng, E, I, H), _switch(rng, E, H, I)
    return mx.MXSwitchGLU(g, u, d), (gw, uw, dw)


EXPERTS = [(1, 1, 1, 32, 32), (1, 8, 32, 256, 64), (3, 4, 6, 95, 33), (4, 10, 64, 512, 128), (11, 6, 16, 128, 96),
           (70, 2, 40, 160, 64), (64, 8, 12, 256, 160), (300, 4, 6, 64, 32), (257, 3, 8, 100, 70),
           # rows too long for the streaming kernel, by pair and sorted; few pairs of many chunks; tiles of 32
           (2, 2, 3, 8192, 32), (30, 2, 12, 8200, 40), (100, 4, 60, 640, 96), (90, 6, 50, 7000, 32), (2, 6, 9, 64, 4096), (40, 4, 10, 64, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,E,H,I", EXPERTS)
def test_experts(dtype, T, k, E, H, I):
    rng = np.random.default_rng(T * 3 + k + E + H)
    glu, ws = _glu(rng, E, H, I)
    x, xv = mc.acts(rng, dtype, T, H)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)])
    if T > 2:
        ids[1, 0], ids[T - 1] = -1, E                      # a pair and a token without an expert
        ids[T // 2] = ids[0]
    w = rng.random((T, k)).astype(np.float32)
    w[ids < 0] = np.nan                                    # not read
    y = glu(x, *_dev(ids, w))
    ref, bar = mc.experts(xv, ids, np.nan_to_num(w.astype(np.float64)), *ws, mc.HALF_STEP[dtype])
    mc.assert_within(y, ref, bar + mc.HALF_STEP[dtype] * (np.abs(ref) + bar), "experts")
    if T > 2:
        assert (y[T - 1] == 0).all()


def test_experts_all_tokens_on_one_expert_and_the_same_twice():
    rng = np.random.default_rng(17)
    glu, ws = _glu(rng, 8, 64, 64)
    x, xv = mc.acts(rng, "bf16", 150, 64)
    ids = np.full((150, 2), 5)
    w = np.full((150, 2), 0.5, np.float32)
    y = glu(x, *_dev(ids, w))
    ref, bar = mc.experts(xv, ids, w.astype(np.float64), *ws, mc.HALF_STEP["bf16"])
    mc.assert_within(y, ref, bar + mc.HALF_STEP["bf16"] * (np.abs(ref) + bar), "one expert")
    assert torch.equal(y, glu(x, *_dev(ids, w)))


def test_block_routes_and_masks():
    """Router and experts together: a padded batch, whose padding may hold anything."""
    from vqlab_amd import mx
    rng = np.random.default_rng(23)
    glu, ws = _glu(rng, 24, 128, 64)
    blk = mx.MXSparseMoeBlock(glu, top_k=4)
    for T in (1, 9, 60, 200):
        x, xv = mc.acts(rng, "bf16", T, 128)
        lg = rng.standard_normal((T, 24)).astype(np.float32)
        mask = rng.random(T) < 0.8
        x[torch.from_numpy(~mask).cuda()] = float("nan")
        lg[~mask] = np.nan
        y = blk(x, *_dev(lg), mask=torch.from_numpy(mask).cuda())
        r = mc.route(lg, 4, True, mask)
        ref, bar = mc.experts(np.nan_to_num(xv), r["ids"], r["w"], *ws, mc.HALF_STEP["bf16"])
        # the routing weights are off by exp and three fp32 roundings
        bar += 64 * 2.0 ** -24 * np.abs(ref) + mc.HALF_STEP["bf16"] * (np.abs(ref) + bar)
        mc.assert_within(y, ref, bar, f"block T={T}")
        assert (y[torch.from_numpy(~mask).cuda()] == 0).all()


# ---------------------------------------------------- streams and captures
def _eager_and_replays(make, n=3):
    """make() -> (run, refill): run() returns outputs; refill(i) puts new inputs in place."""
    run, refill = make()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for i in range(n):
        refill(i)
        g.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in out]
        for a, b in zip(kept, run()):
            assert torch.equal(a, b), f"replay {i}"
        torch.cuda.synchronize()


@pytest.mark.parametrize("N", [1, 40, 200])
@pytest.mark.parametrize("act", [None, "mxfp4"])
def test_linear_captured(N, act):
    def make():
        rng = np.random.default_rng(1)
        lin, _ = _linear(rng, 96, 256, act)
        x, _ = mc.acts(rng, "bf16", N, 256)

        def refill(i):
            x.copy_(mc.acts(np.random.default_rng(i + 9), "bf16", N, 256)[0])
        return (lambda: [lin(x)]), refill
    _eager_and_replays(make)


@pytest.mark.parametrize("T", [1, 12, 100])
def test_block_captured(T):
    from vqlab_amd import mx

    def make():
        rng = np.random.default_rng(1)
        glu, _ = _glu(rng, 16, 128, 64)
        blk = mx.MXSparseMoeBlock(glu, top_k=4)
        x, _ = mc.acts(rng, "bf16", T, 128)
        lg = torch.randn(T, 16, device="cuda")

        def refill(i):
            x.copy_(mc.acts(np.random.default_rng(i + 9), "bf16", T, 128)[0])
            lg.normal_()
        return (lambda: [blk(x, lg)]), refill
    _eager_and_replays(make)


def test_on_two_streams_at_once():
    rng = np.random.default_rng(2)
    lin, w = _linear(rng, 128, 512)
    glu, _ = _glu(rng, 8, 128, 64)
    xs = [mc.acts(rng, "fp16", 100, 512)[0] for _ in range(2)]
    ref = [lin(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(lin(x))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, ref[i % 2])


# ----------------------------------------------------------------- refusals
def test_what_has_no_gradient_says_so():
    from vqlab_amd import mx
    rng = np.random.default_rng(6)
    x, _ = mc.acts(rng, "bf16", 4, 64)
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        mx.mx_quantize(x)
    lin, _ = _linear(rng, 32, 64, act="mxfp4")
    with pytest.raises(RuntimeError, match="no gradient"):
        lin(x)
    glu, _ = _glu(rng, 4, 64, 32)
    ids, w = _dev(np.zeros((4, 2), np.int32), np.ones((4, 2), np.float32))
    with pytest.raises(RuntimeError, match="no gradient"):
        glu(x, ids, w)
    with pytest.raises(RuntimeError, match="no gradient"):
        glu(x.detach(), ids, w.requires_grad_(True))
    with pytest.raises(RuntimeError, match="no gradient"):
        mx.MXSparseMoeBlock(glu, 2)(x, torch.randn(4, 4, device="cuda"))
    with pytest.raises(RuntimeError, match="no gradient"):
        glu.gate_proj(x[:, None, None], ids)
    with torch.no_grad():
        assert lin(x).shape == (4, 32) and glu(x, ids, w).shape == (4, 64)
    plain, _ = _linear(rng, 32, 64)
    d = torch.autograd.grad(plain(x).float().square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):                      # once differentiable
        d.sum().backward()


def test_shapes_and_types_that_do_not_fit():
    from vqlab_amd import mx
    rng = np.random.default_rng(7)
    lin, _ = _linear(rng, 32, 64)
    glu, _ = _glu(rng, 4, 64, 32)
    f = torch.zeros(4, 64, device="cuda")
    for bad in (f[:, :63], f.double(), f.cpu(), torch.zeros((), device="cuda")):
        with pytest.raises(ValueError):
            lin(bad)
    ids, w = _dev(np.zeros((4, 2), np.int32), np.ones((4, 2), np.float32))
    for x, i, v in ((f[:, :32], ids, w), (f[:3], ids, w), (f, ids[:, :1], w), (f[0], ids, w), (f, ids.cpu(), w)):
        with pytest.raises(ValueError):
            glu(x, i, v)
    blk = mx.MXSparseMoeBlock(glu, top_k=2)
    for lg, m in ((torch.zeros(4, 5, device="cuda"), None), (torch.zeros(3, 4, device="cuda"), None),
                  (torch.zeros(4, 4, device="cuda"), torch.ones(3, dtype=torch.bool, device="cuda")),
                  (torch.zeros(4, 4, device="cuda"), torch.ones(4, device="cuda"))):
        with pytest.raises(ValueError):
            blk(f, lg, mask=m)
    with pytest.raises(ValueError):
        mx.MXSparseMoeBlock(glu, top_k=5)(f, torch.zeros(4, 4, device="cuda"))
    with pytest.raises(ValueError):
        glu.gate_proj(f, ids)
    with pytest.raises(ValueError):
        mx.mx_dequantize(*mx.mx_quantize(f), 65)
    with pytest.raises(ValueError):
        mx.mx_dequantize(*mx.mx_quantize(f), 64, torch.float64)


def test_block_from_router_weight_and_no_tokens():
    from vqlab_amd import mx
    rng = np.random.default_rng(8)
    glu, ws = _glu(rng, 6, 64, 32)
    rw = torch.randn(6, 64, device="cuda")
    blk = mx.MXSparseMoeBlock(glu, top_k=2, norm_topk_prob=False, router_weight=rw)
    x, xv = mc.acts(rng, "fp32", 5, 64)
    assert torch.equal(blk(x), blk(x, x.float() @ rw.T))
    assert blk(x[:0]).shape == (0, 64)
    logits = (x.float() @ rw.T).double().cpu().numpy()
    r = mc.route(logits, 2, False)
    ref, bar = mc.experts(xv, r["ids"], r["w"], *ws, 2.0 ** -24)
    bar += 64 * 2.0 ** -24 * np.abs(ref) + 2.0 ** -24 * (np.abs(ref) + bar)
    mc.assert_within(blk(x), ref, bar, "block")


def test_experts_with_weights_beyond_fp16():
    """fp16 x where only some of the projections hold fp16 numbers: pairs and sorted."""
    from vqlab_amd import mx
    rng = np.random.default_rng(9)
    H, I, E = 96, 64, 5

    def sw(OUT, IN, lo):
        codes, scales = mc.weight(rng, E, OUT, IN)
        scales[rng.random(scales.shape) < 0.2] = lo
        return mx.MXSwitchLinear(*_dev(codes, scales), IN), mc.values(codes, scales, IN)
    for los in ((118, 118, 90), (90, 118, 118), (118, 90, 118), (90, 90, 90)):
        (g, gw), (u, uw), (d, dw) = sw(I, H, los[0]), sw(I, H, los[1]), sw(H, I, los[2])
        assert [bool(m._w.f16_exact) for m in (g, u, d)] == [lo > 104 for lo in los]
        glu = mx.MXSwitchGLU(g, u, d)
        for T in (3, 60):
            x, xv = mc.acts(rng, "fp16", T, H)
            ids = np.stack([rng.permutation(E)[:2] for _ in range(T)])
            w = rng.random((T, 2)).astype(np.float32)
            ref, bar = mc.experts(xv, ids, w.astype(np.float64), gw, uw, dw, mc.HALF_STEP["fp16"])
            bar = bar + mc.HALF_STEP["fp16"] * (np.abs(ref) + bar) + 2.0 ** -25
            mc.assert_within(glu(x, *_dev(ids, w)), ref, bar, f"{los} T={T}")


def test_copies_stand_alone():
    """A copied or pickled module describes its own weights, after the first one is gone."""
    import copy
    import io
    from vqlab_amd import mx
    rng = np.random.default_rng(12)
    lin, w = _linear(rng, 40, 96)
    glu, _ = _glu(rng, 6, 64, 32)
    blk = mx.MXSparseMoeBlock(glu, top_k=2)
    x, xv = mc.acts(rng, "bf16", 7, 96)
    z, lg = torch.randn(5, 64, device="cuda"), torch.randn(5, 6, device="cuda")
    ref = blk(z, lg)
    twin, blk2 = copy.deepcopy(lin), copy.deepcopy(blk)
    buf = io.BytesIO()
    torch.save(lin, buf)
    lin._packed[0].zero_()
    glu.down_proj._packed[0].zero_()
    assert torch.equal(blk2(z, lg), ref)
    y, bar = mc.product_bar(xv, w, "bf16")
    mc.assert_within(twin(x), y, bar, "copy")
    buf.seek(0)
    mc.assert_within(torch.load(buf, weights_only=False)(x), y, bar, "pickle")


def test_no_rows_keep_their_gradient():
    rng = np.random.default_rng(13)
    lin, _ = _linear(rng, 40, 96)
    x = torch.zeros(0, 96, device="cuda", requires_grad=True)
    y = lin(x)
    assert y.shape == (0, 40) and torch.autograd.grad(y.sum(), x)[0].shape == (0, 96)


def test_more_tokens_than_a_grid_dimension():
    rng = np.random.default_rng(14)
    glu, ws = _glu(rng, 2, 32, 32)
    T = 70001
    x, xv = mc.acts(rng, "bf16", T, 32)
    ids = rng.integers(0, 2, (T, 1))
    y = glu(x, *_dev(ids, np.full((T, 1), 0.5, np.float32)))
    for part in (slice(0, 40), slice(65500, 65600), slice(T - 40, T)):
        ref, bar = mc.experts(xv[part], ids[part], np.full((T, 1), 0.5)[part], *ws, mc.HALF_STEP["bf16"])
        mc.assert_within(y[part], ref, bar + mc.HALF_STEP["bf16"] * (np.abs(ref) + bar), str(part))
