"""8-bit rows, weights and linears on the GPU against float64 oracles: every type, odd sizes, blocks
at the ends of the range, strides, streams, captured graphs."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import f8_cases as fc
import mx_cases as mc

pytestmark = pytest.mark.gpu

TYPES = ["bf16", "fp16", "fp32"]


def _dev(*arrays):
    return tuple(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays)


def _linear(rng, OUT, IN, act=None, spread=4):
    from vqlab_amd import fp8
    codes, scales, w = fc.weight(rng, OUT, IN, spread)
    return fp8.F8Linear(*_dev(codes, scales), act), w


def _a8_bar(lin, x, dtype):
    """y of x in 8 bits through lin, and its bar."""
    q, s = fc.quantize(x.float().cpu().numpy().reshape(-1, x.shape[-1]))
    w8, sw = _code_values(lin.codes), lin.scales.cpu().numpy()
    y, bar = fc.product_bar(fc.row_values(q, s), fc.weight_values(w8, sw), dtype)
    return y, bar if dtype == "fp32" else bar + 1.01 * fc.instruction_bar(q, s, w8, sw)


def _code_values(codes):
    return fc.decode(codes.view(torch.uint8).cpu().numpy())


def _same(rows, x):
    q, s = fc.quantize(x)
    assert np.array_equal(rows.scales.cpu().numpy().reshape(s.shape), s, equal_nan=True)
    assert np.array_equal(_code_values(rows.codes).reshape(q.shape), q)
    return q, s


# ------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (5, 129), (2, 256), (7, 300), (1, 4096), (17, 1000),
                                       (4, 2055), (600, 136)])
def test_quantize_matches_the_format(dtype, rows, cols):
    from vqlab_amd import fp8
    rng = np.random.default_rng(rows * 7919 + cols)
    x, _ = mc.acts(rng, dtype, rows, cols)
    x *= torch.exp2(torch.randint(-6, 7, (rows, 1), device="cuda")).to(x.dtype)
    got = fp8.f8_quantize(x)
    assert got.codes.dtype == torch.float8_e4m3fn and got.codes.shape == x.shape
    q, s = _same(got, x.float().cpu().numpy())
    for out in TYPES:
        back = fp8.f8_dequantize(*got, mc.torch_dtype(out))
        want = torch.from_numpy((q.astype(np.float32) * np.repeat(s, 128, 1)[:, :cols])).to(back.dtype)
        assert torch.equal(back.cpu(), want)


def test_quantize_borders_and_special_blocks():
    """Every border between two codes and its neighbours under a scale of 1, zeros of both signs, the
    type's extremes, infinities and NaN."""
    from vqlab_amd import fp8
    codes = fc.decode(np.arange(127).astype(np.uint8))
    mid = (codes[1:] + codes[:-1]) / 2
    x = np.concatenate([codes, mid, np.nextafter(mid.astype(np.float32), np.float32(0)).astype(np.float64),
                        np.nextafter(mid.astype(np.float32), np.float32(1e9)).astype(np.float64)])
    x = np.concatenate([x, -x])
    n = -(-x.size // 127)
    b = np.zeros((n, 128))
    b.reshape(n, 128)[:, 0] = 448.0                        # scale 1
    b[:, 1:].reshape(-1)[:0] = 0
    flat = np.zeros(n * 127)
    flat[:x.size] = x
    b[:, 1:] = flat.reshape(n, 127)
    x = torch.from_numpy(b.astype(np.float32)).cuda()
    _same(fp8.f8_quantize(x), b)
    big = torch.finfo(torch.float32).max
    y = torch.zeros(9, 128, device="cuda")
    y[1] = -0.0
    y[2, 5], y[3] = big, 2.0 ** -149
    y[4, 1], y[4, 2] = 448 * 2.0 ** -126, 2.0 ** -126
    y[5, 9], y[6, 3], y[7, 0] = float("inf"), float("nan"), float("-inf")
    y[8] = 2.0 ** -130
    rows = fp8.f8_quantize(y)
    _same(rows, y.cpu().numpy())
    back = fp8.f8_dequantize(*rows, torch.float32).cpu().numpy()
    assert np.isnan(back[5:8]).all() and np.isfinite(np.delete(back, [5, 6, 7], 0)).all()
    assert (back[0] == 0).all() and float(rows.scales[0, 0]) == 2.0 ** -126


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided_rows_and_lead_dimensions(dtype):
    from vqlab_amd import fp8
    rng = np.random.default_rng(5)
    x, _ = mc.acts(rng, dtype, 6, 3, 301)
    for view in (x[:, 1], x[:, 1, 4:297], x.transpose(0, 1), x[::2, :, ::3], x[2, 1]):
        rows = fp8.f8_quantize(view)
        assert rows.codes.shape == view.shape and rows.scales.shape == (*view.shape[:-1], -(-view.shape[-1] // 128))
        _same(rows, view.float().cpu().numpy().reshape(-1, view.shape[-1]))
        assert torch.equal(fp8.f8_dequantize(*rows, torch.float32).reshape(-1, view.shape[-1]),
                           fp8.f8_dequantize(rows.codes.reshape(-1, view.shape[-1]),
                                             rows.scales.reshape(-1, rows.scales.shape[-1]), torch.float32))
    assert fp8.f8_quantize(x[:0]).scales.shape == (0, 3, 3) and fp8.f8_quantize(x[..., :0]).codes.shape == (6, 3, 0)
    assert fp8.f8_dequantize(*fp8.f8_quantize(x[:0])).shape == (0, 3, 301)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("O,I", [(1, 1), (128, 128), (127, 129), (300, 260), (40, 1000), (513, 72)])
def test_quantize_weight(dtype, O, I):
    from vqlab_amd import fp8
    rng = np.random.default_rng(O + I)
    w, wv = mc.acts(rng, dtype, O, I)
    codes, scales = fp8.f8_quantize_weight(w)
    q, s = fc.quantize_weight(wv)
    assert np.array_equal(scales.cpu().numpy(), s)
    assert np.array_equal(_code_values(codes), q)
    back = fp8.f8_dequantize(codes, scales, torch.float32).double().cpu().numpy()
    assert np.array_equal(back, fc.weight_values(q, s).astype(np.float32))
    lin = fp8.F8Linear.from_weight(w)
    assert torch.equal(lin.codes.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(lin.scales, scales)


# ------------------------------------------------------------------- linear
SHAPES = [(1, 16, 32), (1, 64, 4096), (2, 33, 1), (3, 17, 95), (16, 48, 160), (17, 100, 257), (31, 130, 512),
          (33, 64, 1056), (64, 80, 128), (65, 40, 224), (97, 300, 136), (130, 272, 640), (300, 129, 1000),
          (260, 520, 384),
          # every split of k over the waves, rows too long for them, and x through LDS to its last block
          (1, 32, 8192), (3, 32, 8192), (9, 48, 6144), (16, 16, 5120), (20, 33, 8200), (2, 40, 17408), (5, 24, 768),
          (12, 20, 1536), (18, 40, 2048), (30, 40, 3000), (32, 16, 4096), (7, 40, 896), (1, 70000, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,OUT,IN", SHAPES)
def test_linear(dtype, N, OUT, IN):
    rng = np.random.default_rng(N * 1009 + OUT * 31 + IN)
    lin, w = _linear(rng, OUT, IN)
    x, xv = mc.acts(rng, dtype, N, IN)
    y, bar = fc.product_bar(xv, w, dtype)
    mc.assert_within(lin(x), y, bar, "linear")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,OUT,IN", SHAPES)
def test_linear_8_bit_activations(dtype, N, OUT, IN):
    """From x, and from rows that are in 8 bits already."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(N * 11 + OUT + IN)
    lin, w = _linear(rng, OUT, IN, act="fp8")
    x, _ = mc.acts(rng, dtype, N, IN)
    for out in {dtype, "fp32"}:
        y, bar = _a8_bar(lin, x, out)
        got = lin(x, out_dtype=mc.torch_dtype(out))
        mc.assert_within(got, y, bar, "a8 linear")
        assert torch.equal(lin(fp8.f8_quantize(x), out_dtype=got.dtype), got)
    assert lin(x).dtype == x.dtype


@pytest.mark.parametrize("act", [None, "fp8"])
@pytest.mark.parametrize("N", [1, 20, 70, 200])
def test_linear_far_values(N, act):
    """Rows up to the largest number of their type and weights whose scales bring the products back:
    finite throughout. Every row and every block of k has magnitudes of its own."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(N)
    IN, OUT = 384, 48
    codes, _, _ = fc.weight(rng, OUT, IN)
    scales = np.array([[2.0 ** -40, 2.0 ** -20, 2.0 ** -35]], np.float32)
    lin, w = fp8.F8Linear(*_dev(codes, scales), act), fc.weight_values(fc.decode(codes), scales)
    big = torch.finfo(torch.bfloat16).max
    x = torch.from_numpy(rng.uniform(-1, 1, (N, IN)).astype(np.float32)).to(torch.bfloat16)
    x[:, :128] *= big
    x[0, 0] = big
    x[:, 128:256] *= 2.0 ** 100
    for dtype in ("bf16", "fp32"):
        xd = x.to(mc.torch_dtype(dtype)).cuda()
        y, bar = _a8_bar(lin, xd, dtype) if act else fc.product_bar(xd.double().cpu().numpy(), w, dtype)
        mc.assert_within(lin(xd), y, bar, "far values")


@pytest.mark.parametrize("act", [None, "fp8"])
@pytest.mark.parametrize("N", [1, 20, 70, 200])
@pytest.mark.parametrize("IN", [384, 408])
def test_linear_nan_codes_and_scales_stay_in_their_rows(N, act, IN):
    """A NaN code makes its output NaN; a NaN scale those of its 128 rows."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(N + 50)
    codes, scales, _ = fc.weight(rng, 270, IN)
    codes[5, 300], codes[33, 0], codes[269, IN - 1] = 0x7f, 0xff, 0x7f
    scales[1, 2] = np.nan
    lin = fp8.F8Linear(*_dev(codes, scales), act)
    x, _ = mc.acts(rng, "bf16", N, IN)
    x[0] = 0
    y = lin(x).float().cpu().numpy()
    bad = [5, 33, 269, *range(128, 256)]
    assert np.isnan(y[:, bad]).all()
    assert np.isfinite(np.delete(y, bad, 1)).all()


@pytest.mark.parametrize("act", [None, "fp8"])
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
        if r in bad:
            assert not np.isfinite(y[r]).all() and (not act or np.isnan(y[r]).all())
        else:
            assert np.isfinite(y[r]).all()


@pytest.mark.parametrize("act", [None, "fp8"])
def test_linear_views_of_x_and_codes(act):
    """Strided x, an x and codes that start off 16 bytes, lead dimensions, empty x."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(8)
    codes, scales, w = fc.weight(rng, 24, 272)
    raw = torch.zeros(codes.size + 3, dtype=torch.uint8, device="cuda")
    raw[3:] = torch.from_numpy(codes.reshape(-1)).cuda()
    lin = fp8.F8Linear(raw[3:].reshape(24, 272), *_dev(scales), act)
    x, _ = mc.acts(rng, "bf16", 4, 6, 273)
    for view in (x[..., 1:], x[:, ::2, :272], x[1, :, 1:], x[0, 0, :272], x.reshape(-1)[5:5 + 272]):
        y, bar = _a8_bar(lin, view, "bf16") if act else fc.product_bar(view.double().cpu().numpy().reshape(-1, 272), w, "bf16")
        got = lin(view)
        assert got.shape == (*view.shape[:-1], 24)
        mc.assert_within(got.reshape(-1, 24), y, bar, "view")
    assert lin(x[:0, :, :272]).shape == (0, 6, 24)
    if act:
        rows = fp8.f8_quantize(x[..., :272])
        want = lin(x[..., :272])
        assert torch.equal(lin(rows), want)
        assert torch.equal(lin((rows.codes[1:, ::2], rows.scales[1:, ::2])), want[1:, ::2])
        assert torch.equal(lin((rows.codes, rows.scales.contiguous())), want)
        wide = torch.zeros(4, 6, 300, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        wide.view(torch.uint8)[..., 5:277] = rows.codes.view(torch.uint8)
        assert torch.equal(lin((wide[..., 5:277], rows.scales)), want)
        assert torch.equal(lin((rows.codes.view(torch.uint8), rows.scales)), want)
        assert lin(fp8.f8_quantize(x[:0, :, :272])).shape == (0, 6, 24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,OUT,IN", [(1, 32, 64), (3, 33, 95), (20, 1000, 130), (65, 100, 257), (97, 256, 128),
                                      (300, 192, 640), (130, 520, 1000), (2, 17, 1)])
def test_linear_gradient(dtype, N, OUT, IN):
    rng = np.random.default_rng(N + OUT + IN)
    lin, w = _linear(rng, OUT, IN)
    x, _ = mc.acts(rng, dtype, N, IN)
    dy, dv = mc.acts(rng, dtype, N, OUT)
    x.requires_grad_(True)
    dx = torch.autograd.grad(lin(x), x, dy)[0]
    assert dx.dtype == x.dtype
    ref, bar = fc.product_bar(dv, w.T, dtype)
    mc.assert_within(dx, ref, bar, "dx")


def test_linear_gradient_against_differences():
    """A linear map's difference quotient is its derivative, whatever the step."""
    rng = np.random.default_rng(3)
    lin, w = _linear(rng, 20, 270)
    x, xv = mc.acts(rng, "fp32", 2, 270)
    dy, dv = mc.acts(rng, "fp32", 2, 20)
    x.requires_grad_(True)
    dx = torch.autograd.grad(lin(x), x, dy)[0].double().cpu().numpy()
    _, own = fc.product_bar(dv, w.T, "fp32")
    for r, c in ((0, 0), (1, 133), (0, 269)):
        hi, lo = x.detach().clone(), x.detach().clone()
        hi[r, c] += 4
        lo[r, c] -= 4
        diff = ((lin(hi).double() - lin(lo).double()) * dy.double()).sum().item()
        step = float(hi[r, c]) - float(lo[r, c])
        _, bar = fc.product_bar(np.abs(xv) + 4, np.abs(w), "fp32")      # each y is off by its bar, twice, over the step
        assert abs(diff / step - dx[r, c]) <= 2 * (np.abs(dv) * bar).sum() / step + own[r, c]


def test_linear_output_types_and_tangents():
    from vqlab_amd import fp8
    import torch.autograd.forward_ad as fw
    rng = np.random.default_rng(4)
    lin, w = _linear(rng, 40, 256)
    x, xv = mc.acts(rng, "bf16", 5, 256)
    y, bar = fc.product_bar(xv, w, "fp32")
    assert lin(x, out_dtype=torch.float32).dtype == torch.float32
    mc.assert_within(lin(x, out_dtype=torch.float32), y, bar, "fp32 of bf16")
    g = x.clone().requires_grad_(True)
    dy = torch.randn(5, 40, device="cuda")
    dx = torch.autograd.grad(lin(g, out_dtype=torch.float32), g, dy)[0]
    assert dx.dtype == torch.bfloat16
    ref, bar = fc.product_bar(dy.double().cpu().numpy(), w.T, "bf16")
    mc.assert_within(dx, ref, bar, "bf16 dx of fp32 dy")
    with fw.dual_level():
        t, tv = mc.acts(rng, "bf16", 5, 256)
        out = fw.unpack_dual(lin(fw.make_dual(x, t)))
        ref, bar = fc.product_bar(tv, w, "bf16")
        mc.assert_within(out.tangent, ref, bar, "tangent")
    q = fp8.F8Linear(lin.codes, lin.scales, act="fp8")
    assert q(fp8.f8_quantize(x)).dtype == torch.bfloat16


def test_linear_module_state():
    """state_dict holds the rows; loading packs in place; copies, pickles and moves describe their own."""
    import copy
    import pickle
    from vqlab_amd import fp8
    rng = np.random.default_rng(6)
    codes, scales, _ = fc.weight(rng, 50, 300)
    lin = fp8.F8Linear(*_dev(codes, scales))
    sd = lin.state_dict()
    assert sorted(sd) == ["codes", "scales"]
    assert np.array_equal(sd["codes"].view(torch.uint8).cpu().numpy(), codes)
    assert np.array_equal(sd["scales"].cpu().numpy(), scales)
    x, _ = mc.acts(rng, "bf16", 7, 300)
    want = lin(x)
    other = fp8.F8Linear(*_dev(*fc.weight(rng, 50, 300)[:2]))
    assert not torch.equal(other(x), want)
    twin, at = copy.deepcopy(other), other._packed[0].data_ptr()
    other.load_state_dict(sd)
    assert torch.equal(other(x), want) and other._packed[0].data_ptr() == at
    assert not torch.equal(twin(x), want)
    assert torch.equal(pickle.loads(pickle.dumps(lin))(x), want)
    moved = copy.deepcopy(lin).cpu()
    with pytest.raises(ValueError):
        moved(x)
    assert torch.equal(moved.cuda()(x), want)
    moved.half()                                           # casts leave codes and scales what they are
    assert torch.equal(moved(x), want)
    with pytest.raises(RuntimeError, match="codes"):
        other.load_state_dict({"codes": sd["codes"][:, :200], "scales": sd["scales"]})
    with pytest.raises(RuntimeError, match="Missing"):
        other.load_state_dict({"codes": sd["codes"]})


@pytest.mark.parametrize("act", [None, "fp8"])
def test_linear_on_streams_and_in_graphs(act):
    """Two streams at once, and a captured call replayed between eager ones on new inputs."""
    rng = np.random.default_rng(9)
    lin, _ = _linear(rng, 520, 640, act)
    xs = [mc.acts(rng, "bf16", n, 640)[0] for n in (3, 40, 300)]
    want = [lin(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append([lin(x) for x in xs])
        torch.cuda.synchronize()
        for g in got:
            assert all(torch.equal(a, b) for a, b in zip(g, want))
    for i, x in enumerate(xs):
        buf = x.clone()
        neg = lin(-x)                                      # not -lin(x): the matrix cores round both ways alike
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(buf)
        for rep in range(3):
            buf.copy_(x if rep != 1 else -x)
            graph.replay()
            eager = lin(xs[(i + 1) % 3])
            torch.cuda.synchronize()
            assert torch.equal(out, want[i] if rep != 1 else neg)
            assert torch.equal(eager, want[(i + 1) % 3])


def test_linear_gradient_in_a_graph():
    rng = np.random.default_rng(10)
    lin, _ = _linear(rng, 300, 384)
    x, _ = mc.acts(rng, "bf16", 130, 384)
    dy, _ = mc.acts(rng, "bf16", 130, 300)
    x.requires_grad_(True)
    want = torch.autograd.grad(lin(x), x, dy)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(lin(x), x, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(lin(x), x, dy)[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
