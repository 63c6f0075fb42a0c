"""RMS norm with its residual, in 8 bits and as it is, on the GPU against float64: every type, every
number of waves and pieces, strides, ends of the range, gradients against the formula and differences."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import f8_cases as fc
import mx_cases as mc

pytestmark = pytest.mark.gpu

TYPES = ["bf16", "fp16", "fp32"]
EPS = 2.0 ** -24
# every instance of waves and pieces (more than 1024 rows: four pieces a lane), odd ends
SHAPES = [(1, 1), (1, 8), (3, 511), (2, 512), (5, 1000), (4, 2048), (3, 4095), (2, 4096), (3, 8192), (2, 8200), (2, 16384),
          (1, 16383), (1500, 24), (1030, 1001), (1100, 2056), (1025, 4104), (1026, 8200)]


def _inputs(rng, dtype, N, C, res=True):
    x, xv = mc.acts(rng, dtype, N, C)
    w = torch.from_numpy((1 + 0.2 * rng.standard_normal(C)).astype(np.float32)).to(x.dtype).cuda()
    r, rv = mc.acts(rng, dtype, N, C) if res else (None, None)
    return x, xv, w, w.double().cpu().numpy(), r, rv


def _round(dtype):
    return lambda v: torch.from_numpy(v).to(mc.torch_dtype(dtype)).double().numpy()


def _step(dtype, v):
    """Half a step of rounding v into dtype (fp16: below 2^-14 half of 2^-24)."""
    s = mc.HALF_STEP[dtype] * np.abs(v)
    return np.maximum(s, 2.0 ** -25) if dtype == "fp16" else s


def _check(y, h, x, res, w, dtype, eps):
    """h is exact: one rounding of a sum of two numbers (fp32 holds 24 bits of it before: a sum of two
    16-bit numbers is rounded twice, by at most an fp32 half step more). y: the mean is summed in fp64;
    r, h r and its product with w are rounded once each."""
    hv = h.double().cpu().numpy() if h is not None else x
    if res is not None:
        s = x + res
        mc.assert_within(h, s, (1 + 2.0 ** -10) * _step(dtype, s) + 2.0 ** -24 * np.abs(s), "h")
    _, r, ref = fc.norm(hv, None, w, eps, None)
    err = 4 * EPS * np.abs(ref)
    mc.assert_within(y, ref, err + 1.01 * _step(dtype, ref), "y")
    return hv, r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,C", SHAPES)
def test_norm(dtype, N, C):
    from vqlab_amd import fp8
    rng = np.random.default_rng(N * 31 + C)
    x, xv, w, wv, res, rv = _inputs(rng, dtype, N, C)
    y, h = fp8.rms_norm(x, w, 1e-6, residual=res)
    assert y.dtype == h.dtype == x.dtype
    _check(y, h, xv, rv, wv, dtype, 1e-6)
    _check(fp8.rms_norm(x, w, 1e-3), None, xv, None, wv, dtype, 1e-3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,C", SHAPES)
def test_norm_in_8_bits(dtype, N, C):
    """The 8-bit form of a y that is right to 4 fp32 roundings: scales right to as many and their own, a
    code next to a border may fall on its other side (half a step either way, of the code's own size)."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(N * 37 + C)
    x, xv, w, wv, res, rv = _inputs(rng, dtype, N, C)
    rows, h = fp8.rms_norm_f8(x, w, 1e-6, residual=res)
    y32, h2 = fp8.rms_norm(x, w, 1e-6, residual=res)
    assert torch.equal(h, h2)
    _, _, ref = fc.norm(h.double().cpu().numpy(), None, wv, 1e-6, None)
    B = -(-C // 128)
    top = np.abs(np.pad(ref, ((0, 0), (0, -C % 128)))).reshape(N, B, 128).max(-1)
    assert rows.codes.shape == x.shape and rows.scales.shape == (N, B)
    mc.assert_within(rows.scales, np.maximum(top / 448, 2.0 ** -126), 6 * EPS * top / 448, "scales")
    back = fp8.f8_dequantize(*rows, torch.float32).double().cpu().numpy()
    s = np.repeat(rows.scales.double().cpu().numpy(), 128, 1)[:, :C]
    # half a step of the code (2^-4 of the value, 2^-10 among e4m3's subnormals) and the fp32 roundings
    bar = np.maximum(2.0 ** -4 * np.abs(ref), 2.0 ** -10 * s) * (1 + 2.0 ** -10) + 10 * EPS * np.abs(ref)
    assert (np.abs(back - ref) <= bar).all()
    if dtype == "fp32":                                    # the quantiser's own codes of that very y
        q = fp8.f8_quantize(y32)
        assert torch.equal(q.codes.view(torch.uint8), rows.codes.view(torch.uint8)) and torch.equal(q.scales, rows.scales)
    alone = fp8.rms_norm_f8(h, w)
    assert torch.equal(alone.codes.view(torch.uint8), rows.codes.view(torch.uint8))


def _grad_bar(h, r, w, dy, dh, dtype):
    """dx, dw and bars: g, xhat, their product and the row's sum (a tree: log2 C + 8 additions of at most
    8 terms each in a lane) are fp32; dw sums rows in fp32 within a workgroup, at most N additions."""
    dx, dw = fc.norm_grad(h, r, w, dy, dh)
    xh, g = np.abs(h * r), np.abs(dy * w)
    N, C = h.shape
    n = np.log2(C) + 40
    mean = (g * xh).mean(1, keepdims=True)
    err = EPS * (r * (4 * g + xh * (n + 6) * mean) + np.abs(dx) + (0 if dh is None else np.abs(dh)))
    werr = EPS * (N + 4) * (np.abs(dy) * xh).sum(0)
    return dx, err + 1.01 * _step(dtype, np.abs(dx) + err), dw, werr + 1.01 * _step(dtype, np.abs(dw) + werr)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,C", SHAPES + [(2500, 264), (5000, 40)])
def test_norm_gradients(dtype, N, C):
    from vqlab_amd import fp8
    rng = np.random.default_rng(N * 41 + C)
    x, xv, w, wv, res, rv = _inputs(rng, dtype, N, C)
    for t in (x, w, res):
        t.requires_grad_(True)
    y, h = fp8.rms_norm(x, w, 1e-6, residual=res)
    dy, dyv = mc.acts(rng, dtype, N, C)
    dh, dhv = mc.acts(rng, dtype, N, C)
    hv, r = _check(y.detach(), h.detach(), xv, rv, wv, dtype, 1e-6)
    dx, dw, dr = torch.autograd.grad((y, h), (x, w, res), (dy, dh), retain_graph=True)
    assert torch.equal(dx, dr) and dw.dtype == w.dtype and dx.dtype == x.dtype
    rx, bx, rw, bw = _grad_bar(hv, r, wv, dyv, dhv, dtype)
    mc.assert_within(dx, rx, bx, "dx")
    mc.assert_within(dw, rw, bw, "dw")
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)      # y alone
    rx, bx, _, _ = _grad_bar(hv, r, wv, dyv, None, dtype)
    mc.assert_within(dx, rx, bx, "dx of y")
    mc.assert_within(dw, rw, bw, "dw of y")
    dx, dr = torch.autograd.grad(h, (x, res), dh)                       # h alone: a sum
    assert torch.equal(dx, dh) and torch.equal(dr, dh)
    y = fp8.rms_norm(x, w)                                              # no residual
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    _, r, _ = fc.norm(xv, None, wv, 1e-6, None)
    rx, bx, rw, bw = _grad_bar(xv, r, wv, dyv, None, dtype)
    mc.assert_within(dx, rx, bx, "dx without a residual")
    mc.assert_within(dw, rw, bw, "dw without a residual")


def test_norm_gradient_against_differences():
    """The formula's own derivative by central differences in float64."""
    rng = np.random.default_rng(1)
    h, w, dy = rng.standard_normal((2, 7)), rng.standard_normal(7), rng.standard_normal((2, 7))
    f = lambda h, w: (fc.norm(h, None, w, 1e-3, None)[2] * dy).sum()
    dx, dw = fc.norm_grad(h, fc.norm(h, None, w, 1e-3, None)[1], w, dy, None)
    d = 1e-5
    for i in np.ndindex(h.shape):
        a, b = h.copy(), h.copy()
        a[i] += d
        b[i] -= d
        assert abs((f(a, w) - f(b, w)) / (2 * d) - dx[i]) < 1e-8
    for i in range(7):
        a, b = w.copy(), w.copy()
        a[i] += d
        b[i] -= d
        assert abs((f(h, a) - f(h, b)) / (2 * d) - dw[i]) < 1e-8


@pytest.mark.parametrize("N", [3, 1100])
def test_norm_far_values(N):
    """Rows whose squares are no fp32 numbers, rows of zeros (with and without eps), rows of the smallest
    numbers, infinities and NaN in their rows alone."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(N)
    x, _ = mc.acts(rng, "fp32", N, 520)
    w = torch.ones(520, device="cuda")
    x[0] *= 2.0 ** 100
    x[1] *= 2.0 ** -120
    x[2] = 0
    y = fp8.rms_norm(x, w, 0.0)
    ref = fc.norm(x[:2].double().cpu().numpy(), None, np.ones(520), 0.0, None)[2]
    # the second row's h r passes 2^-120 * 2^120: r and the product are rounded once each
    mc.assert_within(y[:2], ref, 4 * EPS * np.abs(ref), "far rows")
    assert torch.isnan(y[2]).all()                         # 0 / 0
    assert (fp8.rms_norm(x, w, 1e-6)[2] == 0).all()
    x[1, 5], x[2, 519] = float("inf"), float("nan")
    for eps in (0.0, 1e-6):
        y = fp8.rms_norm(x, w, eps)
        rows = fp8.rms_norm_f8(x, w, eps)
        back = fp8.f8_dequantize(*rows, torch.float32)
        assert torch.isnan(y[2]).all() and torch.isnan(back[2]).all() and torch.isnan(y[1, 5])
        assert torch.isfinite(y[0]).all() and torch.isfinite(back[0]).all() and torch.isfinite(y[3:]).all()
        assert torch.isnan(back[1, :128]).all()            # inf * 0 in the first block


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_views_types_and_empty(dtype):
    from vqlab_amd import fp8
    rng = np.random.default_rng(2)
    x, _ = mc.acts(rng, dtype, 4, 6, 301)
    res, _ = mc.acts(rng, dtype, 4, 6, 301)
    w = torch.from_numpy(rng.standard_normal(301).astype(np.float32)).cuda()
    for wd in TYPES:
        wt = w.to(mc.torch_dtype(wd))
        for cut in (lambda t: t[..., 1:], lambda t: t[:, ::2, :296], lambda t: t[1, :, 3:299], lambda t: t[0, 0]):
            xc, rc = cut(x), cut(res)
            C = xc.shape[-1]
            y, h = fp8.rms_norm(xc, wt[1:1 + C] if C < 301 else wt, residual=rc)
            assert y.shape == h.shape == xc.shape and y.dtype == x.dtype
            f = lambda t: t.double().cpu().numpy().reshape(-1, C)
            _check(y.reshape(-1, C), h.reshape(-1, C), f(xc), f(rc), f(wt[1:1 + C] if C < 301 else wt)[0], dtype, 1e-6)
            rows, h8 = fp8.rms_norm_f8(xc, wt[1:1 + C] if C < 301 else wt, residual=rc)
            assert torch.equal(h8, h) and rows.codes.shape == xc.shape
    e = x[:0].clone().requires_grad_(True)
    wt = w.clone().requires_grad_(True)
    y = fp8.rms_norm(e, wt)
    de, dw = torch.autograd.grad(y, (e, wt), torch.ones_like(y))
    assert y.shape == de.shape == (0, 6, 301) and (dw == 0).all()
    assert fp8.rms_norm_f8(x[:0], w).scales.shape == (0, 6, 3)


def test_norm_strided_gradient_and_graph():
    """x with rows apart is read in place, backward too; a captured training pass replays."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(3)
    base, _ = mc.acts(rng, "bf16", 40, 800)
    w = torch.ones(512, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    x = base[:, 16:528].requires_grad_(True)
    dy, _ = mc.acts(rng, "bf16", 40, 512)
    y = fp8.rms_norm(x, w)
    want = torch.autograd.grad(y, (x, w), dy)
    c = x.detach().contiguous().requires_grad_(True)
    for a, b in zip(want, torch.autograd.grad(fp8.rms_norm(c, w), (c, w), dy)):
        assert torch.equal(a, b)
    strided = torch.autograd.grad(fp8.rms_norm(c, w), (c, w), dy.t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(strided, want))
    del y
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(fp8.rms_norm(c, w), (c, w), dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(fp8.rms_norm(c, w), (c, w), dy)
        rows = fp8.rms_norm_f8(c.detach(), w.detach())
    eager = fp8.rms_norm_f8(c.detach(), w.detach())
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(rows.codes.view(torch.uint8), eager.codes.view(torch.uint8)) and torch.equal(rows.scales, eager.scales)
