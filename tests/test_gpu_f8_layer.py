"""Norm, 8-bit linears and routing by groups one after the other, as a layer has them; what their
calls refuse; tensors past 2^31 elements; the same tensor twice; two graphs over the same modules."""
from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

import f8_cases as fc
import group_cases as gc
import mx_cases as mc
import test_gpu_norm as tn

pytestmark = pytest.mark.gpu

FORM = dict(score="sigmoid", groups=4, top_groups=2, scale=2.5)
E, K = 16, 3
EPS = 2.0 ** -24


class Layer(torch.nn.Module):
    """norm -> 8-bit rows -> linear -> SiLU -> linear, then norm -> router and MXFP4 experts."""

    def __init__(self, H, I, dtype):
        super().__init__()
        from vqlab_amd import fp8, mx
        rnd = lambda o, i: torch.randn(o, i, device="cuda") / i ** 0.5
        proj = lambda o, i: mx.MXSwitchLinear.from_weight(torch.randn(E, o, i, device="cuda") / i ** 0.5)
        self.n1 = (1 + 0.1 * torch.randn(H, device="cuda")).to(dtype)
        self.n2 = (1 + 0.1 * torch.randn(H, device="cuda")).to(dtype)
        self.up, self.down = fp8.F8Linear.from_weight(rnd(I, H), "fp8"), fp8.F8Linear.from_weight(rnd(H, I))
        self.gate = fp8.F8Linear.from_weight(rnd(E, H))
        self.bias = 0.1 * torch.randn(E, device="cuda")
        self.block = mx.MXSparseMoeBlock(mx.MXSwitchGLU(proj(I, H), proj(I, H), proj(H, I)), K, bias=self.bias, **FORM)

    def forward(self, x, res, keep=None):
        from vqlab_amd import fp8
        rows, h = fp8.rms_norm_f8(x, self.n1, 1e-6, res)
        up = self.up(rows, out_dtype=x.dtype)
        act = torch.nn.functional.silu(up)
        down = self.down(act)
        y, h2 = fp8.rms_norm(down, self.n2, 1e-6, h)
        logits = self.gate(y, out_dtype=torch.float32)
        out = h2 + self.block(y, logits)
        if keep is not None:
            keep.update(rows=rows, h=h, up=up, act=act, down=down, y=y, h2=h2, logits=logits)
        return out


def f64(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("N", [1, 5, 33, 260])
@pytest.mark.parametrize("H,I", [(256, 640), (200, 328)])
def test_a_layer(dtype, N, H, I):
    """Each step against float64 of what the step before it gave; the whole of it again on another
    stream and in a graph, bit for bit."""
    from vqlab_amd import router
    torch.manual_seed(N + H)
    td = mc.torch_dtype(dtype)
    with torch.no_grad():
        layer = Layer(H, I, td)
        x, res = torch.randn(N, H, device="cuda", dtype=td), torch.randn(N, H, device="cuda", dtype=td)
        s = {}
        out = layer(x, res, s)
        w = lambda lin: (fc.decode(lin.codes.view(torch.uint8).cpu().numpy()), lin.scales.cpu().numpy())
        # the norm in 8 bits: h, and codes of the float64 y (a code is off by one step at most where y is near
        # the middle of two; half a step of e4m3 is 2^-4 of the value, of subnormal codes 2^-10 of a scale)
        hv = f64(s["h"])
        _, _, ref = fc.norm(hv, None, f64(layer.n1), 1e-6, None)
        q, sx = fc.decode(s["rows"].codes.view(torch.uint8).cpu().numpy()), s["rows"].scales.cpu().numpy()
        sxr = np.repeat(sx.astype(np.float64), 128, 1)[:, :H]
        assert (np.abs(q * sxr - ref) <= (2.0 ** -4 + 2.0 ** -20) * np.abs(ref) + 2.0 ** -10 * sxr).all()
        # linears
        c8, sw = w(layer.up)
        y, bar = fc.product_bar(q * sxr, fc.weight_values(c8, sw), dtype)
        mc.assert_within(s["up"], y, bar + 1.01 * fc.instruction_bar(q, sx, c8, sw), "up")
        y, bar = fc.product_bar(f64(s["act"]), fc.weight_values(*w(layer.down)), dtype)
        mc.assert_within(s["down"], y, bar, "down")
        tn._check(s["y"], s["h2"], f64(s["down"]), hv, f64(layer.n2), dtype, 1e-6)
        y, bar = fc.product_bar(f64(s["y"]), fc.weight_values(*w(layer.gate)), "fp32")
        mc.assert_within(s["logits"], y, bar, "logits")
        # the block is its routing and its experts
        ids, wts = router.top_k(s["logits"], K, bias=layer.bias, **FORM)
        o = gc.route(f64(s["logits"]), K, bias=f64(layer.bias), score="sigmoid", groups=4, top_groups=2, scale=2.5)
        assert (ids.cpu().numpy() == o["ids"]).all()
        mc.assert_within(wts, o["w"], 64 * EPS * o["w"], "weights")
        assert torch.equal(out, s["h2"] + layer.block.switch_mlp(s["y"], ids, wts))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = layer(x, res)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, other)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = layer(x, res)
        for k in range(3):
            x.copy_(torch.randn_like(x))
            want = layer(x, res)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, want), k


def test_two_graphs_over_the_same_modules():
    """Each graph has its workspaces: replays in turn, and with eager calls between, change nothing."""
    torch.manual_seed(3)
    with torch.no_grad():
        layer = Layer(256, 640, torch.bfloat16)
        xs = [torch.randn(n, 256, device="cuda", dtype=torch.bfloat16) for n in (3, 70)]
        layer(xs[0], xs[0]), layer(xs[1], xs[1])
        graphs = []
        for x in xs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                graphs.append((g, layer(x, x)))
        for _ in range(3):
            for x in xs:
                x.copy_(torch.randn_like(x))
            want = [layer(x, x) for x in xs]
            for (g, _), _x in zip(graphs, xs):
                g.replay()
            graphs[0][0].replay()
            torch.cuda.synchronize()
            for (_, held), w in zip(graphs, want):
                assert torch.equal(held, w)


def test_a_training_step():
    """The gradient through norm, a frozen 8-bit linear and the router, in fp32, against float64.
    d logits is checked against the formula elsewhere; here it is taken as it came. Errors: dy sums O
    exact products in fp32 (O 2^-24 of their magnitudes), the norm's gradient adds at most 32 roundings
    of its terms and passes dy's error on."""
    from vqlab_amd import fp8, router
    torch.manual_seed(9)
    N, H = 130, 384
    lin = fp8.F8Linear.from_weight(torch.randn(64, H, device="cuda") / H ** 0.5)
    x = torch.randn(N, H, device="cuda", requires_grad=True)
    w = (1 + 0.1 * torch.randn(H, device="cuda")).requires_grad_()
    res = torch.randn(N, H, device="cuda", requires_grad=True)
    y, h = fp8.rms_norm(x, w, 1e-6, res)
    logits = lin(y)
    logits.retain_grad(), y.retain_grad()
    r = router.route(logits, 4, score="sigmoid", groups=8, top_groups=4, bias=0.1 * torch.randn(64, device="cuda"))
    c = torch.randn_like(r.weights)
    ((r.weights * c).sum() + 3 * r.balance + 0.5 * r.z + (0.1 * h).sum()).backward()
    W = fc.weight_values(fc.decode(lin.codes.view(torch.uint8).cpu().numpy()), lin.scales.cpu().numpy())
    dl = f64(logits.grad)
    dy, emag = dl @ W, np.abs(dl) @ np.abs(W)
    err = (64 + 20) * EPS * emag
    mc.assert_within(y.grad, dy, err + EPS * np.abs(dy), "dy")
    hv = f64(h)
    _, rr, _ = fc.norm(hv, None, f64(w), 1e-6, None)
    xh = hv * rr
    dx, dw = fc.norm_grad(hv, rr, f64(w), dy, np.full_like(hv, np.float32(0.1)))
    ge = err * np.abs(f64(w)) + 32 * EPS * np.abs(dy * f64(w))
    # the mean: fp32 sums of 16 products in a lane, then 64 bits
    bar = 1.01 * rr * (ge + np.abs(xh) * (ge * np.abs(xh)).mean(1, keepdims=True)) + 32 * EPS * (
        np.abs(dx) + 0.1 + rr * np.abs(xh) * np.abs(dy * f64(w) * xh).mean(1, keepdims=True))
    mc.assert_within(x.grad, dx, bar, "dx")
    assert torch.equal(x.grad, res.grad)
    mc.assert_within(w.grad, dw, 1.01 * ((err + 32 * EPS * np.abs(dy)) * np.abs(xh)).sum(0) + (N + 8) * EPS * np.abs(dy * xh).sum(0),
                     "dw")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("N", [5, 1040])
@pytest.mark.parametrize("C", [1300, 2304, 3300, 5120, 9000, 13320])
def test_norm_of_every_number_of_waves(dtype, N, C):
    tn.test_norm(dtype, N, C)
    tn.test_norm_gradients(dtype, N, C)


def test_the_same_tensor_twice():
    from vqlab_amd import fp8
    x = torch.randn(6, 320, device="cuda", requires_grad=True)
    w = torch.randn(320, device="cuda", requires_grad=True)
    y, h = fp8.rms_norm(x, w, 1e-6, x)
    dy = torch.randn_like(y)
    gx, gw = torch.autograd.grad((y * dy).sum() + h.sum(), (x, w))
    x2 = x.detach().double().requires_grad_()
    w2 = w.detach().double().requires_grad_()
    h2 = x2 + x2
    y2 = h2 * (h2.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * w2
    rx, rw = torch.autograd.grad((y2 * dy.double()).sum() + h2.sum(), (x2, w2))
    # a few dozen roundings of terms of the size of dy w and 1
    assert ((gx - rx).abs() <= 64 * EPS * (1 + 4 * rx.abs().max())).all()
    assert ((gw - rw).abs() <= 64 * EPS * (1 + 4 * rw.abs().max())).all()
    s = torch.randn(320, device="cuda").abs()
    a, b = fp8.rms_norm(s.expand(4, 320), s)[0], fp8.rms_norm(s[None], s)[0]      # x and weight are one, rows too
    assert torch.equal(a, b)


# ------------------------------------------------------------------ far offsets
def test_rows_past_2_to_the_31_elements():
    """The last rows of a tensor of 2^31 elements and more come out as they do alone."""
    from vqlab_amd import fp8
    C, N = 8192, (1 << 18) + 3
    x = torch.zeros(N, C, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, C, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(C, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        q, small = fp8.f8_quantize(x), fp8.f8_quantize(x[-3:])
        assert torch.equal(q.codes[-3:].view(torch.uint8), small.codes.view(torch.uint8))
        assert torch.equal(q.scales[-3:], small.scales)
        assert torch.equal(fp8.f8_dequantize(*q)[-3:], fp8.f8_dequantize(*small))
        del q
        rows, h = fp8.rms_norm_f8(x, w, residual=x)
        few, hf = fp8.rms_norm_f8(x[-3:], w, residual=x[-3:])
        assert torch.equal(h[-3:], hf) and torch.equal(rows.codes[-3:].view(torch.uint8), few.codes.view(torch.uint8))
        del rows, h
    x.requires_grad_(), w.requires_grad_()
    y = fp8.rms_norm(x, w)
    assert torch.equal(y[-3:], fp8.rms_norm(x[-3:], w))
    dy = torch.zeros_like(y)
    dy[-3:] = torch.randn(3, C, device="cuda", dtype=torch.bfloat16)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    t = x.detach()[-3:].clone().requires_grad_()
    tx, tw = torch.autograd.grad(fp8.rms_norm(t, w), (t, w), dy[-3:])
    assert torch.equal(gx[-3:], tx) and (gx[:-3] == 0).all() and torch.equal(gw, tw)


def test_more_rows_than_a_launch_has_threads_for():
    """2^25 rows and more: their waves are more than 2^31 threads."""
    from vqlab_amd import fp8
    N, C = (1 << 25) + 9, 16
    x = torch.ones(N, C, device="cuda", dtype=torch.bfloat16)
    x[-4:] = torch.randn(4, C, device="cuda", dtype=torch.bfloat16)
    x[1 << 25] = 3.0
    w = torch.randn(C, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        y = fp8.rms_norm(x, w)
        assert torch.equal(y[-12:], fp8.rms_norm(x[-12:], w)) and torch.equal(y[:-9], y[:1].expand(N - 9, C))
        rows, few = fp8.rms_norm_f8(x, w), fp8.rms_norm_f8(x[-12:], w)
        assert torch.equal(rows.codes[-12:].view(torch.uint8), few.codes.view(torch.uint8))
        assert torch.equal(rows.scales[-12:], few.scales)


def test_8_bit_rows_far_apart():
    """Rows 16 MB and more apart are laid out first."""
    from vqlab_amd import fp8
    lin = fp8.F8Linear.from_weight(torch.randn(64, 256, device="cuda"), "fp8")
    q = fp8.f8_quantize(torch.randn(40, 256, device="cuda", dtype=torch.bfloat16))
    room = torch.zeros(40, (1 << 24) + 256, device="cuda", dtype=torch.uint8)
    room[:, :256] = q.codes.view(torch.uint8)
    far = room[:, :256].view(fp8.F8)
    assert far.stride(0) > 1 << 24
    for n in (3, 40):
        assert torch.equal(lin((far[:n], q.scales[:n])), lin((q.codes[:n], q.scales[:n])))


@pytest.mark.parametrize("act", [None, "fp8"])
def test_linears_past_2_to_the_31_elements(act):
    """x of more than 2^31 elements, then an output of as many: last rows as they are alone."""
    from vqlab_amd import fp8
    for OUT, IN, N in ((48, 16384, (1 << 17) + 5), (16384, 128, (1 << 17) + 5)):
        lin = fp8.F8Linear.from_weight(torch.randn(OUT, IN, device="cuda") / IN ** 0.5, act)
        x = torch.zeros(N, IN, device="cuda", dtype=torch.bfloat16)
        x[-70:] = torch.randn(70, IN, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            y = lin(x)
        assert (y[:-70] == 0).all()
        ref = x[-70:].double() @ fp8.f8_dequantize(lin.codes, lin.scales, torch.float32).double().t()
        # 2^-8 for bf16's rounding; 8-bit x is 2^-4 off each, at random
        assert ((y[-70:].double() - ref).abs() <= 2.0 ** -7 * ref.abs() + (2.0 ** -8 if act is None else 0.5)).all()
        if act is None:
            dx = lin._dx(y, torch.bfloat16) if OUT > IN else None
            if dx is not None:
                assert (dx[:-70] == 0).all() and torch.isfinite(dx[-70:]).all() and (dx[-70:] != 0).any()
        del x, y


def test_routing_past_2_to_the_31_logits():
    from vqlab_amd import router
    T, n = (1 << 23) + 5, 256
    lg = torch.zeros(T, n, device="cuda", dtype=torch.bfloat16)
    lg[-5:] = torch.randn(5, n, device="cuda", dtype=torch.bfloat16)
    form = dict(score="sigmoid", groups=8, top_groups=4, scale=2.5, bias=0.1 * torch.randn(n, device="cuda"))
    ids, w = router.top_k(lg, 8, **form)
    a, b = router.top_k(lg[-5:], 8, **form)
    assert torch.equal(ids[-5:], a) and ((w[-5:] - b).abs() <= 2.0 ** -18).all()
    lg.requires_grad_()
    r = router.route(lg, 8, **form)
    d, = torch.autograd.grad(r.weights[-5:].sum(), lg)
    assert (d[:1000] == 0).all() and (d[-5:] != 0).any()
    # z: the logits' squared log-sums, log(256)^2 but for five tokens; an fp32 sum of 2^23 in many parts
    assert abs(float(r.z.detach()) / np.log(256.0) ** 2 - 1) < 1e-3 and int(r.counts.sum()) == 8 * T


# ------------------------------------------------------------------ refusals
def test_refusals():
    from vqlab_amd import fp8
    x = torch.randn(4, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    q = fp8.f8_quantize(x)
    codes, scales = fp8.f8_quantize_weight(torch.randn(64, 256, device="cuda"))
    lin, lin8 = fp8.F8Linear(codes, scales), fp8.F8Linear(codes, scales, "fp8")
    bad = [
        (lambda: fp8.f8_quantize(x.int()), ValueError), (lambda: fp8.f8_quantize(x.double()), ValueError),
        (lambda: fp8.f8_quantize(x[0, 0]), ValueError), (lambda: fp8.f8_quantize_weight(x[0]), ValueError),
        (lambda: fp8.f8_dequantize(x, q.scales), ValueError), (lambda: fp8.f8_dequantize(*q, torch.float64), ValueError),
        (lambda: fp8.f8_dequantize(q.codes, q.scales.half()), ValueError),
        (lambda: fp8.f8_dequantize(q.codes, q.scales[:, :1]), ValueError),
        (lambda: fp8.f8_dequantize(q.codes, q.scales.cpu()), ValueError),
        (lambda: fp8.F8Linear(codes.float(), scales), ValueError), (lambda: fp8.F8Linear(codes, scales[:, :1]), ValueError),
        (lambda: fp8.F8Linear(codes, scales.half()), ValueError), (lambda: fp8.F8Linear(codes, scales.cpu()), ValueError),
        (lambda: lin(q), ValueError), (lambda: lin(x[:, :255]), ValueError), (lambda: lin(x.int()), ValueError),
        (lambda: lin(x.cpu()), ValueError), (lambda: lin(x, out_dtype=torch.float64), ValueError),
        (lambda: lin8((q.codes, q.scales[:3])), ValueError), (lambda: lin8((q.codes[:, :128], q.scales[:, :1])), ValueError),
        (lambda: lin8((x, q.scales)), ValueError), (lambda: lin8((q.codes, q.scales.double())), ValueError),
        (lambda: lin8((q.codes.cpu(), q.scales.cpu())), ValueError),
        (lambda: lin8(x.clone().requires_grad_()), RuntimeError),
        (lambda: lin8((q.codes, q.scales.clone().requires_grad_())), RuntimeError),
        (lambda: fp8.f8_quantize(x.clone().requires_grad_()), RuntimeError),
        (lambda: fp8.rms_norm(x, w[:255]), ValueError), (lambda: fp8.rms_norm(x, w.int()), ValueError),
        (lambda: fp8.rms_norm(x, w, -1.0), ValueError), (lambda: fp8.rms_norm(x, w, float("nan")), ValueError),
        (lambda: fp8.rms_norm(x, w, residual=x[:3]), ValueError), (lambda: fp8.rms_norm(x, w, residual=x.half()), ValueError),
        (lambda: fp8.rms_norm(x, w.cpu()), ValueError), (lambda: fp8.rms_norm(x[:, :0], w[:0]), ValueError),
        (lambda: fp8.rms_norm_f8(x, w.clone().requires_grad_()), RuntimeError),
        (lambda: fp8.rms_norm(torch.ones(1, 16385, device="cuda"), torch.ones(16385, device="cuda")), NotImplementedError),
    ]
    for i, (call, error) in enumerate(bad):
        with pytest.raises(error):
            call()
            print("not refused:", i, flush=True)


def test_refused_derivatives():
    from vqlab_amd import fp8, router
    x = torch.randn(4, 256, device="cuda", requires_grad=True)
    w = torch.ones(256, device="cuda", requires_grad=True)
    lin = fp8.F8Linear.from_weight(torch.randn(64, 256, device="cuda"))
    for f in (lambda: fp8.rms_norm(x, w).pow(2).sum(), lambda: lin(x).pow(2).sum(),
              lambda: router.route(x, 4, score="sigmoid").z):
        with pytest.raises(RuntimeError):                   # a derivative of the derivative
            g, = torch.autograd.grad(f(), x, create_graph=True)
            g.sum().backward()
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        fp8.rms_norm(fw.make_dual(x.detach(), torch.ones_like(x)), w)
    with fw.dual_level(), pytest.raises(RuntimeError):
        fp8.rms_norm_f8(fw.make_dual(x.detach(), torch.ones_like(x)), w.detach())


def test_router_forms_are_refused():
    from vqlab_amd import mx, router
    lg = torch.randn(5, 64, device="cuda")
    for call in (router.top_k, router.route):
        for kw, words in ((dict(score="relu"), "score"), (dict(groups=5), "groups"), (dict(groups=8, top_groups=9), "of 8"),
                          (dict(bias=torch.zeros(64)), "device"), (dict(bias=torch.zeros(8, device="cuda")), "bias"),
                          (dict(scale=-1), "scale"), (dict(groups=32, top_groups=1), "top 4 of 2")):
            with pytest.raises(ValueError, match=words):
                call(lg, 4, **kw)
    wide = torch.randn(3, 1024, device="cuda")
    with pytest.raises(NotImplementedError):
        router.top_k(wide, 4, groups=128, top_groups=64)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,OUT,IN", [(1, 100, 5121), (2, 64, 8000), (3, 2000, 7400), (16, 33, 17408), (17, 130, 4104),
                                      (20, 5120, 6016), (32, 48, 20001), (9, 16, 120000)])
def test_few_rows_of_many_blocks(dtype, N, OUT, IN):
    """Rows of more blocks than eight waves hold: ranges of k, added up in their order."""
    import test_gpu_f8 as tf
    tf.test_linear(dtype, N, OUT, IN)
    tf.test_linear_8_bit_activations(dtype, N, OUT, IN)
    tf.test_linear_gradient(dtype, N, min(IN, 9000), OUT)


def _within(got, ref, mag, n, dtype, more=0.0):
    """fc.product_bar's bar, on the GPU: n exact products summed in fp32, scales, slices, one rounding."""
    acc = (n + 20) * EPS * mag + more
    step = mc.HALF_STEP[dtype] * (ref.abs() + acc)
    bar = acc + (step.clamp(min=2.0 ** -25) if dtype == "fp16" else step)
    bad = ((got.double() - ref).abs() > bar).sum()
    assert int(bad) == 0, f"{int(bad)} of {ref.numel()}"


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,OUT,IN", [(49, 4096, 10240), (64, 4100, 10300), (100, 10240, 4096), (129, 4096, 10240),
                                      (200, 10300, 4100), (333, 5120, 8192), (700, 4096, 4096),
                                      (14001, 300, 260), (17000, 257, 384), (20011, 100, 513)])
def test_tiles(dtype, N, OUT, IN):
    """Products large enough for tiles, whatever x: few of them cut along k, and many small ones. In 64 bits
    on the GPU."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(N + OUT + IN)
    codes, s, w = fc.weight(rng, OUT, IN)
    codes, s = torch.from_numpy(codes).cuda(), torch.from_numpy(s).cuda()
    lin, lin8 = fp8.F8Linear(codes, s), fp8.F8Linear(codes, s, "fp8")
    w = torch.from_numpy(w).cuda()
    torch.manual_seed(N)
    x = torch.randn(N, IN, device="cuda").to(mc.torch_dtype(dtype)).requires_grad_()
    y = lin(x)
    xd, aw = x.detach().double(), w.abs()
    _within(y.detach(), xd @ w.t(), xd.abs() @ aw.t(), IN, dtype)
    dy = torch.randn_like(y)
    dx, = torch.autograd.grad(y, x, dy)
    dd = dy.double()
    _within(dx, dd @ w, dd.abs() @ aw, OUT, dtype)
    # 8-bit x: exact into fp32; into 16 bits each group of eight products may lose 7 * 2^-13 of its largest
    q = fp8.f8_quantize(x.detach())
    xd = q.codes.float().double() * q.scales.double().repeat_interleave(128, 1)[:, :IN]
    ref, mag = xd @ w.t(), xd.abs() @ aw.t()
    _within(lin8(q, out_dtype=torch.float32), ref, mag, IN, "fp32")
    if dtype != "fp32":
        pad = lambda t: torch.nn.functional.pad(t.abs().float(), (0, -IN % 8)).unflatten(1, (-1, 8))
        a, b = pad(xd), pad(w)
        top = torch.stack([(a[n][None] * b).amax(-1).sum(-1) for n in range(N)]).double()
        _within(lin8(x.detach()), ref, mag, IN, dtype, 1.01 * 7 * 2.0 ** -13 * top)


@pytest.mark.parametrize("act", [None, "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,OUT,IN", [(100, 4160, 10304), (9000, 300, 1100)])
def test_tiles_keep_to_their_rows(dtype, N, OUT, IN, act):
    """NaN, infinities and far values of x, codes and scales that are NaN: what they do not meet is as ever."""
    from vqlab_amd import fp8
    rng = np.random.default_rng(N + IN)
    codes, s, w = fc.weight(rng, OUT, IN)
    codes[11, 77], codes[270, IN - 1] = 0x7f, 0xff
    s[1, 2] = np.nan                                       # weight rows 128 .. 255
    w = fc.weight_values(fc.decode(codes), s)
    lin = fp8.F8Linear(torch.from_numpy(codes).cuda(), torch.from_numpy(s).cuda(), act)
    w = torch.from_numpy(w).cuda()
    torch.manual_seed(N)
    x = torch.randn(N, IN, device="cuda")
    far = 2.0 ** 12 if dtype == "fp16" else 2.0 ** 100
    x[5] *= far
    x[6] /= far
    x = x.to(mc.torch_dtype(dtype))
    x[17, 3], x[18, IN - 1], x[19, 200] = float("nan"), float("inf"), -float("inf")
    with torch.no_grad():
        out = torch.float32 if act else x.dtype
        y = lin(x, out_dtype=out)
        if act:
            q = fp8.f8_quantize(x)
            xd = q.codes.float().double() * q.scales.double().repeat_interleave(128, 1)[:, :IN]
        else:
            xd = x.double()
    xd = xd.nan_to_num(nan=float("nan"), posinf=float("nan"), neginf=float("nan"))
    ref, mag = xd @ w.t(), xd.abs() @ w.abs().t()
    assert ref.isnan().any(0)[[11, 128, 255, 270]].all() and ref.isnan().any(1)[[17, 18, 19]].all()
    fine = ref.isfinite()
    assert not y[~fine].isfinite().any()
    # x / far in fp16 has numbers below the smallest normal one, which are exact all the same
    _within(torch.where(fine, y.double(), 0), torch.where(fine, ref, 0), torch.where(fine, mag, 0), IN, "fp32" if act else dtype)
