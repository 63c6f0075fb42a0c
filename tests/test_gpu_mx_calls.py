"""How MXFP4 modules and the router are called and kept: types, derivatives, devices, state."""
from __future__ import annotations

import io

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

import mx_cases as mc

pytestmark = pytest.mark.gpu


def _dev(*arrays):
    return tuple(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays)


def _linear(rng, OUT, IN, act=None):
    from vqlab_amd import mx
    codes, scales = mc.weight(rng, OUT, IN)
    return mx.MXLinear(*_dev(codes, scales), IN, act), mc.values(codes, scales, IN)


def _switch(rng, E, OUT, IN):
    from vqlab_amd import mx
    codes, scales = mc.weight(rng, E, OUT, IN)
    return mx.MXSwitchLinear(*_dev(codes, scales), IN), mc.values(codes, scales, IN)


def _glu(rng, E, H, I):
    from vqlab_amd import mx
    (g, gw), (u, uw), (d, dw) = _switch(rng, E, I, H), _switch(rng, E, I, H), _switch(rng, E, H, I)
    return mx.MXSwitchGLU(g, u, d), (gw, uw, dw)


# --------------------------------------------------------------------- ids
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("E", [8, 200, 300])
@pytest.mark.parametrize("T", [3, 250])
def test_ids_of_every_integer_type(dtype, E, T):
    rng = np.random.default_rng(E + T)
    sw, w = _switch(rng, E, 17, 40)
    glu, _ = _glu(rng, E, 32, 32)
    x, xv = mc.acts(rng, "fp32", T, 1, 1, 40)
    top = min(E, 128 if dtype == torch.int8 else 256)      # what every listed type can say
    idx = rng.integers(0, top, (T, 2))
    ids = torch.from_numpy(idx).to(dtype).cuda()
    y = sw(x, ids)
    for t in range(0, T, 9):
        for j in range(2):
            ref, bar = mc.product_bar(xv[t, 0], w[idx[t, j]], "fp32")
            mc.assert_within(y[t, j], ref, bar, f"pair {t}, {j}")
    z, wt = torch.randn(T, 32, device="cuda"), torch.rand(T, 2, device="cuda")
    assert torch.equal(glu(z, ids, wt), glu(z, ids.to(torch.int32), wt))


def test_ids_that_no_integer_type_holds_are_outside():
    rng = np.random.default_rng(1)
    sw, _ = _switch(rng, 4, 16, 32)
    ids = torch.tensor([[2 ** 32 + 1, -2 ** 40, 2 ** 62]], device="cuda")
    assert (sw(torch.ones(1, 1, 1, 32, device="cuda"), ids) == 0).all()


def test_ids_that_are_no_integers_are_refused():
    rng = np.random.default_rng(2)
    glu, _ = _glu(rng, 4, 32, 32)
    x, wt = torch.randn(3, 32, device="cuda"), torch.rand(3, 2, device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.bool):
        ids = torch.ones(3, 2, device="cuda").to(dtype)
        with pytest.raises(ValueError, match="ids"):
            glu(x, ids, wt)
        with pytest.raises(ValueError, match="ids"):
            glu.gate_proj(x[:, None, None], ids)


# ------------------------------------------------- forward-mode derivatives
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N", [1, 20, 130])
def test_linear_forward_mode(dtype, N):
    rng = np.random.default_rng(N)
    lin, w = _linear(rng, 40, 96)
    x, xv = mc.acts(rng, dtype, N, 96)
    t, tv = mc.acts(rng, dtype, N, 96)
    for leaf in (x, x.clone().requires_grad_(True)):
        with fw.dual_level():
            y = fw.unpack_dual(lin(fw.make_dual(leaf, t)))
            assert y.tangent is not None
            mc.assert_within(y.primal, *mc.product_bar(xv, w, dtype), "primal")
            mc.assert_within(y.tangent, *mc.product_bar(tv, w, dtype), "tangent")


def test_what_has_no_gradient_has_no_tangent_either():
    from vqlab_amd import mx, router
    rng = np.random.default_rng(4)
    glu, _ = _glu(rng, 4, 64, 32)
    a4, _ = _linear(rng, 32, 64, act="mxfp4")
    ids, w = _dev(np.zeros((4, 2), np.int32), np.ones((4, 2), np.float32))
    x, lg = torch.randn(4, 64, device="cuda"), torch.randn(4, 4, device="cuda")
    blk = mx.MXSparseMoeBlock(glu, 2)
    with fw.dual_level():
        xd, wd, ld = (fw.make_dual(t, torch.ones_like(t)) for t in (x, w, lg))
        for call in (lambda: mx.mx_quantize(xd), lambda: a4(xd), lambda: glu(xd, ids, w),
                     lambda: glu(x, ids, wd), lambda: glu.gate_proj(xd[:, None, None], ids),
                     lambda: blk(xd, lg), lambda: blk(x, ld)):
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                call()
        with pytest.raises((RuntimeError, NotImplementedError)):
            router.route(ld, 2)
        assert glu(x, ids, w).shape == (4, 64)             # no tangent: as ever
        assert fw.unpack_dual(a4(x)).tangent is None


def test_forward_over_reverse_is_refused():
    """A gradient's own derivative would be dropped by the kernels that compute it."""
    from vqlab_amd import router
    lin, _ = _linear(np.random.default_rng(5), 40, 96)
    with fw.dual_level():
        x = fw.make_dual(torch.randn(3, 96, device="cuda").requires_grad_(True), torch.ones(3, 96, device="cuda"))
        with pytest.raises(RuntimeError, match="gradient of MXLinear"):
            torch.autograd.grad(lin(x).square().sum(), x)
        lg = torch.randn(3, 8, device="cuda", requires_grad=True)
        c = fw.make_dual(torch.ones((), device="cuda"), torch.ones((), device="cuda"))
        with pytest.raises(RuntimeError, match="gradient of the router"):
            torch.autograd.grad(router.route(lg, 2).z * c, lg)


# ------------------------------------------------------------------- router
def test_top_k_refuses_logits_that_want_a_gradient():
    from vqlab_amd import router
    lg = torch.randn(4, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        router.top_k(lg, 2)
    with torch.no_grad():
        ids, w = router.top_k(lg, 2)
    assert torch.equal(ids, router.top_k(lg.detach(), 2)[0]) and not w.requires_grad
    with fw.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
        router.top_k(fw.make_dual(lg.detach(), torch.ones_like(lg)), 2)


def test_losses_can_be_changed_in_place():
    """The other outputs and the gradient stay; a changed token count, which the gradient reads, is
    an error."""
    from vqlab_amd import router
    lg = torch.randn(30, 16, device="cuda", requires_grad=True)
    want = router.route(lg, 4)
    dref = torch.autograd.grad(0.01 * want.balance + 2 * want.z, lg)[0]
    r = router.route(lg, 4)
    r.balance.mul_(0.01)
    r.z.mul_(2)
    assert torch.equal(r.z.detach(), 2 * want.z.detach()) and float(r.tokens) == 30
    assert torch.equal(r.balance.detach(), 0.01 * want.balance.detach())
    assert torch.equal(torch.autograd.grad(r.balance + r.z, lg)[0], dref)
    r = router.route(lg, 4)
    r.tokens.fill_(1e9)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(r.z, lg)


# ------------------------------------------------------------------ modules
def test_a_block_without_logits_says_so():
    from vqlab_amd import mx
    glu, _ = _glu(np.random.default_rng(5), 4, 64, 32)
    with pytest.raises(ValueError, match="router_weight"):
        mx.MXSparseMoeBlock(glu, 2)(torch.randn(3, 64, device="cuda"))


@pytest.mark.parametrize("E,OUT,IN", [(1, 16, 128), (1, 17, 129), (3, 70, 700), (2, 5, 1), (4, 33, 544)])
def test_codes_and_scales_come_back(E, OUT, IN):
    from vqlab_amd import mx
    rng = np.random.default_rng(OUT)
    codes, scales = _dev(*mc.weight(rng, E, OUT, IN))
    sw = mx.MXSwitchLinear(codes, scales, IN)
    assert torch.equal(sw.codes, codes) and torch.equal(sw.scales, scales)
    lin = mx.MXLinear(codes[0], scales[0], IN)
    assert torch.equal(lin.codes, codes[0]) and torch.equal(lin.scales, scales[0])


@pytest.mark.parametrize("assign", [False, True])
def test_state_dict_holds_the_weights(assign):
    from vqlab_amd import mx
    rng = np.random.default_rng(6)
    (glu, ws), (other, _) = _glu(rng, 6, 96, 64), _glu(rng, 6, 96, 64)
    net = torch.nn.ModuleList([glu, _linear(rng, 40, 96)[0]])
    net2 = torch.nn.ModuleList([other, _linear(rng, 40, 96)[0]])
    # weights beyond fp16 in the source only: what is looked up about them follows
    codes, scales = mc.weight(rng, 40, 96)
    scales[::3] = 90
    net[1] = mx.MXLinear(*_dev(codes, scales), 96)
    assert net2[1]._w.f16_exact and not net[1]._w.f16_exact
    buf = io.BytesIO()
    torch.save(net.state_dict(), buf)
    buf.seek(0)
    state = torch.load(buf, weights_only=True, map_location="cpu")
    assert set(state) == {f"0.{p}_proj.{n}" for p in ("gate", "up", "down") for n in ("codes", "scales")} | \
        {"1.codes", "1.scales"}
    assert state["1.codes"].shape == (40, 48) and np.array_equal(state["1.scales"].numpy(), scales)
    net2.load_state_dict(state, assign=assign)
    assert not net2[1]._w.f16_exact
    x, h = torch.randn(7, 96, device="cuda"), torch.randn(7, 96, device="cuda").half()
    ids, w = torch.randint(0, 6, (7, 2), device="cuda"), torch.rand(7, 2, device="cuda")
    assert torch.equal(net2[0](x, ids, w), net[0](x, ids, w)) and torch.equal(net2[1](h), net[1](h))
    lost = dict(state)
    del lost["1.scales"]
    with pytest.raises(RuntimeError, match="1.scales"):
        net2.load_state_dict(lost)
    with pytest.raises(RuntimeError, match="shape"):
        net2.load_state_dict({**state, "1.codes": state["1.codes"][:20], "1.scales": state["1.scales"][:20]})
    with pytest.raises(RuntimeError, match="uint8"):
        net2.load_state_dict({**state, "1.scales": state["1.scales"].int()})
    assert torch.equal(net2[1](h), net[1](h))              # a refused load leaves the module as it was


def test_a_captured_graph_follows_a_load():
    rng = np.random.default_rng(10)
    (lin, _), (other, _) = _linear(rng, 40, 96), _linear(rng, 40, 96)
    x = torch.randn(7, 96, device="cuda", dtype=torch.bfloat16)
    lin(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lin(x)
    for src in (other, _linear(rng, 40, 96)[0], other):
        lin.load_state_dict(src.state_dict())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, src(x))


def test_modules_move_with_their_weights():
    from vqlab_amd import mx
    rng = np.random.default_rng(7)
    glu, _ = _glu(rng, 6, 64, 32)
    blk = mx.MXSparseMoeBlock(glu, 2)
    x, lg = torch.randn(5, 64, device="cuda"), torch.randn(5, 6, device="cuda")
    ref = blk(x, lg)
    blk.to("cpu")
    assert all(not t.is_cuda for t in glu.up_proj._packed[:2]) and not glu.up_proj.codes.is_cuda
    ids = torch.zeros(5, 1, dtype=torch.int32, device="cuda")
    for call in (lambda: blk(x, lg), lambda: glu.gate_proj(x[:, None, None], ids)):
        with pytest.raises(ValueError, match="device"):
            call()
    state = {k: v.clone() for k, v in blk.state_dict().items()}
    blk.cuda()
    assert torch.equal(blk(x, lg), ref)
    assert torch.equal(blk.half()(x, lg), ref)             # codes and scales are no floats
    assert all(torch.equal(v.cpu(), state[k]) for k, v in blk.state_dict().items())
    blk.cpu().load_state_dict(state)                       # packed on the GPU, kept where the module is
    assert torch.equal(blk.cuda()(x, lg), ref)


def test_projections_on_another_device_are_refused():
    from vqlab_amd import mx
    glu, _ = _glu(np.random.default_rng(8), 4, 64, 32)
    x, lg = torch.randn(5, 64, device="cuda"), torch.randn(5, 4, device="cuda")
    ids, w = torch.zeros(5, 2, dtype=torch.int32, device="cuda"), torch.rand(5, 2, device="cuda")
    for name in ("up_proj", "down_proj"):
        getattr(glu, name).cpu()
        with pytest.raises(ValueError, match="device"):
            glu(x, ids, w)
        with pytest.raises(ValueError, match="device"):
            mx.MXSparseMoeBlock(glu, 2)(x, lg)
        getattr(glu, name).cuda()
    assert glu(x, ids, w).shape == (5, 64)


# ------------------------------------------------------------------ streams
@pytest.mark.parametrize("T", [2, 150])
def test_blocks_on_two_streams_at_once(T):
    """Pair by pair and sorted: each call has its own workspace."""
    from vqlab_amd import mx
    rng = np.random.default_rng(9)
    glu, _ = _glu(rng, 8, 128, 64)
    blk = mx.MXSparseMoeBlock(glu, 3)
    xs = [mc.acts(rng, "fp16", T, 128)[0] for _ in range(2)]
    lgs = [torch.randn(T, 8, device="cuda") for _ in range(2)]
    ref = [blk(x, lg) for x, lg in zip(xs, lgs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(6):
        for s, x, lg in zip(streams, xs, lgs):
            with torch.cuda.stream(s):
                got.append(blk(x, lg))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ref[i % 2]) for i, y in enumerate(got))
