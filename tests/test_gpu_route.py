"""The router on the GPU against its float64 formulas: every type, ties, masks, rows of -inf and
NaN, gradients against the formula and against differences."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import mx_cases as mc

pytestmark = pytest.mark.gpu

TYPES = ["fp32", "bf16", "fp16"]
EPS = 2.0 ** -24


def _logits(rng, dtype, T, E, scale=1.0):
    return torch.from_numpy((scale * rng.standard_normal((T, E))).astype(np.float32)).to(mc.torch_dtype(dtype)).cuda()


def _check(lg, k, norm, mask, r, grads=None):
    """Bars: l - max is exact or off by one rounding of a difference of size <= 2 max |l|; exp is
    good to a few units and carries that rounding; a sum of E terms adds E roundings."""
    from vqlab_amd import router
    lv = lg.detach().double().cpu().numpy()
    E = lv.shape[1]
    o = mc.route(lv, k, norm, None if mask is None else mask.cpu().numpy())
    assert np.array_equal(r.ids.cpu().numpy(), o["ids"])
    assert np.array_equal(r.counts.cpu().numpy(), o["counts"])
    assert float(r.tokens) == o["n"]
    span = 2 * np.abs(np.where(np.isfinite(lv), lv, 0)).max() if lv.size else 0.0
    rel = (span + 8 + E + k) * EPS
    mc.assert_within(r.weights, o["w"], rel * np.abs(o["w"]) + 1e-37, "weights")
    # a workgroup's register sums add at most T / 4 roundings, the fp64 rest none
    T = max(lv.shape[0], 1)
    assert abs(float(r.balance.detach()) - o["balance"]) <= (rel + T * EPS) * o["balance"] + 1e-37
    assert abs(float(r.z.detach()) - o["z"]) <= 2 * (rel + T * EPS) * (o["z"] + np.sqrt(o["z"])) + 1e-37
    if grads is not None:
        (dw, gb, gz), d, dtype = grads
        ref = mc.route_grad(o, k, norm, dw.double().cpu().numpy(), float(gb), float(gz))
        dwv = np.abs(dw.double().cpu().numpy())
        n = max(o["n"], 1)
        fmax = abs(float(gb)) * E * o["counts"].max() / (n * n * k)
        # every term of the sum is at most this large, each with the relative error of its factors
        size = o["p"] * (2 * fmax + 2 * abs(float(gz)) / n * (np.abs(o["lse"][:, None]) + 1)
                         + (np.abs(o["w"]) * dwv).sum(1, keepdims=True) * (0 if norm else 1))
        for t in range(lv.shape[0]):
            for j, e in enumerate(o["ids"][t]):
                if e >= 0:
                    size[t, e] += o["w"][t, j] * (dwv[t, j] + (o["w"][t] * dwv[t]).sum())
        bar = 3 * rel * size + mc.HALF_STEP[dtype] * np.abs(ref)
        if dtype == "fp16":
            bar = bar + 2.0 ** -25                       # half a step of fp16's subnormals
        mc.assert_within(d, ref, bar + 1e-37, "gradient")
    return o


CASES = [(1, 1, 1), (1, 8, 2), (5, 8, 8), (33, 60, 6), (64, 64, 4), (100, 65, 10), (257, 256, 8), (40, 300, 10),
         (130, 512, 10), (19, 1000, 3), (9, 2048, 64),
         (2048, 8, 2), (2049, 60, 6), (3001, 96, 10), (2500, 130, 7), (2100, 256, 8), (2222, 300, 10), (2050, 512, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("T,E,k", CASES)
def test_route(dtype, norm, T, E, k):
    from vqlab_amd import router
    rng = np.random.default_rng(T * 31 + E + k)
    lg = _logits(rng, dtype, T, E).requires_grad_(True)
    mask = None if T % 2 else torch.from_numpy(rng.random(T) < 0.7).cuda()
    r = router.route(lg, k, norm, mask)
    dw = torch.randn(T, k, device="cuda")
    gb, gz = torch.tensor(0.7 * T, device="cuda"), torch.tensor(0.3 * T, device="cuda")
    d = torch.autograd.grad((r.weights, r.balance, r.z), lg, (dw, gb, gz))[0]
    assert d.dtype == lg.dtype
    _check(lg, k, norm, mask, r, ((dw, gb, gz), d, dtype))
    ids, w = router.top_k(lg.detach(), k, norm, mask)
    assert torch.equal(ids, r.ids) and torch.equal(w, r.weights)


@pytest.mark.parametrize("T", [3, 3000])
def test_ties_go_to_the_lower_id(T):
    from vqlab_amd import router
    lg = torch.zeros(T, 200, device="cuda")
    lg[1, 70:] = 1.0
    lg[2, ::2] = -0.0
    ids, w = router.top_k(lg, 5)
    assert ids[:3].tolist() == [[0, 1, 2, 3, 4], [70, 71, 72, 73, 74], [0, 1, 2, 3, 4]]
    assert (ids[3:] == torch.arange(5, device="cuda")).all()
    assert torch.allclose(w, torch.full_like(w, 0.2))


@pytest.mark.parametrize("E,k", [(64, 6), (256, 8), (500, 16)])
def test_many_tokens_with_few_distinct_logits(E, k):
    """Coarse logits: rows with more equal candidates than the ranking holds, beside ordinary ones."""
    from vqlab_amd import router
    rng = np.random.default_rng(E)
    lg = torch.from_numpy(np.round(rng.standard_normal((2400, E)) * 2).astype(np.float32) / 2)
    lg[::3] = torch.from_numpy(rng.standard_normal((800, E)).astype(np.float32))
    lg = lg.cuda()
    r = router.route(lg, k)
    _check(lg, k, True, None, r)


@pytest.mark.parametrize("E,k", [(8, 4), (96, 6), (512, 10)])
@pytest.mark.parametrize("more", [0, 2100])
def test_rows_with_few_or_no_experts_left(E, k, more):
    from vqlab_amd import router
    rng = np.random.default_rng(E)
    T = 12 + more
    lg = _logits(rng, "fp32", T, E)
    lg[3] = float("-inf")
    lg[5, 2:] = float("-inf")                              # two experts for k places
    lg[7, 1:] = float("-inf")
    lg[8] = torch.finfo(torch.float32).min                 # the type's lowest value is a number
    lg[9] = 1e30
    mask = torch.ones(T, dtype=torch.bool, device="cuda")
    mask[10] = False
    lg[10] = float("nan")
    lg.requires_grad_(True)
    r = router.route(lg, k, True, mask)
    dw = torch.randn(T, k, device="cuda")
    zero = torch.tensor(0.0, device="cuda")
    gb = torch.tensor(1.0, device="cuda")
    d = torch.autograd.grad((r.weights, r.balance, r.z), lg, (dw, gb, zero))[0]
    assert (r.ids[3] == -1).all() and (r.weights[3] == 0).all() and (d[3] == 0).all()
    assert (r.ids[10] == -1).all() and (r.weights[10] == 0).all() and (d[10] == 0).all()
    assert r.ids[5].tolist()[2:] == [-1] * (k - 2) and abs(float(r.weights[5].sum().detach()) - 1) < 1e-6
    assert r.ids[7].tolist() == [0] + [-1] * (k - 1) and float(r.weights[7, 0].detach()) == 1.0
    assert r.ids[8].tolist() == list(range(k)) and torch.isfinite(r.weights).all()
    assert float(r.tokens) == T - 2 and int(r.counts.sum()) == (T - 2) * k - (k - 2) - (k - 1)
    assert torch.isfinite(d).all()


@pytest.mark.parametrize("T", [4, 2400])
def test_nan_logits_are_loud(T):
    from vqlab_amd import router
    lg = torch.randn(T, 40, device="cuda")
    lg[1, 7] = float("nan")
    lg[2, 3] = float("inf")
    r = router.route(lg, 3)
    assert torch.isnan(r.weights[1]).all() and 7 not in r.ids[1].tolist()
    assert torch.isnan(r.weights[2]).all() and r.ids[2, 0] == 3
    assert torch.isnan(r.balance) and torch.isnan(r.z)
    assert torch.isfinite(r.weights[[0, 3]]).all()


def test_no_tokens_and_no_live_tokens():
    from vqlab_amd import router
    r = router.route(torch.empty(0, 16, device="cuda"), 4)
    assert r.ids.shape == (0, 4) and r.counts.tolist() == [0] * 16
    assert float(r.balance) == 0 and float(r.z) == 0 and float(r.tokens) == 0
    lg = torch.randn(5, 16, device="cuda", requires_grad=True)
    r = router.route(lg, 4, mask=torch.zeros(5, dtype=torch.uint8, device="cuda"))
    assert float(r.balance.detach()) == 0 and r.counts.tolist() == [0] * 16
    d = torch.autograd.grad((r.weights.sum() + r.balance + r.z), lg)[0]
    assert (d == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_logits(dtype):
    from vqlab_amd import router
    rng = np.random.default_rng(9)
    big = _logits(rng, dtype, 40, 130)
    for view in (big[:, 1:97], big[::2, :64], big[:, ::2], big.t()[:30, :40], big[:1].expand(6, 130)):
        leaf = view.detach().requires_grad_(True)
        r = router.route(leaf, 4)
        dw = torch.randn(view.shape[0], 4, device="cuda")
        zero = torch.tensor(0.0, device="cuda")
        d = torch.autograd.grad(r.weights, leaf, dw)[0]
        _check(leaf, 4, True, None, r, ((dw, zero, zero), d, dtype))


def test_gradient_against_differences():
    """Central differences of the float64 formulas at the chosen experts (which a small step does
    not change), for each output alone."""
    from vqlab_amd import router
    rng = np.random.default_rng(2)
    T, E, k = 5, 12, 3
    lg = _logits(rng, "fp32", T, E, 2.0).requires_grad_(True)
    dw = torch.randn(T, k, device="cuda")
    one, zero = torch.tensor(1.0, device="cuda"), torch.tensor(0.0, device="cuda")
    for norm in (True, False):
        r = router.route(lg, k, norm)
        for outs, grads, f in (((r.weights,), (dw,), lambda o: (o["w"] * dw.double().cpu().numpy()).sum()),
                               ((r.balance,), (one,), None), ((r.z,), (one,), lambda o: o["z"])):
            d = torch.autograd.grad(outs, lg, grads, retain_graph=True)[0].double().cpu().numpy()
            base = lg.detach().double().cpu().numpy()
            counts = mc.route(base, k, norm)["counts"]
            if f is None:                                  # counts are held, as choices are
                f = lambda o: E * (counts / (T * k) * o["p"].sum(0) / T).sum()
            h = 1e-5
            for t, e in ((0, 0), (2, 5), (4, 11), (1, int(r.ids[1, 0])), (3, int(r.ids[3, 2]))):
                hi, lo = base.copy(), base.copy()
                hi[t, e] += h
                lo[t, e] -= h
                diff = (f(mc.route(hi, k, norm)) - f(mc.route(lo, k, norm))) / (2 * h)
                # h^2 of the third derivative (of values of order 10), float64 over h, fp32 kernels
                assert abs(diff - d[t, e]) <= 10 * h * h + 1e-9 + 100 * EPS * max(1, abs(diff)), (norm, t, e)


def test_only_some_outputs_are_used():
    from vqlab_amd import router
    lg = torch.randn(20, 32, device="cuda", requires_grad=True)
    r = router.route(lg, 4)
    a = torch.autograd.grad(r.z, lg, retain_graph=True)[0]
    b = torch.autograd.grad(r.balance, lg, retain_graph=True)[0]
    c = torch.autograd.grad(r.z + r.balance, lg)[0]
    assert torch.allclose(a + b, c, atol=1e-6)
    assert not r.ids.requires_grad and not r.counts.requires_grad


def test_same_results_every_time():
    from vqlab_amd import router
    lg = torch.randn(5000, 160, device="cuda", requires_grad=True)
    outs = []
    for _ in range(3):
        r = router.route(lg, 6)
        d = torch.autograd.grad(r.weights.square().sum() + r.balance + r.z, lg)[0]
        outs.append([*r, d])
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


def test_forward_and_backward_captured():
    """A training step's routing recorded once and replayed on new logits."""
    from vqlab_amd import router
    lg = torch.randn(300, 64, device="cuda", requires_grad=True)
    dw = torch.randn(300, 4, device="cuda")
    one = torch.tensor(1.0, device="cuda")

    def run():
        r = router.route(lg, 4)
        d = torch.autograd.grad((r.weights, r.balance, r.z), lg, (dw, one, one))[0]
        return [r.ids, r.weights.detach(), r.counts, r.balance.detach(), r.z.detach(), d]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for i in range(3):
        with torch.no_grad():
            lg.normal_()
        g.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(kept, run())), f"replay {i}"
        torch.cuda.synchronize()


def test_routes_the_vq_layer_the_same():
    """The call's routing is that of the VQ decode layer."""
    from vq_cases import make_module, to_device
    from vqlab_amd import moe, router
    rng = np.random.default_rng(0)
    projs = {}
    for name, (o, i) in (("gate", (128, 256)), ("up", (128, 256)), ("down", (256, 128))):
        projs[name] = make_module(rng, 16, o, i, 4, 256)
    blk = moe.VQSparseMoeBlock.from_modules({n: to_device(m) + (m["pack_bits"],) for n, m in projs.items()},
                                            top_k=4, in_features={"gate": 256, "up": 256, "down": 128})
    lg = torch.randn(7, 16, device="cuda")
    lg[2] = 0.5                                            # ties
    _, ids, w = blk.fused(torch.randn(7, 256, device="cuda", dtype=torch.bfloat16), lg, return_route=True)
    mine, mw = router.top_k(lg, 4)
    assert torch.equal(ids, mine)
    assert torch.allclose(w, mw, rtol=1e-5, atol=0)
