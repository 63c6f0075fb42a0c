"""Routing by sigmoid or softmax scores with a bias and groups on the GPU against float64: every type,
ties, near ties, masks, groups and rows with little left, far logits, gradients."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import group_cases as gc
import mx_cases as mc

pytestmark = pytest.mark.gpu

TYPES = ["fp32", "bf16", "fp16"]
EPS = 2.0 ** -24


def _logits(rng, dtype, T, E, scale=1.0):
    return torch.from_numpy((scale * rng.standard_normal((T, E))).astype(np.float32)).to(mc.torch_dtype(dtype)).cuda()


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _check(lg, k, r, mask=None, grads=None, **form):
    """Bars as of the plain router: l - max and exp carry one rounding of a difference of 2 max |l| and a
    few units, sums of E terms E roundings; a sigmoid a few units more."""
    norm = form.pop("norm_topk_prob", True)
    f = dict(form, bias=_np(form.get("bias")))
    o = gc.route(_np(lg), k, norm=norm, mask=None if mask is None else mask.cpu().numpy(), **f)
    E, T = lg.shape[1], max(lg.shape[0], 1)
    assert np.array_equal(r.ids.cpu().numpy(), o["ids"])
    assert np.array_equal(r.counts.cpu().numpy(), o["counts"]) and float(r.tokens) == o["n"]
    l = o["l"]
    span = 2 * np.abs(np.where(np.isfinite(l), l, 0)).max() if l.size else 0.0
    rel = (span + 16 + E + k) * EPS
    mc.assert_within(r.weights, o["w"], rel * np.abs(o["w"]) + 1e-37, "weights")
    assert abs(float(r.balance.detach()) - o["balance"]) <= (2 * rel + T * EPS) * o["balance"] + 1e-37
    assert abs(float(r.z.detach()) - o["z"]) <= 2 * (rel + T * EPS) * (o["z"] + np.sqrt(o["z"])) + 1e-37
    if grads is not None:
        (dw, gb, gz), d, dtype = grads
        ref, size = gc.grad(o, k, form.get("score", "softmax"), norm, form.get("scale", 1.0), _np(dw), float(gb), float(gz))
        bar = 4 * rel * size + mc.HALF_STEP[dtype] * np.abs(ref) + (2.0 ** -25 if dtype == "fp16" else 0.0)
        mc.assert_within(d, ref, bar + 1e-37, "gradient")
    return o


FORMS = [dict(score="sigmoid"), dict(score="sigmoid", scale=2.5), dict(score="softmax", scale=16.0)]
CASES = [(1, 8, 2, 1, 1, 2), (5, 8, 8, 4, 4, 1), (33, 60, 6, 5, 2, 2), (64, 64, 4, 8, 3, 1), (100, 65, 10, 13, 7, 2),
         (257, 256, 8, 8, 4, 2), (40, 300, 10, 10, 3, 2), (130, 512, 10, 16, 5, 1), (19, 1000, 3, 50, 9, 2),
         (9, 2048, 64, 64, 5, 2), (50, 16, 1, 16, 1, 1),
         (2048, 8, 2, 2, 1, 2), (2049, 60, 6, 5, 2, 2), (3001, 96, 10, 6, 3, 1), (2500, 130, 7, 10, 4, 2),
         (2100, 256, 8, 8, 4, 2), (2222, 300, 10, 12, 5, 2), (2050, 512, 15, 16, 7, 2), (2051, 512, 16, 16, 7, 2),
         (2060, 64, 4, 32, 9, 2), (2070, 320, 6, 5, 1, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS, ids=["sigmoid", "scaled", "softmax"])
@pytest.mark.parametrize("T,E,k,G,kept,top", CASES)
def test_route(dtype, form, T, E, k, G, kept, top):
    from vqlab_amd import router
    rng = np.random.default_rng(T * 31 + E + k)
    for bias in (False, True):
        f = dict(form, groups=G, top_groups=kept, group_top=top, norm_topk_prob=bool((T + bias) % 2))
        if bias:
            f["bias"] = torch.from_numpy((0.1 * rng.standard_normal(E)).astype(np.float32)).cuda()
        lg = _logits(rng, dtype, T, E).requires_grad_(True)
        mask = None if T % 2 else torch.from_numpy(rng.random(T) < 0.7).cuda()
        r = router.route(lg, k, mask=mask, **f)
        dw = torch.randn(T, k, device="cuda")
        gb, gz = torch.tensor(0.7 * T, device="cuda"), torch.tensor(0.3 * T, device="cuda")
        d = torch.autograd.grad((r.weights, r.balance, r.z), lg, (dw, gb, gz))[0]
        assert d.dtype == lg.dtype
        _check(lg, k, r, mask, ((dw, gb, gz), d, dtype), **f)
        ids, w = router.top_k(lg.detach(), k, mask=mask, **f)
        assert torch.equal(ids, r.ids) and torch.equal(w, r.weights)


@pytest.mark.parametrize("T", [60, 3000])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_ties_go_to_the_lower_group_and_id(T, score):
    from vqlab_amd import router
    lg = torch.zeros(T, 64, device="cuda")
    lg[1, 40:] = 1.0
    lg[2, ::2] = -0.0
    for bias in (None, torch.zeros(64, device="cuda")):
        ids, w = router.top_k(lg, 5, score=score, bias=bias, groups=8, top_groups=2)
        want = torch.tensor([0, 1, 2, 3, 4], device="cuda", dtype=torch.int32)
        assert (ids[0] == want).all() and (ids[2:] == want).all() and ids[1].tolist() == [40, 41, 42, 43, 44]
        assert torch.allclose(w, torch.full_like(w, 0.2))
    bias = torch.zeros(64, device="cuda")
    bias[7], bias[63], bias[30] = 1.0, 1.0, 2.0
    ids, _ = router.top_k(lg[3:], 4, score=score, bias=bias, groups=1)
    assert (ids == torch.tensor([30, 7, 63, 0], device="cuda")).all()


@pytest.mark.parametrize("T", [100, 2200])
@pytest.mark.parametrize("E,G,kept,top", [(64, 8, 3, 2), (256, 8, 4, 2), (500, 10, 4, 1)])
def test_coarse_logits_and_biases(T, E, G, kept, top):
    """Few distinct scores: equal sums in many groups, more equal candidates than a token ranks."""
    from vqlab_amd import router
    rng = np.random.default_rng(E + T)
    lg = torch.from_numpy(np.round(rng.standard_normal((T, E)) * 2).astype(np.float32) / 2)
    lg[::3] = torch.from_numpy(rng.standard_normal((len(lg[::3]), E)).astype(np.float32))
    for bias in (None, torch.from_numpy(np.round(rng.standard_normal(E) * 2).astype(np.float32) / 8).cuda()):
        for score in ("sigmoid", "softmax"):
            f = dict(score=score, bias=bias, groups=G, top_groups=kept, group_top=top, scale=2.0)
            _check(lg.cuda(), 8, router.route(lg.cuda(), 8, **f), **f)


@pytest.mark.parametrize("T", [64, 2304])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_near_ties_are_decided_in_64_bits(T, score):
    """Biases that undo the scores' differences to within parts of an fp32 unit: which of two is larger
    shows in 64 bits alone."""
    from vqlab_amd import router
    rng = np.random.default_rng(T)
    E = 48
    lg = rng.standard_normal((T, E)).astype(np.float32)
    lg[1:] = lg[:1]                                        # the same scores in every row ..
    l64 = lg.astype(np.float64)
    s = 1 / (1 + np.exp(-l64[0])) if score == "sigmoid" else np.exp(l64[0]) / np.exp(l64[0]).sum()
    bias = (1.5 - s).astype(np.float32)                    # .. whose c are 1.5 to within half an fp32 unit
    lg[::2] = rng.standard_normal((len(lg[::2]), E)).astype(np.float32)
    lg, bias = torch.from_numpy(lg).cuda(), torch.from_numpy(bias).cuda()
    for f in (dict(groups=1), dict(groups=6, top_groups=2, group_top=2), dict(groups=12, top_groups=4, group_top=1)):
        f = dict(f, score=score, bias=bias)
        f.setdefault("top_groups", 1)
        _check(lg, 6, router.route(lg, 6, **f), **f)


@pytest.mark.parametrize("E,G,k", [(8, 4, 2), (96, 6, 6), (512, 16, 10)])
@pytest.mark.parametrize("more", [0, 2100])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_rows_groups_and_experts_with_little_left(E, G, k, more, score):
    from vqlab_amd import router
    rng = np.random.default_rng(E)
    T = 14 + more
    lg = _logits(rng, "fp32", T, E)
    gs = E // G
    lg[3] = float("-inf")
    lg[5, 2:] = float("-inf")                              # two experts for k places
    lg[6, 1:gs] = float("-inf")                            # a group with one expert
    lg[7, 1:] = float("-inf")
    lg[8, gs:] = float("-inf")                             # one group
    mask = torch.ones(T, dtype=torch.bool, device="cuda")
    mask[10] = False
    lg[10] = float("nan")
    lg.requires_grad_(True)
    bias = 0.1 * torch.randn(E, device="cuda")
    bias[E - 1] = float("-inf")                            # an expert switched off
    for b in (None, bias):
        f = dict(score=score, bias=b, groups=G, top_groups=2, group_top=2)
        r = router.route(lg, k, mask=mask, **f)
        dw = torch.randn(T, k, device="cuda")
        gb, gz = torch.tensor(3.0, device="cuda"), torch.tensor(2.0, device="cuda")
        d = torch.autograd.grad((r.weights, r.balance, r.z), lg, (dw, gb, gz))[0]
        off = lg.detach().clone()
        off[10] = 0
        _check(off, k, r, mask, ((dw, gb, gz), d, "fp32"), **f)
        assert (d[3] == 0).all() and (d[10] == 0).all() and (r.ids[3] == -1).all() and (r.ids[10] == -1).all()


@pytest.mark.parametrize("T", [20, 2080])
@pytest.mark.parametrize("norm", [True, False])
def test_far_logits(T, norm):
    """Sigmoids that vanish in 32 bits (their ratios do not), that are 1 in 32 bits (their order without a
    bias is the logits'), rows around the border between the two forms."""
    from vqlab_amd import router
    rng = np.random.default_rng(T)
    lg = _logits(rng, "fp32", T, 32)
    lg[0] -= 150
    lg[1] -= 300
    lg[2] += 30
    lg[3] *= 40
    lg[4] -= 40
    lg[5] -= 38
    lg[6, :16] -= 90
    lg.requires_grad_(True)
    f = dict(score="sigmoid", groups=4, top_groups=2, group_top=1, norm_topk_prob=norm, scale=1.5)
    r = router.route(lg, 4, **f)
    dw = torch.randn(T, 4, device="cuda")
    gb, gz = torch.tensor(1.0 * T, device="cuda"), torch.tensor(0.0, device="cuda")
    d = torch.autograd.grad((r.weights, r.balance, r.z), lg, (dw, gb, gz))[0]
    _check(lg, 4, r, None, ((dw, gb, gz), d, "fp32"), **f)
    if norm:
        assert torch.allclose(r.weights.sum(1), torch.full((T,), 1.5, device="cuda"))


@pytest.mark.parametrize("T", [30, 2090])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_nan_stays_in_its_row(T, score):
    from vqlab_amd import router
    rng = np.random.default_rng(T)
    lg = _logits(rng, "fp32", T, 64)
    lg[4, 5], lg[9] = float("nan"), float("nan")
    f = dict(score=score, bias=0.1 * torch.randn(64, device="cuda"), groups=8, top_groups=3)
    ids, w = router.top_k(lg, 4, **f)
    assert torch.isnan(w[[4, 9]]).all() and (ids[9] == -1).all() and (ids[4] >= 0).all() and not (ids[4] == 5).any()
    ok = [t for t in range(T) if t not in (4, 9)]
    assert torch.isfinite(w[ok]).all()
    lg[4, 5] = float("-inf")                               # chosen as if it were not there
    again, w2 = router.top_k(lg, 4, **f)
    assert torch.equal(again, ids) and torch.equal(w2[ok], w[ok])


def test_gradient_against_differences():
    """The oracle's formula against central differences of its own weights and losses, choice fixed."""
    rng = np.random.default_rng(0)
    T, E, k = 3, 12, 3
    l = rng.standard_normal((T, E))
    bias = 0.1 * rng.standard_normal(E)
    dw, gb, gz = rng.standard_normal((T, k)), 0.7, 0.3
    for score in ("sigmoid", "softmax"):
        for norm in (True, False):
            f = dict(score=score, bias=bias, groups=4, top_groups=2, group_top=2, norm=norm, scale=2.5)
            base = gc.route(l, k, **f)
            d, _ = gc.grad(base, k, score, norm, 2.5, dw, gb, gz)

            def value(x):
                r = gc.route(x, k, **f)
                assert np.array_equal(r["ids"], base["ids"])
                return (r["w"] * dw).sum() + gb * r["balance"] + gz * r["z"]
            h = 1e-6
            for i in np.ndindex(T, E):
                a, b = l.copy(), l.copy()
                a[i] += h
                b[i] -= h
                assert abs((value(a) - value(b)) / (2 * h) - d[i]) < 1e-7


@pytest.mark.parametrize("T", [70, 2100])
def test_strides_alignment_streams_and_graphs(T):
    from vqlab_amd import router
    rng = np.random.default_rng(T)
    base = _logits(rng, "bf16", T, 300)
    f = dict(score="sigmoid", bias=0.1 * torch.randn(256, device="cuda"), groups=8, top_groups=4, scale=2.5)
    want = router.top_k(base[:, 3:259].contiguous(), 8, **f)
    for view in (base[:, 3:259], base[:, 3:259].t().contiguous().t()):
        got = router.top_k(view, 8, **f)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = base[:, 3:259].detach().requires_grad_(True)
    c = base[:, 3:259].contiguous().requires_grad_(True)
    dw = torch.randn(T, 8, device="cuda")
    d = [torch.autograd.grad(router.route(t, 8, **f).weights, t, dw)[0] for t in (x, c)]
    assert torch.equal(*d)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(router.route(c.detach(), 8, **f))
        torch.cuda.synchronize()
        assert all(torch.equal(g.ids, want[0]) and torch.equal(g.weights, want[1]) for g in got)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(router.route(c, 8, **f).weights, c, dw)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = router.route(c, 8, **f)
        got = torch.autograd.grad(r.weights, c, dw)[0]
    eager = router.route(c.detach(), 8, **f)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, d[0]) and torch.equal(r.ids, eager.ids) and torch.equal(r.counts, eager.counts)
        assert torch.equal(r.balance, eager.balance) and torch.equal(r.z, eager.z)
        router.route(-c.detach(), 8, **f)


def test_empty_and_defaults():
    from vqlab_amd import router
    lg = torch.randn(40, 64, device="cuda")
    a, b = router.route(lg, 4), router.route(lg, 4, groups=8, score="softmax")     # every group kept: the plain router
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    e = router.route(lg[:0], 4, score="sigmoid", groups=8, top_groups=2)
    assert e.ids.shape == (0, 4) and (e.counts == 0).all() and float(e.tokens) == 0 and float(e.balance) == 0
    bias = torch.randn(64, device="cuda").half()
    x = router.top_k(lg, 4, bias=bias)
    y = router.top_k(lg, 4, bias=bias.float())
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


@pytest.mark.parametrize("T", [1, 37, 300])
def test_the_mxfp4_block_by_this_routing(T):
    """MXSparseMoeBlock with a form is its routing and its experts; the bias is a buffer."""
    from vqlab_amd import mx, router
    rng = np.random.default_rng(T)
    E, H, I = 16, 64, 96
    proj = lambda o, i: mx.MXSwitchLinear.from_weight(torch.randn(E, o, i, device="cuda") / i ** 0.5)
    glu = mx.MXSwitchGLU(proj(I, H), proj(I, H), proj(H, I))
    bias = 0.1 * torch.randn(E, device="cuda")
    form = dict(score="sigmoid", groups=4, top_groups=2, scale=2.5)
    block = mx.MXSparseMoeBlock(glu, top_k=3, bias=bias, **form)
    x, _ = mc.acts(rng, "bf16", T, H)
    lg = torch.randn(T, E, device="cuda")
    mask = torch.rand(T, device="cuda") < 0.8
    y = block(x, lg, mask=mask)
    ids, w = router.top_k(lg, 3, mask=mask, bias=bias, **form)
    assert torch.equal(y, glu(x, ids, w))
    assert "bias" in block.state_dict()
    with pytest.raises(ValueError):
        mx.MXSparseMoeBlock(glu, top_k=9, groups=4, top_groups=2)
    plain = mx.MXSparseMoeBlock(glu, top_k=3)
    assert "bias" not in plain.state_dict() and torch.equal(plain(x, lg), mx.MXSparseMoeBlock(glu, 3, groups=4)(x, lg))
