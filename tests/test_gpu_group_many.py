"""Routing by groups of so many tokens that sixteen lanes take one: the cases of few tokens again, every
width of a row, and the ends of what those lanes take."""
from __future__ import annotations

import itertools

import numpy as np
import pytest
import torch

import group_cases as gc
import mx_cases as mc
import test_gpu_group as tg

pytestmark = pytest.mark.gpu

CASES = [(4096, 8, 2, 2, 1, 2), (4097, 60, 6, 5, 2, 2), (4099, 96, 10, 6, 3, 1), (4500, 130, 7, 10, 4, 2),
         (4100, 256, 8, 8, 4, 2), (4222, 300, 10, 12, 5, 2), (4101, 512, 15, 16, 7, 2), (4102, 512, 16, 16, 7, 2),
         (4103, 64, 4, 32, 9, 2), (4104, 320, 6, 5, 1, 1), (4105, 190, 1, 1, 1, 1), (4095, 256, 8, 8, 4, 2)]


@pytest.mark.parametrize("dtype", tg.TYPES)
@pytest.mark.parametrize("form", tg.FORMS, ids=["sigmoid", "scaled", "softmax"])
@pytest.mark.parametrize("T,E,k,G,kept,top", CASES)
def test_route(dtype, form, T, E, k, G, kept, top):
    tg.test_route(dtype, form, T, E, k, G, kept, top)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_ties_nan_and_little_left(score):
    tg.test_ties_go_to_the_lower_group_and_id(4100, score)
    tg.test_near_ties_are_decided_in_64_bits(4352, score)
    tg.test_nan_stays_in_its_row(4110, score)
    for E, G, k in ((8, 4, 2), (96, 6, 6), (512, 16, 10)):
        tg.test_rows_groups_and_experts_with_little_left(E, G, k, 4120, score)


def _choices(l, bias, score, k, G, kept, top):
    """Every choice of ids that 64 bits allow for one row of logits. Softmax scores that are equal as numbers
    (an exponential is a unit of 2^-53 off, the sum of E of them E units in an order that is nobody's
    business), plus biases that add up to the same in two groups, come out up to (E + 8) 2^-53 apart: which of
    two such groups, or experts, is the larger is rounding alone, so each order of them is right."""
    E = len(l)
    ex = np.exp(l - l.max())
    s = 1 / (1 + np.exp(-l)) if score == "sigmoid" else ex / ex.sum()
    c = s + bias
    tol = (E + 8) * 2.0 ** -53 * 2 * np.abs(c).max()
    g = np.sort(c.reshape(G, -1), 1)[:, ::-1][:, :top].sum(1)
    last = np.sort(g)[::-1][kept - 1]
    sure, tied = np.flatnonzero(g > last + tol), np.flatnonzero(np.abs(g - last) <= tol)
    for more in itertools.combinations(tied, kept - len(sure)):
        can = np.isin(np.arange(E) // (E // G), [*sure, *more])
        yield np.argsort(-np.where(can, c, -np.inf), kind="stable")[:k]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,G,kept,top", [(64, 8, 3, 2), (256, 8, 4, 2), (500, 10, 4, 1)])
def test_coarse_logits_and_biases(E, G, kept, top, score):
    """Few distinct scores: equal sums in many groups, more equal candidates than a token ranks. The rows in
    which 64 bits decide go by the oracle, the few in which they do not by one of the orders they allow."""
    from vqlab_amd import router
    T, k = 4100, 8
    rng = np.random.default_rng(E + T)
    lg = torch.from_numpy(np.round(rng.standard_normal((T, E)) * 2).astype(np.float32) / 2)
    lg[::3] = torch.from_numpy(rng.standard_normal((len(lg[::3]), E)).astype(np.float32))
    f = dict(score=score, groups=G, top_groups=kept, group_top=top, scale=2.0)
    tg._check(lg.cuda(), k, router.route(lg.cuda(), k, **f), **f)
    bias = np.round(rng.standard_normal(E) * 2) / 8
    r = router.route(lg.cuda(), k, bias=torch.from_numpy(bias).float().cuda(), **f)
    ids, o = r.ids.cpu().numpy(), gc.route(lg.double().numpy(), k, bias=bias, **f)
    other = np.flatnonzero((ids != o["ids"]).any(1))
    assert len(other) <= T // 50
    for t in other:
        assert any(np.array_equal(ids[t], c) for c in _choices(lg[t].double().numpy(), bias, score, k, G, kept, top)), t
    same = np.setdiff1d(np.arange(T), other)
    mc.assert_within(r.weights[same], o["w"][same], 64 * tg.EPS * E * o["w"][same], "weights")
    assert np.array_equal(r.counts.cpu().numpy(), np.bincount(ids.ravel(), minlength=E))


@pytest.mark.parametrize("norm", [True, False])
def test_far_logits(norm):
    tg.test_far_logits(4128, norm)


def test_strides_alignment_streams_and_graphs():
    tg.test_strides_alignment_streams_and_graphs(4100)


def test_far_and_near_rows_side_by_side():
    """Rows whose largest logit is far from 0 beside others, four tokens to a wave: the log-sum and p of
    each are its own."""
    from vqlab_amd import router
    torch.manual_seed(2)
    T, E = 4100, 128
    lg = torch.randn(T, E, device="cuda")
    lg[::3] += 50 * torch.randn(len(lg[::3]), 1, device="cuda")
    lg[5::7] -= 39.0 + 2 * torch.rand(len(lg[5::7]), 1, device="cuda")      # largest about -40, both sides
    lg.requires_grad_()
    form = dict(score="sigmoid", groups=8, top_groups=4, scale=2.5, bias=0.1 * torch.randn(E, device="cuda"))
    r = router.route(lg, 6, **form)
    dw = torch.randn_like(r.weights)
    gb, gz = torch.tensor(0.7, device="cuda"), torch.tensor(0.2, device="cuda")
    d, = torch.autograd.grad((r.weights, r.balance, r.z), lg, (dw, gb, gz))
    tg._check(lg, 6, r, grads=((dw, gb, gz), d, "fp32"), group_top=2, **form)


@pytest.mark.parametrize("T", [7, 4100])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_groups_of_one_expert(T, score):
    """Scored by two experts where there is one: by that one."""
    from vqlab_amd import router
    rng = np.random.default_rng(T)
    for bias in (None, torch.from_numpy((0.1 * rng.standard_normal(16)).astype(np.float32)).cuda()):
        lg = torch.from_numpy(rng.standard_normal((T, 16)).astype(np.float32)).cuda()
        f = dict(score=score, groups=16, top_groups=9, group_top=2, bias=bias, scale=2.5)
        r = router.route(lg, 6, **f)
        tg._check(lg, 6, r, **f)
        one = router.route(lg, 6, **dict(f, group_top=1))
        assert torch.equal(r.ids, one.ids) and torch.equal(r.weights, one.weights)
