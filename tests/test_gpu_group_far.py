"""Routing by groups where every score of a token is at the lower end of fp32's range: which group and which
expert is the largest is still a question of 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import test_gpu_group as tg

pytestmark = pytest.mark.gpu


def _far(rng, T, E):
    """Rows whose largest logits lie between -80 and -104: their sigmoids run from 1e-35 through the smallest
    normal fp32 number 2^-126 (e^-87.3) to below the smallest of all."""
    top = rng.uniform(-104, -80, (T, 1))
    return torch.from_numpy((top - 4 * rng.random((T, E))).astype(np.float32))


@pytest.mark.parametrize("T", [96, 4100])
@pytest.mark.parametrize("bias", [None, 0.0, 1e-37])
@pytest.mark.parametrize("E,G,kept,top", [(32, 8, 2, 2), (64, 8, 3, 1), (256, 8, 4, 2), (96, 6, 1, 2)])
def test_groups_of_vanishing_scores(E, G, kept, top, bias, T):
    from vqlab_amd import router
    rng = np.random.default_rng(T + E)
    lg = _far(rng, T, E)
    if E == 32:
        # two groups of which the one with the larger sum has the smaller largest score, and the others far below
        lg[7] = -120.0
        lg[7, :2] = torch.tensor([-86.9, -90.0])
        lg[7, 4:6] = torch.tensor([-86.95, -87.5])
    b = None if bias is None else torch.from_numpy((bias * rng.standard_normal(E)).astype(np.float32)).cuda()
    f = dict(score="sigmoid", groups=G, top_groups=kept, group_top=top, bias=b)
    lg = lg.cuda()
    r = router.route(lg, 4, **f)
    tg._check(lg, 4, r, **f)
    ids, w = router.top_k(lg, 4, **f)
    assert torch.equal(ids, r.ids) and torch.equal(w, r.weights)


@pytest.mark.parametrize("bias", [0.0, 1e-37])
def test_experts_of_vanishing_scores(bias):
    """The same of experts chosen by score and bias out of all; and alone or in a large batch it is the same
    choice."""
    from vqlab_amd import router
    rng = np.random.default_rng(3)
    T, E = 4100, 64
    lg = _far(rng, T, E).cuda()
    b = torch.from_numpy((bias * rng.standard_normal(E)).astype(np.float32)).cuda()
    r = router.route(lg, 6, score="sigmoid", bias=b)
    tg._check(lg, 6, r, score="sigmoid", bias=b, group_top=2)
    few, _ = router.top_k(lg[:500], 6, score="sigmoid", bias=b)
    assert torch.equal(few, r.ids[:500])
