"""Gradients of tensors past 2^31 elements, by value: the far rows against float64, every other row zero."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import group_cases as gc
import mx_cases as mc

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def _quiet(t, rows):
    """Every row but the last ones is zero."""
    step = 1 << 14
    return not any(bool(t[i:min(i + step, len(t) - rows)].any()) for i in range(0, len(t) - rows, step))


@pytest.mark.parametrize("OUT,IN", [(48, 16384), (16384, 128), (16384, 136)])
def test_gradient_of_a_linear(OUT, IN):
    """dx (or dy) of more than 2^31 elements. A gradient sums OUT exact products in fp32, in slices, with
    scales, and is rounded once into bfloat16 (half a step, 2^-8 at most of the value)."""
    from vqlab_amd import fp8
    torch.manual_seed(OUT + IN)
    N, far = (1 << 17) + 5, 70
    lin = fp8.F8Linear.from_weight(torch.randn(OUT, IN, device="cuda") / IN ** 0.5)
    W = fp8.f8_dequantize(lin.codes, lin.scales, torch.float32).double()
    x = torch.zeros(N, IN, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = lin(x)
    dy = torch.zeros_like(y)
    dy[-far:] = torch.randn(far, OUT, device="cuda", dtype=torch.bfloat16)
    dx, = torch.autograd.grad(y, x, dy)
    d = dy[-far:].double()
    ref, mag = d @ W, d.abs() @ W.abs()
    acc = (OUT + 20) * EPS * mag
    off = (dx[-far:].double() - ref).abs()
    assert bool((off <= acc + 2.0 ** -8 * (ref.abs() + acc)).all()), float((off - acc - 2.0 ** -8 * ref.abs()).max())
    assert _quiet(dx, far)


@pytest.mark.parametrize("norm", [True, False])
def test_gradient_of_a_router(norm):
    from vqlab_amd import router
    torch.manual_seed(4)
    T, n, k, far = (1 << 23) + 5, 256, 8, 5
    lg = torch.zeros(T, n, device="cuda", dtype=torch.bfloat16)
    lg[-far:] = torch.randn(far, n, device="cuda", dtype=torch.bfloat16)
    form = dict(score="sigmoid", groups=8, top_groups=4, scale=2.5)
    bias = 0.1 * torch.randn(n, device="cuda")
    lg.requires_grad_()
    r = router.route(lg, k, norm_topk_prob=norm, bias=bias, **form)
    dw = torch.zeros_like(r.weights)
    dw[-far:] = torch.randn(far, k, device="cuda")
    d, = torch.autograd.grad(r.weights, lg, dw)
    l = lg[-far:].detach().double().cpu().numpy()
    o = gc.route(l, k, bias=bias.double().cpu().numpy(), norm=norm, group_top=2, **form)
    assert np.array_equal(r.ids[-far:].cpu().numpy(), o["ids"])
    # as test_gpu_group has it: a difference of 2 max |l| rounded, exponentials and sums of E terms
    rel = (2 * np.abs(l).max() + 16 + n + k) * EPS
    mc.assert_within(r.weights[-far:], o["w"], rel * np.abs(o["w"]), "weights")
    ref, size = gc.grad(o, k, "sigmoid", norm, 2.5, dw[-far:].double().cpu().numpy(), 0.0, 0.0)
    mc.assert_within(d[-far:], ref, 4 * rel * size + mc.HALF_STEP["bf16"] * np.abs(ref) + 1e-37, "gradient")
    assert _quiet(d, far)
