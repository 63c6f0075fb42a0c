"""Casts and moves of modules over quantised weights change no output."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import group_cases as gc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [40, 4100])
def test_the_block_chooses_the_same_after_casts(T):
    """Biases of which neighbours differ by less than a 16-bit number holds, over equal scores: rounded, they
    would choose by the lower id."""
    from vqlab_amd import mx
    torch.manual_seed(T)
    E, H, I = 16, 64, 96
    proj = lambda o, i: mx.MXSwitchLinear.from_weight(torch.randn(E, o, i, device="cuda") / i ** 0.5)
    bias = (1 + 1e-5 * torch.arange(E, device="cuda")).float()
    form = dict(score="sigmoid", groups=4, top_groups=2)
    block = mx.MXSparseMoeBlock(mx.MXSwitchGLU(proj(I, H), proj(I, H), proj(H, I)), 3, bias=bias, **form)
    x, lg = torch.randn(T, H, device="cuda", dtype=torch.bfloat16), torch.zeros(T, E, device="cuda")
    want = block(x, lg)
    o = gc.route(np.zeros((1, E)), 3, bias=bias.double().cpu().numpy(), **form)
    assert o["ids"][0].tolist() == [15, 14, 13]
    w = torch.full((T, 3), 1 / 3, device="cuda")
    assert torch.allclose(want, block.switch_mlp(x, torch.tensor([15, 14, 13], device="cuda").expand(T, 3), w), atol=0.02)
    for cast in (lambda: block.half(), lambda: block.bfloat16(), lambda: block.to(torch.bfloat16),
                 lambda: block.cpu().cuda(), lambda: block.type(torch.float16)):
        cast()
        assert block.bias.dtype == torch.float32 and block.bias.is_cuda and torch.equal(block(x, lg), want)


@pytest.mark.parametrize("act", [None, "fp8"])
def test_8_bit_linears_after_casts(act):
    from vqlab_amd import fp8
    torch.manual_seed(1)
    lin = fp8.F8Linear.from_weight(torch.randn(200, 300, device="cuda") * torch.logspace(-6, 6, 300, device="cuda"), act)
    x = torch.randn(9, 300, device="cuda")
    want, codes, scales = lin(x), lin.codes.view(torch.uint8), lin.scales
    for cast in (lambda: lin.half(), lambda: lin.type(torch.float16), lambda: lin.type(torch.bfloat16),
                 lambda: lin.cpu().type(torch.float16).cuda()):
        cast()
        assert torch.equal(lin.codes.view(torch.uint8), codes) and torch.equal(lin.scales, scales)
        assert torch.equal(lin(x), want)
