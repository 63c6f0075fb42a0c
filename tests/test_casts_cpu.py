"""Casts of modules over quantised weights: what decides exactly (the routing bias, the scales of 8-bit
weights) keeps its bits. On the CPU, over modules whose device work is left out."""
from __future__ import annotations

import copy

import pytest
import torch

from vqlab_amd import fp8, mx

CASTS = [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.bfloat16),
         lambda m: m.type(torch.float16), lambda m: m.type(torch.bfloat16), lambda m: m.to("cpu")]
NAMES = ["half", "bfloat16", "double", "to", "type-half", "type-bfloat16", "device"]


class Experts(torch.nn.Module):
    def __init__(self, E):
        super().__init__()
        self.gate_proj = torch.nn.Module()
        self.gate_proj.num_experts = E


def block(bias, **form):
    return mx.MXSparseMoeBlock(Experts(16), 2, bias=bias, score="sigmoid", groups=4, top_groups=2, **form)


@pytest.mark.parametrize("cast", CASTS, ids=NAMES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_routing_bias_keeps_its_bits(cast, dtype):
    bias = (0.1 * torch.randn(16, generator=torch.Generator().manual_seed(1)) + 1 / 3).to(dtype)
    was = bias.clone()
    for m in (block(bias.clone()), torch.nn.Sequential(block(bias.clone()))):
        cast(m)
        b = m if isinstance(m, mx.MXSparseMoeBlock) else m[0]
        assert b.bias.dtype == dtype and torch.equal(b.bias, was)
        assert torch.equal(b.state_dict()["bias"], was) and list(dict(b.named_buffers())) == ["bias"]


def test_the_bias_stays_the_tensor_that_a_training_loop_moves():
    bias = torch.zeros(16)
    b = block(bias)
    b.half().to("cpu")
    bias += 1e-5
    assert torch.equal(b.bias, bias) and float(b.bias[0]) != 0
    strided = torch.arange(32.0)[::2]
    assert torch.equal(block(strided).bfloat16().bias, torch.arange(32.0)[::2])
    with pytest.raises(RuntimeError, match="no"):
        def fail(t):
            raise RuntimeError("no")
        b._apply(fail)
    assert torch.equal(b.bias, bias)                       # a cast that fails loses nothing


def test_blocks_without_a_bias():
    m = mx.MXSparseMoeBlock(Experts(16), 2, score="sigmoid").half()
    assert m.bias is None and "bias" not in m.state_dict()
    plain = mx.MXSparseMoeBlock(Experts(16), 2, router_weight=torch.nn.Parameter(torch.randn(16, 8))).half()
    assert plain.router_weight.dtype == torch.float16

@pytest.mark.parametrize("cast", CASTS, ids=NAMES)
def test_scales_of_8_bit_weights_keep_their_bits(cast):
    g = torch.Generator().manual_seed(2)
    packed = torch.randint(0, 256, (16 * 2 * 256,), generator=g).to(torch.uint8)
    scales = 2.0 ** (200 * torch.rand(1, 2, generator=g) - 120)
    lin = fp8.F8Linear.__new__(fp8.F8Linear)
    torch.nn.Module.__init__(lin)
    lin.out_features, lin.in_features, lin.act, lin._sizes = 32, 256, None, {}
    lin._keep(packed, scales)
    cast(lin)
    assert torch.equal(lin._packed[0], packed) and lin._packed[0].dtype == torch.uint8
    assert torch.equal(lin._packed[1], scales) and lin._packed[1].dtype == torch.float32
    assert lin._packed[1].shape == (1, 2)
    other = copy.deepcopy(lin)
    assert torch.equal(other._packed[1], scales) and other._packed[1].data_ptr() != lin._packed[1].data_ptr()
