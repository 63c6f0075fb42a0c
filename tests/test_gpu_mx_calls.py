"""How MXFP4 modules and the router are called and kept: types, derivatives, devices, state."""
from __future__ import annotations

import numpy as np
import pytest
import torch

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
