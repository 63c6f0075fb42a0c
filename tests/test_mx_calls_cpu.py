"""MXFP4 modules' handling of their arguments, where it needs no GPU."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("E", [8, 200, 300])
def test_ids_keep_their_values(dtype, E):
    """Every id a type holds stays itself or stays outside [0, E)."""
    from vqlab_amd import mx
    lim = torch.iinfo(dtype)
    ids = sorted({max(lim.min, min(lim.max, v)) for v in (0, 1, 7, 100, 199, 255, -1, -7, E, 2 ** 31, 2 ** 32 + 3, -2 ** 40)})
    got = mx._ids32(torch.tensor(ids, dtype=dtype), E)
    assert got.dtype == torch.int32
    for a, b in zip(ids, got.tolist()):
        assert a == b if 0 <= a < E else not 0 <= b < E


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.bool, torch.complex64])
def test_ids_are_integers(dtype):
    from vqlab_amd import mx
    with pytest.raises(ValueError, match="integers"):
        mx._ids32(torch.zeros(3, dtype=dtype), 8)


def test_a_tangent_counts_as_wanting_a_derivative():
    import torch.autograd.forward_ad as fw
    from vqlab_amd import _torch as T
    x = torch.randn(3)
    assert not T.has_tangent(x)
    T.no_grad_here("it", x, x)
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones(3))
        assert T.has_tangent(d) and not T.has_tangent(x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
            T.no_grad_here("it", x, d)
    leaf = torch.randn(3, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        T.no_grad_here("it", leaf)
    with torch.no_grad():
        T.no_grad_here("it", leaf)


@pytest.mark.parametrize("k", [-1, 0, 9])
def test_router_refuses_other_numbers_of_experts(k):
    from vqlab_amd import router
    for call in (router.top_k, router.route):
        with pytest.raises(ValueError, match="of 8 experts"):
            call(torch.zeros(4, 8), k)
