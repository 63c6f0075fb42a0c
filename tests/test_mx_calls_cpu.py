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
