"""The 8-bit tile kernels count the copies they have under way, so they must not spill (as
test_build_resources says of others)."""
from __future__ import annotations

import pytest

from test_build_resources import _kernels


def test_tile_kernels_do_not_spill():
    from vqlab_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("the library is not built")
    found = [k for k in _kernels(_lib.LIB_PATH.read_bytes()) if "k_f8_tiles" in k[".name"]]
    assert len(found) >= 4
    for k in found:
        used = {n: k[n] for n in (".private_segment_fixed_size", ".vgpr_spill_count")}
        assert not any(used.values()), (k[".name"], used)
