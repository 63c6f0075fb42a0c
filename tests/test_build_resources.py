"""What the built library says about its kernels: those that count their outstanding loads should
not spill. A spill is a memory access that the count does not know of; the waits would be for newer
loads than meant, and the loop would stand still where it is to run ahead."""
from __future__ import annotations

import struct

import msgpack
import pytest


def _kernels(data):
    """The kernel records of every code object in the library: AMD's metadata notes (name AMDGPU,
    type 32, a msgpack map)."""
    out, at = [], 0
    while (at := data.find(b"AMDGPU\0\0", at)) >= 0:
        namesz, descsz, kind = struct.unpack_from("<III", data, at - 12)
        if namesz == 7 and kind == 32 and 0 < descsz < len(data) - at - 8:
            out += msgpack.unpackb(data[at + 8:at + 8 + descsz])["amdhsa.kernels"]
        at += 8
    return out


@pytest.mark.parametrize("kernel", ["k_mx_gemm", "k_pgemm"])
def test_kernels_that_count_their_loads_do_not_spill(kernel):
    from vqlab_amd import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("the library is not built")
    found = [k for k in _kernels(_lib.LIB_PATH.read_bytes()) if kernel in k[".name"]]
    assert found
    for k in found:
        used = {n: k[n] for n in (".private_segment_fixed_size", ".vgpr_spill_count")}
        assert not any(used.values()), (k[".name"], used)
