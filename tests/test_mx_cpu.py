"""MXFP4 and the router without a GPU: sizes, and every refusal that is made on the host before
anything is launched. The float64 oracles of the GPU tests are checked against each other here."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import mx_cases as mc


@pytest.fixture(scope="module")
def lib():
    from vqlab_amd import _lib
    return _lib.lib()


def _err(lib):
    return lib.vqk_last_error().decode()


OK, NOTIMPL, EINVAL, ESHARDED, EDEVICE, ENOSPACE = range(6)
P = ctypes.c_void_p(0x10000)          # never read: every call below is refused on the host
BF16, F32 = 1, 2


def _w(E=1, OUT=64, IN=128, codes=0x10000, scales=0x20000):
    from vqlab_amd import _lib as L
    return L.VQKMXWeights(codes, scales, E, OUT, IN, 0)


# ------------------------------------------------------------------ formats
def test_oracle_rounds_to_the_nearest_code():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((20, 96))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0]           # scale 1: the ties
    x[0, 8:32] = 0
    codes, scales = mc.quantize(x)
    v = mc.values(codes, scales, 96)
    assert v[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 4.0]
    step = 2.0 ** (scales.astype(np.float64) - 127).repeat(32, 1)
    top = np.abs(x.reshape(20, 3, 32)).max(-1)
    assert ((4 * step[:, ::32] <= top) & (top < 8 * step[:, ::32])).all()
    # off by at most half the widest step of the grid below 6, by up to 2 past it
    assert (np.abs(v - x) <= np.where(np.abs(x) <= 6 * step, step, 2 * step)).all()
    again = mc.quantize(v)
    assert np.array_equal(mc.values(*again, 96), v)


def test_oracle_special_blocks():
    x = np.zeros((3, 40))
    x[1, 3] = np.inf
    x[2, 39] = -1.0
    codes, scales = mc.quantize(x)
    assert scales.tolist() == [[0, 0], [255, 0], [0, 125]]
    v = mc.values(codes, scales, 40)
    assert np.isnan(v[1, :32]).all() and (v[1, 32:] == 0).all() and v[2, 39] == -1.0


def test_route_oracle_gradient_is_the_derivative():
    rng = np.random.default_rng(1)
    lg, dw = rng.standard_normal((6, 10)), rng.standard_normal((6, 3))
    for norm in (True, False):
        r = mc.route(lg, 3, norm)
        d = mc.route_grad(r, 3, norm, dw, 0.7, 0.3)

        def loss(l):
            o = mc.route(l, 3, norm)
            balance = 10 * (r["counts"] / (6 * 3) * o["p"].sum(0) / 6).sum()
            return (o["w"] * dw).sum() + 0.7 * balance + 0.3 * o["z"]
        for t in range(6):
            for e in range(10):
                hi, lo = lg.copy(), lg.copy()
                hi[t, e] += 1e-5
                lo[t, e] -= 1e-5
                assert abs((loss(hi) - loss(lo)) / 2e-5 - d[t, e]) < 1e-8


# -------------------------------------------------------------------- sizes
@pytest.mark.parametrize("E,OUT,IN,codes,scales", [
    (1, 1, 1, 1024, 256), (1, 16, 128, 1024, 256), (1, 17, 129, 4096, 512), (3, 64, 512, 3 * 16384, 3 * 1024),
    (2, 16, 640, 2 * 5 * 1024, 2 * 2 * 256)])
def test_pack_sizes(lib, E, OUT, IN, codes, scales):
    c, s = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.vqk_mx_pack_bytes(E, OUT, IN, ctypes.byref(c), ctypes.byref(s)) == OK
    assert (c.value, s.value) == (codes, scales)


# ----------------------------------------------------------------- refusals
def test_quantize_refusals(lib):
    assert lib.vqk_mx_quantize(P, 7, 1, 32, 32, P, P, None) == EINVAL and "type" in _err(lib)
    assert lib.vqk_mx_quantize(P, BF16, -1, 32, 32, P, P, None) == EINVAL
    assert lib.vqk_mx_quantize(P, BF16, 2, 32, 31, P, P, None) == EINVAL
    assert lib.vqk_mx_quantize(None, BF16, 1, 32, 32, P, P, None) == EINVAL
    assert lib.vqk_mx_quantize(P, BF16, 1, 32, 32, ctypes.c_void_p(0x10001), P, None) == EINVAL
    assert lib.vqk_mx_quantize(None, BF16, 0, 32, 32, None, None, None) == OK       # no rows
    assert lib.vqk_mx_dequantize(P, P, 1, 32, P, 4, None) == EINVAL
    assert lib.vqk_mx_dequantize(P, P, 1, -1, P, BF16, None) == EINVAL
    assert lib.vqk_mx_dequantize(ctypes.c_void_p(0x10002), P, 1, 32, P, BF16, None) == EINVAL
    assert lib.vqk_mx_dequantize(None, None, 3, 0, None, BF16, None) == OK
    c = ctypes.c_size_t()
    assert lib.vqk_mx_pack_bytes(0, 1, 1, ctypes.byref(c), ctypes.byref(c)) == EINVAL
    assert lib.vqk_mx_pack(ctypes.c_void_p(0x10008), P, 1, 16, 32, P, P, None, None) == EINVAL


def test_linear_refusals(lib):
    n = ctypes.c_size_t()
    r, b = ctypes.byref, _w()

    def call(w=b, x=P, xt=BF16, N=4, act=0, y=P, yt=BF16, ws=P, size=1 << 30):
        return lib.vqk_mx_linear(r(w), x, xt, N, act, y, yt, ws, size, None)
    assert call(w=_w(E=2)) == EINVAL
    assert call(w=_w(OUT=0)) == EINVAL and call(w=_w(codes=0)) == EINVAL
    assert call(w=_w(codes=0x10004)) == EINVAL and call(w=_w(scales=0x20002)) == EINVAL
    assert call(w=_w(OUT=1 << 20, IN=1 << 20)) == NOTIMPL and "4 GB" in _err(lib)
    assert call(xt=6) == EINVAL and call(act=2) == EINVAL and call(yt=6) == EINVAL
    assert call(N=-1) == EINVAL and call(x=None) == EINVAL and call(y=None) == EINVAL
    assert call(N=0, x=None, y=None, ws=None, size=0) == OK
    assert call(act=1, ws=None, size=0) == ENOSPACE
    assert call(xt=F32, size=64) == ENOSPACE and call(N=500, act=1, size=64) == ENOSPACE
    assert call(ws=ctypes.c_void_p(0x10010), act=1) == EINVAL
    assert lib.vqk_mx_linear_workspace(r(b), BF16, 4, 5, r(n)) == EINVAL
    assert lib.vqk_mx_linear_workspace(r(b), BF16, 4, 0, None) == EINVAL
    assert lib.vqk_mx_linear_dx(r(b), P, BF16, 4, P, BF16, None, 0, None) == ENOSPACE
    assert lib.vqk_mx_linear_dx(r(b), P, 5, 4, P, BF16, P, 1 << 30, None) == EINVAL
    assert lib.vqk_mx_linear_dx(r(_w(E=3)), P, BF16, 4, P, BF16, P, 1 << 30, None) == EINVAL
    assert lib.vqk_mx_linear_dx(r(b), None, BF16, 0, None, BF16, None, 0, None) == OK


def test_expert_refusals(lib):
    r = ctypes.byref
    w, up, down = _w(E=4, OUT=64, IN=128), _w(E=4, OUT=64, IN=128), _w(E=4, OUT=128, IN=64)
    n = ctypes.c_size_t()

    def switch(w=w, x=P, xt=BF16, T=4, ids=P, N=8, rep=2, y=P, yt=BF16, ws=P, size=1 << 30):
        return lib.vqk_mx_switch(r(w), x, xt, T, ids, N, rep, y, yt, ws, size, None)
    assert switch(N=9) == EINVAL and switch(rep=0) == EINVAL and switch(xt=3) == EINVAL
    assert switch(ids=None) == EINVAL and switch(size=0) == ENOSPACE
    assert switch(w=_w(E=5000)) == NOTIMPL and switch(ws=ctypes.c_void_p(0x10010)) == EINVAL
    assert switch(T=0, N=0, x=None, ids=None, y=None, ws=None, size=0) == OK

    def experts(g=w, u=up, d=down, xt=BF16, T=4, k=2, ids=P, ws=P, size=1 << 30, yt=BF16):
        return lib.vqk_mx_experts(r(g), r(u), r(d), P, xt, T, ids, P, k, P, yt, ws, size, None)
    assert experts(u=_w(E=4, OUT=32, IN=128)) == EINVAL and experts(d=_w(E=4, OUT=128, IN=96)) == EINVAL
    assert experts(d=_w(E=5, OUT=128, IN=64)) == EINVAL
    assert experts(k=0) == EINVAL and experts(k=5) == EINVAL and experts(T=-1) == EINVAL
    assert experts(ids=None) == EINVAL and experts(size=100) == ENOSPACE and experts(yt=9) == EINVAL
    assert lib.vqk_mx_moe(r(w), r(up), r(down), P, BF16, 4, None, F32, 4, None, 2, 1, P, BF16, P, 1 << 30,
                          None) == EINVAL
    assert lib.vqk_mx_moe(r(w), r(up), r(down), P, BF16, 4, P, F32, 3, None, 2, 1, P, BF16, P, 1 << 30,
                          None) == EINVAL                                 # logits rows of 3 for 4 experts
    assert lib.vqk_mx_moe(r(w), r(up), r(down), P, BF16, 4, P, F32, 4, None, 2, 1, P, BF16, P, 64, None) == ENOSPACE
    assert lib.vqk_mx_experts_workspace(r(w), r(up), r(down), BF16, 4, 2, None) == EINVAL
    assert lib.vqk_mx_moe_workspace(r(w), r(up), r(down), BF16, 4, 9, r(n)) == EINVAL


def test_route_refusals(lib):
    n = ctypes.c_size_t()

    def route(l=P, t=F32, T=4, E=8, ld=8, k=2, ids=P, w=P, counts=P, stats=P, saved=P, ws=P, size=1 << 20):
        return lib.vqk_route(l, t, T, E, ld, None, k, 1, ids, w, counts, stats, saved, ws, size, None)
    assert route(t=4) == EINVAL and route(T=-1) == EINVAL and route(ld=7) == EINVAL
    assert route(k=0) == EINVAL and route(k=9) == EINVAL and route(E=4096, ld=4096) == NOTIMPL
    assert route(E=512, ld=512, k=65) == NOTIMPL
    assert route(l=None) == EINVAL and route(stats=None) == EINVAL and route(size=8) == ENOSPACE
    assert route(saved=ctypes.c_void_p(0x10004)) == EINVAL
    assert lib.vqk_route_workspace(4, 9999, ctypes.byref(n)) == EINVAL
    assert lib.vqk_route_backward(P, F32, 4, 8, 8, 2, 1, P, P, P, P, None, P, P, P, P, None) == EINVAL
    assert lib.vqk_route_backward(P, F32, 0, 8, 8, 2, 1, None, None, None, None, None, None, None, None, None,
                                  None) == OK


def test_modules_refuse_what_they_cannot_take():
    from vqlab_amd import mx, router
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="device"):
        mx.mx_quantize(torch.zeros(2, 32))
    with pytest.raises(ValueError, match="device"):
        mx.MXLinear(codes, scales)
    with pytest.raises(ValueError, match="act"):
        mx.MXLinear(codes, scales, act="int4")
    with pytest.raises(ValueError, match="do not"):
        mx.MXLinear(codes, scales, 65)
    with pytest.raises(ValueError, match="uint8"):
        mx.MXLinear(codes.int(), scales)
    with pytest.raises(ValueError, match=r"\[OUT"):
        mx.MXLinear(codes[None], scales[None])
    with pytest.raises(ValueError, match=r"\[E, OUT"):
        mx.MXSwitchLinear(codes, scales)
    with pytest.raises(ValueError, match="device"):
        router.route(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match=r"\[T, E\]"):
        router.top_k(torch.zeros(8), 2)
    with pytest.raises(ValueError, match="float"):
        router.route(torch.zeros(4, 8, dtype=torch.int32), 2)
