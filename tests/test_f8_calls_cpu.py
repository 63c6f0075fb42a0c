"""Arguments that the 8-bit linears, the norm and the router by groups refuse, where that needs no GPU:
every call here ends in the host's checks, before any address is looked at."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from vqlab_amd import _lib as L

P = 1 << 20                                      # an aligned address that no call reads


@pytest.fixture(scope="module")
def lib():
    return L.lib()


def refused(lib, call, rc):
    assert call == rc, (call, lib.vqk_last_error())
    assert lib.vqk_last_error()


def test_workspaces(lib):
    """What a call reads in place takes none."""
    w, n = ctypes.byref(L.VQKF8Weights(P, P, 256, 512)), ctypes.c_size_t()
    size = lambda q, *a: (q(w, *a, ctypes.byref(n)), n.value)
    assert size(lib.vqk_f8_linear_workspace, L.VQK_BF16, 4, L.VQK_F8_ACT_NONE, L.VQK_BF16) == (0, 0)
    assert size(lib.vqk_f8_linear_workspace, L.VQK_F32, 4, L.VQK_F8_ACT_NONE, L.VQK_F32) == (0, 3 * 4 * 512 * 2)
    assert size(lib.vqk_f8_linear_workspace, L.VQK_BF16, 4, L.VQK_F8_ACT_F8, L.VQK_BF16) == (0, 4 * 512 + 256)
    assert size(lib.vqk_f8_linear_rows_workspace, 512, 4, L.VQK_BF16) == (0, 0)
    assert size(lib.vqk_f8_linear_rows_workspace, 520, 4, L.VQK_BF16) == (0, 4 * 512 + 256)
    assert size(lib.vqk_f8_linear_rows_workspace, 512, 4, L.VQK_F32) == (0, 4 * 512 + 256 + 4 * 1024)


def test_sizes_of_zero_rows_need_nothing(lib):
    """No rows: nothing is read or launched, whatever the addresses."""
    w = L.VQKF8Weights(P, P, 256, 512)
    for call in (lib.vqk_f8_quantize(None, L.VQK_BF16, 0, 128, 128, None, None, 1, 0, None),
                 lib.vqk_f8_dequantize(None, 128, None, 1, 0, 1, 0, 128, None, L.VQK_F32, None),
                 lib.vqk_rms_norm(None, L.VQK_F16, 0, 64, 64, None, 64, None, L.VQK_F16, 1e-6, None, None, None, None,
                                  None, 1, 0, None),
                 lib.vqk_f8_linear(ctypes.byref(w), None, L.VQK_BF16, 0, 0, None, L.VQK_BF16, None, 0, None),
                 lib.vqk_f8_linear_rows(ctypes.byref(w), None, 512, None, 1, 1, 0, None, L.VQK_BF16, None, 0, None),
                 lib.vqk_f8_linear_dx(ctypes.byref(w), None, L.VQK_BF16, 0, None, L.VQK_BF16, None, 0, None)):
        assert call == L.VQK_OK, lib.vqk_last_error()


@pytest.mark.parametrize("change,rc", [
    (dict(t=L.VQK_U8), L.VQK_EINVAL), (dict(rows=-1), L.VQK_EINVAL), (dict(cols=-1), L.VQK_EINVAL),
    (dict(ld=127), L.VQK_EINVAL), (dict(x=None), L.VQK_EINVAL), (dict(codes=None), L.VQK_EINVAL),
    (dict(scales=None), L.VQK_EINVAL), (dict(sr=-1), L.VQK_EINVAL), (dict(sb=-1), L.VQK_EINVAL)])
def test_quantize(lib, change, rc):
    a = dict(x=P, t=L.VQK_BF16, rows=4, cols=128, ld=128, codes=P, scales=P, sr=1, sb=4) | change
    refused(lib, lib.vqk_f8_quantize(a["x"], a["t"], a["rows"], a["cols"], a["ld"], a["codes"], a["scales"], a["sr"],
                                     a["sb"], None), rc)


@pytest.mark.parametrize("change", [dict(t=9), dict(out=-1), dict(inp=-1), dict(ld=99), dict(w=None), dict(codes=None),
                                    dict(scales=None)])
def test_quantize_weight(lib, change):
    a = dict(w=P, t=L.VQK_F32, out=100, inp=100, ld=100, codes=P, scales=P) | change
    refused(lib, lib.vqk_f8_quantize_weight(a["w"], a["t"], a["out"], a["inp"], a["ld"], a["codes"], a["scales"], None),
            L.VQK_EINVAL)


@pytest.mark.parametrize("change", [dict(ld=99), dict(t=L.VQK_I32), dict(per=64), dict(per=0), dict(sr=-1), dict(sb=-4),
                                    dict(codes=None), dict(scales=None), dict(out=None), dict(rows=-3)])
def test_dequantize(lib, change):
    a = dict(codes=P, ld=100, scales=P, sr=1, sb=4, per=1, rows=4, cols=100, out=P, t=L.VQK_F16) | change
    refused(lib, lib.vqk_f8_dequantize(a["codes"], a["ld"], a["scales"], a["sr"], a["sb"], a["per"], a["rows"], a["cols"],
                                       a["out"], a["t"], None), L.VQK_EINVAL)


def test_pack(lib):
    n = ctypes.c_size_t()
    refused(lib, lib.vqk_f8_pack_bytes(0, 128, ctypes.byref(n)), L.VQK_EINVAL)
    refused(lib, lib.vqk_f8_pack_bytes(128, 128, None), L.VQK_EINVAL)
    assert lib.vqk_f8_pack_bytes(17, 129, ctypes.byref(n)) == L.VQK_OK and n.value == 32 * 256
    refused(lib, lib.vqk_f8_pack(None, 16, 128, P, None), L.VQK_EINVAL)
    refused(lib, lib.vqk_f8_pack(P, 16, 128, P + 8, None), L.VQK_EINVAL)
    refused(lib, lib.vqk_f8_unpack(P + 4, 16, 128, P, None), L.VQK_EINVAL)


LINEAR = dict(codes=P, scales=P, out=256, inp=500, x=P, xt=L.VQK_BF16, n=4, act=L.VQK_F8_ACT_NONE, y=P, yt=L.VQK_BF16,
              ws=P, short=0)


def linear(lib, a):
    w = ctypes.byref(L.VQKF8Weights(a["codes"], a["scales"], a["out"], a["inp"]))
    n = ctypes.c_size_t()
    if lib.vqk_f8_linear_workspace(w, a["xt"], a["n"], a["act"], a["yt"], ctypes.byref(n)):
        n.value = 1 << 40                        # refused there as well
    return lib.vqk_f8_linear(w, a["x"], a["xt"], a["n"], a["act"], a["y"], a["yt"], a["ws"], n.value - a["short"], None)


@pytest.mark.parametrize("change,rc", [
    (dict(codes=None), L.VQK_EINVAL), (dict(scales=None), L.VQK_EINVAL), (dict(codes=P + 8), L.VQK_EINVAL),
    (dict(out=0), L.VQK_EINVAL), (dict(inp=-1), L.VQK_EINVAL), (dict(n=-1), L.VQK_EINVAL),
    (dict(xt=L.VQK_U32), L.VQK_EINVAL), (dict(yt=L.VQK_U8), L.VQK_EINVAL), (dict(act=2), L.VQK_EINVAL),
    (dict(x=None), L.VQK_EINVAL), (dict(y=None), L.VQK_EINVAL), (dict(x=P + 8), L.VQK_EINVAL),
    (dict(ws=P + 64), L.VQK_EINVAL), (dict(ws=None), L.VQK_ENOSPACE), (dict(short=1), L.VQK_ENOSPACE)])
def test_linear(lib, change, rc):
    refused(lib, linear(lib, LINEAR | change), rc)


@pytest.mark.parametrize("change,rc", [
    (dict(x=None), L.VQK_EINVAL), (dict(sc=None), L.VQK_EINVAL), (dict(ld=511), L.VQK_EINVAL),
    (dict(sn=-1), L.VQK_EINVAL), (dict(sk=-1), L.VQK_EINVAL), (dict(y=None), L.VQK_EINVAL),
    (dict(x=P + 8), L.VQK_EINVAL),
    (dict(yt=L.VQK_I64), L.VQK_EINVAL), (dict(ws=P + 16), L.VQK_EINVAL), (dict(short=1), L.VQK_ENOSPACE)])
def test_linear_of_rows(lib, change, rc):
    a = dict(x=P, ld=512, sc=P, sn=1, sk=4, n=4, y=P, yt=L.VQK_F32, ws=P, short=0) | change
    w = ctypes.byref(L.VQKF8Weights(P, P, 256, 512))
    n = ctypes.c_size_t()
    if lib.vqk_f8_linear_rows_workspace(w, a["ld"], a["n"], a["yt"], ctypes.byref(n)):
        n.value = 1 << 40
    refused(lib, lib.vqk_f8_linear_rows(w, a["x"], a["ld"], a["sc"], a["sn"], a["sk"], a["n"], a["y"], a["yt"], a["ws"],
                                        n.value - a["short"], None), rc)


@pytest.mark.parametrize("change,rc", [
    (dict(dy=None), L.VQK_EINVAL), (dict(dy=P + 4), L.VQK_EINVAL), (dict(dx=None), L.VQK_EINVAL), (dict(dt=L.VQK_U16), L.VQK_EINVAL),
    (dict(yt=7), L.VQK_EINVAL), (dict(ws=P + 128), L.VQK_EINVAL), (dict(short=1), L.VQK_ENOSPACE)])
def test_linear_gradient(lib, change, rc):
    a = dict(dy=P, dt=L.VQK_F16, n=4, dx=P, yt=L.VQK_F16, ws=P, short=0) | change
    w = ctypes.byref(L.VQKF8Weights(P, P, 256, 512))
    n = ctypes.c_size_t()
    if lib.vqk_f8_linear_dx_workspace(w, a["dt"], a["n"], ctypes.byref(n)):
        n.value = 1 << 40
    refused(lib, lib.vqk_f8_linear_dx(w, a["dy"], a["dt"], a["n"], a["dx"], a["yt"], a["ws"], n.value - a["short"], None), rc)


def norm(lib, **change):
    a = dict(x=P, t=L.VQK_BF16, n=4, c=256, ldx=256, res=P, ldr=256, w=P, wt=L.VQK_F32, eps=1e-6, h=P, y=P, r=None,
             codes=None, scales=None, sr=1, sb=4) | change
    return lib.vqk_rms_norm(a["x"], a["t"], a["n"], a["c"], a["ldx"], a["res"], a["ldr"], a["w"], a["wt"], a["eps"],
                            a["h"], a["y"], a["r"], a["codes"], a["scales"], a["sr"], a["sb"], None)


@pytest.mark.parametrize("change,rc", [
    (dict(t=L.VQK_U8), L.VQK_EINVAL), (dict(wt=L.VQK_I32), L.VQK_EINVAL), (dict(n=-1), L.VQK_EINVAL),
    (dict(n=1 << 31), L.VQK_EINVAL), (dict(c=0), L.VQK_EINVAL), (dict(c=16385, ldx=16385, ldr=16385), L.VQK_ENOTIMPL),
    (dict(eps=-1e-9), L.VQK_EINVAL), (dict(eps=math.nan), L.VQK_EINVAL), (dict(ldx=255), L.VQK_EINVAL),
    (dict(ldr=255), L.VQK_EINVAL), (dict(x=None), L.VQK_EINVAL), (dict(w=None), L.VQK_EINVAL), (dict(h=None), L.VQK_EINVAL),
    (dict(y=None), L.VQK_EINVAL), (dict(codes=P, scales=P), L.VQK_EINVAL), (dict(y=None, codes=P), L.VQK_EINVAL),
    (dict(y=None, codes=P, scales=P, sr=-1), L.VQK_EINVAL), (dict(y=None, codes=P, scales=P, sb=-1), L.VQK_EINVAL)])
def test_norm(lib, change, rc):
    refused(lib, norm(lib, **change), rc)


@pytest.mark.parametrize("change,rc", [
    (dict(h=None), L.VQK_EINVAL), (dict(w=None), L.VQK_EINVAL), (dict(r=None), L.VQK_EINVAL), (dict(dy=None), L.VQK_EINVAL),
    (dict(dx=None), L.VQK_EINVAL), (dict(dw=None), L.VQK_EINVAL), (dict(ld=99), L.VQK_EINVAL),
    (dict(ws=None), L.VQK_ENOSPACE), (dict(short=1), L.VQK_ENOSPACE), (dict(ws=P + 8), L.VQK_EINVAL),
    (dict(c=20000, ld=20000), L.VQK_ENOTIMPL)])
def test_norm_gradient(lib, change, rc):
    a = dict(h=P, n=7, c=100, ld=100, w=P, r=P, dy=P, dh=None, dx=P, dw=P, ws=P, short=0) | change
    n = ctypes.c_size_t()
    if lib.vqk_rms_norm_backward_workspace(a["n"], a["c"], ctypes.byref(n)):
        n.value = 1 << 40
    refused(lib, lib.vqk_rms_norm_backward(a["h"], L.VQK_F16, a["n"], a["c"], a["ld"], a["w"], L.VQK_F32, a["r"], a["dy"],
                                           a["dh"], a["dx"], a["dw"], a["ws"], n.value - a["short"], None), rc)


FORM = dict(score=L.VQK_SCORE_SIGMOID, groups=8, top=4, per=2, scale=2.5, bias=P)


@pytest.mark.parametrize("form,rc", [
    (dict(score=2), L.VQK_EINVAL), (dict(groups=0), L.VQK_EINVAL), (dict(groups=7), L.VQK_EINVAL),
    (dict(groups=128), L.VQK_ENOTIMPL), (dict(top=0), L.VQK_EINVAL), (dict(top=9), L.VQK_EINVAL),
    (dict(per=3), L.VQK_ENOTIMPL), (dict(per=0), L.VQK_ENOTIMPL), (dict(scale=0.), L.VQK_EINVAL),
    (dict(scale=-1.), L.VQK_EINVAL), (dict(scale=math.inf), L.VQK_EINVAL), (dict(scale=math.nan), L.VQK_EINVAL),
    (dict(groups=64, top=1), L.VQK_EINVAL)])     # top 8 of 4 experts
def test_route_forms(lib, form, rc):
    f = FORM | form
    c = L.VQKRouteForm(f["score"], f["groups"], f["top"], f["per"], f["scale"], f["bias"])
    refused(lib, lib.vqk_route_grouped(P, L.VQK_F32, 4, 256, 256, None, ctypes.byref(c), 8, 1, P, P, None, None, None, None,
                                       0, None), rc)
    refused(lib, lib.vqk_route_grouped_backward(P, L.VQK_F32, 4, 256, 256, ctypes.byref(c), 8, 1, P, P, P, P, P, P, P, P, P,
                                                None), rc)


def test_route_arguments(lib):
    c = ctypes.byref(L.VQKRouteForm(*FORM.values()))

    def call(logits=P, t=L.VQK_F32, T=4, E=256, ld=256, form=c, k=8, ids=P, w=P, counts=None, stats=None, saved=None, ws=None,
             size=0):
        return lib.vqk_route_grouped(logits, t, T, E, ld, None, form, k, 1, ids, w, counts, stats, saved, ws, size, None)
    n = ctypes.c_size_t()
    assert lib.vqk_route_workspace(4, 256, ctypes.byref(n)) == L.VQK_OK
    for change in (dict(logits=None), dict(t=L.VQK_U8), dict(T=-1), dict(ld=255), dict(form=None), dict(k=0), dict(k=257),
                   dict(ids=None), dict(w=None), dict(counts=P), dict(stats=P), dict(saved=P + 8),
                   dict(counts=P, stats=P, ws=P + 8, size=n.value)):
        refused(lib, call(**change), L.VQK_EINVAL)
    refused(lib, call(counts=P, stats=P, ws=P, size=n.value - 1), L.VQK_ENOSPACE)
    refused(lib, call(counts=P, stats=P), L.VQK_ENOSPACE)


@pytest.mark.parametrize("change,words", [
    (dict(score="tanh"), "score must be"), (dict(groups=0), "0 groups"), (dict(groups=7), "7 groups"),
    (dict(groups=8, top_groups=9), "top 9 of 8"), (dict(groups=8, top_groups=0), "top 0 of 8"),
    (dict(groups=8, group_top=3), "from 3 experts"), (dict(groups=8, group_top=0), "from 0 experts"),
    (dict(groups=16, top_groups=1), "top 6 of 4"), (dict(scale=0), "positive"), (dict(scale=float("nan")), "positive"),
    (dict(bias=torch.zeros(63)), "bias must be"), (dict(bias=torch.zeros(64, dtype=torch.float64)), "bias must be")])
def test_python_forms(change, words):
    from vqlab_amd import router
    with pytest.raises(ValueError, match=words):
        router.form(64, 6, **change)


def test_python_defaults():
    from vqlab_amd import router
    f = router.form(64, 6, groups=8)
    assert f.plain and (f.top_groups, f.group_top) == (8, 2)
    assert not router.form(64, 6, scale=2.0).plain and not router.form(64, 6, groups=8, top_groups=2).plain
    assert router.form(8, 2, groups=8, top_groups=3).group_top == 2       # of groups of one: that one


def test_python_calls_want_a_gpu():
    from vqlab_amd import fp8, router
    x, w = torch.zeros(2, 128), torch.ones(128)
    for call in (lambda: fp8.f8_quantize(x), lambda: fp8.f8_quantize_weight(x), lambda: fp8.rms_norm(x, w),
                 lambda: fp8.rms_norm_f8(x, w), lambda: fp8.f8_dequantize(x.to(fp8.F8), torch.ones(2, 1)),
                 lambda: fp8.F8Linear(x.to(fp8.F8), torch.ones(1, 1)),
                 lambda: router.top_k(x, 2, score="sigmoid")):
        with pytest.raises(ValueError, match="device"):
            call()
    with pytest.raises(ValueError, match="act must be"):
        fp8.F8Linear(x.to(fp8.F8), torch.ones(1, 1), act="mxfp4")
    with pytest.raises(ValueError, match=r"codes must be \[OUT, IN\]"):
        fp8.F8Linear(torch.zeros(4, dtype=torch.uint8), torch.ones(1, 1))
