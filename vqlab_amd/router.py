"""Router of a mixture of experts: softmax top-k routing with the counts and losses that training
it needs. No counterpart in the reference, whose routers are trained elsewhere; the routing itself
is the one of its MoE block (see vqlab_amd.moe).

    p = softmax(logits); ids = top_k(p); weights = p[ids] (renormalised)
    over the n live tokens:  counts_e = tokens that chose expert e
    balance = E * sum_e counts_e / (n k) * mean_t p_te      (1 where the load is even)
    z       = mean_t logsumexp(logits_t)^2

Gradients reach the logits from weights, balance and z.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib as L
from . import _torch as T


class Route(NamedTuple):
    """ids int32 [T, k] (-1: none), weights fp32 [T, k], counts int32 [E], balance and z fp32
    scalars, tokens fp32 scalar (the live tokens n)."""
    ids: torch.Tensor
    weights: torch.Tensor
    counts: torch.Tensor
    balance: torch.Tensor
    z: torch.Tensor
    tokens: torch.Tensor


def mask_bytes(mask, logits):
    """mask [T] (bool / uint8) of logits [T, E] as contiguous bytes, or None."""
    if mask is None:
        return None
    if mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError(f"mask must be bool or uint8, got {mask.dtype}")
    if mask.shape != logits.shape[:1]:
        raise ValueError(f"mask {tuple(mask.shape)} for logits {tuple(logits.shape)}")
    return mask.contiguous()


def _check(logits, k, mask):
    if logits.ndim != 2:
        raise ValueError(f"logits must be [T, E], got {tuple(logits.shape)}")
    if not 1 <= k <= logits.shape[1]:
        raise ValueError(f"top {k} of {logits.shape[1]} experts")
    T.act_type(logits)
    T.require_cuda(logits, mask)


def _f32(g):
    return g if g.dtype == torch.float32 and g.is_contiguous() else g.float().contiguous()


def rows(logits):
    """logits with contiguous rows, and the elements between them."""
    E = logits.shape[1]
    if logits.stride(1) != 1 or logits.stride(0) < E:
        logits = logits.contiguous()
    return logits, max(logits.stride(0), E)


def top_k(logits, k, norm_topk_prob=True, mask=None):
    """ids int32 [T, k] and weights fp32 [T, k] of logits [T, E], one launch: the routing of a
    serving step. mask [T] (bool / uint8): 0 marks padding, whose ids are -1. Logits that want a
    gradient are refused: that is route's."""
    k = int(k)
    _check(logits, k, mask)
    T.no_grad_here("router.top_k", logits)
    with T.on_device(logits):
        lg, ld = rows(logits)
        m = mask_bytes(mask, lg)
        mp = None if m is None else m.data_ptr()
        n, E = lg.shape
        ids = torch.empty((n, k), dtype=torch.int32, device=lg.device)
        w = torch.empty((n, k), dtype=torch.float32, device=lg.device)
        L.check(L.lib().vqk_route(lg.data_ptr(), T.act_type(lg), n, E, ld, mp, k,
                                  int(norm_topk_prob), ids.data_ptr(), w.data_ptr(), None, None,
                                  None, None, 0, T.raw_stream(lg)), "route")
    return ids, w


_sizes = {}                                     # (tokens, experts) -> workspace bytes


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, norm, mask):
        with T.on_device(logits):
            lg, ld = rows(logits)
            m = mask_bytes(mask, lg)
            mp = None if m is None else m.data_ptr()
            n, E = lg.shape
            dev = lg.device
            ids = torch.empty((n, k), dtype=torch.int32, device=dev)
            w = torch.empty((n, k), dtype=torch.float32, device=dev)
            counts = torch.empty(E, dtype=torch.int32, device=dev)
            stats = torch.empty(3, dtype=torch.float32, device=dev)
            saved = torch.empty((n, 2), dtype=torch.float32, device=dev)
            lib = L.lib()
            size = _sizes.get((n, E))
            if size is None:
                ws = ctypes.c_size_t()
                L.check(lib.vqk_route_workspace(n, E, ctypes.byref(ws)), "route")
                if len(_sizes) > 4096:
                    _sizes.clear()
                size = _sizes[(n, E)] = ws.value
            work = torch.empty(size, dtype=torch.uint8, device=dev)
            L.check(lib.vqk_route(lg.data_ptr(), T.act_type(lg), n, E, ld, mp, k, norm,
                                  ids.data_ptr(), w.data_ptr(), counts.data_ptr(),
                                  stats.data_ptr(), saved.data_ptr(), work.data_ptr(), size,
                                  T.raw_stream(lg)), "route")
        balance, z, tokens = stats.unbind()
        # no views, so that a loss can be scaled in place: the backward pass reads neither
        balance, z = balance.data, z.data
        ctx.save_for_backward(lg, ids, w, counts, stats, saved)
        ctx.k, ctx.norm, ctx.ld = k, norm, ld
        ctx.mark_non_differentiable(ids, counts, tokens)
        ctx.set_materialize_grads(False)
        return ids, w, counts, balance, z, tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _ids, dw, _counts, db, dz, _tokens):
        lg, ids, w, counts, stats, saved = ctx.saved_tensors
        T.no_grad_here("The gradient of the router", *(g for g in (dw, db, dz) if g is not None))
        n, E = lg.shape
        with T.on_device(lg):
            d = torch.empty((n, E), dtype=lg.dtype, device=lg.device)
            grads = [None if g is None else _f32(g) for g in (dw, db, dz)]
            L.check(L.lib().vqk_route_backward(
                lg.data_ptr(), T.act_type(lg), n, E, ctx.ld, ctx.k, ctx.norm, ids.data_ptr(),
                w.data_ptr(), counts.data_ptr(), stats.data_ptr(), saved.data_ptr(),
                *(None if g is None else g.data_ptr() for g in grads), d.data_ptr(),
                T.raw_stream(lg)), "route backward")
        return d, None, None, None


def route(logits, k, norm_topk_prob=True, mask=None):
    """Route of logits [T, E] (fp16, bf16 or fp32), differentiable in the logits. mask [T] (bool /
    uint8): 0 marks padding, which gets ids -1, weights 0 and a zero gradient and enters neither
    counts nor losses; so does a token whose logits are all -inf. The gradient reads ids, weights,
    counts and tokens again: copy them before anything changes them in place, a collective among it."""
    k = int(k)
    _check(logits, k, mask)
    return Route(*_RouteFn.apply(logits, k, int(norm_topk_prob), mask))
