"""Router of a mixture of experts: softmax top-k routing with the counts and losses that training
it needs. No counterpart in the reference, whose routers are trained elsewhere; the routing itself
is the one of its MoE block (see vqlab_amd.moe).

    p = softmax(logits); ids = top_k(p); weights = p[ids] (renormalised)
    over the n live tokens:  counts_e = tokens that chose expert e
    balance = E * sum_e counts_e / (n k) * mean_t p_te      (1 where the load is even)
    z       = mean_t logsumexp(logits_t)^2

Gradients reach the logits from weights, balance and z.

Other forms of the scores (score, bias, groups, top_groups, group_top, scale of top_k and route):

    s = sigmoid(logits) or softmax(logits); c = s + bias
    group score = sum of the group_top largest c of a group (groups equal runs of experts)
    ids = top_k(c) in the top_groups best groups; weights = scale * s[ids] (/ their sum)
    balance goes by p = s / sum(s)

c is compared in 64 bits (without a bias experts are in the order of their logits). The bias steers
the choice alone and takes no gradient: a buffer that a training loop moves against the counts.
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


SCORES = {"softmax": L.VQK_SCORE_SOFTMAX, "sigmoid": L.VQK_SCORE_SIGMOID}


class Form(NamedTuple):
    """How scores are made and chosen among (see the module's head); `plain` is softmax by itself."""
    score: str = "softmax"
    bias: torch.Tensor = None
    groups: int = 1
    top_groups: int = 1
    group_top: int = 2
    scale: float = 1.0

    @property
    def plain(self):
        return self.score == "softmax" and self.bias is None and self.top_groups == self.groups and self.scale == 1.0


def form(E, k, score="softmax", bias=None, groups=1, top_groups=None, group_top=None, scale=1.0):
    """A checked Form for E experts, top_groups all of them and group_top 2 unless given (a group of one
    expert scores as that)."""
    if score not in SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    groups = int(groups)
    if groups < 1 or E % groups:
        raise ValueError(f"{groups} groups of {E} experts")
    top_groups = groups if top_groups is None else int(top_groups)
    group_top = 2 if group_top is None else int(group_top)
    if not 1 <= top_groups <= groups:
        raise ValueError(f"top {top_groups} of {groups} groups")
    if group_top not in (1, 2):
        raise ValueError(f"a group's score from {group_top} experts (1 or 2 are taken)")
    if k > top_groups * (E // groups):
        raise ValueError(f"top {k} of {top_groups * (E // groups)} experts in {top_groups} groups")
    scale = float(scale)
    if not 0 < scale <= 3.4e38:
        raise ValueError(f"scale must be a positive number, got {scale}")
    if bias is not None:
        if bias.shape != (E,) or bias.dtype not in T.ACT_TYPES:
            raise ValueError(f"bias must be float16, bfloat16 or float32 [{E}], got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.detach().float()
    return Form(score, bias, groups, top_groups, group_top, scale)


def _c_form(f, bias):
    """The form as the library reads it; bias: its contiguous tensor, or None."""
    return L.VQKRouteForm(SCORES[f.score], f.groups, f.top_groups, f.group_top, f.scale,
                          None if bias is None else bias.data_ptr())


def rows(logits):
    """logits with contiguous rows, and the elements between them."""
    E = logits.shape[1]
    if logits.stride(1) != 1 or logits.stride(0) < E:
        logits = logits.contiguous()
    return logits, max(logits.stride(0), E)


def top_k(logits, k, norm_topk_prob=True, mask=None, score="softmax", bias=None, groups=1, top_groups=None,
          group_top=None, scale=1.0):
    """ids int32 [T, k] and weights fp32 [T, k] of logits [T, E], one launch: the routing of a
    serving step. mask [T] (bool / uint8): 0 marks padding, whose ids are -1. score .. scale: see the
    module's head. Logits that want a gradient are refused: that is route's."""
    k = int(k)
    _check(logits, k, mask)
    f = form(logits.shape[1], k, score, bias, groups, top_groups, group_top, scale)
    T.require_cuda(logits, f.bias)
    T.no_grad_here("router.top_k", logits)
    return _top_k(logits, k, norm_topk_prob, mask, f)


def _top_k(logits, k, norm_topk_prob, mask, f):
    with T.on_device(logits):
        lg, ld = rows(logits)
        m = mask_bytes(mask, lg)
        mp = None if m is None else m.data_ptr()
        n, E = lg.shape
        ids = lg.new_empty((n, k), dtype=torch.int32)
        w = lg.new_empty((n, k), dtype=torch.float32)
        if f.plain:
            rc = L.lib().vqk_route(lg.data_ptr(), T.act_type(lg), n, E, ld, mp, k, int(norm_topk_prob),
                                   ids.data_ptr(), w.data_ptr(), None, None, None, None, 0, T.raw_stream(lg))
        else:
            b = None if f.bias is None else f.bias.contiguous()
            rc = L.lib().vqk_route_grouped(lg.data_ptr(), T.act_type(lg), n, E, ld, mp,
                                           ctypes.byref(_c_form(f, b)), k, int(norm_topk_prob), ids.data_ptr(),
                                           w.data_ptr(), None, None, None, None, 0, T.raw_stream(lg))
        if rc:
            L.check(rc, "route")
    return ids, w


_sizes = {}                                     # (tokens, experts) -> workspace bytes


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, norm, mask, f):
        with T.on_device(logits):
            lg, ld = rows(logits)
            m = mask_bytes(mask, lg)
            mp = None if m is None else m.data_ptr()
            n, E = lg.shape
            plain = f.plain
            ids = lg.new_empty((n, k), dtype=torch.int32)
            w = lg.new_empty((n, k), dtype=torch.float32)
            counts = lg.new_empty(E, dtype=torch.int32)
            stats = lg.new_empty(3, dtype=torch.float32)
            saved = lg.new_empty((n, 2 if plain else 4), dtype=torch.float32)
            lib = L.lib()
            size = _sizes.get((n, E))
            if size is None:
                ws = ctypes.c_size_t()
                L.check(lib.vqk_route_workspace(n, E, ctypes.byref(ws)), "route")
                if len(_sizes) > 4096:
                    _sizes.clear()
                size = _sizes[(n, E)] = ws.value
            work = lg.new_empty(size, dtype=torch.uint8)
            out = (ids.data_ptr(), w.data_ptr(), counts.data_ptr(), stats.data_ptr(), saved.data_ptr(),
                   work.data_ptr(), size, T.raw_stream(lg))
            if plain:
                c_form, rc = None, lib.vqk_route(lg.data_ptr(), T.act_type(lg), n, E, ld, mp, k, norm, *out)
            else:
                bias = None if f.bias is None else f.bias.contiguous()
                c_form = _c_form(f, bias)
                rc = lib.vqk_route_grouped(lg.data_ptr(), T.act_type(lg), n, E, ld, mp, ctypes.byref(c_form), k, norm, *out)
                c_form.bias = None                          # the gradient reads no bias
            if rc:
                L.check(rc, "route")
        balance, z, tokens = stats.unbind()
        # no views, so that a loss can be scaled in place: the backward pass reads neither
        balance, z = balance.data, z.data
        ctx.save_for_backward(lg, ids, w, counts, stats, saved)
        ctx.k, ctx.norm, ctx.ld, ctx.form = k, norm, ld, c_form
        ctx.mark_non_differentiable(ids, counts, tokens)
        ctx.set_materialize_grads(False)
        return ids, w, counts, balance, z, tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _ids, dw, _counts, db, dz, _tokens):
        lg, ids, w, counts, stats, saved = ctx.saved_tensors
        for g in (dw, db, dz):
            if g is not None:
                T.no_grad_here("The gradient of the router", g)
        n, E = lg.shape
        with T.on_device(lg):
            d = lg.new_empty((n, E))
            grads = [None if g is None else _f32(g) for g in (dw, db, dz)]
            at = (ctx.k, ctx.norm, ids.data_ptr(), w.data_ptr(), counts.data_ptr(), stats.data_ptr(),
                  saved.data_ptr(), *(None if g is None else g.data_ptr() for g in grads), d.data_ptr(),
                  T.raw_stream(lg))
            if ctx.form is None:
                rc = L.lib().vqk_route_backward(lg.data_ptr(), T.act_type(lg), n, E, ctx.ld, *at)
            else:
                rc = L.lib().vqk_route_grouped_backward(lg.data_ptr(), T.act_type(lg), n, E, ctx.ld,
                                                        ctypes.byref(ctx.form), *at)
            if rc:
                L.check(rc, "route backward")
        return d, None, None, None, None


def route(logits, k, norm_topk_prob=True, mask=None, score="softmax", bias=None, groups=1, top_groups=None,
          group_top=None, scale=1.0):
    """Route of logits [T, E] (fp16, bf16 or fp32), differentiable in the logits. mask [T] (bool /
    uint8): 0 marks padding, which gets ids -1, weights 0 and a zero gradient and enters neither
    counts nor losses; so does a token whose logits are all -inf. score .. scale: see the module's
    head. The gradient reads ids, weights, counts and tokens again: copy them before anything changes
    them in place, a collective among it."""
    k = int(k)
    _check(logits, k, mask)
    f = form(logits.shape[1], k, score, bias, groups, top_groups, group_top, scale)
    T.require_cuda(logits, f.bias)
    return Route(*_RouteFn.apply(logits, k, int(norm_topk_prob), mask, f))
