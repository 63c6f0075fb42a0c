"""MXFP4 (microscaled 4-bit) weights for PyTorch-ROCm, beside the VQ modules. No counterpart in
the reference, whose formats are vector-quantised: this is the OCP microscaling format that
gfx950's matrix cores multiply directly.

A row of C values is ceil(C / 32) blocks of 32: 16 bytes of 4-bit codes each (element 2i in the
low half of byte i) and one scale byte s, value = e2m1(code) * 2^(s - 127); s = 255 is a block of
NaN (include/vqk.h).

  mx_quantize(x) -> codes, scales         mx_dequantize(codes, scales, cols, dtype)
  MXLinear(codes, scales, in_features)    bias-free linear, like VQLinear
  MXSwitchLinear                          routed linears, called like VQSwitchLinear
  MXSwitchGLU, MXSparseMoeBlock           routed experts with their weighted sum, and routing in front
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib as L
from . import _torch as T
from . import router

BLOCK = 32


def _blocks(cols):
    return -(-int(cols) // BLOCK)


def mx_quantize(x):
    """x [..., C] (fp16, bf16, fp32) -> codes uint8 [..., 16 B], scales uint8 [..., B],
    B = ceil(C / 32). Each block's scale is 2^(floor(log2(max |x|)) - 2), at least 2^-127; elements
    are rounded to nearest (ties to even), past 6 to 6. A block with an infinity or NaN becomes NaN.
    Not differentiable."""
    T.require_cuda(x)
    xt = T.act_type(x)
    if x.ndim == 0:
        raise ValueError("mx_quantize takes rows, got a scalar")
    T.no_grad_here("mx_quantize", x)
    C, B = x.shape[-1], _blocks(x.shape[-1])
    with T.on_device(x):
        if x.ndim == 2 and x.stride(1) == 1 and x.stride(0) >= C:
            rows, ld = x, x.stride(0)                  # rows apart: read where they are
        else:
            rows, ld = x.contiguous(), C
        n = x.numel() // C if C else 0
        lead = x.shape[:-1]
        codes = torch.empty((*lead, 16 * B), dtype=torch.uint8, device=x.device)
        scales = torch.empty((*lead, B), dtype=torch.uint8, device=x.device)
        L.check(L.lib().vqk_mx_quantize(rows.data_ptr(), xt, n, C, ld, codes.data_ptr(),
                                        scales.data_ptr(), T.raw_stream(x)), "mx_quantize")
    return codes, scales


def _check_mx(codes, scales, cols, what):
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"{what}: codes and scales must be uint8, got {codes.dtype}, {scales.dtype}")
    B = _blocks(cols)
    if codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != 16 * B or scales.shape[-1] != B:
        raise ValueError(f"{what}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not "
                         f"hold rows of {cols} values ({16 * B} and {B} bytes)")


def mx_dequantize(codes, scales, cols, dtype=torch.bfloat16):
    """The values [..., cols] that codes and scales stand for, in dtype (exact in bf16 and fp32; 2^128
    and more, which scales of 253 and 254 can say, are infinite)."""
    T.require_cuda(codes, scales)
    _check_mx(codes, scales, cols, "mx_dequantize")
    if dtype not in T.ACT_TYPES:
        raise ValueError(f"dtype must be float16, bfloat16 or float32, got {dtype}")
    with T.on_device(codes):
        codes, scales = _aligned(codes, 4), scales.contiguous()
        out = torch.empty((*scales.shape[:-1], int(cols)), dtype=dtype, device=codes.device)
        n = out.numel() // int(cols) if cols else 0
        L.check(L.lib().vqk_mx_dequantize(codes.data_ptr(), scales.data_ptr(), n, int(cols),
                                          out.data_ptr(), T.ACT_TYPES[dtype],
                                          T.raw_stream(codes)), "mx_dequantize")
    return out


def _aligned(t, n):
    """t contiguous, its first byte at a multiple of n."""
    t = t.contiguous()
    return t if t.data_ptr() % n == 0 else t.clone()


_IDS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _ids32(ids, E):
    """ids as int32; a wider id keeps being outside [0, E) when it is."""
    if ids.dtype not in _IDS:
        raise ValueError(f"expert ids must be integers (uint8, int8 .. int64), got {ids.dtype}")
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, E)
    return ids.to(torch.int32).contiguous()


def _desc(packed, E, OUT, IN):
    codes, scales, f16_exact = packed
    return L.VQKMXWeights(codes.data_ptr(), scales.data_ptr(), E, OUT, IN, f16_exact)


def _pack(codes, scales, E, OUT, IN):
    """Codes and scales of E weights in the kernels' operand order (laid out once), and whether
    every weight is an fp16 number (looked up once: the one wait for the GPU here)."""
    T.require_cuda(codes, scales)
    nc, ns = ctypes.c_size_t(), ctypes.c_size_t()
    L.check(L.lib().vqk_mx_pack_bytes(E, OUT, IN, ctypes.byref(nc), ctypes.byref(ns)), "MXFP4 weight")
    with T.on_device(codes):
        codes, scales = _aligned(codes, 16), scales.contiguous()
        pc = torch.empty(nc.value, dtype=torch.uint8, device=codes.device)
        ps = torch.empty(ns.value, dtype=torch.uint8, device=codes.device)
        inexact = torch.zeros(1, dtype=torch.int32, device=codes.device)
        L.check(L.lib().vqk_mx_pack(codes.data_ptr(), scales.data_ptr(), E, OUT, IN, pc.data_ptr(),
                                    ps.data_ptr(), inexact.data_ptr(), T.raw_stream(codes)),
                "MXFP4 weight")
        return pc, ps, int(inexact.item() == 0)


def _ws_bytes(sizes, key, query, *args):
    """Workspace bytes of a call, asked of the library once for each (shape, type)."""
    n = sizes.get(key)
    if n is None:
        ws = ctypes.c_size_t()
        L.check(query(*args, ctypes.byref(ws)), "workspace")
        if len(sizes) > 4096:
            sizes.clear()
        n = sizes[key] = ws.value
    return n


def _work(like, n):
    """A workspace of n bytes beside `like`, and its address (None, None: none needed)."""
    if not n:
        return None, None
    t = torch.empty(n, dtype=torch.uint8, device=like.device)
    return t, t.data_ptr()


class _Packed(torch.nn.Module):
    """A module over packed weights: `_packed` tensors, `_shape` (E, OUT, IN), and the descriptor
    `_w` of them that the library reads, which a copy or a move makes anew. `codes` and `scales`
    are the rows they were packed from, and what state_dict() holds."""

    _rows = 3                                   # dimensions of codes and scales

    def _set(self, codes, scales, E, OUT, IN):
        self._shape = (int(E), int(OUT), int(IN))
        self._sizes = {}
        self._keep(_pack(codes, scales, *self._shape))

    def _keep(self, packed):
        self._packed = packed
        self._w = _desc(packed, *self._shape)

    def _unpack(self, i, a, b, cols):
        """Packed tensor i, [E, RT, groups, 4, 16, n], with its row of 16 moved to the front and its
        last dimensions in the order a, b: rows [E, OUT, cols]."""
        E, OUT, _ = self._shape
        t = self._packed[i].view(E, -(-OUT // 16), -1, 4, 16, (16, 4)[i])
        t = t.permute(0, 1, 4, 2, a, b).reshape(E, -(-OUT // 16) * 16, -1)[:, :OUT, :cols]
        return (t if self._rows == 3 else t[0]).contiguous()

    @property
    def codes(self):
        """Codes uint8 [(E,) OUT, 16 B], unpacked by each access."""
        return self._unpack(0, 3, 5, 16 * _blocks(self._shape[2]))

    @property
    def scales(self):
        """Scales uint8 [(E,) OUT, B], unpacked by each access."""
        return self._unpack(1, 5, 3, _blocks(self._shape[2]))

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "codes"], destination[prefix + "scales"] = self.codes, self.scales

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys,
                              unexpected_keys, error_msgs):
        names = (prefix + "codes", prefix + "scales")
        super()._load_from_state_dict({k: v for k, v in state_dict.items() if k not in names}, prefix,
                                      local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        lost = [n for n in names if n not in state_dict]
        if lost:
            missing_keys.extend(lost)
            return
        B = _blocks(self._shape[2])
        rows = self._shape[3 - self._rows:2]
        wrong = [f"{n}: {t.dtype} of shape {tuple(t.shape)}, the module holds uint8 of shape {(*rows, c)}"
                 for n, t, c in zip(names, map(state_dict.get, names), (16 * B, B))
                 if t.dtype != torch.uint8 or t.shape != (*rows, c)]
        if wrong:
            error_msgs.extend(wrong)
            return
        here = self._packed[0].device
        at = here if here.type == "cuda" else "cuda"       # packed by a GPU, kept where the module is
        new = _pack(*(state_dict[n].to(at) for n in names), *self._shape)
        for old, t in zip(self._packed, new[:2]):          # in place: captured graphs read these
            old.copy_(t)
        self._keep((*self._packed[:2], new[2]))

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        codes, scales, exact = self._packed
        self._keep((fn(codes).to(torch.uint8), fn(scales).to(torch.uint8), exact))
        return self

    def __getstate__(self):
        state = self.__dict__.copy()
        del state["_w"]
        return state

    def __setstate__(self, state):
        super().__setstate__(state)
        self._keep(self._packed)


class _LinearFn(torch.autograd.Function):
    """y = x . W^T with a frozen W; the gradient reaches x, a tangent of x comes through."""

    @staticmethod
    def forward(ctx, x, mod):
        ctx.mod = mod
        return mod._product(x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        T.no_grad_here("The gradient of MXLinear", dy)
        return ctx.mod._dx(dy), None

    @staticmethod
    def jvp(ctx, dx, _mod):
        return ctx.mod._product(dx)


class MXLinear(_Packed):
    """Bias-free linear whose weight is MXFP4: codes uint8 [OUT, 16 B], scales uint8 [OUT, B]
    (the module keeps its own copy, in the kernels' operand order; state_dict holds the rows).
    in_features may be any width of the last block (default: all 32 of it). act: None multiplies x
    as it is (bf16, fp16 and fp32 enter exactly, but for bits under 2^-126; fp32 sums); "mxfp4"
    quantises x's rows as mx_quantize does. Differentiable in x with act None; the weight is
    frozen."""

    _rows = 2

    def __init__(self, codes, scales, in_features=None, act=None):
        super().__init__()
        if act not in (None, "mxfp4"):
            raise ValueError(f"act must be None or 'mxfp4', got {act!r}")
        if codes.ndim != 2:
            raise ValueError(f"codes must be [OUT, bytes], got {tuple(codes.shape)}")
        IN = int(scales.shape[-1]) * BLOCK if in_features is None else int(in_features)
        _check_mx(codes, scales, IN, "MXLinear")
        self.in_features, self.out_features, self.act = IN, int(codes.shape[0]), act
        self._set(codes, scales, 1, self.out_features, IN)

    @classmethod
    def from_weight(cls, weight, act=None):
        """The linear of a weight [OUT, IN], quantised here."""
        return cls(*mx_quantize(weight.detach()), weight.shape[1], act)

    input_dims = property(lambda self: self.in_features)
    output_dims = property(lambda self: self.out_features)

    def _product(self, x):
        IN, OUT = self.in_features, self.out_features
        act = L.VQK_MX_ACT_NONE if self.act is None else L.VQK_MX_ACT_MXFP4
        xt, lib, w = T.act_type(x), L.lib(), ctypes.byref(self._w)
        with T.on_device(x):
            xf = T.rows_of(x, IN)
            N = xf.shape[0]
            y = x.new_empty((*x.shape[:-1], OUT))
            size = _ws_bytes(self._sizes, (N, xt), lib.vqk_mx_linear_workspace, w, xt, N, act)
            work, wp = _work(x, size)
            rc = lib.vqk_mx_linear(w, xf.data_ptr(), xt, N, act, y.data_ptr(), xt, wp, size,
                                   T.raw_stream(x))
            if rc:
                L.check(rc, "MXLinear")
        return y

    def _dx(self, dy):
        IN, OUT = self.in_features, self.out_features
        dt, lib, w = T.act_type(dy), L.lib(), ctypes.byref(self._w)
        with T.on_device(dy):
            d = T.rows_of(dy, OUT)
            N = d.shape[0]
            dx = dy.new_empty((*dy.shape[:-1], IN))
            size = _ws_bytes(self._sizes, (N, dt, "dx"), lib.vqk_mx_linear_dx_workspace, w, dt, N)
            work, wp = _work(dy, size)
            L.check(lib.vqk_mx_linear_dx(w, d.data_ptr(), dt, N, dx.data_ptr(), dt, wp, size,
                                         T.raw_stream(dy)), "MXLinear gradient")
        return dx

    def forward(self, x):
        if x.device != self._packed[0].device:
            raise ValueError(f"MXLinear on {self._packed[0].device}, x on {x.device}")
        if x.ndim == 0 or x.shape[-1] != self.in_features:
            raise ValueError(f"MXLinear: x {tuple(x.shape)} for in_features {self.in_features}")
        if self.act is not None:
            T.no_grad_here("MXLinear(act='mxfp4')", x)
        elif (x.requires_grad and torch.is_grad_enabled()) or T.has_tangent(x):
            return _LinearFn.apply(x, self)
        return self._product(x)


class MXSwitchLinear(_Packed):
    """E bias-free linears in MXFP4, one picked by each index: codes uint8 [E, OUT, 16 B], scales
    uint8 [E, OUT, B]. forward(x [..., 1, 1, IN] or [..., k, 1, IN], indices [..., k]) ->
    [..., k, 1, OUT], as VQSwitchLinear; an index outside [0, E) gives zeros. Serving only: no
    gradient."""

    def __init__(self, codes, scales, in_features=None):
        super().__init__()
        if codes.ndim != 3:
            raise ValueError(f"codes must be [E, OUT, bytes], got {tuple(codes.shape)}")
        IN = int(scales.shape[-1]) * BLOCK if in_features is None else int(in_features)
        _check_mx(codes, scales, IN, "MXSwitchLinear")
        self.num_experts, self.output_dims, self.input_dims = int(codes.shape[0]), int(codes.shape[1]), IN
        self._set(codes, scales, self.num_experts, self.output_dims, IN)

    @classmethod
    def from_weight(cls, weight):
        """The experts of a weight [E, OUT, IN], quantised here."""
        return cls(*mx_quantize(weight.detach()), weight.shape[2])

    def forward(self, x, indices):
        T.require_cuda(x, indices, self._packed[0])
        T.no_grad_here("MXSwitchLinear", x)
        IN, OUT, k = self.input_dims, self.output_dims, int(indices.shape[-1])
        lead = tuple(indices.shape[:-1])
        if x.ndim < 3 or x.shape[-1] != IN or tuple(x.shape[:-3]) != lead or x.shape[-2] != 1 or \
                x.shape[-3] not in (1, k):
            raise ValueError(f"MXSwitchLinear: x {tuple(x.shape)} for indices {tuple(indices.shape)}, "
                             f"in_features {IN}")
        xt, lib, w = T.act_type(x), L.lib(), ctypes.byref(self._w)
        with T.on_device(x):
            xf = T.rows_of(x, IN)
            eidx = _ids32(indices.reshape(-1), self.num_experts)
            rows, N = xf.shape[0], eidx.numel()
            y = x.new_empty((*lead, k, 1, OUT))
            size = _ws_bytes(self._sizes, (rows, N, xt), lib.vqk_mx_switch_workspace, w, xt, rows, N)
            work, wp = _work(x, size)
            L.check(lib.vqk_mx_switch(w, xf.data_ptr(), xt, rows, eidx.data_ptr(), N,
                                      N // rows if rows else 1, y.data_ptr(), xt, wp, size,
                                      T.raw_stream(x)), "MXSwitchLinear")
        return y


class MXSwitchGLU(torch.nn.Module):
    """SwitchGLU with MXFP4 projections: forward(x [T, H], ids [T, k], weights [T, k]) ->
    sum_j weights_j * down_j(silu(gate_j(x)) * up_j(x)), [T, H]. Ids outside [0, E) add nothing.
    The SwiGLU rows are kept in 16 bits of bf16's range (24 for fp32 x). Serving only: no
    gradient."""

    def __init__(self, gate_proj: MXSwitchLinear, up_proj: MXSwitchLinear, down_proj: MXSwitchLinear):
        super().__init__()
        g, u, d = gate_proj, up_proj, down_proj
        if (g.num_experts, g.output_dims, g.input_dims) != (u.num_experts, u.output_dims, u.input_dims) or \
                (d.num_experts, d.output_dims, d.input_dims) != (g.num_experts, g.input_dims, g.output_dims):
            raise ValueError("MXSwitchGLU: gate, up [E, I, H] and down [E, H, I] do not fit together")
        self.gate_proj, self.up_proj, self.down_proj = g, u, d
        self._sizes = {}

    def _refs(self, *ts):
        """The projections' descriptors; they and the tensors ts are on one device."""
        m = self._modules
        g, u, d = m["gate_proj"], m["up_proj"], m["down_proj"]
        T.require_cuda(*ts, g._packed[0], u._packed[0], d._packed[0])
        return [ctypes.byref(p._w) for p in (g, u, d)]

    def forward(self, x, ids, weights):
        refs = self._refs(x, ids, weights)
        T.no_grad_here("MXSwitchGLU", x, weights)
        H = self.gate_proj.input_dims
        if x.ndim != 2 or x.shape[1] != H or ids.ndim != 2 or ids.shape[0] != x.shape[0] or \
                ids.shape != weights.shape:
            raise ValueError(f"MXSwitchGLU: x {tuple(x.shape)}, ids {tuple(ids.shape)}, weights "
                             f"{tuple(weights.shape)} for hidden size {H}")
        xt, lib, (n, k) = T.act_type(x), L.lib(), ids.shape
        with T.on_device(x):
            ids = _ids32(ids, self.gate_proj.num_experts)
            wts = weights.to(torch.float32).contiguous()
            x = x.contiguous()
            y = x.new_empty(x.shape)
            size = _ws_bytes(self._sizes, (n, k, xt), lib.vqk_mx_experts_workspace, *refs, xt, n, k)
            work, wp = _work(x, size)
            rc = lib.vqk_mx_experts(*refs, x.data_ptr(), xt, n, ids.data_ptr(), wts.data_ptr(), k,
                                    y.data_ptr(), xt, wp, size, T.raw_stream(x))
            if rc:
                L.check(rc, "MXSwitchGLU")
        return y


class MXSparseMoeBlock(torch.nn.Module):
    """Top-k routing and MXFP4 experts: forward(x [T, H], logits [T, E], mask [T]) ->
    [T, H]; without logits they are x . router_weight^T. mask: 0 marks padding, whose rows are
    zero and take no expert's time. form: keyword arguments of router.top_k beyond its softmax (score,
    bias, groups, top_groups, group_top, scale); the bias is a buffer, whose type casts of the module
    leave as it is."""

    form = {}

    def __init__(self, switch_mlp: MXSwitchGLU, top_k: int, norm_topk_prob: bool = True,
                 router_weight=None, **form):
        super().__init__()
        self.switch_mlp, self.top_k = switch_mlp, int(top_k)
        self.norm_topk_prob, self.router_weight = bool(norm_topk_prob), router_weight
        self._sizes = {}
        if form:
            router.form(switch_mlp.gate_proj.num_experts, self.top_k, **form)      # a ValueError where it does not fit
            self.register_buffer("bias", form.pop("bias", None))
            self.form = form

    def _apply(self, fn, recurse=True):
        bias = self._buffers.get("bias")
        if bias is None:
            return super()._apply(fn, recurse)
        self._buffers["bias"] = None
        try:
            super()._apply(fn, recurse)
            # as bytes, whose values casts keep: a rounded bias chooses other experts
            flat = bias.detach().contiguous().view(torch.uint8)
            moved = fn(flat)
            if moved is not flat:
                bias = moved.to(torch.uint8).view(bias.dtype)
        finally:
            self._buffers["bias"] = bias
        return self

    def forward(self, x, logits=None, mask=None):
        if logits is None:
            if self.router_weight is None:
                raise ValueError("MXSparseMoeBlock without a router_weight needs logits")
            logits = x.float() @ self.router_weight.float().T
        T.no_grad_here("MXSparseMoeBlock", x, logits)
        g = self.switch_mlp.gate_proj
        ws = self.switch_mlp._refs(x, logits, mask)
        if x.ndim != 2 or x.shape[1] != g.input_dims or logits.shape != (x.shape[0], g.num_experts):
            raise ValueError(f"MXSparseMoeBlock: x {tuple(x.shape)}, logits {tuple(logits.shape)} for "
                             f"{g.num_experts} experts of width {g.input_dims}")
        bias = self._buffers.get("bias")
        if self.form or bias is not None:
            return self.switch_mlp(x, *router.top_k(logits, self.top_k, self.norm_topk_prob, mask, bias=bias, **self.form))
        m = router.mask_bytes(mask, logits)
        xt, lib, k = T.act_type(x), L.lib(), self.top_k
        n = x.shape[0]
        with T.on_device(x):
            x = x.contiguous()
            lg, ld = router.rows(logits)
            y = x.new_empty(x.shape)
            size = _ws_bytes(self._sizes, (n, xt, k), lib.vqk_mx_moe_workspace, *ws, xt, n, k)
            work, wp = _work(x, size)
            rc = lib.vqk_mx_moe(*ws, x.data_ptr(), xt, n, lg.data_ptr(), T.act_type(lg), ld,
                                None if m is None else m.data_ptr(), k, int(self.norm_topk_prob),
                                y.data_ptr(), xt, wp, size, T.raw_stream(x))
            if rc:
                L.check(rc, "MXSparseMoeBlock")
        return y
