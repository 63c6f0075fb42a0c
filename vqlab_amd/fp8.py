"""8-bit floating point (e4m3) weights with block scales for PyTorch-ROCm, and the RMS norm whose
output is in 8 bits already. No counterpart in the reference, whose formats are vector-quantised:
this is what block-scaled 8-bit checkpoints hold.

A weight [OUT, IN] has codes (torch.float8_e4m3fn) and an fp32 scale for each 128 x 128 of it, rows of
activations one for each 128 of their columns; value = code * scale (include/vqk.h).

  f8_quantize(x) -> F8Rows(codes, scales)      f8_quantize_weight(w) -> codes, scales
  f8_dequantize(codes, scales, dtype)
  F8Linear(codes, scales, act)                 bias-free linear, like MXLinear
  rms_norm, rms_norm_f8                        with the residual's addition in front
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib as L
from . import _torch as T
from .mx import _work, _ws_bytes

BLOCK = 128
F8 = torch.float8_e4m3fn


class F8Rows(NamedTuple):
    """codes float8_e4m3fn [..., C] and scales fp32 [..., ceil(C / 128)] of rows in 8 bits (the scales
    of one block lie side by side in memory: a view of [blocks, rows])."""
    codes: torch.Tensor
    scales: torch.Tensor


def _blocks(n):
    return -(-int(n) // BLOCK)


def _rows_in(x, C):
    """x [..., C] as rows, their number and the elements between them."""
    if x.ndim == 2 and x.stride(1) == 1 and x.stride(0) >= C:
        return x, x.shape[0], x.stride(0)              # rows apart: read where they are
    x = x.contiguous()
    return x, x.numel() // C if C else 0, C


def _aligned(x):
    """x, or a copy of it, at an address that the products read from."""
    return x.clone() if x.data_ptr() & 15 else x


def _rows_out(like, lead, n, C):
    """Room for rows [*lead, C] in 8 bits."""
    codes = like.new_empty((*lead, C), dtype=F8)
    scales = torch.empty_strided((n, _blocks(C)), (1, n), dtype=torch.float32, device=like.device)
    return codes, scales, scales if len(lead) == 1 else scales.view(*lead, _blocks(C))


def f8_quantize(x):
    """Rows x [..., C] (fp16, bf16, fp32) in 8 bits. A block's scale is its largest magnitude / 448, at
    least 2^-126; a code is value * (1 / scale) rounded to nearest, ties to even. A block with an
    infinity or NaN becomes NaN. Not differentiable."""
    T.require_cuda(x)
    xt = T.act_type(x)
    if x.ndim == 0:
        raise ValueError("f8_quantize takes rows, got a scalar")
    T.no_grad_here("f8_quantize", x)
    C = x.shape[-1]
    with T.on_device(x):
        rows, n, ld = _rows_in(x, C)
        codes, scales, view = _rows_out(x, x.shape[:-1], n, C)
        L.check(L.lib().vqk_f8_quantize(rows.data_ptr(), xt, n, C, ld, codes.data_ptr(), scales.data_ptr(),
                                        1, n, T.raw_stream(x)), "f8_quantize")
    return F8Rows(codes, view)


def f8_quantize_weight(w):
    """Codes float8_e4m3fn [OUT, IN] and scales fp32 [ceil(OUT / 128), ceil(IN / 128)] of a weight (fp16,
    bf16, fp32), quantised as f8_quantize does over blocks of 128 x 128."""
    T.require_cuda(w)
    wt = T.act_type(w)
    if w.ndim != 2:
        raise ValueError(f"f8_quantize_weight takes [OUT, IN], got {tuple(w.shape)}")
    T.no_grad_here("f8_quantize_weight", w)
    O, I = w.shape
    with T.on_device(w):
        rows, _, ld = _rows_in(w, I)
        codes = torch.empty((O, I), dtype=F8, device=w.device)
        scales = torch.empty((_blocks(O), _blocks(I)), dtype=torch.float32, device=w.device)
        L.check(L.lib().vqk_f8_quantize_weight(rows.data_ptr(), wt, O, I, ld, codes.data_ptr(),
                                               scales.data_ptr(), T.raw_stream(w)), "f8_quantize_weight")
    return codes, scales


def _codes(codes, what):
    if codes.dtype not in (F8, torch.uint8):
        raise ValueError(f"{what}: codes must be float8_e4m3fn (or its bytes as uint8), got {codes.dtype}")
    return codes


def _strided(codes, scales, C, what):
    """Rows in 8 bits as the library reads them: codes, their stride, scales [n, blocks] and their
    strides, the number of rows."""
    _codes(codes, what)
    if scales.dtype != torch.float32:
        raise ValueError(f"{what}: scales must be float32, got {scales.dtype}")
    if codes.ndim == 0 or codes.shape[-1] != C or scales.shape != (*codes.shape[:-1], _blocks(C)):
        raise ValueError(f"{what}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not rows "
                         f"of {C} with a scale for each {BLOCK}")
    codes, n, ldc = _rows_in(codes, C)
    if scales.ndim != 2:
        scales = scales.reshape(n, _blocks(C))         # a view where the strides allow it
    if n == 1:                                         # one row: its stride says nothing
        return codes, ldc, scales, 0, scales.stride(1), n
    return codes, ldc, scales, scales.stride(0), scales.stride(1), n


def f8_dequantize(codes, scales, dtype=torch.bfloat16):
    """The values of rows in 8 bits (scales [..., ceil(C / 128)]), or of a weight (scales [ceil(OUT / 128),
    ceil(IN / 128)], where that is not the shape of rows), in dtype: code * scale in fp32, rounded once.
    Not differentiable."""
    T.require_cuda(codes, scales)
    if dtype not in T.ACT_TYPES:
        raise ValueError(f"dtype must be float16, bfloat16 or float32, got {dtype}")
    if codes.ndim == 0:
        raise ValueError("f8_dequantize takes rows, got a scalar")
    T.no_grad_here("f8_dequantize", scales)
    C = codes.shape[-1]
    per = 1
    with T.on_device(codes):
        if codes.ndim == 2 and scales.ndim == 2 and scales.shape != (codes.shape[0], _blocks(C)) and \
                scales.shape == (_blocks(codes.shape[0]), _blocks(C)):
            if scales.dtype != torch.float32:
                raise ValueError(f"f8_dequantize: scales must be float32, got {scales.dtype}")
            per = BLOCK
            rows, n, ldc = _rows_in(_codes(codes, "f8_dequantize"), C)
            so, sk, sc = scales.stride(0), scales.stride(1), scales
        else:
            rows, ldc, sc, so, sk, n = _strided(codes, scales, C, "f8_dequantize")
        out = codes.new_empty(codes.shape, dtype=dtype)
        rc = L.lib().vqk_f8_dequantize(rows.data_ptr(), ldc, sc.data_ptr(), so, sk, per, n, C, out.data_ptr(),
                                       T.ACT_TYPES[dtype], T.raw_stream(codes))
        if rc:
            L.check(rc, "f8_dequantize")
    return out


class _LinearFn(torch.autograd.Function):
    """y = x . W^T with a frozen W; the gradient reaches x, a tangent of x comes through."""

    @staticmethod
    def forward(ctx, x, mod, out_dtype):
        ctx.mod, ctx.dtypes = mod, (x.dtype, out_dtype)
        return mod._product(x, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        T.no_grad_here("The gradient of F8Linear", dy)
        return ctx.mod._dx(dy, ctx.dtypes[0]), None, None

    @staticmethod
    def jvp(ctx, dx, _mod, _dtype):
        return ctx.mod._product(dx, ctx.dtypes[1])


class F8Linear(torch.nn.Module):
    """Bias-free linear whose weight is in 8 bits: codes float8_e4m3fn (or uint8) [OUT, IN], scales fp32
    [ceil(OUT / 128), ceil(IN / 128)] (the module keeps its own copy, in the kernels' operand order;
    state_dict holds the rows). act: None multiplies x as it is (every finite bf16, fp16 and fp32 value
    enters exactly, but for bits under 2^-110; fp32 sums); "fp8" quantises x's rows as f8_quantize does.
    With act "fp8" x may also be F8Rows, as f8_quantize and rms_norm_f8 make them. The output has x's
    type, of F8Rows bfloat16, or out_dtype; into float32 products of 8-bit x are exact, into 16 bits they
    keep about 14 bits (include/vqk.h). Differentiable in x with act None; the weight is frozen."""

    def __init__(self, codes, scales, act=None):
        super().__init__()
        if act not in (None, "fp8"):
            raise ValueError(f"act must be None or 'fp8', got {act!r}")
        if codes.ndim != 2 or 0 in codes.shape:
            raise ValueError(f"codes must be [OUT, IN], got {tuple(codes.shape)}")
        self.out_features, self.in_features, self.act = int(codes.shape[0]), int(codes.shape[1]), act
        self._sizes = {}
        self._keep(*self._pack(codes, scales))

    @classmethod
    def from_weight(cls, weight, act=None):
        """The linear of a weight [OUT, IN], quantised here."""
        return cls(*f8_quantize_weight(weight.detach()), act)

    input_dims = property(lambda self: self.in_features)
    output_dims = property(lambda self: self.out_features)

    def _scale_shape(self):
        return _blocks(self.out_features), _blocks(self.in_features)

    def _pack(self, codes, scales):
        T.require_cuda(codes, scales)
        _codes(codes, "F8Linear")
        if scales.dtype != torch.float32 or scales.shape != self._scale_shape():
            raise ValueError(f"F8Linear: scales must be float32 {self._scale_shape()}, got {scales.dtype} "
                             f"{tuple(scales.shape)}")
        O, I = self.out_features, self.in_features
        size = ctypes.c_size_t()
        L.check(L.lib().vqk_f8_pack_bytes(O, I, ctypes.byref(size)), "F8Linear")
        with T.on_device(codes):
            codes = codes.detach().contiguous()
            packed = torch.empty(size.value, dtype=torch.uint8, device=codes.device)
            L.check(L.lib().vqk_f8_pack(codes.data_ptr(), O, I, packed.data_ptr(), T.raw_stream(codes)), "F8Linear")
            return packed, scales.detach().clone(memory_format=torch.contiguous_format)

    def _keep(self, packed, scales):
        self._packed = (packed, scales)
        self._w = ctypes.byref(L.VQKF8Weights(packed.data_ptr(), scales.data_ptr(), self.out_features, self.in_features))

    @property
    def codes(self):
        """Codes float8_e4m3fn [OUT, IN], unpacked by each access."""
        O, I = self.out_features, self.in_features
        packed = self._packed[0]
        rows = packed.view(-(-O // 16), _blocks(I), 2, 4, 16, 16).permute(0, 4, 1, 3, 2, 5)
        return rows.reshape(-(-O // 16) * 16, -1)[:O, :I].contiguous().view(F8)

    @property
    def scales(self):
        """Scales fp32 [ceil(OUT / 128), ceil(IN / 128)], a copy by each access."""
        return self._packed[1].clone()

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
        codes, scales = (state_dict[n] for n in names)
        if codes.shape != (self.out_features, self.in_features) or codes.dtype not in (F8, torch.uint8) or \
                scales.shape != self._scale_shape() or scales.dtype != torch.float32:
            error_msgs.append(f"{names[0]}: {codes.dtype} {tuple(codes.shape)} with scales {scales.dtype} "
                              f"{tuple(scales.shape)}, the module holds float8_e4m3fn "
                              f"{(self.out_features, self.in_features)} with float32 {self._scale_shape()}")
            return
        here = self._packed[0].device
        at = here if here.type == "cuda" else "cuda"       # packed by a GPU, kept where the module is
        for old, new in zip(self._packed, self._pack(codes.to(at), scales.to(at))):
            old.copy_(new)                                 # in place: captured graphs read these

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        packed, scales = self._packed
        # as bytes, whose values casts keep (type() casts integers too)
        self._keep(fn(packed).to(torch.uint8), fn(scales.view(torch.uint8)).to(torch.uint8).view(torch.float32))
        return self

    def __getstate__(self):
        state = self.__dict__.copy()
        del state["_w"]
        return state

    def __setstate__(self, state):
        super().__setstate__(state)
        self._keep(*self._packed)

    def _product(self, x, out_dtype):
        IN, OUT = self.in_features, self.out_features
        act = L.VQK_F8_ACT_NONE if self.act is None else L.VQK_F8_ACT_F8
        xt, yt, lib, w = T.act_type(x), T.ACT_TYPES[out_dtype], L.lib(), self._w
        with T.on_device(x):
            xf = _aligned(T.rows_of(x, IN))
            N = xf.shape[0]
            y = x.new_empty((*x.shape[:-1], OUT), dtype=out_dtype)
            size = _ws_bytes(self._sizes, (N, xt, yt), lib.vqk_f8_linear_workspace, w, xt, N, act, yt)
            work, wp = _work(x, size)
            rc = lib.vqk_f8_linear(w, xf.data_ptr(), xt, N, act, y.data_ptr(), yt, wp, size, T.raw_stream(x))
            if rc:
                L.check(rc, "F8Linear")
        return y

    def _rows_product(self, rows, out_dtype):
        lib, w = L.lib(), self._w
        with T.on_device(rows.codes):
            codes, ldc, scales, sn, sk, N = _strided(*rows, self.in_features, "F8Linear")
            if codes.data_ptr() & 15:
                codes, ldc = codes.clone(memory_format=torch.contiguous_format), self.in_features
            y = scales.new_empty((*rows.codes.shape[:-1], self.out_features), dtype=out_dtype)
            yt = T.ACT_TYPES[out_dtype]
            size = _ws_bytes(self._sizes, (N, ldc, yt, "rows"), lib.vqk_f8_linear_rows_workspace, w, ldc, N, yt)
            work, wp = _work(codes, size)
            rc = lib.vqk_f8_linear_rows(w, codes.data_ptr(), ldc, scales.data_ptr(), sn, sk, N, y.data_ptr(),
                                        yt, wp, size, T.raw_stream(codes))
            if rc:
                L.check(rc, "F8Linear")
        return y

    def _dx(self, dy, dtype):
        IN, OUT = self.in_features, self.out_features
        dt, lib, w = T.act_type(dy), L.lib(), self._w
        with T.on_device(dy):
            d = _aligned(T.rows_of(dy, OUT))
            N = d.shape[0]
            dx = torch.empty((*dy.shape[:-1], IN), dtype=dtype, device=dy.device)
            size = _ws_bytes(self._sizes, (N, dt, "dx"), lib.vqk_f8_linear_dx_workspace, w, dt, N)
            work, wp = _work(dy, size)
            L.check(lib.vqk_f8_linear_dx(w, d.data_ptr(), dt, N, dx.data_ptr(), T.ACT_TYPES[dtype], wp, size,
                                         T.raw_stream(dy)), "F8Linear gradient")
        return dx

    def forward(self, x, out_dtype=None):
        if out_dtype is not None and out_dtype not in T.ACT_TYPES:
            raise ValueError(f"out_dtype must be float16, bfloat16 or float32, got {out_dtype}")
        if isinstance(x, tuple):
            if self.act is None:
                raise ValueError("F8Linear takes rows in 8 bits with act='fp8' only")
            rows = F8Rows(*x)
            T.require_cuda(*rows, self._packed[0])
            T.no_grad_here("F8Linear of rows in 8 bits", rows.scales)
            return self._rows_product(rows, out_dtype or torch.bfloat16)
        if x.device != self._packed[0].device:
            raise ValueError(f"F8Linear on {self._packed[0].device}, x on {x.device}")
        if x.ndim == 0 or x.shape[-1] != self.in_features:
            raise ValueError(f"F8Linear: x {tuple(x.shape)} for in_features {self.in_features}")
        T.act_type(x)
        out_dtype = out_dtype or x.dtype
        if self.act is not None:
            T.no_grad_here("F8Linear(act='fp8')", x)
        elif (x.requires_grad and torch.is_grad_enabled()) or T.has_tangent(x):
            return _LinearFn.apply(x, self, out_dtype)
        return self._product(x, out_dtype)


# ------------------------------------------------------------------ norm
def _check_norm(x, weight, eps, residual, what):
    T.require_cuda(x, weight, residual)
    T.act_type(x), T.act_type(weight)
    if x.ndim == 0 or x.shape[-1] == 0 or weight.shape != x.shape[-1:]:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} for x {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{what}: residual {residual.dtype} {tuple(residual.shape)} for x {x.dtype} {tuple(x.shape)}")
    if not eps >= 0:
        raise ValueError(f"{what}: eps={eps}")


def _norm(x, weight, eps, residual, f8, want_r):
    """h (None without a residual), r or None, and y or F8Rows."""
    C = x.shape[-1]
    with T.on_device(x):
        rows, n, ld = _rows_in(x, C)
        res, _, ldr = _rows_in(residual, C) if residual is not None else (None, 0, C)
        w = weight.contiguous()
        h = None if residual is None else x.new_empty(x.shape)
        r = x.new_empty(n, dtype=torch.float32) if want_r else None
        y = codes = scales = None
        if f8:
            codes, scales, view = _rows_out(x, x.shape[:-1], n, C)
        else:
            y = x.new_empty(x.shape)
        at = [None if t is None else t.data_ptr() for t in (res, h, y, r, codes, scales)]
        rc = L.lib().vqk_rms_norm(rows.data_ptr(), T.act_type(x), n, C, ld, at[0], ldr, w.data_ptr(), T.act_type(w),
                                  float(eps), at[1], at[2], at[3], at[4], at[5], 1, n, T.raw_stream(x))
        if rc:
            L.check(rc, "rms_norm")
    return h, r, F8Rows(codes, view) if f8 else y


_norm_sizes = {}                                # (rows, columns) -> workspace bytes


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        h, r, y = _norm(x, weight, eps, residual, False, True)
        ctx.save_for_backward(x if h is None else h, weight, r)
        ctx.has_res = h is not None
        ctx.set_materialize_grads(False)
        return (y, h) if ctx.has_res else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, r = ctx.saved_tensors
        for g in (dy, dh):
            if g is not None:
                T.no_grad_here("The gradient of rms_norm", g)
        if dy is None:                                 # through h alone
            return dh, None, dh if ctx.has_res else None, None
        C = h.shape[-1]
        lib = L.lib()
        with T.on_device(h):
            rows, n, ld = _rows_in(h, C)
            w, dy = weight.contiguous(), dy.contiguous()
            dh = None if dh is None else dh.contiguous()
            dx, dw = h.new_empty(h.shape), w.new_empty(C)
            size = _ws_bytes(_norm_sizes, (n, C), lib.vqk_rms_norm_backward_workspace, n, C)
            work, wp = _work(h, size)
            rc = lib.vqk_rms_norm_backward(rows.data_ptr(), T.act_type(h), n, C, ld, w.data_ptr(), T.act_type(w),
                                           r.data_ptr(), dy.data_ptr(), None if dh is None else dh.data_ptr(),
                                           dx.data_ptr(), dw.data_ptr(), wp, size, T.raw_stream(h))
            if rc:
                L.check(rc, "rms_norm gradient")
        return dx, dw, dx if ctx.has_res else None, None


def rms_norm(x, weight, eps=1e-6, residual=None):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension of x [..., C] (fp16, bf16, fp32; C at
    most 16384), h = x + residual rounded once to their type; with a residual y, h, otherwise y. eps 0 is
    for rows of a root mean square of 2^-128 and more. Differentiable in x, residual and weight."""
    _check_norm(x, weight, eps, residual, "rms_norm")
    ts = (x, weight) if residual is None else (x, weight, residual)
    for t in ts:
        if T.has_tangent(t):
            raise RuntimeError("rms_norm has no forward-mode derivative")
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        return _NormFn.apply(x, weight, residual, eps)
    h, _, y = _norm(x, weight, eps, residual, False, False)
    return y if residual is None else (y, h)


def rms_norm_f8(x, weight, eps=1e-6, residual=None):
    """The same with y in 8 bits, as f8_quantize makes them of the fp32 y: F8Rows, or F8Rows and h. For
    F8Linear(act="fp8"). Not differentiable."""
    _check_norm(x, weight, eps, residual, "rms_norm_f8")
    T.no_grad_here("rms_norm_f8", *(t for t in (x, weight, residual) if t is not None))
    h, _, rows = _norm(x, weight, eps, residual, True, False)
    return rows if residual is None else (rows, h)
