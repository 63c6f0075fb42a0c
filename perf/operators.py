"""Microscaled 4-bit weights and the router of a mixture of experts, as cases that can be timed.

Four kinds of operator:

  quant    rows to MXFP4 (blocks of 32 along the row: one power-of-two scale, 4-bit elements) and
           back to the values they stand for
  linear   y = x . W^T with W in MXFP4; x as it comes, or itself quantised to MXFP4 ("a4"); with
           "train" the gradient of x as well
  experts  one block of experts in MXFP4: softmax top-k routing, SwiGLU of the routed experts,
           weighted sum
  route    that routing by itself, for training: expert ids and weights, tokens per expert, the
           balance and z losses, and the gradient of the logits

A block of 32 values has the scale 2^e, e = floor(log2(largest magnitude)) - 2 (at least -127),
stored as e + 127; an element is its value / 2^e rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3,
4, 6 (ties to the even code, larger values to 6) under its sign. Weights are N(0, 1 / columns),
quantised so; activations and router logits are N(0, 1).
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token's activations, quantised before a product: launch latency
        dict(name="quant_row_4096", kind="quant", rows=1, cols=4096, dtype="bf16"),
        # an MLP weight quantised when a checkpoint is written
        dict(name="quant_weight_17408", kind="quant", rows=17408, cols=5120, dtype="bf16"),
        # one token through an attention-sized projection
        dict(name="linear_decode_4096", kind="linear", rows=1, inp=4096, out=4096, a4=False, train=False,
             dtype="bf16"),
        # twenty sequences decoded together through an MLP gate
        dict(name="linear_decode_20_rows", kind="linear", rows=20, inp=5120, out=17408, a4=False,
             train=False, dtype="bf16"),
        # a short prompt of odd length through an MLP down projection
        dict(name="linear_prompt_333", kind="linear", rows=333, inp=17408, out=5120, a4=False,
             train=False, dtype="fp16"),
        # a long prompt (or one chunk of it) through an MLP gate, both sides in 4 bits
        dict(name="linear_prompt_2048_a4", kind="linear", rows=2048, inp=5120, out=17408, a4=True,
             train=False, dtype="bf16"),
        # a training step through a frozen MLP down projection: its output and the gradient of x
        dict(name="linear_train_2048", kind="linear", rows=2048, inp=17408, out=5120, a4=False,
             train=True, dtype="bf16"),
        # one token through a layer of 256 small experts: the inner loop of decoding
        dict(name="experts_decode_e256", kind="experts", tokens=1, hidden=2048, inter=512, experts=256,
             top_k=8, pad=0.0, dtype="bf16"),
        # a verify batch of speculative decoding through 512 larger experts, one or two pairs each
        dict(name="experts_verify_e512_64", kind="experts", tokens=64, hidden=4096, inter=1024,
             experts=512, top_k=10, pad=0.0, dtype="bf16"),
        # a padded batch of prompts through the layer of small experts: 60 pairs or so for each
        dict(name="experts_prompt_e256_2048", kind="experts", tokens=2048, hidden=2048, inter=512,
             experts=256, top_k=8, pad=0.07, dtype="bf16"),
        # the router in a training step over 32 sequences
        dict(name="route_65536_e256", kind="route", tokens=65536, experts=256, top_k=8, norm=True,
             pad=0.0, dtype="fp32"),
        # a small padded batch over more experts, logits straight from a 16-bit product
        dict(name="route_509_e512", kind="route", tokens=509, experts=512, top_k=10, norm=True,
             pad=0.2, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng, lo, hi):
    """A model dimension: mostly a multiple of 256, else of the block, now and then neither."""
    step = rng.choice([256, 256, 256, BLOCK, BLOCK, 1])
    return max(BLOCK, int(_log_int(rng, lo, hi) / step + 0.5) * step)


def _draw_quant(rng):
    return dict(kind="quant", rows=_log_int(rng, 1, 17408), cols=_dim(rng, 64, 5120),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _draw_linear(rng):
    inp, out = _dim(rng, 512, 17408), _dim(rng, 512, 17408)
    rows = rng.choice([_log_int(rng, 1, 64), _log_int(rng, 65, 2048)])
    a4 = rng.random() < 0.4
    train = not a4 and rng.random() < 0.35
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    rows = max(1, min(rows, 2048 * 5120 * 17408 // (inp * out)))
    return dict(kind="linear", rows=rows, inp=inp, out=out, a4=a4, train=train, dtype=dtype)


def _draw_experts(rng):
    experts = rng.choice([8, 60, 64, 96, 128, 160, 256, 384, 512])
    top_k = min(experts, rng.choice([1, 2, 4, 6, 8, 10]))
    hidden, inter = BLOCK * _log_int(rng, 16, 128), BLOCK * _log_int(rng, 8, 32)
    tokens = rng.choice([_log_int(rng, 1, 8), _log_int(rng, 9, 128), _log_int(rng, 129, 2048)])
    cap = 2048 * 8 * 2048 * 512 // (top_k * hidden * inter)       # the largest listed layer's work
    return dict(kind="experts", tokens=max(1, min(tokens, cap)), hidden=hidden, inter=inter,
                experts=experts, top_k=top_k, pad=rng.choice([0.0, 0.0, 0.3]),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _draw_route(rng):
    experts = rng.choice([8, 60, 64, 128, 160, 256, 384, 512])
    tokens = _log_int(rng, 1, 65536 * 256 // max(256, experts))
    return dict(kind="route", tokens=tokens, experts=experts,
                top_k=min(experts, rng.choice([1, 2, 4, 6, 8, 10])), norm=rng.random() < 0.7,
                pad=rng.choice([0.0, 0.0, 0.25]), dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))


def draw(rng):
    return rng.choice([_draw_quant, _draw_linear, _draw_linear, _draw_experts, _draw_experts,
                       _draw_route])(rng)


# ------------------------------------------------------------ plain forms
_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _table(device, dtype):
    return torch.tensor(_VALUES + [-v for v in _VALUES], dtype=dtype, device=device)


def _quantize(x):
    """Rows [..., C] -> packed codes uint8 [..., B * 16] (the earlier element in the low four bits)
    and scales uint8 [..., B], B = ceil(C / 32)."""
    x = x.float()
    pad = -x.shape[-1] % BLOCK
    if pad:
        x = torch.nn.functional.pad(x, (0, pad))
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax).exponent - 3                  # floor(log2(amax)) - 2
    e = torch.where(amax > 0, e, -127).clamp(min=-127)
    half = e // 2
    a = torch.ldexp(torch.ldexp(b.abs(), -half), half - e)      # 2^127 and more in two steps
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, t in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (a > t if i % 2 == 0 else a >= t)       # a tie goes to the even one of two codes
    code += (torch.signbit(b)).to(torch.uint8) * 8
    code = code.reshape(*x.shape[:-1], -1, 2)
    return code[..., 0] + code[..., 1] * 16, (e + 127).to(torch.uint8).squeeze(-1)


def _values(codes, scales, cols, dtype=torch.float32):
    """The values that packed codes and scales stand for, [..., cols]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    v = _table(codes.device, dtype)[c]
    s = torch.ldexp(torch.ones((), dtype=dtype, device=codes.device), scales.int() - 127)
    v = v.reshape(*scales.shape, BLOCK) * s[..., None]
    return v.flatten(-2)[..., :cols]


def _plain_quant(s):
    codes, scales = _quantize(s["x"])
    return _values(codes, scales, s["x"].shape[-1]).to(s["x"].dtype)


def _plain_linear(s):
    case, x = s["case"], s["x"].float()
    if case["a4"]:
        x = _values(*_quantize(x), case["inp"])
    w = _values(s["codes"], s["scales"], case["inp"])
    y = (x @ w.T).to(s["x"].dtype)
    if not case["train"]:
        return y
    return y, (s["dy"].float() @ w).to(s["x"].dtype)


def _plain_route(s, grads=True):
    """Ids, weights, counts, balance, z and the gradient of the logits, or the first two."""
    case = s["case"]
    E, k = case["experts"], case["top_k"]
    logits = s["logits"].detach().float()
    keep = s["mask"] if s["mask"] is not None else torch.ones_like(logits[:, 0], dtype=torch.bool)
    m = logits.max(-1, keepdim=True).values
    ex = torch.exp(logits - m)
    total = ex.sum(-1, keepdim=True)
    p = ex / total
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    sel = p.gather(1, order)
    norm = case.get("norm", True)
    w = sel / sel.sum(-1, keepdim=True) if norm else sel
    ids = torch.where(keep[:, None], order, -1).int()
    w = torch.where(keep[:, None], w, 0.0)
    if not grads:
        return ids, w
    n = keep.sum().clamp(min=1).double()
    counts = torch.zeros(E + 1, dtype=torch.int32, device=p.device)
    counts.index_add_(0, torch.where(keep[:, None], order, E).flatten(),
                      torch.ones(order.numel(), dtype=torch.int32, device=p.device))
    counts = counts[:E]
    kp = keep[:, None].double()
    lse = (m + torch.log(total)).double()
    P = (p.double() * kp).sum(0) / n
    c = counts.double()
    balance = (E * (c / (n * k) * P).sum()).float()
    z = ((lse * lse * kp).sum() / n).float()
    # the gradient: of the balance and z losses, then of the weights
    gb, gz = s["gb"].double(), s["gz"].double()
    pd = p.double()
    f = gb * E / (n * n * k) * c
    d = pd * (f - (pd * f).sum(-1, keepdim=True)) + gz * 2 / n * lse * pd
    dw = s["dw"].double()
    if norm:
        wd = w.double()
        d.scatter_add_(1, order, wd * (dw - (wd * dw).sum(-1, keepdim=True)))
    else:
        sd = sel.double()
        d.scatter_add_(1, order, sd * dw)
        d -= pd * (sd * dw).sum(-1, keepdim=True)
    d = torch.where(keep[:, None], d, 0.0)
    return ids, w, counts, balance, z, d.to(s["logits"].dtype)


def _plain_experts(s):
    case = s["case"]
    T, E, k, H, I = (case[n] for n in ("tokens", "experts", "top_k", "hidden", "inter"))
    ids, w = _plain_route(s, grads=False)
    x = s["x"].float()
    y = torch.zeros_like(x)

    def weight(name, e, cols):
        codes, scales = s["w"][name]
        return _values(codes[e], scales[e], cols)

    if T * k < E:                                       # a weight for each pair
        for j in range(k):
            for t in range(T):
                e = ids[t, j].clamp(min=0).long()[None]         # on the GPU: no look at its value
                g = x[t:t + 1] @ weight("gate", e, H)[0].T
                u = x[t:t + 1] @ weight("up", e, H)[0].T
                y[t] += w[t, j] * ((g * torch.sigmoid(g) * u) @ weight("down", e, I)[0].T)[0]
    else:                                               # every expert over all tokens
        for e in range(E):
            g, u = x @ weight("gate", e, H).T, x @ weight("up", e, H).T
            we = torch.where(ids == e, w, 0.0).sum(-1, keepdim=True)
            y += we * ((g * torch.sigmoid(g) * u) @ weight("down", e, I).T)
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(0x3B5D + 7907 * int(seed))


def _weight(g, out, inp):
    """Packed codes and scales of a weight ~ N(0, 1 / inp), made in slices of rows."""
    nb = -(-inp // BLOCK)
    codes = torch.empty(out, nb * 16, dtype=torch.uint8, device="cuda")
    scales = torch.empty(out, nb, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // inp)
    for r in range(0, out, step):
        n = min(step, out - r)
        codes[r:r + n], scales[r:r + n] = _quantize(
            torch.randn(n, inp, device="cuda", generator=g) / math.sqrt(inp))
    return codes, scales


def _experts(g, E, out, inp):
    codes, scales = _weight(g, E * out, inp)
    return codes.reshape(E, out, -1), scales.reshape(E, out, -1)


def _mask(g, case):
    if not case["pad"]:
        return None
    return torch.rand(case["tokens"], device="cuda", generator=g) >= case["pad"]


def _inputs(case, seed):
    """Every tensor of the case, from the seed alone."""
    g, kind = _gen(seed), case["kind"]
    dt = DTYPES[case["dtype"]]

    def acts(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dt)

    if kind == "quant":
        return dict(x=acts(case["rows"], case["cols"]))
    if kind == "linear":
        codes, scales = _weight(g, case["out"], case["inp"])
        s = dict(codes=codes, scales=scales, x=acts(case["rows"], case["inp"]))
        if case["train"]:
            s["dy"] = acts(case["rows"], case["out"])
        return s
    if kind == "experts":
        E, H, I = case["experts"], case["hidden"], case["inter"]
        return dict(w={"gate": _experts(g, E, I, H), "up": _experts(g, E, I, H),
                       "down": _experts(g, E, H, I)},
                    x=acts(case["tokens"], H), mask=_mask(g, case),
                    logits=torch.randn(case["tokens"], E, device="cuda", generator=g))
    return dict(logits=acts(case["tokens"], case["experts"]), mask=_mask(g, case),
                # of a loss summed over the tokens
                dw=torch.randn(case["tokens"], case["top_k"], device="cuda", generator=g),
                gb=torch.tensor(0.01 * case["tokens"], device="cuda"),
                gz=torch.tensor(0.001 * case["tokens"], device="cuda"))


# -------------------------------------------------------------- one pass
def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if not own:
        return s
    from vqlab_amd import mx
    if case["kind"] == "linear":
        s["module"] = mx.MXLinear(s.pop("codes"), s.pop("scales"), case["inp"],
                                  act="mxfp4" if case["a4"] else None)
        s["x"].requires_grad_(case["train"])
    elif case["kind"] == "experts":
        w, H, I = s.pop("w"), case["hidden"], case["inter"]
        glu = mx.MXSwitchGLU(mx.MXSwitchLinear(*w["gate"], H), mx.MXSwitchLinear(*w["up"], H),
                             mx.MXSwitchLinear(*w["down"], I))
        s["module"] = mx.MXSparseMoeBlock(glu, top_k=case["top_k"], norm_topk_prob=True)
    elif case["kind"] == "route":
        s["logits"].requires_grad_(True)
    return s


def run(state):
    case = state["case"]
    if not own:
        plain = dict(quant=_plain_quant, linear=_plain_linear, experts=_plain_experts,
                     route=_plain_route)[case["kind"]]
        with torch.no_grad():
            return plain(state)
    from vqlab_amd import mx, router
    if case["kind"] == "quant":
        codes, scales = mx.mx_quantize(state["x"])
        return mx.mx_dequantize(codes, scales, case["cols"], state["x"].dtype)
    if case["kind"] == "linear":
        y = state["module"](state["x"])
        if not case["train"]:
            return y
        return y.detach(), torch.autograd.grad(y, state["x"], state["dy"])[0]
    if case["kind"] == "experts":
        return state["module"](state["x"], state["logits"], mask=state["mask"])
    r = router.route(state["logits"], case["top_k"], norm_topk_prob=case["norm"], mask=state["mask"])
    d = torch.autograd.grad((r.weights, r.balance, r.z), state["logits"],
                            (state["dw"], state["gb"], state["gz"]))[0]
    return r.ids, r.weights.detach(), r.counts, r.balance.detach(), r.z.detach(), d


# ------------------------------------------------------------------ work
def _mx_bytes(rows, cols):
    return rows * -(-cols // BLOCK) * 17


def work(case):
    kind, act = case["kind"], 4 if case["dtype"] == "fp32" else 2
    if kind == "quant":
        r, c = case["rows"], case["cols"]
        # in, codes and scales out; codes and scales in, values out
        return dict(bytes=2 * r * c * act + 2 * _mx_bytes(r, c), flops=4 * r * c)
    if kind == "linear":
        r, i, o = case["rows"], case["inp"], case["out"]
        n = 2 if case["train"] else 1
        return dict(bytes=_mx_bytes(o, i) + n * r * (i + o) * act, flops=2 * n * r * i * o)
    if kind == "experts":
        T, H, I, E, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "top_k"))
        live = T * (1 - case["pad"])
        touched = E * (1 - (1 - k / E) ** live)                 # expected, of uniform routing
        return dict(bytes=int(touched * (2 * _mx_bytes(I, H) + _mx_bytes(H, I)) + 2 * T * H * act
                              + T * E * 4), flops=int(6 * live * k * H * I))
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    # logits in, ids and weights out; logits, ids, weights and their gradient in, gradient out
    return dict(bytes=3 * T * E * act + 5 * T * k * 4 + E * 4, flops=20 * T * E)


# --------------------------------------------------------- 64-bit results
def _exact_round(x):
    """x in 64 bits, each block of 32 rounded to the grid of its scale."""
    x = x.double()
    C = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -C % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    log = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    log = torch.where(torch.exp2(log) > top, log - 1, log)
    log = torch.where(torch.exp2(log + 1) <= top, log + 1, log)
    scale = torch.exp2((log - 2).clamp(min=-127))
    a = (b / scale).abs()
    # the spacing of the grid at a: 0.5 up to 2, then 1, then 2; round() takes ties to even
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.copysign(q, b) * scale).flatten(-2)[..., :C]


def _exact_weight(codes, scales, cols):
    lo, hi = (codes % 16).long(), (codes // 16).long()
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.long, device=codes.device)
    c[..., 0::2], c[..., 1::2] = lo, hi
    mag, sign = c % 8, 1 - 2 * (c // 8).double()
    exp, frac = mag // 2, (mag % 2).double()
    v = torch.where(exp == 0, frac * 0.5, (1 + frac / 2) * torch.exp2(exp.double() - 1)) * sign
    s = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)
    return (v * s)[..., :cols]


def _exact_route(case, s):
    E, k = case["experts"], case["top_k"]
    l = s["logits"].double()
    keep = s["mask"] if s["mask"] is not None else torch.ones(l.shape[0], dtype=torch.bool, device=l.device)
    ids = torch.argsort(-l, dim=-1, stable=True)[:, :k]
    return l, keep, ids


@torch.no_grad()
def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "quant":
        return _exact_round(s["x"])
    if kind == "linear":
        x = _exact_round(s["x"]) if case["a4"] else s["x"].double()
        y = torch.empty(case["rows"], case["out"], dtype=torch.float64, device="cuda")
        dx = torch.zeros(case["rows"], case["inp"], dtype=torch.float64, device="cuda")
        for r in range(0, case["out"], 1024):
            w = _exact_weight(s["codes"][r:r + 1024], s["scales"][r:r + 1024], case["inp"])
            y[:, r:r + 1024] = x @ w.T
            if case["train"]:
                dx += s["dy"][:, r:r + 1024].double() @ w
        return (y, dx) if case["train"] else y
    if kind == "experts":
        l, keep, ids = _exact_route(case, s)
        sel = torch.softmax(l.gather(1, ids), -1)               # renormalised over the chosen
        x = s["x"].double()
        y = torch.zeros_like(x)
        H, I = case["hidden"], case["inter"]
        for e in ids[keep].unique().tolist():
            t, j = ((ids == e) & keep[:, None]).nonzero(as_tuple=True)
            gate, up, down = (_exact_weight(s["w"][n][0][e], s["w"][n][1][e], c)
                              for n, c in (("gate", H), ("up", H), ("down", I)))
            g = x[t] @ gate.T
            y.index_add_(0, t, sel[t, j, None] * ((g / (1 + torch.exp(-g)) * (x[t] @ up.T)) @ down.T))
        return y
    # the losses by their definition, their gradient (and that of the weights) by differentiating it
    with torch.enable_grad():
        l, keep, ids = _exact_route(case, s)
        l.requires_grad_(True)
        E, k, n = case["experts"], case["top_k"], max(1, int(keep.sum()))
        p = torch.softmax(l, -1)
        w = p.gather(1, ids)
        if case["norm"]:
            w = w / w.sum(-1, keepdim=True)
        w = torch.where(keep[:, None], w, torch.zeros_like(w))
        share = torch.bincount(ids[keep].flatten(), minlength=E).double() / (n * k)
        balance = E * (share * p[keep].sum(0) / n).sum()
        z = (torch.logsumexp(l[keep], -1) ** 2).sum() / n
        total = (w * s["dw"].double()).sum() + s["gb"].double() * balance + s["gz"].double() * z
        d = torch.autograd.grad(total, l)[0]
    return None, w.detach(), None, balance.detach(), z.detach(), d
