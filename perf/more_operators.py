"""Linears in 8-bit floating point, the norm that feeds them, and routing by groups of experts, as
cases that can be timed.

Four kinds of operator:

  norm    h = x + residual, y = h / rms(h) * weight; y in 8 bits with scales for serving, or with
          "train" as it is, with the gradients of x, residual (the same) and weight
  linear  y = x . W^T with W in 8 bits and a scale for each block of 128 x 128; x as it comes, or
          itself in 8 bits ("a8"); with "train" the gradient of x as well
  feed    the two together: the norm's 8-bit rows straight into the linear
  route   ids and weights of the k experts of a token, chosen by score + bias out of the best groups
          of experts; with "train" also tokens per expert, the balance and z losses, and the gradient
          of the logits

Eight bits are e4m3 (finite: up to 448). A block is 128 values of a row, or 128 x 128 of a weight; its
scale is its largest magnitude / 448 (at least 2^-126), an element is value * (1 / scale) rounded to the
nearest code, ties to even. Scale, reciprocal and product are 32-bit numbers. Weights are
N(0, 1 / columns), quantised so; activations, residuals and logits are N(0, 1).

Routing: s = sigmoid(logits) or softmax(logits), c = s + bias. A group's score is the sum of its
`group_top` largest c; the k largest c of the `top_groups` best groups are chosen, ties to the lowest
index. Weights are s of the chosen (norm: divided by their sum) times `scale`; the balance loss goes by
p = s / sum(s).
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token's hidden state before a layer's first product: launch latency
        dict(name="norm_decode_4096", kind="norm", rows=1, cols=4096, train=False, dtype="bf16"),
        # a prompt before an MLP
        dict(name="norm_prompt_2048", kind="norm", rows=2048, cols=5120, train=False, dtype="fp16"),
        # a training step over eight sequences of 2048
        dict(name="norm_train_16384", kind="norm", rows=16384, cols=4096, train=True, dtype="bf16"),
        # eight sequences decoded together, from the residual stream through an MLP gate
        dict(name="feed_decode_8_rows", kind="feed", rows=8, inp=5120, out=17408, dtype="bf16"),
        # one token through an attention-sized projection
        dict(name="linear_decode_4096", kind="linear", rows=1, inp=4096, out=4096, a8=False, train=False,
             dtype="bf16"),
        # twenty sequences decoded together through an MLP gate, both sides in 8 bits
        dict(name="linear_decode_20_rows_a8", kind="linear", rows=20, inp=5120, out=17408, a8=True,
             train=False, dtype="bf16"),
        # a short prompt of odd length through an MLP down projection
        dict(name="linear_prompt_333", kind="linear", rows=333, inp=17408, out=5120, a8=False, train=False,
             dtype="fp16"),
        # a long prompt (or one chunk of it) through an MLP gate, both sides in 8 bits
        dict(name="linear_prompt_2048_a8", kind="linear", rows=2048, inp=5120, out=17408, a8=True,
             train=False, dtype="bf16"),
        # a training step through a frozen MLP down projection: its output and the gradient of x
        dict(name="linear_train_2048", kind="linear", rows=2048, inp=17408, out=5120, a8=False, train=True,
             dtype="bf16"),
        # a decode batch through 256 experts in 8 groups, 4 of them kept
        dict(name="route_decode_64_e256", kind="route", tokens=64, experts=256, top_k=8, score="sigmoid",
             bias=True, groups=8, top_groups=4, group_top=2, norm=True, scale=2.5, pad=0.0, train=False,
             dtype="fp32"),
        # the same router in a training step over 32 sequences of 2048
        dict(name="route_train_65536_e256", kind="route", tokens=65536, experts=256, top_k=8,
             score="sigmoid", bias=True, groups=8, top_groups=4, group_top=2, norm=True, scale=2.5, pad=0.0,
             train=True, dtype="fp32"),
        # a small padded batch, softmax scores as they are, groups by their best expert, 16-bit logits
        dict(name="route_train_509_e160", kind="route", tokens=509, experts=160, top_k=6, score="softmax",
             bias=False, groups=8, top_groups=3, group_top=1, norm=False, scale=16.0, pad=0.2, train=True,
             dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng, lo, hi):
    """A model dimension: mostly a multiple of 256, else of the block, of 8, or odd."""
    step = rng.choice([256, 256, 256, BLOCK, BLOCK, 8, 1])
    return max(64, int(_log_int(rng, lo, hi) / step + 0.5) * step)


def _draw_norm(rng):
    train = rng.random() < 0.4
    cols = _dim(rng, 64, 8192)
    rows = max(1, min(_log_int(rng, 1, 16384), 16384 * 4096 // cols))
    return dict(kind="norm", rows=rows, cols=cols, train=train, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _draw_linear(rng):
    inp, out = _dim(rng, 256, 17408), _dim(rng, 256, 17408)
    rows = rng.choice([_log_int(rng, 1, 64), _log_int(rng, 65, 2048)])
    a8 = rng.random() < 0.5
    train = not a8 and rng.random() < 0.4
    rows = max(1, min(rows, 2048 * 5120 * 17408 // (inp * out)))
    return dict(kind="linear", rows=rows, inp=inp, out=out, a8=a8, train=train,
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _draw_feed(rng):
    inp, out = _dim(rng, 256, 8192), _dim(rng, 256, 17408)
    rows = max(1, min(_log_int(rng, 1, 2048), 2048 * 5120 * 17408 // (inp * out)))
    return dict(kind="feed", rows=rows, inp=inp, out=out, dtype=rng.choice(["bf16", "fp16"]))


def _draw_route(rng):
    experts = rng.choice([16, 60, 64, 128, 160, 192, 256, 384, 512])
    groups = rng.choice([g for g in (1, 2, 4, 5, 8, 16) if experts % g == 0])
    top_groups = rng.randint(1, groups)
    group_top = rng.choice([1, 2])
    top_k = min(top_groups * (experts // groups), rng.choice([1, 2, 4, 6, 8, 10]))
    train = rng.random() < 0.6
    tokens = _log_int(rng, 1, 65536 * 256 // max(256, experts))
    return dict(kind="route", tokens=tokens, experts=experts, top_k=top_k,
                score=rng.choice(["sigmoid", "sigmoid", "softmax"]), bias=rng.random() < 0.7, groups=groups,
                top_groups=top_groups, group_top=group_top, norm=rng.random() < 0.7,
                scale=rng.choice([1.0, 2.5, 16.0]), pad=rng.choice([0.0, 0.0, 0.25]), train=train,
                dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))


def draw(rng):
    return rng.choice([_draw_norm, _draw_linear, _draw_linear, _draw_feed, _draw_route])(rng)


# ------------------------------------------------------------ plain forms
def _codes(v, amax):
    """Values v of blocks with the largest magnitude amax -> codes as values, and scales."""
    s = (amax / torch.full_like(amax, 448.0)).clamp(min=2.0 ** -126)
    inv = torch.ones_like(s) / s
    return (v * inv).to(torch.float8_e4m3fn).float(), s


def _quantize_rows(x):
    """The values in 32 bits that rows [N, C] have in 8 bits."""
    N, C = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -C % BLOCK)).reshape(N, -1, BLOCK)
    q, s = _codes(b, b.abs().amax(-1, keepdim=True))
    return (q * s).reshape(N, -1)[:, :C]


def _quantize_weight(w):
    """Codes [OUT, IN] (e4m3) and scales [ceil(OUT / 128), ceil(IN / 128)] of a weight in 32 bits."""
    O, I = w.shape
    b = torch.nn.functional.pad(w, (0, -I % BLOCK, 0, -O % BLOCK))
    b = b.reshape(b.shape[0] // BLOCK, BLOCK, b.shape[1] // BLOCK, BLOCK)
    q, s = _codes(b, b.abs().amax((1, 3), keepdim=True))
    q = q.reshape(b.shape[0] * BLOCK, -1)[:O, :I]
    return q.to(torch.float8_e4m3fn), s[:, 0, :, 0].contiguous()


def _weight_values(codes, scales):
    O, I = codes.shape
    s = scales.repeat_interleave(BLOCK, 0)[:O].repeat_interleave(BLOCK, 1)[:, :I]
    return codes.float() * s


def _plain_norm(s):
    """h rounded to x's type, the norm of that in 32 bits, and its 1 / rms."""
    h = (s["x"].float() + s["res"].float()).to(s["x"].dtype)
    hf = h.float()
    r = 1.0 / torch.sqrt((hf.double() * hf.double()).mean(-1, keepdim=True) + EPS)
    xhat = (hf.double() * r).float()
    return h, xhat, r.float(), xhat * s["weight"].float()


def _run_plain_norm(s):
    dt = s["x"].dtype
    h, xhat, r, y = _plain_norm(s)
    if not s["case"]["train"]:
        return _quantize_rows(y).to(torch.bfloat16), h
    dy = s["dy"].float()
    g = dy * s["weight"].float()
    mean = (g.double() * xhat.double()).mean(-1, keepdim=True).float()
    dx = r * (g - xhat * mean) + s["dh"].float()
    dw = (dy * xhat).sum(0, dtype=torch.float64)
    return y.to(dt), h, dx.to(dt), dw.to(s["weight"].dtype)


def _plain_feed(s):
    h, _, _, y = _plain_norm(s)
    return (_quantize_rows(y) @ _weight_values(s["codes"], s["scales"]).T).to(s["x"].dtype), h


def _plain_linear(s):
    x = s["x"].float()
    if s["case"]["a8"]:
        x = _quantize_rows(x)
    w = _weight_values(s["codes"], s["scales"])
    y = (x @ w.T).to(s["x"].dtype)
    if not s["case"]["train"]:
        return y
    return y, (s["dy"].float() @ w).to(s["x"].dtype)


def _plain_route(s):
    case = s["case"]
    T, E, k, G = case["tokens"], case["experts"], case["top_k"], case["groups"]
    logits = s["logits"].detach().double()              # 64 bits: which of two near scores is larger
    keep = s["mask"] if s["mask"] is not None else torch.ones_like(logits[:, 0], dtype=torch.bool)
    m = logits.max(-1, keepdim=True).values
    ex = torch.exp(logits - m)
    total = ex.sum(-1, keepdim=True)
    soft = ex / total
    sig = case["score"] == "sigmoid"
    sc = 1.0 / (1.0 + torch.exp(-logits)) if sig else soft
    c = sc if s["bias"] is None else sc + s["bias"].double()
    if G > 1:
        by = torch.sort(c.reshape(T, G, E // G), dim=-1, descending=True).values
        best = by[..., :case["group_top"]].sum(-1)
        out = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, case["top_groups"]:]
        drop = torch.zeros(T, G, dtype=torch.bool, device=c.device).scatter_(1, out, True)
        c = torch.where(drop.repeat_interleave(E // G, 1), -math.inf, c)
    order = torch.sort(c, dim=-1, descending=True, stable=True).indices[:, :k]
    sel = sc.gather(1, order)
    w0 = sel / sel.sum(-1, keepdim=True) if case["norm"] else sel
    ids = torch.where(keep[:, None], order, -1).int()
    w = torch.where(keep[:, None], (case["scale"] * w0).float(), 0.0)
    if not case["train"]:
        return ids, w
    n = keep.sum().clamp(min=1).double()
    counts = torch.zeros(E + 1, dtype=torch.int32, device=c.device)
    counts.index_add_(0, torch.where(keep[:, None], order, E).flatten(),
                      torch.ones(order.numel(), dtype=torch.int32, device=c.device))
    counts = counts[:E]
    p = sc / sc.sum(-1, keepdim=True)
    live = keep[:, None].double()
    lse = m + torch.log(total)
    f = counts.double() * E / (n * n * k)
    balance = (f * (p * live).sum(0)).sum().float()
    z = ((lse * lse * live).sum() / n).float()
    # through the scores: d log(s) / d l is 1 - sigmoid(l), or the softmax's own
    f = s["gb"].double() * f
    d = p * (f - (p * f).sum(-1, keepdim=True))
    dw = s["dw"].double() * case["scale"]
    up = w0 * dw
    chosen = up - w0 * up.sum(-1, keepdim=True) if case["norm"] else up
    d.scatter_add_(1, order, chosen)
    if sig:
        d = d * (1.0 - sc)
    elif not case["norm"]:
        d = d - soft * up.sum(-1, keepdim=True)
    d = d + s["gz"].double() * 2 / n * lse * soft
    d = torch.where(keep[:, None], d, 0.0)
    return ids, w, counts, balance, z, d.to(s["logits"].dtype)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(0x5E1F + 6151 * int(seed))


def _weight(g, out, inp):
    """Codes and scales of a weight ~ N(0, 1 / inp), made in slices of whole blocks of rows."""
    codes = torch.empty(out, inp, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(-(-out // BLOCK), -(-inp // BLOCK), device="cuda")
    step = max(1, (1 << 25) // inp // BLOCK) * BLOCK
    for r in range(0, out, step):
        n = min(step, out - r)
        codes[r:r + n], scales[r // BLOCK:-(-(r + n) // BLOCK)] = _quantize_weight(
            torch.randn(n, inp, device="cuda", generator=g) / math.sqrt(inp))
    return codes, scales


def _inputs(case, seed):
    """Every tensor of the case, from the seed alone."""
    g, kind = _gen(seed), case["kind"]
    dt = DTYPES[case["dtype"]]

    def acts(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dt)

    if kind in ("norm", "feed"):
        rows, cols = case["rows"], case["cols"] if kind == "norm" else case["inp"]
        s = dict(x=acts(rows, cols), res=acts(rows, cols),
                 weight=(1 + 0.1 * torch.randn(cols, device="cuda", generator=g)).to(dt))
        if kind == "feed":
            s["codes"], s["scales"] = _weight(g, case["out"], cols)
        elif case["train"]:
            s["dy"], s["dh"] = acts(rows, cols), acts(rows, cols)
        return s
    if kind == "linear":
        codes, scales = _weight(g, case["out"], case["inp"])
        s = dict(codes=codes, scales=scales, x=acts(case["rows"], case["inp"]))
        if case["train"]:
            s["dy"] = acts(case["rows"], case["out"])
        return s
    T, E = case["tokens"], case["experts"]
    s = dict(logits=acts(T, E), mask=None, bias=None)
    if case["pad"]:
        s["mask"] = torch.rand(T, device="cuda", generator=g) >= case["pad"]
    if case["bias"]:
        s["bias"] = 0.05 * torch.randn(E, device="cuda", generator=g)
    if case["train"]:
        # of a loss summed over the tokens
        s["dw"] = torch.randn(T, case["top_k"], device="cuda", generator=g)
        s["gb"], s["gz"] = (torch.tensor(f * T, device="cuda") for f in (0.01, 0.001))
    return s


# -------------------------------------------------------------- one pass
def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if not own:
        return s
    from vqlab_amd import fp8
    if case["kind"] in ("linear", "feed"):
        a8 = case["kind"] == "feed" or case["a8"]
        s["module"] = fp8.F8Linear(s.pop("codes"), s.pop("scales"), act="fp8" if a8 else None)
    if case.get("train"):
        for name in ("x", "res", "weight", "logits"):
            if name in s:
                s[name].requires_grad_(True)
    return s


def run(state):
    case = state["case"]
    if not own:
        plain = dict(norm=_run_plain_norm, feed=_plain_feed, linear=_plain_linear, route=_plain_route)
        with torch.no_grad():
            return plain[case["kind"]](state)
    from vqlab_amd import fp8, router
    if case["kind"] == "norm":
        if not case["train"]:
            rows, h = fp8.rms_norm_f8(state["x"], state["weight"], EPS, residual=state["res"])
            return fp8.f8_dequantize(*rows), h
        y, h = fp8.rms_norm(state["x"], state["weight"], EPS, residual=state["res"])
        dx, dw = torch.autograd.grad((y, h), (state["x"], state["weight"]), (state["dy"], state["dh"]))
        return y.detach(), h.detach(), dx, dw
    if case["kind"] == "feed":
        rows, h = fp8.rms_norm_f8(state["x"], state["weight"], EPS, residual=state["res"])
        return state["module"](rows, out_dtype=state["x"].dtype), h
    if case["kind"] == "linear":
        y = state["module"](state["x"])
        if not case["train"]:
            return y
        return y.detach(), torch.autograd.grad(y, state["x"], state["dy"])[0]
    form = dict(norm_topk_prob=case["norm"], mask=state["mask"], score=case["score"], bias=state["bias"],
                groups=case["groups"], top_groups=case["top_groups"], group_top=case["group_top"],
                scale=case["scale"])
    if not case["train"]:
        return router.top_k(state["logits"], case["top_k"], **form)
    r = router.route(state["logits"], case["top_k"], **form)
    d = torch.autograd.grad((r.weights, r.balance, r.z), state["logits"],
                            (state["dw"], state["gb"], state["gz"]))[0]
    return r.ids, r.weights.detach(), r.counts, r.balance.detach(), r.z.detach(), d


# ------------------------------------------------------------------ work
def _f8_bytes(rows, cols):
    return rows * cols + rows * -(-cols // BLOCK) * 4


def work(case):
    kind, act = case["kind"], 4 if case["dtype"] == "fp32" else 2
    if kind == "norm":
        r, c = case["rows"], case["cols"]
        if case["train"]:                                   # x, residual, dy, dh in; y, h, dx out
            return dict(bytes=7 * r * c * act + 2 * c * act, flops=16 * r * c)
        # x and residual in, h and the 8-bit rows out; the rows in, their values out
        return dict(bytes=r * c * (3 * act + 2) + 2 * _f8_bytes(r, c) + c * act, flops=10 * r * c)
    if kind in ("linear", "feed"):
        r, i, o = case["rows"], case["inp"], case["out"]
        w = i * o + -(-i // BLOCK) * -(-o // BLOCK) * 4
        n = 2 if case.get("train") else 1
        more = 2 * r * i * act if kind == "feed" else 0     # the residual in, h out
        return dict(bytes=w + n * r * (i + o) * act + more, flops=2 * n * r * i * o)
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    if not case["train"]:
        return dict(bytes=T * E * act + 2 * T * k * 4, flops=10 * T * E)
    # logits in, ids and weights out; logits, ids, weights and their gradient in, gradient out
    return dict(bytes=3 * T * E * act + 5 * T * k * 4 + E * 4, flops=25 * T * E)


# --------------------------------------------------------- 64-bit results
def _grid(q):
    """q in 64 bits rounded to the values of e4m3: three bits after the first, multiples of 2^-9."""
    mag = q.abs().clamp(min=2.0 ** -6)
    e = torch.floor(torch.log2(mag))
    e = torch.where(torch.exp2(e) > mag, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= mag, e + 1, e)
    step = torch.exp2(e - 3)
    return (torch.round(q / step) * step).clamp(-448.0, 448.0)


def _f32(v):
    """v in 64 bits, rounded to a 32-bit number."""
    return v.float().double()


def _exact_rows(x, stored):
    """Rows in 64 bits as their 8-bit form says; stored: with the roundings of its 32-bit numbers."""
    fl = _f32 if stored else (lambda v: v)
    C = x.shape[1]
    b = torch.cat([x, x.new_zeros(x.shape[0], -C % BLOCK)], 1).unflatten(1, (-1, BLOCK))
    s = fl(b.abs().amax(-1, keepdim=True) / 448).clamp(min=2.0 ** -126)
    return (_grid(fl(b * fl(1 / s))) * s).flatten(1)[:, :C]


def _exact_norm(s):
    h = (s["x"].double() + s["res"].double()).to(s["x"].dtype).double()     # 53 bits hold the sum's rounding
    return h, h / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[1] + EPS) * s["weight"].double()


def _exact_product(x, s, dy=None):
    """x . W^T in 64 bits, a block of 128 rows of W after the other; with dy also dy . W."""
    codes, scales = s["codes"], s["scales"].double()
    O, I = codes.shape
    y = torch.empty(x.shape[0], O, dtype=torch.float64, device="cuda")
    dx = torch.zeros_like(x) if dy is not None else None
    per = 8 * BLOCK
    for r in range(0, O, per):
        w = codes[r:r + per].double()
        f = scales[r // BLOCK:(r + per) // BLOCK]
        rows = torch.arange(w.shape[0], device="cuda") // BLOCK
        cols = torch.arange(I, device="cuda") // BLOCK
        w *= f[rows][:, cols]
        y[:, r:r + per] = x @ w.T
        if dy is not None:
            dx += dy[:, r:r + per] @ w
    return y if dy is None else (y, dx)


def _exact_route(case, s):
    E, k, G = case["experts"], case["top_k"], case["groups"]
    keep = s["mask"] if s["mask"] is not None else torch.ones(case["tokens"], dtype=torch.bool, device="cuda")
    with torch.enable_grad():                               # the gradient by differentiating the definition
        l = s["logits"].double().requires_grad_(True)
        score = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.softmax(l, -1)
        with torch.no_grad():
            c = score if s["bias"] is None else score + s["bias"].double()
            g = c.unflatten(1, (G, E // G))
            gs = g.topk(case["group_top"], -1).values.sum(-1)
            rank = (gs[:, None, :] > gs[:, :, None]).sum(-1)                # groups with a better score
            lower = torch.ones(G, G, dtype=torch.bool, device="cuda").tril(-1)
            rank = rank + ((gs[:, None, :] == gs[:, :, None]) & lower).sum(-1)
            c = g.masked_fill((rank >= case["top_groups"])[..., None], -math.inf).flatten(1)
            ids = torch.argsort(-c, dim=-1, stable=True)[:, :k]
        w = score.gather(1, ids)
        if case["norm"]:
            w = w / w.sum(-1, keepdim=True)
        w = torch.where(keep[:, None], w * case["scale"], torch.zeros_like(w))
        if not case["train"]:
            return None, w.detach()
        n = max(1, int(keep.sum()))
        share = torch.bincount(ids[keep].flatten(), minlength=E).double() / (n * k)
        p = score / score.sum(-1, keepdim=True)
        balance = E * (share * p[keep].sum(0) / n).sum()
        z = (torch.logsumexp(l[keep], -1) ** 2).sum() / n
        total = (w * s["dw"].double()).sum() + s["gb"].double() * balance + s["gz"].double() * z
        d = torch.autograd.grad(total, l)[0]
    return None, w.detach(), None, balance.detach(), z.detach(), d


@torch.no_grad()
def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "linear":
        x = s["x"].double()
        return _exact_product(_exact_rows(x, True) if case["a8"] else x, s,
                              s["dy"].double() if case["train"] else None)
    if kind == "route":
        return _exact_route(case, s)
    if kind == "feed" or not case["train"]:
        h, y = _exact_norm(s)
        y = _exact_rows(y, False)
        return (_exact_product(y, s) if kind == "feed" else y), h
    with torch.enable_grad():
        w = s["weight"].double().requires_grad_(True)
        h = _exact_norm(s)[0].requires_grad_(True)
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w
        dx, dw = torch.autograd.grad((y, h), (h, w), (s["dy"].double(), s["dh"].double()))
    return y.detach(), h.detach(), dx, dw
