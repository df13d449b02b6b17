"""Performance cases of the operators around the head's grouped products: the norm
that takes the residual in, rows on their way to their experts and back, and products
of microscaled operands.

Kinds of case (``case["kind"]``):

* ``norm``: root-mean-square norm of (rows, width), with ``residual`` of the sum of the
  input and a residual, which comes out too; with ``format`` the result is quantised
  (8 bits with a power of two for every 32 values);
* ``rows``: (tokens, k) expert numbers sorted by expert, tokens' rows copied to their
  experts' places, and the experts' rows summed back with weights;
* ``quantize``: rows to microscaled 8-bit values;
* ``product``: rows quantised (``act``) and, in ragged groups, times one microscaled
  matrix per group (``wgt``).

A case with ``train`` runs forward and backward and returns outputs and gradients.
``run`` computes an operator in its plain form, in 32 bits and rounded once, or, where
``own`` is set, makes the calls of this repository.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
BLOCK = 32  # values that share a scale
# of the element formats: the largest value, its exponent, the smallest normal exponent, fraction bits, bytes
LARGEST = {"e2m1": 6.0, "e4m3": 448.0}
EMAX = {"e2m1": 2, "e4m3": 8}
EMIN = {"e2m1": 0, "e4m3": -6}
FRACTION = {"e2m1": 1, "e4m3": 3}
ELEMENT = {"e2m1": 0.5, "e4m3": 1.0}


def _norm(dtype, rows, width, residual=True, train=True, format="", params=None):
    return dict(kind="norm", dtype=dtype, rows=rows, width=width, residual=residual, train=train, format=format,
                params=params or dtype)


def _rows(dtype, tokens, k, experts, width, dropped=0.0, train=True, params="f32"):
    """dropped: the share of the assignments that have no expert (a number outside 0 .. experts - 1)."""
    return dict(kind="rows", dtype=dtype, tokens=tokens, k=k, experts=experts, width=width, dropped=dropped, train=train,
                params=params)


def _quantize(dtype, rows, width):
    return dict(kind="quantize", dtype=dtype, rows=rows, width=width, train=False)


def _product(dtype, act, wgt, groups, rows, K, N, pad=0):
    return dict(kind="product", dtype=dtype, act=act, wgt=wgt, groups=groups, rows=rows, K=K, N=N, pad=pad, train=False)


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # one image's queries in inference, a call bound by its launch
        named("norm_f32_queries", _norm("f32", 200, 256, train=False)),
        # pixel tokens of four 1024 x 1024 images at stride 16 in a wide decoder, trained
        named("norm_bf16_train", _norm("bf16", 16384, 1024)),
        # an odd width, no residual, weights kept in float32
        named("norm_f16_odd", _norm("f16", 4097, 1153, residual=False, params="f32")),
        # a prompt's tokens on their way into products of 8-bit operands
        named("norm_bf16_to_e4m3", _norm("bf16", 8192, 4096, train=False, format="e4m3")),
        # single tokens: the router's choice of two of 32 experts
        named("rows_bf16_tokens", _rows("bf16", 16, 2, 32, 2048, train=False)),
        # a training batch, eight of 64 experts to a token
        named("rows_bf16_train", _rows("bf16", 8192, 8, 64, 1024, params="bf16")),
        # one expert to a token, an odd width, and a quarter of the tokens over the experts' capacity
        named("rows_f32_dropped", _rows("f32", 20011, 1, 16, 257, dropped=0.25)),
        # the activations of a batch
        named("quantize_bf16", _quantize("bf16", 16384, 2048)),
        # an odd number of rows from float32
        named("quantize_f32", _quantize("f32", 1001, 4128)),
        # single tokens through many experts: most groups hold none or one
        named("product_bf16_tokens", _product("bf16", "e4m3", "e2m1", 32, 32, 2048, 1024)),
        # a prompt's tokens through an expert's first product, 4-bit weights, room behind the last group
        named("product_f16_prompt", _product("f16", "e4m3", "e2m1", 8, 4096, 1024, 2736, pad=37)),
        # a batch's tokens sorted by expert, both operands in 4 bits
        named("product_bf16_batch", _product("bf16", "e2m1", "e2m1", 16, 16384, 1024, 4096)),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm", "rows", "rows", "rows", "quantize", "product", "product", "product"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    e = BYTES[dtype]
    while True:
        if kind == "norm":
            rows, width = _log_uniform(rng, 1, 100000), _log_uniform(rng, 32, 8192)
            if rng.random() < 0.6:  # most models' widths
                width = width // 32 * 32
            train = rng.random() < 0.6
            format = rng.choice(["", "e4m3"]) if not train and width % BLOCK == 0 else ""
            if rows * width * e <= 2 ** 26:
                return _norm(dtype, rows, width, rng.random() < 0.6, train, format, rng.choice([dtype, dtype, "f32"]))
        elif kind == "rows":
            tokens, k, experts = _log_uniform(rng, 1, 65536), rng.choice([1, 2, 2, 4, 8, 5]), _log_uniform(rng, 8, 256)
            width = _log_uniform(rng, 32, 8192)
            if rng.random() < 0.7:
                width = width // 32 * 32
            if tokens * k * width * e <= 1.1e8:
                return _rows(dtype, tokens, k, experts, width, rng.choice([0.0, 0.0, 0.1, 0.5]), rng.random() < 0.6,
                             rng.choice([dtype, "f32"]))
        elif kind == "quantize":
            rows, width = _log_uniform(rng, 1, 100000), max(1, _log_uniform(rng, 1, 300)) * BLOCK
            if rows * width * e <= 2 ** 27:
                return _quantize(dtype, rows, width)
        else:
            groups, rows = _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 16384)
            K, N = _log_uniform(rng, 2, 160) * BLOCK, _log_uniform(rng, 64, 5000)
            if rng.random() < 0.6:
                K, N = max(128, K // 128 * 128), max(16, N // 16 * 16)
            act, wgt = rng.choice([("e4m3", "e2m1"), ("e4m3", "e2m1"), ("e2m1", "e2m1"), ("e4m3", "e4m3"), ("e2m1", "e4m3")])
            if rows * K * N <= 3.4e10 and rows * (K + N) <= 6.0e7 and groups * K * N <= 6.7e7:
                return _product(dtype, act, wgt, groups, rows, K, N, rng.choice([0, 0, _log_uniform(rng, 1, 300)]))


# ---- microscaled values, in plain form ------------------------------------------
def _blocks(x, format):
    """Blocks of 32 values divided by their scales, and the scales' exponents: the largest magnitude's
    exponent less the format's, within 8 bits."""
    v = x.float().unflatten(-1, (-1, BLOCK))
    largest = v.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(largest).exponent - 1 - EMAX[format]
    exponent = torch.where(largest > 0, exponent, -127).clamp(-127, 127)
    return (v.double() * torch.exp2(-exponent.double())).float(), exponent


def _round(q, format):
    """The nearest values of the format, ties to the even code, held to the largest."""
    q = q.clamp(-LARGEST[format], LARGEST[format])
    if format == "e4m3":
        return q.to(torch.float8_e4m3fn).float()
    m = q.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    return torch.copysign(torch.round(m / step) * step, q)


def _scales(exponent):
    """As they are kept: 8 bits, the exponent and 127."""
    return (exponent.squeeze(-1) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _pack(q):
    """Codes of 4-bit values, two to a byte, the first in the low bits."""
    m = q.abs()
    code = torch.where(m < 2, 2 * m, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8)
    code = (code + 8 * torch.signbit(q).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2]


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values(codes, scales):
    """What kept codes and scales stand for, float32."""
    if codes.dtype == torch.uint8:
        table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
        q = table[torch.stack((codes & 15, codes >> 4), -1).long().flatten(-2)]
    else:
        q = codes.float()
    return (q.unflatten(-1, (-1, BLOCK)) * scales.float().unsqueeze(-1)).flatten(-2)


# ---- inputs ---------------------------------------------------------------------
def _offsets(case, seed, device):
    """Borders of the groups: uneven shares, some groups with none; and where each row goes when the groups
    lie one after another, padded to the longest."""
    rng = np.random.default_rng(seed)
    share = rng.gamma(2.0, size=case["groups"])
    counts = rng.multinomial(case["rows"], share / share.sum())
    offsets = np.concatenate([[0], np.cumsum(counts)])
    most = max(1, int(counts.max()))
    group = np.repeat(np.arange(case["groups"]), counts)
    slot = group * most + np.arange(case["rows"]) - offsets[group]
    return torch.from_numpy(offsets).to(device), torch.from_numpy(slot).to(device), most


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype, train, kind = DTYPES[case["dtype"]], case["train"], case["kind"]

    def normal(*shape, to=dtype, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=gen, device=device).mul_(scale).add_(shift).to(to)

    def leaf(x):
        return x.requires_grad_(train)

    def activations(rows, width):  # a few channels are larger than the others
        channel = torch.exp(0.7 * torch.randn(width, generator=gen, device=device))
        return (torch.randn(rows, width, generator=gen, device=device) * channel).to(dtype)

    s = dict(kind=kind, train=train)
    if kind == "norm":
        rows, width = case["rows"], case["width"]
        s["format"] = case["format"]
        s["x"] = leaf(normal(rows, width))
        s["residual"] = leaf(activations(rows, width)) if case["residual"] else None
        s["weight"] = leaf(normal(width, to=DTYPES[case["params"]], scale=0.1, shift=1.0))
        if train:
            s["dy"] = normal(rows, width, scale=0.02)
            s["ds"] = normal(rows, width, scale=0.02) if case["residual"] else None
    elif kind == "rows":
        T, k, E, D = case["tokens"], case["k"], case["experts"], case["width"]
        s["experts"] = E
        liked = 0.5 * torch.randn(E, generator=gen, device=device)  # uneven experts
        score = torch.randn(T, E, generator=gen, device=device) + liked
        top, ids = score.topk(k, dim=1)
        out = torch.rand(T, k, generator=gen, device=device) < case["dropped"]
        s["ids"] = torch.where(out, E, ids)
        s["weights"] = leaf(torch.softmax(top, 1).to(DTYPES[case["params"]]))
        s["x"] = leaf(normal(T, D))
        s["y"] = leaf(normal(T * k, D))  # the experts' results
        if train:
            s["dxs"] = normal(T * k, D, scale=0.02)
            s["dout"] = normal(T, D, scale=0.02)
    elif kind == "quantize":
        s["x"] = activations(case["rows"], case["width"])
    else:
        G, K, N = case["groups"], case["K"], case["N"]
        s["act"], s["dtype"], s["N"] = case["act"], dtype, N
        s["x"] = activations(case["rows"] + case["pad"], K)
        # a layer's weights, quantised when it was loaded
        scaled, exponent = _blocks(normal(G, N, K, scale=K ** -0.5), case["wgt"])
        q = _round(scaled, case["wgt"])
        s["codes"] = _pack(q) if case["wgt"] == "e2m1" else q.flatten(-2).to(torch.float8_e4m3fn)
        s["scales"] = _scales(exponent)
        s["offsets"], s["slot"], s["most"] = _offsets(case, seed, device)
    return s


# ---- plain forms ----------------------------------------------------------------
def _plain_norm(s):
    x, w = s["x"].float(), s["weight"].float()
    dt = s["x"].dtype
    out = ()
    if s["residual"] is not None:
        total = (x + s["residual"].float()).to(dt)
        x, out = total.float(), (total,)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    h = x * r
    y = h * w
    if s["format"]:
        scaled, exponent = _blocks(y, s["format"])
        return (_round(scaled, s["format"]).flatten(-2).to(torch.float8_e4m3fn), _scales(exponent), *out)
    if not s["train"]:
        return (y.to(dt), *out)
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - h * (g * h).mean(-1, keepdim=True))
    dw = (dy * h).sum(0).to(s["weight"].dtype)
    if s["residual"] is None:
        return y.to(dt), dx.to(dt), dw
    dx = (dx + s["ds"].float()).to(dt)
    return y.to(dt), *out, dx, dx, dw


def _plain_rows(s):
    ids, E, x, y, w = s["ids"], s["experts"], s["x"], s["y"], s["weights"]
    T, k = ids.shape
    key = torch.where((ids >= 0) & (ids < E), ids, E).flatten()
    order = torch.sort(key, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(T * k, device=order.device)
    offsets = (key[:, None] < torch.arange(E + 1, device=key.device)).sum(0)
    kept = (key < E).view(T, k, 1)
    slots = slots.view(T, k)
    xs = torch.where((torch.arange(T * k, device=order.device) < offsets[E])[:, None], x[order // k], 0)
    rows = torch.where(kept, y[slots].float(), 0.0)  # (T, k, D)
    out = (rows * w.float().unsqueeze(-1)).sum(1).to(y.dtype)
    if not s["train"]:
        return order, slots, offsets, xs, out
    dx = torch.where(kept, s["dxs"][slots].float(), 0.0).sum(1).to(x.dtype)
    dout = s["dout"].float().unsqueeze(1)
    dy = torch.empty(T * k, y.shape[1], device=y.device)
    dy[slots.flatten()] = torch.where(kept, dout * w.float().unsqueeze(-1), 0.0).flatten(0, 1)
    dw = (rows * dout).sum(-1).to(w.dtype)
    return order, slots, offsets, xs, out, dx, dy.to(y.dtype), dw


def _plain_product(s):
    scaled, exponent = _blocks(s["x"], s["act"])
    x = (_round(scaled, s["act"]) * torch.exp2(exponent.float())).flatten(-2)
    w, slot, most = _values(s["codes"], s["scales"]), s["slot"], s["most"]
    G, n = w.shape[0], slot.shape[0]
    padded = x.new_zeros(G * most, x.shape[1])
    padded[slot] = x[:n]
    y = torch.bmm(padded.view(G, most, -1), w.transpose(1, 2)).flatten(0, 1)
    out = x.new_zeros(x.shape[0], s["N"])
    out[:n] = y[slot]
    return out.to(s["dtype"])


@torch.no_grad()
def _plain(s):
    if s["kind"] == "norm":
        return _plain_norm(s)
    if s["kind"] == "rows":
        return _plain_rows(s)
    if s["kind"] == "quantize":
        scaled, exponent = _blocks(s["x"], "e4m3")
        return _round(scaled, "e4m3").flatten(-2).to(torch.float8_e4m3fn), _scales(exponent)
    return _plain_product(s)


def run(state):
    if not own:
        return _plain(state)
    from mask_loss_amd.functions import (from_experts, grouped_matmul_mx, mx_quantize, rms_norm, rms_norm_mx,
                                         sort_by_expert, to_experts)
    s, train = state, state["train"]
    if s["kind"] == "norm":
        if s["format"]:
            return rms_norm_mx(s["x"], s["weight"], EPS, s["residual"], format=s["format"])
        y = rms_norm(s["x"], s["weight"], EPS, s["residual"])
        if not train:
            return y if s["residual"] is not None else (y,)
        if s["residual"] is None:
            return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"]))
        grads = torch.autograd.grad(y, (s["x"], s["residual"], s["weight"]), (s["dy"], s["ds"]))
        return (y[0].detach(), y[1].detach(), *grads)
    if s["kind"] == "rows":
        order = sort_by_expert(s["ids"], s["experts"])
        xs = to_experts(s["x"], order)
        out = from_experts(s["y"], order, s["weights"])
        plan = (order.order, order.slots, order.offsets)
        if not train:
            return (*plan, xs, out)
        grads = torch.autograd.grad((xs, out), (s["x"], s["y"], s["weights"]), (s["dxs"], s["dout"]))
        return (*plan, xs.detach(), out.detach(), *grads)
    if s["kind"] == "quantize":
        return mx_quantize(s["x"], "e4m3")
    codes, scales = mx_quantize(s["x"], s["act"])
    return grouped_matmul_mx(codes, scales, s["codes"], s["scales"], s["offsets"], dtype=s["dtype"])


def work(case):
    e, train = BYTES[case["dtype"]], case["train"]
    if case["kind"] == "norm":
        n, res = case["rows"] * case["width"], case["residual"]
        w = case["width"] * BYTES[case["params"]]
        if case["format"]:
            return {"bytes": (3 if res else 1) * n * e + n * (1 + 1 / BLOCK) + w, "flops": 8 * n}
        # x, residual, sum, y; then dy, the sum's gradient, dx (the same for both)
        return {"bytes": ((4 if res else 2) + (3 if res else 2) * train) * n * e + (1 + train) * w,
                "flops": (14 if train else 6) * n}
    if case["kind"] == "rows":
        small = case["tokens"] * case["k"] * (24 + (1 + train) * BYTES[case["params"]]) + 8 * (case["experts"] + 1)
        n = case["tokens"] * case["width"]
        return {"bytes": (4 if train else 2) * n * (1 + case["k"]) * e + small,
                "flops": n * case["k"] * (6 if train else 2)}
    if case["kind"] == "quantize":
        n = case["rows"] * case["width"]
        return {"bytes": n * (e + 1 + 1 / BLOCK), "flops": 4 * n}
    rows = case["rows"] + case["pad"]
    read = rows * case["K"] * e + case["groups"] * case["N"] * case["K"] * (ELEMENT[case["wgt"]] + 1 / BLOCK)
    return {"bytes": read + rows * case["N"] * e, "flops": 2 * case["rows"] * case["K"] * case["N"]}


# ---- definitions in 64 bits -----------------------------------------------------
def _exact_mx(x, format):
    """(values in the format, scales): the scale is the power of two that brings the block's largest magnitude into
    the format's last binade, the values the nearest multiples of their own binade's step."""
    v = x.double().reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    top = v.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(top > 0, top, 2.0 ** -140)))
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))  # log2 rounds
    scale = torch.exp2((e - EMAX[format]).clamp(-127, 127))
    v = v / scale
    binade = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** EMIN[format])))
    step = torch.exp2(binade - FRACTION[format])
    v = (torch.round(v / step) * step).clamp(-LARGEST[format], LARGEST[format])
    return v.reshape(x.shape), scale.squeeze(-1)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        x, w = s["x"].double(), s["weight"].double()
        out = ()
        if case["residual"]:
            total = s["x"].float() + s["residual"].float()  # the one rounding that the definition has
            x = total.to(s["x"].dtype).double()
            out = (x,)
        D = case["width"]
        rms = torch.sqrt((x * x).sum(1, keepdim=True) / D + EPS)
        y = x / rms * w
        if case["format"]:
            return (*_exact_mx(y, case["format"]), *out)
        if not case["train"]:
            return (y, *out)
        dy = s["dy"].double()
        dh = dy * w
        # y = x w / rms; d rms = x dx / (D rms)
        dx = dh / rms - x * (dh * x).sum(1, keepdim=True) / (D * rms ** 3)
        dw = torch.einsum("rd,rd->d", dy, x / rms)
        if not case["residual"]:
            return y, dx, dw
        dx = dx + s["ds"].double()
        return y, *out, dx, dx, dw
    if case["kind"] == "rows":
        ids, E, T, k = s["ids"].cpu().numpy(), case["experts"], case["tokens"], case["k"]
        flat = np.where((ids < 0) | (ids >= E), E, ids).reshape(-1)
        order = np.concatenate([np.flatnonzero(flat == g) for g in range(E + 1)])
        slots = np.zeros(T * k, dtype=np.int64)
        slots[order] = np.arange(T * k)
        offsets = np.concatenate([[0], np.cumsum([(flat == g).sum() for g in range(E)])]).astype(np.int64)
        kept = int(offsets[E])
        dev = s["x"].device
        at = torch.from_numpy(order[:kept]).to(dev)
        x, y, w = s["x"].double(), s["y"].double(), s["weights"].double()
        token, weight = at // k, w.reshape(-1)[at][:, None]
        xs = torch.zeros_like(y)
        xs[:kept] = x[token]
        out = torch.zeros_like(x).index_add_(0, token, y[:kept] * weight)
        plan = tuple(torch.from_numpy(a).to(dev) for a in (order, slots.reshape(T, k), offsets))
        if not case["train"]:
            return (*plan, xs, out)
        dout = s["dout"].double()[token]
        dx = torch.zeros_like(x).index_add_(0, token, s["dxs"].double()[:kept])
        dy = torch.zeros_like(y)
        dy[:kept] = dout * weight
        dw = torch.zeros(T * k, dtype=torch.float64, device=dev)
        dw[at] = (dout * y[:kept]).sum(1)
        return (*plan, xs, out, dx, dy, dw.view(T, k))
    if case["kind"] == "quantize":
        return _exact_mx(s["x"], "e4m3")
    values, scale = _exact_mx(s["x"], case["act"])
    x = values * scale.repeat_interleave(BLOCK, 1)
    w = _values(s["codes"], s["scales"]).double()
    edges = s["offsets"].tolist()
    y = x.new_zeros(x.shape[0], case["N"])
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        y[lo:hi] = x[lo:hi] @ w[g].T
    return y
