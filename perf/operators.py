"""Performance cases of the head in front of the matching loss: the norm of a
decoder's queries and the products of each group's rows with the group's matrix
(an image's queries with its features, an expert's rows with its weights).

Kinds of case (``case["kind"]``):

* ``norm``: layer norm of (rows, width);
* ``masks``: mask logits, the queries of every image times that image's feature
  map, for all queries of all layers or, with ``rows``, for a ragged set per image;
* ``grouped``: rows in ragged groups times one matrix per group.

A case with ``train`` runs forward and backward and returns the output and every
gradient, the others run the forward alone.  ``run`` computes an operator in its
plain form, in 32 bits and rounded once, or, where ``own`` is set, makes the
calls of this repository.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def _norm(dtype, rows, width, params=None, train=True):
    """params: the type of weight and bias (the input's own where it is None)."""
    return dict(kind="norm", dtype=dtype, rows=rows, width=width, params=params or dtype, train=train)


def _masks(dtype, L, B, Q, C, H, W, rows=0, pad=0, train=True):
    """rows: 0 for Q queries of each layer and image, else so many rows in one
    ragged group per image, with `pad` rows behind the last group."""
    return dict(kind="masks", dtype=dtype, L=L, B=B, Q=Q, C=C, H=H, W=W, rows=rows, pad=pad, train=train)


def _grouped(dtype, groups, rows, K, N, transposed, pad=0, train=True):
    """transposed: matrices stored (N, K) as linear layers keep them, else (K, N)."""
    return dict(kind="grouped", dtype=dtype, groups=groups, rows=rows, K=K, N=N, transposed=transposed, pad=pad,
                train=train)


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # one image's 200 queries in inference: a call bound by its launch
        named("norm_f32_queries", _norm("f32", 200, 256, train=False)),
        # the decoder norm over ten layers' queries of a training batch
        named("norm_bf16_layers", _norm("bf16", 10 * 16 * 200, 256)),
        # pixel tokens of eight 1024 x 1024 images at strides 8, 16 and 32
        named("norm_f16_pixels", _norm("f16", 8 * (16384 + 4096 + 1024), 256)),
        # an odd width, its rows on no vector boundary
        named("norm_f32_odd", _norm("f32", 2048, 1153)),
        # wide rows of a large backbone, weights kept in float32
        named("norm_bf16_wide", _norm("bf16", 16384, 4096, params="f32")),
        # the headline of the matching step: 16 images, 200 queries, 256 x 256 logits;
        # the largest case
        named("masks_bf16_256", _masks("bf16", 1, 16, 200, 256, 256, 256)),
        # ten layers that share the features of two images, not square, float32
        named("masks_f32_layers", _masks("f32", 10, 2, 100, 256, 100, 168)),
        # inference: masks of the predictions that were kept, few per image
        named("masks_bf16_kept", _masks("bf16", 1, 8, 0, 256, 256, 256, rows=160, train=False)),
        # the matched queries of each image on a map of odd size, in a buffer with room behind them
        named("masks_f16_matched", _masks("f16", 1, 3, 0, 256, 97, 131, rows=190, pad=41)),
        # a batch's tokens sorted by expert, forward and backward
        named("experts_bf16_train", _grouped("bf16", 16, 16384, 1024, 4096, True)),
        # single tokens on their way through many experts: most groups hold none or one
        named("experts_bf16_tokens", _grouped("bf16", 32, 32, 2048, 1024, True, train=False)),
        # a prompt's tokens through an expert's first product, matrices stored (K, N)
        named("experts_f16_prompt", _grouped("f16", 8, 4096, 1024, 2736, False, train=False)),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "masks", "masks", "grouped", "grouped"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    train = rng.random() < 0.7
    while True:
        if kind == "norm":
            rows, width = _log_uniform(rng, 1, 200000), _log_uniform(rng, 32, 8192)
            if rng.random() < 0.5:  # most models' widths
                width = max(32, width // 32 * 32)
            if rows * width <= 2 ** 26:
                return _norm(dtype, rows, width, rng.choice([dtype, dtype, "f32"]), train)
        elif kind == "masks":
            L, B, Q = rng.choice([1, 1, 1, 3, 10]), _log_uniform(rng, 1, 16), _log_uniform(rng, 20, 300)
            C = rng.choice([64, 128, 256, 256, 512, _log_uniform(rng, 32, 512)])
            H, W = _log_uniform(rng, 24, 512), _log_uniform(rng, 24, 512)
            if rng.random() < 0.6:
                H, W = max(8, H // 8 * 8), max(8, W // 8 * 8)
            rows = pad = 0
            if rng.random() < 0.5:
                L, rows, pad = 1, _log_uniform(rng, 1, B * Q), rng.choice([0, 0, _log_uniform(rng, 1, 200)])
                Q = 0
            cells = H * W * max(rows, L * B * Q)
            small = 4 if dtype == "f32" else 1  # float32 products take longer
            if cells <= 2.0e8 / small and B * C * H * W <= 2.6e8 / small and cells * C <= 5.0e10 / small:
                return _masks(dtype, L, B, Q, C, H, W, rows, pad, train)
        else:
            groups, rows = _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 16384)
            K, N = _log_uniform(rng, 128, 4096), _log_uniform(rng, 128, 4096)
            if rng.random() < 0.7:
                K, N = K // 16 * 16, N // 16 * 16
            small = 4 if dtype == "f32" else 1
            if rows * K * N <= 5.0e10 / small and groups * K * N <= 1.3e8:
                return _grouped(dtype, groups, rows, K, N, rng.random() < 0.5, rng.choice([0, 0, _log_uniform(rng, 1, 300)]),
                                train)


def _counts(case, seed, groups, rows):
    """Rows of each group: uneven shares, some groups with none."""
    rng = np.random.default_rng(seed)
    share = rng.gamma(2.0, size=groups)
    return rng.multinomial(rows, share / share.sum())


def _plan(counts, layers, device):
    """Group borders, and where each row goes when the groups that share a matrix
    lie one after another, padded to the longest."""
    offsets = np.concatenate([[0], np.cumsum(counts)])
    matrices = len(counts) // layers
    per_matrix = counts.reshape(layers, matrices)
    before = np.cumsum(per_matrix, axis=0) - per_matrix  # rows of earlier layers in the same matrix
    most = max(1, int(per_matrix.sum(axis=0).max()))
    group = np.repeat(np.arange(len(counts)), counts)
    slot = (group % matrices) * most + before.reshape(-1)[group] + np.arange(offsets[-1]) - offsets[group]
    return torch.from_numpy(offsets).to(device), torch.from_numpy(slot).to(device), most


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype, train = DTYPES[case["dtype"]], case["train"]

    def normal(*shape, to=dtype, scale=1.0, shift=0.0):
        x = torch.randn(*shape, generator=gen, device=device).mul_(scale).add_(shift)
        return x.to(to)

    def leaf(x):
        return x.requires_grad_(train)

    s = dict(kind=case["kind"], train=train)
    if case["kind"] == "norm":
        rows, width, params = case["rows"], case["width"], DTYPES[case["params"]]
        s["x"] = leaf((torch.randn(rows, width, generator=gen, device=device)
                       + torch.randn(width, generator=gen, device=device)).to(dtype))
        s["weight"] = leaf(normal(width, to=params, scale=0.1, shift=1.0))
        s["bias"] = leaf(normal(width, to=params, scale=0.1))
        if train:
            s["dy"] = normal(rows, width, scale=0.02)
        return s
    if case["kind"] == "masks":
        L, B, Q, C, H, W = (case[k] for k in "LBQCHW")
        s["weight"] = leaf(normal(B, C, H, W, scale=2.0 * C ** -0.5))
        if case["rows"]:
            counts, L = _counts(case, seed, B, case["rows"]), 1
            s["x"] = leaf(normal(case["rows"] + case["pad"], C))
            s["ragged"] = True
            if train:
                s["dy"] = normal(case["rows"] + case["pad"], H, W, scale=0.02)
        else:
            counts = np.full(L * B, Q)
            s["x"] = leaf(normal(L, B, Q, C))
            s["ragged"] = False
            if train:  # the matching's gradient: a quarter of the queries are matched
                s["dy"] = normal(L, B, Q, H, W, scale=0.02)
                s["dy"].mul_((torch.rand(L, B, Q, 1, 1, generator=gen, device=device) < 0.25).to(dtype))
        s["transposed"] = False
    else:
        G, K, N, L = case["groups"], case["K"], case["N"], 1
        counts = _counts(case, seed, G, case["rows"])
        s["transposed"] = case["transposed"]
        s["weight"] = leaf(normal(*((G, N, K) if case["transposed"] else (G, K, N)), scale=K ** -0.5))
        s["x"] = leaf(normal(case["rows"] + case["pad"], K))
        if train:
            s["dy"] = normal(case["rows"] + case["pad"], N, scale=0.02)
    s["offsets"], s["slot"], s["most"] = _plan(counts, L, device)
    return s


@torch.no_grad()
def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    xc = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(xc.square().mean(-1, keepdim=True) + EPS)
    h = xc * r
    y = (h * w + b).to(s["x"].dtype)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return (y, dx.to(s["x"].dtype), (dy * h).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["bias"].dtype))


@torch.no_grad()
def _plain_grouped(s):
    x, w, slot, most = s["x"], s["weight"], s["slot"], s["most"]
    n, K, G = slot.shape[0], x.shape[-1], w.shape[0]
    wm = w.float().flatten(2)
    wm = wm.transpose(1, 2) if s["transposed"] else wm
    N = wm.shape[2]

    def lay_out(rows):  # (R, width) -> (G, most, width), zeros behind each group's rows
        out = rows.new_zeros(G * most, rows.shape[1], dtype=torch.float32)
        out[slot] = rows[:n].float()
        return out.view(G, most, -1)

    def put_back(padded, like):
        out = torch.zeros(like, dtype=torch.float32, device=x.device)
        out.view(-1, padded.shape[2])[:n] = padded.reshape(G * most, -1)[slot]
        return out.to(x.dtype)

    xp = lay_out(x.reshape(-1, K))
    y = put_back(torch.bmm(xp, wm), (*x.shape[:-1], *(w.shape[2:] if w.dim() == 4 else (N,))))
    if not s["train"]:
        return y
    dyp = lay_out(s["dy"].reshape(-1, N))
    dx = put_back(torch.bmm(dyp, wm.transpose(1, 2)), x.shape)
    dw = torch.bmm(dyp.transpose(1, 2), xp) if s["transposed"] else torch.bmm(xp.transpose(1, 2), dyp)
    return y, dx, dw.reshape(w.shape).to(w.dtype)


def run(state):
    if not own:
        return _plain_norm(state) if state["kind"] == "norm" else _plain_grouped(state)
    from mask_loss_amd.functions import grouped_matmul, layer_norm, mask_logits
    x, w = state["x"], state["weight"]
    leaves = (x, w)
    if state["kind"] == "norm":
        y = layer_norm(x, w, state["bias"], EPS)
        leaves = (x, w, state["bias"])
    elif state["kind"] == "masks":
        y = mask_logits(x, w, state["offsets"] if state["ragged"] else None)
    else:
        y = grouped_matmul(x, w, state["offsets"], transposed=state["transposed"])
    if not state["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))


def _sizes(case):
    """(rows in groups, rows in all, K, N, matrices) of a product's case."""
    if case["kind"] == "masks":
        rows = case["rows"] or case["L"] * case["B"] * case["Q"]
        return rows, rows + case["pad"], case["C"], case["H"] * case["W"], case["B"]
    return case["rows"], case["rows"] + case["pad"], case["K"], case["N"], case["groups"]


def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "norm":
        n, p = case["rows"] * case["width"], 2 * case["width"] * BYTES[case["params"]]
        return {"bytes": (4 * n * e + 2 * p) if case["train"] else (2 * n * e + p),
                "flops": (18 if case["train"] else 7) * n}
    used, rows, K, N, G = _sizes(case)
    io = (rows * K + G * K * N + rows * N) * e
    return {"bytes": 2 * io if case["train"] else io, "flops": 2 * used * K * N * (3 if case["train"] else 1)}


@torch.no_grad()
def exact(case, seed):
    """The operators' definitions in 64 bits, group by group."""
    s = prepare(case, seed)
    x, w = s["x"].double(), s["weight"].double()
    if case["kind"] == "norm":
        D = case["width"]
        b = s["bias"].double()
        mean = x.sum(1) / D
        var = (x * x).sum(1) / D - mean * mean
        sd = torch.sqrt(var + EPS)
        hat = (x - mean[:, None]) / sd[:, None]
        y = hat * w + b
        if not case["train"]:
            return y
        dy = s["dy"].double()
        dhat = dy * w
        # y = hat * w + b with hat = (x - mean) / sd: through hat, the mean and the deviation
        along = (dhat * hat).sum(1) / D
        dx = (dhat - dhat.sum(1)[:, None] / D - hat * along[:, None]) / sd[:, None]
        return y, dx, torch.einsum("rd,rd->d", dy, hat), dy.sum(0)
    used, rows, K, N, G = _sizes(case)
    x2, w2 = x.reshape(rows, K), (w.transpose(1, 2) if s["transposed"] else w.reshape(G, K, N))
    edges = s["offsets"].tolist()
    y = x.new_zeros(rows, N)
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        y[lo:hi] = x2[lo:hi] @ w2[g % G]
    shape = (*s["x"].shape[:-1], *(s["weight"].shape[2:] if case["kind"] == "masks" else (N,)))
    if not case["train"]:
        return y.view(shape)
    dy = s["dy"].double().reshape(rows, N)
    dx, dw = torch.zeros_like(x2), torch.zeros_like(w2)
    for g, (lo, hi) in enumerate(zip(edges, edges[1:])):
        dx[lo:hi] = dy[lo:hi] @ w2[g % G].T
        dw[g % G] += x2[lo:hi].T @ dy[lo:hi]
    dw = dw.transpose(1, 2) if s["transposed"] else dw
    return y.view(shape), dx.view(s["x"].shape), dw.reshape(s["weight"].shape)
