"""Operators of serving in block-scaled 8 bits, case by case: activations in E4M3 with one scale for each row and 128 columns, weights in E4M3
with one scale for each 128 x 128, and what an engine computes with them.

``norm`` is the RMS norm with the residual's addition that leaves such rows, ``linear`` a projection's product, ``experts`` the products of
rows sorted by expert, ``gated`` a gate-up product (of a dense layer or by expert) with SwiGLU that leaves such rows for the next one. Sizes are the
layers of this package's models (2048 wide with 128 experts of 768, 2560 and 4096 wide dense ones) from a single token of the
tail of a rollout to the prompts of a step, and odd ones whose last blocks are partial.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK, TOP, LEAST, EPS = 128, 448.0, 1e-10, 1e-6
ROW_TILE = 128


def listed():
    return [
        # the tail of a rollout: one token's norm before the router, which wants it in bf16 too (latency)
        dict(name="norm-1", kind="norm", rows=1, width=2048, residual=True, keep=True),
        # a short prompt enters a layer
        dict(name="norm-777", kind="norm", rows=777, width=2560, residual=False, keep=False),
        # the prompts of a step between attention and a dense layer's gate-up product
        dict(name="norm-16384", kind="norm", rows=16384, width=4096, residual=True, keep=False),
        # one token's q, k and v
        dict(name="linear-1", kind="linear", rows=1, n=5120, k=2048, given=True, residual=False),
        # a decode batch of a dense model on its way back into the residual stream
        dict(name="linear-23", kind="linear", rows=23, n=2560, k=9728, given=True, residual=True),
        # sizes whose last blocks are partial on every side, activations that arrive in bf16
        dict(name="linear-301-odd", kind="linear", rows=301, n=1000, k=1040, given=False, residual=False),
        # the attention output of the prompts of a step: bf16 rows, residual
        dict(name="linear-8192", kind="linear", rows=8192, n=4096, k=4096, given=False, residual=True),
        # the gate-up product of a dense model's prompts (the largest)
        dict(name="gated-8192", kind="gated", groups=0, rows=8192, top_k=1, inter=12288, k=4096),
        # the beginning of a rollout: 64 running rows, eight experts each of 128: a few rows an expert, some without any
        dict(name="gated-experts-64", kind="gated", groups=128, rows=64, top_k=8, inter=768, k=2048),
        # the prompts of a step
        dict(name="gated-experts-8192", kind="gated", groups=128, rows=8192, top_k=8, inter=768, k=2048),
        # nine running rows back into the residual stream
        dict(name="experts-9", kind="experts", groups=128, rows=9, top_k=8, n=2048, k=768),
        # the prompts of a step
        dict(name="experts-8192", kind="experts", groups=128, rows=8192, top_k=8, n=2048, k=768),
    ]


def draw(rng):
    """One more case of the same ranges; sizes are drawn over their logarithm."""
    size = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    wide = lambda lo, hi: max(16, size(lo, hi) // 16 * 16)  # noqa: E731
    kind = rng.choice(["norm", "linear", "linear", "gated", "gated", "experts"])
    if kind == "norm":
        return dict(kind=kind, rows=size(1, 16384), width=wide(512, 4096), residual=rng.random() < 0.5, keep=rng.random() < 0.5)
    if kind == "linear":
        return dict(kind=kind, rows=size(1, 8192), n=size(128, 6144), k=wide(256, 9728), given=rng.random() < 0.5, residual=rng.random() < 0.5)
    if kind == "gated" and rng.random() < 0.4:
        return dict(kind=kind, groups=0, rows=size(1, 8192), top_k=1, inter=wide(256, 12288), k=wide(512, 4096))
    top_k = rng.randint(1, 8)
    case = dict(kind=kind, groups=rng.choice([8, 32, 60, 128]), rows=size(1, 8192), top_k=top_k, k=wide(512, 2048))
    return case | (dict(inter=wide(256, 768)) if kind == "gated" else dict(n=size(512, 2048)))


# ---------------------------------------------------------------------------------------------- inputs
def _blocks(n):
    return -(-n // BLOCK)


def _weight(shape, gen):
    """A matrix, or one for each expert, as a checkpoint holds it: E4M3 values and the scales of their 128 x 128 blocks."""
    *lead, n, k = shape
    w = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(0.02)
    rows, cols = _blocks(n), _blocks(k)
    padded = torch.zeros(*lead, rows * BLOCK, cols * BLOCK, device="cuda", dtype=torch.bfloat16)
    padded[..., :n, :k] = w
    amax = padded.view(*lead, rows, BLOCK, cols, BLOCK).abs().amax((-3, -1)).float()
    scales = amax.clamp_min(LEAST) / TOP
    wide = scales.repeat_interleave(BLOCK, -2).repeat_interleave(BLOCK, -1)[..., :n, :k]
    return (w.float() / wide).clamp(-TOP, TOP).to(torch.float8_e4m3fn), scales


def _activations(rows, k, gen):
    """Rows as they come out of a transformer's layers: channels of different size, a few of them far larger than the others."""
    channel = torch.randn(k, generator=gen, device="cuda").mul_(0.5).exp_()
    channel *= 1 + 20 * (torch.rand(k, generator=gen, device="cuda") < 0.005)
    return (torch.randn(rows, k, generator=gen, device="cuda") * channel).to(torch.bfloat16)


def _plan(case, gen):
    """The rows of every expert, and the row tiles {expert, first row, rows, 0} that the router's sort leaves: experts are not equally liked."""
    groups, rows, top_k = case["groups"], case["rows"], case["top_k"]
    liked = torch.randn(groups, generator=gen, device="cuda") * 0.5
    noise = -torch.log(-torch.log(torch.rand(rows, groups, generator=gen, device="cuda").clamp(1e-6, 1 - 1e-6)))
    ids = (liked + noise).topk(top_k, dim=1).indices
    counts = torch.bincount(ids.flatten(), minlength=groups).tolist()
    tiles, first = [], 0
    for g, c in enumerate(counts):
        tiles += [(g, first + a, min(ROW_TILE, c - a), 0) for a in range(0, c, ROW_TILE)]
        first += c
    live = len(tiles)
    tiles += [(0, 0, 0, 0)] * (groups + first // ROW_TILE + 1 - live)  # as many as there can be for this many rows
    counts = torch.tensor(counts, device="cuda")
    group = torch.repeat_interleave(torch.arange(groups, device="cuda"), counts)
    place = torch.arange(first, device="cuda") - (counts.cumsum(0) - counts)[group]  # of a row among its expert's
    return dict(most=int(counts.max()), group=group, place=place, tiles=torch.tensor(tiles, dtype=torch.int32, device="cuda"),
                live=torch.tensor([live], dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, s = case["kind"], dict(case=case)
    if kind == "norm":
        s["x"] = _activations(case["rows"], case["width"], gen)
        s["residual"] = _activations(case["rows"], case["width"], gen) if case["residual"] else None
        s["weight"] = (1 + 0.1 * torch.randn(case["width"], generator=gen, device="cuda")).to(torch.bfloat16)
        return s
    n = 2 * case["inter"] if kind == "gated" else case["n"]
    groups = case.get("groups", 0)
    lead = ((groups,) if groups else ()) + ((2,) if kind == "gated" else ())  # gate and up are two matrices, with blocks of their own
    wq, ws = _weight((*lead, n // 2 if kind == "gated" else n, case["k"]), gen)
    s["wq"], s["ws"] = (wq.flatten(-3, -2), ws.flatten(-3, -2)) if kind == "gated" else (wq, ws)
    s["plan"] = _plan(case, gen) if groups else None
    rows = case["rows"] * case.get("top_k", 1)
    x = _activations(rows, case["k"], gen)
    if case.get("given", True):
        s["xq"], s["xs"] = _quantized(x.float())
    else:
        s["x"] = x
    s["residual"] = _activations(rows, n, gen) if case.get("residual") else None
    return s


# ---------------------------------------------------------------------------------------------- the plain form, in 32 bits
def _quantized(x):
    """E4M3 rows and the scales of their blocks of 128 columns."""
    rows, k = x.shape
    padded = torch.nn.functional.pad(x, (0, -k % BLOCK))
    scales = padded.view(rows, -1, BLOCK).abs().amax(-1).clamp_min(LEAST) / TOP
    q = (x / scales.repeat_interleave(BLOCK, 1)[:, :k]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return q, scales


def _values(q, scales, by=(1,), dtype=torch.float32):
    """The numbers that 8-bit values and their scales stand for."""
    wide = scales.to(dtype).repeat_interleave(BLOCK, -1)
    if 0 in by:
        wide = wide.repeat_interleave(BLOCK, -2)
    return q.to(dtype) * wide[..., :q.shape[-2], :q.shape[-1]]


def _product(s, x):
    wq, ws = s["wq"], s["ws"]
    if s["case"]["kind"] == "gated":
        w = _values(wq.unflatten(-2, (2, -1)), ws.unflatten(-2, (2, -1)), (0, 1)).flatten(-3, -2)
    else:
        w = _values(wq, ws, (0, 1))
    plan = s["plan"]
    if plan is None:
        return x @ w.t()
    padded = x.new_zeros(w.shape[0], plan["most"], x.shape[1])
    padded[plan["group"], plan["place"]] = x
    return torch.bmm(padded, w.transpose(1, 2))[plan["group"], plan["place"]]


def _plain(s):
    case = s["case"]
    if case["kind"] == "norm":
        h = s["x"]
        if case["residual"]:
            h = (h.float() + s["residual"].float()).to(torch.bfloat16)
        f = h.float()
        y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
        q, scales = _quantized(y)
        out = dict(q=q, scales=scales)
        if case["residual"]:
            out["sum"] = h
        if case["keep"]:
            out["y"] = y.to(torch.bfloat16)
        return out
    xq, xs = (s["xq"], s["xs"]) if "xq" in s else _quantized(s["x"].float())
    y = _product(s, _values(xq, xs))
    if case["kind"] == "gated":
        gate, up = y.chunk(2, dim=-1)
        q, scales = _quantized(gate / (1 + torch.exp(-gate)) * up)
        return dict(q=q, scales=scales)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(torch.bfloat16))


# ---------------------------------------------------------------------------------------------- the framework's calls
def _framework(s):
    from miles_b200.ops import fp8_block as F8

    case = s["case"]
    if case["kind"] == "norm":
        rows, total, y = F8.rmsnorm_rows(s["x"], s["weight"], EPS, s["residual"], keep=case["keep"])
        out = dict(q=rows.q, scales=rows.scales)
        if case["residual"]:
            out["sum"] = total
        if case["keep"]:
            out["y"] = y
        return out
    w = F8.Fp8Weight(s["wq"], s["ws"], halves=2 if case["kind"] == "gated" else 1)
    x = F8.Fp8Rows(s["xq"], s["xs"]) if "xq" in s else s["x"]
    plan = (s["plan"]["tiles"], s["plan"]["live"]) if s["plan"] is not None else None
    if case["kind"] == "gated":
        rows = F8.gated_linear(x, w) if plan is None else F8.grouped_gated_linear(x, w, *plan)
        return dict(q=rows.q, scales=rows.scales)
    return dict(y=F8.linear(x, w, s["residual"]) if plan is None else F8.grouped_linear(x, w, *plan))


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "norm":
        n, scales = case["rows"] * case["width"], case["rows"] * _blocks(case["width"])
        return dict(bytes=2 * n + n + 4 * scales + 2 * case["width"] + (4 * n if case["residual"] else 0) + (2 * n if case["keep"] else 0), flops=8 * n)
    rows, k = case["rows"] * case.get("top_k", 1), case["k"]
    n = 2 * case["inter"] if case["kind"] == "gated" else case["n"]
    groups = case.get("groups", 0)
    # an expert that no row chose is not read; every row's choices are taken as equally likely here
    live = groups * (1 - (1 - case["top_k"] / groups) ** case["rows"]) if groups else 1
    moved = live * (n * k + 4 * _blocks(n) * _blocks(k)) + (rows * k + 4 * rows * _blocks(k) if case.get("given", True) else 2 * rows * k)
    if case["kind"] == "gated":
        moved += rows * case["inter"] + 4 * rows * _blocks(case["inter"])
    else:
        moved += 2 * rows * n + (2 * rows * n if case.get("residual") else 0)
    return dict(bytes=int(moved), flops=2 * rows * n * k)


# ---------------------------------------------------------------------------------------------- in 64 bits, from the definitions
def _rows64(v):
    """Scales of blocks of 128 columns, and the values over them before they are rounded to 8 bits."""
    scales = torch.stack([b.abs().amax(1) for b in v.split(BLOCK, dim=1)], 1).clamp(min=LEAST) / TOP
    return torch.cat([b / scales[:, i:i + 1] for i, b in enumerate(v.split(BLOCK, dim=1))], 1), scales


def _matrix64(q, scales, halves):
    if halves == 2:
        n, rows = q.shape[0] // 2, scales.shape[0] // 2
        return torch.cat([_matrix64(q[:n], scales[:rows], 1), _matrix64(q[n:], scales[rows:], 1)])
    out = q.double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            out[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scales[i, j].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        h = s["x"].double()
        if case["residual"]:
            h = (h + s["residual"].double()).to(torch.bfloat16).double()  # what is stored is what is normalised
        y = h / ((h * h).sum(1, keepdim=True) / case["width"] + EPS).sqrt() * s["weight"].double()
        q, scales = _rows64(y)
        out = dict(q=q, scales=scales)
        if case["residual"]:
            out["sum"] = s["x"].double() + s["residual"].double()
        if case["keep"]:
            out["y"] = y
        return out
    if "xq" in s:
        xq, xs = s["xq"].double(), s["xs"].double()
    else:
        v, xs32 = _rows64(s["x"].double())
        xs = xs32.float().double()  # a scale is a 32-bit number, and its rows are rounded to 8 bits
        xq = (s["x"].double() / xs.repeat_interleave(BLOCK, 1)[:, :v.shape[1]]).float().clamp(-TOP, TOP).to(torch.float8_e4m3fn).double()
    x = torch.cat([b * xs[:, i:i + 1] for i, b in enumerate(xq.split(BLOCK, dim=1))], 1)
    halves = 2 if case["kind"] == "gated" else 1
    if s["plan"] is None:
        y = x @ _matrix64(s["wq"], s["ws"], halves).t()
    else:
        y = x.new_zeros(x.shape[0], s["wq"].shape[1])
        for g, first, rows, _ in s["plan"]["tiles"].tolist():
            if rows:
                y[first:first + rows] = x[first:first + rows] @ _matrix64(s["wq"][g], s["ws"][g], halves).t()
    if case["kind"] == "gated":
        gate, up = y[:, :case["inter"]], y[:, case["inter"]:]
        q, scales = _rows64(gate * torch.sigmoid(gate) * up)
        return dict(q=q, scales=scales)
    return dict(y=y if s["residual"] is None else y + s["residual"].double())
