"""Operators of the 8-bit feed-forward and of experts chosen by scores, as cases to time: each in a plain form (elementary torch operations) and, where
``own`` is true, through the package's entry points.  Widths are the ones ``bench.py`` and its workloads run (0.5b: 896 / 4864, 7b: 3584 / 18944).

``boundary``  ``rms_residual_fp8``: residual addition, weighted expert rows, norm, e4m3 with a scale for every 128 columns.
``quantize``  ``quantize_fp8``: an activation (none, gelu, silu gate) and the same 8-bit form.
``linear``    ``linear_fp8``: product of e4m3 rows and e4m3 weights, scales per 128 columns of a row and per 128 x 128 block of the weights.
``route``     ``route_by_scores``: scores to chosen experts, their weights, and the rows of the matrix sorted by expert."""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
FP8 = torch.float8_e4m3fn
BLOCK = 128
LEAST = 2.0 ** -100  # what a block's largest magnitude counts as at least
MOST = 448.0         # the largest e4m3 value
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # a decode step of one user
        dict(name="boundary_1", kind="boundary", rows=1, width=896, stream="fp32", delta="fp32", top=0, plain=False),
        # a decode batch behind a layer of experts, whose weighted rows are added here; the router reads the plain rows
        dict(name="boundary_64_experts", kind="boundary", rows=64, width=3584, stream="fp32", delta="fp32", top=2, plain=True),
        # a prompt batch of a model that keeps its residual in 16 bits
        dict(name="boundary_8192", kind="boundary", rows=8192, width=3584, stream="bf16", delta="bf16", top=0, plain=False),
        # behind the first product of a dense feed-forward: a decode batch of odd size, a prompt batch with gate
        dict(name="gelu_37", kind="quantize", rows=37, width=4864, act="gelu_tanh", dtype="bf16"),
        dict(name="gate_8192", kind="quantize", rows=8192, width=18944, act="silu_gate", dtype="bf16"),
        # products: one user (latency), a decode batch (weights from HBM), unequal prompts with sums that feed the residual, a prompt batch
        dict(name="linear_1", kind="linear", rows=1, k=896, features=4864, out="bf16"),
        dict(name="linear_64", kind="linear", rows=64, k=3584, features=18944, out="bf16"),
        dict(name="linear_1171", kind="linear", rows=1171, k=4864, features=896, out="fp32"),
        dict(name="linear_8192", kind="linear", rows=8192, k=3584, features=18944, out="bf16"),
        # routing: one user and few experts; a decode batch and a prompt batch over many experts in groups, with a bias for balance
        dict(name="route_1", kind="route", rows=1, experts=16, top=2, score="softmax", bias=False, groups=1, top_groups=1, dtype="bf16"),
        dict(name="route_64", kind="route", rows=64, experts=256, top=8, score="sigmoid", bias=True, groups=8, top_groups=4, dtype="fp32"),
        dict(name="route_8191", kind="route", rows=8191, experts=256, top=8, score="sigmoid", bias=True, groups=8, top_groups=4, dtype="fp32"),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(("boundary", "quantize", "linear", "linear", "route"))
    if kind == "boundary":
        stream = rng.choice(("fp32", "fp32", "bf16"))
        return dict(kind=kind, rows=_log(rng, 1, 8192), width=rng.choice((896, 1022, 2048, 3584, 4102, _log(rng, 100, 4096))), stream=stream,
                    delta="bf16" if stream == "bf16" else rng.choice(("fp32", "bf16")), top=rng.choice((0, 0, 1, 2, 6)), plain=rng.random() < 0.5)
    if kind == "quantize":
        return dict(kind=kind, rows=_log(rng, 1, 8192), width=rng.choice((896, 1021, 4864, 18944, _log(rng, 100, 18944))),
                    act=rng.choice(("none", "gelu_tanh", "silu_gate")), dtype=rng.choice(("bf16", "bf16", "fp32")))
    if kind == "linear":
        k, features = rng.choice(((896, 4864), (4864, 896), (3584, 4608), (3584, 18944), (18944, 3584), (_log(rng, 100, 5000), _log(rng, 100, 5000))))
        return dict(kind=kind, rows=_log(rng, 1, 8192 if k * features <= 3584 * 18944 else 4096), k=k, features=features, out=rng.choice(("bf16", "bf16", "fp32")))
    experts, groups = rng.choice(((8, 1), (16, 1), (60, 1), (64, 8), (128, 1), (160, 8), (256, 8), (384, 1), (_log(rng, 8, 384), 1)))
    top_groups = 1 if groups == 1 else rng.randint(2, groups)
    return dict(kind=kind, rows=_log(rng, 1, 8192), experts=experts, top=rng.randint(1, min(8, experts // groups * top_groups)),
                score=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.6, groups=groups, top_groups=top_groups,
                dtype=rng.choice(("fp32", "bf16")))


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def _rows8(n: int, width: int) -> torch.Tensor:
    """e4m3 rows that start on 16-byte boundaries."""
    return torch.empty((n, _up(width, 16)), dtype=FP8, device=DEV)[:, :width]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    n, kind = case["rows"], case["kind"]
    state = dict(case=case)
    if kind == "boundary":
        width, top = case["width"], case["top"]
        channel = 1.0 + 9.0 * (torch.rand(width, generator=g, device=DEV) < 0.01)  # a few channels of a residual are much larger
        state["x"] = (rnd(n, width) * channel).to(DTYPES[case["stream"]])
        state["delta"] = (0.3 * rnd(n, width)).to(DTYPES[case["delta"]])
        state["weight"] = 1.0 + 0.2 * rnd(width)
        if top:
            rows = _up(n * top, 8) + 8
            state["pairs"] = 0.5 * rnd(rows, width)
            state["pair_slots"] = torch.randperm(rows, generator=g, device=DEV)[: n * top].view(n, top).to(torch.int32)
            state["pair_slots"][torch.rand(n, top, generator=g, device=DEV) < 0.03] = -1  # tokens that had fewer experts
            state["pair_weights"] = torch.rand(n, top, generator=g, device=DEV)
    elif kind == "quantize":
        state["z"] = rnd(n, case["width"] * (2 if case["act"] == "silu_gate" else 1)).to(DTYPES[case["dtype"]])
    elif kind == "linear":
        k, f = case["k"], case["features"]
        blocks = -(-k // BLOCK)
        state["x"], state["w"] = _rows8(n, k), _rows8(f, k)
        # values as a block's scaling leaves them: the largest of a block near 448
        state["x"].copy_((rnd(n, k) * 130).clamp(-MOST, MOST))
        state["w"].copy_((rnd(f, k) * 110).clamp(-MOST, MOST))
        state["x_scales"] = (0.5 + torch.rand(blocks, n, generator=g, device=DEV)) / 130
        state["w_scales"] = (0.5 + torch.rand(-(-f // BLOCK), blocks, generator=g, device=DEV)) * 0.02 / 110
    else:
        e = case["experts"]
        liked = rnd(e)  # some experts are liked by all tokens; the bias was learned against that
        state["logits"] = (1.3 * rnd(n, e) + 0.7 * liked).to(DTYPES[case["dtype"]])
        state["bias"] = -0.08 * liked + 0.02 * rnd(e) if case["bias"] else None
    return state


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _blocks8(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows as e4m3 values [n, width] and scales [blocks, n]."""
    n, width = v.shape
    b = F.pad(v, (0, -width % BLOCK)).view(n, -1, BLOCK)
    scales = b.abs().amax(-1).clamp(min=LEAST) / MOST
    q = (b / scales[..., None]).clamp(-MOST, MOST).to(FP8)
    return q.view(n, -1)[:, :width], scales.t().contiguous()


def _plain_boundary(s: dict) -> dict:
    c, y = s["case"], s["x"].float() + s["delta"].float()
    if c["top"]:
        at = s["pair_slots"].long()
        rows = s["pairs"][at.clamp(min=0)] * torch.where(at < 0, 0.0, s["pair_weights"])[..., None]
        y = y + rows.sum(1)
    x_out = y.to(s["x"].dtype)
    y = x_out.float()
    v = y * (1.0 / (y.square().mean(-1, keepdim=True) + EPS).sqrt()) * s["weight"]
    q, scales = _blocks8(v)
    return dict(x=x_out, q=q, scales=scales, out=v.to(torch.bfloat16) if c["plain"] else None)


def _plain_quantize(s: dict) -> dict:
    z, act = s["z"].float(), s["case"]["act"]
    if act == "gelu_tanh":
        z = 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    elif act == "silu_gate":
        gate, up = z.chunk(2, dim=1)
        z = gate / (1.0 + torch.exp(-gate)) * up
    q, scales = _blocks8(z)
    return dict(q=q, scales=scales)


def _plain_linear(s: dict) -> torch.Tensor:
    k, f = s["case"]["k"], s["case"]["features"]
    x = s["x"].float() * s["x_scales"].t().repeat_interleave(BLOCK, 1)[:, :k]
    w = s["w"].float() * s["w_scales"].repeat_interleave(BLOCK, 0)[:f].repeat_interleave(BLOCK, 1)[:, :k]
    return (x @ w.t()).to(DTYPES[s["case"]["out"]])


def _layout(ids: torch.Tensor, experts: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of the matrix sorted by expert: segments start at multiples of eight, pairs in their order inside."""
    n, top = ids.shape
    flat = ids.reshape(-1).long()
    there = flat >= 0
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, torch.where(there, flat, experts), torch.ones_like(flat))[:experts]
    padded = (counts + 7) // 8 * 8
    first = padded.cumsum(0) - padded
    before = counts.cumsum(0) - counts
    order = torch.sort(torch.where(there, flat, experts), stable=True).indices
    place = torch.empty_like(flat)
    place[order] = torch.arange(n * top, device=ids.device)
    e = flat.clamp(min=0)
    slots = torch.where(there, first[e] + place - before[e], -1)
    return slots.view(n, top).to(torch.int32), torch.stack((first, counts), 1).to(torch.int32)


def _plain_route(s: dict) -> dict:
    c = s["case"]
    n, e, g, top = c["rows"], c["experts"], c["groups"], c["top"]
    l = s["logits"].double()  # choices lie next to borders: 64 bits
    score = torch.softmax(l, 1) if c["score"] == "softmax" else 1.0 / (1.0 + torch.exp(-l))
    chosen_by = score if s["bias"] is None else score + s["bias"].double()
    if g > 1:
        best = torch.sort(chosen_by.view(n, g, e // g), dim=2, descending=True).values[..., :2].sum(2)
        keep = torch.sort(best, dim=1, descending=True, stable=True).indices[:, : c["top_groups"]]
        kept = torch.zeros((n, g), dtype=torch.bool, device=l.device).scatter_(1, keep, True)
        chosen_by = torch.where(kept.repeat_interleave(e // g, 1), chosen_by, -math.inf)
    ids = torch.sort(chosen_by, dim=1, descending=True, stable=True).indices[:, :top]
    weights = score.gather(1, ids)
    weights = (weights / weights.sum(1, keepdim=True)).float()
    slots, segs = _layout(ids, e)
    return dict(ids=ids.to(torch.int32), weights=weights, slots=slots, segs=segs)


def _own(s: dict):
    from spikeinfer_b200.kernels import fp8, routing

    c, kind = s["case"], s["case"]["kind"]
    if kind == "boundary":
        x_out = torch.empty_like(s["x"])
        out = torch.empty(s["x"].shape, dtype=torch.bfloat16, device=DEV) if c["plain"] else None
        pairs = {k: s[k] for k in ("pairs", "pair_slots", "pair_weights")} if c["top"] else {}
        q, scales = fp8.rms_residual_fp8(s["x"], s["weight"], eps=EPS, delta=s["delta"], x_out=x_out, out=out, **pairs)
        return dict(x=x_out, q=q, scales=scales, out=out)
    if kind == "quantize":
        q, scales = fp8.quantize_fp8(s["z"], c["act"])
        return dict(q=q, scales=scales)
    if kind == "linear":
        return fp8.linear_fp8(s["x"], s["x_scales"], s["w"], s["w_scales"], out_dtype=DTYPES[c["out"]])
    r = routing.route_by_scores(s["logits"], c["top"], score=c["score"], bias=s["bias"], groups=c["groups"], top_groups=c["top_groups"])
    return dict(ids=r.ids, weights=r.weights, slots=r.slots, segs=r.segs)


def run(state: dict):
    if own:
        return _own(state)
    return {"boundary": _plain_boundary, "quantize": _plain_quantize, "linear": _plain_linear, "route": _plain_route}[state["case"]["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case: dict) -> dict:
    n, kind = case["rows"], case["kind"]
    size = lambda d: 4 if d == "fp32" else 2
    if kind == "boundary":
        w, top = case["width"], case["top"]
        per = 2 * size(case["stream"]) + size(case["delta"]) + 1 + (2 if case["plain"] else 0) + 4 * top
        return dict(bytes=n * w * per + 4 * w + 4 * n * -(-w // BLOCK) + 8 * n * top, flops=n * w * (8 + 2 * top))
    if kind == "quantize":
        w, gate = case["width"], case["act"] == "silu_gate"
        return dict(bytes=n * w * (size(case["dtype"]) * (2 if gate else 1) + 1) + 4 * n * -(-w // BLOCK), flops=n * w * 10)
    if kind == "linear":
        k, f = case["k"], case["features"]
        blocks = -(-k // BLOCK)
        return dict(bytes=(n + f) * k + 4 * blocks * (n + -(-f // BLOCK)) + n * f * size(case["out"]), flops=2 * n * k * f)
    e, top = case["experts"], case["top"]
    return dict(bytes=n * e * size(case["dtype"]) + (4 * e if case["bias"] else 0) + 12 * n * top + 8 * e, flops=n * e * 20)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _nearest_e4m3(a: torch.Tensor) -> torch.Tensor:
    """The e4m3 value next to each of ``a`` (half to even): steps of 2^-3 of the power of two below, of 2^-9 under 2^-6."""
    _, exponent = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), (exponent - 1).clamp(min=-6) - 3)
    return (torch.round(a / step) * step).clamp(-MOST, MOST)


def _exact_blocks(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    n, width = v.shape
    blocks = -(-width // BLOCK)
    block_of = torch.arange(width, device=v.device) // BLOCK
    most = torch.zeros((n, blocks), dtype=v.dtype, device=v.device).scatter_reduce_(1, block_of.expand(n, width), v.abs(), "amax")
    scales = torch.maximum(most, torch.full_like(most, LEAST)) / MOST
    return _nearest_e4m3(v / scales[:, block_of]), scales.t()


def exact(case: dict, seed: int):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "boundary":
        y = s["x"].double() + s["delta"].double()
        for j in range(case["top"]):
            at = s["pair_slots"][:, j].long()
            row = s["pairs"].double().index_select(0, at.clamp(min=0)) * s["pair_weights"][:, j, None].double()
            y += torch.where(at[:, None] >= 0, row, torch.zeros_like(row))
        x_out = y
        if case["stream"] != "fp32":
            y = y.to(s["x"].dtype).double()
        v = y / torch.sqrt((y * y).sum(1, keepdim=True) / case["width"] + EPS) * s["weight"].double()
        q, scales = _exact_blocks(v)
        return dict(x=x_out, q=q, scales=scales, out=v if case["plain"] else None)
    if kind == "quantize":
        z = s["z"].double()
        if case["act"] == "gelu_tanh":
            z = z * torch.sigmoid(2.0 * (2.0 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3))
        elif case["act"] == "silu_gate":
            z = z[:, : case["width"]] * torch.sigmoid(z[:, : case["width"]]) * z[:, case["width"]:]
        q, scales = _exact_blocks(z)
        return dict(q=q, scales=scales)
    if kind == "linear":
        k, f = case["k"], case["features"]
        out = torch.zeros((case["rows"], f), dtype=torch.float64, device=DEV)
        sw = s["w_scales"].double()[torch.arange(f, device=DEV) // BLOCK]
        for b0 in range(0, k, 8 * BLOCK):  # eight blocks at a time
            cols = torch.arange(b0, min(k, b0 + 8 * BLOCK), device=DEV)
            part = s["x"][:, b0: b0 + len(cols)].double() * s["x_scales"].double()[cols // BLOCK].t()
            out.addmm_(part, (s["w"][:, b0: b0 + len(cols)].double() * sw[:, cols // BLOCK]).t())
        return out
    l = s["logits"].double()
    raw = torch.exp(l - torch.logsumexp(l, 1, keepdim=True)) if case["score"] == "softmax" else torch.sigmoid(l)
    by = raw + s["bias"].double() if case["bias"] else raw.clone()
    n, e, g = case["rows"], case["experts"], case["groups"]
    if g > 1:
        two = by.view(n, g, -1).topk(2, dim=2).values.sum(2)
        lost = torch.ones((n, g), dtype=torch.bool, device=DEV)
        lost.scatter_(1, two.topk(case["top_groups"], dim=1).indices, False)
        by.view(n, g, -1)[lost] = -math.inf
    ids = by.topk(case["top"], dim=1).indices
    weights = raw.gather(1, ids)
    return dict(ids=None, weights=weights / weights.sum(1, keepdim=True), slots=None, segs=None)
