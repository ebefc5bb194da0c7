"""Plain float64 forms of the 8-bit operators and of the experts chosen by scores (CPU, no code shared with the product)."""
from __future__ import annotations

import math

import torch

LEAST = 2.0 ** -100


def e4m3_step(a: torch.Tensor) -> torch.Tensor:
    """Distance of neighbouring e4m3 values at ``a``."""
    _, exponent = torch.frexp(torch.where(a == 0, 2.0 ** -9, a.double()))
    return torch.ldexp(torch.ones_like(a, dtype=torch.float64), (exponent - 1).clamp(min=-6) - 3)


def block_scales(v: torch.Tensor) -> torch.Tensor:
    """``[blocks, n]``: largest finite magnitude of every 128 columns (an infinity as the largest fp32 value) over 448."""
    n, width = v.shape
    out = torch.zeros(-(-width // 128), n, dtype=torch.float64)
    for b in range(out.shape[0]):
        part = v[:, 128 * b: 128 * b + 128].abs()
        part = torch.where(part.isnan(), 0.0, part).clamp(max=torch.finfo(torch.float32).max)
        out[b] = part.amax(1).clamp(min=LEAST) / 448
    return out


def spread(scales: torch.Tensor, width: int) -> torch.Tensor:
    """Scales ``[blocks, n]`` as factors ``[n, width]``."""
    return scales.double().t()[:, torch.arange(width) // 128]


def boundary(x, delta=None, pairs=None, slots=None, weights=None) -> torch.Tensor:
    y = x.double().clone()
    if delta is not None:
        y += delta.double()
    if pairs is not None:
        for t in range(slots.shape[0]):
            for j in range(slots.shape[1]):
                if 0 <= slots[t, j] < pairs.shape[0]:
                    y[t] += weights[t, j].double() * pairs[slots[t, j]].double()
    return y


def rms_norm(y: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    return y.double() / torch.sqrt(y.double().square().mean(1, keepdim=True) + eps) * w.double()


def activation(z: torch.Tensor, act: str) -> torch.Tensor:
    z = z.double()
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu_gate":
        half = z.shape[1] // 2
        return z[:, :half] / (1 + torch.exp(-z[:, :half])) * z[:, half:]
    return z


def linear(x, x_scales, w, w_scales) -> tuple[torch.Tensor, torch.Tensor]:
    """The product, and the sums of the magnitudes of its terms."""
    k = x.shape[1]
    a = x.double() * spread(x_scales, k)
    b = w.double() * w_scales.double()[torch.arange(w.shape[0]) // 128][:, torch.arange(k) // 128]
    return a @ b.t(), a.abs() @ b.abs().t()


def route(logits, top, *, score="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0, active=None):
    """ids, weights, slots, segs, token by token."""
    n, experts = logits.shape
    ids, weights = torch.full((n, top), -1, dtype=torch.int64), torch.zeros(n, top, dtype=torch.float64)
    for t in range(n):
        if active is not None and int(active[t]) != 1:
            continue
        l = [-math.inf if math.isnan(v) else min(v, torch.finfo(torch.float32).max) for v in logits[t].double().tolist()]
        if score == "softmax":
            m = max(l)
            e = [0.0 if v == -math.inf else math.exp(v - m) for v in l]
            s = [v / max(sum(e), 1e-300) for v in e]
        else:
            s = [0.0 if v < -709 else 1 / (1 + math.exp(-v)) for v in l]
        c = [s[i] + (float(bias[i].double()) if bias is not None else 0.0) for i in range(experts)]
        c = [-math.inf if l[i] == -math.inf or math.isnan(c[i]) else c[i] for i in range(experts)]
        per = experts // groups
        if groups > 1:
            worth = []
            for g in range(groups):
                there = sorted((v for v in c[g * per: (g + 1) * per] if v > -math.inf), reverse=True)[:2]
                worth.append(sum(there) if there else -math.inf)
            kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:top_groups]
            c = [c[i] if i // per in kept else -math.inf for i in range(experts)]
        order = [i for i in sorted(range(experts), key=lambda i: (-c[i], i)) if c[i] > -math.inf][:top]
        total = sum(s[i] for i in order)
        for j, i in enumerate(order):
            ids[t, j] = i
            weights[t, j] = (s[i] / total if total > 0 else 0.0) * scale if renormalize else s[i] * scale
    slots, segs, at = torch.full((n, top), -1, dtype=torch.int64), [], 0
    for e in range(experts):
        where = [(t, j) for t in range(n) for j in range(top) if ids[t, j] == e] if n * top * experts < 2_000_000 else (ids == e).nonzero().tolist()
        segs.append((at, len(where)))
        for r, (t, j) in enumerate(where):
            slots[t, j] = at + r
        at += -(-len(where) // 8) * 8
    return ids, weights, slots, torch.tensor(segs)
