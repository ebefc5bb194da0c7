"""Experts chosen by scores (CUDA): scores, bias, groups and the best few, and the rows of the matrix sorted by expert.

The route is what :func:`.experts.experts_forward` takes; its weights go to the layer boundary (:func:`.fp8.rms_residual_fp8`).  Where a token's id names its
experts, :class:`.experts.ExpertRouter` routes."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib
from .dense import _call, _f32, _ptr
from .experts import LayerRoute
from .fp8 import one_device

_SCORES = {"softmax": _lib.SCORE_SOFTMAX, "sigmoid": _lib.SCORE_SIGMOID}
MAX_EXPERTS, MAX_TOP = 1024, 32


@dataclass
class ScoreRoute(LayerRoute):
    ids: torch.Tensor
    """int32 ``[n, top]``: the experts of a token, the best first, -1 where there are no more."""
    weights: torch.Tensor
    """fp32 ``[n, top]``."""


def route_by_scores(logits: torch.Tensor, top: int, *, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1, top_groups: int = 1,
                    renormalize: bool = True, scale: float = 1.0, active: torch.Tensor | None = None) -> ScoreRoute:
    """The ``top`` experts of every row of ``logits [n, experts]`` (fp32 or bf16, unit column stride).

    ``s = softmax(logits)`` or ``sigmoid(logits)``; the choice goes by ``c = s + bias``, the weights are ``s`` of the chosen, divided by their sum with
    ``renormalize``, times ``scale``.  ``groups > 1``: experts lie in that many equal runs, a run counts the sum of its best two ``c``, and only the best
    ``top_groups`` runs stay.  Equal ones go by index, comparisons have the outcome of 64-bit arithmetic.  An expert whose logit or ``c`` is NaN or
    -infinity is never chosen; rows whose ``active`` (int32 ``[n]``) is not 1, and choices that are left over, get id -1, weight 0 and slot -1.
    Slots are handed out in the order of the rows, so they do not depend on timing."""
    _lib.require_cuda(logits, "route_by_scores logits")
    if logits.ndim != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or logits.shape[1] < 1 or (logits.shape[1] > 1 and logits.stride(1) != 1) \
            or (logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]):
        raise ValueError("logits must be [n, experts], fp32 or bf16, with unit column stride")
    n, experts = logits.shape
    if score not in _SCORES:
        raise ValueError(f"unknown score {score!r} (known: {', '.join(_SCORES)})")
    if experts > MAX_EXPERTS or not 1 <= top <= MAX_TOP:
        raise ValueError(f"at most {MAX_EXPERTS} experts and 1 to {MAX_TOP} of them a token")
    if groups < 1 or experts % groups or not 1 <= top_groups <= groups:
        raise ValueError("experts must be a multiple of groups, top_groups one of them to all")
    if top > experts // groups * top_groups:
        raise ValueError(f"{top} experts of {top_groups} groups of {experts // groups}")
    _f32(bias, "bias", experts)
    if active is not None and (active.dtype != torch.int32 or active.numel() != n or not active.is_contiguous()):
        raise ValueError("active must be contiguous int32 [n]")
    device = logits.device
    one_device(device, bias, active)
    lib = _lib.load()
    ids, slots, bits = torch.empty((3, n, top), dtype=torch.int32, device=device).unbind(0)  # one allocation: it costs more than a launch
    weights = bits.view(torch.float32)
    segs = torch.empty((experts, 2), dtype=torch.int32, device=device)
    need = int(lib.spk_route_scores_workspace_bytes(n, experts))
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    a = _lib.RouteScoresArgs(
        logits=logits.data_ptr(), bias=_ptr(bias), active=_ptr(active), ids=ids.data_ptr(), weights=weights.data_ptr(), slots=slots.data_ptr(),
        segs=segs.data_ptr(), workspace=_ptr(ws), workspace_bytes=need, logits_stride=max(experts, logits.stride(0)), n=n,
        dtype=_lib.dtype_code(logits.dtype), experts=experts, top=top, groups=groups, top_groups=top_groups, score=_SCORES[score],
        renormalize=renormalize, scale=scale)
    _call("spk_route_scores", a, device)
    return ScoreRoute(slots, segs, ids, weights)
