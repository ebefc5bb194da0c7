"""Operators in 8 bits (CUDA): layer boundary, activation and product with e4m3 values.

Activations are e4m3 ``[n, width]`` with fp32 scales ``[ceil(width / 128), n]``, one for every row and 128 columns; weights are e4m3 ``[features, k]`` with
fp32 scales ``[ceil(features / 128), ceil(k / 128)]``, one for every block of 128 x 128.  A value stands for ``value * scale``.  Rows start on
16-byte boundaries: a width that is no multiple of 16 is a view of a wider matrix (:func:`rows_fp8`).  The kernels are in the full library
(``python -m spikeinfer_b200.build``), not in those that serve one model from a fresh checkout."""
from __future__ import annotations

import torch

from .. import _lib
from .dense import _call, _f32, _ptr

FP8 = torch.float8_e4m3fn
BLOCK = 128
_F32, _BF16 = torch.float32, torch.bfloat16
_FLOATS = (_F32, _BF16)
_ACTS = {"none": _lib.ACT_NONE, "gelu_tanh": _lib.ACT_GELU_TANH, "silu_gate": _lib.ACT_SILU_GATE}


def rows_fp8(n: int, width: int, device) -> torch.Tensor:
    """An e4m3 ``[n, width]`` matrix, not filled, whose rows start on 16-byte boundaries."""
    return torch.empty_strided((n, width), (-(-width // 16) * 16, 1), dtype=FP8, device=device)


def _scales(n: int, width: int, device) -> torch.Tensor:
    return torch.empty_strided((-(-width // BLOCK), n), (n, 1), dtype=_F32, device=device)


def _row_stride(t: torch.Tensor, what: str) -> int:
    if t.ndim == 2 and t.dtype is FP8:
        (row, column), (n, width) = t.stride(), t.shape
        if n <= 1 or width == 1:  # torch gives an axis of one any stride
            row, column = row if n > 1 else -(-width // 16) * 16, 1 if width == 1 else column
        if column == 1 and row >= width > 0 and not row % 16 and not t.data_ptr() % 16:
            return row
    raise ValueError(f"{what} must be e4m3 [rows, columns] with unit column stride and rows that start on 16-byte boundaries")


def one_device(device: torch.device, *tensors: torch.Tensor | None) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"all tensors must be on {device}: one is on {t.device}")


@torch.no_grad()
def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A weight matrix ``[features, k]`` as e4m3 values and scales for blocks of 128 x 128, for :func:`linear_fp8`; done once, when a model is loaded.  As in the
    activations, NaN stays NaN and is not the largest of its block, and an infinity counts as the largest finite value."""
    f, k = w.shape
    fb, kb = -(-f // BLOCK), -(-k // BLOCK)
    x = w.new_zeros((fb * BLOCK, kb * BLOCK), dtype=torch.float32)
    x[:f, :k] = w
    x = x.view(fb, BLOCK, kb, BLOCK)
    most = x.abs().nan_to_num_(nan=0.0, posinf=torch.finfo(torch.float32).max).amax(dim=(1, 3))
    scales = most.clamp(min=2.0 ** -100) / 448.0
    out = rows_fp8(f, k, w.device)
    out.copy_((x / scales[:, None, :, None]).clamp(-448.0, 448.0).view(fb * BLOCK, kb * BLOCK)[:f, :k])
    return out, scales.contiguous()


def rms_residual_fp8(x: torch.Tensor, weight: torch.Tensor, *, eps: float, delta: torch.Tensor | None = None, x_out: torch.Tensor | None = None,
                     pairs: torch.Tensor | None = None, pair_slots: torch.Tensor | None = None, pair_weights: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One layer boundary: ``y = x + delta + sum_j pair_weights[t, j] * pairs[pair_slots[t, j]]`` in the dtype of ``x``, to ``x_out`` (may be ``x``);
    returns ``rmsnorm(y) * weight`` as e4m3 values and scales, and writes it to ``out`` (fp32 or bf16) where given.  Up to 32768 columns.

    ``x`` is fp32 (``delta`` fp32 or bf16) or bf16 (``delta`` bf16), ``pairs`` what :func:`.experts.experts_forward` returned, ``pair_slots`` and
    ``pair_weights`` a route's (:func:`.routing.route_by_scores`); a negative slot adds nothing."""
    _lib.require_cuda(x, "rms_residual_fp8 input")
    if x.ndim != 2 or not x.is_contiguous() or x.dtype not in _FLOATS:
        raise ValueError("x must be contiguous [n, width], fp32 or bf16")
    n, width = x.shape
    _f32(weight, "weight", width)
    if delta is not None and (delta.shape != x.shape or not delta.is_contiguous()
                              or delta.dtype not in (_FLOATS if x.dtype == _F32 else (_BF16,))):
        raise ValueError("delta must be contiguous and of the shape of x, fp32 or bf16 beside fp32, bf16 beside bf16")
    if x_out is not None and (x_out.shape != x.shape or x_out.dtype != x.dtype or not x_out.is_contiguous()):
        raise ValueError("x_out must be contiguous, of the shape and dtype of x")
    if out is not None and (out.shape != x.shape or out.dtype not in _FLOATS or not out.is_contiguous()):
        raise ValueError("out must be contiguous and of the shape of x, fp32 or bf16")
    if pairs is None and (pair_slots is not None or pair_weights is not None):
        raise ValueError("pair_slots and pair_weights name rows of pairs")
    if pairs is not None:
        _f32(pairs, "pairs")
        if pairs.ndim != 2 or pairs.shape[1] != width or pairs.shape[0] < 1:
            raise ValueError("pairs must be [rows, width]")
        if pair_slots is None or pair_slots.ndim != 2 or pair_slots.shape[0] != n or pair_slots.shape[1] < 1 or pair_slots.dtype != torch.int32 \
                or not pair_slots.is_contiguous():
            raise ValueError("pair_slots must be contiguous int32 [n, top]")
        if pair_weights is None or pair_weights.shape != pair_slots.shape:
            raise ValueError("pair_weights must be [n, top]")
        _f32(pair_weights, "pair_weights")
    device = x.device
    one_device(device, weight, delta, x_out, out, pairs, pair_slots, pair_weights, status)
    q, scales = rows_fp8(n, width, device), _scales(n, width, device)
    a = _lib.RmsResidualFp8Args(
        x=x.data_ptr(), delta=_ptr(delta), x_out=_ptr(x_out), w=weight.data_ptr(), pairs=_ptr(pairs), pair_slots=_ptr(pair_slots),
        pair_weights=_ptr(pair_weights), out=_ptr(out), q=q.data_ptr(), scales=scales.data_ptr(), pair_rows=0 if pairs is None else pairs.shape[0], n=n,
        width=width, q_stride=q.stride(0), scale_stride=n, pair_top=0 if pairs is None else pair_slots.shape[1], x_dtype=_lib.dtype_code(x.dtype),
        delta_dtype=0 if delta is None else _lib.dtype_code(delta.dtype), out_dtype=0 if out is None else _lib.dtype_code(out.dtype), eps=eps,
        status=_ptr(status))
    _call("spk_rms_residual_fp8", a, x.device)
    return q, scales


def quantize_fp8(z: torch.Tensor, act: str = "none") -> tuple[torch.Tensor, torch.Tensor]:
    """``act(z)`` as e4m3 values and scales: ``"none"``, ``"gelu_tanh"``, or ``"silu_gate"`` (``silu(z[:, :w]) * z[:, w:]``).  ``z`` is fp32 or bf16 with
    unit column stride."""
    _lib.require_cuda(z, "quantize_fp8 input")
    if act not in _ACTS:
        raise ValueError(f"unknown activation {act!r} (known: {', '.join(_ACTS)})")
    if z.ndim != 2 or z.dtype not in _FLOATS or z.shape[1] < 1 or (z.shape[1] > 1 and z.stride(1) != 1) or (z.shape[0] > 1 and z.stride(0) < z.shape[1]) \
            or (act == "silu_gate" and z.shape[1] % 2):
        raise ValueError("z must be [n, width], fp32 or bf16, with unit column stride; an even width for the gate")
    n, width = z.shape[0], z.shape[1] // (2 if act == "silu_gate" else 1)
    q, scales = rows_fp8(n, width, z.device), _scales(n, width, z.device)
    a = _lib.QuantizeFp8Args(z=z.data_ptr(), q=q.data_ptr(), scales=scales.data_ptr(), z_stride=max(z.shape[1], z.stride(0)), q_stride=q.stride(0), scale_stride=n, n=n,
                             width=width, act=_ACTS[act], dtype=_lib.dtype_code(z.dtype))
    _call("spk_quantize_fp8", a, z.device)
    return q, scales


def linear_fp8(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *, out_dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """``x w^T`` of e4m3 rows ``[n, k]`` and weights ``[features, k]`` with their scales, 32-bit sums, in ``out_dtype`` (fp32 or bf16).  ``out`` may be a column
    range of a row-major matrix."""
    _lib.require_cuda(x, "linear_fp8 input")
    x_stride, w_stride = _row_stride(x, "x"), _row_stride(w, "w")
    (n, k), features = x.shape, w.shape[0]
    blocks = -(-k // BLOCK)
    if w.shape[1] != k or features < 1:
        raise ValueError(f"w is {tuple(w.shape)}, x has {k} columns")
    if x_scales.dtype != torch.float32 or x_scales.shape != (blocks, n) or (n > 1 and x_scales.stride(1) != 1) or (blocks > 1 and x_scales.stride(0) < n):
        raise ValueError("x_scales must be fp32 [ceil(k / 128), n] with unit stride along the rows")
    if w_scales.dtype != torch.float32 or w_scales.shape != (-(-features // BLOCK), blocks) or not w_scales.is_contiguous():
        raise ValueError("w_scales must be contiguous fp32 [ceil(features / 128), ceil(k / 128)]")
    if out is None:
        out = torch.empty((n, features), dtype=out_dtype, device=x.device)
    if out.shape != (n, features) or out.dtype != out_dtype or out_dtype not in _FLOATS or (features > 1 and out.stride(1) != 1) \
            or (n > 1 and out.stride(0) < features):
        raise ValueError("out must be [n, features] in out_dtype, fp32 or bf16, with unit column stride")
    one_device(x.device, x_scales, w, w_scales, out, status)
    a = _lib.LinearFp8Args(x=x.data_ptr(), w=w.data_ptr(), x_scales=x_scales.data_ptr(), w_scales=w_scales.data_ptr(), out=out.data_ptr(),
                           x_stride=x_stride, w_stride=w_stride, x_scale_stride=max(n, x_scales.stride(0)), w_scale_stride=blocks,
                           out_stride=max(features, out.stride(0)), n=n, k=k, features=features, out_dtype=_lib.dtype_code(out_dtype),
                           status=_ptr(status))
    _call("spk_linear_fp8", a, x.device)
    return out
