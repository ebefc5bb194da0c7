"""CPU: host checks of the 8-bit operators and of the experts chosen by scores; the oracle against closed forms.  No call here launches a kernel."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from oracle import fp8_oracle as fo
from spikeinfer_b200 import _lib
from spikeinfer_b200.kernels import fp8 as k8
from spikeinfer_b200.kernels import routing as kr

ROOT = Path(__file__).resolve().parent.parent


def test_argument_structs_have_the_header_layout(tmp_path):
    names = {"spk_rms_residual_fp8_args": _lib.RmsResidualFp8Args, "spk_quantize_fp8_args": _lib.QuantizeFp8Args, "spk_linear_fp8_args": _lib.LinearFp8Args,
             "spk_route_scores_args": _lib.RouteScoresArgs}
    lines = [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for c, s in names.items() for f, _ in s._fields_]
    lines += [f'printf("{c} %zu\\n", sizeof({c}));' for c in names]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "spikeinfer_b200.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    for c, s in names.items():
        assert int(got[c]) == ctypes.sizeof(s)
        for f, _ in s._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(s, f).offset, (c, f)


def refuses(fn, args, code, **changed):
    for k, v in changed.items():
        setattr(args, k, v)
    assert fn(ctypes.byref(args), None) == code, changed


def test_boundary_arguments(lib):
    fn = lib.spk_rms_residual_fp8
    new = lambda: _lib.RmsResidualFp8Args(x=256, w=256, q=256, scales=256, n=4, width=40, q_stride=48, scale_stride=4, x_dtype=_lib.F32)
    assert fn(None, None) == -4
    refuses(fn, new(), 0, n=0, scale_stride=0)
    for code, changed in ((-2, dict(n=-1)), (-2, dict(width=0)), (-2, dict(width=1 << 16)), (-2, dict(scale_stride=3)), (-1, dict(x_dtype=_lib.F16)),
                          (-1, dict(delta=256, delta_dtype=_lib.F16)), (-1, dict(x_dtype=_lib.BF16, delta=256, delta_dtype=_lib.F32)), (-1, dict(out=256, out_dtype=_lib.U8)),
                          (-3, dict(q_stride=40)), (-3, dict(q_stride=32)), (-3, dict(q=264)), (-4, dict(x=None)), (-4, dict(w=None)), (-4, dict(scales=None)),
                          (-4, dict(pairs=256, pair_top=2, pair_rows=8)), (-2, dict(pairs=256, pair_slots=256, pair_weights=256, pair_rows=8)),
                          (-2, dict(pairs=256, pair_slots=256, pair_weights=256, pair_top=1)), (-7, dict(n=1 << 32, scale_stride=1 << 32))):
        refuses(fn, new(), code, **changed)


def test_quantize_arguments(lib):
    fn = lib.spk_quantize_fp8
    new = lambda: _lib.QuantizeFp8Args(z=256, q=256, scales=256, z_stride=80, q_stride=48, scale_stride=4, n=4, width=40, act=_lib.ACT_SILU_GATE, dtype=_lib.F32)
    assert fn(None, None) == -4
    refuses(fn, new(), 0, n=0)
    for code, changed in ((-2, dict(n=-1)), (-2, dict(width=0)), (-2, dict(scale_stride=3)), (-3, dict(z_stride=79)), (-3, dict(q_stride=47)), (-3, dict(q=8)),
                          (-1, dict(dtype=_lib.F16)), (-6, dict(act=3)), (-6, dict(act=-1)), (-4, dict(z=None)), (-4, dict(scales=None))):
        refuses(fn, new(), code, **changed)


def test_linear_arguments(lib):
    fn = lib.spk_linear_fp8
    new = lambda: _lib.LinearFp8Args(x=256, w=256, x_scales=256, w_scales=256, out=256, x_stride=208, w_stride=208, x_scale_stride=4, w_scale_stride=2, out_stride=9,
                                     n=4, k=200, features=9, out_dtype=_lib.BF16)
    assert fn(None, None) == -4
    refuses(fn, new(), 0, n=0)
    for code, changed in ((-2, dict(n=-1)), (-2, dict(k=0)), (-2, dict(features=0)), (-3, dict(x_stride=200)), (-3, dict(w_stride=192)), (-3, dict(x=264)), (-3, dict(w=8)),
                          (-3, dict(x_scale_stride=3)), (-3, dict(w_scale_stride=1)), (-3, dict(out_stride=8)), (-1, dict(out_dtype=_lib.F16)), (-4, dict(x=None)),
                          (-4, dict(out=None)), (-4, dict(w_scales=None)), (-7, dict(n=1 << 31, x_scale_stride=1 << 31))):
        refuses(fn, new(), code, **changed)


def test_route_arguments(lib):
    fn = lib.spk_route_scores
    assert lib.spk_route_scores_workspace_bytes(0, 8) == 0 and lib.spk_route_scores_workspace_bytes(400, 8) >= 13 * 8 * 4
    new = lambda: _lib.RouteScoresArgs(logits=256, ids=256, weights=256, slots=256, segs=256, workspace=256, workspace_bytes=1 << 20, logits_stride=64, n=400, dtype=_lib.F32,
                                       experts=64, top=6, groups=8, top_groups=2, score=_lib.SCORE_SIGMOID, renormalize=1, scale=1.0)
    assert fn(None, None) == -4
    for code, changed in ((-2, dict(n=-1)), (-2, dict(experts=0)), (-2, dict(experts=2048)), (-2, dict(top=0)), (-2, dict(top=33)), (-2, dict(groups=7)), (-2, dict(groups=0)),
                          (-2, dict(top_groups=0)), (-2, dict(top_groups=9)), (-2, dict(top=17)), (-1, dict(dtype=_lib.F16)), (-6, dict(score=2)), (-7, dict(n=1 << 25)),
                          (-4, dict(logits=None)), (-4, dict(ids=None)), (-4, dict(segs=None)), (-3, dict(logits_stride=63)), (-5, dict(workspace=None)),
                          (-5, dict(workspace_bytes=8))):
        refuses(fn, new(), code, **changed)


def test_operators_refuse_cpu_tensors():
    x, w = torch.zeros(2, 32), torch.zeros(2, 32).to(torch.float8_e4m3fn)
    for call in (lambda: k8.rms_residual_fp8(x, torch.ones(32), eps=1e-5), lambda: k8.quantize_fp8(x), lambda: k8.linear_fp8(w, torch.ones(1, 2), w, torch.ones(1, 1)),
                 lambda: kr.route_by_scores(x, 2)):
        with pytest.raises(_lib.SpkError):
            call()


def test_oracle_against_closed_forms():
    assert fo.e4m3_step(torch.tensor([1.0, 1.9, 2.0, 256.0, 2.0 ** -6, 2.0 ** -7, 0.0])).tolist() == [0.125, 0.125, 0.25, 32.0, 2.0 ** -9, 2.0 ** -9, 2.0 ** -9]
    q, s = k8.quantize_weight(torch.eye(200) * 3)
    assert q[5, 5].float() == 448 and q[150, 150].float() == 448 and float(s[0, 0]) == pytest.approx(3 / 448) and float(s[0, 1]) == pytest.approx(2.0 ** -100 / 448)
    ids, weights, slots, segs = fo.route(torch.tensor([[0.0, 1.0, 1.0], [5.0, -float("inf"), 0.0]]), 2)
    assert ids.tolist() == [[1, 2], [0, 2]] and weights[0].tolist() == [0.5, 0.5] and slots.tolist() == [[8, 16], [0, 17]] and segs.tolist() == [[0, 1], [8, 1], [16, 2]]
    ids, *_ = fo.route(torch.tensor([[9.0, -9.0, 3.0, 3.0]]), 2, score="sigmoid", groups=2, top_groups=1)
    assert ids.tolist() == [[2, 3]]
    out, size = fo.linear(torch.ones(1, 130).to(torch.float8_e4m3fn), torch.tensor([[2.0], [3.0]]), (-torch.ones(1, 130)).to(torch.float8_e4m3fn), torch.tensor([[5.0, 7.0]]))
    assert float(out) == -(128 * 10 + 2 * 21) and float(size) == 128 * 10 + 2 * 21
