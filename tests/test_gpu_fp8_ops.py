"""GPU: the 8-bit operators and the experts chosen by scores, each alone, against plain forms in float64.

Tolerances count roundings: u = 2^-24 is half a step of fp32, 2^-8 of bf16, 2^-4 of e4m3."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8_oracle as fo
from spikeinfer_b200 import _lib
from spikeinfer_b200.kernels import dense as kn
from spikeinfer_b200.kernels import experts as ke
from spikeinfer_b200.kernels import fp8 as k8
from spikeinfer_b200.kernels import routing as kr

pytestmark = pytest.mark.gpu
F32, BF, FP8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -24
HALF = {F32: U, BF: 2.0 ** -8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def holds8(q, scales, v, rel):
    """q and scales are the 8-bit form of v, known to a relative error of `rel`."""
    v = v.double().cpu()
    width = v.shape[1]
    want = fo.block_scales(v)
    assert q.dtype == FP8 and q.shape == v.shape and scales.shape == want.shape and scales.dtype == F32
    assert ((scales.double().cpu() - want).abs() <= (rel + 2 * U) * want).all()
    s = fo.spread(scales.cpu(), width)
    got = q.cpu().double()
    off = (got * s - v).abs()
    # half a step of the quotient, whose own error (that of v, two roundings) can reach over the middle between two values
    assert (off <= (0.5 * fo.e4m3_step(v / s) + (rel + 4 * U) * 512) * s).all()
    assert ((off <= 0.5 * fo.e4m3_step(v / s) * s * (1 + 64 * U) + (rel + 4 * U) * v.abs())).all()
    for b in range(want.shape[0]):  # the largest of a block is 448
        there = want[b] > fo.LEAST / 448
        assert (got[:, 128 * b: 128 * b + 128].abs().amax(1)[there] == 448).all()


# ---- boundary --------------------------------------------------------------------------------------------------------
# v = y * rms * w: a sum of squares over at most 21 roundings a term, its root half of that, and five more: 16 u
NORM = 16 * U


@pytest.mark.parametrize("stream,delta_dtype", [(F32, F32), (F32, BF), (F32, None), (BF, BF), (BF, None)])
@pytest.mark.parametrize("n,width,top", [(1, 1, 0), (1, 45, 1), (37, 88, 3), (5, 129, 0), (3, 896, 0), (2, 1022, 2), (64, 3584, 2), (7, 1028, 6), (3, 9001, 2),
                                         (2, 32768, 1), (700, 256, 0), (601, 1030, 2), (600, 900, 0), (593, 1004, 0), (640, 2056, 0)])
def test_boundary(dev, n, width, top, stream, delta_dtype):
    g = gen(n * 7 + width)
    rnd = lambda *s: torch.randn(*s, generator=g)
    x, w, eps = rnd(n, width).to(stream), 1 + 0.3 * rnd(width), 1e-5
    delta = None if delta_dtype is None else rnd(n, width).to(delta_dtype)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    args, more = {}, 0.0
    if top:
        rows = n * top + 5
        slots = torch.randperm(rows, generator=g)[: n * top].view(n, top).to(torch.int32)
        slots[torch.rand(n, top, generator=g) < 0.2] = -1
        pairs, weights = rnd(rows, width), torch.rand(n, top, generator=g)
        pairs[[r for r in range(rows) if r not in set(slots.flatten().tolist())]] = float("nan")
        args = dict(pairs=pairs, slots=slots, weights=weights)
        more = fo.boundary(torch.zeros(n, width), None, pairs.abs(), slots, weights)
    y = fo.boundary(x, delta, **args)
    size = x.double().abs() + (0 if delta is None else delta.double().abs()) + more
    d = lambda t: None if t is None else t.to(dev)
    on = dict(pairs=d(args["pairs"]), pair_slots=d(args["slots"]), pair_weights=d(args["weights"])) if top else {}
    x_out = torch.full((n, width), 7.0, dtype=stream, device=dev)
    for out_dtype in (BF, F32):
        out = torch.full((n, width), 7.0, dtype=out_dtype, device=dev)
        xd = d(x)
        q, scales = k8.rms_residual_fp8(xd, d(w), eps=eps, delta=d(delta), x_out=x_out, out=out, status=status, **on)
        assert torch.equal(xd, d(x))
        assert ((x_out.double().cpu() - y).abs() <= (top + 2) * U * size + (HALF[BF] * (y.abs() + 2 * U * size) if stream == BF else 0)).all()
        v = fo.rms_norm(x_out.cpu(), w, eps)  # of what is stored
        assert ((out.double().cpu() - v).abs() <= (NORM + HALF[out_dtype]) * (1 + 2 * U) * v.abs()).all()
        holds8(q, scales, v, NORM)
    # in place, without the plain output: the same bits
    xd = d(x)
    q2, s2 = k8.rms_residual_fp8(xd, d(w), eps=eps, delta=d(delta), x_out=xd, status=status, **on)
    assert torch.equal(xd, x_out) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, scales)
    # and without keeping the sum
    q2, s2 = k8.rms_residual_fp8(d(x), d(w), eps=eps, delta=d(delta), status=status, **on)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, scales)
    assert int(status.item()) == 0


def test_boundary_of_matrices_at_odd_places(dev):
    """Views that begin off every boundary but their own elements', many rows and few: the bits of aligned ones."""
    for n, width in ((700, 512), (5, 512)):
        for stream, delta_dtype in ((F32, F32), (F32, BF), (BF, BF)):
            place = lambda t, off: torch.empty(t.numel() + off, dtype=t.dtype, device=dev)[off:].view(t.shape).copy_(t)
            x, delta, w = torch.randn(n, width, device=dev).to(stream), torch.randn(n, width, device=dev).to(delta_dtype), torch.rand(width, device=dev)
            run = lambda x, delta, w, x_out, out: (x_out, out, *k8.rms_residual_fp8(x, w, eps=1e-5, delta=delta, x_out=x_out, out=out))
            want = run(x, delta, w, torch.empty_like(x), torch.empty(n, width, dtype=BF, device=dev))
            for offs in ((1, 0, 0, 0, 0), (0, 1, 0, 0, 0), (0, 0, 1, 0, 0), (0, 0, 0, 1, 0), (0, 0, 0, 0, 1), (2, 2, 2, 2, 2), (4, 4, 4, 4, 4), (0, 4, 0, 0, 0)):
                got = run(*(place(t, o) for t, o in zip((x, delta, w, want[0], want[1]), offs)))
                v = fo.rms_norm(got[0].cpu(), w.cpu(), 1e-5)
                assert torch.equal(got[0], want[0])
                assert ((got[1].double().cpu() - v).abs() <= (NORM + HALF[BF]) * (1 + 2 * U) * v.abs()).all()
                holds8(got[2], got[3], v, NORM)


def test_boundary_reports_slots_that_do_not_exist(dev):
    x, w = torch.randn(4, 64, device=dev), torch.ones(64, device=dev)
    pairs, weights = torch.randn(8, 64, device=dev), torch.ones(4, 2, device=dev)
    slots = torch.tensor([[0, 1], [8, 2], [-1, -5], [3, 2 ** 30]], dtype=torch.int32, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    x_out = torch.empty_like(x)
    k8.rms_residual_fp8(x, w, eps=1e-5, x_out=x_out, pairs=pairs, pair_slots=slots, pair_weights=weights, status=status)
    assert int(status.item()) == _lib.STATUS_BAD_SLOT
    want = fo.boundary(x.cpu(), None, pairs.cpu(), slots.cpu(), weights.cpu())
    assert ((x_out.double().cpu() - want).abs() <= 4 * U * 10).all()


def test_values_that_are_not_finite_and_blocks_of_nothing(dev):
    z = torch.zeros(6, 300)
    z[0, 3], z[0, 200] = float("nan"), 2.0
    z[1, 5], z[1, 6], z[1, 140] = float("inf"), 1.0, -float("inf")
    z[2, :128] = float("nan")
    z[3, 17] = 1e-35
    z[4, 0], z[4, 1] = 3e38, 1e30
    z[5, 299] = -5.0
    q, s = k8.quantize_fp8(z.to(dev))
    q, s = q.double().cpu(), s.double().cpu()
    top = torch.finfo(torch.float32).max
    assert q[0, 3].isnan() and int(q.isnan().sum()) == 129
    assert abs(float(s[0, 1]) / (top / 448) - 1) < 4 * U and q[1, 5] == 448 and q[1, 6] == 0 and q[1, 140] == -448
    assert q[2, :128].isnan().all() and (s[0, [0, 2, 3, 5]] == torch.tensor(2.0 ** -100 / 448, dtype=F32).double()).all()
    assert q[4, 0] == 448 and q[4, 1] == 0 and q[5, 299] == -448 and q[0, 200] == 448
    assert torch.isfinite(s).all() and (s > 0).all()


# ---- activations -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["none", "gelu_tanh", "silu_gate"])
@pytest.mark.parametrize("n,width,pad", [(1, 1, 0), (3, 45, 3), (37, 4864, 0), (130, 896, 8), (5, 1021, 1), (2, 18944, 0), (65, 128, 0), (33, 130, 2)])
def test_quantize(dev, n, width, pad, act, dtype):
    z = 3 * torch.randn(n, width * (2 if act == "silu_gate" else 1), generator=gen(n + width)).to(dtype)
    big = torch.full((n, z.shape[1] + pad), float("nan"), dtype=dtype, device=dev)
    view = big[:, pad // 2: pad // 2 + z.shape[1]]
    view.copy_(z)
    q, scales = k8.quantize_fp8(view, act)
    v = fo.activation(z, act)
    # the exponential and what stands in its exponent (|z| <= 18: its three roundings and the function's 2 ulp at up to 200), the quotient and the product
    rel = 0.0 if act == "none" else (1300 if act == "gelu_tanh" else 64) * U
    want = fo.block_scales(v)
    assert ((scales.double().cpu() - want).abs() <= (rel + 2 * U) * want).all()
    s = fo.spread(scales.cpu(), width)
    off = (q.double().cpu() * s - v).abs()
    # far tails of the gelu are off by more; under 1e-4 of its block's largest a value is under 0.0448 of the scale, so under 2^-4, where half a step is 2^-9 or less
    keep = v.abs() > 1e-4 * 448 * s
    assert (off <= 0.5 * fo.e4m3_step(v / s) * s * (1 + 64 * U) + (rel + 4 * U) * v.abs())[keep | (act == "none")].all()
    assert (off <= 1.01 * 2.0 ** -9 * s)[~keep].all()


# ---- products --------------------------------------------------------------------------------------------------------
def operands(n, k, f, dev, seed, pad=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x, w = (torch.full((r, -(-k // 16) * 16 + 16 * pad), float("nan"), device=dev).to(FP8)[:, :k] for r in (n, f))  # NaN behind the columns
    x.copy_((150 * torch.randn(n, k, generator=g, device=dev)).clamp(-448, 448))
    w.copy_((150 * torch.randn(f, k, generator=g, device=dev)).clamp(-448, 448))
    blocks = -(-k // 128)
    sx = torch.exp2(4 * torch.randn(blocks, n + pad, generator=g, device=dev))[:, :n]  # a row's blocks differ by a lot: a scale at the wrong place shows
    sw = torch.exp2(2 * torch.randn(-(-f // 128), blocks, generator=g, device=dev))
    return x, sx, w, sw


def check_linear(out, x, sx, w, sw):
    want, size = fo.linear(x.cpu(), sx.cpu(), w.cpu(), sw.cpu())
    # products are exact.  A tensor-core step adds 32 of them and the sum so far, each cut to 23 bits or more of the largest: 4 steps of 33 terms within
    # 2^-23 of the block's magnitudes; then a product of scales, a product with it and a sum per block
    tol = (132 * 2.0 ** -23 + (3 + -(-x.shape[1] // 128)) * U) * size
    off = (out.double().cpu() - want).abs()
    assert (off <= tol + HALF[out.dtype] * (want.abs() + tol)).all(), float((off / size.clamp(min=1e-300)).max())


SIZES = [(1, 16, 1), (1, 45, 7), (1, 128, 128), (3, 129, 130), (1, 896, 4864), (16, 256, 300), (17, 384, 129), (31, 1000, 257), (33, 640, 200), (64, 3584, 896),
         (65, 128, 512), (100, 4864, 130), (128, 512, 128), (129, 1021, 255), (200, 2048, 1000), (300, 1152, 640), (513, 300, 777), (1171, 4864, 896), (5, 2100, 300), (64, 2050, 900), (20, 1100, 2000), (130, 2100, 200), (90, 2304, 1100),
         (2600, 260, 4000), (2563, 130, 4111)]


@pytest.mark.parametrize("out_dtype", [BF, F32])
@pytest.mark.parametrize("n,k,f", SIZES)
def test_linear(dev, n, k, f, out_dtype):
    x, sx, w, sw = operands(n, k, f, dev, n + k + f)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = k8.linear_fp8(x, sx, w, sw, out_dtype=out_dtype, status=status)
    check_linear(out, x, sx, w, sw)
    assert torch.equal(out, k8.linear_fp8(x, sx, w, sw, out_dtype=out_dtype)) and int(status.item()) == 0


@pytest.mark.parametrize("n,k,f", [(5, 300, 200), (70, 512, 390), (260, 1000, 520)])
def test_linear_into_a_column_range_of_strided_operands(dev, n, k, f):
    x, sx, w, sw = operands(n, k, f, dev, 5, pad=3)
    for dtype in (BF, F32):
        big = torch.full((n + 2, f + 9), 7.0, dtype=dtype, device=dev)
        k8.linear_fp8(x, sx, w, sw, out_dtype=dtype, out=big[1: n + 1, 4: f + 4])
        check_linear(big[1: n + 1, 4: f + 4], x, sx, w, sw)
        big[1: n + 1, 4: f + 4] = 7.0
        assert (big == 7.0).all()


def test_linear_of_single_values(dev):
    """One value of x and one of w at a time: the product lands where it belongs, with its own block's scales."""
    n, k, f = 150, 400, 300
    for t, c, o in [(0, 0, 0), (149, 399, 299), (127, 128, 128), (128, 127, 127), (16, 255, 256), (77, 384, 255)]:
        x, w = k8.rows_fp8(n, k, dev), k8.rows_fp8(f, k, dev)
        x.zero_()
        w.zero_()
        x[t, c], w[o, c] = 3.5, -20.0
        sx = torch.arange(1, 4 * n + 1, device=dev, dtype=F32).view(4, n)
        sw = torch.arange(1, 13, device=dev, dtype=F32).view(3, 4) / 8
        out = k8.linear_fp8(x, sx, w, sw, out_dtype=F32)
        want = torch.zeros(n, f)
        want[t, o] = -70.0 * float(sx[c // 128, t]) * float(sw[o // 128, c // 128])
        assert torch.equal(out.cpu(), want)


def test_linear_rows_do_not_depend_on_their_neighbours(dev):
    x, sx, w, sw = operands(40, 500, 300, dev, 11)
    want = k8.linear_fp8(x, sx, w, sw, out_dtype=F32)
    x[7], x[21, 3] = float("nan"), float("nan")
    sx[:, 9] = float("inf")
    got = k8.linear_fp8(x, sx, w, sw, out_dtype=F32)
    rows = [t for t in range(40) if t not in (7, 21, 9)]
    assert torch.equal(got[rows], want[rows]) and got[7].isnan().all() and got[21].isnan().all() and not torch.isfinite(got[9]).any()


def test_quantized_weights(dev):
    w = torch.randn(300, 200, generator=gen(3)).to(dev)
    w[:128, 128:] = 0
    q, s = k8.quantize_weight(w)
    assert q.shape == (300, 200) and s.shape == (3, 2) and q.stride(0) % 16 == 0
    back = q.double().cpu() * s.double().cpu()[torch.arange(300) // 128][:, torch.arange(200) // 128]
    assert ((back - w.double().cpu()).abs() <= 2.0 ** -4 * (1 + 4 * U) * w.double().cpu().abs() + 2.0 ** -10 * float(s.max())).all()


# ---- routes ----------------------------------------------------------------------------------------------------------
def check_route(r, logits, top, **kw):
    cpu = {k: (v.cpu() if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}
    ids, weights, slots, segs = fo.route(logits.cpu(), top, **cpu)
    assert torch.equal(r.ids.cpu().long(), ids)
    # 32-bit weights: the difference in the exponent (half a step of its size, up to the 88 where the exponential ends), two exponentials (2 ulp each), up to 37 sums of positive terms, their
    # quotient, the sum of up to 32 choices and its quotient, the scale; what lies below the exponential's range is zero
    spread = 88.0
    assert ((r.weights.double().cpu() - weights).abs() <= (spread + 8 + 37 + 1 + 6 + 2) * U * weights + 1e-37 * max(1.0, kw.get("scale", 1.0))).all()
    assert torch.equal(r.slots.cpu().long(), slots) and torch.equal(r.segs.cpu().long(), segs)


ROUTES = [(1, 16, 2, 1, 1), (1, 1, 1, 1, 1), (3, 5, 5, 1, 1), (64, 256, 8, 8, 4), (33, 60, 4, 1, 1), (257, 64, 6, 8, 3), (40, 160, 6, 8, 3), (9, 384, 8, 1, 1), (7, 1024, 32, 1, 1),
          (5, 1024, 16, 32, 2), (300, 8, 2, 4, 2), (31, 12, 2, 12, 5), (65, 100, 7, 4, 2), (1000, 37, 3, 1, 1), (2000, 24, 2, 1, 1)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("score,biased", [("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)])
@pytest.mark.parametrize("n,experts,top,groups,top_groups", ROUTES)
def test_route(dev, n, experts, top, groups, top_groups, score, biased, dtype):
    g = gen(n + experts)
    logits = (2 * torch.randn(n, experts, generator=g)).to(dtype)
    bias = 0.1 * torch.randn(experts, generator=g) if biased else None
    more = dict(score=score, bias=None if bias is None else bias.to(dev), groups=groups, top_groups=top_groups)
    wide = torch.full((n, experts + 3), 99.0, dtype=dtype, device=dev)
    wide[:, 1: experts + 1] = logits.to(dev)
    r = kr.route_by_scores(wide[:, 1: experts + 1], top, **more)
    check_route(r, logits, top, **more)
    r = kr.route_by_scores(logits.to(dev), top, renormalize=False, scale=2.5, **more)
    check_route(r, logits, top, renormalize=False, scale=2.5, **more)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_equal_masked_and_missing_scores(dev, score):
    inf, nan = float("inf"), float("nan")
    logits = torch.zeros(12, 8)
    logits[1] = torch.tensor([1, 2, 2, 1, 2, 1, 2, 0.0])
    logits[2] = -inf
    logits[3, :7] = -inf
    logits[4] = nan
    logits[5] = torch.tensor([nan, 1, -inf, 3, nan, -inf, 2, nan])
    logits[6] = torch.tensor([inf, 0, inf, 0, 0, 0, 0, 0])
    logits[7] = torch.tensor([-inf, -inf, 1, -inf, -inf, -inf, 0.5, -inf])
    logits[8] = -400.0
    logits[9] = torch.tensor([80.0, 81, 82, 83, 84, 85, 86, 87]) / 4  # sigmoids that are all 1 or next to it in 32 bits
    logits[10] = torch.finfo(F32).min
    logits[11] = torch.tensor([1.0, 1.0000001, 1.0000002, 1, 1, 1, 1, 1])
    for bias in (None, torch.tensor([0, -inf, 0, nan, 0.5, inf, 0, 0]), torch.full((8,), -3.0)):
        for groups, top_groups, top in ((1, 1, 4), (4, 2, 4), (2, 1, 3), (8, 3, 3), (4, 4, 8)):
            for active in (None, torch.tensor([1, 0, 1, 1, 2, 1, 1, 1, 1, -1, 1, 1], dtype=torch.int32)):
                more = dict(score=score, groups=groups, top_groups=top_groups, bias=None if bias is None else bias.to(dev), active=None if active is None else active.to(dev))
                check_route(kr.route_by_scores(logits.to(dev), top, **more), logits, top, **more)


def test_route_tells_neighbours_of_64_bits_apart(dev):
    """Scores that are equal in 32 bits and not in 64, and biases that make up for a difference to the last bit but some."""
    g = gen(5)
    base = torch.randn(1, 64, generator=g).expand(200, 64)
    logits = (base + 1e-7 * torch.randn(200, 64, generator=g)).contiguous()
    bias = -torch.sigmoid(base[0].double()).to(F32)
    for groups, top_groups in ((1, 1), (8, 2)):
        more = dict(score="sigmoid", bias=bias.to(dev), groups=groups, top_groups=top_groups)
        check_route(kr.route_by_scores(logits.to(dev), 8, **more), logits, 8, **more)


def test_nothing_is_a_size(dev):
    q, s = k8.rms_residual_fp8(torch.empty(0, 64, device=dev), torch.ones(64, device=dev), eps=1e-5)
    assert q.shape == (0, 64) and s.shape == (1, 0)
    q, s = k8.quantize_fp8(torch.empty(0, 200, dtype=BF, device=dev), "silu_gate")
    assert q.shape == (0, 100) and s.shape == (1, 0)
    x, sx, w, sw = operands(1, 64, 10, dev, 1)
    assert k8.linear_fp8(x[:0], sx[:, :0], w, sw).shape == (0, 10)
    r = kr.route_by_scores(torch.empty(0, 9, device=dev), 3)
    assert r.ids.shape == (0, 3) and torch.equal(r.segs.cpu(), torch.zeros(9, 2, dtype=torch.int32))


# ---- together --------------------------------------------------------------------------------------------------------
def rel(got, want) -> float:
    return float((got.double().cpu() - want).pow(2).mean().sqrt() / want.pow(2).mean().sqrt().clamp(min=1e-30))


class Block:
    """A pre-norm block with an 8-bit dense feed-forward and, beside it, experts chosen by scores."""

    def __init__(self, dev, width=256, ff=384, experts=16, top=3, eff=72, seed=1):
        g = torch.Generator(device=dev).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.width, self.top = width, top
        self.w1, self.w2 = 1 + 0.2 * rnd(width), 1 + 0.2 * rnd(width)
        self.up, self.down = k8.quantize_weight(rnd(ff, width) / width ** 0.5), k8.quantize_weight(rnd(width, ff) / ff ** 0.5)
        self.router, self.bias = rnd(experts, width) / width ** 0.5, 0.05 * rnd(experts)
        self.parts = [[(rnd(*s) / s[1] ** 0.5).to(BF) for _ in range(experts)] for s in ((eff, width), (eff, width), (width, eff))]
        self.experts = ke.ExpertWeights(*self.parts, top=top)

    def run(self, x, delta, status):
        n, s = x.shape[0], {}
        s["x1"], s["h"] = torch.empty_like(x), torch.empty(n, self.width, dtype=BF, device=x.device)
        s["q1"], s["s1"] = k8.rms_residual_fp8(x, self.w1, eps=1e-5, delta=delta, x_out=s["x1"], out=s["h"], status=status)
        s["z"] = k8.linear_fp8(s["q1"], s["s1"], *self.up, status=status)
        s["q2"], s["s2"] = k8.quantize_fp8(s["z"], "gelu_tanh")
        s["ff"] = k8.linear_fp8(s["q2"], s["s2"], *self.down, out_dtype=F32, status=status)
        s["logits"] = s["h"].float() @ self.router.t()
        r = s["route"] = kr.route_by_scores(s["logits"], self.top, score="sigmoid", bias=self.bias, groups=4, top_groups=2)
        rows = self.experts.sorted_matrix(n, self.width)
        kn.rms_residual(x=s["x1"], w2=self.w1, eps=1e-5, out2=rows, out2_slots=r.slots, out2_tiled=self.experts.tiled, status=status)
        s["pairs"] = ke.experts_forward(rows, self.experts, r, status)
        s["x2"] = torch.empty_like(x)
        s["q3"], s["s3"] = k8.rms_residual_fp8(s["x1"], self.w2, eps=1e-5, delta=s["ff"], x_out=s["x2"], pairs=s["pairs"], pair_slots=r.slots, pair_weights=r.weights,
                                               status=status)
        return s


@pytest.mark.parametrize("n", [1, 6, 70, 300])
def test_a_block_of_them(dev, n):
    block = Block(dev)
    g = torch.Generator(device=dev).manual_seed(n)
    x, delta = torch.randn(n, block.width, generator=g, device=dev), torch.randn(n, block.width, generator=g, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    s = block.run(x, delta, status)
    assert int(status.item()) == 0
    c = {k: v.cpu() for k, v in s.items() if isinstance(v, torch.Tensor)}
    holds8(s["q1"], s["s1"], fo.rms_norm(c["x1"], block.w1.cpu(), 1e-5), NORM)
    check_linear(s["z"], s["q1"], s["s1"], *block.up)
    check_linear(s["ff"], s["q2"], s["s2"], *block.down)
    check_route(s["route"], s["logits"], block.top, score="sigmoid", bias=block.bias, groups=4, top_groups=2)
    # the experts' products by token, on the norm as it was rounded for them
    h, r = c["h"].double(), s["route"]
    gates, ups, downs = ([w.double().cpu() for w in part] for part in block.parts)
    want = fo.boundary(c["x1"], c["ff"])
    for t in range(n):
        for j in range(block.top):
            e = int(r.ids[t, j])
            y = h[t] @ gates[e].t()
            want[t] += float(r.weights[t, j]) * ((y / (1 + torch.exp(-y)) * (h[t] @ ups[e].t())).to(BF).double() @ downs[e].t())
    assert rel(s["x2"], want) < 4e-3  # the experts' inner products are rounded to bf16, 2^-8 each at most, and are a part of the sum
    holds8(s["q3"], s["s3"], fo.rms_norm(c["x2"], block.w2.cpu(), 1e-5), NORM)


def test_a_captured_block_and_one_beside_it(dev):
    """A captured block replayed on new inputs, while another stream runs the same operators: both as if alone."""
    block, other = Block(dev, seed=1), Block(dev, seed=2)
    new = lambda n, seed: torch.randn(n, block.width, generator=torch.Generator(device=dev).manual_seed(seed), device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    n = 300
    x, delta = new(n, 1), new(n, 2)
    block.run(x, delta, status)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = block.run(x, delta, status)
    keep = ("x2", "q3", "s3", "ff", "pairs")
    bits = lambda t: t.contiguous().view(torch.uint8)
    alone = {}
    for seed in (5, 6):
        alone[seed] = {k: v.clone() for k, v in block.run(new(n, seed), new(n, seed + 50), status).items() if k in ("x2", "q3", "s3", "ff")}
    y = new(40, 9), new(40, 10)
    quiet = other.run(*y, status)["x2"].clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for seed in (5, 6, 5):
        x.copy_(new(n, seed))
        delta.copy_(new(n, seed + 50))
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            beside = [other.run(*y, status)["x2"] for _ in range(5)]
        torch.cuda.synchronize()
        for k, want in alone[seed].items():
            assert torch.equal(bits(held[k]), bits(want)), k
        assert all(torch.equal(b, quiet) for b in beside)
    assert int(status.item()) == 0 and keep


def test_two_streams_of_products_and_routes(dev):
    """Every form of the product, and routes of both, on two streams at once: the bits of one after the other."""
    sizes = [(2600, 260, 4000), (5, 2100, 300), (90, 2304, 1100), (200, 2048, 1000), (64, 2050, 900), (2600, 260, 4000)]
    work = [operands(*z, dev, i) for i, z in enumerate(sizes)]
    logits = [torch.randn(n, 64, generator=torch.Generator(device=dev).manual_seed(n), device=dev) for n in (60, 700, 3000)]
    run = lambda: [k8.linear_fp8(*w) for w in work] + [t for l in logits for r in (kr.route_by_scores(l, 4),) for t in (r.ids, r.weights, r.slots, r.segs)]
    want = run()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(run())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


# ---- refusals --------------------------------------------------------------------------------------------------------
def test_refusals(dev):
    x, w = torch.randn(4, 48, device=dev), torch.ones(48, device=dev)
    slots, weights, pairs = torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.ones(4, 2, device=dev), torch.randn(8, 48, device=dev)
    b = lambda **k: (lambda: k8.rms_residual_fp8(**(dict(x=x, weight=w, eps=1e-5) | k)))
    q, s = k8.quantize_fp8(x)
    qw, sw = k8.quantize_weight(torch.randn(10, 48, device=dev))
    f = lambda **k: (lambda: k8.linear_fp8(**(dict(x=q, x_scales=s, w=qw, w_scales=sw) | k)))
    r = lambda logits=torch.randn(4, 12, device=dev), top=3, **k: (lambda: kr.route_by_scores(logits, top, **k))
    experts = lambda **k: (lambda: ke.ExpertWeights([pairs] * 4, [pairs] * 4, [pairs.t().contiguous()] * 4, **k))
    for call in (b(x=x.half()), b(x=x[:, ::2]), b(x=x[0]), b(weight=w[:47]), b(weight=w.to(BF)), b(delta=x[:3]), b(delta=x.half()), b(x=x.to(BF), delta=x), b(x_out=x.to(BF)),
                 b(x_out=torch.empty(4, 96, device=dev)[:, ::2]), b(out=x.half()), b(pairs=pairs), b(pairs=pairs, pair_slots=slots), b(pair_weights=weights),
                 b(pairs=pairs, pair_slots=slots.long(), pair_weights=weights), b(pairs=pairs, pair_slots=slots[:3], pair_weights=weights[:3]),
                 b(pairs=pairs, pair_slots=slots, pair_weights=weights[:, :1]), b(pairs=pairs[:, :40], pair_slots=slots, pair_weights=weights), b(delta=x.cpu()),
                 lambda: k8.quantize_fp8(x, "relu"), lambda: k8.quantize_fp8(x.half()), lambda: k8.quantize_fp8(x.t()), lambda: k8.quantize_fp8(x[:, :47], "silu_gate"),
                 f(x=x), f(x=q[:, :40]), f(x=q[:, 1:]), f(w=qw.t()), f(x_scales=s.t()), f(x_scales=s.double()), f(x_scales=s[:, :3]), f(w_scales=sw.t().contiguous().expand(2, 1)),
                 f(out_dtype=torch.float16), f(out=torch.empty(4, 10, device=dev)), f(out=torch.empty(4, 20, dtype=BF, device=dev)[:, ::2]), f(w=qw.cpu()), f(x_scales=s.cpu()),
                 r(top=0), r(top=13), r(top=33), r(logits=torch.randn(4, 2000, device=dev)), r(logits=torch.randn(4, 12, device=dev).half()), r(logits=torch.randn(12, 4, device=dev).t()),
                 r(score="tanh"), r(groups=5), r(groups=4, top_groups=5), r(groups=4, top_groups=0), r(groups=6, top_groups=1), r(bias=torch.zeros(11, device=dev)),
                 r(bias=torch.zeros(12, device=dev).to(BF)), r(bias=torch.zeros(12)), r(active=torch.ones(4, device=dev)), r(active=torch.ones(3, dtype=torch.int32, device=dev)),
                 experts(), experts(top=0), experts(top=5), experts(top=2, table=torch.zeros(9, 2, dtype=torch.int64, device=dev)),
                 lambda: ke.experts_forward(pairs, experts(top=2)(), kr.route_by_scores(torch.randn(4, 4, device=dev), 3)),
                 lambda: ke.ExpertRouter([experts(top=2)()], 9)):
        with pytest.raises((ValueError, TypeError)):
            call()


def test_rows_beyond_32_bit_offsets(dev):
    n, width = 140_000, 16_384  # 2.3 billion elements
    z = torch.randn(1000, width, device=dev).to(BF).repeat(n // 1000, 1)
    z[-3:] = 2 * z[-3:] + 1
    q, s = k8.quantize_fp8(z)
    few, scales = k8.quantize_fp8(z[-3:])
    assert torch.equal(q[-3:].view(torch.uint8), few.view(torch.uint8)) and torch.equal(s[:, -3:], scales)
    w, delta = torch.rand(width, device=dev), z
    x_out = torch.empty_like(z)
    q, s = k8.rms_residual_fp8(z, w, eps=1e-5, delta=delta, x_out=x_out)
    y = torch.empty(3, width, dtype=BF, device=dev)
    few, scales = k8.rms_residual_fp8(z[-3:], w, eps=1e-5, delta=delta[-3:], x_out=y)
    assert torch.equal(x_out[-3:], y)
    holds8(q[-3:].clone(), s[:, -3:].clone(), fo.rms_norm(y.cpu(), w.cpu(), 1e-5), NORM)
    holds8(few, scales, fo.rms_norm(y.cpu(), w.cpu(), 1e-5), NORM)
    del z, q, x_out, delta
    x, sx, w8, sw = operands(120_000, 256, 18_000, dev, 3)
    out = k8.linear_fp8(x, sx, w8, sw)  # 2.16 billion elements
    for at in (slice(119_900, 120_000), slice(0, 50)):
        check_linear(out[at], x[at], sx[:, at], w8, sw)
