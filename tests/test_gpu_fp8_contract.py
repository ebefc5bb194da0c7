"""GPU: the 8-bit operators and the routes by scores where their contract says more than a tolerance."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8_oracle as fo
from spikeinfer_b200 import _lib
from spikeinfer_b200.kernels import fp8 as k8
from spikeinfer_b200.kernels import routing as kr

from test_gpu_fp8_ops import BF, F32, FP8, HALF, NORM, U, check_linear, check_route, gen, operands

pytestmark = pytest.mark.gpu


# ---- the 8-bit value and its scale ----------------------------------------------------------------------------------
def is_quotient(q, scales, v):
    """scales are most / 448 and q is v / scale to the nearest, both as 32-bit divisions round them: no other value, at a tie neither."""
    v = v.float().cpu()
    n, width = v.shape
    blocks = -(-width // 128)
    padded = torch.zeros(n, blocks * 128)
    padded[:, :width] = v
    padded = padded.view(n, blocks, 128)
    most = torch.where(padded.isnan(), 0.0, padded.abs()).clamp(max=torch.finfo(F32).max).amax(2).clamp(min=fo.LEAST)
    want = most / 448.0
    assert torch.equal(scales.cpu(), want.t())
    values = (padded / want[..., None]).clamp(-448.0, 448.0).to(FP8).view(n, -1)[:, :width]
    assert torch.equal(torch.nan_to_num(q.cpu().float(), nan=-1000.0), torch.nan_to_num(values.float(), nan=-1000.0))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,width,pad", [(37, 4864, 0), (300, 1021, 1), (300, 1022, 2), (3000, 896, 0), (3000, 898, 0), (2500, 897, 0), (8192, 4864, 0)])
def test_values_are_the_nearest_to_the_quotient(dev, n, width, pad, dtype):
    """16-bit values over a scale of few bits lie between two 8-bit ones often (one in a thousand): the even one is theirs."""
    z = torch.full((n, width + pad), float("nan"), dtype=dtype, device=dev)[:, pad // 2: pad // 2 + width]
    z.copy_(torch.randn(n, width, generator=torch.Generator(device=dev).manual_seed(n + width), device=dev))
    if dtype == F32:
        z.mul_(2.0 ** torch.randint(-90, 100, (n, 1), generator=torch.Generator(device=dev).manual_seed(1), device=dev))
    q, scales = k8.quantize_fp8(z)
    is_quotient(q, scales, z)


@pytest.mark.parametrize("stream", [F32, BF])
@pytest.mark.parametrize("n,width", [(5, 512), (3, 1022), (7, 1021), (64, 3584), (700, 256), (2000, 3584), (1300, 1030)])
def test_boundary_rounds_what_it_writes(dev, n, width, stream):
    g = torch.Generator(device=dev).manual_seed(n + width)
    x, delta = (torch.randn(n, width, generator=g, device=dev).to(stream) for _ in range(2))
    out = torch.empty(n, width, device=dev)
    q, scales = k8.rms_residual_fp8(x, 1 + 0.2 * torch.randn(width, generator=g, device=dev), eps=1e-5, delta=delta, out=out)
    is_quotient(q, scales, out)


def test_quotients_of_values_that_are_not_finite(dev):
    inf, nan = float("inf"), float("nan")
    top = torch.finfo(F32).max
    for dtype in (F32, BF):
        for width in (512, 514, 513):
            z = torch.randn(6, width, generator=gen(width)) * torch.tensor([1.0, 1e-30, 1e30, 1e-32, 1.0, 1.0])[:, None]
            z[0, 3], z[0, 200], z[2, 5], z[2, 300], z[4, 7], z[5] = nan, inf, -inf, top, -top, 0.0
            z = z.to(dtype)
            q, scales = k8.quantize_fp8(z.to(dev))
            is_quotient(q, scales, z)


# ---- choices ---------------------------------------------------------------------------------------------------------
def rows_of(*rows, experts=12):
    """Rows of logits; where a row is short, experts behind it that can't be chosen."""
    out = torch.full((len(rows), experts), -float("inf"))
    for r, row in zip(out, rows):
        r[: len(row)] = torch.tensor(row)
    return out


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("times", [1, 70])
def test_equal_experts_at_the_cut_hide_none_behind_them(dev, times, dtype):
    """The last of the chosen equals the next one, and one behind both that 32 bits cannot tell from them is better."""
    sigmoid = rows_of([17, 17, 40, 0], [20, 20, 20, 25, 0, 0, 0, 0], [30, 30, 30, 30, 30, 30, 30, 31, 33, 35, 36, 36], [17, 17, 17, 40], [-200, -200, -100], [-120, -120, -120, -119, -120])
    softmax = rows_of([0, -200, -200, -100], [0, -150, -150, -150, -150, -149], [0, -120, -120, -120, -110, -115], [5, 5, -300, -300, -299])
    flat = rows_of([-20, -20, -19, -50], [-22, -22, -22, -22, -21], [-18, -18, -18, -17, -17])  # beside a bias that is 1 for all
    one = torch.ones(12)
    for logits, score, bias in ((sigmoid, "sigmoid", None), (softmax, "softmax", None), (flat, "sigmoid", one), (rows_of([0, -22, -22, -21], [0, -30, -30, -30, -29]), "softmax", one)):
        logits = logits.repeat(times, 1).to(dtype)
        for top in (1, 2, 3, 4, 8):
            for groups, top_groups in ((1, 1), (3, 2)):
                if top <= 12 // groups * top_groups:
                    more = dict(score=score, bias=None if bias is None else bias.to(dev), groups=groups, top_groups=top_groups)
                    check_route(kr.route_by_scores(logits.to(dev), top, **more), logits, top, **more)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top", [(16, 2), (64, 6), (200, 1), (256, 8), (300, 4), (700, 5)])
def test_choices_among_few_and_saturated_logits(dev, experts, top, score):
    """Logits of a few values: ties at every cut, saturated ones among them, single better experts far behind."""
    g = gen(experts)
    values = torch.tensor([17.0, 17.5, 20.0, 30.0, 36.0, 40.0, -100.0, -200.0])
    logits = values[torch.randint(0, 8, (40, experts), generator=g)]
    logits[:20] = 20.0
    logits[torch.arange(10), torch.randint(0, experts, (10,), generator=g)] = 25.0
    logits[20:30] = torch.where(torch.rand(10, experts, generator=g) < 0.9, 17.0, logits[20:30])
    logits[10] = 0.0
    logits[11] = 0.0
    logits[11, experts - 1] = 1e-9
    for bias in (None, torch.full((experts,), 2.0)):
        more = dict(score=score, bias=None if bias is None else bias.to(dev))
        check_route(kr.route_by_scores(logits.to(dev), top, **more), logits, top, **more)


# ---- products ----------------------------------------------------------------------------------------------------------
def test_a_product_of_many_tiles_by_pairs(dev):
    """Some ten milliseconds in one launch, beyond any one wait's share: the last rows and features are right, nothing ran out, and again."""
    n, k, f = 33_000, 18_944, 16_400
    x, sx, w, sw = operands(n, k, f, dev, 7)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = k8.linear_fp8(x, sx, w, sw, status=status)
    assert torch.equal(out, k8.linear_fp8(x, sx, w, sw, status=status)) and int(status.item()) == 0
    fb = 16_256  # a block's first feature
    for at in (slice(0, 20), slice(n - 140, n)):
        check_linear(out[at, fb:], x[at], sx[:, at], w[fb:], sw[fb // 128:])


# ---- rows of many tokens' choices -------------------------------------------------------------------------------------
def rows_in_order(r, experts):
    """slots and segs follow from the ids: segments of multiples of eight rows, the pairs of an expert in their order."""
    ids = r.ids.cpu().long()
    n, top = ids.shape
    flat = torch.where(ids < 0, experts, ids).flatten()
    counts = torch.bincount(flat, minlength=experts + 1)[:experts]
    first = torch.cumsum((counts + 7) // 8 * 8, 0) - (counts + 7) // 8 * 8
    order = torch.sort(flat, stable=True).indices
    place = torch.empty_like(flat)
    place[order] = torch.arange(n * top)
    e = flat.clamp(max=experts - 1)
    slots = torch.where(flat < experts, first[e] + place - (torch.cumsum(counts, 0) - counts)[e], -1)
    assert torch.equal(r.slots.cpu().long().flatten(), slots) and torch.equal(r.segs.cpu().long(), torch.stack((first, counts), 1))


@pytest.mark.parametrize("n,experts,top", [(2369, 24, 3), (5000, 40, 4), (5000, 256, 8)])
def test_routes_of_32_tokens_a_word(dev, n, experts, top):
    logits = torch.randn(n, experts, generator=gen(n))
    groups, top_groups = (8, 4) if experts == 256 else (1, 1)
    more = dict(score="sigmoid", groups=groups, top_groups=top_groups)
    r = kr.route_by_scores(logits.to(dev), top, **more)
    check_route(r, logits, top, **more)
    rows_in_order(r, experts)


@pytest.mark.parametrize("n,experts,top", [(32_768, 16, 2), (32_769, 16, 2), (70_001, 64, 6), (300_000, 33, 1), (1_000_003, 8, 2)])
def test_routes_beyond_what_a_cta_counts(dev, n, experts, top):
    """More words than every CTA of the layout counts by itself (1024): counts by chunks, the last of each cut short."""
    g = torch.Generator(device=dev).manual_seed(n)
    logits = torch.randn(n, experts, generator=g, device=dev)
    active = (torch.rand(n, generator=g, device=dev) < 0.97).to(torch.int32)
    logits[torch.rand(n, generator=g, device=dev) < 0.01] = -float("inf")
    r = kr.route_by_scores(logits, top, active=active)
    rows_in_order(r, experts)
    want = torch.sort(logits.double().softmax(1), dim=1, descending=True, stable=True).indices[:, :top]
    there = (active == 1) & (logits[:, 0] > -float("inf"))
    assert torch.equal(r.ids[there].long(), want[there]) and (r.ids[~there] == -1).all()
    again = kr.route_by_scores(logits, top, active=active)
    assert torch.equal(r.slots, again.slots) and torch.equal(r.segs, again.segs)


def test_routes_of_many_tokens_in_a_graph_beside_others(dev):
    n, experts = 50_000, 48
    x, other = (torch.randn(n, experts, generator=torch.Generator(device=dev).manual_seed(s), device=dev) for s in (1, 2))
    want = [kr.route_by_scores(t, 4) for t in (x, other)]
    held = x.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        kr.route_by_scores(held, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = kr.route_by_scores(held, 4)
    for t, w in ((other, want[1]), (x, want[0])):
        held.copy_(t)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        beside = [kr.route_by_scores(other, 4) for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(captured.slots, w.slots) and torch.equal(captured.segs, w.segs) and torch.equal(captured.weights, w.weights)
        assert all(torch.equal(b.slots, want[1].slots) and torch.equal(b.segs, want[1].segs) for b in beside)


# ---- single rows -----------------------------------------------------------------------------------------------------
def test_the_stride_of_a_single_row_is_of_no_account(dev):
    one = lambda t, stride: t.as_strided((1, t.shape[1]), (stride, 1))
    for act in ("none", "silu_gate"):
        z = torch.randn(1, 300, generator=gen(2)).to(dev)
        want, scales = k8.quantize_fp8(z, act)
        got, s = k8.quantize_fp8(one(z, 1), act)
        assert torch.equal(got.float(), want.float()) and torch.equal(s, scales)
    column = torch.randn(5, 7, generator=gen(3)).to(dev)[:, 2:3]  # nor that of a single column
    got, s = k8.quantize_fp8(column)
    want, scales = k8.quantize_fp8(column.clone())
    assert torch.equal(got.float(), want.float()) and torch.equal(s, scales)
    x, sx, w, sw = operands(1, 200, 1, dev, 4)
    want = k8.linear_fp8(x, sx, w, sw)
    for stride in (1, 200, 208):
        assert torch.equal(k8.linear_fp8(one(x, stride), sx, one(w, stride), sw), want)
    for bad in (one(x, 200)[:, 8:], torch.empty(2, 200, dtype=FP8, device=dev)[:, :40].t(), torch.empty(2, 200, dtype=FP8, device=dev)[:, :45]):
        with pytest.raises(ValueError):
            k8.linear_fp8(bad, sx, w, sw)


# ---- scales far from one ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,k,f", [(5, 300, 200), (40, 2100, 300), (130, 400, 300), (130, 2100, 200), (600, 300, 2600), (1171, 200, 4864), (2600, 260, 4000)])
def test_products_of_scales_beyond_32_bits(dev, n, k, f):
    """A block's two scales need not have a product in 32 bits: what counts is the block's term."""
    x, sx, w, sw = operands(n, k, f, dev, n)
    sx.fill_(1.0)
    sw.fill_(1.0)
    top = 2.0 ** 70
    sx[1], sw[:, 1] = top, top  # block 1: 2^140, beside nothing, and beside products of 2^-18
    x[:, 128:256] = 0.0
    x[1::2, 130] = 2.0 ** -9
    w[:, 130] = 2.0 ** -9
    out = k8.linear_fp8(x, sx, w, sw, out_dtype=F32)
    assert torch.isfinite(out[1::2]).all() and (out[1::2] > 2.0 ** 121).all()
    check_linear(out, x, sx, w, sw)
    near = k8.linear_fp8(x, torch.ones_like(sx), w, sw, out_dtype=F32)
    sx[1, 1:] = 1.0  # row 0 alone is far: the others keep their bits
    assert torch.equal(k8.linear_fp8(x, sx, w, sw, out_dtype=F32)[1:], near[1:])
    # far below: products of 2^-138, of which 32 bits hold a few, known to within 2^-150 each
    g = torch.Generator(device=dev).manual_seed(k)
    x, _, w, _ = operands(n, k, f, dev, n + 1)
    size = x.double().cpu().abs() @ w.double().cpu().abs().t()
    sx.copy_((0.5 + torch.rand(sx.shape, generator=g, device=dev)) * 2.0 ** -72)
    sw.copy_((0.5 + torch.rand(sw.shape, generator=g, device=dev)) * 2.0 ** -66)
    want, _ = fo.linear(x.cpu(), sx.cpu(), w.cpu(), sw.cpu())
    off = (k8.linear_fp8(x, sx, w, sw, out_dtype=F32).double().cpu() - want).abs()
    assert (off <= 2.0 ** -150 * size * (1 + 132 * 2.0 ** -23) + 2.0 ** -16 * 2.0 ** -136 * size).all()  # 132 x 2^-23 of the terms: under 2^-16 of them, scales under 1.5^2 x 2^-138
    # blocks of zeros as quantize_fp8 leaves them, beside scales of any size; a scale of zero is zero beside any other
    sx.fill_(1.0)
    sw.fill_(1.0)
    sx[1], x[:, 128:256] = 2.0 ** -100 / 448, 0.0
    sw[:, 1] = 2.0 ** -40
    check_linear(k8.linear_fp8(x, sx, w, sw, out_dtype=F32), x, sx, w, sw)
    sx[0], sw[:, 0] = 0.0, 2.0 ** 120
    check_linear(k8.linear_fp8(x, sx, w, sw, out_dtype=F32), x, sx, w, sw)


@pytest.mark.parametrize("n", [7, 8, 9, 63, 64, 113, 120, 127, 128])
@pytest.mark.parametrize("experts,top", [(16, 16), (256, 32), (1000, 32)])
def test_routes_that_one_cluster_hands_out(dev, n, experts, top):
    """One to sixteen tokens a CTA and up to 32 choices each: the most that a launch of one cluster keeps."""
    logits = torch.randn(n, experts, generator=gen(n + top))
    r = kr.route_by_scores(logits.to(dev), top)
    check_route(r, logits, top)
    rows_in_order(r, experts)


# ---- every form, beyond the first turn of its rings --------------------------------------------------------------------
# (rows of a tile, parts of k) of the sizes that take it; every CTA has 33 or more blocks of 128 columns, so that stages, accumulators and groups of scales are used again
FORMS = {(rows, parts): [(n, 4300 * parts, f)] for rows, n in ((16, 13), (32, 29), (64, 61)) for parts, f in ((1, 8200), (2, 4120), (4, 1100), (8, 300))}
FORMS |= {(128, 4): [(130, 17_100, 200)], (128, 2): [(300, 8500, 1500)], (128, 1): [(1171, 4300, 1200), (1171, 4300, 4864), (1171, 896, 4864)],  # one tile a CTA, two and three
          (256, 1): [(2600, 4300, 4000), (2600, 3584, 4000)]}


@pytest.mark.parametrize("out_dtype", [BF, F32])
@pytest.mark.parametrize("rows,parts,n,k,f", [(*form, *size) for form, sizes in FORMS.items() for size in sizes])
def test_products_of_every_form(dev, rows, parts, n, k, f, out_dtype):
    assert _lib.load().spk_linear_fp8_form(n, k, f) == 16 * rows + parts
    x, sx, w, sw = operands(n, k, f, dev, n + k + f)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = k8.linear_fp8(x, sx, w, sw, out_dtype=out_dtype, status=status)
    want, size = fo.linear(x, sx, w, sw)
    tol = (132 * 2.0 ** -23 + (3 + -(-k // 128)) * U) * size  # as check_linear
    assert ((out.double() - want).abs() <= tol + HALF[out_dtype] * (want.abs() + tol)).all()
    assert torch.equal(out, k8.linear_fp8(x, sx, w, sw, out_dtype=out_dtype)) and int(status.item()) == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("act", ["gelu_tanh", "silu_gate"])
@pytest.mark.parametrize("n,width", [(600, 4864), (600, 3502), (600, 3501), (8192, 4864)])
def test_activations_of_several_blocks_at_a_time(dev, n, width, act, dtype):
    """Two blocks at a time from 16384 on, four (16-bit rows on 16-byte boundaries) from 262144 on; bounds as test_quantize counts them."""
    g = torch.Generator(device=dev).manual_seed(n + width)
    z = (3 * torch.randn(n, width * (2 if act == "silu_gate" else 1), generator=g, device=dev)).to(dtype)
    q, scales = k8.quantize_fp8(z, act)
    v, rel = fo.activation(z, act), (1300 if act == "gelu_tanh" else 64) * U
    blocks = -(-width // 128)
    most = torch.nn.functional.pad(v.abs(), (0, blocks * 128 - width)).view(n, blocks, 128).amax(2).clamp(min=fo.LEAST)
    assert ((scales.t().double() - most / 448).abs() <= (rel + 2 * U) * most / 448).all()
    s = scales.double().t().repeat_interleave(128, 1)[:, :width]
    off = (q.double() * s - v).abs()
    keep = v.abs() > 1e-4 * 448 * s
    assert (off <= 0.5 * fo.e4m3_step(v / s) * s * (1 + 64 * U) + (rel + 4 * U) * v.abs())[keep].all()
    assert (off <= 1.01 * 2.0 ** -9 * s)[~keep].all()
    few = k8.quantize_fp8(z[-5:].contiguous(), act)  # a block's values do not depend on how many are taken at once
    assert torch.equal(q[-5:].float(), few[0].float()) and torch.equal(scales[:, -5:], few[1])


@pytest.mark.parametrize("stream,delta_dtype", [(BF, BF), (BF, None), (F32, F32), (F32, BF), (F32, None)])
@pytest.mark.parametrize("n,width", [(8192, 3584), (5001, 896), (9000, 128), (4000, 8192), (4000, 1000)])
def test_boundaries_of_many_rows_a_cta(dev, n, width, stream, delta_dtype):
    """The streaming form gives a CTA more rows than it has stages (three): up to 19 here."""
    g = torch.Generator(device=dev).manual_seed(n + width)
    x = torch.randn(n, width, generator=g, device=dev).to(stream)
    delta = None if delta_dtype is None else torch.randn(n, width, generator=g, device=dev).to(delta_dtype)
    w, eps = 1 + 0.3 * torch.randn(width, generator=g, device=dev), 1e-5
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    x_out, out = x.clone(), torch.empty(n, width, device=dev)
    q, scales = k8.rms_residual_fp8(x_out, w, eps=eps, delta=delta, x_out=x_out, out=out, status=status)  # in place
    y = x.float() if delta is None else x.float() + delta.float()
    assert torch.equal(x_out, y.to(stream))  # one rounding to 32 bits, and to the stream's
    v = fo.rms_norm(x_out, w, eps)
    assert ((out.double() - v).abs() <= (NORM + U) * (1 + 2 * U) * v.abs()).all()
    is_quotient(q, scales, out)
    short = torch.empty(n, width, dtype=BF, device=dev)
    q2, s2 = k8.rms_residual_fp8(x, w, eps=eps, delta=delta, out=short, status=status)
    assert torch.equal(short, out.to(BF)) and torch.equal(q2.float(), q.float()) and torch.equal(s2, scales) and int(status.item()) == 0
