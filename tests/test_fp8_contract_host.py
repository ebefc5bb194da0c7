"""CPU: host sides of the 8-bit operators and of the routes by scores: workspaces, weights, forms."""
from __future__ import annotations

import torch

from spikeinfer_b200.kernels import fp8 as k8

from test_gpu_fp8_contract import FORMS


def test_workspace_of_many_tokens_holds_counts_by_chunks(lib):
    """A bit for every token and expert, 32 to a word, four words at a time; beyond 1024 words a count for every 64 of them, and the sums."""
    need = lib.spk_route_scores_workspace_bytes
    for experts in (1, 7, 256):
        assert need(128, experts) == 0
        for n in (2400, 5000, 32_768):
            assert need(n, experts) == -(-n // 128) * 16 * experts
        for n in (32_769, 70_000, 1 << 24):
            words = -(-n // 32)
            assert need(n, experts) == -(-words // 4) * 16 * experts + (-(-words // 64) + 1) * 4 * experts


def test_weights_that_are_not_finite_stay_alone():
    """NaN is NaN and not the largest of its block, an infinity counts as the largest finite value: the rule of the activations."""
    inf, nan, top = float("inf"), float("nan"), torch.finfo(torch.float32).max
    for dtype in (torch.float32, torch.bfloat16):
        w = torch.randn(200, 300, generator=torch.Generator().manual_seed(1)).to(dtype)
        w[3, 5] = 0.0
        want, _ = k8.quantize_weight(w)
        bad = w.clone()
        bad[3, 5], bad[150, 20], bad[130, 299] = nan, inf, -inf
        bad[:128, 256:] = nan
        q, s = k8.quantize_weight(bad)
        values = q.float()
        assert torch.isfinite(s).all() and float(s[0, 2]) == float(torch.tensor(2.0 ** -100) / 448)
        assert values[3, 5].isnan() and values[:128, 256:].isnan().all() and int(values.isnan().sum()) == 1 + 128 * 44
        assert float(s[1, 0]) == float(s[1, 2]) == float(torch.tensor(top) / 448) and values[150, 20] == 448 and values[130, 299] == -448
        rest = torch.ones(200, 300, dtype=torch.bool)  # blocks without an infinity: as they were
        rest[3, 5] = False
        rest[:128, 256:] = rest[128:, :128] = rest[128:, 256:] = False
        assert torch.equal(values[rest], want.float()[rest])
        assert (values[128:, :128] == 0).sum() >= 72 * 128 - 1  # next to 3e38 there is nothing left of the others


def test_every_form_of_the_product_is_tested_beyond_its_rings(lib):
    """The sizes of test_products_of_every_form take the forms that they stand for, all that a sweep of sizes meets, and long parts of k; a changed rule shows here."""
    form = lambda n, k, f: divmod(lib.spk_linear_fp8_form(n, k, f), 16)
    for want, sizes in FORMS.items():
        assert all(form(*size) == want for size in sizes), (want, sizes)
        assert max(-(-k // 128) // want[1] for _, k, _ in sizes) >= 33
    met = {form(n, k, f) for n in (1, 20, 40, 65, 130, 600, 1171, 8192) for k in (100, 900, 2100, 4864, 18_944) for f in (100, 900, 2000, 4864, 8192, 18_944)}
    assert met == set(FORMS)
    assert lib.spk_linear_fp8_form(0, 5, 5) == lib.spk_linear_fp8_form(5, 0, 5) == lib.spk_linear_fp8_form(5, 5, 0) == 0
    # tiles of 128 x 128: more than one a CTA (148 SMs), and more blocks of k than the ring of scales holds (four groups of eight)
    assert any(-(-n // 128) * -(-f // 128) > 148 and k > 32 * 128 for n, k, f in FORMS[128, 1])
