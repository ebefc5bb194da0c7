"""CPU: host sides of the 8-bit operators and of the routes by scores: workspaces, weights, forms."""
from __future__ import annotations




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
