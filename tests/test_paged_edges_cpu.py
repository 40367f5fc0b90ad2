"""Sizes that the paged cache's operators take and refuse, without a GPU."""
import pytest
import torch

from tiktok_techjam_2026_track3_amd import _lib, ops

BAD_SIZE = -2


def views(names, tokens, heads, B, most, kv_heads=8, ragged=True):
    shapes = tuple(torch.Size((tokens, kv_heads if n in ("k", "v") else heads, 128)) for n in names)
    return ops._paged_views(torch.Size((9, kv_heads, 16, 128)), torch.Size((B, 4)), (4, 1), most, ragged, names, (torch.float16,) * len(names),
                            shapes, tuple(torch.empty(s, device="meta").stride() for s in shapes))


@pytest.mark.parametrize("tokens,heads,B,most", [
    (30000, 32, 24, 16000), (4159, 32, 64, 4096), (2304, 32, 257, 2048), ((1 << 18) - 1, 32, 2, 1 << 18), (8, 64, 1 << 20, 1 << 20),
    (5, 8, 1, (1 << 20) - 1)])
def test_what_counts_is_how_many_tokens_there_are(tokens, heads, B, most):
    sizes = views(("q",), tokens, heads, B, most)[1]
    assert _lib.lib().mi355_attn_paged_workspace_bytes(sizes) >= 0


@pytest.mark.parametrize("tokens,heads,B,most,ragged", [
    (1 << 18, 32, 2, 1 << 18, True), (1 << 18, 32, 1, 1 << 18, False), (5, 8, 1, (1 << 20) + 1, True), (5, 8, 1 << 20, (1 << 20) + 1, True)])
def test_attention_refuses_more(tokens, heads, B, most, ragged):
    with pytest.raises(ValueError, match="too many for one call"):
        views(("q",), tokens, heads, B, most, ragged=ragged)
    sizes = _lib.i64_array((B, most, tokens, heads, 8, 128, 9, 16, 4, 4))
    assert _lib.lib().mi355_attn_paged_workspace_bytes(sizes) == BAD_SIZE


@pytest.mark.parametrize("names", [("k", "v"), ("k", "v", "q")])
def test_append_takes_what_its_launch_does(names):
    for tokens, B, most in ((30000, 24, 16000), (1 << 18, 1, 1 << 18), (1 << 18, 64, 1 << 18), (1 << 20, 1 << 20, 1), (5, 1 << 20, 97)):
        views(names, tokens, 64, B, most)
    for B, most in ((1 << 20, 98), (8, (1 << 24) + 1)):
        with pytest.raises(ValueError, match="too many for one call"):
            views(names, 5, 64, B, most)
