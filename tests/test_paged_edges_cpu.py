"""Sizes that the paged cache's operators take and refuse and the frequencies of rotary plans, without a GPU."""
from decimal import Decimal, localcontext

import pytest
import torch

from paged_edges_reference import pi_of
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


@pytest.mark.parametrize("kw", [
    dict(base=10000.0), dict(base=500000.0), dict(base=1.0), dict(base=0.01), dict(base=1e300), dict(base=10000.0, scaling="linear", factor=3.0),
    dict(base=10000.0, scaling="base", factor=16.0), dict(base=10000.0, scaling="parts", factor=8.0, original=4096),
    dict(base=1e6, scaling="parts", factor=3.3, original=8192.5, slow=0.5, fast=7), dict(freqs=[2.5, -2.5, 1e-30, -1e-30, 0.0, 1e17, -1e17, 1e300])])
def test_frequencies_are_rounded_once(monkeypatch, kw):
    """The fractions of a turn times 2^64 of a plan are the nearest whole numbers, computed here with 700 digits."""
    dim = 16
    seen = []
    monkeypatch.setattr(torch.Tensor, "to", lambda self, *a, **k: seen.append(self) or self)
    ops.rotary_plan(dim, **kw)
    with localcontext() as c:
        c.prec = 700
        two_pi, base, factor = 2 * pi_of(700), Decimal(kw.get("base", 1.0)), Decimal(kw.get("factor", 1.0))
        if kw.get("scaling") == "base":
            base = base * (factor.ln() * dim / (dim - 2)).exp()
        f = [Decimal(x) for x in kw["freqs"]] if "freqs" in kw else [(base.ln() * -j / 8).exp() for j in range(8)]
        if kw.get("scaling") == "linear":
            f = [x / factor for x in f]
        if kw.get("scaling") == "parts":
            slow, fast, original = Decimal(kw.get("slow", 1.0)), Decimal(kw.get("fast", 32.0)), Decimal(kw["original"])
            for j, x in enumerate(f):
                r = original * x / two_pi
                g = 0 if r <= slow else 1 if r >= fast else (r - slow) / (fast - slow)
                f[j] = x * (g + (1 - g) / factor)
        for x, turn in zip(f, seen[0].tolist()):
            off = abs((x / two_pi * 2 ** 64 - turn) % 2 ** 64)
            assert min(off, 2 ** 64 - off) <= Decimal("0.5000001"), (x, turn, off)


@pytest.mark.parametrize("turns,dim", [
    (torch.zeros(31, dtype=torch.int64), 64), (torch.zeros(0, dtype=torch.int64), 2), (torch.zeros(64, dtype=torch.int64)[::2], 64),
    (torch.zeros(32, dtype=torch.int32), 64), (torch.zeros(32, 1, dtype=torch.int64), 64), (torch.zeros(32), 64),
    (torch.zeros(0, dtype=torch.int64), 0), (torch.zeros(3, dtype=torch.int64), 7), (torch.zeros(257, dtype=torch.int64), 514)])
def test_plans_that_the_kernels_would_read_beyond_are_refused(turns, dim):
    with pytest.raises(ValueError):
        ops.RotaryPlan(turns, dim, False, 1.0)
    assert ops.RotaryPlan(torch.zeros(32, dtype=torch.int64), 64, False, 1.0).dim == 64


@pytest.mark.parametrize("amplitude", [1e39, -1e300, float("nan")])
def test_amplitudes_beyond_fp32_are_refused(amplitude):
    """(the kernels take it in fp32, where it would be an infinity)"""
    with pytest.raises(ValueError, match="amplitude"):
        ops.rotary_plan(64, amplitude=amplitude, device="cpu")
