"""The token-generation operators on inputs whose results show every key and every weight: a missing, doubled or
misweighted one is far outside rounding (which the oracle checks of itself, on the CPU).

Projections: small whole x, scales of powers of two, whole zero points and biases. A weight enters as 16 + q, a
group's sum is corrected by -(16 + z) times the sum of x, both whole and below 2^24, and what is added up is a
multiple of the least scale; as long as the sum of all magnitudes stays below 2^24 of those, every order of
summation is exact in 32 bits, and the output is that number, rounded once if it is of 16 bits.

Attention: V is 1 in one element per block of 64 keys, so that an element of the output is the weight of its blocks. With
P |V| = |ref| the bounds are relative (u = half a step of a type): 2 u for probabilities taken as one term, 2 u^2 as
two (fp16: 2^-24 of the row's largest a key), 2^-20 for the exponent of scores below 1 and the exponential, u for the
output, and for the numerator's and the probabilities' sums over n keys, 32 keys at a time, then those one after the
other (at most all of them), then at most 512 ranges, 2 (n / 32 + 544) 2^-24.
"""
import math

import pytest
import torch

from tiktok_techjam_2026_track3_amd import _lib

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16]


def _ops():
    from tiktok_techjam_2026_track3_amd import ops
    return ops


# ------------------------------------------------------------------------------ 4-bit projections
def whole_numbers(M, N, K, group, zeros, bias, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-3, 4, (M, K), generator=g).to(dtype)
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scale = (2.0 ** torch.randint(-2, 3, (N, K // group), generator=g)).to(dtype)
    zero = torch.randint(0, 64 if zeros == "any" else 16, (N, K // group), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randint(-8, 9, (N,), generator=g).float() if bias else None
    return x, w, scale, zero, b


# (M, N, K, group): each kernel, number of rows and waves that a call is given by its size
SIZES = [
    # one row in registers: one and two chunks, one, two and four waves a feature
    (1, 61, 512, 32), (1, 300, 2048, 64), (1, 75, 2176, 128), (1, 101, 4096, 32), (1, 30, 8192, 128), (1, 9001, 8064, 64),
    (1, 18, 16384, 32), (1, 4100, 12288, 128), (1, 33, 16256, 128),
    # two and four rows
    (2, 50, 4224, 64), (2, 33, 8192, 32), (2, 4099, 6144, 128), (2, 9, 16384, 64), (2, 2050, 8320, 128), (3, 21, 8224, 32),
    (4, 19, 16320, 64), (4, 1030, 16384, 128),
    # up to 16 rows held in registers: 1, 2, 4, 6 and 8 steps a wave, ranges of k that overlap, tiles that are walked
    (2, 17, 128, 128), (16, 300, 1024, 64), (5, 4200, 160, 32), (9, 8300, 1088, 64), (16, 50, 2080, 32), (3, 4097, 4096, 32),
    (7, 20, 4224, 128), (12, 100, 6144, 32), (16, 40, 6208, 64), (4, 33, 8192, 128), (11, 4500, 8128, 64),
    # beyond: one tile of features to eight waves, two to four; less than a step
    (16, 33, 6176, 32), (5, 30, 8256, 64), (16, 9, 16448, 64), (1, 20, 16512, 128), (16, 12300, 8320, 128), (6, 30, 64, 32), (16, 7, 96, 32),
    # 32 and 64 rows a tile: K below a batch of steps, one and two tiles of features
    (20, 40, 480, 32), (32, 70, 448, 64), (17, 64, 1024, 128), (25, 8200, 704, 64), (32, 33, 8192, 32), (20, 20, 16384, 128),
    (33, 40, 384, 128), (64, 96, 8192, 64), (40, 8200, 640, 128), (65, 50, 544, 32), (200, 31, 4160, 64),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,group", SIZES)
def test_i4_whole_numbers(gpu, dtype, M, N, K, group):
    """Equal in every output, fp32 and 16-bit, with zero points of 4 bits, of more, and without, with and without a bias."""
    ops = _ops()
    for zeros, bias in (("4 bits", False), ("any", True), (None, True)):
        x, w, scale, zero, b = whole_numbers(M, N, K, group, zeros, bias, dtype, M + N + K)
        xd, wd, sd, zd, bd = (t.to(gpu) if t is not None else None for t in (x, w, scale, zero, b))
        q = torch.stack((wd & 15, wd >> 4), -1).view(N, K // group, group).double()
        values = ((q - (zd.double()[..., None] if zeros else 8.0)) * sd.double()[..., None]).view(N, K)
        ref = xd.double() @ values.t().contiguous()
        if bias:
            ref += bd.double()
        most = (xd.abs().double() @ values.abs().t().contiguous()).max()
        assert float(most) + 8 < 2.0 ** 24 * 2.0 ** -2  # exact in any order
        assert torch.equal(ops.linear_i4(xd, wd, sd, zd, bd, out_dtype=torch.float32).double(), ref)
        if float(ref.abs().max()) < torch.finfo(dtype).max:
            assert torch.equal(ops.linear_i4(xd, wd, sd, zd, bd), ref.to(dtype))


@pytest.mark.parametrize("M,N,K,group", [(1, 18, 16384, 32), (4, 19, 16320, 64), (16, 40, 6208, 64), (5, 30, 8256, 64), (20, 20, 16384, 128)])
def test_i4_whole_numbers_show_every_group(gpu, M, N, K, group):
    """(The oracle alone: without any one group of 32 neighbouring k, nearly every output is another.)"""
    x, w, scale, zero, _ = whole_numbers(M, N, K, group, "4 bits", False, torch.float16, M + N + K)
    q = torch.stack((w & 15, w >> 4), -1).view(N, K // group, group).double()
    values = ((q - zero.double()[..., None]) * scale.double()[..., None]).view(N, K // 32, 32)
    parts = torch.einsum("mgk,ngk->gmn", x.double().view(M, K // 32, 32), values)
    assert float((parts != 0).double().mean()) > 0.9
    assert bool((parts != 0).flatten(1).any(1).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,group", [(1, 2048, 32), (1, 4096, 64), (1, 8192, 128), (1, 16384, 64), (2, 8192, 64), (2, 16384, 128), (4, 16384, 32),
                                       (16, 4096, 64), (16, 8192, 128), (16, 6144, 32), (16, 16512, 128), (32, 8192, 64), (64, 16384, 128)])
def test_i4_one_hot_rows_of_long_sums(gpu, dtype, M, K, group):
    """One-hot rows read single weights back, from both ends and all over K."""
    ops = _ops()
    N = 37
    _, w, scale, zero, _ = whole_numbers(1, N, K, group, "4 bits", False, dtype, K + M)
    wd, sd, zd = w.to(gpu), scale.to(gpu), zero.to(gpu)
    q = torch.stack((wd & 15, wd >> 4), -1).view(N, K // group, group).double()
    values = ((q - zd.double()[..., None]) * sd.double()[..., None]).view(N, K)
    at = torch.cat((torch.arange(64), torch.arange(K - 64, K), torch.arange(256) * (K // 256) + torch.arange(256) % 32))
    at = at.clamp_max(K - 1)[:len(at) // M * M].to(gpu)
    x = torch.zeros(M, K, dtype=dtype, device=gpu)
    rows = torch.arange(M, device=gpu)
    for k in at.view(-1, M):
        x.zero_()
        x[rows, k] = 1
        assert torch.equal(ops.linear_i4(x, wd, sd, zd).double(), values[:, k].t())


# ------------------------------------------------------------------------------ attention, range by range
def blocks(keys, kv_heads, D, dtype, seed):
    """K with one score a block of 64 keys (times q's first element, 1), V that is 1 in the block's element."""
    g = torch.Generator().manual_seed(seed)
    block = torch.arange(keys) // 64
    k, v = torch.zeros(keys, kv_heads, D), torch.zeros(keys, kv_heads, D)
    score = torch.randint(-2, 3, (keys // 64 + 1, kv_heads), generator=g) / 4.0
    k[:, :, 0] = score[block]
    v[torch.arange(keys), :, block % D] = 1
    return k.to(dtype), v.to(dtype)


def ones_q(*shape):
    q = torch.zeros(*shape)
    q[..., 0] = 1
    return q


def weights64(k, v, keys, terms, dtype):
    """The output of a row that sees the first ``keys`` keys of one head, its bound, and what any one range of 256
    keys less would change of it, relative to the bound."""
    if keys <= 0:
        z = torch.zeros(k.shape[1], dtype=torch.float64)
        return z, z + 1e-30, math.inf
    s = k[:keys, 0].double()
    p = torch.exp(s)
    pv = p[:, None] * v[:keys].double()
    ref = pv.sum(0) / p.sum()
    rel = 2 * UNIT[dtype] ** terms + 2.0 ** -20 + (keys / 32 + 544) * 2.0 ** -23 + UNIT[dtype] * (1 + UNIT[dtype])
    least = 2.0 ** -24 * keys / float(p.sum()) if dtype == torch.float16 else 0.0
    tol = rel * ref + least + 2.0 ** -25
    n = -(-keys // 256) * 256
    pad = torch.zeros(n - keys, v.shape[1], dtype=torch.float64)
    of_range = torch.cat((pv, pad)).view(n // 256, 256, -1).sum(1)
    p_range = torch.cat((p, pad[:, 0])).view(n // 256, 256).sum(1)
    without = (pv.sum(0) - of_range) / (p.sum() - p_range)[:, None].clamp_min(1e-30)
    seen = float(((without - ref).abs() / tol).amax(1).min()) if n > 256 else math.inf
    return ref, tol, seen


def check(name, out, ref, tol):
    worst = float(((out.cpu().double() - ref).abs() / tol).max())
    print(f"{name}: worst err/bound {worst:.3f}", flush=True)
    assert worst <= 1.0, name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 80])
@pytest.mark.parametrize("q_lens,k_lens,H,Hkv", [
    ([1], [20001], 4, 2), ([3, 1, 2], [5000, 1, 300], 6, 2), ([1, 1], [70000, 3], 8, 1),   # few rows
    ([70], [4001], 4, 2), ([90, 2, 200], [3000, 2500, 900], 5, 1)])                        # tiles of 64 rows, both kinds
@pytest.mark.parametrize("causal", [True, False])
def test_packed_every_range_counts(gpu, dtype, D, q_lens, k_lens, H, Hkv, causal):
    ops = _ops()
    plan = ops.packed_plan(q_lens, k_lens, heads=H, kv_heads=Hkv, head_dim=D, causal=causal, device=gpu)
    assert plan.counts[2] > 0
    kv = [blocks(m, Hkv, D, dtype, i + m) for i, m in enumerate(k_lens)]
    out = ops.attention_packed(ones_q(sum(q_lens), H, D).to(dtype).to(gpu), torch.cat([k for k, _ in kv]).to(gpu),
                               torch.cat([v for _, v in kv]).to(gpu), plan, scale=1.0)
    q0 = 0
    for i, (n, m, (k, v)) in enumerate(zip(q_lens, k_lens, kv)):
        terms = 2 if n * H // Hkv <= 32 and plan.counts[1] else 1
        for t in sorted({0, n // 2, n - 1}):
            for h in (0, H - 1):
                y = h * Hkv // H
                ref, tol, seen = weights64(k[:, y], v[:, y], m - n + t + 1 if causal else m, terms, dtype)
                assert seen > 3
                check(f"sequence {i} token {t} head {h}", out[q0 + t, h], ref, tol)
        q0 += n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,n,H,Hkv,D,P,room", [
    # up to 32 ranges are joined by one wave a row, more by four; H that is no multiple of the rows of a work-group
    (1, 1, 3, 1, 64, 256 * 31, 256), (1, 1, 3, 1, 64, 256 * 32, 256), (1, 1, 5, 1, 128, 256 * 33 + 7, 300), (2, 1, 6, 2, 64, 20000, 9000),
    (1, 2, 7, 1, 64, 70000, 500), (1, 1, 2, 2, 256, 33000, 40), (3, 1, 3, 3, 80, 0, 33000), (1, 3, 1, 1, 16, 17000, 100), (1, 1, 9, 3, 192, 30000, 1000),
    # tiles of 16, 32, 64 and 128 rows of the prefix beside 16 and 32 (one and several) of the caches
    (4, 1, 4, 1, 64, 3000, 600), (4, 1, 8, 1, 64, 3000, 600), (2, 1, 32, 1, 64, 3000, 600), (2, 1, 32, 1, 128, 9000, 2000), (2, 1, 32, 1, 256, 3000, 600),
    (4, 1, 16, 1, 80, 3000, 600), (20, 1, 32, 1, 64, 3000, 600), (20, 2, 8, 1, 128, 5000, 600), (3, 17, 4, 2, 64, 3000, 600), (1, 50, 2, 1, 128, 2000, 700)])
def test_prefix_every_range_counts(gpu, dtype, B, n, H, Hkv, D, P, room):
    ops = _ops()
    ranges = _lib.lib().mi355_attn_shared_prefix_workspace_bytes(B, n, H, Hkv, D, P, room) // (B * n * H * (D + 2) * 4)
    assert ranges > 32 if P + room >= 256 * 32 + 256 else 0 < ranges <= 32
    kp, vp = blocks(P, Hkv, D, dtype, 1)
    own = [blocks(room, Hkv, D, dtype, 2 + b) for b in range(B)]
    lens = [room - b * (room // (B + 1)) for b in range(B)]
    out = ops.attention_shared_prefix(
        ones_q(B, n, H, D).to(dtype).to(gpu), kp.to(gpu), vp.to(gpu), torch.stack([k for k, _ in own]).to(gpu),
        torch.stack([v for _, v in own]).to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), scale=1.0)
    terms = 1 if B * n * H // Hkv > 64 else 2
    for b in sorted({0, B // 2, B - 1}):
        for t in sorted({0, n - 1}):
            for h in (0, H - 1):
                y = h * Hkv // H
                k, v = torch.cat((kp[:, y], own[b][0][:, y])), torch.cat((vp[:, y], own[b][1][:, y]))
                ref, tol, seen = weights64(k, v, P + max(0, lens[b] - n + t + 1), terms, dtype)
                assert seen > 3
                check(f"sequence {b} token {t} head {h}", out[b, t, h], ref, tol)


# ------------------------------------------------------------------------------ two terms
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["packed", "whole", "16 rows", "32 rows", "64 rows", "own"])
def test_probabilities_of_two_terms(gpu, dtype, form):
    """Where a probability enters P · V as two terms, the outputs are off by their own rounding alone. With V of both
    signs an output is about 1 / sqrt(n) of P |V| for n keys that count, and so is the sum of n roundings by u: one
    term would add as much again as the output's rounding, sqrt(2) of it in all, two add 2 u^2 of P |V|, below a tenth
    of it for n up to 40."""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    D, Hkv, room, P = 64, 2, 40, 1200 if form not in ("packed", "whole", "own") else 24
    B, H = {"16 rows": (3, 8), "32 rows": (6, 8), "64 rows": (12, 8)}.get(form, (3, 8))
    if form == "own":
        P, room = 0, 1300
    q = torch.randn(B, 1, H, D, generator=g).to(dtype)
    kp, vp = (torch.randn(P, Hkv, D, generator=g).to(dtype) for _ in range(2))
    ko, vo = (torch.randn(B, room, Hkv, D, generator=g).to(dtype) for _ in range(2))
    # all but 40 keys count nothing
    nothing = -3e4 if dtype == torch.float16 else -1e30
    kp[20 if P > 40 else P:, :, 0] = nothing
    ko[:, 40:, :, 0] = nothing
    q[..., 0] = 1
    lens = [20 if P > 40 else 16 if form == "whole" else room] * B
    args = [t.to(gpu) for t in (q, kp, vp, ko, vo)]
    if form == "packed":
        plan = ops.packed_plan([1] * B, [room] * B, heads=H, kv_heads=Hkv, head_dim=D, device=gpu)
        assert plan.counts[0] == 0
        out = ops.attention_packed(args[0][:, 0].contiguous(), args[3].flatten(0, 1), args[4].flatten(0, 1), plan)[:, None]
        P = 0
    else:
        out = ops.attention_shared_prefix(*args, torch.tensor(lens, dtype=torch.int32, device=gpu))
    ref = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            y = h * Hkv // H
            k, v = (torch.cat((a[:P, y], c[b, :lens[b], y])).double() for a, c in ((kp, ko), (vp, vo)))
            ref[b, 0, h] = torch.softmax(k @ q[b, 0, h].double() * D ** -0.5, 0) @ v
    err = (out.cpu().double() - ref).norm()
    rounding = (ref.to(dtype).double() - ref).norm()
    print(f"{form} {dtype}: {float(err / rounding):.4f}", flush=True)
    assert float(err) <= 1.1 * float(rounding)
