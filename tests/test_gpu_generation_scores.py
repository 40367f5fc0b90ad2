"""Token-generation attention at scores of every size: finite ones give finite outputs, however large.

Scores are exact here (one element of q and of K that is not 0, powers of two and 1.5 times those), and any two that
differ, and whose product with log2 e is 2^24 or more, differ by millions. Error bounds (u = half a step of a type): 2 u of
P |V| for probabilities taken as one term, 2 u^2 as two (fp16: 2^-24 a key), 2^-18 for exponents down to -32 and the
exponential, for the sums over n keys (32 at a time, one after the other, and at most 512 ranges) 2 (n / 32 + 544) 2^-24,
the output u |ref|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16]


def _ops():
    from tiktok_techjam_2026_track3_amd import ops
    return ops


def check(name, out, ref, tol):
    worst = float(((out.cpu().double() - ref).abs() / tol).max())
    print(f"{name}: worst err/bound {worst:.3f}", flush=True)
    assert worst <= 1.0, name


def far_inputs(rows, keys, D, Hkv, dtype, seed):
    """q of one element, 1 to 2^14 (bf16 2^60) from row to row, K of one, +-1 or 1.5 times a power of two up to that."""
    g = torch.Generator().manual_seed(seed)
    most = 14 if dtype == torch.float16 else 60
    q, k = torch.zeros(rows, D), torch.zeros(keys, Hkv, D)
    q[:, 0] = 2.0 ** ((torch.arange(rows) * 4) % (most + 1)).float()
    size = torch.randint(-most // 2, most + 1, (keys, Hkv), generator=g) - most // 2 * (torch.rand(keys, Hkv, generator=g) < 0.9)
    k[:, :, 0] = (1 + torch.randint(0, 2, (keys, Hkv), generator=g) / 2) * 2.0 ** size * (1 - 2 * torch.randint(0, 2, (keys, Hkv), generator=g))
    return q.to(dtype), k.to(dtype), torch.randn(keys, Hkv, D, generator=g).to(dtype)


def far64(q, k, v, last, terms, dtype):
    s = q[:, :1].double() @ k[:, :1].double().t()
    s[torch.arange(k.shape[0])[None] >= last[:, None]] = -math.inf
    p = torch.nan_to_num(torch.softmax(s, 1))
    ref, pv = p @ v.double(), p @ v.double().abs()
    least = k.shape[0] * 2.0 ** -24 * v.double().abs().max() if dtype == torch.float16 else 0.0
    return ref, (2 * UNIT[dtype] ** terms + 2.0 ** -18 + (k.shape[0] / 32 + 544) * 2.0 ** -23) * pv + least + UNIT[dtype] * ref.abs() + 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("q_lens,k_lens,H,Hkv,terms", [([150] * 20, [150] * 20, 16, 16, 1), ([200, 40], [200, 47], 4, 2, 1),
                                                       ([7, 16], [130, 77], 4, 2, 2), ([40], [4000], 4, 2, 1), ([3], [3000], 4, 2, 2)])
def test_packed_scores_of_every_size(gpu, dtype, D, sign, q_lens, k_lens, H, Hkv, terms):
    """Finite scores give finite outputs, however large: what is taken off them is not rounded away from them. With
    sign -1 all of the keys a row sees first are far below 0."""
    ops = _ops()
    T = sum(q_lens)
    q, k, v = far_inputs(T * H, sum(k_lens), D, Hkv, dtype, T)
    if sign < 0:
        k = -k.abs()
    q = q.view(T, H, D)
    plan = ops.packed_plan(q_lens, k_lens, heads=H, kv_heads=Hkv, head_dim=D, device=gpu)
    out = ops.attention_packed(q.to(gpu), k.to(gpu), v.to(gpu), plan, scale=1.0).cpu()
    q0 = k0 = 0
    for i, (n, m) in enumerate(zip(q_lens, k_lens)):
        for h in (0, H - 1) if i < 4 else ():
            y = h * Hkv // H
            ref, tol = far64(q[q0:q0 + n, h], k[k0:k0 + m, y], v[k0:k0 + m, y], torch.arange(n) + m - n + 1, terms, dtype)
            check(f"sequence {i} head {h}", out[q0:q0 + n, h], ref, tol)
        q0, k0 = q0 + n, k0 + m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("B,n,H,Hkv,P,room", [(2, 1, 8, 2, 300, 200), (2, 1, 8, 2, 1500, 200), (4, 1, 16, 2, 1500, 200), (3, 4, 8, 2, 1500, 200), (9, 2, 16, 2, 1500, 200)])
def test_prefix_scores_of_every_size(gpu, dtype, sign, B, n, H, Hkv, P, room):
    ops = _ops()
    D = 64
    q, kp, vp = far_inputs(B * n * H, P, D, Hkv, dtype, 1)
    q = q.view(B, n, H, D)
    _, ko, vo = far_inputs(1, B * room, D, Hkv, dtype, 2)
    ko, vo = ko.view(B, room, Hkv, D), vo.view(B, room, Hkv, D)
    if sign < 0:
        kp, ko = -kp.abs(), -ko.abs()
    lens = [room - 30 * b % room for b in range(B)]
    out = ops.attention_shared_prefix(*(t.to(gpu) for t in (q, kp, vp, ko, vo)), torch.tensor(lens, dtype=torch.int32, device=gpu), scale=1.0).cpu()
    terms = 1 if B * n * H // Hkv > 64 else 2
    for b in range(B):
        for h in (0, H - 1):
            y = h * Hkv // H
            ref, tol = far64(q[b, :, h], torch.cat((kp[:, y], ko[b, :lens[b], y])), torch.cat((vp[:, y], vo[b, :lens[b], y])),
                             torch.arange(n) + P + lens[b] - n + 1, terms, dtype)
            check(f"sequence {b} head {h}", out[b, :, h], ref, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,P", [(4, 300), (4, 1500), (40, 1500)])
@pytest.mark.parametrize("huge", [2.0 ** 14, math.inf])
def test_rows_beside_large_scores_keep_their_bits(gpu, dtype, B, P, huge):
    """A sequence whose scores are huge or infinite is a row beside others of the batch: theirs stay as they are."""
    ops = _ops()
    H, Hkv, D, room = 4, 2, 64, 100
    g = torch.Generator().manual_seed(B + P)
    q, kp, vp, ko, vo = (torch.randn(*s, generator=g).to(dtype).to(gpu) for s in (
        (B, 1, H, D), (P, Hkv, D), (P, Hkv, D), (B, room, Hkv, D), (B, room, Hkv, D)))
    lens = torch.full((B,), room, dtype=torch.int32, device=gpu)
    clean = ops.attention_shared_prefix(q, kp * 100, vp, ko * 100, vo, lens, scale=1.0)
    q2 = q.clone()
    q2[1] *= huge
    out = ops.attention_shared_prefix(q2, kp * 100, vp, ko * 100, vo, lens, scale=1.0)
    keep = [b for b in range(B) if b != 1]
    assert torch.equal(out[keep], clean[keep])
    assert bool(torch.isfinite(out[1]).all()) == (huge < math.inf)
