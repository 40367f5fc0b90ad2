"""The paged cache's operators at their edges, against plain arithmetic in 64 bits (paged_reference) and themselves."""

import math
from decimal import Decimal, localcontext

import pytest
import torch

from paged_edges_reference import pi_of
from paged_reference import DTYPES, UNIT, attention64, check, empty_cache, rand

pytestmark = pytest.mark.gpu


def _ops():
    from tiktok_techjam_2026_track3_amd import ops
    return ops


def on_gpu(cache):
    return _ops().PagedCache(*[t.cuda() for t in cache])


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def tables(tokens, page, seed, wide):
    """(table, pages): every sequence has pages of its own for so many tokens, in any order; wide: with room for 2^17 tokens of
    pages that do not exist, so that the work is shared out evenly."""
    width = max(1, -(-max(tokens) // page))
    pages = len(tokens) * width + 2
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(pages, generator=g)[:len(tokens) * width].to(torch.int32).view(len(tokens), width)
    if wide:
        table = torch.cat((table, torch.full((len(tokens), (1 << 17) // page - width), -1, dtype=torch.int32)), 1)
    return table, pages


def poison(q):
    """Fills and frees memory that a new output of q's size may be made of."""
    trash = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    del trash


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("B", [3, 70])
@pytest.mark.parametrize("most,D", [(3, 64), (40, 64), (40, 192), (40, 256), (3, 256)])
def test_more_tokens_than_most(most, D, B, wide):
    """Those behind the first `most` of a sequence are left out, as if neither the offsets nor the lengths counted them;
    their rows, and those before the first sequence's, are zeros in new outputs and left in given ones."""
    ops = _ops()
    page = 16
    rng = torch.Generator().manual_seed(70)
    new = [most + 300, 2, most, 0, most + 1][:B] + [int(n) for n in torch.randint(0, most + 3, (max(0, B - 5),), generator=rng)]
    offsets = [4]
    for n in new:
        offsets.append(offsets[-1] + n)
    T = offsets[-1] + 5
    cut = [max(0, n - most) for n in new]
    lens = [n + 7 + 11 * (b % 4) for b, n in enumerate(new)]
    kept_lens = [m - c for m, c in zip(lens, cut)]
    kept = [r for a, n, c in zip(offsets, new, cut) for r in range(a, a + n - c)]
    packed = [0]
    for n, c in zip(new, cut):
        packed.append(packed[-1] + n - c)
    others = sorted(set(range(T)) - set(kept))
    table, pages = tables(kept_lens, page, 71, wide)
    cache = empty_cache(pages, 2, page, D, seed=72)
    q, k, v = rand((T, 4, D), torch.bfloat16, 73).cuda(), rand((T, 2, D), torch.bfloat16, 74).cuda(), rand((T, 2, D), torch.bfloat16, 75).cuda()
    plan = ops.rotary_plan(D)
    batch = ops.PagedBatch(table.cuda(), i32(lens), most, i32(offsets))
    alone = ops.PagedBatch(table.cuda(), i32(kept_lens), most, i32(packed))
    dev, want = on_gpu(cache), on_gpu(cache)
    ref = ops.paged_append(want, k[kept], v[kept], alone, plan, q[kept])
    poison(q)
    turned = ops.paged_append(dev, k, v, batch, plan, q)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(dev, name).view(torch.uint8), getattr(want, name).view(torch.uint8)), name
    assert torch.equal(turned[kept], ref) and not turned[others].any()
    given = ops.paged_append(on_gpu(cache), k, v, batch, plan, q, q_out=torch.full_like(q, 3.0))
    assert torch.equal(given[kept], ref) and (given[others] == 3).all()

    poison(q)
    out = ops.attention_paged(turned, dev, batch)
    assert not out[others].any()
    cpu = tuple(getattr(want, name).cpu() for name in ("k", "v", "k_scale", "v_scale"))
    check(out[kept], *attention64(ref.cpu(), cpu, table, kept_lens, packed, D ** -0.5, most))
    assert torch.equal(out[kept], ops.attention_paged(ref, want, alone))
    given = ops.attention_paged(turned, dev, batch, out=torch.full_like(q, 3.0))
    assert torch.equal(given[kept], out[kept]) and (given[others] == 3).all()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("most,D", [(3, 64), (40, 64), (40, 256)])
def test_more_tokens_than_most_in_replays(most, D, wide):
    """A captured step whose offsets and lengths outgrow `most` later, and come back."""
    ops = _ops()
    page, T = 16, 2 * most + 20
    table, pages = tables([150, 150], page, 76, wide)
    plan = ops.rotary_plan(D)
    q, kv = rand((T, 4, D), torch.float16, 77).cuda(), rand((T, 2, D), torch.float16, 78).cuda()
    cache = empty_cache(pages, 2, page, D, seed=79)
    dev = on_gpu(cache)
    lens, offsets = i32([100, 90]), i32([0, most, 2 * most])
    batch = ops.PagedBatch(table.cuda(), lens, most, offsets)

    def step(c):
        turned = ops.paged_append(c, kv, kv, batch, plan, q)
        return turned, ops.attention_paged(turned, c, batch)

    step(dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, out = step(dev)
    for at, n in (([0, most, 2 * most], [100, 90]), ([0, most + 9, 2 * most + 10], [101, 95]), ([2, 3, 2 * most + 20], [60, 120]),
                  ([0, most, 2 * most], [100, 90]), ([0, 2 * most + 20, 2 * most + 20], [130, 5])):
        lens.copy_(i32(n))
        offsets.copy_(i32(at))
        graph.replay()
        torch.cuda.synchronize()
        got = turned.clone(), out.clone()
        others = [r for r in range(T) if not any(a <= r < min(b, a + most) for a, b in zip(at, at[1:]))]
        assert not got[0][others].any() and not got[1][others].any()
        copy = ops.PagedCache(dev.k.clone(), dev.v.clone(), dev.k_scale.clone(), dev.v_scale.clone())
        eager = step(copy)
        assert torch.equal(got[0], eager[0])
        assert torch.equal(got[1], eager[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("most", [1, 3, 40])
def test_rows_beside_far_scores_keep_their_bits(dtype, wide, most):
    """A row's result does not depend on the scores of the other rows of its tile: neither on how far they are from 0 nor on
    when their maximum moves (fp16 queries become infinities with the largest factor, and their rows NaN)."""
    ops = _ops()
    D, page, lens = 128, 64, [3000, 517]
    table, pages = tables(lens, page, 90, wide)
    k, v, ks, vs = empty_cache(pages, 2, page, D, seed=91)
    cache = on_gpu((k, v, ks * 64, vs))
    batch = ops.PagedBatch(table.cuda(), i32(lens), most)
    q = 0.05 * rand((2 * most, 16, D), torch.float32, 92)
    changed = [(0, 1), (0, 6), (most, 0), (most, 12), (2 * most - 1, 15)]
    others = torch.ones(2 * most, 16, dtype=torch.bool)
    for at in changed:
        others[at] = False
    want = ops.attention_paged(q.to(dtype).cuda(), cache, batch)
    for factor in (0.1, 3.0, 30.0, 1e5, 6e5):
        other = q.clone()
        for at in changed:
            other[at] *= factor
        got = ops.attention_paged(other.to(dtype).cuda(), cache, batch)
        assert torch.equal(got[others.cuda()], want[others.cuda()]), factor


def lifted(ref, tol, sees, top):
    """attention64's bound for fp16 probabilities that are rounded once, with 2^-33 of the largest one as their smallest half
    step (2^8 times the running maximum's is their unit, 2^-25 fp16's half step) in place of 2^-25."""
    return ref, tol - sees * top * (2.0 ** -25 - 2.0 ** -33)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D", [64, 256])
def test_keys_far_below_a_sink(D, wide):
    """A key of no value 18 and 20 (in e's powers) above 12000 others: what those weigh together is not lost."""
    ops = _ops()
    page, keys, most = 64, 12000, 40
    table, pages = tables([keys], page, 80, wide)
    k, v, ks, vs = empty_cache(pages, 1, page, D)
    ks.fill_(1.0)
    vs.fill_(0.125)
    k.copy_(rand(k.shape, torch.float32, 81).to(k.dtype))
    v.copy_((2 + rand(v.shape, torch.float32, 82)).to(v.dtype))
    k[..., 0] = torch.zeros(()).to(k.dtype)
    sink = int(table[0, 0])
    k[sink, 0, 0] = torch.zeros(D).to(k.dtype)
    k[sink, 0, 0, 0] = torch.tensor(16.0).to(k.dtype)
    v[sink, 0, 0] = torch.zeros(D).to(v.dtype)
    q = 0.02 * rand((most, 1, D), torch.float32, 83)
    q[::2, 0, 0], q[1::2, 0, 0] = 18.0, 20.0
    q = q.half()
    scale, cache = 0.0625, (k, v, ks, vs)
    got = ops.attention_paged(q.cuda(), on_gpu(cache), ops.PagedBatch(table.cuda(), i32([keys]), most), scale=scale)
    ref, tol = lifted(*attention64(q, cache, table, [keys], [0, most], scale), keys, float((v.float().abs().amax() * 0.125)))
    assert (tol < 0.25 * ref.abs()).double().mean() > 0.5  # (the bound is well below what it measures)
    check(got, ref, tol)
    few = torch.cat([ops.attention_paged(q[i:i + 8].cuda(), on_gpu(cache), ops.PagedBatch(table.cuda(), i32([keys - most + i + 8]), 8), scale=scale)
                     for i in range(0, most, 8)])
    check(few, ref, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("far,step", [(0, 1), (2 ** 22, 1), (2 ** 25, 4), (-2 ** 26, 8)])
@pytest.mark.parametrize("most", [1, 40])
def test_scores_that_rise(dtype, far, step, most):
    """Whole scores (2's powers) that rise by up to 16 from a unit of 32 keys to the next, near 0 and far from it: exact in fp32,
    so that a weight is off by its exponential's 2^-20 and its own rounding, and none may overflow its type."""
    ops = _ops()
    D, page = 64, 32
    rises = [0, 7, 8, 6, 14, 15, 16, 9, 1, 0, 12, 13, 15, 7, 8, 15, 16, 14, 0, 3, 15, 15, 8, 7]
    keys = page * len(rises)
    table, pages = tables([keys], page, 84, False)
    k, v, ks, vs = empty_cache(pages, 1, page, D)
    ks.fill_(1.0)
    vs.fill_(2.0 ** -3)
    v.copy_((448 * torch.rand(v.shape, generator=torch.Generator().manual_seed(85))).to(v.dtype))
    at, score = 0, []  # in steps
    for u, r in enumerate(rises):
        at += -(-r // step)
        row = torch.zeros(D)
        row[0], row[1], row[2] = at // 16, at % 16, 256
        k[table[0, u].long(), 0] = row.to(k.dtype)
        score += [at * step] * page
    q = torch.zeros(most, 1, D)
    q[..., 0], q[..., 1], q[..., 2] = 16, 1, far / step / 256
    got = ops.attention_paged(q.to(dtype).cuda(), on_gpu((k, v, ks, vs)), ops.PagedBatch(table.cuda(), i32([keys]), most),
                              scale=math.log(2.0) * step).double().cpu()
    score = torch.tensor(score, dtype=torch.float64)
    values = v.double()[table[0].long(), 0].reshape(keys, D) * 2.0 ** -3
    many = most > 32
    for i in range(most):
        sees = keys - most + i + 1
        w = torch.softmax(score[:sees] * math.log(2.0), 0)
        ref = w @ values[:sees]
        rel = (2 * UNIT[dtype] if many else 2.0 ** -16) + 2 * 2.0 ** -20 + sees * 2.0 ** -23 + UNIT[dtype]
        tol = rel * ref + (sees * 2.0 ** (-25 if abs(far) >= 2 ** 24 else -33) * 56 if many and dtype == torch.float16 else 0.0)
        assert ((got[i, 0] - ref).abs() <= tol).all(), (i, got[i, 0, :4], ref[:4], tol[:4])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("most", [2, 40])
def test_mantissas_of_v_scales_do_not_count(dtype, most):
    ops = _ops()
    D, page, lens = 128, 32, [300, 77]
    table, pages = tables(lens, page, 86, False)
    k, v, ks, vs = empty_cache(pages, 2, page, D, seed=87)
    q = rand((2 * most, 4, D), dtype, 88).cuda()
    batch = ops.PagedBatch(table.cuda(), i32(lens), most)
    want = ops.attention_paged(q, on_gpu((k, v, ks, vs)), batch)
    factor = 1 + 0.99 * torch.rand(vs.shape, generator=torch.Generator().manual_seed(89))
    assert torch.equal(ops.attention_paged(q, on_gpu((k, v, ks, vs * factor)), batch), want)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("B,most", [(129, 16384), (129, 1 << 20), (300, 1 << 20)])
def test_a_large_bound_on_the_new_tokens(B, most, wide):
    """Many sequences of which one may have a long piece: what counts is how many tokens there are."""
    ops = _ops()
    D, page = 32, 16
    new = [1] * B
    new[57] = 150
    lens = [n + 3 + 13 * (b % 5) for b, n in enumerate(new)]
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    table, pages = tables(lens, page, 93, False)
    cache = empty_cache(pages, 2, page, D, seed=94)
    if wide:
        table = torch.cat((table, torch.full((len(lens), 200), -1, dtype=torch.int32)), 1)
    q, k, v = (rand((offsets[-1], h, D), torch.float16, 95 + h) for h in (4, 2, 2))
    batch = ops.PagedBatch(table.cuda(), i32(lens), most, i32(offsets))
    dev, want, plan = on_gpu(cache), on_gpu(cache), ops.rotary_plan(D)
    if most == 16384:
        turned = ops.paged_append(dev, k.cuda(), v.cuda(), batch, plan, q.cuda())
        ref = ops.paged_append(want, k.cuda(), v.cuda(), ops.PagedBatch(table.cuda(), i32(lens), 150, i32(offsets)), plan, q.cuda())
        assert torch.equal(turned, ref) and torch.equal(dev.k.view(torch.uint8), want.k.view(torch.uint8))
        assert torch.equal(dev.v.view(torch.uint8), want.v.view(torch.uint8))
    cpu = tuple(t.cpu() for t in (dev.k, dev.v, dev.k_scale, dev.v_scale))
    check(ops.attention_paged(q.cuda(), dev, batch), *attention64(q, cpu, table, lens, offsets, D ** -0.5, most))


@pytest.mark.parametrize("base,dim", [(10000.0, 64), (500000.0, 128)])
def test_rotary_positions_up_to_2_33(base, dim):
    """Angles are off by 2^-31 of a turn at most: sines and cosines of their exact values, against the kernel's."""
    ops = _ops()
    positions = [2 ** 33, -2 ** 33, 2 ** 33 - 12345, 2 ** 31 + 7, -2 ** 31, 2 ** 26 + 1, 10 ** 6, 3]
    x = rand((len(positions), 1, dim), torch.float32, 96)
    pi, h = pi_of(60), dim // 2
    with localcontext() as c:
        c.prec = 60
        turns = [(Decimal(base).ln() * -2 * j / dim).exp() / (2 * pi) for j in range(h)]
        angle = torch.tensor([[float((p * t) % 1 * 2 * pi) for t in turns] for p in positions], dtype=torch.float64)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., :h].double(), x[..., h:].double()
    ref = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    # 2 pi 2^-31 of the angle; 2^-21 as in rotate64; the output's rounding
    tol = (2.0 ** -28 + 2.0 ** -21) * (a.abs() + b.abs()).repeat(1, 1, 2) + UNIT[torch.float32] * ref.abs()
    got = ops.rotary(x.cuda(), torch.tensor(positions).cuda(), ops.rotary_plan(dim, base))
    check(got, ref, tol)


def test_caches_that_require_gradients_are_refused():
    ops = _ops()
    x, kv = (torch.zeros(1, h, 64, dtype=torch.float16, device="cuda") for h in (4, 2))
    batch, plan = ops.PagedBatch(i32([[0]]), i32([1])), ops.rotary_plan(64)
    for at in range(4):
        parts = [t.cuda() for t in empty_cache(2, 2, 16, 64)]
        parts[at].requires_grad_()
        cache = ops.PagedCache(*parts)
        for call in (lambda: ops.attention_paged(x, cache, batch), lambda: ops.paged_append(cache, kv, kv, batch, plan, x)):
            with pytest.raises(ValueError, match="no backward"):
                call()
            with torch.no_grad():
                call()


def test_caches_with_tangents_are_refused():
    from torch.autograd import forward_ad
    ops = _ops()
    x, kv = (torch.zeros(1, h, 64, dtype=torch.float16, device="cuda") for h in (4, 2))
    batch, plan = ops.PagedBatch(i32([[0]]), i32([1])), ops.rotary_plan(64)
    k, v, ks, vs = (t.cuda() for t in empty_cache(2, 2, 16, 64))
    with torch.no_grad(), forward_ad.dual_level():
        cache = ops.PagedCache(k, v, ks, forward_ad.make_dual(vs, torch.ones_like(vs)))
        for call in (lambda: ops.attention_paged(x, cache, batch), lambda: ops.paged_append(cache, kv, kv, batch, plan, x)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


def test_an_append_of_more_rows_than_the_attention_takes():
    """2^23 rows of queries and more in one call: the same as in two, and as the rotation alone in fp32. That one is rounded to
    fp32 (2^-24 of it), ours to fp16 (2^-11, below 2^-14 2^-25) either from there or from the sum as it is: the compiler's
    choice, so that fp16 results of the two kernels can be neighbours where fp32 has the middle between them."""
    ops = _ops()
    D, page, T, H, cut = 16, 1024, 270001, 32, 100000
    assert T * H > 1 << 23
    width = -(-T // page)
    table = torch.randperm(width, generator=torch.Generator().manual_seed(97)).to(torch.int32)[None].cuda()
    g = torch.Generator(device="cuda").manual_seed(98)
    q, k, v = (torch.randn(T, h, D, device="cuda", generator=g).half() for h in (H, 1, 1))
    plan, one, two = ops.rotary_plan(D), ops.paged_cache(width, 1, D, page), ops.paged_cache(width, 1, D, page)
    turned = ops.paged_append(one, k, v, ops.PagedBatch(table, i32([T]), T), plan, q)
    for a, b in ((0, cut), (cut, T)):
        part = ops.paged_append(two, k[a:b], v[a:b], ops.PagedBatch(table, i32([b]), b - a), plan, q[a:b])
        assert torch.equal(part, turned[a:b])
    for a in range(0, T, 1 << 16):
        part = ops.rotary(q[a:a + (1 << 16)].float(), torch.arange(a, min(T, a + (1 << 16)), device="cuda"), plan).double()
        tol = (UNIT[torch.float16] + 2.0 ** -23) * part.abs() + 2.0 ** -25
        assert ((turned[a:a + (1 << 16)].double() - part).abs() <= tol).all()
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(one, name).view(torch.uint8), getattr(two, name).view(torch.uint8))
