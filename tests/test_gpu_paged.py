"""Rotary positions, appending to a paged e4m3 cache and attention over its pages against plain arithmetic in 64 bits,
and the three together as generation steps use them. Error bounds stand at the formulas (paged_reference)."""
import math

import pytest
import torch

from paged_reference import (BLOCK, DTYPES, UNIT, attention64, block_scale, check, empty_cache, frequencies, packed,
                             rand, rotate64, values64)

pytestmark = pytest.mark.gpu


def _ops():
    from tiktok_techjam_2026_track3_amd import ops
    return ops


def on_gpu(cache):
    return _ops().PagedCache(*[t.cuda() for t in cache])


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def tables(lens, page, seed, spare=3):
    """(table [B, width], pages): every sequence has pages of its own, in any order."""
    width = max(1, -(-max([0, *lens]) // page)) + 1
    pages = len(lens) * width + spare
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:len(lens) * width].to(torch.int32).view(len(lens), width), pages


def widened(table, page):
    """The table with room for 2^17 tokens, of pages that do not exist: a call whose work is shared out evenly, whatever
    the lengths are."""
    return torch.cat((table, torch.full((table.shape[0], (1 << 17) // page - table.shape[1]), -1, dtype=torch.int32)), 1)


# rotary

@pytest.mark.parametrize("dtype", [*DTYPES, torch.float32])
@pytest.mark.parametrize("shape,rot,interleaved", [
    ((1, 1, 64), 64, False), ((3, 5, 128), 128, False), ((7, 1, 80), 32, True), ((2, 3, 80), 40, False), ((4, 2, 96), 48, True),
    ((5, 3, 6), 2, False), ((9, 2, 10), 6, True), ((33, 4, 256), 256, True), ((2, 17, 3, 64), 64, False), ((1, 300, 9, 128), 64, True),
    ((70, 1, 512), 512, False), ((3, 70, 192), 192, False), ((2, 3, 72), 24, False)])
def test_rotary(dtype, shape, rot, interleaved):
    ops = _ops()
    x = rand(shape, dtype, sum(shape))
    g = torch.Generator().manual_seed(rot)
    positions = torch.randint(-50, 3_000_000, shape[:-2], generator=g)
    plan = ops.rotary_plan(rot, interleaved=interleaved, amplitude=1.25)
    for inverse in (False, True):
        ref, tol = rotate64(x, positions, frequencies(rot), interleaved, 1.25, inverse)
        for pos in (positions.cuda(), positions.int().cuda()):
            check(ops.rotary(x.cuda(), pos, plan, inverse), ref, tol + UNIT[dtype] * ref.abs(), "rotary")
    y = x.cuda()
    assert ops.rotary(y, positions.cuda(), plan, out=y) is y  # in place
    check(y, *(lambda r, t: (r, t + UNIT[dtype] * r.abs()))(*rotate64(x, positions, frequencies(rot), interleaved, 1.25)))


@pytest.mark.parametrize("scaling", ["linear", "base", "parts", "freqs"])
def test_rotary_scalings(scaling):
    ops = _ops()
    f = frequencies(64)
    if scaling == "linear":
        want, kw = [x / 8 for x in f], dict(scaling="linear", factor=8.0)
    elif scaling == "base":
        want, kw = frequencies(64, 10000.0 * 8 ** (64 / 62)), dict(scaling="base", factor=8.0)
    elif scaling == "parts":
        want = []
        for x in f:
            r = 2048 * x / (2 * math.pi)
            g = min(1, max(0, (r - 1) / 3))
            want.append(x * (g + (1 - g) / 8))
        kw = dict(scaling="parts", factor=8.0, original=2048, slow=1.0, fast=4.0)
    else:
        want = [-3.0, 0.0, 100.0, 1e-9] * 8
        kw = dict(freqs=want)
    x = rand((50, 2, 64), torch.float32, 1)
    positions = torch.randint(0, 1_000_000, (50,), generator=torch.Generator().manual_seed(2))
    ref, tol = rotate64(x, positions, want)
    # (64-bit products on both sides: 2^-52 of an angle of up to 10^8)
    tol = tol + 1e-7 * max(1.0, max(map(abs, want))) * x.abs().amax(-1, keepdim=True)
    check(ops.rotary(x.cuda(), positions.cuda(), ops.rotary_plan(64, **kw)), ref, tol + UNIT[torch.float32] * ref.abs())


def test_rotary_far_positions():
    """A position of 2^31 and beyond: 64 bits of a double's frequency, 2^-53 relative, leave 2^-20 of a turn."""
    ops = _ops()
    x = rand((4, 1, 32), torch.float32, 3)
    positions = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 31 + 12345, 2 ** 31 - 2])
    ref, tol = rotate64(x, positions, frequencies(32))
    check(ops.rotary(x.cuda(), positions.cuda(), ops.rotary_plan(32)), ref, tol + 2.0 ** -17 * x.abs().amax(-1, keepdim=True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_views(dtype):
    """Queries and keys of a packed projection, a broadcast position, odd strides and bases, a strided output."""
    ops = _ops()
    plan = ops.rotary_plan(16)
    qkv = rand((6, 12, 32), dtype, 5).cuda()
    positions = torch.arange(6, device="cuda") + 100
    ref, tol = rotate64(qkv[:, :8].cpu(), positions.cpu(), frequencies(16))
    tol = tol + UNIT[dtype] * ref.abs()
    check(ops.rotary(qkv[:, :8], positions, plan), ref, tol)
    keep = qkv[:, 8:].clone()
    ops.rotary(qkv[:, :8], positions, plan, out=qkv[:, :8])
    check(qkv[:, :8], ref, tol)
    assert torch.equal(qkv[:, 8:], keep)
    flat = rand((6 * 101 + 3,), dtype, 6).cuda()
    x = torch.as_strided(flat, (6, 3, 32), (101, 33, 1), 1)
    ref, tol = rotate64(x.cpu(), positions.cpu(), frequencies(16))
    out = torch.zeros(6, 3, 2, 32, dtype=dtype, device="cuda")
    ops.rotary(x, positions, plan, out=out[:, :, 1])
    check(out[:, :, 1], ref, tol + UNIT[dtype] * ref.abs())
    assert not out[:, :, 0].any()
    x = rand((3, 4, 2, 32), dtype, 7).cuda().transpose(0, 1)  # [4, 3, 2, 32]
    positions = torch.arange(3, device="cuda").expand(4, 3)
    ref, tol = rotate64(x.cpu(), positions.cpu(), frequencies(16))
    check(ops.rotary(x, positions, plan), ref, tol + UNIT[dtype] * ref.abs())
    assert ops.rotary(x[:0], positions[:0], plan).shape == (0, 3, 2, 32)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_larger_than_the_caches(interleaved):
    """Outputs of 32 MiB and more are stored another way; the append's queries likewise, and to the same bits."""
    ops = _ops()
    T, H, D = 4100, 34, 128
    x = rand((T, H, D), torch.bfloat16, 50)
    positions = torch.arange(T) + 77
    plan = ops.rotary_plan(96, interleaved=interleaved)
    ref, tol = rotate64(x, positions, frequencies(96), interleaved)
    got = ops.rotary(x.cuda(), positions.cuda(), plan)
    check(got, ref, tol + UNIT[torch.bfloat16] * ref.abs())
    k = rand((T, 2, D), torch.bfloat16, 51).cuda()
    table = torch.arange(5, dtype=torch.int32, device="cuda")[None]
    cache = ops.paged_cache(5, 2, D, 1024)
    assert torch.equal(ops.paged_append(cache, k, k, ops.PagedBatch(table, i32([T + 77]), T), plan, x.cuda()), got)


def test_rotary_is_its_own_gradient():
    """The inverse is the transposed map: differences of sum(w y), and against autograd of the formula."""
    ops = _ops()
    plan = ops.rotary_plan(32, amplitude=0.75)
    x, w = rand((5, 2, 48), torch.float32, 8), rand((5, 2, 48), torch.float32, 9)
    positions = torch.arange(5) * 1000
    got = ops.rotary(w.cuda(), positions.cuda(), plan, inverse=True).cpu()
    leaf = x.double().requires_grad_()
    y, _ = rotate64(leaf, positions, frequencies(32), False, 0.75)
    (y * w.double()).sum().backward()
    _, tol = rotate64(w, positions, frequencies(32), False, 0.75)
    check(got, leaf.grad, tol + UNIT[torch.float32] * leaf.grad.abs())
    step = torch.zeros_like(x)
    for at in ((0, 0, 0), (2, 1, 17), (4, 0, 40)):
        step.zero_()
        step[at] = 1.0
        d = [(ops.rotary((x + e * step).cuda(), positions.cuda(), plan).cpu().double() * w).sum() for e in (1.0, -1.0)]
        # (the map is linear: a difference over a step of 2 is exact but for the roundings of about 100 terms)
        assert abs((d[0] - d[1]) / 2 - got[at]) <= 100 * 2.0 ** -20


# append

def append64(cache, k, v, table, lens, offsets, positions_freqs=None, interleaved=False, amplitude=1.0):
    """The cache (CPU tensors) after an append, with tolerances of K's values; V and scales are exact."""
    kb, vb, ks, vs = [t.clone() for t in cache]
    pages, _, page, D = kb.shape
    slack = torch.zeros(kb.shape, dtype=torch.float64)
    touched = torch.zeros(kb.shape[:3], dtype=torch.bool)
    kx = k.double()
    err = torch.zeros_like(kx)
    if positions_freqs is not None:
        pos = torch.cat([torch.arange(m - (offsets[b + 1] - offsets[b]), m) for b, m in enumerate(lens)])
        kx, err = rotate64(k[:len(pos)], pos, positions_freqs, interleaved, amplitude)
    want_k = values64(kb, ks)
    for b, m in enumerate(lens):
        n, first = offsets[b + 1] - offsets[b], offsets[b]
        for block in range(min(m - n, 0) // BLOCK, (m - 1) // BLOCK + 1):
            lo, hi = max(m - n, block * BLOCK), min(m, block * BLOCK + BLOCK)
            if hi <= lo or block < 0 or block * BLOCK // page >= table.shape[1]:
                continue
            at, row = int(table[b, block * BLOCK // page]), block * BLOCK % page
            if not 0 <= at < pages:
                continue
            i0, t0, t1 = first + lo - (m - n), lo - block * BLOCK, hi - block * BLOCK
            for h in range(kb.shape[1]):
                for new, e, bytes_, scales, exact in ((kx, err, kb, ks, False), (v.double(), None, vb, vs, True)):
                    x = new[i0:i0 + hi - lo, h]
                    finite = x[x.isfinite()].abs()
                    top = float(finite.max()) if finite.numel() else 0.0
                    s = block_scale(top)
                    if not exact:  # (a scale that the fp32 rotation's error decides says nothing)
                        near = e[i0:i0 + hi - lo, h]
                        assert block_scale(float((x.abs() + near).max())) == s == block_scale(float((x.abs() - near).max())), "pick another seed"
                    old = float(scales[at, h, row // BLOCK]) if t0 else 0.0
                    s = max(s, old)
                    if t0 and s > old:
                        part = bytes_[at, h, row:row + t0].float() * (old / s)
                        bytes_[at, h, row:row + t0] = part.to(torch.float8_e4m3fn)
                        if not exact:
                            want_k[at, h, row:row + t0] = bytes_[at, h, row:row + t0].double() * s
                    scales[at, h, row // BLOCK] = s
                    if exact:
                        y = (x / s).float()
                        y = torch.where(y.isinf(), math.nan, y)
                        bytes_[at, h, row + t0:row + t1] = y.to(torch.float8_e4m3fn)
                    else:
                        want_k[at, h, row + t0:row + t1] = x
                        slack[at, h, row + t0:row + t1] = torch.maximum(x.abs() * 2.0 ** -4, torch.tensor(s * 2.0 ** -10)) \
                            * (1 + 2.0 ** -16) + e[i0:i0 + hi - lo, h]
                        touched[at, h, row + t0:row + t1] = True
    return kb, vb, ks, vs, want_k, slack, touched


def check_cache(got, want):
    kb, vb, ks, vs, want_k, slack, touched = want
    assert torch.equal(got.k_scale.cpu(), ks) and torch.equal(got.v_scale.cpu(), vs)
    a, b = got.v.cpu().float(), vb.float()
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    bytes_ = got.k.cpu()
    assert torch.equal(bytes_.view(torch.uint8)[~touched], kb.view(torch.uint8)[~touched])
    check(values64(bytes_, ks)[touched], want_k[touched], slack[touched], "k")


APPENDS = [
    # new, lens, heads, kv_heads, D, page, rot
    ([1, 1, 1], [1, 17, 400], 8, 2, 64, 16, 64),
    ([1] * 70, list(range(1, 71)), 4, 4, 32, 32, 16),
    ([0, 5, 0, 33], [9, 5, 0, 100], 6, 3, 128, 64, 128),
    ([16, 17, 15, 1], [16, 33, 31, 32], 2, 1, 80, 16, 40),
    ([40, 7], [300, 7], 3, 1, 96, 128, 48),
    ([3, 2], [5, 40], 2, 2, 256, 1024, 256),
    ([9], [70], 4, 1, 192, 256, 8),
    ([2, 3], [12, 70], 5, 5, 16, 64, 16),
    ([50], [61], 2, 1, 48, 32, 32),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", APPENDS)
def test_append(dtype, interleaved, case):
    new, lens, H, kvh, D, page, rot = case
    ops = _ops()
    offsets = packed(new)
    T = offsets[-1]
    table, pages = tables(lens, page, T)
    cache = empty_cache(pages, kvh, page, D, seed=11)
    k, v, q = (rand((T, h, D), dtype, 20 + i, s) for i, (h, s) in enumerate(((kvh, 2.0), (kvh, 0.3), (H, 1.0))))
    plan = ops.rotary_plan(rot, interleaved=interleaved, amplitude=1.5)
    want = append64(cache, k, v, table, lens, offsets, frequencies(rot), interleaved, 1.5)
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(new, lens)])
    ref, tol = rotate64(q, pos, frequencies(rot), interleaved, 1.5)
    uniform = len(set(new)) == 1
    for off in ([None] if uniform else []) + [i32(offsets)]:
        dev = on_gpu(cache)
        batch = ops.PagedBatch(table.cuda(), i32(lens), max(new), off)
        got = ops.paged_append(dev, k.cuda(), v.cuda(), batch, plan, q.cuda())
        check(got, ref, tol + UNIT[dtype] * ref.abs(), "q")
        check_cache(dev, want)
        before = [t.view(torch.uint8).clone() for t in (dev.k, dev.v, dev.k_scale, dev.v_scale)]
        qg = q.cuda()
        assert ops.paged_append(dev, k.cuda(), v.cuda(), batch, plan, qg, q_out=qg) is qg  # the same again, in place
        assert torch.equal(qg, got)
        assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, (dev.k, dev.v, dev.k_scale, dev.v_scale)))
    # neither positions nor queries
    dev = on_gpu(cache)
    assert ops.paged_append(dev, k.cuda(), v.cuda(), ops.PagedBatch(table.cuda(), i32(lens), max(new), i32(offsets))) is None
    check_cache(dev, append64(cache, k, v, table, lens, offsets))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_values(dtype):
    """Zeros, infinities, NaN, the type's largest and least values, ties, and a scale that grows over its tokens."""
    ops = _ops()
    D, page = 32, 32
    top = torch.finfo(dtype).max
    rows = torch.zeros(9, 1, D)
    rows[1] = 1.0
    rows[2, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    rows[3] = torch.linspace(-1, 1, D)
    rows[4] = torch.arange(D) * 28.0  # steps and half steps
    rows[5] = 600.0
    rows[6] = top
    rows[7] = torch.finfo(dtype).smallest_normal
    rows[8] = math.inf
    v = rows.to(dtype)
    table, pages = tables([9], page, 1)
    cache = empty_cache(pages, 1, page, D, seed=3)
    for split in ([9], [1, 2, 3, 1, 1, 1], [1] * 9):
        dev, host, done = on_gpu(cache), cache, 0
        for n in split:
            done += n
            part = v[done - n:done].contiguous()
            want = append64(host, torch.zeros_like(part), part, table, [done], [0, n])
            ops.paged_append(dev, torch.zeros_like(part).cuda(), part.cuda(), ops.PagedBatch(table.cuda(), i32([done]), n))
            check_cache(dev, want)
            host = (dev.k.cpu(), *want[1:4])


def test_append_pages_that_do_not_exist():
    """Tokens without a page are not written, whatever the table says; nothing else changes."""
    ops = _ops()
    D, page, lens, new = 64, 16, [40, 200, 3, 20], [30, 5, 8, 4]
    table, pages = tables([64] * 4, page, 5)
    table[0, 1], table[0, 2], table[3, 1] = -1, pages, -2 ** 31
    cache = empty_cache(pages, 2, page, D, seed=4)
    offsets = packed(new)
    k, v, q = (rand((offsets[-1], 2, D), torch.bfloat16, 30 + i) for i in range(3))
    dev = on_gpu(cache)
    plan = ops.rotary_plan(64)
    got = ops.paged_append(dev, k.cuda(), v.cuda(), ops.PagedBatch(table.cuda(), i32(lens), 30, i32(offsets)), plan, q.cuda())
    check_cache(dev, append64(cache, k, v, table, lens, offsets, frequencies(64)))
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(new, lens)])
    ref, tol = rotate64(q, pos, frequencies(64))
    check(got, ref, tol + UNIT[torch.bfloat16] * ref.abs())


def test_append_rows_of_no_sequence():
    ops = _ops()
    table, pages = tables([20], 16, 6)
    cache = empty_cache(pages, 1, 16, 32)
    x = rand((9, 1, 32), torch.float16, 7).cuda()
    batch = ops.PagedBatch(table.cuda(), i32([20]), 5, i32([0, 4]))
    plan = ops.rotary_plan(32)
    dev = on_gpu(cache)
    got = ops.paged_append(dev, x, x.clone(), batch, plan, x.clone())
    assert got[:4].any() and not got[4:].any()
    out = torch.full_like(x, 5.0)
    ops.paged_append(dev, x, x.clone(), batch, plan, x.clone(), q_out=out)
    assert torch.equal(out[:4], got[:4]) and bool((out[4:] == 5.0).all())
    got = ops.attention_paged(x, dev, batch)
    assert got[:4].any() and not got[4:].any()
    out = torch.full_like(x, 5.0)
    ops.attention_paged(x, dev, batch, out=out)
    assert torch.equal(out[:4], got[:4]) and bool((out[4:] == 5.0).all())


# attention

ATTENDS = [
    # new, lens, heads, kv_heads, D, page
    ([1, 1, 1], [1, 17, 300], 8, 2, 64, 16),
    ([1], [33], 1, 1, 16, 16),
    ([1, 1], [700, 5], 4, 2, 32, 64),
    ([1] * 67, [3 + 7 * (i % 11) for i in range(67)], 4, 1, 48, 32),
    ([1, 1], [2500, 900], 8, 8, 128, 128),
    ([0, 5, 2, 0], [40, 5, 600, 0], 6, 3, 80, 16),
    ([3, 1], [2, 1], 4, 2, 64, 16),           # tokens before position 0
    ([7], [2000], 8, 1, 96, 256),
    ([1], [3000], 8, 2, 256, 64),
    ([6, 2], [700, 1], 12, 4, 192, 32),
    ([20, 33], [20, 400], 4, 1, 128, 16),
    ([100], [150], 2, 1, 64, 1024),
    ([1, 1], [0, 4], 2, 2, 64, 16),           # an empty sequence
    ([40, 1], [300, 1300], 8, 2, 256, 64),
    ([70, 3, 0, 41], [70, 900, 5, 1500], 6, 2, 128, 64),
    ([33], [5000], 1, 1, 192, 128),
    ([1] * 3, [5000, 40, 1024], 12, 3, 80, 16),
    ([200], [200], 4, 4, 48, 32),
    ([9, 1], [1100, 2080], 16, 4, 96, 256),
    ([17, 1, 2], [900, 2000, 2], 6, 2, 256, 32),
    ([90, 3], [90, 1400], 4, 2, 192, 16),
]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ATTENDS)
def test_attention(dtype, case, wide):
    new, lens, H, kvh, D, page = case
    ops = _ops()
    offsets = packed(new)
    table, pages = tables(lens, page, sum(lens))
    table = widened(table, page) if wide else table
    cache = empty_cache(pages, kvh, page, D, seed=5)
    q = rand((offsets[-1], H, D), dtype, 6, 1.5)
    ref, tol = attention64(q, cache, table, lens, offsets, D ** -0.5)
    dev = on_gpu(cache)
    for off in ([None] if len(set(new)) == 1 else []) + [i32(offsets)]:
        batch = ops.PagedBatch(table.cuda(), i32(lens), max(new), off)
        got = ops.attention_paged(q.cuda(), dev, batch)
        check(got, ref, tol, "attention")
        assert torch.equal(got, ops.attention_paged(q.cuda(), dev, batch))
    more = ops.PagedBatch(table.cuda(), i32(lens), max(new) + 40, i32(offsets))  # `most` need not be exact
    ref, tol = attention64(q, cache, table, lens, offsets, D ** -0.5, max(new) + 40)
    check(ops.attention_paged(q.cuda(), dev, more), ref, tol, "attention")


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_views(dtype):
    """Queries of a packed projection, a strided output, a scale of its own, a table that is part of a larger one."""
    ops = _ops()
    lens, D, page = [100, 37, 260], 64, 32
    table, pages = tables(lens, page, 8)
    cache = empty_cache(pages, 2, page, D, seed=9)
    qkv = rand((3, 8, D), dtype, 10).cuda()
    ref, tol = attention64(qkv[:, :4].cpu(), cache, table, lens, packed([1, 1, 1]), 0.3)
    big = torch.full((4, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    big[1:, 2:2 + table.shape[1]] = table.cuda()
    out = torch.zeros(3, 5, D + 4, dtype=dtype, device="cuda")
    batch = ops.PagedBatch(big[1:, 2:2 + table.shape[1]], i32(lens))
    got = ops.attention_paged(qkv[:, :4], on_gpu(cache), batch, 0.3, out=out[:, :4, :D])
    check(got, ref, tol)
    assert not out[:, 4].any() and not out[:, :, D:].any()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D", [64, 80, 128, 192, 256])
def test_attention_what_is_not_seen(D, wide, many):
    """Stale bytes behind a sequence's end and NaN in keys and values: only the tokens that see them change."""
    ops = _ops()
    page, lens, new = 16, [50, 700, 33], [3, 4, 2]
    table, pages = tables(lens, page, 12)
    own = table.shape[1]
    table = widened(table, page) if wide else table
    offsets = packed(new)
    cache = empty_cache(pages, 2, page, D, seed=13)
    q = rand((offsets[-1], 4, D), torch.bfloat16, 14)
    dev = on_gpu(cache)
    most = 40 if many else 4  # (more than 32 rows: another kernel)
    batch = ops.PagedBatch(table.cuda(), i32(lens), most, i32(offsets))
    clean = ops.attention_paged(q.cuda(), dev, batch)
    ref, tol = attention64(q, cache, table, lens, offsets, D ** -0.5, most)
    check(clean, ref, tol)
    for b, m in enumerate(lens):
        for p in range(m, own * page):
            for t in (dev.k, dev.v):
                t.view(torch.uint8)[int(table[b, p // page]), :, p % page] = 0x7f
        last = -(-m // BLOCK) * BLOCK  # scales of blocks behind the end
        for p in range(last, own * page, BLOCK):
            dev.k_scale[int(table[b, p // page]), :, p % page // BLOCK] = math.nan
            dev.v_scale[int(table[b, p // page]), :, p % page // BLOCK] = math.inf
    assert torch.equal(ops.attention_paged(q.cuda(), dev, batch), clean)
    # NaN in the newest value of each sequence: element 5 of the last token alone
    for b, m in enumerate(lens):
        dev.v.view(torch.uint8)[int(table[b, (m - 1) // page]), :, (m - 1) % page, 5] = 0xff
    got = ops.attention_paged(q.cuda(), dev, batch)
    rows = [offsets[b + 1] - 1 for b in range(3)]
    assert got[rows][:, :, 5].isnan().all()
    got[rows, :, 5] = clean[rows, :, 5]
    check(got, ref, tol)
    # NaN in its key too: the whole last token
    for b, m in enumerate(lens):
        dev.k.view(torch.uint8)[int(table[b, (m - 1) // page]), :, (m - 1) % page, 1] = 0x7f
    got = ops.attention_paged(q.cuda(), dev, batch)
    assert got[rows].isnan().all()
    got[rows] = clean[rows]
    check(got, ref, tol)
    # a NaN that everyone sees
    dev.v.view(torch.uint8)[int(table[1, 0]), 1, 3, 7] = 0x7f
    got = ops.attention_paged(q.cuda(), dev, batch)
    assert got[3:7, 2:, 7].isnan().all() and not got[3:6, :2].isnan().any() and not got[0:2].isnan().any()


@pytest.mark.parametrize("most", [6, 40])
def test_attention_pages_that_do_not_exist(most):
    ops = _ops()
    D, page, lens, new = 64, 16, [40, 40, 130, 30], [2, 2, 1, 6]
    table, pages = tables([64] * 4, page, 15)  # room for 80 tokens: the third sequence's 130 do not fit
    table[0, 1], table[3, 1], table[1, 4] = -1, pages, 2 ** 31 - 1  # (the last one is not reached)
    offsets = packed(new)
    lens[3] = 18  # tokens at positions 12 to 17: two of them see the page that is missing
    cache = empty_cache(pages, 2, page, D, seed=16)
    q = rand((offsets[-1], 2, D), torch.float16, 17)
    ref, tol = attention64(q, cache, table, lens, offsets, D ** -0.5, most)
    assert ref[:2].isnan().all() and not ref[2:4].isnan().any() and ref[4].isnan().all() and ref[9:].isnan().all()
    got = ops.attention_paged(q.cuda(), on_gpu(cache), ops.PagedBatch(table.cuda(), i32(lens), most, i32(offsets)))
    check(got, ref, tol)


@pytest.mark.parametrize("most", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_large_scores(dtype, most):
    """Scores far apart, all far from zero, and one that takes everything."""
    ops = _ops()
    D, page, lens = 64, 32, [600, 900]
    table, pages = tables(lens, page, 18)
    cache = empty_cache(pages, 1, page, D, seed=19)
    for factor in (30.0, 3000.0):
        q = rand((2, 4, D), dtype, 20, factor)
        ref, tol = attention64(q, cache, table, lens, packed([1, 1]), D ** -0.5, most)
        for t in (table, widened(table, page)):
            got = ops.attention_paged(q.cuda(), on_gpu(cache), ops.PagedBatch(t.cuda(), i32(lens), most, i32([0, 1, 2])))
            check(got, ref, tol)


@pytest.mark.parametrize("most", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_rows_beside_bad_ones(dtype, most):
    """Queries with NaN and infinities: their own outputs alone are NaN, and the other rows keep their bits."""
    ops = _ops()
    D, page, lens = 128, 32, [90, 1200]
    table, pages = tables(lens, page, 30)
    dev = on_gpu(empty_cache(pages, 2, page, D, seed=31))
    q = rand((2, 8, D), dtype, 32)
    for t in (table, widened(table, page)):
        batch = ops.PagedBatch(t.cuda(), i32(lens), most, i32([0, 1, 2]))
        clean = ops.attention_paged(q.cuda(), dev, batch)
        bad = q.clone()
        bad[0, 1, 3], bad[1, 4, 0], bad[1, 7, 127] = math.nan, math.inf, -math.inf
        got = ops.attention_paged(bad.cuda(), dev, batch)
        for r in ((0, 1), (1, 4), (1, 7)):
            assert got[r].isnan().all()
            got[r] = clean[r]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("most", [2, 40])
def test_lengths_and_offsets_that_make_no_sense(most):
    """Read on the device, checked there: nothing outside the tensors is touched, and a sequence that makes sense is right."""
    ops = _ops()
    D, page, lens = 64, 16, [2 ** 31 - 1, -2 ** 31, 60, -5, 2 ** 31 - 1]
    table, pages = tables([60] * 5, page, 33)
    table[4] = torch.tensor([2 ** 31 - 1, -2 ** 31, pages, -1, 2 ** 30])
    cache = empty_cache(pages, 2, page, D, seed=34)
    q, k = rand((9, 4, D), torch.float16, 35), rand((9, 2, D), torch.float16, 36)
    for offsets in ([-7, 2, 3, 5, 4, 2 ** 31 - 1], [0, 2, 3, 5, 7, 9], [2 ** 31 - 1, 0, 3, 5, -2 ** 31, 9]):
        # a row that two sequences name holds either's result (a start below 0 counts as 0)
        own = [r for r in (3, 4) if sum(max(a, 0) <= r < min(b, max(a, 0) + most) for a, b in zip(offsets, offsets[1:])) == 1]
        rows = [r - 3 for r in own]
        for t in (table, widened(table, page)):
            batch = ops.PagedBatch(t.cuda(), i32(lens), most, i32(offsets))
            dev = on_gpu(cache)
            got = ops.attention_paged(q.cuda(), dev, batch)
            ref, tol = attention64(q[3:5], cache, table[2:3], [60], [0, 2], D ** -0.5, most)
            check(got[own], ref[rows], tol[rows])
            turned = ops.paged_append(dev, k.cuda(), k.cuda(), batch, ops.rotary_plan(D), q.cuda())
            ref, tol = rotate64(q[3:5], torch.tensor([58, 59]), frequencies(D))
            check(turned[own], ref[rows], (tol + UNIT[torch.float16] * ref.abs())[rows])
            one = on_gpu(cache)
            ops.paged_append(one, k[3:5].cuda(), k[3:5].cuda(), ops.PagedBatch(table[2:3].cuda(), i32([60]), 2), ops.rotary_plan(D))
            at = int(table[2, 3])
            assert torch.equal(dev.k.view(torch.uint8)[at], one.k.view(torch.uint8)[at])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_prompt_rows_and_later_scales(D, dtype):
    """V far larger in later blocks, of the same 32 keys and behind them: rows that do not see those keep their digits."""
    ops = _ops()
    page, lens = 64, [80]
    table, pages = tables(lens, page, 43)
    cache = empty_cache(pages, 1, page, D, seed=44)
    scales = cache[3][table[0, :2].long(), 0].view(-1)  # of the sequence's blocks
    scales[:] = torch.tensor([2.0 ** e for e in (-12, 30, 30, -12, 60, 0, 0, 0)])
    cache[3][table[0, :2].long(), 0] = scales.view(2, -1)
    q = rand((80, 1, D), dtype, 45)
    for t in (table, widened(table, page)):
        got = ops.attention_paged(q.cuda(), on_gpu(cache), ops.PagedBatch(t.cuda(), i32(lens), 80))
        ref, tol = attention64(q[:16], cache, t, [16], [0, 16], D ** -0.5, 80)
        check(got[:16], ref, tol)
        if dtype == torch.bfloat16:  # (elsewhere the results leave the type)
            ref, tol = attention64(q, cache, t, lens, [0, 80], D ** -0.5)
            check(got, ref, tol)


@pytest.mark.parametrize("most", [3, 40])
def test_pools_beyond_32_bits(most):
    """K and V of more than 2^32 bytes each, and tables for more keys than the last-level cache holds: the same bits as
    from small pools and tables."""
    ops = _ops()
    D, page, H = 256, 1024, 8
    pages, width = 2100, 100
    cache = ops.paged_cache(pages, H, D, page)
    assert cache.k.numel() > 1 << 32
    lens = [2500, 9000]
    table = torch.full((2, width), -1, dtype=torch.int32)
    table[0, :3] = torch.tensor([2099, 2052, 7])
    table[1, :9] = torch.arange(2060, 2069)
    used = torch.cat((table[0, :3], table[1, :9])).long()
    small = ops.paged_cache(13, H, D, page)
    near = torch.full((2, 60), -1, dtype=torch.int32)
    near[0, :3], near[1, :9] = torch.arange(1, 4), torch.arange(4, 13)
    results = []
    for c, t in ((cache, table), (small, near)):
        g = torch.Generator(device="cuda").manual_seed(46)
        new = torch.randn(sum(lens), H, D, device="cuda", generator=g).half()
        ops.paged_append(c, new, new.flip(0), ops.PagedBatch(t.cuda(), i32(lens), max(lens), i32(packed(lens))), ops.rotary_plan(D))
        q = torch.randn(2 * most, H, D, device="cuda", generator=g).half()
        results.append(ops.attention_paged(q, c, ops.PagedBatch(t.cuda(), i32(lens), most)))
        at = used.cuda() if c is cache else torch.arange(1, 13, device="cuda")
        results[-1:] = [results[-1], c.k.view(torch.uint8)[at], c.v.view(torch.uint8)[at], c.k_scale[at], c.v_scale[at]]
    assert results[0].isfinite().all() and results[0].abs().max() > 0
    for a, b in zip(results[:5], results[5:]):
        assert torch.equal(a, b)
    used = set(used.tolist())
    others = torch.tensor([i for i in range(pages) if i not in used], device="cuda")
    assert cache.k_scale[others].abs().max() == 0 and cache.v_scale[others].abs().max() == 0


def test_many_sequences():
    """More than 64, and more than 1024, sequences; some without a token."""
    ops = _ops()
    D, page = 32, 16
    g = torch.Generator().manual_seed(37)
    for B in (130, 1500):
        new = torch.randint(0, 3, (B,), generator=g).tolist()
        lens = [n + int(torch.randint(0, 60, (1,), generator=g)) for n in new]
        offsets = packed(new)
        table, pages = tables(lens, page, B)
        cache = empty_cache(pages, 1, page, D, seed=38)
        q = rand((offsets[-1], 2, D), torch.bfloat16, 39)
        ref, tol = attention64(q, cache, table, lens, offsets, D ** -0.5)
        for t in (table, widened(table, page)) if B < 1000 else (table,):
            check(ops.attention_paged(q.cuda(), on_gpu(cache), ops.PagedBatch(t.cuda(), i32(lens), 2, i32(offsets))), ref, tol)


def test_append_in_place_on_a_packed_projection():
    """q, k and v as views of one buffer: queries rotated in place are refused only where they share elements."""
    ops = _ops()
    D, page = 64, 16
    table, pages = tables([40], page, 41)
    cache = on_gpu(empty_cache(pages, 2, page, D))
    plan = ops.rotary_plan(D)
    qkv = rand((5, 8, D), torch.bfloat16, 42).cuda()
    batch = ops.PagedBatch(table.cuda(), i32([40]), 5)
    want = ops.paged_append(cache, qkv[:, 4:6], qkv[:, 6:], batch, plan, qkv[:, :4])
    bytes_ = cache.k.view(torch.uint8).clone()
    keep = qkv[:, 4:].clone()
    ops.paged_append(cache, qkv[:, 4:6], qkv[:, 6:], batch, plan, qkv[:, :4], q_out=qkv[:, :4])
    assert torch.equal(qkv[:, :4], want) and torch.equal(qkv[:, 4:], keep) and torch.equal(cache.k.view(torch.uint8), bytes_)
    with pytest.raises(ValueError, match="shares memory"):
        ops.paged_append(cache, qkv[:, 3:5], qkv[:, 6:], batch, plan, qkv[:, :4], q_out=qkv[:, :4])
    with pytest.raises(ValueError, match="shares memory"):
        ops.paged_append(cache, qkv[:, 4:6], qkv[:, 6:], batch, plan, qkv[:, 1:5], q_out=qkv[:, :4])


def test_refusals_on_the_gpu():
    ops = _ops()
    D = 64
    cache = ops.paged_cache(4, 2, D, 16)
    x, kv = torch.zeros(2, 4, D, dtype=torch.float16, device="cuda"), torch.zeros(2, 2, D, dtype=torch.float16, device="cuda")
    batch = ops.PagedBatch(i32([[0], [1]]), i32([3, 4]))
    plan = ops.rotary_plan(D)
    cases = [
        (TypeError, lambda: ops.attention_paged(x.float(), cache, batch)),
        (ValueError, lambda: ops.attention_paged(x[:1], cache, batch)),
        (ValueError, lambda: ops.attention_paged(x, cache, batch, scale=0.0)),
        (ValueError, lambda: ops.attention_paged(x, cache, batch, out=x)),
        (ValueError, lambda: ops.attention_paged(x[..., :32], cache, batch)),
        (ValueError, lambda: ops.attention_paged(x.clone().requires_grad_(), cache, batch)),
        (ValueError, lambda: ops.attention_paged(x.cpu(), cache, batch)),
        (ValueError, lambda: ops.paged_append(cache, kv, kv, batch, None, x)),
        (ValueError, lambda: ops.paged_append(cache, kv, kv, batch, ops.rotary_plan(20), x)),
        (ValueError, lambda: ops.paged_append(cache, kv, kv, batch, ops.rotary_plan(128), x)),
        (ValueError, lambda: ops.paged_append(cache, kv, kv, batch, plan, q_out=x)),
        (ValueError, lambda: ops.paged_append(cache, kv, kv, batch, plan, x, q_out=x.transpose(0, 1))),
        (ValueError, lambda: ops.paged_append(cache, x, kv, batch)),
        (TypeError, lambda: ops.paged_append(cache, kv, kv.bfloat16(), batch)),
        (ValueError, lambda: ops.paged_append(cache, cache.k.view(torch.float16)[0, :, :2].transpose(0, 1)[..., :32].repeat(1, 1, 2), kv.requires_grad_(), batch)),
        (ValueError, lambda: ops.rotary(x, torch.arange(2, device="cuda"), plan, out=x[:, :, :].flip(0)[:1])),
        (ValueError, lambda: ops.rotary(x, torch.arange(3, device="cuda"), plan)),
        (ValueError, lambda: ops.rotary(x, torch.arange(2), plan)),
        (TypeError, lambda: ops.rotary(x, torch.arange(2, device="cuda"), plan, out=x.float())),
    ]
    for i, (error, call) in enumerate(cases):
        with pytest.raises(error):
            call()
            print("case", i)
    long = torch.zeros(3, 4, D, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        ops.rotary(long[:2], torch.arange(2, device="cuda"), plan, out=long[1:])
    whole = cache.k.view(torch.float16).view(-1)[:2 * 2 * D].view(2, 2, D)  # the cache's own bytes
    with pytest.raises(ValueError, match="shares memory"):
        ops.paged_append(cache, whole, torch.zeros_like(whole), batch)


def test_rows_of_no_sequence_in_a_long_buffer():
    """Packed tokens that end long before the buffer does: zeros behind them in new outputs, nothing in given ones."""
    ops = _ops()
    D, page, T = 64, 16, 5000
    table, pages = tables([50, 3], page, 47)
    cache = on_gpu(empty_cache(pages, 2, page, D, seed=48))
    q, kv, plan = rand((T, 4, D), torch.bfloat16, 49).cuda(), rand((T, 2, D), torch.bfloat16, 50).cuda(), ops.rotary_plan(D)
    batch, exact = (ops.PagedBatch(table.cuda(), i32([50, 3]), 6, o) for o in (i32([0, 4, 5]), i32([0, 4, 5])))
    trash = torch.full((T, 4, D), 7.0, dtype=torch.bfloat16, device="cuda")
    del trash  # (what a new output may be made of)
    turned = ops.paged_append(cache, kv, kv, batch, plan, q)
    given = ops.paged_append(cache, kv, kv, batch, plan, q, q_out=torch.full_like(q, 3.0))
    assert (turned[5:] == 0).all() and (given[5:] == 3).all() and torch.equal(turned[:5], given[:5])
    out = ops.attention_paged(turned, cache, batch)
    assert (out[5:] == 0).all() and torch.equal(out[:5], ops.attention_paged(turned[:5].clone(), cache, exact))


@pytest.mark.parametrize("most", [1, 40])
def test_pages_in_several_tables(most):
    """A shared beginning, and a page twice in one table."""
    ops = _ops()
    D, page, lens = 96, 32, [100, 130, 128]
    table = torch.tensor([[5, 2, 7, 1, 0], [5, 2, 7, 3, 6], [4, 4, 5, 4, 9]], dtype=torch.int32)
    cache = empty_cache(10, 2, page, D, seed=59)
    q = rand((3 * most, 4, D), torch.bfloat16, 60)
    ref, tol = attention64(q, cache, table, lens, [most * i for i in range(4)], D ** -0.5)
    for t in (table, widened(table, page)):
        check(ops.attention_paged(q.cuda(), on_gpu(cache), ops.PagedBatch(t.cuda(), i32(lens), most)), ref, tol)


def test_nothing_to_do():
    """No sequences, no rows, no new tokens, tables without columns."""
    ops = _ops()
    D, page = 64, 16
    cache = on_gpu(empty_cache(4, 2, page, D, seed=51))
    kept = cache.k.view(torch.uint8).clone(), cache.v.view(torch.uint8).clone()
    plan = ops.rotary_plan(D)
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    for T, batch in ((0, ops.PagedBatch(none, i32([]))), (5, ops.PagedBatch(none, i32([]), 3, i32([0]))),
                     (4, ops.PagedBatch(i32([[0], [1]]), i32([3, 9]), 2, i32([0, 0, 0]))),
                     (0, ops.PagedBatch(i32([[0], [1]]), i32([3, 9]), 0))):
        q, kv = rand((T, 4, D), torch.float16, 52).cuda(), rand((T, 2, D), torch.float16, 53).cuda()
        for got in (ops.attention_paged(q, cache, batch), ops.paged_append(cache, kv, kv, batch, plan, q)):
            assert got.shape == q.shape and not got.any()
        given = torch.full_like(q, 2.0)
        ops.attention_paged(q, cache, batch, out=given)
        ops.paged_append(cache, kv, kv, batch, plan, q, q_out=given)
        assert (given == 2).all()
    q, kv = rand((2, 4, D), torch.float16, 54).cuda(), rand((2, 2, D), torch.float16, 55).cuda()
    batch = ops.PagedBatch(torch.zeros(2, 0, dtype=torch.int32, device="cuda"), i32([1, 5]))
    assert ops.attention_paged(q, cache, batch).isnan().all()
    turned = ops.paged_append(cache, kv, kv, batch, plan, q)
    assert torch.equal(turned, ops.rotary(q, torch.tensor([0, 4], device="cuda"), plan))
    assert torch.equal(cache.k.view(torch.uint8), kept[0]) and torch.equal(cache.v.view(torch.uint8), kept[1])


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    ops = _ops()
    cache = on_gpu(empty_cache(2, 2, 16, 64, seed=56))
    batch = ops.PagedBatch(i32([[0], [1]]), i32([3, 4]))
    q, kv = rand((2, 4, 64), torch.float16, 57).cuda(), rand((2, 2, 64), torch.float16, 58).cuda()
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(ValueError):
            ops.attention_paged(dual, cache, batch)
        with pytest.raises(ValueError):
            ops.paged_append(cache, kv, kv, batch, ops.rotary_plan(64), dual)


# together

@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_generation_steps(dtype, wide):
    """Two prompts admitted into the cache, then steps of both (and a graph of one step, replayed with lengths that grow on
    the device), each against 64 bits over what the cache holds."""
    ops = _ops()
    H, kvh, D, page, rot = 8, 2, 64, 16, 64
    prompts = [37, 90]
    plan = ops.rotary_plan(rot)
    table, pages = tables([200, 200], page, 21)
    table = widened(table, page) if wide else table
    cache = ops.paged_cache(pages, kvh, D, page)
    table_gpu, lens = table.cuda(), i32(prompts)
    offsets = packed(prompts)
    qkv = rand((offsets[-1], H + 2 * kvh, D), dtype, 22).cuda()
    q, k, v = qkv[:, :H], qkv[:, H:H + kvh], qkv[:, H + kvh:]
    batch = ops.PagedBatch(table_gpu, lens, max(prompts), i32(offsets))
    turned = ops.paged_append(cache, k, v, batch, plan, q)
    out = ops.attention_paged(turned, cache, batch)
    host = [t.cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    ref, tol = attention64(turned.cpu(), host, table, prompts, offsets, D ** -0.5)
    check(out, ref, tol)
    # the cache's K is the rotated one: e4m3 is within 2^-4 of it, or half a least step of its block's scale
    positions = torch.cat([torch.arange(n) for n in prompts])
    kr, kt = rotate64(k.cpu(), positions, frequencies(rot))
    held = values64(host[0], host[2])
    for i in (0, 16, 36, 37, 100, 126):
        b, p = (0, i) if i < 37 else (1, i - 37)
        at = int(table[b, p // page])
        step = host[2][at, :, p % page // BLOCK].double()[:, None] * 2.0 ** -10
        assert ((held[at, :, p % page] - kr[i]).abs() <= kr[i].abs() * 2.0 ** -4 * 1.001 + step + kt[i]).all()

    step = ops.PagedBatch(table_gpu, lens)
    x = torch.zeros(2, H + 2 * kvh, D, dtype=dtype, device="cuda")

    def one():
        lens.add_(1)
        t = ops.paged_append(cache, x[:, H:H + kvh], x[:, H + kvh:], step, plan, x[:, :H])
        return t, ops.attention_paged(t, cache, step)

    graph = None
    for i in range(12):
        x.copy_(rand(x.shape, dtype, 100 + i))
        if i == 3:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            keep = lens.clone()
            with torch.cuda.graph(graph):
                t, o = one()
            lens.copy_(keep)
        if graph is None:
            t, o = one()
        else:
            graph.replay()
            torch.cuda.synchronize()
        host = [a.cpu() for a in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        now = [n + i + 1 for n in prompts]
        assert lens.tolist() == now
        ref, tol = rotate64(x[:, :H].cpu(), torch.tensor(now) - 1, frequencies(rot))
        check(t, ref, tol + UNIT[dtype] * ref.abs(), "queries")
        ref, tol = attention64(t.cpu(), host, table, now, [0, 1, 2], D ** -0.5)
        check(o, ref, tol, "step %d" % i)
        eager = ops.attention_paged(t, cache, step)  # eager work between replays
        assert torch.equal(eager, o)


@pytest.mark.parametrize("wide", [False, True])
def test_side_stream_and_two_at_once(wide):
    ops = _ops()
    lens, D, page = [3000, 1000], 128, 64
    table, pages = tables(lens, page, 23)
    table = widened(table, page) if wide else table
    dev = on_gpu(empty_cache(pages, 2, page, D, seed=24))
    batch = ops.PagedBatch(table.cuda(), i32(lens))
    q = [rand((2, 8, D), torch.bfloat16, 25 + i).cuda() for i in range(2)]
    want = [ops.attention_paged(x, dev, batch) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.attention_paged(q[i], dev, batch))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
