"""The operators of token generation against plain implementations in 64 bits: attention over packed
prompts with grouped heads, attention of new tokens behind a shared prefix, projections with 4-bit
weights, and the three together as a generation step uses them.

Error bounds, from the roundings of the operators (u = half a step of a type):
  attention: a probability is rounded to u_p (2^-8 bf16, 2^-11 fp16; fp16 ones below 2^-14 to 2^-25) and
    enters the numerator and the sum, so 2 u_p (P |V|), where P |V| = sum_j p_j |v_j|; its exponent
    c s - mu carries (D + 3) 2^-24 c max_j sum_d |q_d k_jd| and the exponential 2^-22, both twice in
    the same way; fp32 sums over n keys n 2^-23; the output u_out |ref|.
  projection: fp32 sums of K terms, K 2^-24 on sum_k |x| (magic + 15 + |z|) s (the operands carry
    1024 or 128 until the zero point is taken off; fp16 takes it off exactly before, so 15 + |z|), and
    the output u_out |ref|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DTYPES = [torch.float16, torch.bfloat16]


def _ops():
    from tiktok_techjam_2026_track3_amd import ops
    return ops


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def attention64(q, k, v, last, scale):
    """Rows q [n, D] over keys k, v [m, D]: row i sees keys j < last[i]. Returns (ref, error bound)."""
    dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    n, m, D = q.shape[0], k.shape[0], q.shape[1]
    if m == 0 or n == 0:
        return torch.zeros(n, D, dtype=torch.float64), torch.zeros(n, D, dtype=torch.float64)
    seen = torch.arange(m)[None, :] < last[:, None]
    s = torch.where(seen, q @ k.t() * scale, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, 1))  # (rows that see nothing)
    vs = torch.where(seen.any(0)[:, None], v, 0.0)
    ref = p @ vs
    c = scale * 1.4427
    score = (D + 3) * 2.0 ** -24 * c * (torch.where(seen, q.abs() @ k.abs().t(), 0.0).amax(1))
    pv = p @ vs.abs()
    rel = 2 * UNIT[dtype] + 2 * (2.0 ** -22 + score) + m * 2.0 ** -23
    small = m * 2.0 ** -25 * vs.abs().max() if dtype == torch.float16 else 0.0
    return ref, rel[:, None] * pv + small + UNIT[dtype] * ref.abs() + 2.0 ** -24


def packed64(q, k, v, q_lens, k_lens, causal, scale):
    ref = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros_like(ref)
    g = q.shape[1] // max(1, k.shape[1])
    q0 = k0 = 0
    for n, m in zip(q_lens, k_lens):
        last = torch.arange(n) + m - n + 1 if causal else torch.full((n,), m)
        for h in range(q.shape[1]):
            ref[q0:q0 + n, h], tol[q0:q0 + n, h] = attention64(
                q[q0:q0 + n, h], k[k0:k0 + m, h // g], v[k0:k0 + m, h // g], last, scale)
        q0, k0 = q0 + n, k0 + m
    return ref, tol


def check(name, out, ref, tol):
    out = out.detach().cpu().double()
    assert out.shape == ref.shape
    assert bool(torch.isfinite(out).all()), f"{name}: not finite"
    err = (out - ref).abs()
    worst = float((err / tol.clamp_min(1e-30)).max()) if err.numel() else 0.0
    print(f"{name}: max err {float(err.max()) if err.numel() else 0:.3g}, worst err/bound {worst:.3f}", flush=True)
    assert worst <= 1.0


# ------------------------------------------------------------------------------ packed prompts
def run_packed(gpu, dtype, q_lens, k_lens, H, Hkv, D, causal, seed=1, scale=None):
    ops = _ops()
    q = _rand((sum(q_lens), H, D), dtype, seed)
    k = _rand((sum(k_lens), Hkv, D), dtype, seed + 1)
    v = _rand((sum(k_lens), Hkv, D), dtype, seed + 2)
    plan = ops.packed_plan(q_lens, k_lens, heads=H, kv_heads=Hkv, head_dim=D, causal=causal, device=gpu)
    out = ops.attention_packed(q.to(gpu), k.to(gpu), v.to(gpu), plan, scale=scale)
    ref, tol = packed64(q, k, v, q_lens, k_lens, causal, scale or D ** -0.5)
    check(f"packed {dtype} D={D} H={H}/{Hkv} q={q_lens} k={k_lens} causal={causal} counts={list(plan.counts)}", out, ref, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_head_dims(gpu, dtype, D, causal):
    """Every head dim, sequences that end inside row and key tiles, a single token, an empty one."""
    run_packed(gpu, dtype, [37, 1, 0, 130, 64], [37, 1, 0, 130, 64], 4, 2, D, causal)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 1), (5, 5), (8, 1), (12, 4), (64, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_groups(gpu, H, Hkv, causal):
    """Groups that do not divide a tile of rows, and one whose token is a tile of its own."""
    run_packed(gpu, torch.bfloat16, [33, 7, 65], [33, 7, 65], H, Hkv, 64, causal, seed=5)


@pytest.mark.parametrize("q_lens,k_lens", [
    ([1, 1, 1], [1, 77, 300]),        # single tokens
    ([5, 40], [133, 40 + 511]),       # pieces of a prompt against a longer context
    ([40, 9, 3], [7, 0, 3]),          # more tokens than keys: the first see nothing; no keys at all
    ([0, 0], [0, 5]), ([], []),
])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_lengths(gpu, dtype, q_lens, k_lens, causal):
    run_packed(gpu, dtype, q_lens, k_lens, 6, 2, 64, causal, seed=9)


@pytest.mark.parametrize("dtype,D,H,Hkv", [(torch.bfloat16, 128, 16, 4), (torch.float16, 64, 24, 8), (torch.float16, 256, 16, 8),
                                          (torch.bfloat16, 80, 16, 16), (torch.float16, 16, 16, 8), (torch.bfloat16, 32, 16, 8),
                                          (torch.float16, 48, 16, 8), (torch.float16, 96, 16, 8), (torch.bfloat16, 192, 16, 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_large_tiles(gpu, dtype, D, H, Hkv, causal):
    """Enough rows for the large tiles, tiles that end inside a sequence's rows and keys."""
    q_lens = [1025, 700, 2, 511]
    k_lens = [1025, 1003, 66, 511]
    ops = _ops()
    plan = ops.packed_plan(q_lens * 4, k_lens * 4, heads=H, kv_heads=Hkv, head_dim=D, causal=causal, device=gpu)
    assert plan.tile_rows == 128
    q, k, v = (_rand((sum(n) * 4, h, D), dtype, 20 + i) for i, (n, h) in enumerate([(q_lens, H), (k_lens, Hkv), (k_lens, Hkv)]))
    out = ops.attention_packed(q.to(gpu), k.to(gpu), v.to(gpu), plan).cpu()
    # a head of each group of the first and the last sequences
    q0 = k0 = 0
    for i, (n, m) in enumerate(zip(q_lens * 4, k_lens * 4)):
        if i in (0, 1, 2, 15):
            for h in (0, H - 1):
                last = torch.arange(n) + m - n + 1 if causal else torch.full((n,), m)
                ref, tol = attention64(q[q0:q0 + n, h], k[k0:k0 + m, h * Hkv // H], v[k0:k0 + m, h * Hkv // H], last, D ** -0.5)
                check(f"sequence {i} head {h}", out[q0:q0 + n, h], ref, tol)
        q0, k0 = q0 + n, k0 + m


@pytest.mark.parametrize("D", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_lens,k_lens", [
    ([1], [20001]),                      # one token, many ranges
    ([3, 1, 2], [5000, 1, 0]),           # few rows, split and whole, one without keys
    ([70], [4001]),                      # wide tiles in ranges; the last rows' range reaches furthest
    ([90, 2, 200], [3000, 2500, 150]),   # both lists; more tokens than keys
])
def test_packed_split_keys(gpu, dtype, D, q_lens, k_lens):
    """Few rows against many keys: tiles in ranges of keys that are joined, also where causal rows end
    before a range."""
    ops = _ops()
    assert ops.packed_plan(q_lens, k_lens, heads=4, kv_heads=2, head_dim=D, device=gpu).counts[2] > 0
    run_packed(gpu, dtype, q_lens, k_lens, 4, 2, D, True, seed=17)
    run_packed(gpu, dtype, q_lens, k_lens, 4, 2, D, False, seed=18)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_packed_split_what_a_row_does_not_see(gpu, bad):
    """... and a later token's not-finite K and V, in a range that some rows of the tile see nothing of."""
    ops = _ops()
    n, m, H, D = 40, 4000, 4, 64
    q, k, v = _rand((n, H, D), torch.float16, 71), _rand((m, 2, D), torch.float16, 72), _rand((m, 2, D), torch.float16, 73)
    plan = ops.packed_plan([n], [m], heads=H, kv_heads=2, head_dim=D, device=gpu)
    assert plan.counts[2] > 0
    ref, tol = packed64(q, k, v, [n], [m], True, D ** -0.5)
    k[m - 1, :, 0], v[m - 1] = bad, bad
    out = ops.attention_packed(q.to(gpu), k.to(gpu), v.to(gpu), plan).cpu()
    check("rows before it", out[:n - 1], ref[:n - 1], tol[:n - 1])
    assert not bool(torch.isfinite(out[n - 1]).any())
    k[:], v[m - 1] = 0, 0  # every score of the first rows' keys -inf: NaN
    k[:, :, 0] = -math.inf
    out = ops.attention_packed(torch.ones_like(q).to(gpu), k.to(gpu), v.to(gpu), plan).cpu()
    assert bool(torch.isnan(out).all())


@pytest.mark.parametrize("scale", [0.02, 1.0, 6.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_scales(gpu, dtype, scale):
    """From nearly uniform rows to rows that one key takes (the running maximum moves by far)."""
    run_packed(gpu, dtype, [300], [300], 2, 1, 64, True, seed=31, scale=scale)


def test_packed_views_and_rows_behind(gpu):
    """q, k, v as views of one projection, an output with head and token gaps; rows behind the last
    token, and the gaps, stay as they were; a larger q than the plan's tokens."""
    ops = _ops()
    H, Hkv, D, lens = 4, 2, 64, [19, 50]
    T = sum(lens)
    x = _rand((T + 5, (H + 2 * Hkv) * D + 24), torch.float16, 41).to(gpu)
    q = x[:, :H * D].view(T + 5, H, D)
    k = x[:, H * D:(H + Hkv) * D].view(T + 5, Hkv, D)
    v = x[:, (H + Hkv) * D:(H + 2 * Hkv) * D].view(T + 5, Hkv, D)
    buf = torch.full((T + 5, H, D + 4), 7.0, device=gpu, dtype=torch.float16)
    plan = ops.packed_plan(lens, heads=H, kv_heads=Hkv, head_dim=D, device=gpu)
    got = ops.attention_packed(q, k, v, plan, out=buf[..., :D])
    assert got.data_ptr() == buf.data_ptr()
    ref, tol = packed64(q.cpu()[:T], k.cpu()[:T], v.cpu()[:T], lens, lens, True, D ** -0.5)
    check("views", buf[:T, :, :D], ref, tol)
    assert bool((buf[T:] == 7.0).all()) and bool((buf[..., D:] == 7.0).all())
    assert bool((ops.attention_packed(q, k, v, plan)[T:] == 0).all())
    # a head of k / v that all heads share through a stride of 0
    one = k[:, :1].expand(T + 5, Hkv, D)
    out = ops.attention_packed(q, one, one, plan)[:T]
    ref, tol = packed64(q.cpu()[:T], one.cpu()[:T], one.cpu()[:T], lens, lens, True, D ** -0.5)
    check("one shared head", out, ref, tol)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_what_a_row_does_not_see(gpu, dtype, bad):
    """Not-finite K and V of a later token (in the same tile of keys and in a later one) reach only the
    rows that see it; the next sequence's and those behind the last never do."""
    ops = _ops()
    H, Hkv, D, lens = 4, 2, 64, [100, 41]
    T = sum(lens)
    q, k, v = _rand((T, H, D), dtype, 51), _rand((T + 3, Hkv, D), dtype, 52), _rand((T + 3, Hkv, D), dtype, 53)
    plan = ops.packed_plan(lens, heads=H, kv_heads=Hkv, head_dim=D, device=gpu)
    for at in (20, 99, 100, 120):
        k2, v2 = k.clone(), v.clone()
        k2[at, :, 3], v2[at] = bad, bad
        k2[T:], v2[T:] = bad, bad
        out = ops.attention_packed(q.to(gpu), k2.to(gpu), v2.to(gpu), plan).cpu()
        first = at  # the token itself is the first that sees it
        end = 100 if at < 100 else T
        clean = [i for i in range(T) if not first <= i < end]
        ref, tol = packed64(q, k[:T], v[:T], lens, lens, True, D ** -0.5)
        check(f"{bad} at {at}", out[clean], ref[clean], tol[clean])
        if bad != bad:
            assert bool(torch.isnan(out[first:end]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_infinite_scores(gpu, dtype):
    """Scores of -inf are probability 0; a row of nothing else is NaN, as softmax's; NaN in a query
    stays in its row."""
    ops = _ops()
    D, n = 32, 70
    q, k, v = torch.ones(n, 1, D).to(dtype), _rand((n, 1, D), dtype, 61), _rand((n, 1, D), dtype, 62)
    k[:40, 0, 0] = -math.inf
    k[45, 0, 0] = -math.inf
    q[66, 0, 5] = math.nan
    plan = ops.packed_plan([n], heads=1, kv_heads=1, head_dim=D, device=gpu)
    out = ops.attention_packed(q.to(gpu), k.to(gpu), v.to(gpu), plan).cpu()
    assert bool(torch.isnan(out[:40]).all()) and bool(torch.isnan(out[66]).all())
    keep = [j for j in range(40, n) if j != 45]
    for i in (40, 45, 46, 65, 67, 69):
        seen = [j for j in keep if j <= i]
        ref, tol = attention64(q[i:i + 1, 0], k[seen, 0], v[seen, 0], torch.tensor([len(seen)]), D ** -0.5)
        check(f"row {i}", out[i:i + 1, 0], ref, tol)


def test_packed_same_bits_again_and_on_another_stream(gpu):
    ops = _ops()
    lens = [300, 17, 64]
    q, k, v = (_rand((sum(lens), h, 128), torch.bfloat16, 70 + h).to(gpu) for h in (8, 2, 4))
    v = v[:, :2]
    plan = ops.packed_plan(lens, heads=8, kv_heads=2, head_dim=128, device=gpu)
    first = ops.attention_packed(q, k, v, plan)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = ops.attention_packed(q, k, v, plan)
    side.synchronize()
    assert torch.equal(first, again)
    # a sequence's rows do not depend on its neighbours
    alone = ops.packed_plan([17], heads=8, kv_heads=2, head_dim=128, device=gpu)
    assert torch.equal(ops.attention_packed(q[300:317], k[300:317], v[300:317], alone), first[300:317])


def test_packed_graph_replay(gpu):
    ops = _ops()
    lens = [90, 31]
    plan = ops.packed_plan(lens, heads=4, kv_heads=4, head_dim=64, device=gpu)
    q, k, v = (_rand((sum(lens), 4, 64), torch.float16, 80 + i).to(gpu) for i in range(3))
    out = torch.empty_like(q)
    ops.attention_packed(q, k, v, plan, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_packed(q, k, v, plan, out=out)
    for i in range(3):
        q.copy_(_rand(q.shape, q.dtype, 90 + i))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attention_packed(q, k, v, plan))


# ------------------------------------------------------------------------------ shared prefix
def prefix64(q, kp, vp, ko, vo, lens, scale):
    B, n, H, D = q.shape
    g, P = H // kp.shape[1], kp.shape[0]
    ref, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        m = min(max(int(lens[b]), 0), ko.shape[1])
        last = (torch.arange(n) + m - n + 1).clamp_min(0) + P
        for h in range(H):
            k = torch.cat((kp[:, h // g], ko[b, :m, h // g]))
            v = torch.cat((vp[:, h // g], vo[b, :m, h // g]))
            ref[b, :, h], tol[b, :, h] = attention64(q[b, :, h], k, v, last, scale)
    return ref, tol


def run_prefix(gpu, dtype, B, n, H, Hkv, D, P, room, lens, seed=1, behind=None):
    ops = _ops()
    q = _rand((B, n, H, D), dtype, seed)
    kp, vp = _rand((P, Hkv, D), dtype, seed + 1), _rand((P, Hkv, D), dtype, seed + 2)
    ko, vo = _rand((B, room, Hkv, D), dtype, seed + 3), _rand((B, room, Hkv, D), dtype, seed + 4)
    ref, tol = prefix64(q, kp, vp, ko, vo, lens, D ** -0.5)
    if behind is not None:  # what the caches hold behind their lengths
        for b in range(B):
            m = min(max(lens[b], 0), room)
            ko[b, m:], vo[b, m:] = behind, behind
    out = ops.attention_shared_prefix(*(t.to(gpu) for t in (q, kp, vp, ko, vo)),
                                      torch.tensor(lens, dtype=torch.int32, device=gpu))
    check(f"prefix {dtype} B={B} n={n} H={H}/{Hkv} D={D} P={P} room={room} lens={lens}", out, ref, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("P", [333, 1333])
def test_prefix_head_dims(gpu, dtype, D, P):
    """Prefix and cache by one work-group (up to 1024 keys), and in ranges that are joined."""
    run_prefix(gpu, dtype, 3, 1, 4, 2, D, P, 130, [130, 1, 64], behind=math.nan)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,n,H,Hkv", [(1, 1, 1, 1), (2, 1, 32, 2), (9, 1, 8, 2), (20, 1, 8, 2), (40, 1, 8, 2), (5, 3, 12, 2),
                                       (2, 40, 4, 4)])
@pytest.mark.parametrize("P", [500, 1500])
def test_prefix_row_tiles(gpu, D, B, n, H, Hkv, P):
    """Batches and groups that fill 16, 32, 64 and several 128 rows of the prefix, and own rows of one
    tile and of several."""
    g = torch.Generator().manual_seed(B * n)
    lens = [int(x) for x in torch.randint(n, 101, (B,), generator=g)]
    run_prefix(gpu, torch.bfloat16, B, n, H, Hkv, D, P, 100, lens, seed=B, behind=math.inf)


@pytest.mark.parametrize("P,room,lens", [
    (0, 40, [0, 1, 40]),       # no prefix; a sequence without a key gives zeros
    (77, 0, [0, 0, 0]),        # no caches
    (0, 0, [0, 0, 0]),
    (1, 1, [1, 0, 1]),
    (129, 65, [-3, 70, 65]),   # lengths outside [0, room] are clamped
    (1290, 65, [-3, 70, 65]),
    (0, 3000, [2999, 0, 1]),
    (64, 4000, [3999, 5, 2049]),  # several splits of a cache, most of them empty
    (5000, 16, [16, 3, 0]),
])
@pytest.mark.parametrize("n", [1, 4])
def test_prefix_lengths(gpu, P, room, lens, n):
    run_prefix(gpu, torch.float16, 3, n, 8, 2, 64, P, room, lens, seed=7, behind=math.nan)


@pytest.mark.parametrize("B,n", [(2, 40), (600, 1)])
def test_prefix_without_any_keys(gpu, B, n):
    """Neither prefix nor caches, where rows or work-groups are too many for one launch of whole rows."""
    ops = _ops()
    q = _rand((B, n, 4, 64), torch.bfloat16, 1).to(gpu)
    none, caches = q.new_empty(0, 2, 64), q.new_empty(B, 0, 2, 64)
    out = torch.full_like(q, math.nan)
    ops.attention_shared_prefix(q, none, none, caches, caches, torch.zeros(B, dtype=torch.int32, device=gpu), out=out)
    assert not out.any()


@pytest.mark.parametrize("P", [200, 1200])
def test_prefix_strides_and_out(gpu, P):
    """Caches as views of one buffer for K and V, a strided query and output."""
    ops = _ops()
    B, n, H, Hkv, D, room = 4, 2, 8, 4, 64, 96
    cache = _rand((B, room, 2, Hkv, D), torch.bfloat16, 11).to(gpu)
    pre = _rand((2, Hkv, P, D), torch.bfloat16, 12).to(gpu)  # head-major
    kp, vp = (pre[i].transpose(0, 1) for i in range(2))
    q = _rand((B, n, H + 3, D), torch.bfloat16, 13).to(gpu)[:, :, :H]
    buf = torch.full((B, n + 1, H, D), 3.0, device=gpu, dtype=torch.bfloat16)
    lens = [96, 2, 50, 33]
    lt = torch.tensor(lens, dtype=torch.int32, device=gpu)
    ops.attention_shared_prefix(q, kp, vp, cache[:, :, 0], cache[:, :, 1], lt, out=buf[:, :n])
    ref, tol = prefix64(q.cpu(), kp.cpu(), vp.cpu(), cache[:, :, 0].cpu(), cache[:, :, 1].cpu(), lens, D ** -0.5)
    check("strides", buf[:, :n], ref, tol)
    assert bool((buf[:, n:] == 3.0).all())


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("P", [0, 100, 1100])
def test_prefix_later_tokens(gpu, bad, P):
    """A not-finite V of the last new token does not reach the new tokens before it."""
    ops = _ops()
    B, n, H, D, room = 2, 3, 4, 64, 50
    q, kp, vp, ko, vo = (_rand(s, torch.float16, 21 + i) for i, s in enumerate(
        [(B, n, H, D), (P, 2, D), (P, 2, D), (B, room, 2, D), (B, room, 2, D)]))
    lens = [50, 17]
    ref, tol = prefix64(q, kp, vp, ko, vo, lens, D ** -0.5)
    for b in range(B):
        ko[b, lens[b] - 1, :, 0], vo[b, lens[b] - 1] = bad, bad
    out = ops.attention_shared_prefix(*(t.to(gpu) for t in (q, kp, vp, ko, vo)),
                                      torch.tensor(lens, dtype=torch.int32, device=gpu)).cpu()
    check("earlier tokens", out[:, :2], ref[:, :2], tol[:, :2])
    assert not bool(torch.isfinite(out[:, 2]).any())


@pytest.mark.parametrize("at", ["prefix", "own"])
@pytest.mark.parametrize("P", [70, 1070])
def test_prefix_infinite_scores(gpu, at, P):
    """A range of keys with no finite score counts nothing; a row with none at all is NaN."""
    ops = _ops()
    B, H, D, room = 2, 2, 32, 40
    q = torch.ones(B, 1, H, D).half()
    kp, vp, ko, vo = (_rand(s, torch.float16, 31 + i) for i, s in enumerate([(P, 2, D), (P, 2, D), (B, room, 2, D), (B, room, 2, D)]))
    lens = [40, 0]
    if at == "prefix":
        kp[:, :, 0] = -math.inf
    else:
        ko[:, :, :, 0] = -math.inf
    out = ops.attention_shared_prefix(*(t.to(gpu) for t in (q, kp, vp, ko, vo)),
                                      torch.tensor(lens, dtype=torch.int32, device=gpu)).cpu()
    for b in range(B):
        for h in range(H):
            k, v = (ko[b, :lens[b], h], vo[b, :lens[b], h]) if at == "prefix" else (kp[:, h], vp[:, h])
            if k.shape[0] == 0:
                assert bool(torch.isnan(out[b, 0, h]).all())
                continue
            ref, tol = attention64(q[b, :, h], k, v, torch.tensor([k.shape[0]]), D ** -0.5)
            check(f"{at} {b} {h}", out[b, :, h], ref, tol)


@pytest.mark.parametrize("P", [300, 3000])
def test_prefix_graph_follows_lengths(gpu, P):
    """A captured step replayed while the caches grow, beside a second graph and eager calls."""
    ops = _ops()
    B, H, D, room = 5, 8, 64, 200

    def inputs(seed):
        return [_rand(s, torch.float16, seed + i).to(gpu) for i, s in enumerate(
            [(B, 1, H, D), (P, 2, D), (P, 2, D), (B, room, 2, D), (B, room, 2, D)])]

    sets = [inputs(100), inputs(200)]
    lens = [torch.tensor([1, 5, 9, 0, 20], dtype=torch.int32, device=gpu) for _ in sets]
    outs, graphs = [], []
    for args, n in zip(sets, lens):
        ops.attention_shared_prefix(*args, n)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.attention_shared_prefix(*args, n))
        graphs.append(graph)
    for i in range(4):
        for args, n in zip(sets, lens):
            n.add_(30)
            args[0].copy_(_rand(args[0].shape, torch.float16, 300 + i))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for args, n, out in zip(sets, lens, outs):
            assert torch.equal(out, ops.attention_shared_prefix(*args, n))


# ------------------------------------------------------------------------------ 4-bit projections
def weights(N, K, group, zeros, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scale = (torch.rand(N, K // group, generator=g) + 0.2).to(dtype)
    zero = torch.randint(0, 256 if zeros == "any" else 16, (N, K // group), generator=g, dtype=torch.uint8) if zeros else None
    return w, scale, zero


def linear64(x, w, scale, zero, bias, group, out_dtype):
    N, K = w.shape[0], 2 * w.shape[1]
    q = torch.stack((w & 15, w >> 4), -1).reshape(N, K).double()
    z = (zero.double() if zero is not None else torch.full(scale.shape, 8.0, dtype=torch.float64)).repeat_interleave(group, 1)
    s = scale.double().repeat_interleave(group, 1)
    x = x.double()
    ref = x @ ((q - z) * s).t() + (bias.double() if bias is not None else 0.0)
    magic = 0 if scale.dtype == torch.float16 else 128
    # the zero point is taken off twice at most (sum and correction), each sum rounded K times
    tol = 2 * (K + 8) * 2.0 ** -24 * (x.abs() @ ((magic + 15 + z) * s).t()) + (UNIT[out_dtype] + 2.0 ** -23) * ref.abs() + 2.0 ** -24
    return ref, tol


def run_i4(gpu, dtype, M, N, K, group, zeros=True, bias=True, out_dtype=None, seed=1):
    ops = _ops()
    x = _rand((M, K), dtype, seed)
    w, scale, zero = weights(N, K, group, zeros, dtype, seed)
    b = _rand((N,), torch.float32, seed + 1) if bias else None
    out = ops.linear_i4(x.to(gpu), w.to(gpu), scale.to(gpu), zero.to(gpu) if zero is not None else None,
                        b.to(gpu) if bias else None, out_dtype=out_dtype)
    assert out.dtype == (out_dtype or dtype)
    ref, tol = linear64(x, w, scale, zero, b, group, out.dtype)
    check(f"i4 {dtype} M={M} N={N} K={K} group={group} zeros={zeros}", out, ref, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [None, "4 bits", "any"])
def test_i4_groups(gpu, dtype, group, zeros):
    """K that ends inside a step of 128, features that end inside a tile."""
    run_i4(gpu, dtype, 3, 101, 5 * group, group, zeros, seed=group)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,group", [(1, 1, 32, 32), (1, 16, 128, 128), (2, 17, 96, 32), (15, 33, 4096, 128),
                                         (16, 300, 2048, 64), (17, 64, 1024, 128), (33, 40, 544, 32), (64, 96, 8192, 64),
                                         (65, 50, 256, 128), (200, 31, 192, 64), (1, 17000, 256, 128), (5, 1000, 11008, 128),
                                         # one to four rows in registers: each of its numbers of chunks and waves
                                         (1, 7, 512, 128), (1, 300, 2048, 64), (1, 101, 4096, 32), (1, 30, 8192, 128), (1, 18, 16384, 32),
                                         (2, 33, 2016, 32), (2, 50, 2176, 128), (2, 20, 6144, 64), (2, 9, 16384, 64), (3, 21, 1024, 32),
                                         (4, 77, 4064, 32), (3, 50, 8064, 64), (4, 19, 16320, 64), (1, 9001, 544, 32), (4, 70000, 512, 128),
                                         (1, 20, 16512, 128)])
def test_i4_sizes(gpu, dtype, M, N, K, group):
    """One row to several tiles of rows, few and many work-groups (both wave counts)."""
    run_i4(gpu, dtype, M, N, K, group, seed=M)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,group", [
    # x in registers: each number of steps, ranges of k that overlap and one that does not, one tile a work-group and several
    (16, 37, 128, 128), (8, 6000, 128, 128), (5, 4200, 160, 32), (2, 33, 1024, 64), (9, 8300, 1088, 64), (16, 50, 2080, 32), (3, 4097, 4128, 32),
    (2, 19, 4096, 128), (7, 20, 4224, 128), (12, 100, 6144, 32), (16, 40, 6208, 64), (4, 33, 8192, 128), (11, 4500, 992, 32),
    # not: two tiles a wave, batches that overlap, less than a batch
    (16, 33, 6176, 32), (16, 12300, 8320, 128), (6, 30, 64, 32), (20, 40, 480, 32), (17, 9000, 576, 64), (40, 8200, 640, 128),
    (16, 9, 16448, 64), (25, 70, 704, 64)])
def test_i4_held_rows(gpu, dtype, M, N, K, group):
    run_i4(gpu, dtype, M, N, K, group, zeros=None if N % 2 else True, bias=N % 3 != 0, seed=K)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_i4_held_rows_every_value(gpu, dtype, group):
    """One-hot rows, 16 at a time, read back exactly, where the ranges of k of the waves overlap."""
    ops = _ops()
    N, K = 20, 1152
    w, _, zero = weights(N, K, group, "4 bits", dtype, group)
    scale = 2.0 ** torch.randint(-3, 4, (N, K // group), generator=torch.Generator().manual_seed(1)).to(dtype)
    eye = torch.eye(K, dtype=dtype, device=gpu)
    args = [t.to(gpu) for t in (w, scale, zero)]
    out = torch.cat([ops.linear_i4(eye[i:i + 16], *args) for i in range(0, K, 16)]).cpu()
    q = torch.stack((w & 15, w >> 4), -1).reshape(N, K).double()
    ref = (q - zero.double().repeat_interleave(group, 1)) * scale.double().repeat_interleave(group, 1)
    assert torch.equal(out.double(), ref.t())


@pytest.mark.parametrize("dtype", DTYPES)
def test_i4_fp32_output_and_no_bias(gpu, dtype):
    run_i4(gpu, dtype, 9, 130, 1024, 64, None, bias=False, out_dtype=torch.float32, seed=3)


def test_i4_every_value(gpu):
    """One-hot rows read the weights back: every position of a group's words, exactly."""
    ops = _ops()
    for dtype in DTYPES:
        for group in (32, 64, 128):
            N, K = 20, 384
            w, _, zero = weights(N, K, group, "4 bits", dtype, group)
            scale = 2.0 ** torch.randint(-3, 4, (N, K // group), generator=torch.Generator().manual_seed(1)).to(dtype)
            out = ops.linear_i4(torch.eye(K, dtype=dtype, device=gpu), w.to(gpu), scale.to(gpu), zero.to(gpu)).cpu()
            q = torch.stack((w & 15, w >> 4), -1).reshape(N, K).double()
            ref = (q - zero.double().repeat_interleave(group, 1)) * scale.double().repeat_interleave(group, 1)
            assert torch.equal(out.double(), ref.t()), (dtype, group)


@pytest.mark.parametrize("M,K", [(5, 256), (3, 1024)])
def test_i4_strides_and_out(gpu, M, K):
    """Row-strided x and out; what lies between and behind the rows stays."""
    ops = _ops()
    N = 70
    x = _rand((M, K + 40), torch.float16, 1).to(gpu)[:, 8:8 + K]
    w, scale, zero = (t.to(gpu) for t in weights(N, K, 64, "4 bits", torch.float16, 2))
    buf = torch.full((M + 1, N + 3), 5.0, device=gpu, dtype=torch.float16)
    ops.linear_i4(x, w, scale, zero, out=buf[:M, :N])
    ref, tol = linear64(x.cpu(), w.cpu(), scale.cpu(), zero.cpu(), None, 64, torch.float16)
    check("strided", buf[:M, :N], ref, tol)
    assert bool((buf[M:] == 5.0).all()) and bool((buf[:, N:] == 5.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_i4_small_values(gpu, dtype):
    """x of fp16's subnormal range and scales near the least: nothing is flushed to zero."""
    ops = _ops()
    for M in (1, 2, 4, 9):
        x = (_rand((M, 640), torch.float32, M) * 2.0 ** -18).to(dtype)
        w, scale, zero = weights(40, 640, 64, "4 bits", dtype, 12)
        scale = (scale.float() * 2.0 ** -10).to(dtype)
        out = ops.linear_i4(x.to(gpu), w.to(gpu), scale.to(gpu), zero.to(gpu), out_dtype=torch.float32).cpu().double()
        ref, tol = linear64(x, w, scale, zero, None, 64, torch.float32)
        tol = tol - 2.0 ** -24 + 2.0 ** -149
        assert bool(((out - ref).abs() <= tol).all()), M


def test_i4_rows_stand_alone(gpu):
    """A not-finite row of x stays in its row; a row's bits do not depend on the others of its tile."""
    ops = _ops()
    w, scale, zero = (t.to(gpu) for t in weights(64, 512, 128, "4 bits", torch.bfloat16, 4))
    x = _rand((16, 512), torch.bfloat16, 5).to(gpu)
    for M in (2, 4):  # the kernel of few rows
        x2 = x[:M].clone()
        x2[1, 7] = math.nan
        got, clean = ops.linear_i4(x2, w, scale, zero), ops.linear_i4(x[:M].contiguous(), w, scale, zero)
        keep = [i for i in range(M) if i != 1]
        assert torch.equal(got[keep], clean[keep]) and bool(torch.isnan(got[1]).all())
    clean = ops.linear_i4(x, w, scale, zero)
    x2 = x.clone()
    x2[3, 7], x2[9, 100] = math.nan, math.inf
    got = ops.linear_i4(x2, w, scale, zero)
    keep = [i for i in range(16) if i not in (3, 9)]
    assert torch.equal(got[keep], clean[keep])
    assert bool(torch.isnan(got[3]).all()) and not bool(torch.isfinite(got[9]).any())
    assert torch.equal(ops.linear_i4(x[4:10], w, scale, zero), clean[4:10])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("symmetric", [False, True])
def test_quant_groups_i4_round_trip(gpu, dtype, symmetric):
    """Quantised weights are within half a step (and the scale's rounding) of the weights."""
    ops = _ops()
    w = _rand((40, 256), dtype, 6).to(gpu)
    w[3, :64] = 0
    w[4, 64:128] = 2.5
    q, scale, zero = ops.quant_groups_i4(w, 64, symmetric)
    values = torch.stack((q & 15, q >> 4), -1).reshape(40, 256).double()
    z = zero.double().repeat_interleave(64, 1) if zero is not None else 8.0
    s = scale.double().repeat_interleave(64, 1)
    err = ((values - z) * s - w.double()).abs()
    # half a step for the value, half for a zero point between two values, and 15 (or 7) roundings of the scale
    assert bool((err <= s * (0.5 + (0 if symmetric else 0.5) + 16 * UNIT[dtype])).all())
    assert bool((((values - z) * s)[3, :64] == 0).all())


def test_i4_graph_replay(gpu):
    ops = _ops()
    w, scale, zero = (t.to(gpu) for t in weights(300, 1024, 128, "4 bits", torch.float16, 8))
    x = _rand((2, 1024), torch.float16, 9).to(gpu)
    ops.linear_i4(x, w, scale, zero)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_i4(x, w, scale, zero)
    for i in range(3):
        x.copy_(_rand(x.shape, x.dtype, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.linear_i4(x, w, scale, zero))


# ------------------------------------------------------------------------------ refusals, far offsets
def test_refusals_on_the_gpu(gpu):
    """What the kernels are not made for raises before anything is launched."""
    ops = _ops()
    q, k = torch.zeros(8, 4, 64, device=gpu).half(), torch.zeros(8, 2, 64, device=gpu).half()
    plan = ops.packed_plan([5, 3], heads=4, kv_heads=2, head_dim=64, device=gpu)
    cache, lens = torch.zeros(8, 10, 2, 64, device=gpu).half(), torch.zeros(8, dtype=torch.int32, device=gpu)
    q4 = q.unsqueeze(1)
    x, w = torch.zeros(3, 128, device=gpu).half(), torch.zeros(10, 64, dtype=torch.uint8, device=gpu)
    s, z, b = torch.ones(10, 2, device=gpu).half(), torch.zeros(10, 2, dtype=torch.uint8, device=gpu), torch.zeros(10, device=gpu)
    packed, prefix, i4 = ops.attention_packed, ops.attention_shared_prefix, ops.linear_i4
    odd = torch.zeros(8 * 2 * 64 + 1, device=gpu).half()[1:].view(8, 2, 64)
    grad = q.clone().requires_grad_()
    own = [k, k, cache, cache, lens]
    for error, call in [
        (TypeError, lambda: packed(q.float(), k.float(), k.float(), plan)), (TypeError, lambda: packed(q, k.bfloat16(), k, plan)),
        (ValueError, lambda: packed(q[:7], k, k, plan)), (ValueError, lambda: packed(q, k[:, :1], k, plan)),
        (ValueError, lambda: packed(q, k, k[:7], plan)), (ValueError, lambda: packed(q[..., :32], k, k, plan)),
        (ValueError, lambda: packed(q, odd, k, plan)), (ValueError, lambda: packed(q, k[:1].expand(8, 2, 64), k, plan)),
        (ValueError, lambda: packed(q, k, k, plan, scale=0.0)), (ValueError, lambda: packed(q, k, k, plan, scale=math.inf)),
        (ValueError, lambda: packed(q, k, k, plan, scale=math.nan)), (ValueError, lambda: packed(q, k, k, plan, out=q)),
        (ValueError, lambda: packed(q, k, k, plan, out=q.new_zeros(8, 4, 32))), (TypeError, lambda: packed(q, k, k, plan, out=q.float())),
        (ValueError, lambda: packed(q, k, k, plan, out=q.new_zeros(1, 4, 64).expand(8, 4, 64))),
        (ValueError, lambda: packed(q, k, k, plan, out=torch.empty_like(q).requires_grad_())),
        (ValueError, lambda: prefix(q4, *own, out=torch.empty_like(q4).requires_grad_())),
        (ValueError, lambda: i4(x, w, s, z, b, out=x.new_empty(3, 10).requires_grad_())),
        (ValueError, lambda: packed(grad, k, k, plan)), (ValueError, lambda: packed(q.cpu(), k, k, plan)),
        (ValueError, lambda: packed(q, k.cpu(), k, plan)),
        (TypeError, lambda: prefix(q4.float(), *own)), (TypeError, lambda: prefix(q4, k.bfloat16(), *own[1:])),
        (ValueError, lambda: prefix(q, *own)), (ValueError, lambda: prefix(q4[:7], *own)), (ValueError, lambda: prefix(q4[:, :, :3], *own)),
        (ValueError, lambda: prefix(q4, k[:7], *own[1:])), (ValueError, lambda: prefix(q4, k, k, cache[:, :9], cache, lens)),
        (ValueError, lambda: prefix(q4, *own[:4], lens.long())), (ValueError, lambda: prefix(q4, *own[:4], lens[:7])),
        (ValueError, lambda: prefix(q4, *own[:4], torch.zeros(16, dtype=torch.int32, device=gpu)[::2])),
        (ValueError, lambda: prefix(q4, *own, out=q4)), (ValueError, lambda: prefix(q4, *own[:4], lens.cpu())),
        (ValueError, lambda: prefix(grad.unsqueeze(1), *own)), (ValueError, lambda: prefix(q4, *own, scale=-1.0)),
        (ValueError, lambda: prefix(q4[..., :40], k[..., :40], k[..., :40], cache[..., :40], cache[..., :40], lens)),
        (TypeError, lambda: i4(x.float(), w, s, z, b)), (TypeError, lambda: i4(x, w, s.bfloat16(), z, b)),
        (TypeError, lambda: i4(x, w, s, z, b, out_dtype=torch.bfloat16)), (ValueError, lambda: i4(x, w[:9], s, z, b)),
        (ValueError, lambda: i4(x[:, :96], w, s, z, b)), (ValueError, lambda: i4(x, w, s[:, :1], z, b)),
        (ValueError, lambda: i4(x, w.char(), s, z, b)), (ValueError, lambda: i4(x, w, s, z.int(), b)), (ValueError, lambda: i4(x, w, s, z, b.half())),
        (ValueError, lambda: i4(x, w, torch.ones(2, 10, device=gpu).half().t(), z, b)), (ValueError, lambda: i4(x.t().contiguous().t(), w, s, z, b)),
        (ValueError, lambda: i4(torch.zeros(3, 129, device=gpu).half()[:, 1:], w, s, z, b)), (ValueError, lambda: i4(x[0], w, s, z, b)),
        (ValueError, lambda: i4(x, w, s, z, b, out=x[:, :10])), (ValueError, lambda: i4(x, w, s, z, b, out=x.new_zeros(10, 3).t())),
        (ValueError, lambda: i4(x.clone().requires_grad_(), w, s, z, b)), (ValueError, lambda: i4(x, w.cpu(), s, z, b)),
    ]:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        packed(grad, k, k, plan)
    i4(x, w, s, z, b)


def test_offsets_past_32_bits(gpu):
    """A sequence of a cache, tokens of a prefix and features of a weight that start past 2^32 elements or bytes."""
    ops = _ops()
    H, Hkv, D, P, room = 4, 2, 64, 290, 50
    far, apart = 1 << 32, 1 << 24
    big = torch.empty(far + room * Hkv * D, device=gpu, dtype=torch.float16)
    ko = big.as_strided((2, room, Hkv, D), (far, Hkv * D, D, 1))
    wide = torch.empty(P * apart, device=gpu, dtype=torch.float16)
    kp = wide.as_strided((P, Hkv, D), (apart, D, 1))
    vo, vp = _rand((2, room, Hkv, D), torch.float16, 2).to(gpu), _rand((P, Hkv, D), torch.float16, 3).to(gpu)
    ko.copy_(_rand((2, room, Hkv, D), torch.float16, 4))
    kp.copy_(_rand((P, Hkv, D), torch.float16, 5))
    q = _rand((2, 1, H, D), torch.float16, 6).to(gpu)
    lens = [50, 33]
    ref, tol = prefix64(q.cpu(), kp.cpu(), vp.cpu(), ko.cpu(), vo.cpu(), lens, D ** -0.5)
    lt = torch.tensor(lens, dtype=torch.int32, device=gpu)
    check("far caches and tokens", ops.attention_shared_prefix(q, kp, vp, ko, vo, lt), ref, tol)
    plan = ops.packed_plan([2], [P], heads=H, kv_heads=Hkv, head_dim=D, device=gpu)
    qq = q[:, 0].contiguous()
    ref, tol = packed64(qq.cpu(), kp.cpu(), vp.cpu(), [2], [P], True, D ** -0.5)
    check("far tokens", ops.attention_packed(qq, kp, vp, plan), ref, tol)
    del big, wide, ko, kp
    N, K = (1 << 17) + 40, 65536  # 4 GiB of weights and more
    w = torch.empty(N, K // 2, dtype=torch.uint8, device=gpu)
    tail, scale, zero = weights(40, K, 128, "4 bits", torch.float16, 7)
    w[-40:] = tail.to(gpu)
    s = torch.ones(N, K // 128, device=gpu, dtype=torch.float16)
    z = torch.zeros(N, K // 128, device=gpu, dtype=torch.uint8)
    s[-40:], z[-40:] = scale.to(gpu), zero.to(gpu)
    x = _rand((2, K), torch.float16, 8, 0.05)
    ref, tol = linear64(x, tail, scale, zero, None, 128, torch.float16)
    check("far features", ops.linear_i4(x.to(gpu), w, s, z)[:, -40:], ref, tol)
    K = 16384  # ... and of the kernel of few rows
    w = w.view(-1)[:((1 << 19) + 40) * (K // 2)].view(-1, K // 2)
    tail, scale, zero = weights(40, K, 128, "4 bits", torch.float16, 9)
    w[-40:] = tail.to(gpu)
    s, z = (t.view(-1)[:w.shape[0] * 128].view(-1, 128) for t in (s, z))
    s[-40:], z[-40:] = scale.to(gpu), zero.to(gpu)
    ref, tol = linear64(x[:, :K].contiguous(), tail, scale, zero, None, 128, torch.float16)
    check("far features", ops.linear_i4(x[:, :K].contiguous().to(gpu), w, s, z)[:, -40:], ref, tol)


# ------------------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", DTYPES)
def test_generation_steps(gpu, dtype):
    """A shared instruction and each user's question as packed prompts, then tokens one at a time: the
    projections on 4-bit weights, the new K and V put into the caches, attention behind the shared
    instruction. The last step's context equals a packed call over each sequence's whole history, and
    a captured step the eager one."""
    ops = _ops()
    H, Hkv, D, B, P, room = 8, 2, 64, 3, 150, 64
    d = H * D
    width = (H + 2 * Hkv) * D
    wq = ops.quant_groups_i4(_rand((width, d), dtype, 1, d ** -0.5).to(gpu), 128)
    wo = ops.quant_groups_i4(_rand((d, d), dtype, 2, d ** -0.5).to(gpu), 64, symmetric=True)

    def project(x):
        y = ops.linear_i4(x, *wq)
        return (y[:, :H * D].view(-1, H, D), y[:, H * D:(H + Hkv) * D].view(-1, Hkv, D),
                y[:, (H + Hkv) * D:].view(-1, Hkv, D))

    qp, kp, vp = project(_rand((P, d), dtype, 3).to(gpu))
    asks = [30, 1, 47]
    q, k, v = project(_rand((sum(asks), d), dtype, 4).to(gpu))
    plan = ops.packed_plan(asks, [P + n for n in asks], heads=H, kv_heads=Hkv, head_dim=D, device=gpu)
    ko = torch.full((B, room, Hkv, D), math.nan, device=gpu, dtype=dtype)
    vo = ko.clone()
    keys, values = [], []
    at = 0
    for b, n in enumerate(asks):
        ko[b, :n], vo[b, :n] = k[at:at + n], v[at:at + n]
        keys += [kp, k[at:at + n]]
        values += [vp, v[at:at + n]]
        at += n
    prompt = ops.attention_packed(q, torch.cat(keys), torch.cat(values), plan)
    last = prompt[torch.tensor(asks, device=gpu).cumsum(0) - 1]  # each question's last token
    lens = torch.tensor(asks, dtype=torch.int32, device=gpu)
    rows = torch.arange(B, device=gpu)
    x = torch.empty(B, d, device=gpu, dtype=dtype)
    x.copy_(ops.linear_i4(last.reshape(B, d), *wo))

    def step():
        q, k, v = project(x)
        ko[rows, lens.long()], vo[rows, lens.long()] = k, v
        lens.add_(1)
        ctx = ops.attention_shared_prefix(q.unsqueeze(1), kp, vp, ko, vo, lens)
        x.copy_(ops.linear_i4(ctx.view(B, d), *wo))
        return q, ctx

    for _ in range(2):
        q, ctx = step()
    saved = [t.clone() for t in (x, ko, vo, lens)]
    q, ctx = step()
    whole = ops.packed_plan([1] * B, [P + int(n) for n in lens.tolist()], heads=H, kv_heads=Hkv, head_dim=D, device=gpu)
    ks = torch.cat([t for b, n in enumerate(lens.tolist()) for t in (kp, ko[b, :n])])
    vs = torch.cat([t for b, n in enumerate(lens.tolist()) for t in (vp, vo[b, :n])])
    ref, tol = packed64(q.cpu(), ks.cpu(), vs.cpu(), [1] * B, [P + int(n) for n in lens.tolist()], True, D ** -0.5)
    check("step", ctx.view(B, H, D), ref, tol)
    check("packed history", ops.attention_packed(q, ks, vs, whole), ref, tol)

    eager = [x.clone()]
    for _ in range(2):
        step()
        eager.append(x.clone())
    for t, s in zip((x, ko, vo, lens), saved):
        t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, s in zip((x, ko, vo, lens), saved):
        t.copy_(s)
    for want in eager:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want)
