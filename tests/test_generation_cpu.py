"""Refusals and host-side work of the token-generation operators, without a GPU: the C entry points
reject bad arguments before they launch anything, the packed plan covers every row once, and the
Python wrappers name what is wrong."""
import ctypes as C

import pytest
import torch

from tiktok_techjam_2026_track3_amd import _lib, ops

F32, F16, BF16 = 0, 1, 2
BAD_SIZE, NULL, DTYPE, ALIGN, HEAD, UNSUP = -2, -1, -3, -4, -5, -6


def plan(q_lens, k_lens, heads=4, kv_heads=2, head_dim=64, causal=1):
    n = len(q_lens)
    arr = C.c_int32 * max(1, n)
    counts, rows = _lib.i64_array((0, 0, 0, 0)), C.c_int32(0)
    args = (arr(*q_lens), arr(*k_lens), n, heads, kv_heads, head_dim, causal)
    st = _lib.lib().mi355_attn_packed_plan(*args, 0, 0, counts, C.byref(rows))
    if st:
        return st, None, counts, 0
    entries = torch.empty(sum(counts[:3]), 8, dtype=torch.int32)
    if entries.numel():
        assert _lib.lib().mi355_attn_packed_plan(*args, entries.data_ptr(), len(entries) - 1, counts,
                                                 C.byref(rows)) == BAD_SIZE  # too small a buffer
        st = _lib.lib().mi355_attn_packed_plan(*args, entries.data_ptr(), len(entries), counts, C.byref(rows))
    return st, entries.tolist(), list(counts), rows.value


@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads", [
    ([5], [5], 4, 2), ([0, 3, 0, 900, 1], [4, 3, 0, 900, 77], 12, 4), ([4096] * 3, [5000, 4096, 100], 32, 8), ([], [], 1, 1),
    ([1] * 200, list(range(200)), 8, 8), ([1, 1], [70000, 3], 8, 1), ([40, 8, 1], [9000, 20000, 1000], 8, 2),
    ([33, 32], [5000, 5000], 1, 1), ([500], [10], 4, 4), ([100, 1], [100, 512], 4, 2), ([100, 1], [100, 513], 4, 2)])
@pytest.mark.parametrize("causal", [0, 1])
def test_plan_covers_every_row_and_key_once(q_lens, k_lens, heads, kv_heads, causal):
    """Each row's visible keys are covered by ranges without gap or overlap, a tile in one range writes its
    rows itself, the ranges of a split one have partial rows of their own that a join names; lists are
    longest first."""
    st, entries, (wide, narrow, joins, slots), rows = plan(q_lens, k_lens, heads, kv_heads, causal=causal)
    assert st == 0 and len(entries) == wide + narrow + joins
    g = heads // kv_heads
    few = [m for n, m in zip(q_lens, k_lens) if 0 < n * g <= 32]
    limit = 0 if wide and len(few) * kv_heads <= 256 and max(few, default=0) <= 512 else 32  # rows of narrow tiles
    tiles = {}
    for i, (q0, q_len, k0, k_len, row0, k_begin, k_stop, slot) in enumerate(entries[:wide + narrow]):
        tiles.setdefault((q0, q_len, k0, k_len, row0), []).append((k_begin, k_stop, slot))
        assert (q_len * g > limit) == (i < wide)
    for part in (entries[:wide], entries[wide:wide + narrow]):
        keys = [t[6] - t[5] for t in part]
        assert keys == sorted(keys, reverse=True)
    joined = {(j[0], j[3]): j for j in entries[wide + narrow:]}
    assert len(joined) == joins
    want, used, q0, k0 = set(), [], 0, 0
    for n, m in zip(q_lens, k_lens):
        step = rows if n * g > limit else 32
        for r in range(0, n * g, step):
            want.add((q0, n, k0, m, r))
            real = min(step, n * g - r)
            last = (r + real - 1) // g
            keys = max(0, min(m, last + m - n + 1)) if causal else m
            ranges = sorted(tiles[(q0, n, k0, m, r)])
            assert ranges[0][0] == 0 and ranges[-1][1] == keys
            assert all(a[1] == b[0] for a, b in zip(ranges, ranges[1:]))
            if len(ranges) == 1:
                assert ranges[0][2] == -1 and (q0, r) not in joined
            else:
                assert all(a[0] < a[1] for a in ranges)
                j = joined[(q0, r)]
                assert j == [q0, n, m, r, real, ranges[0][2], len(ranges), 0]
                assert [a[2] for a in ranges] == [j[5] + real * i for i in range(len(ranges))]
                used += [x for a in ranges for x in range(a[2], a[2] + real)]
        q0, k0 = q0 + n, k0 + m
    assert set(tiles) == want
    assert sorted(used) == list(range(slots))


@pytest.mark.parametrize("kw,status", [
    (dict(heads=3), BAD_SIZE), (dict(heads=0), BAD_SIZE), (dict(kv_heads=0), BAD_SIZE), (dict(head_dim=8), HEAD),
    (dict(head_dim=0), HEAD), (dict(q_lens=[-1]), BAD_SIZE), (dict(k_lens=[-1]), BAD_SIZE),
    (dict(q_lens=[1 << 29], heads=8, kv_heads=1), BAD_SIZE), (dict(q_lens=[1 << 25], k_lens=[1], heads=4096, kv_heads=4096), BAD_SIZE), (dict(q_lens=[1 << 29, 1 << 29], k_lens=[1, 1]), BAD_SIZE)])
def test_plan_refusals(kw, status):
    kw = {"q_lens": [4], "k_lens": [4], **kw}
    assert plan(**kw)[0] == status


def test_plan_null_pointers():
    counts, rows = _lib.i64_array((0, 0, 0, 0)), C.c_int32(0)
    f = _lib.lib().mi355_attn_packed_plan
    assert f(None, None, 1, 4, 2, 64, 1, 0, 0, counts, C.byref(rows)) == NULL
    assert f(None, None, 0, 4, 2, 64, 1, 0, 0, None, C.byref(rows)) == NULL


PACKED = dict(dtype=F16, Q=64, K=64, V=64, O=64, heads=4, kv_heads=2, head_dim=64, qs=(256, 64), ks=(128, 64),
              vs=(128, 64), os=(256, 64), scale=0.125, causal=1, tiles=64, counts=(3, 2, 1, 100), tile_rows=64,
              ws=64, ws_bytes=100 * 2 * 66 * 4)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=F32), DTYPE), (dict(dtype=9), DTYPE), (dict(heads=3), BAD_SIZE), (dict(kv_heads=0), BAD_SIZE),
    (dict(counts=(-1, 0, 0, 0)), BAD_SIZE), (dict(counts=(1 << 30, 0, 0, 0)), BAD_SIZE), (dict(counts=None), NULL),
    (dict(ws=0), NULL), (dict(ws=72), ALIGN), (dict(ws_bytes=100 * 2 * 66 * 4 - 1), BAD_SIZE), (dict(head_dim=40), HEAD), (dict(tile_rows=48), UNSUP),
    (dict(scale=0.0), UNSUP), (dict(scale=-1.0), UNSUP), (dict(scale=float("inf")), UNSUP), (dict(scale=float("nan")), UNSUP),
    (dict(Q=0), NULL), (dict(O=0), NULL), (dict(tiles=0), NULL), (dict(Q=72), ALIGN), (dict(K=68), ALIGN), (dict(V=8), ALIGN),
    (dict(O=68), ALIGN), (dict(qs=(257, 64)), ALIGN), (dict(ks=(132, 64)), ALIGN), (dict(vs=(128, 4)), ALIGN),
    (dict(os=(256, 62)), ALIGN), (dict(ks=(56, 64)), BAD_SIZE), (dict(vs=(0, 64)), BAD_SIZE), (dict(ks=(1 << 25, 64)), BAD_SIZE)])
def test_packed_entry_refusals(kw, status):
    a = {**PACKED, **kw}
    i64 = _lib.i64_array
    assert _lib.lib().mi355_attn_packed(
        a["dtype"], a["Q"], a["K"], a["V"], a["O"], a["heads"], a["kv_heads"], a["head_dim"], i64(a["qs"]), i64(a["ks"]),
        i64(a["vs"]), i64(a["os"]), a["scale"], a["causal"], a["tiles"], i64(a["counts"]) if a["counts"] else None,
        a["tile_rows"], a["ws"], a["ws_bytes"], None) == status


PREFIX = dict(dtype=F16, ptrs=[64] * 7, B=2, n=1, heads=4, kv_heads=2, head_dim=64, P=1000, room=50, qs=(256, 256, 64),
              kps=(128, 64), vps=(128, 64), kos=(6400, 128, 64), vos=(6400, 128, 64), os=(256, 256, 64), scale=0.125, ws=64,
              ws_bytes=1 << 30)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=F32), DTYPE), (dict(heads=5), BAD_SIZE), (dict(B=-1), BAD_SIZE), (dict(B=60000, n=100), BAD_SIZE), (dict(n=-1), BAD_SIZE), (dict(P=-1), BAD_SIZE),
    (dict(room=1 << 30), BAD_SIZE), (dict(head_dim=24), HEAD), (dict(scale=0.0), UNSUP), (dict(scale=float("nan")), UNSUP),
    (dict(ws=0), NULL), (dict(ws_bytes=16), BAD_SIZE), (dict(ws=72), ALIGN), (dict(kps=(56, 64)), BAD_SIZE),
    (dict(vos=(6400, 64, 64), kv_heads=2, head_dim=128), BAD_SIZE), (dict(qs=(256, 256, 63)), ALIGN),
    (dict(kos=(6401, 128, 64)), ALIGN), (dict(os=(256, 256, 2)), ALIGN),
    *[(dict(ptrs=[0 if j == i else 64 for j in range(7)]), NULL) for i in range(7)],
    *[(dict(ptrs=[72 if j == i else 64 for j in range(7)]), ALIGN) for i in range(5)]])
def test_prefix_entry_refusals(kw, status):
    a = {**PREFIX, **kw}
    i64 = _lib.i64_array
    q, kp, vp, ko, vo, lens, out = a["ptrs"]
    assert _lib.lib().mi355_attn_shared_prefix(
        a["dtype"], q, kp, vp, ko, vo, lens, out, a["B"], a["n"], a["heads"], a["kv_heads"], a["head_dim"], a["P"], a["room"],
        i64(a["qs"]), i64(a["kps"]), i64(a["vps"]), i64(a["kos"]), i64(a["vos"]), i64(a["os"]), a["scale"], a["ws"],
        a["ws_bytes"], None) == status


def test_prefix_workspace_size():
    f = _lib.lib().mi355_attn_shared_prefix_workspace_bytes
    assert f(2, 1, 4, 2, 64, 0, 0) == 0
    assert f(2, 1, 4, 2, 64, 974, 50) == 0  # a work-group goes through all keys of its rows
    assert f(2, 1, 4, 2, 64, 975, 50) == (4 + 1) * 2 * 4 * (64 + 2) * 4  # ranges of 256 keys
    assert f(2, 17, 4, 2, 64, 100, 50) == 2 * 2 * 17 * 4 * (64 + 2) * 4  # more than 32 rows
    assert f(2, 1, 4, 3, 64, 100, 50) == BAD_SIZE and f(2, 1, 4, 2, 65, 100, 50) == HEAD
    assert f(64, 1, 32, 8, 128, 1 << 20, 4096) > 0


I4 = dict(dtype=F16, odt=F16, X=64, ldx=256, W=64, s=64, Y=64, ldy=100, M=3, N=100, K=256, group=64)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=F32), DTYPE), (dict(odt=BF16), DTYPE), (dict(odt=7), DTYPE), (dict(group=16), UNSUP), (dict(group=0), UNSUP),
    (dict(K=224), BAD_SIZE), (dict(M=-1), BAD_SIZE), (dict(N=(1 << 26) + 1), BAD_SIZE), (dict(K=1 << 27, group=128), BAD_SIZE), (dict(N=-1), BAD_SIZE), (dict(ldx=248), BAD_SIZE), (dict(ldy=99), BAD_SIZE),
    (dict(ldx=260), ALIGN), (dict(X=72), ALIGN), (dict(W=68), ALIGN), (dict(X=0), NULL), (dict(W=0), NULL), (dict(s=0), NULL),
    (dict(Y=0), NULL)])
def test_i4_entry_refusals(kw, status):
    a = {**I4, **kw}
    assert _lib.lib().mi355_linear_i4(a["dtype"], a["odt"], a["X"], a["ldx"], a["W"], a["s"], 0, 0, a["Y"], a["ldy"], a["M"],
                                      a["N"], a["K"], a["group"], None) == status


def test_wrappers_refuse_cpu_tensors():
    q, k = torch.zeros(4, 4, 64, dtype=torch.float16), torch.zeros(4, 2, 64, dtype=torch.float16)
    p = ops.PackedPlan(4, 4, 4, 2, 64, True, 64, _lib.i64_array((0, 0, 0, 0)), torch.zeros(0, 8, dtype=torch.int32), 0)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention_packed(q, k, k, p)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention_shared_prefix(q[None], k, k, k[None], k[None], torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_i4(torch.zeros(1, 64).half(), torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1).half())


@pytest.mark.parametrize("kw", [
    dict(q_lens=[1], k_lens=[1, 2]), dict(q_lens=[-1]), dict(q_lens=[1 << 30]), dict(q_lens=[4], kv_heads=3),
    dict(q_lens=[4], heads=0), dict(q_lens=[4], head_dim=8), dict(q_lens=[4], device="cpu")])
def test_packed_plan_wrapper_refusals(kw):
    kw = {"heads": 4, "kv_heads": 2, "head_dim": 64, **kw}
    with pytest.raises(ValueError):
        ops.packed_plan(kw.pop("q_lens"), kw.pop("k_lens", None), **kw)


@pytest.mark.parametrize("w,group", [(torch.zeros(4, 64), 64), (torch.zeros(4, 64).half(), 48), (torch.zeros(4, 96).half(), 64),
                                     (torch.zeros(64).half(), 64)])
def test_quant_groups_i4_refusals(w, group):
    with pytest.raises(ValueError):
        ops.quant_groups_i4(w, group)


def test_quant_groups_i4_values():
    """Two-level groups come back exactly; the even k is in the low half of a byte."""
    w = torch.zeros(2, 64, dtype=torch.float16)
    w[0, ::2], w[0, 1::2], w[1] = 0.0, 15.0, -7.0
    q, s, z = ops.quant_groups_i4(w, 32)
    assert q.shape == (2, 32) and s.shape == z.shape == (2, 2)
    assert bool((q[0] == 0xF0).all()) and bool((s[0] == 1).all()) and bool((z[0] == 0).all())
    values = torch.stack((q & 15, q >> 4), -1).reshape(2, 64).float()
    assert bool((((values - z.repeat_interleave(32, 1)) * s.float().repeat_interleave(32, 1))[1] + 7).abs().max() < 0.01)
    q, s, z = ops.quant_groups_i4(w, 32, symmetric=True)
    assert z is None and bool((q[1] == 0x11).all()) and bool((s[1] == 1).all())


@pytest.mark.parametrize("shape,stride,kw", [
    ((4, 2, 64), (128, 64, 2), {}), ((4, 2, 64), (130, 64, 1), {}), ((4, 2, 64), (128, 68, 1), {}),
    ((4, 2, 64), (56, 64, 1), dict(kv_axis=0)), ((4, 2, 64), (0, 64, 1), dict(kv_axis=0)), ((4, 2, 64), (1 << 25, 64, 1), dict(kv_axis=0)),
    ((4, 2, 64), (0, 64, 1), dict(written=True)), ((4, 2, 64), (128, 0, 1), dict(written=True)), ((4, 2, 64), (64, 128, 1), dict(written=True)),
    ((4, 2, 64), (128, 32, 1), dict(written=True))])
def test_view_refusals(shape, stride, kw):
    with pytest.raises(ValueError):
        ops._rows_strides("t", shape, stride, 8, **kw)


@pytest.mark.parametrize("shape,stride,kw,want", [
    ((4, 2, 64), (128, 64, 1), {}, (128, 64)), ((4, 2, 64), (64, 256, 1), dict(written=True), (64, 256)),
    ((1, 2, 64), (3, 64, 1), dict(kv_axis=0), (64, 64)), ((4, 1, 64), (64, 5, 1), {}, (64, 0)),
    ((4, 2, 64), (64, 0, 1), dict(kv_axis=0), (64, 0)), ((0, 2, 64), (128, 64, 1), dict(kv_axis=0), (64, 0))])
def test_view_strides(shape, stride, kw, want):
    """Axes of one element have any stride; heads may share one K / V head; orders other than the usual."""
    assert ops._rows_strides("t", shape, stride, 8, **kw) == want


def _dma_asm(*between):
    return "\n".join(["attn_rows_x:", "  v_readfirstlane_b32 s6, v1", *between, "  s_mov_b32 m0, s20", "  s_nop 0",
                      "  buffer_load_dwordx4 v2, s[4:7], s9 offen lds", "  s_endpgm", ".Lfunc_end0:"])


@pytest.mark.parametrize("between,bad", [
    ([], True), (["  s_add_i32 s8, s8, 1"] * 2, True), (["  s_add_i32 s8, s8, 1"] * 3, False), (["  s_nop 2"], False),
    (["  s_mov_b32 s6, s30"], False),                       # written again by the scalar ALU
    (["  s_cmp_eq_u32 s6, s30"], True),                     # only read
    (["  s_branch .L1", ".L0:", "  s_nop 7", ".L1:"], True)])  # over a branch
def test_build_finds_scalars_read_too_soon(between, bad):
    """The build's check of LDS-DMA loads whose resource the vector ALU has just written."""
    from tiktok_techjam_2026_track3_amd import _lib  # noqa: F401  (the package's build attribute is a function)
    import importlib
    B = importlib.import_module("tiktok_techjam_2026_track3_amd.build")
    assert bool(B.dma_hazards(_dma_asm(*between))) == bad
    if bad:
        with pytest.raises(RuntimeError):
            B.check_dma_hazards("x.hip", _dma_asm(*between))


def test_packed_plan_takes_whole_lengths():
    with pytest.raises(TypeError):
        ops.packed_plan([2.5], heads=4, head_dim=64)
