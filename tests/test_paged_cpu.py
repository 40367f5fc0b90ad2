"""Refusals of the rotary and paged-cache operators without a GPU: the C entry points reject bad arguments before they
launch anything, the Python wrappers name what is wrong; and the plain reference that the GPU tests use."""
import math

import pytest
import torch

from paged_reference import block_scale, empty_cache, frequencies, rotate64, values64
from tiktok_techjam_2026_track3_amd import _lib, ops

F32, F16, BF16 = 0, 1, 2
BAD_SIZE, NULL, DTYPE, ALIGN, HEAD, UNSUP = -2, -1, -3, -4, -5, -6
i64 = _lib.i64_array


ROTARY = dict(dtype=F16, X=64, Y=64, pos=64, freqs=64, n0=1, n1=4, heads=2, head_dim=64, rot=64, sizes=True,
              strides=(0, 1, 0, 128, 64, 0, 128, 64))


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), DTYPE), (dict(n0=-1), BAD_SIZE), (dict(n1=1 << 32), BAD_SIZE), (dict(n0=1 << 16, n1=1 << 16), BAD_SIZE),
    (dict(heads=70000), BAD_SIZE), (dict(heads=-1), BAD_SIZE), (dict(head_dim=63), HEAD), (dict(head_dim=514), HEAD),
    (dict(rot=66), HEAD), (dict(rot=0), HEAD), (dict(rot=3), HEAD), (dict(X=0), NULL), (dict(Y=0), NULL), (dict(pos=0), NULL),
    (dict(freqs=0), NULL), (dict(sizes=False), NULL), (dict(strides=None), NULL), (dict(n1=0), 0), (dict(heads=0), 0)])
def test_rotary_entry_refusals(kw, status):
    a = {**ROTARY, **kw}
    sizes = i64([a[k] for k in ("n0", "n1", "heads", "head_dim", "rot")])
    assert _lib.lib().mi355_rotary(a["dtype"], a["X"], a["Y"], a["pos"], 1, a["freqs"], 1.0, sizes if a["sizes"] else None,
                                   i64(a["strides"]) if a["strides"] else None, 0, 0, None) == status


APPEND = dict(dtype=F16, K=64, V=64, Q=64, QO=64, ck=64, cv=64, ks=64, vs=64, table=64, row=4, lens=64, off=64, B=2, most=3,
              tokens=6, heads=4, kv_heads=2, head_dim=64, pages=9, page=16, width=4, strides=(128, 64, 128, 64, 256, 64, 256, 64),
              freqs=64, rot=64)


def sizes_of(a):
    return i64([a[k] for k in ("B", "most", "tokens", "heads", "kv_heads", "head_dim", "pages", "page", "width", "row")])


def strides_but(at, value):
    return tuple(value if i == at else s for i, s in enumerate(APPEND["strides"]))


SIZES = [
    (dict(dtype=F32), DTYPE), (dict(head_dim=40), HEAD), (dict(B=-1), BAD_SIZE), (dict(B=(1 << 20) + 1), BAD_SIZE),
    (dict(most=-1), BAD_SIZE), (dict(tokens=1 << 30), BAD_SIZE), (dict(heads=5), BAD_SIZE), (dict(kv_heads=0), BAD_SIZE),
    (dict(pages=1 << 30), BAD_SIZE), (dict(page=8), BAD_SIZE), (dict(page=48), BAD_SIZE), (dict(page=2048), BAD_SIZE),
    (dict(width=1 << 26), BAD_SIZE), (dict(width=-1), BAD_SIZE), (dict(off=0, tokens=5), BAD_SIZE),
    (dict(row=-1), BAD_SIZE), (dict(row=1 << 30), BAD_SIZE), (dict(strides=None), NULL)]


@pytest.mark.parametrize("kw,status", SIZES + [
    *[({k: 0}, NULL) for k in ("K", "V", "QO", "ck", "cv", "ks", "vs", "table", "lens", "freqs")],
    (dict(rot=4), HEAD), (dict(rot=72), HEAD), (dict(rot=20), HEAD), (dict(K=72), ALIGN), (dict(V=68), ALIGN), (dict(Q=72), ALIGN),
    (dict(QO=72), ALIGN), (dict(ck=72), ALIGN), (dict(cv=72), ALIGN), *[(dict(strides=strides_but(i, 132)), ALIGN) for i in range(8)], (dict(most=1 << 29, B=1 << 10), BAD_SIZE), (dict(B=0), 0),
    (dict(tokens=0), 0), (dict(most=0), 0)])
def test_append_entry_refusals(kw, status):
    a = {**APPEND, **kw}
    assert _lib.lib().mi355_paged_append(
        a["dtype"], a["K"], a["V"], a["Q"], a["QO"], a["ck"], a["cv"], a["ks"], a["vs"], a["table"], a["lens"], a["off"],
        sizes_of(a), i64(a["strides"]) if a["strides"] else None, a["freqs"], a["rot"], 0, 1.0, 1, None) == status


@pytest.mark.parametrize("kw,status", SIZES + [
    *[({k: 0}, NULL) for k in ("Q", "QO", "ck", "cv", "ks", "vs", "table", "lens")],
    (dict(pages=0), BAD_SIZE), (dict(scale=0.0), UNSUP), (dict(scale=-1.0), UNSUP), (dict(scale=math.nan), UNSUP),
    (dict(scale=math.inf), UNSUP), (dict(Q=72), ALIGN), (dict(QO=68), ALIGN), (dict(ck=72), ALIGN), (dict(cv=8), ALIGN),
    *[(dict(strides=strides_but(i, 130)), ALIGN) for i in range(4)], (dict(width=129, ws=0), BAD_SIZE), (dict(width=129, ws_bytes=64), BAD_SIZE),
    (dict(width=129, ws=72), BAD_SIZE), (dict(B=1 << 11, most=1 << 10, tokens=1 << 21), BAD_SIZE), (dict(B=0), 0), (dict(tokens=0), 0)])
def test_attention_entry_refusals(kw, status):
    a = {**APPEND, "scale": 0.125, "ws": 64, "ws_bytes": 1 << 30, **kw}
    assert _lib.lib().mi355_attn_paged(
        a["dtype"], a["Q"], a["ck"], a["cv"], a["ks"], a["vs"], a["table"], a["lens"], a["off"], a["QO"], sizes_of(a),
        i64(a["strides"]) if a["strides"] else None, a["scale"], 1, a["ws"], a["ws_bytes"], None) == status


def test_attention_workspace():
    def f(**kw):
        return _lib.lib().mi355_attn_paged_workspace_bytes(sizes_of({**APPEND, "tokens": 0, **kw}))

    assert f(width=128) == 0  # 2048 keys: a work-group for each job
    assert f(width=129) > 0 and f(width=129) % 16 == 0
    assert f(kv_heads=3) == BAD_SIZE and f(head_dim=40) == HEAD and f(page=24) == BAD_SIZE
    assert _lib.lib().mi355_attn_paged_workspace_bytes(None) == NULL


def cache(pages=3, kv_heads=2, page=16, D=64):
    return ops.PagedCache(*empty_cache(pages, kv_heads, page, D))


def int32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    batch = ops.PagedBatch(int32(2, 1), int32(2))
    plan = ops.RotaryPlan(torch.zeros(32, dtype=torch.int64), 64, False, 1.0)
    with pytest.raises(ValueError, match="GPU"):
        ops.rotary(x, torch.arange(2), plan)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_append(cache(), x, x, batch, plan, x)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention_paged(x, cache(), batch)


@pytest.mark.parametrize("kw", [
    dict(dim=0), dict(dim=7), dict(dim=514), dict(base=0.0), dict(base=-1.0), dict(base=math.inf), dict(factor=0.0),
    dict(scaling="other"), dict(scaling="parts"), dict(scaling="parts", original=0), dict(scaling="parts", original=5, slow=2.0, fast=2.0),
    dict(dim=2, scaling="base"), dict(freqs=[1.0]), dict(freqs=[math.nan] * 32), dict(freqs=[1.0] * 32, scaling="linear"),
    dict(amplitude=math.inf), dict(scaling="base", factor=1e300), dict(device="cpu")])
def test_rotary_plan_refusals(kw):
    with pytest.raises(ValueError):
        ops.rotary_plan(**{"dim": 64, **kw})


@pytest.mark.parametrize("x,positions,out", [
    (((4, 2, 64), torch.int8), ((4,), torch.int64), None), (((64,), torch.float16), ((), torch.int64), None),
    (((4, 2, 64), torch.float16), ((5,), torch.int64), None), (((4, 2, 64), torch.float16), ((4,), torch.float32), None),
    (((4, 2, 62), torch.float16), ((4,), torch.int64), None), (((4, 2, 65), torch.float16), ((4,), torch.int64), None),
    (((4, 2, 514), torch.float16), ((4,), torch.int64), None), (((4, 2, 64), torch.float16), ((4,), torch.int64), (4, 3, 64))])
def test_rotary_view_refusals(x, positions, out):
    def stride(shape):
        return torch.empty(shape, device="meta").stride()

    with pytest.raises((TypeError, ValueError)):
        ops._rotary_views(x[1], torch.Size(x[0]), stride(x[0]), positions[1], torch.Size(positions[0]), stride(positions[0]),
                          None if out is None else torch.Size(out), None if out is None else stride(out), 64)


@pytest.mark.parametrize("change", [
    lambda k, v, ks, vs: (k[0], v[0], ks, vs), lambda k, v, ks, vs: (k, v[:2], ks, vs), lambda k, v, ks, vs: (k.view(torch.uint8), v, ks, vs),
    lambda k, v, ks, vs: (k, v, ks[:2], vs), lambda k, v, ks, vs: (k, v, ks.double(), vs), lambda k, v, ks, vs: (k[:, :, :8], v[:, :, :8], ks, vs),
    lambda k, v, ks, vs: (k.transpose(0, 1), v.transpose(0, 1), ks.transpose(0, 1), vs.transpose(0, 1)),
    lambda k, v, ks, vs: (k[..., :40].contiguous(), v[..., :40].contiguous(), ks, vs), lambda k, v, ks, vs: (k, k, ks, vs),
    lambda k, v, ks, vs: (k, v, ks, ks), lambda k, v, ks, vs: (k[:0], v[:0], ks[:0], vs[:0])])
def test_cache_refusals(change):
    with pytest.raises((TypeError, ValueError)):
        ops.PagedCache(*change(*empty_cache(3, 2, 16, 64)))


@pytest.mark.parametrize("kw", [
    dict(table=torch.zeros(2, 3)), dict(table=int32(2)), dict(table=int32(3, 2).t()), dict(lens=int32(3)), dict(lens=torch.zeros(2)),
    dict(lens=int32(4)[::2]), dict(offsets=int32(2)), dict(offsets=torch.zeros(3)), dict(offsets=int32(6)[::2]), dict(most=-1),
    dict(most=1 << 30)])
def test_batch_refusals(kw):
    with pytest.raises(ValueError):
        ops.PagedBatch(**{"table": int32(2, 3), "lens": int32(2), **kw})


@pytest.mark.parametrize("names,shapes,kw", [
    (("q",), ((2, 4, 64),), dict(dtypes=(torch.float32,))), (("q",), ((2, 3, 64),), {}), (("q",), ((2, 4, 32),), {}),
    (("q",), ((3, 4, 64),), {}), (("q",), ((2, 64),), {}), (("q", "out"), ((2, 4, 64), (2, 2, 64)), {}),
    (("q", "out"), ((2, 4, 64), (3, 4, 64)), dict(ragged=True)), (("k", "v"), ((2, 4, 64), (2, 2, 64)), {}),
    (("k", "v"), ((2, 2, 64), (2, 2, 64)), dict(dtypes=(torch.float16, torch.bfloat16))), (("k", "v", "q"), ((2, 2, 64), (2, 2, 64), (1, 4, 64)), {}),
    (("q",), ((2, 4, 64),), dict(table=(2, 1 << 26))), (("q",), ((2, 4, 64),), dict(strides=((256, 60, 1),))),
    (("q",), ((2, 4, 64),), dict(strides=((256, 64, 2),))), (("q", "out"), ((2, 4, 64), (2, 4, 64)), dict(strides=((256, 64, 1), (0, 64, 1)))),
    (("q",), ((2, 4, 64),), dict(ragged=True, most=1 << 21))])
def test_paged_view_refusals(names, shapes, kw):
    shapes = tuple(torch.Size(s) for s in shapes)
    strides = kw.get("strides", tuple(torch.empty(s, device="meta").stride() for s in shapes))
    with pytest.raises((TypeError, ValueError)):
        ops._paged_views(torch.Size((9, 2, 16, 64)), torch.Size(kw.get("table", (2, 4))), (4, 1), kw.get("most", 1), kw.get("ragged", False),
                         names, kw.get("dtypes", (torch.float16,) * len(names)), shapes, strides)


def test_reference_scale_and_rotation():
    assert block_scale(448.0) == 1.0 and block_scale(449.0) == 2.0 and block_scale(0.0) == 2.0 ** -118
    assert block_scale(448 * 2.0 ** -118) == 2.0 ** -118 and block_scale(450 * 2.0 ** -118) == 2.0 ** -117
    x = torch.randn(3, 2, 8, dtype=torch.float64)
    p = torch.tensor([0, 5, 1000])
    y, _ = rotate64(x, p, frequencies(8))
    back, _ = rotate64(y, p, frequencies(8), inverse=True)
    assert torch.equal(y[0], x[0]) and (back - x).abs().max() < 1e-12
    k, v, ks, vs = empty_cache(2, 1, 32, 16, seed=1)
    assert values64(k, ks).isfinite().all() and values64(v, vs).shape == (2, 1, 32, 16)
