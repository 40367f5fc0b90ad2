"""What the token-generation operators do at the edges of their documentation, as far as it shows without a
GPU: how long a plan's table lives, 4-bit weights of every magnitude,
what profiles and the build look for."""
import importlib
import re
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from tiktok_techjam_2026_track3_amd import _lib, ops, profiling


# ------------------------------------------------------------------------------ a plan's table
@pytest.mark.parametrize("current,capturing,told", [(11, False, False), (12, False, True), (12, True, False)])
def test_plan_tells_the_allocator_of_other_streams(monkeypatch, current, capturing, told):
    """A call on another stream than the table's is made known to the allocator, which otherwise hands a dropped
    plan's block out again while that stream still has to read it."""
    seen = []
    tiles = SimpleNamespace(record_stream=seen.append)
    plan = ops.PackedPlan(4, 4, 4, 2, 64, True, 64, _lib.i64_array((0, 0, 0, 0)), tiles, 0, stream=11)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: current)
    monkeypatch.setattr(ops, "_current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: ("stream", device, current))
    plan.used_on(3)
    assert seen == ([("stream", 3, current)] if told else [])


@pytest.mark.parametrize("current,capturing", [(3, {3}), (0, {3}), (0, {0}), (3, set())])
def test_capture_is_asked_of_the_plans_device(monkeypatch, current, capturing):
    """... which need not be the current one."""
    at = [current]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            at.append(self.index)

        def __exit__(self, *_):
            at.pop()

    monkeypatch.setattr(ops, "_current_device", lambda: at[-1])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: at[-1] in capturing)
    assert ops._capturing(3) == (3 in capturing) and at == [current]


# ------------------------------------------------------------------------------ 4-bit weights
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def dequantised(q, scale, zero, group):
    n, k = q.shape[0], 2 * q.shape[1]
    v = torch.stack((q & 15, q >> 4), -1).reshape(n, k).double()
    z = zero.double().repeat_interleave(group, 1) if zero is not None else 8.0
    return (v - z) * scale.double().repeat_interleave(group, 1)


@pytest.mark.parametrize("dtype,exps", [(torch.float16, range(0, 25)), (torch.bfloat16, (0, 60, 110, 120, 124, 126, 128, 130, 133))])
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_quant_groups_i4_of_every_magnitude(dtype, exps, symmetric, group):
    """The error relative to the group's own range, down to weights of a few of the type's least numbers. A step
    is range / 15 (largest / 7), its scale off by u of it, or, below the least normal number, up to a least number
    more; a value is off by half a step, the zero point by another half, and by the scale's error over 15 (7) steps
    where it was rounded down."""
    least = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    for e in exps:
        w = (torch.randn(24, 256, generator=torch.Generator().manual_seed(e)) * 2.0 ** -e).to(dtype)
        w[3, :group] = 0
        q, scale, zero = ops.quant_groups_i4(w, group, symmetric)
        assert scale.dtype == dtype and bool((scale > 0).all())
        x = w.double().reshape(24, -1, group)
        span = x.abs().amax(2) / 7 if symmetric else (x.amax(2).clamp_min(0) - x.amin(2).clamp_max(0)) / 15
        bound = (span + least) * (0.5 + (0 if symmetric else 0.5) + 16 * UNIT[dtype])
        err = (dequantised(q, scale, zero, group).reshape(x.shape) - x).abs().amax(2)
        assert bool((err <= bound).all()), (e, float((err / bound).max()))


def test_quant_groups_i4_least_numbers_come_back():
    """Weights that are up to 15 of fp16's least numbers are kept exactly."""
    step = 2.0 ** -24
    w = (torch.randint(0, 16, (8, 64), generator=torch.Generator().manual_seed(1)).double() * step).to(torch.float16)
    w[:, 0], w[:, 32] = 0, 15 * step
    w[:, 1], w[:, 33] = 15 * step, 0
    got = dequantised(*ops.quant_groups_i4(w, 32), 32)
    assert torch.equal(got, w.double())


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_quant_groups_i4_refuses_what_is_not_finite(bad, symmetric):
    for dtype in UNIT:
        w = torch.ones(4, 64, dtype=dtype)
        w[2, 40] = bad
        with pytest.raises(ValueError, match="finite"):
            ops.quant_groups_i4(w, 32, symmetric)
    w = torch.full((4, 64), 3e38, dtype=torch.bfloat16)
    w[:, ::2] = -3e38
    if symmetric:  # +-7 steps reach it
        assert bool(torch.isfinite(ops.quant_groups_i4(w, 32, True)[1]).all())
    else:
        with pytest.raises(ValueError, match="finite"):
            ops.quant_groups_i4(w, 32)


def test_quant_groups_i4_without_rows_or_columns():
    q, scale, zero = ops.quant_groups_i4(torch.zeros(0, 64).half(), 32)
    assert q.shape == (0, 32) and scale.shape == zero.shape == (0, 2)
    with pytest.raises(ValueError):
        ops.quant_groups_i4(torch.zeros(4, 0).half(), 32)


# ------------------------------------------------------------------------------ profiles and the build's checks
def test_profiles_name_every_kernel():
    """The profiler's summaries know every kernel of the library's sources by its own name."""
    csrc = Path(ops.__file__).parent / "csrc"
    names = [n for f in sorted(csrc.iterdir()) for n in re.findall(r"__global__[^;{]*?\bvoid\s+(\w+)\s*\(", f.read_text())]
    assert len(names) > 15 and "linear_i4_held" in names
    for n in names:
        assert profiling.short_name(f"_ZN12_GLOBAL__N_1{len(n)}{n}IDF16_Li64EEEvNS_4ArgsE") == f"{n}<f16,64>"


@pytest.mark.parametrize("vector,bad", [
    ("v_mad_u64_u32 v[2:3], s[6:7], v4, v5, v[6:7]", True), ("v_mad_i64_i32 v[2:3], s[4:5], v4, v5, 0", True),
    ("v_add_co_u32_e64 v2, s[6:7], v3, v4", True), ("v_addc_co_u32_e64 v2, s[6:7], v3, v4, s[8:9]", True),
    ("v_subbrev_co_u32_e64 v2, s[6:7], v3, v4, vcc", True), ("v_div_scale_f32 v2, s[6:7], v3, v4, v5", True),
    ("v_addc_co_u32_e64 v2, vcc, v3, v4, s[6:7]", False),    # carry in only
    ("v_cndmask_b32_e64 v2, v3, v4, s[6:7]", False), ("v_add_u32_e64 v2, s6, v3", False)])
def test_build_sees_carries_as_writes(vector, bad):
    """A carry or scale mask that the vector ALU leaves in scalar registers is a write like any other to the check of
    LDS-DMA loads."""
    build = importlib.import_module("tiktok_techjam_2026_track3_amd.build")
    asm = "\n".join(["attn_rows_x:", "  " + vector, "  s_mov_b32 m0, s20", "  s_nop 0",
                     "  buffer_load_dwordx4 v2, s[4:7], s9 offen lds", "  s_endpgm", ".Lfunc_end0:"])
    assert bool(build.dma_hazards(asm)) == bad


# ------------------------------------------------------------------------------ derivatives
def test_forward_mode_tangents_are_found():
    """A dual tensor is refused, under no_grad too, which leaves forward mode on; plain ones in a level are not."""
    x = torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            ops._no_tangent(None, x, dual)
        ops._no_tangent(x, None, forward_ad.unpack_dual(dual).primal)
