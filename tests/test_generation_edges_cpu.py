"""What the token-generation operators do at the edges of their documentation, as far as it shows without a
GPU: how long a plan's table lives."""
import importlib
from types import SimpleNamespace

import pytest
import torch

from tiktok_techjam_2026_track3_amd import _lib, ops


# ------------------------------------------------------------------------------ a plan's table
@pytest.mark.parametrize("current,capturing,told", [(11, False, False), (12, False, True), (12, True, False)])
def test_plan_tells_the_allocator_of_other_streams(monkeypatch, current, capturing, told):
    """A call on another stream than the table's is made known to the allocator, which otherwise hands a dropped
    plan's block out again while that stream still has to read it."""
    seen = []
    tiles = SimpleNamespace(record_stream=seen.append)
    plan = ops.PackedPlan(4, 4, 4, 2, 64, True, 64, _lib.i64_array((0, 0, 0, 0)), tiles, 0, stream=11)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: current)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: ("stream", device, current))
    plan.used_on(3)
    assert seen == ([("stream", 3, current)] if told else [])
