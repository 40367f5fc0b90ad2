"""The token-generation operators where their documentation allows what the first tests do not do: plans
dropped while another stream still has to read them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ops():
    from tiktok_techjam_2026_track3_amd import ops
    return ops


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


# ------------------------------------------------------------------------------ a plan's table
def test_plan_dropped_while_another_stream_has_to_read_it(gpu):
    """A plan made on the default stream, used on a side stream that is behind, and dropped: its block is not
    handed out again before the side stream is done, so that later tables do not land in it."""
    ops = _ops()
    lens = [300, 17, 64, 5]
    q, k, v = (_rand((sum(lens), h, 64), torch.bfloat16, 70 + h).to(gpu) for h in (4, 2, 2))
    kw = dict(heads=4, kv_heads=2, head_dim=64, device=gpu)
    want = ops.attention_packed(q, k, v, ops.packed_plan(lens, **kw))
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    plan = ops.packed_plan(lens, **kw)
    shape, where = plan.tiles.shape, plan.tiles.data_ptr()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        ops.attention_packed(q, k, v, plan, out=out)
    del plan
    later = [torch.empty(shape, dtype=torch.int32, device=gpu) for _ in range(8)]
    busy = not side.query()
    assert all(t.data_ptr() != where for t in later) or not busy
    for t in later:
        t.zero_()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
