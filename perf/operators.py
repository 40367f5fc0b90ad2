"""Operators of token generation: attention over packed prompts with grouped heads, attention of a
batch's new tokens against a prefix they share and their own caches, and projections with 4-bit
weights. Each case is one call; ``run`` makes it in plain torch operations, or, with ``own``, over the
package's public entry points.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # three short prompts of a chat front end: a call whose time is its launches
        dict(name="packed tiny", op="packed", dtype="fp16", seqs=3, lo=1, hi=40, ctx=0, lens=1, heads=8,
             kv_heads=2, dim=64, causal=True),
        # an admission batch: prompts of very different lengths, eight query heads to a K/V head
        dict(name="packed ragged", op="packed", dtype="bf16", seqs=24, lo=33, hi=2011, ctx=0, lens=2,
             heads=32, kv_heads=4, dim=128, causal=True),
        # one long document
        dict(name="packed long", op="packed", dtype="bf16", seqs=1, lo=8192, hi=8192, ctx=0, lens=3,
             heads=32, kv_heads=8, dim=128, causal=True),
        # the next piece of prompts taken in pieces: new tokens against a longer context, no grouping
        dict(name="packed pieces", op="packed", dtype="fp16", seqs=8, lo=200, hi=512, ctx=5000, lens=4,
             heads=16, kv_heads=16, dim=64, causal=True),
        # a few chats behind a short instruction: latency
        dict(name="prefix small", op="prefix", dtype="fp16", batch=4, tokens=1, prefix=300, room=128,
             lens=5, heads=8, kv_heads=2, dim=64),
        # a serving batch behind a long instruction
        dict(name="prefix batch", op="prefix", dtype="bf16", batch=64, tokens=1, prefix=8192, room=1024,
             lens=6, heads=32, kv_heads=8, dim=128),
        # questions on one long document
        dict(name="prefix long", op="prefix", dtype="fp16", batch=16, tokens=1, prefix=65521, room=4096,
             lens=7, heads=32, kv_heads=8, dim=128),
        # drafted tokens checked four at a time, no grouping
        dict(name="prefix draft", op="prefix", dtype="bf16", batch=24, tokens=4, prefix=2047, room=777,
             lens=8, heads=16, kv_heads=16, dim=64),
        # the smallest model's projection for one token
        dict(name="i4 small", op="i4", dtype="fp16", rows=1, n=256, k=256, group=32, zeros=False,
             bias=True),
        # packed QKV projection of one token at d_model 4096
        dict(name="i4 token", op="i4", dtype="fp16", rows=1, n=12288, k=4096, group=128, zeros=True,
             bias=True),
        # FFN input projection of a small batch
        dict(name="i4 batch", op="i4", dtype="bf16", rows=16, n=16384, k=4096, group=128, zeros=True,
             bias=False),
        # FFN output projection of an odd batch: few features, a long sum
        dict(name="i4 tall", op="i4", dtype="bf16", rows=7, n=4096, k=16384, group=64, zeros=False,
             bias=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("packed", "prefix", "i4"))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "i4":
        group = rng.choice((32, 64, 128))
        n, k = _log_int(rng, 64, 16384), group * _log_int(rng, max(1, 128 // group), 16384 // group)
        return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, 16), n=n, k=min(k, 64 * 10 ** 6 // n // group * group),
                    group=group, zeros=rng.random() < 0.5, bias=rng.random() < 0.5)
    kv_heads, grouped = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 8))
    heads, dim, lens = kv_heads * grouped, rng.choice((32, 64, 64, 80, 128, 128)), rng.randrange(1 << 30)
    if op == "packed":
        seqs = _log_int(rng, 1, 48)
        hi = _log_int(rng, 8, max(8, int(8192 / seqs ** 0.6)))
        return dict(op=op, dtype=dtype, seqs=seqs, lo=rng.choice((1, 1 + hi // 3)), hi=hi,
                    ctx=rng.choice((0, 0, _log_int(rng, 16, 4096))), lens=lens, heads=heads,
                    kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.8)
    batch = _log_int(rng, 1, 64)
    return dict(op=op, dtype=dtype, batch=batch, tokens=rng.choice((1, 1, 1, 2, 5)),
                prefix=_log_int(rng, 64, 32768), room=_log_int(rng, 16, 2048), lens=lens, heads=heads,
                kv_heads=kv_heads, dim=dim)


def _packed_lens(case):
    """(query lengths, key lengths): lengths between lo and hi (over their logarithm), keys up to ctx more."""
    rng = random.Random(case["lens"])
    q = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    return q, [n + (rng.randint(case["ctx"] // 2, case["ctx"]) if case["ctx"] else 0) for n in q]


def _own_lens(case):
    """Keys in each sequence's own cache, its new tokens among them."""
    rng = random.Random(case["lens"])
    return [rng.randint(min(case["tokens"], case["room"]), case["room"]) for _ in range(case["batch"])]


def prepare(case, seed):
    dtype, dev = _DTYPES[case["dtype"]], "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    st = dict(case)
    if case["op"] == "i4":
        n, k, group = case["n"], case["k"], case["group"]
        st["x"] = (rand(case["rows"], k) * (1 + 3 * (rand(1, k) > 2.5))).to(dtype)  # a few channels stand out
        st["w"] = torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8)
        st["scale"] = ((0.5 + torch.rand(n, k // group, generator=g, device=dev)) * 0.2 * k ** -0.5).to(dtype)
        st["zero"] = (torch.randint(5, 11, (n, k // group), generator=g, device=dev, dtype=torch.uint8)
                      if case["zeros"] else None)
        st["b"] = rand(n) * 0.1 if case["bias"] else None
        return st
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    channel = 0.5 * rand(kh, d)  # keys have a mean of their own in each channel
    if case["op"] == "packed":
        q_lens, k_lens = _packed_lens(case)
        tq, tk = sum(q_lens), sum(k_lens)
        st.update(q=rand(tq, h, d).to(dtype), k=(rand(tk, kh, d) + channel).to(dtype), v=rand(tk, kh, d).to(dtype))
        st.update(q_lens=torch.tensor(q_lens, device=dev), k_lens=torch.tensor(k_lens, device=dev),
                  max_q=max(q_lens), max_k=max(k_lens))
        st["plan"] = _ops().packed_plan(q_lens, k_lens, heads=h, kv_heads=kh, head_dim=d,
                                        causal=case["causal"], device=dev) if own else None
        return st
    b, n, room = case["batch"], case["tokens"], case["room"]
    st.update(q=rand(b, n, h, d).to(dtype), kp=(rand(case["prefix"], kh, d) + channel).to(dtype),
              vp=rand(case["prefix"], kh, d).to(dtype), ks=(rand(b, room, kh, d) + channel).to(dtype),
              vs=rand(b, room, kh, d).to(dtype))
    st["own_lens"] = torch.tensor(_own_lens(case), device=dev, dtype=torch.int32)
    return st


def _ops():
    from tiktok_techjam_2026_track3_amd import ops
    return ops


def run(st):
    if own:
        ops = _ops()
        if st["op"] == "packed":
            return ops.attention_packed(st["q"], st["k"], st["v"], st["plan"])
        if st["op"] == "prefix":
            return ops.attention_shared_prefix(st["q"], st["kp"], st["vp"], st["ks"], st["vs"], st["own_lens"])
        return ops.linear_i4(st["x"], st["w"], st["scale"], st["zero"], st["b"])
    return {"packed": _plain_packed, "prefix": _plain_prefix, "i4": _plain_i4}[st["op"]](st)


def _softmax(s):
    """Softmax of the last axis, zeros where it holds nothing but -inf."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_packed(st):
    """The sequences padded to the longest, one batched product for the scores and one for the outputs."""
    q, k, v, dev = st["q"], st["k"], st["v"], st["q"].device
    (tq, h, d), kh = q.shape, k.shape[1]
    g = h // kh
    lq, lk, mq, mk = st["q_lens"], st["k_lens"], st["max_q"], st["max_k"]
    n = lq.numel()
    q0, k0 = lq.cumsum(0) - lq, lk.cumsum(0) - lk
    iq, ik = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
    at_q = (q0[:, None] + iq).clamp_max(tq - 1)
    at_k = (k0[:, None] + ik).clamp_max(k.shape[0] - 1)
    qp = q[at_q].float().view(n, mq, kh, g, d).permute(0, 2, 1, 3, 4).reshape(n, kh, mq * g, d)
    kp = k[at_k].float().permute(0, 2, 3, 1).contiguous()
    vp = v[at_k].float().permute(0, 2, 1, 3).contiguous()
    seen = (ik < lk[:, None])[:, None, :]
    if st["causal"]:
        seen = seen & (ik <= iq[:, None] + (lk - lq)[:, None, None])
    s = torch.matmul(qp, kp).mul_(d ** -0.5).view(n, kh, mq, g, mk)
    s.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    o = torch.matmul(_softmax(s).view(n, kh, mq * g, mk), vp)
    o = o.view(n, kh, mq, g, d).permute(0, 2, 1, 3, 4).reshape(n * mq, h, d)
    rows = torch.arange(tq, device=dev)
    seq = torch.searchsorted(lq.cumsum(0), rows, right=True)
    return o[seq * mq + rows - q0[seq]].to(q.dtype)


def _plain_prefix(st):
    """Scores against the prefix as one product for the whole batch, against the caches as a batched one."""
    q, dev = st["q"], st["q"].device
    (b, n, h, d), (p, kh), room = q.shape, st["kp"].shape[:2], st["ks"].shape[1]
    g = h // kh
    qf = q.float().view(b, n, kh, g, d).permute(2, 0, 1, 3, 4).contiguous()  # [kh, b, n, g, d]
    own_q = qf.permute(1, 0, 2, 3, 4).reshape(b, kh, n * g, d)
    sp = torch.matmul(qf.view(kh, b * n * g, d), st["kp"].float().permute(1, 2, 0).contiguous())
    ss = torch.matmul(own_q, st["ks"].float().permute(0, 2, 3, 1).contiguous())
    j, i = torch.arange(room, device=dev), torch.arange(n, device=dev)
    seen = j <= (st["own_lens"][:, None] - n + i)[:, :, None]  # [b, n, room]
    ss = ss.view(b, kh, n, g, room).masked_fill(~seen[:, None, :, None, :], -math.inf)
    s = torch.cat((sp.view(kh, b, n, g, p).permute(1, 0, 2, 3, 4), ss), -1) * d ** -0.5
    w = _softmax(s)
    op = torch.matmul(w[..., :p].permute(1, 0, 2, 3, 4).reshape(kh, b * n * g, p),
                      st["vp"].float().permute(1, 0, 2).contiguous())
    os = torch.matmul(w[..., p:].reshape(b, kh, n * g, room), st["vs"].float().permute(0, 2, 1, 3).contiguous())
    o = op.view(kh, b, n, g, d).permute(1, 2, 0, 3, 4) + os.view(b, kh, n, g, d).permute(0, 2, 1, 3, 4)
    return o.reshape(b, n, h, d).to(q.dtype)


def _plain_i4(st):
    x, w = st["x"], st["w"]
    n, k = st["n"], st["k"]
    q = torch.stack((w & 15, w >> 4), -1).view(n, -1, st["group"]).float()  # the even k is the low half
    z = st["zero"].float() if st["zero"] is not None else torch.full_like(st["scale"], 8.0).float()
    y = torch.matmul(x.float(), ((q - z[..., None]) * st["scale"].float()[..., None]).view(n, k).t())
    return (y if st["b"] is None else y + st["b"]).to(x.dtype)


def exact(case, seed):
    """The definitions in 64 bits: one sequence (and one K/V head) at a time, 4-bit values by division."""
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "i4":
        w, g = st["w"].to(torch.int64), case["group"]
        q = torch.empty(case["n"], case["k"], dtype=f64, device=w.device)
        q[:, 0::2], q[:, 1::2] = w % 16, w // 16
        z = st["zero"].to(f64) if st["zero"] is not None else 8.0 + 0 * st["scale"].to(f64)
        q = (q - z.repeat_interleave(g, 1)) * st["scale"].to(f64).repeat_interleave(g, 1)
        y = st["x"].to(f64) @ q.t().contiguous()
        return y if st["b"] is None else y + st["b"].to(f64)
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(st["q"].shape, dtype=f64, device=st["q"].device)

    def one(q, k, v, last):
        """q [n, d], keys up to last[i] for row i."""
        s = (q.to(f64) @ k.to(f64).t().contiguous()) / math.sqrt(d)
        s[torch.arange(k.shape[0], device=q.device)[None, :] > last[:, None]] = -math.inf
        return torch.softmax(s, 1) @ v.to(f64)

    if case["op"] == "packed":
        q_lens, k_lens = _packed_lens(case)
        q0 = k0 = 0
        for lq, lk in zip(q_lens, k_lens):
            last = torch.arange(lq, device=out.device) + (lk - lq) if case["causal"] else \
                torch.full((lq,), lk - 1, device=out.device)
            for x in range(h):
                y = x * kh // h
                out[q0:q0 + lq, x] = one(st["q"][q0:q0 + lq, x], st["k"][k0:k0 + lk, y],
                                         st["v"][k0:k0 + lk, y], last)
            q0, k0 = q0 + lq, k0 + lk
        return out
    for b, length in enumerate(_own_lens(case)):
        n, p = case["tokens"], case["prefix"]
        last = torch.arange(n, device=out.device) + (p + length - n)
        for y in range(kh):
            k = torch.cat((st["kp"][:, y], st["ks"][b, :length, y]))
            v = torch.cat((st["vp"][:, y], st["vs"][b, :length, y]))
            for x in range(y * (h // kh), (y + 1) * (h // kh)):
                out[b, :, x] = one(st["q"][b, :, x], k, v, last)
    return out


def work(case):
    if case["op"] == "i4":
        m, n, k = case["rows"], case["n"], case["k"]
        groups = n * k // case["group"]
        return dict(bytes=n * k // 2 + groups * (3 if case["zeros"] else 2) + 2 * m * (k + n)
                    + (4 * n if case["bias"] else 0), flops=2 * m * n * k)
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "packed":
        q_lens, k_lens = _packed_lens(case)
        pairs = sum(lq * lk - (lq * (lq - 1) // 2 if case["causal"] else 0) for lq, lk in zip(q_lens, k_lens))
        return dict(bytes=2 * d * (2 * h * sum(q_lens) + 2 * kh * sum(k_lens)), flops=4 * d * h * pairs)
    lens, n, b = _own_lens(case), case["tokens"], case["batch"]
    pairs = b * n * case["prefix"] + sum(n * length - n * (n - 1) // 2 for length in lens)
    return dict(bytes=2 * d * (2 * h * b * n + 2 * kh * (case["prefix"] + sum(lens))), flops=4 * d * h * pairs)
