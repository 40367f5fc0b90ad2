"""The paged cache's operators in plain 64-bit arithmetic, for its tests."""
import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DTYPES = [torch.float16, torch.bfloat16]
BLOCK = 16


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def frequencies(dim, base=10000.0):
    return [base ** (-2.0 * j / dim) for j in range(dim // 2)]


def rotate64(x, positions, freqs, interleaved=False, amplitude=1.0, inverse=False):
    """x [..., heads, D] in 64 bits, positions of its leading shape: (result, bound of an fp32 evaluation: sine and
    cosine 2^-22.4 off, three roundings on each product)."""
    x, n = x.double(), 2 * len(freqs)
    t = positions.double()[..., None, None] * torch.tensor(freqs, dtype=torch.float64)
    c, s = amplitude * torch.cos(t), amplitude * torch.sin(-t if inverse else t)
    a, b = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    y, tol = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    tol[..., a] = tol[..., b] = abs(amplitude) * 2.0 ** -21 * (x[..., a].abs() + x[..., b].abs())
    return y, tol


def block_scale(top):
    """Least power of two s with top <= 448 s, at least 2^-118."""
    if top <= 448 * 2.0 ** -118:
        return 2.0 ** -118
    m, e = math.frexp(top)
    return 2.0 ** (e - 9 + (m > 0.875))


def empty_cache(pages, kv_heads, page, D, seed=None):
    """CPU tensors of a cache; with a seed, full of values."""
    k, v = (torch.zeros(pages, kv_heads, page, D, dtype=torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros(pages, kv_heads, page // BLOCK) for _ in range(2))
    if seed is not None:
        for i, (t, s) in enumerate(((k, ks), (v, vs))):
            x = rand((pages, kv_heads, page // BLOCK, BLOCK * D), torch.float32, seed + i)
            x = x * torch.exp2(rand((pages, kv_heads, page // BLOCK, 1), torch.float32, seed + 7 + i))
            s.copy_(torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1) / 448))))
            t.copy_((x / s[..., None]).view(t.shape).to(torch.float8_e4m3fn))
    return k, v, ks, vs


def values64(t, s):
    """What a cache's bytes stand for, [pages, kv_heads, page, D]."""
    pages, kv_heads, page, D = t.shape
    x = t.double().view(pages, kv_heads, page // BLOCK, BLOCK, D) * s.double()[..., None, None]
    return x.view(t.shape)


def attention64(q, cache, table, lens, offsets, scale, most=None):
    """q [tokens, heads, D] over cache (k, v, k_scale, v_scale): (result, error bound). Errors: scores (D + 4) 2^-24 scale
    sum |q| |k| and exponentials 2^-20, both in numerator and denominator; probabilities as two bf16 terms 2^-16, or where
    `most` new tokens make more than 32 rows, rounded to q's type in numerator and denominator (fp16 ones below 2^-14 by
    2^-25); sums of m terms m 2^-23; the output's rounding."""
    rows = (max(b - a for a, b in zip(offsets, offsets[1:])) if most is None else most) * (q.shape[1] // cache[0].shape[1])
    once = rows > 32
    k, v = values64(cache[0], cache[2]), values64(cache[1], cache[3])
    pages, kv_heads, page, D = k.shape
    T, H, _ = q.shape
    ref = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros_like(ref)
    for b, m in enumerate(lens):
        first, n = offsets[b], offsets[b + 1] - offsets[b]
        room = min(max(m, 0), table.shape[1] * page)
        for y in range(kv_heads):
            kk, vv = torch.full((room, D), math.nan, dtype=torch.float64), torch.full((room, D), math.nan, dtype=torch.float64)
            for p0 in range(0, room, page):
                at, stop = int(table[b, p0 // page]), min(room, p0 + page)
                if 0 <= at < pages:
                    kk[p0:stop], vv[p0:stop] = k[at, y, :stop - p0], v[at, y, :stop - p0]
            for i in range(n):
                sees = m - n + i + 1
                for x in range(y * (H // kv_heads), (y + 1) * (H // kv_heads)):
                    if sees <= 0:
                        continue
                    if sees > room:
                        ref[first + i, x] = math.nan
                        continue
                    qq = q[first + i, x].double()
                    s = kk[:sees] @ qq * scale
                    w = torch.softmax(s, 0)
                    o = w @ vv[:sees]
                    rel = (2 * UNIT[q.dtype] if once else 2.0 ** -16) + 2 * (2.0 ** -20 + (D + 4) * 2.0 ** -24 * scale * (kk[:sees].abs() @ qq.abs()).max()) + sees * 2.0 ** -23
                    ref[first + i, x] = o
                    tol[first + i, x] = rel * (w @ vv[:sees].abs()) + UNIT[q.dtype] * o.abs() + 2.0 ** -24
                    if once and q.dtype == torch.float16:
                        tol[first + i, x] += sees * 2.0 ** -25 * vv[:sees].abs().amax()
    return ref, tol


def packed(new):
    """offsets of sequences with `new` new tokens each."""
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def check(got, ref, tol, name=""):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{name}: NaN at other places"
    off = ((got - ref).abs() - tol).nan_to_num(-1.0)
    if not off.numel():
        return
    worst = int(off.argmax())
    assert off.max() <= 0, f"{name}: element {worst} is {got.flatten()[worst]}, not {ref.flatten()[worst]} +- {tol.flatten()[worst]}"
