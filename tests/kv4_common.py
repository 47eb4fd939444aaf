"""Plain 64-bit forms of the 4-bit KV cache and of rotary positions, for the tests."""
from __future__ import annotations

import torch

D = 128


def parts(pool: torch.Tensor, page: int, group: int):
    """K codes, K pairs, V codes, V pairs of a pool [..., bytes] (copies): codes
    [..., page, 128] as integers, pairs [..., page, 128 / group, 2] float16."""
    ng = D // group
    half = page * (64 + 4 * ng)
    out = []
    for at in (0, 1):
        h = pool[..., at * half:(at + 1) * half]
        c = h[..., :page * 64].reshape(*pool.shape[:-1], page, 64).int()
        out.append(torch.stack([c & 15, c >> 4], -1).flatten(-2))
        out.append(h[..., page * 64:].contiguous().view(torch.float16).reshape(*pool.shape[:-1], page, ng, 2))
    return out


def values(codes: torch.Tensor, pairs: torch.Tensor) -> torch.Tensor:
    """scale * code + zero in 64 bits, [..., 128]."""
    p = pairs.double().repeat_interleave(D // pairs.shape[-2], dim=-2)
    return codes.double() * p[..., 0] + p[..., 1]


def quantise32(x: torch.Tensor, group: int):
    """The format's codes [..., 128] and pairs [..., 128 / group, 2] of x in FP32,
    operation by operation."""
    g = x.float().unflatten(-1, (D // group, group))
    mn, mx = g.amin(-1), g.amax(-1)
    z = mn.clamp(-65504, 65504).half()
    s = ((mx - mn) / 15).clamp(0, 65504).half()
    inv = torch.where(s > 0, 1.0 / s.float(), torch.zeros_like(s.float()))[..., None]
    n = ((g - z.float()[..., None]) * inv).round().clamp(0, 15)
    return n.flatten(-2).int(), torch.stack([s, z], -1)


def pack(x: torch.Tensor, v: torch.Tensor, page: int, group: int) -> torch.Tensor:
    """Pool [pages, heads, bytes] of keys x and values v [pages, heads, page, 128]."""
    out = []
    for t in (x, v):
        n, p = quantise32(t, group)
        n = n.to(torch.uint8)
        out += [(n[..., 0::2] | (n[..., 1::2] << 4)).flatten(-2), p.flatten(-3).contiguous().view(torch.uint8)]
    return torch.cat(out, -1).contiguous()


def rotate64(x: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor | None, interleaved: bool, scale: float):
    """x [tokens, heads, dim] rotated in 64 bits."""
    x = x.double().clone()
    if inv_freq is None:
        return x
    h = inv_freq.numel()
    t = pos.double()[:, None, None] * inv_freq.double()
    c, s = scale * t.cos(), scale * t.sin()
    i = torch.arange(h)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    x1, x2 = x[..., a], x[..., b]
    x[..., a], x[..., b] = x1 * c - x2 * s, x2 * c + x1 * s
    return x


def rotation_bound(x: torch.Tensor, inv_freq, interleaved: bool, scale: float) -> torch.Tensor:
    """Error bound of the FP32 rotation, per element.  A half turn in FP32 is off by
    2^-25, pi 2^-25 rad of angle; sincospif by 2 units in the last place; the
    factor, two products and the sum round once each: together
    (pi 2^-25 + 2 * 2^-23 + 3 * 2^-24) = 5.1e-7 of scale * (|x1| + |x2|)."""
    b = torch.zeros_like(x.double())
    if inv_freq is None:
        return b
    h = inv_freq.numel()
    i = torch.arange(h)
    p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    both = 5.1e-7 * abs(scale) * (x[..., p].double().abs() + x[..., q].double().abs())
    b[..., p], b[..., q] = both, both
    return b


def rounding(ref: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Half a step of ``dtype`` at ref, subnormals included."""
    fi = torch.finfo(dtype)
    return torch.maximum(ref.abs() * (fi.eps / 2), torch.tensor(fi.tiny * fi.eps / 2, dtype=torch.float64))


def attend64(q, pools, page, group, table, lens, scaling):
    """Decode attention in 64 bits over pools (device, host) [pages, heads, bytes];
    entries outside their pool read as zeros, sequences of no tokens give zeros."""
    B, Hq, _ = q.shape
    kv = next(p for p in pools if p is not None).shape[1]
    vals = [None if p is None else (values(*parts(p, page, group)[:2]), values(*parts(p, page, group)[2:])) for p in pools]
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        rows = []
        for j in range(-(-n // page)):
            e = int(table[b, j])
            tier, idx = (0, e) if e >= 0 else (1, -1 - e)
            ok = vals[tier] is not None and idx < vals[tier][0].shape[0]
            rows.append([vals[tier][a][idx] if ok else torch.zeros(kv, page, D, dtype=torch.float64) for a in (0, 1)])
        k, v = (torch.cat([r[a] for r in rows], 1)[:, :n] for a in (0, 1))
        w = torch.softmax(torch.einsum("hsd,htd->hst", q[b].double().reshape(kv, -1, D), k) * scaling, -1)
        out[b] = torch.einsum("hst,htd->hsd", w, v).reshape(Hq, D)
    return out


def random_pool(pages, heads, page, group, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(pages, heads, page, D, generator=g) * spread + 0.7 * torch.randn(1, heads, 1, D, generator=g)
    v = torch.randn(pages, heads, page, D, generator=g) * spread
    return pack(k, v, page, group)
