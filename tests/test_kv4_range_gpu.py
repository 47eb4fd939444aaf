"""4-bit decode attention over rows whose tokens and groups differ in magnitude and in
weight: every output is held to a bound of its own row and group."""
import math

import pytest
import torch

from kv4_common import D, pack, parts, rounding, values

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _exact(q, pool, page, group, table, lens, scaling):
    """Outputs in 64 bits and the bound of each, [B, Hq, 128].

    With p the weights, s, c and z the scale, code and zero of V and v = s c + z, an output
    sum_t p v may be off by
    * half a step of the dtype, its one rounding;
    * products p s rounded to float16 (bfloat16 outputs) or to two float16 terms: 2^-11 or
      2^-21 of sum p s c.  Those below 2^-14 of a chunk's unit are off by up to 2^-25 of it, a
      unit being at most the sum of the chunk's products: 64 tokens x 15 x 2^-25 < 2^-15 of sum p s;
    * FP32 sums.  A warp has at most 16 chunks here, each 4 steps of two terms and two
      products with the accumulator: below 200 roundings of 2^-23 (a matrix instruction may
      truncate), of partial sums of at most 17 sum p (15 s + |z|), a 16th of which reaches an
      odd dim: 1.2 x 200 x 2^-23 < 2^-15 of sum p (15 s + |z|);
    * scores off by e: weights by e relative, outputs by 2 e sum p |v|.  A score is summed over
      the n dims where q is not 0 (the others add exact zeros), then takes a scale, a zero, the
      scaling and the largest score's difference: (n + 8) x 2^-23 of sum |q| (s c + |z|), K's;
      exp2 and its argument add 2^-21."""
    B, Hq, _ = q.shape
    kc, kp, vc, vp = parts(pool, page, group)
    kv, width = pool.shape[1], group
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        ids = table[b, :-(-n // page)].long()
        row = lambda t: t[ids].transpose(0, 1).flatten(1, 2)[:, :n].double()  # noqa: E731 [heads, tokens, ...]
        k = values(row(kc), row(kp))
        s, z = (row(vp)[..., i].repeat_interleave(width, -1) for i in (0, 1))
        c = row(vc)
        v = s * c + z
        x = q[b].double().view(kv, -1, D)
        ks, kz = (row(kp)[..., i].repeat_interleave(width, -1) for i in (0, 1))
        p = torch.softmax(torch.einsum("hqd,htd->hqt", x, k) * scaling, -1)
        mass = lambda t: torch.einsum("hqt,htd->hqd", p, t)  # noqa: E731
        nnz = (x != 0).sum(-1, keepdim=True)
        e = torch.einsum("hqd,htd->hqt", x.abs(), ks * row(kc) + kz.abs()).amax(-1, keepdim=True)
        e = e * abs(scaling) * (nnz + 8) * 2.0**-23 + 2.0**-21
        o = mass(v)
        two = q.dtype == torch.float16
        t = (rounding(o, q.dtype) + mass(s * c) * (2.0**-21 if two else 2.0**-11) + mass(s) * 2.0**-15
             + mass(15 * s + z.abs()) * 2.0**-15 + 2 * e * mass(v.abs()))
        out[b], tol[b] = o.view(Hq, D), t.view(Hq, D)
    return out, tol


def _run(kind, lens, page, group, dtype, seed, wide, counters):
    from directaccesskernel_b200 import kv4

    g = torch.Generator().manual_seed(seed)
    B, Hkv, share = len(lens), 2, 5
    n_pages = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(n_pages), generator=g)
    width = max(max(n_pages), 513 // page + 1 if wide else 1)  # beyond 512 tokens rows may be split
    table = torch.zeros(B, width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(n_pages):
        table[b, :n] = ids[at:at + n].int()
        at += n
    k = torch.randn(sum(n_pages), Hkv, page, D, generator=g)
    v = torch.randn(sum(n_pages), Hkv, page, D, generator=g)
    # Scores are q . k over dims 0 and 2 alone: a row's first token gets a score of `sink` nats above 0.
    q = torch.zeros(B, Hkv * share, D)
    q[..., 0] = torch.tensor([4.0, 2.0, 4.0, 1.0, 4.0] * Hkv)
    q[..., 2] = torch.tensor([0.5, -0.5, 0.25, 0.5, 0.0] * Hkv)
    k[..., 0] *= 0.05
    what, amount = kind
    sink = amount if what.startswith("sink") else 11.8  # e^11.8 = 2^17
    for b in range(B):
        if lens[b] == 0:
            continue
        first = (int(table[b, 0]), slice(None), 0)
        k[first][:, 0] = sink / 4
        mid = lens[b] // 2
        loud = (int(table[b, mid // page]), slice(None), mid % page)
        if what == "sink":
            v[first] /= 100
        elif what == "sink0":
            v[first] = 0
        elif what == "silent" and mid > 0:  # no weight, a large V
            k[loud][:, 0] = -12.0
            v[loud] *= amount
        elif what == "both" and mid > 0:
            v[first] *= 1e-3
            k[loud][:, 0] = -12.0
            v[loud] *= amount
    if what == "group":
        v[..., group:2 * group] *= amount
    pool = pack(k, v, page, group)
    q = q.to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    cnt = torch.zeros(kv4.merge_counter_count(B, Hkv * share, Hkv), dtype=torch.int32, device="cuda") if counters else None
    got = kv4.decode_paged_q4(q.cuda(), pool.cuda(), None, table.cuda(), lens_t.cuda(), 1.0, merge_counters=cnt).cpu().double()
    ref, tol = _exact(q, pool, page, group, table, lens, 1.0)
    worst = ((got - ref).abs() / tol.clamp(min=1e-300)).amax()
    assert ((got - ref).abs() <= tol).all(), f"{worst:.3g} times the bound"


KINDS = [("sink", 13.9), ("sink", 16.7), ("sink0", 30.0), ("sink0", 75.0), ("silent", 256.0), ("silent", 1024.0), ("both", 1e3), ("group", 64.0),
         ("group", 1024.0)]


@pytest.mark.parametrize("kind", KINDS, ids=lambda k: f"{k[0]}{k[1]:g}")
@pytest.mark.parametrize("lens,wide,counters", [([130], False, False), ([500], True, False), ([5000], True, True),
                                                ([5000], True, False), ([0, 1, 63, 700, 2500, 65, 1300], True, True)],
                         ids=["short", "pieces", "split", "merged", "ragged"])
@pytest.mark.parametrize("page,group", [(16, 32), (32, 64), (64, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_mixed_magnitudes(kind, lens, wide, counters, page, group, dtype):
    if kind[0] == "group" and group == D:
        pytest.skip("one group")
    _run(kind, lens, page, group, dtype, 7, wide, counters)


def _attend(q, pool, page, lens, scaling):
    """decode_paged_q4 over rows whose pages lie one after the other, and its table."""
    from directaccesskernel_b200 import kv4

    n_pages = [-(-n // page) for n in lens]
    table = torch.zeros(len(lens), max(n_pages), dtype=torch.int32)
    at = 0
    for b, n in enumerate(n_pages):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    got = kv4.decode_paged_q4(q.cuda(), pool.cuda(), None, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scaling)
    return got.cpu().double(), table


@pytest.mark.parametrize("ratio", [200.0, 1000.0, 30000.0])
@pytest.mark.parametrize("channel", [4, 5])
@pytest.mark.parametrize("page,group", [(16, 32), (32, 64), (64, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_query_with_an_outlier_channel(ratio, channel, page, group, dtype):
    """One channel of the query is far larger than the rest and meets keys of exactly 0
    there: the scores are the other channels', whose bits must not be lost to it."""
    g = torch.Generator().manual_seed(3)
    lens, Hkv, share = [2, 40, 700], 2, 4
    pages = sum(-(-n // page) for n in lens)
    k = torch.randn(pages, Hkv, page, D, generator=g).abs()
    k[..., channel] = 0  # its group's minimum: code 0, zero 0
    v = torch.randn(pages, Hkv, page, D, generator=g)
    q = torch.randn(len(lens), Hkv * share, D, generator=g)
    q[..., channel] = ratio
    q, pool = q.to(dtype), pack(k, v, page, group)
    scaling = 1 / math.sqrt(D)
    got, table = _attend(q, pool, page, lens, scaling)
    ref, tol = _exact(q, pool, page, group, table, lens, scaling)
    worst = ((got - ref).abs() / tol).amax()
    assert ((got - ref).abs() <= tol).all(), f"{worst:.3g} times the bound"


@pytest.mark.parametrize("size", [-126, -90, 100, 113, 118, 120, 126])
@pytest.mark.parametrize("page,group", [(16, 32), (32, 64), (64, 128)])
def test_attend_queries_over_the_whole_range_of_bfloat16(size, page, group):
    """Queries of 2^size with a scaling that brings the scores back to ordinary size, and,
    for large ones, a scaling that leaves the largest score's token alone."""
    g = torch.Generator().manual_seed(size + 200)
    lens, Hkv, share = [3, 130, 600], 1, 4
    pages = sum(-(-n // page) for n in lens)
    k, v = (torch.randn(pages, Hkv, page, D, generator=g) for _ in range(2))
    q = torch.randn(len(lens), Hkv * share, D, generator=g).clamp(-1.9, 1.9).to(torch.bfloat16)
    pool = pack(k, v, page, group)
    scaling = 2.0 ** -(size + 3)
    got, table = _attend(q * 2.0**size, pool, page, lens, scaling)
    assert torch.isfinite(q * 2.0**size).all()
    ref, tol = _exact(q * 2.0**size, pool, page, group, table, lens, scaling)
    assert ((got - ref).abs() <= tol).all()
    if size >= 100:
        got, _ = _attend(q * 2.0**size, pool, page, lens, 0.5)
        # Scores are 0.5 x 2^size times those of q, whose two largest lie further apart than
        # FP32 sums of 128 products can be off; the other weights are 0.
        kc, kp = parts(pool, page, group)[:2]
        for b, n in enumerate(lens):
            ids = table[b, :-(-n // page)].long()
            keys = values(kc[ids], kp[ids])[:, 0].reshape(-1, D)[:n]
            s = q[b].double() @ keys.T
            two = s.topk(2, -1).values
            assert (two[:, 0] - two[:, 1] > 2 * 136 * 2.0**-23 * (q[b].double().abs() @ keys.abs().T).amax()).all()
            vc, vp = parts(pool, page, group)[2:]
            rows = values(vc[ids], vp[ids])[:, 0].reshape(-1, D)[:n]
            s16 = vp[ids][:, 0, ..., 0].double().repeat_interleave(group, -1).reshape(-1, D)[:n]
            top = s.argmax(-1)
            assert ((got[b] - rows[top]).abs() <= rounding(rows[top], torch.bfloat16) + 15 * s16[top] * 2.0**-11 + 2.0**-14).all()


@pytest.mark.parametrize("nats", [20.0, 55.0, 65.0])
@pytest.mark.parametrize("n", [357, 5000])
@pytest.mark.parametrize("page,group", [(16, 32), (32, 64), (64, 128)])
def test_attend_one_token_beside_a_silent_sink(nats, n, page, group):
    """Token 255 has the largest score and no V, token 78 comes `nats` below it with all there
    is of V, the others lie 160 nats further down: whole chunks with products of 0 follow 78's."""
    g = torch.Generator().manual_seed(9)
    pages, Hkv, share = -(-n // page), 2, 3
    k, v = (torch.randn(pages, Hkv, page, D, generator=g) for _ in range(2))
    k[..., 0] = -40.0
    k[78 // page, :, 78 % page, 0] = 0.0
    k[255 // page, :, 255 % page, 0] = nats / 4
    v[255 // page, :, 255 % page] = 0
    q = torch.zeros(1, Hkv * share, D)
    q[..., 0] = 4.0
    q, pool = q.to(torch.bfloat16), pack(k, v, page, group)
    got, table = _attend(q, pool, page, [n], 1.0)
    ref, tol = _exact(q, pool, page, group, table, [n], 1.0)
    worst = ((got - ref).abs() / tol).amax()
    assert ((got - ref).abs() <= tol).all(), f"{worst:.3g} times the bound"
