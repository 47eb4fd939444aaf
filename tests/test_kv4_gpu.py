"""The 4-bit KV cache on the GPU, against plain 64-bit forms: append with rotary,
read-back and decode attention, and the three together."""
import math

import pytest
import torch

from kv4_common import (D, attend64, pack, parts, quantise32, random_pool, rotate64, rotation_bound, rounding, values)

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def _kv4():
    from directaccesskernel_b200 import kv4

    return kv4


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ append
def _append_case(T, B, Hq, Hkv, page, group, rotary_dim, inter, scale, dtype, seed, pad=0, tiers=True, decode=False):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D + pad, generator=g).to(dtype)
    if decode:
        seq, pos = torch.arange(T), torch.randint(0, 100, (T,), generator=g)
    else:  # distinct (sequence, position) pairs in any order
        pick = torch.randperm(B * 100, generator=g)[:T]
        seq, pos = pick // 100, pick % 100
    width = -(-100 // page)
    ids = torch.randperm(B * width, generator=g).view(B, width)
    table = torch.where(ids % 3 == 0, -1 - ids // 3, ids - ids // 3 - 1) if tiers else ids  # a third on the host
    n_dev, n_host = B * width, (B * width + 2) // 3 if tiers else 0
    inv = (1.0 / 10000 ** (torch.arange(0, rotary_dim, 2).float() / rotary_dim)) if rotary_dim else None
    return qkv, seq, pos, table, n_dev, n_host, inv


@pytest.mark.parametrize("T,B,Hq,Hkv,page,group,rotary_dim,inter,scale,pad,decode", [
    (1, 1, 1, 1, 16, 128, 128, False, 1.0, 0, True),
    (5, 5, 8, 2, 32, 32, 128, False, 1.0, 8, True),
    (33, 33, 32, 8, 64, 128, 64, False, 1.2, 0, True),
    (257, 3, 4, 1, 16, 64, 64, True, 1.0, 0, False),
    (100, 2, 0, 3, 32, 128, 128, True, 1.1, 0, False),
    (77, 4, 3, 3, 64, 32, 6, True, 1.0, 24, False),
    (130, 2, 5, 5, 16, 32, 48, False, 1.0, 0, False),
    (190, 2, 2, 1, 64, 64, 0, False, 1.0, 0, False),
])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append(T, B, Hq, Hkv, page, group, rotary_dim, inter, scale, pad, decode, dtype):
    kv4 = _kv4()
    qkv, seq, pos, table, n_dev, n_host, inv = _append_case(T, B, Hq, Hkv, page, group, rotary_dim, inter, scale, dtype,
                                                            T + Hq, pad, decode=decode)
    bytes_ = kv4.page_bytes(page, group)
    dev = torch.full((n_dev, Hkv, bytes_), 0xAB, dtype=torch.uint8, device="cuda")
    host = torch.full((n_host, Hkv, bytes_), 0xAB, dtype=torch.uint8).pin_memory()
    q_out = torch.empty(T, Hq, D, dtype=dtype, device="cuda") if Hq else None
    kv4.rope_kv_append_q4(qkv.cuda()[:, :(Hq + 2 * Hkv) * D], pos.int().cuda(), inv.cuda() if inv is not None else None, Hq,
                          q_out, dev, host, table.int().cuda(), seq_index=None if decode else seq.int().cuda(),
                          interleaved=inter, rope_scale=scale)
    torch.cuda.synchronize()
    x = qkv[:, :(Hq + 2 * Hkv) * D].reshape(T, -1, D)
    if Hq:
        ref = rotate64(x[:, :Hq], pos, inv, inter, scale)
        assert ((q_out.cpu().double() - ref).abs()
                <= rounding(ref, dtype) + rotation_bound(x[:, :Hq], inv, inter, scale) * 1.01).all()
    kc, kp, vc, vp = [torch.cat([a, b]) for a, b in zip(parts(dev.cpu(), page, group), parts(host, page, group))]
    ids = table[seq, pos // page]
    ids = torch.where(ids < 0, n_dev - 1 - ids, ids)
    slot = pos % page
    # v: the format's definition, bit by bit.
    n, p = quantise32(x[:, Hq + Hkv:], group)
    assert torch.equal(vc[ids, :, slot], n) and torch.equal(vp[ids, :, slot], p)
    # k: within half a step of the rotated value, where scale and zero are those of
    # the rotated group to one float16 rounding (2^-11 relative) and the rotation's error.
    ref = rotate64(x[:, Hq:Hq + Hkv], pos, inv, inter, scale)
    err = rotation_bound(x[:, Hq:Hq + Hkv], inv, inter, scale)
    gr, ge = ref.unflatten(-1, (-1, group)), err.unflatten(-1, (-1, group)).amax(-1)
    s, z = kp[ids, :, slot].double().unbind(-1)
    mn, mx = gr.amin(-1), gr.amax(-1)
    tiny = 2.0**-24  # float16's smallest step
    assert ((z - mn).abs() <= mn.abs() * 2**-11 + ge + tiny).all()
    assert ((s - (mx - mn) / 15).abs() <= (mx - mn) / 15 * (2**-11 + 2**-23) + ge + tiny).all()
    got = values(kc[ids, :, slot], kp[ids, :, slot])
    # code * scale reaches at most 15 scale roundings (15 s 2^-11) and one zero rounding short of an end.
    room = s / 2 * (1 + 2**-20) + 15 * s * 2**-11 + z.abs() * 2**-11 + 2 * ge + 16 * tiny
    assert ((got - ref).abs() <= room.repeat_interleave(group, -1)).all()
    # Nothing else is written.
    touched = torch.zeros(n_dev + n_host, page, dtype=torch.bool)
    touched[ids, slot] = True
    for t, fill in ((kc, 0xB), (vc, 0xB)):
        low = t[..., 0::2].transpose(1, 2)[~touched]
        assert (low == fill).all()
    for t in (kp, vp):
        assert (t.view(torch.int16).transpose(1, 2)[~touched] == torch.tensor(0xABAB - 65536, dtype=torch.int16)).all()


@pytest.mark.parametrize("T,Hq,Hkv,page,group,rotary_dim,inter", [
    (2371, 1, 1, 64, 128, 128, False), (4739, 2, 1, 16, 64, 64, True), (5003, 0, 3, 32, 32, 48, False),
    (3001, 16, 3, 64, 64, 128, False), (9998, 6, 3, 32, 128, 0, False), (4737, 11, 7, 64, 32, 128, True)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_of_many_tokens_is_that_of_few(T, Hq, Hkv, page, group, rotary_dim, inter, dtype):
    """Many tokens share a CTA: one call writes the bytes that calls of 500 tokens write
    (which test_append compares with the formula), in both tiers."""
    kv4 = _kv4()
    B = 101
    qkv, seq, pos, table, n_dev, n_host, inv = _append_case(T, B, Hq, Hkv, page, group, rotary_dim, inter, 1.1, dtype, T)
    qkv, pos, seq, table = qkv.cuda(), pos.int().cuda(), seq.int().cuda(), table.int().cuda()
    inv = inv.cuda() if inv is not None else None
    got = []
    for step in (T, 500):
        dev = torch.full((n_dev, Hkv, kv4.page_bytes(page, group)), 0xAB, dtype=torch.uint8, device="cuda")
        host = torch.full((n_host, Hkv, kv4.page_bytes(page, group)), 0xAB, dtype=torch.uint8).pin_memory()
        q_out = torch.zeros(T, Hq, D, dtype=dtype, device="cuda")
        for i in range(0, T, step):
            n = slice(i, min(T, i + step))
            kv4.rope_kv_append_q4(qkv[n], pos[n], inv, Hq, q_out[n] if Hq else None, dev, host, table, seq_index=seq[n],
                                  interleaved=inter, rope_scale=1.1)
        torch.cuda.synchronize()
        got.append((dev, host, q_out))
    for one, other in zip(*got):
        assert torch.equal(one, other)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_append_of_extreme_values(group):
    """Constant groups, the type's extremes, infinities and NaN: finite, saturated contents."""
    kv4 = _kv4()
    rows = torch.randn(7, 1, D, generator=torch.Generator().manual_seed(1))
    rows[0] = 0.0
    rows[1] = -3.25
    rows[2, 0, 5], rows[2, 0, 70] = 3e38, -3e38
    rows[3, 0, 9] = math.inf
    rows[4, 0, 100] = -math.inf
    rows[5, 0, ::2] = math.nan
    rows[6] = math.nan
    x = rows.to(torch.bfloat16)
    qkv = torch.cat([x, x], 1).reshape(7, 2 * D).cuda()
    pool = torch.zeros(1, 1, kv4.page_bytes(16, group), dtype=torch.uint8, device="cuda")
    kv4.rope_kv_append_q4(qkv, _i32(list(range(7))), None, 0, None, pool, None, _i32([[0]]), seq_index=_i32([0] * 7))
    kc, kp, vc, vp = parts(pool.cpu(), 16, group)
    assert torch.equal(kc, vc) and torch.equal(kp, vp)
    got = values(vc, vp)[0, 0, :7]
    assert torch.isfinite(got).all()
    n, p = quantise32(x[:3, 0], group)
    assert torch.equal(vc[0, 0, :3], n) and torch.equal(vp[0, 0, :3], p)
    assert (got[0] == 0).all() and (got[1] == -3.25).all()
    assert (vc[0, 0, 5, ::2] == 0).all()
    keep = x[5, 0, 1::2].double()  # numbers beside NaN: the group's range is theirs
    s = vp[0, 0, 5].double()[:, 0].repeat_interleave(group // 2)
    assert ((got[5, 1::2] - keep).abs() <= s / 2 + 15 * s * 2**-11 + 4 * 2**-11).all()
    k, v = kv4.kv_read_q4(pool, None, _i32([[0]]), _i32(list(range(7))), seq_index=_i32([0] * 7), dtype=torch.bfloat16)
    assert torch.isfinite(k).all() and torch.equal(k, v)


def test_append_records_bad_entries_and_writes_the_rest():
    from directaccesskernel_b200 import _lib, runtime

    kv4 = _kv4()
    pool = torch.zeros(2, 1, kv4.page_bytes(16, 32), dtype=torch.uint8, device="cuda")
    host = torch.zeros(1, 1, kv4.page_bytes(16, 32), dtype=torch.uint8).pin_memory()
    qkv = torch.randn(6, 3 * D, generator=torch.Generator().manual_seed(2)).half().cuda()
    q_out = torch.empty(6, 1, D, dtype=torch.float16, device="cuda")
    table = _i32([[0, 2], [-2, 1]])
    assert runtime.device_status() == 0
    # (seq 0, page 1 -> 2: outside), (seq 1, page 0 -> host 1: outside), negative, past the table, sequence 2, and a good one
    kv4.rope_kv_append_q4(qkv, _i32([20, 3, -1, 32, 0, 17]), None, 1, q_out, pool, host, table,
                          seq_index=_i32([0, 1, 0, 0, 2, 1]))
    assert runtime.device_status(clear=True) == _lib.DAK_ERR_INVALID_ARG
    kc, _, vc, _ = parts(pool.cpu(), 16, 32)
    n, _ = quantise32(qkv.cpu()[5].view(3, D)[1:], 32)
    assert torch.equal(kc[1, 0, 1], n[0]) and torch.equal(vc[1, 0, 1], n[1])
    kc[1, 0, 1], vc[1, 0, 1] = 0, 0
    assert not kc.any() and not vc.any() and not host.any()
    assert torch.equal(q_out.view(6, D), qkv[:, :D])  # q needs no page
    k, v = kv4.kv_read_q4(pool, host, table, _i32([20, 17]), seq_index=_i32([0, 1]))
    assert runtime.device_status(clear=True) == _lib.DAK_ERR_INVALID_ARG
    assert not k[0].any() and not v[0].any() and k[1].any()


# -------------------------------------------------------------------- read
@pytest.mark.parametrize("page,group,Hkv,T", [(16, 32, 1, 1), (32, 64, 3, 70), (64, 128, 8, 333), (16, 128, 2, 1000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_read(page, group, Hkv, T, dtype):
    kv4 = _kv4()
    pool, host = random_pool(5, Hkv, page, group, 3), random_pool(4, Hkv, page, group, 4)
    table = torch.tensor([[0, -1, 4], [-4, 2, 3]])
    g = torch.Generator().manual_seed(T)
    seq, pos = torch.randint(0, 2, (T,), generator=g), torch.randint(0, 3 * page, (T,), generator=g)  # repeats too
    k, v = kv4.kv_read_q4(pool.cuda(), host.pin_memory(), table.int().cuda(), pos.int().cuda(), seq_index=seq.int().cuda(),
                          dtype=dtype)
    both = torch.cat([pool, host])
    e = table[seq, pos // page]
    e = torch.where(e < 0, 4 - e, e)
    for got, (c, p) in zip((k, v), ((0, 1), (2, 3))):
        c, p = parts(both, page, group)[c][e, :, pos % page], parts(both, page, group)[p][e, :, pos % page]
        p = p.float().repeat_interleave(group, dim=-2)
        assert torch.equal(got.cpu(), (c.float() * p[..., 0] + p[..., 1]).to(dtype))


def test_read_of_no_tokens_and_given_outputs():
    kv4 = _kv4()
    pool = random_pool(2, 2, 16, 32, 5).cuda()
    k, v = kv4.kv_read_q4(pool, None, _i32([[0, 1]]), _i32([]), seq_index=_i32([]))
    assert k.shape == v.shape == (0, 2, D)
    k2, v2 = torch.empty(1, 2, D, dtype=torch.float16, device="cuda"), torch.empty(1, 2, D, dtype=torch.float16, device="cuda")
    k, v = kv4.kv_read_q4(pool, None, _i32([[0, 1]]), _i32([31]), k_out=k2, v_out=v2)
    assert k is k2 and v is v2
    with pytest.raises(RuntimeError, match="k_out"):
        kv4.kv_read_q4(pool, None, _i32([[0, 1]]), _i32([31]), dtype=torch.bfloat16, k_out=k2, v_out=v2)


# --------------------------------------------------------------- attention
def _bound(ref, q, k_abs, v_range, scaling, dtype):
    """Absolute error bound of the attention kernel's arithmetic.
    * the output is rounded once: half a step of the dtype;
    * softmax weights times V's scale are rounded to float16 before the product
      (2^-11 relative), so sum_t p_t scale n is off by at most 2^-11 of the
      largest code part, 15 scale = v_range;
    * scores are FP32 sums of 128 products: off by at most 128 * 2^-23 of
      sum |q||k|, and by 2^-22 in exp2 and its argument; a weight error of d moves
      the output by at most 2 d max|v| <= 2 d v_max."""
    q = q.double()
    score = scaling * torch.where(torch.isfinite(q), q, torch.zeros_like(q)).abs().sum(-1).amax() * k_abs
    d = score * 2.0**-16 + 2.0**-20
    return rounding(ref, dtype) + 2.0**-11 * v_range + 2 * d * (v_range + ref[torch.isfinite(ref)].abs().amax())


def _attend(B, Hq, Hkv, page, group, lens, dtype, seed, *, wide=False, width=None, host_every=0, q_pad=0, counters=False,
            max_seq_len=None, spread=1.0, q_scale=1.0, share_out=False):
    kv4 = _kv4()
    g = torch.Generator().manual_seed(seed)
    lens = torch.tensor(lens)
    pages = [-(-max(0, int(n)) // page) for n in lens]
    width = max(width or 1, max(pages), 513 // page + 1 if wide else 1)  # beyond 512 tokens rows may be split
    ids = torch.randperm(sum(pages), generator=g).tolist()
    table = torch.full((B, width), 2**30, dtype=torch.int64)  # entries past a sequence are never read
    n_dev = n_host = 0
    for b in range(B):
        for j in range(pages[b]):
            v = ids.pop()
            if host_every and (b + j) % host_every == 0:
                table[b, j], n_host = -1 - v, max(n_host, v + 1)
            else:
                table[b, j], n_dev = v, max(n_dev, v + 1)
    pool = random_pool(max(1, n_dev), Hkv, page, group, seed + 1, spread)
    host = random_pool(n_host, Hkv, page, group, seed + 2, spread) if n_host else None
    q = (torch.randn(B, Hq, D + q_pad, generator=g) * q_scale).to(dtype)
    scaling = 1 / math.sqrt(D)
    limit = max_seq_len or width * page
    cnt = torch.zeros(kv4.merge_counter_count(B, Hq, Hkv), dtype=torch.int32, device="cuda") if counters else None
    got = kv4.decode_paged_q4(q.cuda()[..., :D], pool.cuda(), host.pin_memory() if host is not None else None,
                              table.int().cuda(), lens.int().cuda(), scaling, max_seq_len=max_seq_len,
                              merge_counters=cnt)
    if counters:
        assert not cnt.any()
    ref = attend64(q[..., :D], (pool, host), page, group, table, lens.clamp(max=limit), scaling)
    both = [p for p in (pool, host) if p is not None]
    k_abs = max(values(*parts(p, page, group)[:2]).abs().amax() for p in both)
    v_range = max(15 * parts(p, page, group)[3][..., 0].double().amax() for p in both)
    return got.cpu().double(), ref, _bound(ref, q[..., :D], k_abs, v_range, scaling, dtype)


@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [63], [64], [65], [130], [1000]])
@pytest.mark.parametrize("page,group", [(16, 32), (32, 64), (64, 128)])
@pytest.mark.parametrize("wide", [False, True])
def test_attend_lengths(lens, page, group, wide):
    got, ref, tol = _attend(1, 4, 1, page, group, lens, torch.float16, lens[0], wide=wide)
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize("share", [1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 16, 20])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide", [False, True])
def test_attend_shared_heads(share, dtype, wide):
    got, ref, tol = _attend(2, 2 * share, 2, 16, 64, [100, 70], dtype, share, wide=wide)
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize("counters", [False, True])
@pytest.mark.parametrize("page,group,host_every", [(16, 32, 2), (16, 64, 0), (16, 128, 3), (32, 64, 1), (32, 128, 2),
                                                   (32, 32, 0), (64, 32, 2), (64, 64, 3), (64, 128, 0), (64, 128, 3)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_ragged_tiers_and_splits(counters, page, group, host_every, dtype):
    """Rows of no tokens, one token, page ends, all pages on the host, rows over several CTAs."""
    lens = [0, 1, 777, 64, 500, 2049, 0, 333]
    got, ref, tol = _attend(8, 8, 2, page, group, lens, dtype, page + group, host_every=host_every, counters=counters)
    assert ((got - ref).abs() <= tol).all()
    assert not got[0].any() and not got[6].any()


def test_attend_long_row_and_strided_query():
    got, ref, tol = _attend(1, 8, 1, 64, 128, [40003], torch.bfloat16, 7, q_pad=8)
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize("max_seq_len", [1, 100, 513, 700])
def test_attend_cuts_rows_at_max_seq_len(max_seq_len):
    got, ref, tol = _attend(2, 4, 2, 16, 32, [800, 90], torch.float16, 8, max_seq_len=max_seq_len)
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize("spread,q_scale", [(1e-4, 1.0), (300.0, 1e-3), (1.0, 200.0), (30.0, 30.0), (1e-4, 3e4)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide", [False, True])
def test_attend_large_and_small_values(spread, q_scale, dtype, wide):
    """Tiny V scales (float16 subnormals after the weights), one-hot softmax, large q."""
    got, ref, tol = _attend(2, 5, 1, 32, 64, [400, 33], dtype, 11, wide=wide, spread=spread, q_scale=q_scale)
    fine = torch.isfinite(ref)  # 3e4 takes some float16 queries to infinity: no reference there
    assert fine.any() and (fine.all() or (dtype == torch.float16 and q_scale == 3e4))
    assert torch.isfinite(got[fine]).all()
    assert ((got - ref).abs() <= tol)[fine].all()


def test_attend_ignores_what_lies_behind_the_last_token():
    """Unused slots of the last page may hold anything, NaN and infinite pairs included."""
    kv4 = _kv4()
    page, group, n = 64, 32, 75
    pool = random_pool(2, 2, page, group, 12)
    clean = pool.clone()
    half = page * (64 + 16)
    for at in (0, half):  # slots 11.. of page 1
        pool[1, :, at + 11 * 64:at + page * 64] = 0xFF
        pool[1, :, at + page * 64 + 11 * 16:at + half] = torch.tensor([0, 0x7E, 0, 0xFC], dtype=torch.uint8).repeat(53 * 4)
    q = torch.randn(1, 6, D, generator=torch.Generator().manual_seed(1)).half().cuda()
    args = (None, _i32([[0, 1]]), _i32([n]), 0.1)
    a, b = (kv4.decode_paged_q4(q, p.cuda(), *args) for p in (clean, pool))
    assert torch.equal(a, b) and torch.isfinite(a).all()


def test_attend_bad_pages_read_zeros_and_are_recorded():
    from directaccesskernel_b200 import _lib, runtime

    kv4 = _kv4()
    pool = random_pool(3, 1, 16, 64, 13)
    table = torch.tensor([[0, 3, 1], [-1, 2, 0]])
    q = torch.randn(2, 3, D, generator=torch.Generator().manual_seed(2)).half()
    assert runtime.device_status() == 0
    got = kv4.decode_paged_q4(q.cuda(), pool.cuda(), None, table.int().cuda(), _i32([40, 48]), 0.1)
    assert runtime.device_status(clear=True) == _lib.DAK_ERR_INVALID_ARG
    ref = attend64(q, (pool, None), 16, 64, table, [40, 48], 0.1)
    v_range = 15 * parts(pool, 16, 64)[3][..., 0].double().amax()
    k_abs = values(*parts(pool, 16, 64)[:2]).abs().amax()
    assert ((got.cpu().double() - ref).abs() <= _bound(ref, q, k_abs, v_range, 0.1, torch.float16)).all()


def test_attend_nan_query_stays_in_its_row():
    kv4 = _kv4()
    pool = random_pool(4, 1, 16, 32, 14).cuda()
    q = torch.randn(2, 4, D, generator=torch.Generator().manual_seed(3)).half()
    table, lens = _i32([[0, 1], [2, 3]]), _i32([30, 30])
    good = kv4.decode_paged_q4(q.cuda(), pool, None, table, lens, 0.1)
    q[0, 2, 5] = math.nan
    bad = kv4.decode_paged_q4(q.cuda(), pool, None, table, lens, 0.1)
    assert torch.isnan(bad[0, 2]).all()
    keep = torch.ones(2, 4, dtype=torch.bool)
    keep[0, 2] = False
    assert torch.equal(bad.cpu()[keep], good.cpu()[keep])


def test_attend_same_bits_with_counters_and_every_time():
    kv4 = _kv4()
    pool = random_pool(40, 2, 64, 128, 15).cuda()
    q = torch.randn(2, 16, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    table, lens = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20), _i32([1280, 901])
    cnt = torch.zeros(kv4.merge_counter_count(2, 16, 2), dtype=torch.int32, device="cuda")
    first = kv4.decode_paged_q4(q, pool, None, table, lens, 0.09)
    for _ in range(5):
        assert torch.equal(kv4.decode_paged_q4(q, pool, None, table, lens, 0.09, merge_counters=cnt), first)
        assert torch.equal(kv4.decode_paged_q4(q, pool, None, table, lens, 0.09), first)


@pytest.mark.parametrize("counters", [True, False])
@pytest.mark.parametrize("Hq", [8, 72])
def test_attend_in_place(Hq, counters):
    """out over the query, with rows that are split, whole and empty."""
    kv4 = _kv4()
    g = torch.Generator().manual_seed(Hq)
    lens = [9000, 0, 70, 4000, 1, 2049]
    pool = random_pool(200, 4, 64, 128, Hq).cuda()
    table = torch.randint(0, 200, (6, 141), generator=g, dtype=torch.int32).cuda()
    q = torch.randn(6, Hq, D, generator=g).to(torch.bfloat16).cuda()
    cnt = torch.zeros(kv4.merge_counter_count(6, Hq, 4), dtype=torch.int32, device="cuda") if counters else None
    want = kv4.decode_paged_q4(q, pool, None, table, _i32(lens), 0.1, merge_counters=cnt)
    assert kv4.decode_paged_q4(q, pool, None, table, _i32(lens), 0.1, merge_counters=cnt, out=q) is q
    assert torch.equal(q, want)


def test_attend_refusals():
    kv4 = _kv4()
    pool = random_pool(4, 2, 16, 32, 16).cuda()
    q = torch.zeros(2, 4, D, dtype=torch.float16, device="cuda")
    table, lens = _i32([[0, 1], [2, 3]]), _i32([3, 4])
    ok = dict(query=q, pool_dev=pool, pool_host=None, block_table=table, seq_lens=lens, scaling=0.1)
    for bad, msg in ((dict(query=q[..., :64]), "128"), (dict(query=q.float()), "float16"), (dict(query=q[:, :3]), "divide"),
                     (dict(pool_dev=pool[:, :, ::2]), "contiguous"), (dict(pool_dev=None), "no KV pool"),
                     (dict(pool_host=pool.cpu()), "pinned"), (dict(pool_host=pool), "pinned"),
                     (dict(pool_host=torch.zeros(1, 1, pool.shape[2], dtype=torch.uint8).pin_memory()), "share"),
                     (dict(block_table=table.long()), "int32"), (dict(block_table=table[:1]), "one row"),
                     (dict(seq_lens=lens.cpu()), "seq_lens"), (dict(seq_lens=lens[:1]), "seq_lens"),
                     (dict(max_seq_len=33), "max_seq_len"), (dict(max_seq_len=0), "max_seq_len"),
                     (dict(out=torch.empty(2, 4, D, device="cuda")), "out"),
                     (dict(out=torch.empty(2, 4, 2 * D, dtype=torch.float16, device="cuda")[..., ::2]), "contiguous"),
                     (dict(query=torch.zeros(2, 4, 2 * D + 4, dtype=torch.float16, device="cuda")[..., :D]), "strides"),
                     (dict(out=torch.empty(8 * D + 4, dtype=torch.float16, device="cuda")[4:].view(2, 4, D)), "aligned")):
        with pytest.raises(RuntimeError, match=msg):
            kv4.decode_paged_q4(**{**ok, **bad})
    big = dict(ok, block_table=_i32([[0] * 40, [0] * 40]))
    for bad, msg in ((dict(scratch=torch.empty(10, device="cuda")), "scratch"),
                     (dict(scratch=torch.empty(10**6, device="cuda", dtype=torch.float16)), "scratch"),
                     (dict(merge_counters=torch.zeros(3, dtype=torch.int32, device="cuda")), "merge_counters")):
        with pytest.raises(RuntimeError, match=msg):
            kv4.decode_paged_q4(**{**big, **bad})


def test_attend_many_rows_and_dealt_ranges():
    """More rows than CTAs, ranges that begin and end within rows, given scratch."""
    kv4 = _kv4()
    g = torch.Generator().manual_seed(40)
    B, Hq, Hkv, page = 150, 24, 4, 16
    lens = torch.randint(0, 200, (B,), generator=g)
    lens[::7] = 0
    lens[5], lens[149] = 1500, 700
    pages = -(-lens // page)
    pool = random_pool(97, Hkv, page, 64, 41)
    table = torch.randint(0, 97, (B, int(pages.max())), generator=g)  # shared pages
    q = torch.randn(B, Hq, D, generator=g).to(torch.bfloat16)
    scratch = torch.full((kv4.scratch_floats(B, Hq, Hkv, page, 64, 16 * table.shape[1]),), float("nan"), device="cuda")
    ref = attend64(q, (pool, None), page, 64, table, lens, 0.088)
    k_abs, v_range = values(*parts(pool, page, 64)[:2]).abs().amax(), 15 * parts(pool, page, 64)[3][..., 0].double().amax()
    for cnt in (None, torch.zeros(kv4.merge_counter_count(B, Hq, Hkv), dtype=torch.int32, device="cuda")):
        got = kv4.decode_paged_q4(q.cuda(), pool.cuda(), None, table.int().cuda(), lens.int().cuda(), 0.088, scratch=scratch,
                                  merge_counters=cnt)
        assert ((got.cpu().double() - ref).abs() <= _bound(ref, q, k_abs, v_range, 0.088, torch.bfloat16)).all()
        assert cnt is None or not cnt.any()


@pytest.mark.parametrize("B,Hq,Hkv,longest", [(3, 2, 1, 30000), (31, 4, 2, 4000), (32, 8, 1, 6000), (33, 4, 1, 9000),
                                              (70, 3, 3, 1500), (97, 2, 1, 4000), (128, 1, 1, 3000), (129, 16, 1, 2000),
                                              (260, 2, 2, 700), (297, 1, 1, 900)])
@pytest.mark.parametrize("even", [False, True])
def test_attend_batches_of_every_deal(B, Hq, Hkv, longest, even):
    """Lengths over the logarithm, some zero, or nearly even: pieces of rows, rows and
    ranges, the lengths in one to many blocks of 32, both ways to merge alike."""
    kv4 = _kv4()
    g = torch.Generator().manual_seed(B + longest)
    u = torch.rand(B, generator=g, dtype=torch.float64)
    lens = (longest - 60 * u if even else torch.exp(u * math.log(longest))).long()
    lens[2::5] = longest if even else 0
    lens[B // 2] = longest
    table = torch.randint(0, 61, (B, -(-longest // 64)), generator=g)  # shared pages
    pool = random_pool(61, Hkv, 64, 128, B)
    q = torch.randn(B, Hq, D, generator=g).to(torch.bfloat16)
    cnt = torch.zeros(kv4.merge_counter_count(B, Hq, Hkv), dtype=torch.int32, device="cuda")
    one, two = (kv4.decode_paged_q4(q.cuda(), pool.cuda(), None, table.int().cuda(), lens.int().cuda(), 0.088,
                                    scratch=torch.full((kv4.scratch_floats(B, Hq, Hkv, 64, 128, 64 * table.shape[1]),),
                                                       float("nan"), device="cuda"), merge_counters=c) for c in (cnt, None))
    assert torch.equal(one, two) and not cnt.any()
    some = torch.cat([torch.arange(min(B, 6)), torch.randint(0, B, (12,), generator=g), torch.tensor([B // 2, B - 1])])
    ref = attend64(q[some], (pool, None), 64, 128, table[some], lens[some], 0.088)
    k_abs, v_range = values(*parts(pool, 64, 128)[:2]).abs().amax(), 15 * parts(pool, 64, 128)[3][..., 0].double().amax()
    assert ((one[some.cuda()].cpu().double() - ref).abs() <= _bound(ref, q, k_abs, v_range, 0.088, torch.bfloat16)).all()
    zero = (lens == 0).nonzero().flatten().cuda()
    assert not one[zero].any() and torch.isfinite(one).all()


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_then_steps_in_a_graph_on_another_stream(dtype):
    """A prompt appended in one call, then single tokens by a captured and
    replayed step on a stream of its own, over both tiers."""
    kv4 = _kv4()
    B, Hq, Hkv, page, group, n0, steps = 3, 6, 2, 16, 32, 45, 6
    g = torch.Generator().manual_seed(21)
    total = n0 + steps
    x = torch.randn(B, total, Hq + 2 * Hkv, D, generator=g).to(dtype)
    inv = 1.0 / 10000 ** (torch.arange(0, D, 2).float() / D)
    width = -(-total // page)
    table = torch.tensor([[(b * width + j) if j else -1 - b for j in range(width)] for b in range(B)])
    dev = torch.zeros(B * width, Hkv, kv4.page_bytes(page, group), dtype=torch.uint8, device="cuda")
    host = torch.zeros(B, Hkv, kv4.page_bytes(page, group), dtype=torch.uint8).pin_memory()
    tab, inv_d = table.int().cuda(), inv.cuda()
    seq = torch.arange(B).repeat_interleave(n0)
    pos = torch.arange(n0).repeat(B)
    q_all = torch.empty(B * n0, Hq, D, dtype=dtype, device="cuda")
    kv4.rope_kv_append_q4(x[:, :n0].reshape(B * n0, -1).cuda(), pos.int().cuda(), inv_d, Hq, q_all, dev, host, tab,
                          seq_index=seq.int().cuda())
    qkv = torch.empty(B, (Hq + 2 * Hkv) * D, dtype=dtype, device="cuda")
    where, lens = _i32([n0] * B), _i32([n0 + 1] * B)
    q_buf = torch.empty(B, Hq, D, dtype=dtype, device="cuda")
    out = torch.empty(B, Hq, D, dtype=dtype, device="cuda")
    cnt = torch.zeros(kv4.merge_counter_count(B, Hq, Hkv), dtype=torch.int32, device="cuda")

    def step():
        kv4.rope_kv_append_q4(qkv, where, inv_d, Hq, q_buf, dev, host, tab)
        kv4.decode_paged_q4(q_buf, dev, host, tab, lens, 0.088, out=out, merge_counters=cnt)
        where.add_(1)
        lens.add_(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qkv.copy_(x[:, n0].reshape(B, -1).cuda())
        step()  # warm-up: the first token
        first = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        got = [first]
        for i in range(1, steps):
            qkv.copy_(x[:, n0 + i].reshape(B, -1).cuda())
            graph.replay()
            got.append(out.clone())
    torch.cuda.synchronize()
    dev_c = dev.cpu()
    for i, o in enumerate(got):
        q = rotate64(x[:, n0 + i, :Hq], torch.full((B,), n0 + i), inv, False, 1.0).to(dtype)
        ref = attend64(q, (dev_c, host), page, group, table, [n0 + i + 1] * B, 0.088)
        v_range = 15 * max(parts(p, page, group)[3][..., 0].double().amax() for p in (dev_c, host))
        k_abs = max(values(*parts(p, page, group)[:2]).abs().amax() for p in (dev_c, host))
        # q may round the other way where the FP32 rotation lies at a rounding border: one step of q.
        flip = 0.088 * torch.finfo(dtype).eps * q.double().abs().sum(-1).amax() * k_abs * 2.0**-4
        tol = _bound(ref, q, k_abs, v_range, 0.088, dtype) + 2 * flip * v_range
        assert ((o.cpu().double() - ref).abs() <= tol).all()
    k, v = kv4.kv_read_q4(dev, host, tab, pos.int().cuda(), seq_index=seq.int().cuda(), dtype=dtype)
    err = (k.cpu().double() - rotate64(x[:, :n0, Hq:Hq + Hkv].reshape(B * n0, Hkv, D), pos, inv, False, 1.0)).abs()
    # Half a step of the group: its range is below 2 * 6 (normal values, rotated pairs), 1/30 of it, roundings aside.
    assert err.max() <= 12 / 30 + 0.03


def test_pack_of_the_tests_is_the_formats():
    """The tests' own packing and the append write the same bytes (no rotation)."""
    kv4 = _kv4()
    g = torch.Generator().manual_seed(30)
    k, v = (torch.randn(3, 2, 32, D, generator=g).half() for _ in range(2))
    want = pack(k, v, 32, 64)
    pool = torch.zeros_like(want, device="cuda")
    qkv = torch.cat([k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)], 2).reshape(96, -1).cuda()
    kv4.rope_kv_append_q4(qkv, torch.arange(32, dtype=torch.int32, device="cuda").repeat(3), None, 0, None, pool, None,
                          _i32([[0], [1], [2]]), seq_index=torch.arange(3, dtype=torch.int32, device="cuda").repeat_interleave(32))
    assert torch.equal(pool.cpu(), want)


def test_pools_beyond_32_bit_offsets():
    """Pages whose bytes lie past 4 GiB: append, read, attend and copy."""
    from directaccesskernel_b200.kv_pages import copy_pages

    kv4 = _kv4()
    n = 2**32 // kv4.page_bytes(64, 128) + 40
    pool = torch.empty(n, 1, kv4.page_bytes(64, 128), dtype=torch.uint8, device="cuda")
    small = random_pool(3, 1, 64, 128, 50)
    pool[n - 3:] = small.cuda()
    table, lens = _i32([[n - 1, n - 3, n - 2]]), _i32([150])
    q = torch.randn(1, 8, D, generator=torch.Generator().manual_seed(5)).half().cuda()
    got = kv4.decode_paged_q4(q, pool, None, table, lens, 0.1)
    assert torch.equal(got, kv4.decode_paged_q4(q, small.cuda(), None, _i32([[2, 0, 1]]), lens, 0.1))
    x = torch.randn(1, 2 * D, generator=torch.Generator().manual_seed(6)).half().cuda()
    kv4.rope_kv_append_q4(x, _i32([149]), None, 0, None, pool, None, table)
    k, v = kv4.kv_read_q4(pool, None, table, _i32([149]))
    codes, pairs = quantise32(x.cpu().view(2, D), 128)
    want = values(codes, pairs).half()
    assert torch.equal(k.cpu()[0, 0], want[0]) and torch.equal(v.cpu()[0, 0], want[1])
    copy_pages(pool, None, [n - 2], [n - 9])
    assert torch.equal(pool[n - 9], pool[n - 2])


def test_entry_points_refuse_another_device_or_the_cpu():
    kv4 = _kv4()
    pool = random_pool(2, 1, 16, 32, 51)
    q = torch.zeros(1, 1, D, dtype=torch.float16, device="cuda")
    one, table = _i32([3]), _i32([[0, 1]])
    for call in (lambda: kv4.decode_paged_q4(q, pool, None, table, one, 1.0),
                 lambda: kv4.kv_read_q4(pool, None, table, one),
                 lambda: kv4.kv_read_q4(pool.cuda(), None, table, one.cpu()),
                 lambda: kv4.rope_kv_append_q4(torch.zeros(1, 2 * D, dtype=torch.float16, device="cuda"), one, None, 0, None,
                                               pool, None, table)):
        with pytest.raises(RuntimeError, match="device|CUDA"):
            call()


def test_two_streams_with_their_own_scratch():
    """The same batch on two streams at once, each with scratch and counters of its own."""
    kv4 = _kv4()
    pool = random_pool(60, 2, 32, 64, 52).cuda()
    q = torch.randn(3, 10, D, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).cuda()
    table = torch.randint(0, 60, (3, 100), generator=torch.Generator().manual_seed(8)).int().cuda()
    lens = _i32([3200, 1700, 900])
    want = kv4.decode_paged_q4(q, pool, None, table, lens, 0.09)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            cnt = torch.zeros(kv4.merge_counter_count(3, 10, 2), dtype=torch.int32, device="cuda")
            outs.append([kv4.decode_paged_q4(q, pool, None, table, lens, 0.09, merge_counters=cnt) for _ in range(10)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for out in outs for o in out)


def test_steps_whose_lengths_change_under_one_graph():
    """A graph captured with a long max_seq_len replayed for lengths from none to the limit."""
    kv4 = _kv4()
    page, group, width = 16, 32, 130
    pool = random_pool(200, 1, page, group, 53)
    table = torch.randint(0, 200, (2, width), generator=torch.Generator().manual_seed(9))
    q = torch.randn(2, 4, D, generator=torch.Generator().manual_seed(10)).half()
    dev, tab, qd, lens = pool.cuda(), table.int().cuda(), q.cuda(), _i32([5, 9])
    cnt = torch.zeros(kv4.merge_counter_count(2, 4, 1), dtype=torch.int32, device="cuda")
    out = torch.empty_like(qd)
    kv4.decode_paged_q4(qd, dev, None, tab, lens, 0.1, out=out, merge_counters=cnt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv4.decode_paged_q4(qd, dev, None, tab, lens, 0.1, out=out, merge_counters=cnt)
    v_range = 15 * parts(pool, page, group)[3][..., 0].double().amax()
    k_abs = values(*parts(pool, page, group)[:2]).abs().amax()
    for pair in ([0, 0], [1, 2080], [2080, 0], [64, 65], [700, 1300]):
        lens.copy_(torch.tensor(pair, dtype=torch.int32))
        graph.replay()
        ref = attend64(q, (pool, None), page, group, table, pair, 0.1)
        assert ((out.cpu().double() - ref).abs() <= _bound(ref, q, k_abs, v_range, 0.1, torch.float16)).all()
        assert not cnt.any()
