"""The operators of the 4-bit paged KV cache and the rotary positions in front of it, as cases to time and compare.

A 4-bit cache pool is uint8 [pages, kv_heads, bytes]; one (page, head) slab of P tokens holds, in order,
K codes [P, 64] (dim 2i in the low nibble of byte i), K (scale, zero) float16 pairs [P, 128 / group, 2], V codes, V pairs;
the value of code n is scale * n + zero.  A block-table entry v >= 0 names device page v, v < 0 host page -1 - v.
"""
import math

import torch

own = False

D = 128  # head dimension of the cache
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of 8 sequences: q and k heads of the fused projection, latency-bound.
        dict(name="rotary step 8", op="rotary", tokens=8, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, scale=1.0, far=8192, dtype="bf16"),
        # A long prompt at far positions of a context-extended model (attention factor above one).
        dict(name="rotary prompt 8192", op="rotary", tokens=8192, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, scale=1.1386294, far=131072, dtype="bf16"),
        # One decode step of the 70B-shaped decoder, 32 sequences, all heads on one GPU.
        dict(name="append step 32", op="append", tokens=32, seqs=32, q_heads=64, kv_heads=8, page=64, group=128,
             rotary_dim=128, interleaved=False, scale=1.0, start=16384, dtype="fp16"),
        # Three ragged prompts in one call, part of the head rotated in interleaved pairs, small groups and pages.
        dict(name="append prompts 4099", op="append", tokens=4099, seqs=3, q_heads=32, kv_heads=8, page=32, group=32,
             rotary_dim=64, interleaved=True, scale=1.0, start=100, dtype="bf16"),
        # A short prefix back to 16 bit, for the attention of the tokens that follow it.
        dict(name="read 257", op="read", tokens=257, seqs=1, kv_heads=8, page=16, group=64, dtype="fp16"),
        # Long prefixes of four sequences back to 16 bit.
        dict(name="read 4 x 16384", op="read", tokens=65536, seqs=4, kv_heads=8, page=64, group=128, dtype="bf16"),
        # The first tokens of a chat: one sequence, latency-bound.
        dict(name="attend 1 x 130", op="attend", seqs=1, length=130, ragged=False, kv_heads=8, share=4, page=64,
             group=128, host=0.0, dtype="bf16"),
        # One rank of eight of the 70B-shaped decoder: 32 sequences, one KV head.
        dict(name="attend 32 x 16384 x 1", op="attend", seqs=32, length=16384, ragged=False, kv_heads=1, share=8, page=64,
             group=128, host=0.0, dtype="fp16"),
        # The same batch with every KV head on one GPU: the largest.
        dict(name="attend 32 x 16384 x 8", op="attend", seqs=32, length=16384, ragged=False, kv_heads=8, share=8, page=64,
             group=128, host=0.0, dtype="bf16"),
        # A served batch: lengths from one token up, small groups, an eighth of each sequence's pages in host memory.
        dict(name="attend ragged tiers", op="attend", seqs=24, length=6001, ragged=True, kv_heads=2, share=5, page=32,
             group=32, host=0.125, dtype="bf16"),
        # Forking a few sequences: their last, partly filled pages, in every layer.
        dict(name="fork 8 pages", op="pages", kind="within", slabs=32, pages=64, moves=8, kv_heads=8, page=64, group=128),
        # Compaction after a wave of sequences has left.
        dict(name="compact 397 pages", op="pages", kind="within", slabs=16, pages=1024, moves=397, kv_heads=8, page=64,
             group=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "read", "attend", "attend", "pages"])
    dtype = rng.choice(["bf16", "fp16"])
    page, group = rng.choice([16, 32, 64]), rng.choice([32, 64, 128])
    if op == "rotary":
        d = rng.choice([64, 96, 128, 256])
        inter = rng.random() < 0.5
        r = rng.choice([d, d // 2, 32, rng.randrange(2, d + 1, 2) if inter else 16 * rng.randrange(1, d // 16 + 1)])
        return dict(op=op, tokens=_log(rng, 1, 4096), q_heads=rng.choice([1, 4, 8, 14, 32]), kv_heads=rng.choice([1, 2, 8]),
                    head_dim=d, rotary_dim=r, interleaved=inter, scale=rng.choice([1.0, 1.2079]),
                    far=_log(rng, 100, 1000000), dtype=dtype)
    if op == "append":
        inter = rng.random() < 0.5
        r = rng.choice([0, 128, 64, rng.randrange(2, 129, 2) if inter else 16 * rng.randrange(1, 9)])
        seqs = _log(rng, 1, 64)
        tokens = seqs if rng.random() < 0.4 else max(seqs, _log(rng, 1, 8192))
        kv = rng.choice([1, 2, 3, 8])
        return dict(op=op, tokens=tokens, seqs=seqs, q_heads=kv * rng.choice([1, 2, 4, 5, 8]), kv_heads=kv, page=page,
                    group=group, rotary_dim=r, interleaved=inter, scale=rng.choice([1.0, 1.2079]),
                    start=_log(rng, 1, 20000), dtype=dtype)
    if op == "read":
        seqs = _log(rng, 1, 16)
        return dict(op=op, tokens=max(seqs, _log(rng, 1, 65536)), seqs=seqs, kv_heads=rng.choice([1, 2, 3, 8]), page=page,
                    group=group, dtype=dtype)
    if op == "attend":
        kv, share = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 16])
        seqs = _log(rng, 1, 64)
        length = _log(rng, 1, min(131072, 4000000 // (kv * seqs * max(1, share // 8))))
        return dict(op=op, seqs=seqs, length=length, ragged=rng.random() < 0.6, kv_heads=kv, share=share, page=page,
                    group=group, host=0.0 if kv * seqs * length > 400000 or rng.random() < 0.7 else rng.choice([0.2, 1.0]),
                    dtype=dtype)
    pages = _log(rng, 16, 1024)
    kind = rng.choice(["within", "within", "out", "in"])
    return dict(op=op, kind=kind, slabs=rng.choice([1, 2, 7, 16]) if kind == "within" else 1, pages=pages,
                moves=_log(rng, 1, pages // 2 if kind == "within" else min(pages // 2, 100)), kv_heads=rng.choice([1, 2, 8]),
                page=page, group=group)


# ----------------------------------------------------------------- inputs
def _slab(page, group):
    return 2 * page * (64 + 512 // group)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _store(pool, v0, x, page, group, at):
    """Codes and (scale, zero) of x [pages, heads, page, 128] into the K (at = 0) or V (at = 1) half of pool[v0:...]."""
    ng = 128 // group
    half, cb = page * (64 + 4 * ng), page * 64
    g = x.float().unflatten(-1, (ng, group))
    mn, mx = g.amin(-1), g.amax(-1)
    z, s = mn.half(), ((mx - mn) / 15).half()
    n = ((g - z.float()[..., None]) / s.float()[..., None].clamp(min=1e-12)).round_().clamp_(0, 15).flatten(-2).to(torch.uint8)
    to = pool[v0:v0 + x.shape[0], :, at * half:(at + 1) * half]
    to[..., :cb] = (n[..., 0::2] | (n[..., 1::2] << 4)).flatten(-2)
    to[..., cb:] = torch.stack([s, z], -1).flatten(-3).contiguous().view(torch.uint8)


def _filled(pages, heads, page, group, g):
    """A pool of normally distributed keys and values, with channels that are off centre as real keys have them."""
    pool = torch.empty(pages, heads, _slab(page, group), dtype=torch.uint8, device="cuda")
    off = torch.randn(2, heads, 1, D, generator=g, device="cuda") * torch.tensor([0.8, 0.2], device="cuda").view(2, 1, 1, 1)
    step = max(1, 16_000_000 // (heads * page * D))
    for v0 in range(0, pages, step):
        for at in (0, 1):
            x = torch.randn(min(step, pages - v0), heads, page, D, generator=g, device="cuda")
            _store(pool, v0, x + off[at], page, group, at)
    return pool


def _spread(case, seed):
    """Tokens of a call over its sequences: positions, their sequence and a table of shuffled pages."""
    g = torch.Generator().manual_seed(seed)
    T, B, P = case["tokens"], case["seqs"], case["page"]
    counts = torch.tensor([T // B + (b < T % B) for b in range(B)])
    first = torch.randint(0, case.get("start", 0) + 1, (B,), generator=g)
    seq = torch.repeat_interleave(torch.arange(B), counts)
    pos = torch.arange(T) - (torch.cumsum(counts, 0) - counts)[seq] + first[seq]
    width = -(-int(pos.max() + 1) // P)
    used = -(-(first + counts) // P) - first // P  # pages that this call's tokens touch; the others stay page 0
    table = torch.zeros(B, width, dtype=torch.int32)
    ids = torch.randperm(int(used.sum()), generator=g).to(torch.int32)
    at = 0
    for b in range(B):
        lo, n = int(first[b]) // P, int(used[b])
        table[b, lo:lo + n] = ids[at:at + n]
        at += n
    i32 = lambda t: t.to("cuda", torch.int32)  # noqa: E731
    return i32(pos), i32(seq), table.cuda(), int(used.sum())


def _freqs(r):
    return 1.0 / (500000.0 ** (torch.arange(0, r, 2, dtype=torch.float32, device="cuda") / max(r, 1)))


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    dt = DTYPES.get(case.get("dtype"))
    s = dict(case=case)
    if op == "rotary":
        T, H, d = case["tokens"], case["q_heads"] + case["kv_heads"], case["head_dim"]
        qkv = torch.randn(T, (H + case["kv_heads"]) * d, generator=g, device="cuda").to(dt)
        s["x"] = qkv.view(T, -1, d)[:, :H]  # q and k heads of the fused projection
        s["out"] = torch.empty(T, H, d, dtype=dt, device="cuda")
        s["inv_freq"] = _freqs(case["rotary_dim"])
        s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda", dtype=torch.int32)
    elif op == "append":
        s["positions"], s["seq"], s["table"], pages = _spread(case, seed)
        T, H = case["tokens"], case["q_heads"] + 2 * case["kv_heads"]
        s["qkv"] = torch.randn(T, H * D, generator=g, device="cuda").to(dt)
        s["inv_freq"] = _freqs(case["rotary_dim"]) if case["rotary_dim"] else None
        s["q_out"] = torch.empty(T, case["q_heads"], D, dtype=dt, device="cuda")
        s["pool"] = _filled(pages, case["kv_heads"], case["page"], case["group"], g)
        if case["tokens"] == case["seqs"]:
            s["seq"] = None  # a decode step: token t belongs to sequence t
    elif op == "read":
        s["positions"], s["seq"], s["table"], pages = _spread(case, seed)
        s["pool"] = _filled(pages, case["kv_heads"], case["page"], case["group"], g)
    elif op == "attend":
        B, P, S = case["seqs"], case["page"], case["length"]
        c = torch.Generator().manual_seed(seed)
        lens = torch.full((B,), S)
        if case["ragged"]:  # over the logarithm, one of them the longest
            lens = torch.exp(torch.rand(B, generator=c, dtype=torch.float64) * math.log(S)).round().long().clamp(1, S)
            lens[int(torch.randint(0, B, (1,), generator=c))] = S
        width = -(-S // P)
        n = -(-lens // P)
        host = (n * case["host"]).round().long()  # a sequence's first pages
        table = torch.zeros(B, width, dtype=torch.int32)
        dev_ids = torch.randperm(max(1, int((n - host).sum())), generator=c).to(torch.int32)
        d0 = h0 = 0
        for b in range(B):
            h, m = int(host[b]), int(n[b])
            table[b, :h] = -1 - torch.arange(h0, h0 + h, dtype=torch.int32)
            table[b, h:m] = dev_ids[d0:d0 + m - h]
            h0, d0 = h0 + h, d0 + m - h
        s["table"], s["lens"] = table.cuda(), lens.to("cuda", torch.int32)
        Hq = case["kv_heads"] * case["share"]
        s["q"] = torch.randn(B, Hq, D, generator=g, device="cuda").to(dt)
        s["pool"] = _filled(max(1, d0), case["kv_heads"], P, case["group"], g)
        s["host"] = _filled(h0, case["kv_heads"], P, case["group"], g).cpu().pin_memory() if h0 else None
        s["counters"] = torch.zeros(B * case["kv_heads"] * max(1, -(-case["share"] // 8)), dtype=torch.int32, device="cuda")
    else:
        c = torch.Generator().manual_seed(seed)
        shape = (case["slabs"], case["pages"], case["kv_heads"], _slab(case["page"], case["group"]))
        s["pool"] = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
        ids = torch.randperm(case["pages"], generator=c).to(torch.int32)
        m = case["moves"]
        s["src"], s["dst"] = ids[:m].clone(), ids[m:2 * m].clone()
        s["host"] = None
        if case["kind"] != "within":
            s["host"] = torch.randint(0, 256, shape, generator=c, dtype=torch.uint8).pin_memory()
            s["dst" if case["kind"] == "out" else "src"] = -1 - torch.randperm(case["pages"], generator=c)[:m].to(torch.int32)
    return s


# ------------------------------------------------------------- plain forms
def _rotated(x, positions, inv_freq, interleaved, scale):
    """x [tokens, heads, dim] in 32 bits, its first 2 * inv_freq.numel() dims rotated by positions * inv_freq."""
    x = x.float()
    if inv_freq is None:
        return x
    r = 2 * inv_freq.numel()
    t = positions.double()[:, None] * inv_freq.double()  # 64 bits: far positions
    c, n = (t.cos() * scale).float()[:, None], (t.sin() * scale).float()[:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    y1, y2 = a * c - b * n, b * c + a * n
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., r:]], -1)


def _quantised(x, group):
    """Codes [..., 64] and (scale, zero) [..., 128 / group, 2] of x [..., 128]."""
    g = x.unflatten(-1, (128 // group, group))
    mn, mx = g.amin(-1), g.amax(-1)
    z = mn.clamp(-65504, 65504).half()
    s = ((mx - mn) / 15).clamp(max=65504).half()
    sf = s.float()[..., None]
    inv = torch.where(sf > 0, 1.0 / sf, torch.zeros_like(sf))
    n = ((g - z.float()[..., None]) * inv).round().clamp(0, 15).flatten(-2).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.stack([s, z], -1)


def _parts(pool, page, group):
    """K codes, K pairs, V codes and V pairs of a pool, as views [..., page, 64] and [..., page, 128 / group, 2]."""
    ng = 128 // group
    cb, pb = page * 64, page * 4 * ng
    codes = lambda o: pool[..., o:o + cb].unflatten(-1, (page, 64))  # noqa: E731
    pairs = lambda o: pool[..., o + cb:o + cb + pb].view(torch.float16).unflatten(-1, (page, ng, 2))  # noqa: E731
    return codes(0), pairs(0), codes(cb + pb), pairs(cb + pb)


def _values(codes, pairs, group):
    """32-bit values [..., 128] of codes [..., 64] and pairs [..., 128 / group, 2]."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (128 // group, group))
    p = pairs.float()
    return (n * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _rows(positions, seq, table, page):
    """Page and slot of each token."""
    pos = positions.long()
    seq = torch.arange(pos.numel(), device=pos.device) if seq is None else seq.long()
    return table[seq, pos // page].long(), pos % page


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "rotary":
        s["out"].copy_(_rotated(s["x"], s["positions"], s["inv_freq"], case["interleaved"], case["scale"]))
        return s["out"]
    page, group = case["page"], case["group"]
    if op == "append":
        dt, kv = s["qkv"].dtype, case["kv_heads"]
        x = s["qkv"].view(case["tokens"], -1, D)
        y = _rotated(x[:, :-kv], s["positions"], s["inv_freq"], case["interleaved"], case["scale"])
        s["q_out"].copy_(y[:, :-kv])
        at, slot = _rows(s["positions"], s["seq"], s["table"], page)
        kc, kp, vc, vp = _parts(s["pool"], page, group)
        kc[at, :, slot], kp[at, :, slot] = _quantised(y[:, -kv:], group)
        vc[at, :, slot], vp[at, :, slot] = _quantised(x[:, -kv:].float(), group)
        return (s["q_out"], _values(kc[at, :, slot], kp[at, :, slot], group).to(dt),
                _values(vc[at, :, slot], vp[at, :, slot], group).to(dt))
    if op == "read":
        dt = DTYPES[case["dtype"]]
        at, slot = _rows(s["positions"], s["seq"], s["table"], page)
        kc, kp, vc, vp = _parts(s["pool"], page, group)
        return (_values(kc[at, :, slot], kp[at, :, slot], group).to(dt),
                _values(vc[at, :, slot], vp[at, :, slot], group).to(dt))
    if op == "attend":
        pool, at = s["pool"], s["table"].long()
        if s["host"] is not None:
            at = torch.where(at < 0, pool.shape[0] - 1 - at, at)
            pool = torch.cat([pool, s["host"].to(pool.device, non_blocking=True)])
        kc, kp, vc, vp = _parts(pool[at], page, group)  # [seqs, pages, heads, page, ...]
        B, Hq, kv = case["seqs"], s["q"].shape[1], case["kv_heads"]
        k = _values(kc, kp, group).transpose(1, 2).flatten(2, 3)  # [seqs, heads, tokens, 128]
        q = s["q"].float().view(B, kv, -1, D)
        w = torch.matmul(q, k.transpose(-1, -2)) * (1 / math.sqrt(D))
        del k
        w = w.masked_fill(torch.arange(w.shape[-1], device=w.device) >= s["lens"].view(B, 1, 1, 1), -math.inf)
        w = torch.exp(w - w.amax(-1, keepdim=True))
        v = _values(vc, vp, group).transpose(1, 2).flatten(2, 3)
        return (torch.matmul(w, v) / w.sum(-1, keepdim=True)).view(B, Hq, D).to(s["q"].dtype)
    pool, host = s["pool"], s["host"]
    src, dst = s["src"].long(), s["dst"].long()
    if case["kind"] == "within":
        pool[:, dst.to(pool.device)] = pool[:, src.to(pool.device)]
        return pool
    if case["kind"] == "out":
        host[:, -1 - dst] = pool[:, src.to(pool.device)].cpu()
    else:
        pool[:, dst.to(pool.device)] = host[:, -1 - src].to(pool.device)
    return pool, host


# --------------------------------------------------------------------- run
def run(state):
    s = state
    case, op = s["case"], s["case"]["op"]
    if not own:
        return _plain(s)
    if op == "rotary":
        from directaccesskernel_b200.decode_ops import rotary

        return rotary(s["x"], s["positions"], s["inv_freq"], interleaved=case["interleaved"], rope_scale=case["scale"],
                      out=s["out"])
    if op == "append":
        from directaccesskernel_b200.kv4 import kv_read_q4, rope_kv_append_q4

        rope_kv_append_q4(s["qkv"], s["positions"], s["inv_freq"], case["q_heads"], s["q_out"], s["pool"], None, s["table"],
                          seq_index=s["seq"], interleaved=case["interleaved"], rope_scale=case["scale"])
        k, v = kv_read_q4(s["pool"], None, s["table"], s["positions"], seq_index=s["seq"], dtype=s["qkv"].dtype)
        return s["q_out"], k, v
    if op == "read":
        from directaccesskernel_b200.kv4 import kv_read_q4

        return kv_read_q4(s["pool"], None, s["table"], s["positions"], seq_index=s["seq"], dtype=DTYPES[case["dtype"]])
    if op == "attend":
        from directaccesskernel_b200.kv4 import decode_paged_q4

        return decode_paged_q4(s["q"], s["pool"], s["host"], s["table"], s["lens"], 1 / math.sqrt(D),
                               max_seq_len=case["length"], merge_counters=s["counters"])
    from directaccesskernel_b200.kv_pages import copy_pages

    copy_pages(s["pool"], s["host"], s["src"], s["dst"], page_dim=1)
    return s["pool"] if s["host"] is None else (s["pool"], s["host"])


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "rotary":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return dict(bytes=4 * n * case["head_dim"] + 4 * case["tokens"], flops=3 * n * case["rotary_dim"])
    tok = _slab(case["page"], case["group"]) // case["page"]  # bytes of one token of one head, K and V
    if op == "append":  # qkv in, q and the cache rows out, the rows' values back
        T, hq, kv = case["tokens"], case["q_heads"], case["kv_heads"]
        return dict(bytes=T * (2 * D * (2 * hq + 2 * kv) + kv * tok + kv * tok + 4 * D * kv),
                    flops=T * (3 * (hq + kv) * case["rotary_dim"] + 12 * D * kv))
    if op == "read":
        n = case["tokens"] * case["kv_heads"]
        return dict(bytes=n * (tok + 4 * D), flops=4 * n * D)
    if op == "attend":
        kv, hq = case["kv_heads"], case["kv_heads"] * case["share"]
        n, S = case["seqs"], case["length"]
        # The mean of lengths that are even over their logarithm; one of them is the longest.
        total = n * S if not case["ragged"] or S < 2 else S + (n - 1) * (S - 1) / math.log(S)
        return dict(bytes=total * kv * tok + 4 * n * hq * D, flops=4 * total * hq * D)
    n = case["slabs"] * case["moves"] * case["kv_heads"] * _slab(case["page"], case["group"])
    return dict(bytes=2 * n, flops=0)


# ------------------------------------------------------------------- exact
def _turn64(x, pos, inv_freq, interleaved, scale):
    """The rotation as a product of complex numbers, in 64 bits."""
    x = x.double().clone()
    if inv_freq is None:
        return x
    h = inv_freq.numel()
    t = torch.outer(pos.double(), inv_freq.double())
    e = torch.polar(torch.full_like(t, scale), t)[:, None]
    i = torch.arange(h, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    z = torch.complex(x[..., a], x[..., b]) * e
    x[..., a], x[..., b] = z.real, z.imag
    return x


def _through64(x, group):
    """What the cache holds of x [..., 128]: float16 scale and zero, 16 steps."""
    out = torch.empty_like(x)
    for j in range(0, D, group):
        g = x[..., j:j + group]
        lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        zero, scale = lo.half().double(), ((hi - lo) / 15).half().double()
        n = torch.where(scale > 0, torch.round((g - zero) / scale).clamp(0, 15), torch.zeros_like(g))
        out[..., j:j + group] = zero + n * scale
    return out


def _held64(row, page, group, at):
    """Values [pages, heads, page, 128] in 64 bits of slabs [pages, heads, bytes], K (at = 0) or V (at = 1)."""
    n, heads, ng = row.shape[0], row.shape[1], D // group
    half = row[..., at * (row.shape[-1] // 2):(at + 1) * (row.shape[-1] // 2)]
    c = half[..., :64 * page].reshape(n, heads, page, 64).int()
    p = half[..., 64 * page:].contiguous().view(torch.float16).reshape(n, heads, page, ng, 2).double()
    out = torch.empty(n, heads, page, D, dtype=torch.float64, device=row.device)
    out[..., 0::2], out[..., 1::2] = (c % 16).double(), (c // 16).double()
    for j in range(ng):
        v = out[..., j * group:(j + 1) * group]
        v.mul_(p[..., j, 0:1]).add_(p[..., j, 1:2])
    return out


def exact(case, seed):
    op = case["op"]
    if op == "pages":
        return None
    s = prepare(case, seed)
    if op == "rotary":
        return _turn64(s["x"], s["positions"], s["inv_freq"], case["interleaved"], case["scale"])
    page, group = case["page"], case["group"]
    if op == "append":
        T, hq, kv = case["tokens"], case["q_heads"], case["kv_heads"]
        x = s["qkv"].reshape(T, hq + 2 * kv, D)
        q = _turn64(x[:, :hq], s["positions"], s["inv_freq"], case["interleaved"], case["scale"])
        k = _turn64(x[:, hq:hq + kv], s["positions"], s["inv_freq"], case["interleaved"], case["scale"])
        return q, _through64(k, group), _through64(x[:, hq + kv:].double(), group)
    if op == "read":
        seq = torch.arange(case["tokens"], device="cuda") if s["seq"] is None else s["seq"].long()
        v = s["table"][seq, s["positions"].long() // page].long()
        o = s["positions"].long() % page
        return tuple(_held64(s["pool"], page, group, at)[v, :, o] for at in (0, 1))
    B, kv, share = case["seqs"], case["kv_heads"], case["share"]
    out = torch.zeros(B, kv * share, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = int(s["lens"][b])
        ids = s["table"][b, :-(-n // page)].long()
        row = torch.empty(ids.numel(), *s["pool"].shape[1:], dtype=torch.uint8, device="cuda")
        row[ids >= 0] = s["pool"][ids[ids >= 0]]
        if s["host"] is not None:
            row[ids < 0] = s["host"][(-1 - ids[ids < 0]).cpu()].cuda()
        k, v = (_held64(row, page, group, at).permute(1, 0, 2, 3).reshape(kv, -1, D)[:, :n] for at in (0, 1))
        q = s["q"][b].double().view(kv, share, D)
        w = torch.softmax(torch.einsum("hsd,htd->hst", q, k) / math.sqrt(D), -1)
        out[b] = torch.einsum("hst,htd->hsd", w, v).reshape(-1, D)
    return out
