"""Copying cache pages within and between the tiers."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pools(lead, dev, host, rest, dtype=torch.uint8, seed=0):
    g = torch.Generator().manual_seed(seed)

    def one(n):
        t = torch.randint(0, 256, (*lead, n, *rest), generator=g, dtype=torch.int32)
        return t.to(dtype)

    return one(dev).cuda() if dev else None, one(host).pin_memory() if host else None


def _expect(dev, host, src, dst, dim):
    d, h = (None if t is None else t.cpu().clone().movedim(dim, 0) for t in (dev, host))
    rows = [(d[s] if s >= 0 else h[-1 - s]).clone() for s in src]
    for v, r in zip(dst, rows):
        (d if v >= 0 else h)[v if v >= 0 else -1 - v] = r
    return tuple(None if t is None else t.movedim(0, dim) for t in (d, h))


@pytest.mark.parametrize("lead,dev,host,rest,dtype,src,dst", [
    ((), 4, 0, (16,), torch.uint8, [1], [3]),
    ((3,), 6, 5, (2, 2176), torch.uint8, [0, -1, -5, 4], [-2, 5, -3, 1]),
    ((2, 2), 5, 3, (2, 16, 128), torch.float16, [-1, 2, 2, 0], [1, 3, -2, -3]),
    ((7,), 9, 0, (3, 8704), torch.uint8, [8, 8, 8, 0], [1, 2, 3, 4]),
    ((), 3, 3, (8, 10240), torch.uint8, [2, -3], [-1, 0]),
    ((2,), 2, 2, (1040,), torch.bfloat16, [0, -2], [-1, 1]),
    ((5,), 3, 2, (4,), torch.float32, [], []),
])
def test_copy_pages(lead, dev, host, rest, dtype, src, dst):
    from directaccesskernel_b200.kv_pages import copy_pages

    d, h = _pools(lead, dev, host, rest, dtype)
    want = _expect(d, h, src, dst, len(lead))
    copy_pages(d, h, src, dst, page_dim=len(lead))
    torch.cuda.synchronize()
    for got, ref in zip((d, h), want):
        assert got is None or torch.equal(got.cpu(), ref)


@pytest.mark.parametrize("n", [119, 120, 121, 3584, 3585, 8000])
def test_copy_many_pages(n):
    """Both parameter sizes and several launches; the list may change after the call."""
    from directaccesskernel_b200.kv_pages import copy_pages

    d, _ = _pools((2,), 2 * n, 0, (48,), seed=n)
    g = torch.Generator().manual_seed(n)
    ids = torch.randperm(2 * n, generator=g)
    src, dst = ids[:n].clone(), ids[n:].to(torch.int32)
    want = d.clone()
    want[:, ids[n:].cuda()] = d[:, ids[:n].cuda()]
    copy_pages(d, None, src, dst, page_dim=1)
    dst.zero_()
    assert torch.equal(d, want)


def test_copy_in_a_graph_and_on_another_stream():
    from directaccesskernel_b200.kv_pages import copy_pages

    d, h = _pools((4,), 6, 2, (2304,), seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        copy_pages(d, h, [0, -1], [3, 4], page_dim=1)
    d[:, 0] = 7
    h[:, 0] = 9
    graph.replay()
    torch.cuda.synchronize()
    assert (d[:, 3] == 7).all() and (d[:, 4] == 9).all()


def test_refusals_come_before_any_copy():
    from directaccesskernel_b200.kv_pages import copy_pages

    d, h = _pools((2,), 4, 2, (32,), seed=6)
    before = d.clone()
    for src, dst, msg in (([0], [4], "outside"), ([0, 1], [2, 2], "twice"), ([0, 1], [1, 2], "both"), ([-3], [0], "outside"),
                          ([0], [1, 2], "same length"), (torch.tensor([0.0]), [1], "CPU tensor"),
                          (torch.tensor([0], device="cuda"), [1], "CPU tensor"), (torch.tensor([2**40]), [1], "int32"),
                          (list(range(4000)), [5000] * 4000, "twice"), (list(range(4000)), list(range(4000)), "both"),
                          ([0] * 4000, list(range(1, 4001)), "outside")):
        with pytest.raises(RuntimeError, match=msg):
            copy_pages(d, h, src, dst, page_dim=1)
    for kw, msg in ((dict(pool_host=torch.zeros(2, 2, 32, dtype=torch.uint8)), "pinned"), (dict(page_dim=3), "page_dim"),
                    (dict(pool_dev=d[..., :16]), "contiguous"), (dict(pool_dev=d[:1]), "differ"),
                    (dict(pool_dev=d.float()), "differ")):
        with pytest.raises(RuntimeError, match=msg):
            copy_pages(**{**dict(pool_dev=d, pool_host=h, src=[0], dst=[1], page_dim=1), **kw})
    assert torch.equal(d, before)


def test_forked_sequences_part_ways():
    """PageTable and copy_pages around the 16-bit cache: a fork shares full pages,
    copies the open one, moves to the host and is compacted; attention over both
    sequences stays that of their own tokens."""
    import math

    import oracle
    from conftest import rel_err
    from directaccesskernel_b200.attention import decode_paged, kv_append_paged
    from directaccesskernel_b200.kv_pages import PageTable, copy_pages

    P, Hq, Hkv, d = 16, 4, 2, 128
    g = torch.Generator().manual_seed(8)
    kd, vd = (torch.zeros(12, Hkv, P, d, dtype=torch.float16, device="cuda") for _ in range(2))
    kh, vh = (torch.zeros(6, Hkv, P, d, dtype=torch.float16).pin_memory() for _ in range(2))
    t = PageTable(12, 6, P)
    toks = {"a": [], "b": []}

    def moves(m):
        for dev, host in ((kd, kh), (vd, vh)):
            copy_pages(dev, host, *m)

    def append(seq):
        t.grow(seq, len(toks[seq]) + 1)
        k, v = (torch.randn(1, Hkv, d, generator=g).half() for _ in range(2))
        kv_append_paged(k.cuda(), v.cuda(), kd, vd, kh, vh, t.block_table([seq], 8).cuda(),
                        torch.tensor([len(toks[seq])], dtype=torch.int32, device="cuda"))
        toks[seq].append((k[0], v[0]))

    t.grow("hole", 40)
    for _ in range(37):
        append("a")
    moves(t.fork("a", "b", 37))
    toks["b"] = list(toks["a"])
    for i in range(15):
        append("a")
        if i % 2:
            append("b")
    moves(t.move("a", 0, 2, True))
    t.free("hole")
    moves(t.compact())
    for _ in range(3):
        append("b")
    q = torch.randn(2, Hq, d, generator=g).half()
    lens = [len(toks["a"]), len(toks["b"])]
    out = decode_paged(q.cuda(), kd, vd, kh, vh, t.block_table(["a", "b"], 8).cuda(),
                       torch.tensor(lens, dtype=torch.int32, device="cuda"), 1 / math.sqrt(d), 64)
    for i, s in enumerate("ab"):
        k, v = (torch.stack([x[j] for x in toks[s]], 1)[None].numpy() for j in (0, 1))
        ref = oracle.decode_attention(q[i:i + 1, :, None].numpy(), k, v, None, 1 / math.sqrt(d))[:, 0]
        assert rel_err(out[i:i + 1].float().cpu().numpy(), ref) < 2e-3
