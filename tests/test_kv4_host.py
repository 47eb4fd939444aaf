"""Host side of the 4-bit KV cache, the rotary frequencies and the page table:
formats, refusals before any launch, bookkeeping.  No GPU."""
import ctypes

import pytest
import torch

from directaccesskernel_b200 import _lib, kv4
from directaccesskernel_b200.decode_ops import rope_frequencies, rotary
from directaccesskernel_b200.kv_pages import MAX_MOVES, PageTable, copy_pages

BUF = 0x10000  # never dereferenced: every call below fails its checks first


def _status(fn, *args):
    st = fn(*args)
    return st, _lib.LIB.dak_last_error_message().decode()


def _cache(**kw):
    c = _lib.Kv4Cache()
    for k, v in dict(pool_dev=BUF, dev_pages=4, block_table=BUF, table_stride=2, max_pages=2, batch=3, kv_heads=2,
                     page_size=16, group=32, **kw).items():
        setattr(c, k, v)
    return c


def test_page_bytes_name_one_format_each():
    seen = {}
    for p in kv4.PAGE_SIZES:
        for g in kv4.GROUPS:
            n = kv4.page_bytes(p, g)
            assert n == 2 * p * (64 + 4 * 128 // g) and n % 16 == 0
            assert n not in seen
            seen[n] = (p, g)
            assert kv4.page_format(torch.empty(0, 1, n, dtype=torch.uint8)) == (p, g)
    with pytest.raises(RuntimeError, match="no page_bytes"):
        kv4.page_format(torch.empty(1, 1, 2177, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="page_size"):
        kv4.page_bytes(48, 32)
    assert kv4.merge_counter_count(3, 40, 4) == 3 * 4 * 2


@pytest.mark.parametrize("bad,status,msg", [
    (dict(page_size=48), _lib.DAK_ERR_UNSUPPORTED, "page_size"),
    (dict(group=16), _lib.DAK_ERR_UNSUPPORTED, "group"),
    (dict(batch=0), _lib.DAK_ERR_INVALID_ARG, "positive"),
    (dict(kv_heads=0), _lib.DAK_ERR_INVALID_ARG, "positive"),
    (dict(table_stride=1), _lib.DAK_ERR_INVALID_ARG, "table_stride"),
    (dict(block_table=None), _lib.DAK_ERR_INVALID_ARG, "block_table"),
    (dict(dev_pages=0), _lib.DAK_ERR_INVALID_ARG, "tier"),
    (dict(host_pages=3), _lib.DAK_ERR_INVALID_ARG, "tier"),
    (dict(pool_dev=None, dev_pages=0), _lib.DAK_ERR_INVALID_ARG, "no KV pool"),
    (dict(pool_dev=BUF + 8), _lib.DAK_ERR_ALIGNMENT, "aligned"),
])
def test_cache_refusals(bad, status, msg):
    c = _cache(**{k: v for k, v in bad.items() if k == "host_pages"})
    for k, v in bad.items():
        setattr(c, k, v)
    a = _lib.AttnQ4Args()
    for fn, args in ((_lib.LIB.dak_attn_decode_paged_q4, (ctypes.byref(c), ctypes.byref(a), None)),
                     (_lib.LIB.dak_rope_kv_append_q4, (ctypes.byref(c), ctypes.byref(_lib.Kv4AppendArgs()), None)),
                     (_lib.LIB.dak_kv_read_q4, (ctypes.byref(c), BUF, BUF, BUF, BUF, 4, _lib.DTYPE_F16, None))):
        st, text = _status(fn, *args)
        assert st == status and msg in text, text


@pytest.mark.parametrize("bad,status,msg", [
    (dict(dtype=_lib.DTYPE_F32), _lib.DAK_ERR_UNSUPPORTED, "float16"),
    (dict(num_q_heads=5), _lib.DAK_ERR_INVALID_ARG, "multiple of kv_heads"),
    (dict(num_q_heads=0), _lib.DAK_ERR_INVALID_ARG, "multiple of kv_heads"),
    (dict(max_seq_len=33), _lib.DAK_ERR_INVALID_ARG, "max_seq_len"),
    (dict(max_seq_len=0), _lib.DAK_ERR_INVALID_ARG, "max_seq_len"),
    (dict(query=None), _lib.DAK_ERR_INVALID_ARG, "query"),
    (dict(q_stride_h=100), _lib.DAK_ERR_ALIGNMENT, "strides"),
    (dict(o_stride_b=513), _lib.DAK_ERR_ALIGNMENT, "strides"),
    (dict(out=BUF + 2), _lib.DAK_ERR_ALIGNMENT, "aligned"),
    (dict(o_stride_b=0), _lib.DAK_ERR_INVALID_ARG, "overlap"),
    (dict(o_stride_h=64), _lib.DAK_ERR_INVALID_ARG, "overlap"),
])
def test_attention_refusals(bad, status, msg):
    a = _lib.AttnQ4Args()
    for k, v in {**dict(query=BUF, q_stride_b=512, q_stride_h=128, seq_lens=BUF, out=BUF, o_stride_b=512, o_stride_h=128,
                        num_q_heads=4, max_seq_len=32, scaling=0.1, dtype=_lib.DTYPE_F16), **bad}.items():
        setattr(a, k, v)
    st, text = _status(_lib.LIB.dak_attn_decode_paged_q4, ctypes.byref(_cache()), ctypes.byref(a), None)
    assert st == status and msg in text, text


def test_attention_refuses_lengths_near_2_to_31():
    c = _cache()
    c.max_pages = c.table_stride = 2**27
    a = _lib.AttnQ4Args(BUF, 512, 128, BUF, BUF, 512, 128, BUF, 1 << 40, None, 4, 2**31 - 1, 0.1, _lib.DTYPE_F16)
    st, text = _status(_lib.LIB.dak_attn_decode_paged_q4, ctypes.byref(c), ctypes.byref(a), None)
    assert st == _lib.DAK_ERR_UNSUPPORTED and "max_seq_len" in text, text


def test_attention_scratch():
    """None for short rows that fit the GPU at once, else two slots of 8 heads for
    every CTA; a call with less is refused."""
    c = _cache()
    assert _lib.LIB.dak_attn_q4_scratch(ctypes.byref(c), 4, 32) == 0 == kv4.scratch_floats(3, 4, 2, 16, 32, 32)
    assert _lib.LIB.dak_attn_q4_scratch(ctypes.byref(c), 5, 32) < 0
    assert kv4.scratch_floats(1, 8, 1, 64, 128, 513) == 2 * 3 * 8 * 130  # 9 chunks: 3 CTAs of 4 warps
    sms = _lib.constants().num_sms
    assert kv4.scratch_floats(64, 64, 8, 64, 128, 16384) == 2 * 2 * sms * 8 * 130  # two CTAs per SM
    c.max_pages = c.table_stride = 64
    a = _lib.AttnQ4Args()
    for k, v in dict(query=BUF, q_stride_b=512, q_stride_h=128, seq_lens=BUF, out=BUF, o_stride_b=512, o_stride_h=128,
                     num_q_heads=4, max_seq_len=1000, scaling=0.1, dtype=_lib.DTYPE_F16, scratch=BUF, scratch_floats=100).items():
        setattr(a, k, v)
    st, text = _status(_lib.LIB.dak_attn_decode_paged_q4, ctypes.byref(c), ctypes.byref(a), None)
    assert st == _lib.DAK_ERR_INVALID_ARG and "scratch" in text


@pytest.mark.parametrize("bad,status,msg", [
    (dict(dtype=99), _lib.DAK_ERR_UNSUPPORTED, "float16"),
    (dict(tokens=-1), _lib.DAK_ERR_INVALID_ARG, "negative"),
    (dict(tokens=4, seq_index=None), _lib.DAK_ERR_INVALID_ARG, "one token per sequence"),
    (dict(positions=None), _lib.DAK_ERR_INVALID_ARG, "positions"),
    (dict(q_out=None), _lib.DAK_ERR_INVALID_ARG, "q_out"),
    (dict(ld=1016), _lib.DAK_ERR_INVALID_ARG, "row stride"),
    (dict(ld=1028), _lib.DAK_ERR_ALIGNMENT, "multiple of 8"),
    (dict(rotary_dim=130), _lib.DAK_ERR_INVALID_ARG, "rotary_dim"),
    (dict(rotary_dim=24), _lib.DAK_ERR_UNSUPPORTED, "multiple of 16"),
    (dict(rotary_dim=7, interleaved=1), _lib.DAK_ERR_INVALID_ARG, "even"),
    (dict(inv_freq=None), _lib.DAK_ERR_INVALID_ARG, "inv_freq"),
])
def test_append_refusals(bad, status, msg):
    a = _lib.Kv4AppendArgs()
    for k, v in {**dict(qkv=BUF, ld=1024, positions=BUF, seq_index=BUF, inv_freq=BUF, rope_scale=1.0, q_out=BUF, tokens=3,
                        q_heads=4, rotary_dim=128, dtype=_lib.DTYPE_BF16), **bad}.items():
        setattr(a, k, v)
    st, text = _status(_lib.LIB.dak_rope_kv_append_q4, ctypes.byref(_cache()), ctypes.byref(a), None)
    assert st == status and msg in text, text


def test_read_refuses_one_output_for_both():
    st, text = _status(_lib.LIB.dak_kv_read_q4, ctypes.byref(_cache()), BUF, BUF, BUF, BUF, 4, _lib.DTYPE_F16, None)
    assert st == _lib.DAK_ERR_INVALID_ARG and "overlap" in text, text


@pytest.mark.parametrize("src", [[0.5], [[0, 1]], [1 << 31], ["0"], torch.tensor([0.0]), torch.tensor([[0]]),
                                 torch.tensor([1 << 31])])
def test_page_lists_are_whole_numbers(src):
    from directaccesskernel_b200.kv_pages import _entries

    with pytest.raises(RuntimeError):
        _entries(src, "src")
    assert _entries([], "src").numel() == 0 and _entries((1, -2), "src").tolist() == [1, -2]


def test_rotary_refusals():
    def call(tokens=2, heads=2, d=128, r=128, inter=0, st=(256, 128, 256, 128), x=BUF, out=BUF, dtype=_lib.DTYPE_F16):
        a = _lib.RotaryArgs(x, st[0], st[1], BUF, BUF, out, st[2], st[3], tokens, heads, d, r, inter, 1.0, dtype)
        return _status(_lib.LIB.dak_rotary, ctypes.byref(a), None)

    assert call(dtype=_lib.DTYPE_F32)[0] == _lib.DAK_ERR_UNSUPPORTED
    for kw, status, msg in ((dict(heads=0), _lib.DAK_ERR_INVALID_ARG, "positive"),
                            (dict(d=1032), _lib.DAK_ERR_INVALID_ARG, "1024"),
                            (dict(d=100, r=32), _lib.DAK_ERR_ALIGNMENT, "multiple of 8"),
                            (dict(r=136), _lib.DAK_ERR_INVALID_ARG, "head_dim"),
                            (dict(r=40), _lib.DAK_ERR_UNSUPPORTED, "16"),
                            (dict(st=(252, 128, 256, 128)), _lib.DAK_ERR_ALIGNMENT, "strides"),
                            (dict(out=BUF + 4), _lib.DAK_ERR_ALIGNMENT, "aligned"),
                            (dict(st=(256, 128, 0, 128)), _lib.DAK_ERR_INVALID_ARG, "overlap"),
                            (dict(st=(256, 128, 256, 0)), _lib.DAK_ERR_INVALID_ARG, "overlap"),
                            (dict(x=None), _lib.DAK_ERR_INVALID_ARG, "required")):
        st, text = call(**kw)
        assert st == status and msg in text, (kw, text)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary(torch.zeros(2, 2, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32), torch.zeros(64))


@pytest.mark.parametrize("n", [2, 9, 120, 1000, MAX_MOVES])
@pytest.mark.parametrize("stride", [1, 16, 4096])
def test_copy_finds_hazards_in_long_lists(n, stride):
    g = torch.Generator().manual_seed(n)
    ids = (torch.randperm(2 * n, generator=g) * stride).to(torch.int32)
    ids[::3] = -1 - ids[::3]  # some on the host

    def message(src, dst):
        return _status(_lib.LIB.dak_copy_pages, BUF, 2 * n * stride, BUF, 2 * n * stride, 64, 1, 0, 0, src.data_ptr(),
                       dst.data_ptr(), n, None)[1]

    src, dst = ids[:n].clone(), ids[n:].clone()
    assert not any(w in message(src, dst) for w in ("twice", "both", "outside"))
    assert not any(w in message(src[:1].repeat(n), dst) for w in ("twice", "both", "outside"))  # one page to many
    for i, j in ((0, n - 1), (n // 2, 0)):
        two = dst.clone()
        two[i] = two[j]
        assert f"page {int(dst[j])} is a destination twice" in message(src, two)
        two = src.clone()
        two[i] = dst[j]
        assert f"page {int(dst[j])} is both" in message(two, dst)


def test_copy_refusals():
    def call(src, dst, dev=4, host=4, page=64, slabs=1, strides=(256, 256), pool=BUF, n=None):
        s, d = torch.tensor(src, dtype=torch.int32), torch.tensor(dst, dtype=torch.int32)
        return _status(_lib.LIB.dak_copy_pages, pool if dev else None, dev, BUF if host else None, host, page, slabs,
                       *strides, s.data_ptr(), d.data_ptr(), len(src) if n is None else n, None)

    for args, kw, status, msg in (
            (([0], [4]), {}, _lib.DAK_ERR_INVALID_ARG, "outside"),
            (([-5], [0]), {}, _lib.DAK_ERR_INVALID_ARG, "outside"),
            (([0], [-1]), dict(host=0), _lib.DAK_ERR_INVALID_ARG, "outside"),
            (([0, 1], [2, 2]), {}, _lib.DAK_ERR_INVALID_ARG, "destination twice"),
            (([0, 1], [1, 2]), {}, _lib.DAK_ERR_INVALID_ARG, "source and a destination"),
            (([3], [3]), {}, _lib.DAK_ERR_INVALID_ARG, "source and a destination"),
            (([0], [1]), dict(page=24), _lib.DAK_ERR_ALIGNMENT, "16 bytes"),
            (([0], [1]), dict(slabs=2, strides=(128, 256)), _lib.DAK_ERR_INVALID_ARG, "slab stride"),
            (([0], [1]), dict(slabs=0), _lib.DAK_ERR_INVALID_ARG, "positive"),
            (([0], [1]), dict(n=MAX_MOVES + 1), _lib.DAK_ERR_INVALID_ARG, "per call")):
        st, text = call(*args, **kw)
        assert st == status and msg in text, (args, kw, text)
    with pytest.raises(RuntimeError, match="no KV pool"):
        copy_pages(None, None, [0], [1])
    with pytest.raises(RuntimeError, match="CUDA device"):
        copy_pages(torch.zeros(2, 16, dtype=torch.uint8), None, [0], [1])


@pytest.mark.parametrize("call", ["append", "read", "attend"])
def test_python_entry_points_refuse_cpu_tensors(call):
    pool = torch.zeros(2, 1, kv4.page_bytes(16, 32), dtype=torch.uint8)
    table = torch.zeros(1, 2, dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="current CUDA device"):
        if call == "append":
            kv4.rope_kv_append_q4(torch.zeros(1, 384, dtype=torch.float16), one, None, 1,
                                  torch.zeros(1, 1, 128, dtype=torch.float16), pool, None, table)
        elif call == "read":
            kv4.kv_read_q4(pool, None, table, one)
        else:
            kv4.decode_paged_q4(torch.zeros(1, 1, 128, dtype=torch.float16), pool, None, table, one, 1.0)


# ------------------------------------------------------------- frequencies
@pytest.mark.parametrize("scaling", [
    dict(rope_type="default"), dict(rope_type="linear", factor=4.0),
    dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192),
    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096),
    dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=2048, beta_fast=16, beta_slow=2, attention_factor=1.25),
    dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=4096, mscale=1.0, mscale_all_dim=0.707),
])
def test_rope_frequencies_match_transformers(scaling):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    theta, d = 500000.0, 128
    cfg = LlamaConfig(hidden_size=1024, num_attention_heads=8, head_dim=d, max_position_embeddings=131072,
                      rope_parameters=dict(scaling, rope_theta=theta))
    inv, attention = rope_frequencies(d, theta, scaling, device="cpu")
    kind = scaling["rope_type"]
    if kind == "default":
        ref, ref_attention = 1.0 / theta ** (torch.arange(0, d, 2).double() / d), 1.0
    else:
        ref, ref_attention = ROPE_INIT_FUNCTIONS[kind](cfg, torch.device("cpu"))
    # transformers works in FP32: theta ** x is off by about |ln| 2^-24, a few steps.
    torch.testing.assert_close(inv.double(), ref.double(), rtol=32 * 2.0**-24, atol=0)
    assert abs(attention - ref_attention) < 1e-6


def test_rope_frequencies_refusals():
    with pytest.raises(RuntimeError, match="not supported"):
        rope_frequencies(128, 1e4, dict(rope_type="longrope"), device="cpu")
    with pytest.raises(RuntimeError, match="max_position"):
        rope_frequencies(128, 1e4, dict(rope_type="yarn", factor=2.0), device="cpu")
    with pytest.raises(RuntimeError, match="even"):
        rope_frequencies(7, device="cpu")


# -------------------------------------------------------------- page table
def _check(t: PageTable):
    """Every page is free or held, never both, and reference counts are the rows'."""
    held = {}
    for row in t._rows.values():
        for v in row:
            held[v] = held.get(v, 0) + 1
    assert held == t._refs
    free = t._free_dev + t._free_host
    assert len(set(free)) == len(free) and not set(free) & set(held)
    assert set(free) | set(held) == set(range(t.dev_pages)) | set(range(-t.host_pages, 0))


def test_page_table_grow_fork_free():
    t = PageTable(6, 3, 16)
    assert t.grow("a", 33) == [0, 1, 2] and t.grow("a", 48) == [] and t.grow("b", 1, host=True) == [-1]
    src, dst = t.fork("a", "c", 40)  # two full pages shared, the third copied
    assert (src, dst) == ([2], [3]) and t.pages("c") == [0, 1, 3]
    assert t.fork("a", "d", 32) == ([], []) and t.pages("d") == [0, 1]
    assert t.fork("b", "e", 1) == ([-1], [-2])
    assert t.fork("a", "empty", 0) == ([], []) and t.pages("empty") == []
    _check(t)
    t.free("a")
    assert t.pages("d") == [0, 1] and t.free_pages() == (3, 1)
    _check(t)
    table = t.block_table(["c", "e", "empty"], 4)
    assert table.tolist() == [[0, 1, 3, 0], [-2, 0, 0, 0], [0, 0, 0, 0]] and table.dtype == torch.int32
    with pytest.raises(RuntimeError, match="at least 3"):
        t.block_table(["c"], 2)
    for s in ("c", "d", "e", "b", "empty"):
        t.free(s)
    assert t.free_pages() == (6, 3)
    _check(t)


def test_page_table_out_of_pages_changes_nothing():
    t = PageTable(2, 0, 16)
    t.grow("a", 20)
    for call in (lambda: t.grow("b", 1), lambda: t.grow("a", 33), lambda: t.fork("a", "b", 20), lambda: t.move("a", 0, 1, True)):
        with pytest.raises(RuntimeError, match="out of"):
            call()
        _check(t)
        assert t.pages("a") == [0, 1] and "b" not in t._rows
    with pytest.raises(RuntimeError, match="fewer"):
        t.fork("a", "b", 33)
    with pytest.raises(RuntimeError, match="exists"):
        t.fork("a", "a", 16)


def test_page_table_move_and_compact_keep_the_contents():
    """Random operations; a dictionary of page contents stands in for the pools."""
    import random

    rng = random.Random(3)
    t = PageTable(24, 12, 8)
    data, want, names = {}, {}, iter(range(10**6))

    def copy(src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for a, b in [(data[s], d) for s, d in zip(src, dst)]:
            data[b] = a

    for _ in range(600):
        op = rng.choice(["new", "grow", "fork", "free", "move", "compact"])
        seqs = list(want)
        try:
            if op == "new" or not seqs:
                s = next(names)
                new = t.grow(s, rng.randrange(1, 40), host=rng.random() < 0.3)
                want[s] = []
            elif op == "grow":
                s = rng.choice(seqs)
                new = t.grow(s, 8 * len(want[s]) + rng.randrange(1, 20), host=rng.random() < 0.3)
            else:
                new = None
            if new is not None:
                for v in new:
                    data[v] = next(names)
                    want[s].append(data[v])
                continue
            s = rng.choice(seqs)
            if op == "fork" and want[s]:
                tokens = rng.randrange(0, 8 * len(want[s]) + 1)
                n = next(names)
                copy(*t.fork(s, n, tokens))
                want[n] = want[s][:-(-tokens // 8)]
            elif op == "free":
                t.free(s)
                del want[s]
            elif op == "move" and want[s]:
                i = rng.randrange(len(want[s]))
                copy(*t.move(s, i, rng.randrange(len(want[s]) - i + 1), rng.random() < 0.5))
            elif op == "compact":
                copy(*t.compact())
                live = [v for v in t._refs if v >= 0]
                assert sorted(live) == list(range(len(live)))
        except RuntimeError as e:
            assert "out of" in str(e)
        _check(t)
        for s, rows in want.items():
            assert [data[v] for v in t.pages(s)] == rows


# ------------------------------------------------------------ decoder's sizes
def test_decoder_shapes_with_scaled_rotary_and_4_bit_pages():
    from directaccesskernel_b200 import decode
    from directaccesskernel_b200.llama_tp import LlamaShape, budget_fraction

    cfg = decode.llama_config("llama-3-70b")
    s = LlamaShape.from_config(cfg)
    assert s.rope_scaling is None
    # 136, 144 or 160 bytes per token, head and layer instead of 512.
    full = s.kv_bytes_per_rank(8, 32, 16384)
    for group, per in ((128, 136), (64, 144), (32, 160)):
        assert s.kv_bytes_per_rank(8, 32, 16384, kv_bits=4, kv_group=group) * 512 == full * per
    assert budget_fraction(s, 4, 32, 16384, 60 * 10**9) > 0.2
    assert budget_fraction(s, 4, 32, 16384, 60 * 10**9, kv_bits=4) == 0.0
    cfg.rope_parameters = dict(rope_type="yarn", factor=4.0, rope_theta=1e4, original_max_position_embeddings=4096)
    assert LlamaShape.from_config(cfg).rope_scaling["factor"] == 4.0
    cfg.rope_parameters = dict(rope_type="longrope", factor=4.0, rope_theta=1e4)
    with pytest.raises(ValueError, match="not supported"):
        LlamaShape.from_config(cfg)
