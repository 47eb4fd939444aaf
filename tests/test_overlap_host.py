"""Outputs that would overlap themselves or an input are refused before any launch.  No GPU."""
import ctypes
import random

import pytest

from directaccesskernel_b200 import _lib

BUF = 0x100000  # never dereferenced: calls that pass the checks of overlaps fail the one of pointers
OVERLAP = "overlap"


def _refusal(fn, *args):
    assert fn(*args) == _lib.DAK_ERR_INVALID_ARG
    return _lib.LIB.dak_last_error_message().decode()


def _starts(p, shape, strides):
    return [p + 2 * (i * strides[0] + j * strides[1]) for i in range(shape[0]) for j in range(shape[1])]


def _meet(a, b, n):
    """Whether blocks of n bytes at a and at b share a byte; b None: two blocks of a."""
    both = sorted([(x, 0) for x in a] + ([(x, 1) for x in b] if b is not None else []))
    if b is None:
        return any(y[0] - x[0] < n for x, y in zip(both, both[1:]))
    near = {0: None, 1: None}
    for x, of in both:
        other = near[1 - of]
        if other is not None and x - other < n:
            return True
        near[of] = x
    return False


def _rotary(tokens, heads, dim, x, xs, out, os):
    a = _lib.RotaryArgs(x, *xs, BUF, BUF, out, *os, tokens, heads, dim, 16, 0, 1.0, _lib.DTYPE_F16)
    return _refusal(_lib.LIB.dak_rotary, ctypes.byref(a), None)


@pytest.mark.parametrize("tokens,heads,xs,out,os,refused", [
    (4, 3, (384, 128), BUF, (384, 128), False),               # in place
    (4, 3, (640, 128), BUF, (640, 128), False),               # in place within a fused projection
    (4, 3, (384, 128), 1 << 30, (128, 128), True),            # token t + 1 over head 1 of token t
    (4, 3, (384, 128), 1 << 30, (256, 128), True),            # token t + 1 over head 2
    (4, 3, (384, 128), 1 << 30, (128, 512), False),           # head-major
    (5, 3, (384, 128), 1 << 30, (128, 512), True),            # its fifth token over the next head
    (4, 3, (0, 0), 1 << 30, (384, 128), False),               # one head for all
    (4, 3, (768, 128), BUF + 2 * 384, (768, 128), False),     # between the rows of x
    (4, 3, (768, 128), BUF + 2 * 256, (768, 128), True),      # over the last head of each
    (4, 3, (384, 128), BUF + 2 * 384, (384, 128), True),      # a token on
    (4, 3, (384, 128), BUF, (128, 512), True),                # x transposed over itself
    (1, 3, (0, 128), BUF + 2 * 128, (0, 128), True),
    (1, 3, (7 * 8, 128), BUF, (9 * 8, 128), False),           # one token: its stride does not count
    (4, 3, (384, 128), BUF + 2 * 384 * 4, (384, 128), False), # right behind x
    (4, 3, (-384, 128), BUF, (384, 128), True),
])
def test_rotary_outputs(tokens, heads, xs, out, os, refused):
    assert (OVERLAP in _rotary(tokens, heads, 128, BUF, xs, out, os)) == refused


def test_rotary_outputs_against_all_pairs():
    """Random small grids: refused exactly where two blocks of out, or one of out and one of x
    that is not the same call in place, share an element."""
    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        T, H, d = rng.randint(1, 5), rng.randint(1, 5), 16
        xs, os = ([8 * rng.randint(-12, 12) for _ in range(2)] for _ in range(2))
        if rng.random() < 0.4:
            os = list(xs)
        out = BUF + 16 * rng.randint(-40, 40)
        x_at, o_at = _starts(BUF, (T, H), xs), _starts(out, (T, H), os)
        same = out == BUF and (T == 1 or xs[0] == os[0]) and (H == 1 or xs[1] == os[1])
        want = _meet(o_at, None, 2 * d) or (not same and _meet(x_at, o_at, 2 * d))
        assert (OVERLAP in _rotary(T, H, d, BUF, xs, out, os)) == want, (T, H, xs, os, out - BUF)
        seen[want] += 1
    assert min(seen.values()) > 300


def _cache(**kw):
    c = _lib.Kv4Cache()
    for k, v in {**dict(pool_dev=1 << 40, dev_pages=4, block_table=1 << 41, table_stride=2, max_pages=2, batch=3, kv_heads=2,
                        page_size=16, group=32), **kw}.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("batch,heads,qs,out,os,refused", [
    (3, 4, (512, 128), BUF, (512, 128), False),               # over the query itself
    (3, 4, (512, 128), 1 << 30, (512, 128), False),
    (3, 4, (512, 128), 1 << 30, (128, 128), True),            # the next sequence over head 1
    (3, 4, (512, 128), 1 << 30, (384, 128), True),            # over the last head
    (3, 4, (512, 128), 1 << 30, (128, 384), False),           # head-major
    (3, 4, (512, 128), 1 << 30, (128, 256), True),
    (3, 4, (768, 128), BUF + 2 * 128, (768, 128), True),      # a head on
    (3, 4, (1024, 128), BUF + 2 * 512, (1024, 128), False),   # between the query's rows
    (3, 4, (512, 128), BUF, (128, 384), True),                # over the query in another order
    (1, 4, (0, 128), BUF, (9 * 8, 128), False),               # one sequence: its stride does not count
])
def test_attention_outputs(batch, heads, qs, out, os, refused):
    a = _lib.AttnQ4Args(BUF, *qs, BUF, out, *os, None, 0, None, heads, 32, 0.1, _lib.DTYPE_F16)
    assert (OVERLAP in _refusal(_lib.LIB.dak_attn_decode_paged_q4, ctypes.byref(_cache(batch=batch)), ctypes.byref(a), None)) == refused


@pytest.mark.parametrize("tokens,ld,q_out,refused", [
    (3, 1024, BUF, True),
    (3, 1024, BUF - 2 * 3 * 512, False),       # right before qkv
    (3, 1024, BUF - 2 * 3 * 512 + 16, True),
    (3, 1024, BUF + 2 * 3 * 1024, False),      # right behind it
    (3, 1024, BUF + 2 * 3 * 1024 - 16, True),
    (3, 4096, BUF + 2 * 1024, False),          # between its rows
    (3, 2048, BUF + 2 * 1024, True),           # where they leave less room
    (1, 4096, BUF + 2 * 512, True),
    (0, 1024, BUF, False),
])
def test_append_outputs(tokens, ld, q_out, refused):
    a = _lib.Kv4AppendArgs()
    for k, v in dict(qkv=BUF, ld=ld, positions=BUF, seq_index=BUF, inv_freq=BUF, rope_scale=1.0, q_out=q_out, tokens=tokens,
                     q_heads=4, rotary_dim=128, dtype=_lib.DTYPE_BF16).items():
        setattr(a, k, v)
    assert (OVERLAP in _refusal(_lib.LIB.dak_rope_kv_append_q4, ctypes.byref(_cache()), ctypes.byref(a), None)) == refused


@pytest.mark.parametrize("behind,refused", [(0, True), (16, True), (2 * 3 * 2 * 128 - 16, True), (2 * 3 * 2 * 128, False),
                                            (16 - 2 * 3 * 2 * 128, True), (-2 * 3 * 2 * 128, False)])
def test_read_outputs(behind, refused):
    text = _refusal(_lib.LIB.dak_kv_read_q4, ctypes.byref(_cache()), BUF, BUF, BUF, BUF + behind, 3, _lib.DTYPE_F16, None)
    assert (OVERLAP in text) == refused
