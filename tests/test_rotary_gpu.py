"""Rotary positions on the GPU against the rotation in 64 bits."""
import pytest
import torch

from kv4_common import rotate64, rotation_bound, rounding

pytestmark = pytest.mark.gpu


def _case(T, H, d, r, seed, dtype, far=5000):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, d, generator=g).to(dtype)
    pos = torch.randint(-5, far, (T,), generator=g, dtype=torch.int32)
    inv = 1.0 / 500000 ** (torch.arange(0, r, 2).float() / r)
    return x, pos, inv


def _check(got, x, pos, inv, inter, scale):
    ref = rotate64(x, pos, inv, inter, scale)
    r = 2 * inv.numel()
    assert torch.equal(got.cpu()[..., r:], x[..., r:])
    assert ((got.cpu().double() - ref).abs()
            <= rounding(ref, x.dtype) + rotation_bound(x, inv, inter, scale) * 1.01).all()


@pytest.mark.parametrize("T,H,d,r,inter", [
    (1, 1, 128, 128, False), (1, 1, 8, 2, True), (7, 3, 64, 32, False), (33, 5, 96, 96, False), (64, 2, 256, 64, True),
    (5, 40, 128, 126, True), (3, 2, 80, 16, False), (1000, 9, 128, 128, False), (9, 1, 1024, 1024, False),
    (2, 130, 128, 64, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 1.1386])
def test_rotary(T, H, d, r, inter, dtype, scale):
    from directaccesskernel_b200.decode_ops import rotary

    x, pos, inv = _case(T, H, d, r, T + d, dtype)
    got = rotary(x.cuda(), pos.cuda(), inv.cuda(), interleaved=inter, rope_scale=scale)
    _check(got, x, pos, inv, inter, scale)


@pytest.mark.parametrize("inter", [False, True])
def test_rotary_at_far_positions(inter):
    from directaccesskernel_b200.decode_ops import rotary

    x, _, inv = _case(6, 2, 128, 128, 1, torch.float16)
    pos = torch.tensor([131071, 10**6 + 1, 2**31 - 1, -2**31, 0, 16777217], dtype=torch.int32)
    _check(rotary(x.cuda(), pos.cuda(), inv.cuda(), interleaved=inter), x, pos, inv, inter, 1.0)


def test_rotary_of_a_fused_projection_in_place():
    """q and k heads of a padded [tokens, (Hq + 2 Hkv) d] buffer rotated where they
    lie; v and the padding stay as they were."""
    from directaccesskernel_b200.decode_ops import rotary

    T, Hq, Hkv, d = 19, 6, 2, 128
    g = torch.Generator().manual_seed(3)
    buf = torch.randn(T, (Hq + 2 * Hkv) * d + 16, generator=g).half()
    _, pos, inv = _case(T, 1, d, 64, 4, torch.float16)
    dev = buf.cuda()
    view = dev[:, :(Hq + 2 * Hkv) * d].view(T, -1, d)[:, :Hq + Hkv]
    assert rotary(view, pos.cuda(), inv.cuda(), out=view) is view
    x = buf[:, :(Hq + Hkv) * d].reshape(T, -1, d)
    _check(view, x, pos, inv, False, 1.0)
    assert torch.equal(dev.cpu()[:, (Hq + Hkv) * d:], buf[:, (Hq + Hkv) * d:])


def test_rotary_head_major_strides_and_passing_infinities():
    from directaccesskernel_b200.decode_ops import rotary

    x, pos, inv = _case(12, 4, 64, 20, 5, torch.bfloat16)
    x[3, 1, 21:30] = float("inf")
    x[4, 0, 63] = float("nan")
    hm = x.transpose(0, 1).contiguous().cuda().transpose(0, 1)  # [tokens, heads, d] over a head-major buffer
    out = torch.empty(4, 12, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    got = rotary(hm, pos.cuda(), inv.cuda(), interleaved=True, out=out).cpu()
    assert torch.equal(got[..., 20:].view(torch.int16), x[..., 20:].view(torch.int16))
    ref = rotate64(x, pos, inv, True, 1.0)[..., :20]
    assert ((got[..., :20].double() - ref).abs()
            <= rounding(ref, torch.bfloat16) + rotation_bound(x, inv, True, 1.0)[..., :20] * 1.01).all()


def test_rotary_keeps_lengths_and_inverts():
    """A rotation by t and then by -t gives the input back, two roundings away."""
    from directaccesskernel_b200.decode_ops import rotary

    x, pos, inv = _case(50, 3, 128, 128, 6, torch.float16)
    once = rotary(x.cuda(), pos.cuda(), inv.cuda())
    back = rotary(once, (-pos).cuda(), inv.cuda()).cpu().double()
    half = x.double()[..., :64].abs() + x.double()[..., 64:].abs()
    # The first rounding (2^-11 of at most |x1| + |x2| in either partner) comes back through the second rotation.
    tol = 2 * 2.0**-11 * torch.cat([half, half], -1) + rounding(x.double(), torch.float16) + 1e-6 + 2.0**-24
    assert ((back - x.double()).abs() <= tol).all()


def test_rotary_of_nothing_and_refusals():
    from directaccesskernel_b200.decode_ops import rotary

    x, pos, inv = _case(4, 2, 128, 64, 7, torch.float16)
    x, pos, inv = x.cuda(), pos.cuda(), inv.cuda()
    assert rotary(x[:0], pos[:0], inv).shape == (0, 2, 128)
    for kw, msg in ((dict(x=x.float()), "float16"), (dict(positions=pos.long()), "int32"), (dict(positions=pos[:3]), "per token"),
                    (dict(inv_freq=inv.double()), "float32"), (dict(inv_freq=torch.ones(65, device="cuda")), "head_dim / 2"),
                    (dict(out=torch.empty_like(x[:2])), "out must match"), (dict(x=x[..., 1:125]), "multiple of 8"), (dict(x=x[..., ::2]), "contiguous"),
                    (dict(inv_freq=inv[:20]), "multiple of 16")):
        with pytest.raises(RuntimeError, match=msg):
            rotary(**{**dict(x=x, positions=pos, inv_freq=inv), **kw})
