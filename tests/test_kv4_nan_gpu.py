"""What the 4-bit cache holds of NaN."""
import math

import pytest
import torch

from kv4_common import D, parts, quantise32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_of_groups_of_nothing_but_nan(group, dtype):
    """Such a group is stored as zeros and read back as zeros; the groups beside it are as ever, and
    a NaN among numbers is their minimum."""
    from directaccesskernel_b200 import kv4

    rows = torch.randn(4, 1, D, generator=torch.Generator().manual_seed(1))
    x = rows.clone()
    x[0] = math.nan
    x[1, :, :group] = math.nan
    x[2, :, 3] = math.nan
    x = x.to(dtype)
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = torch.full((1, 1, kv4.page_bytes(16, group)), 255, dtype=torch.uint8, device="cuda")
    at = (i32([[0]]), i32([0, 1, 2, 3]))
    kv4.rope_kv_append_q4(torch.cat([x, x], 1).reshape(4, 2 * D).cuda(), at[1], None, 0, None, pool, None, at[0],
                          seq_index=i32([0] * 4))
    k, v = (t.cpu().float()[:, 0] for t in kv4.kv_read_q4(pool, None, *at, seq_index=i32([0] * 4), dtype=dtype))
    kc, kp, vc, vp = (t[0, 0, :4] for t in parts(pool.cpu(), 16, group))
    assert torch.equal(kc, vc) and torch.equal(kp.view(torch.int16), vp.view(torch.int16)) and torch.equal(k, v)
    assert not vc[0].any() and not vp[0].view(torch.int16).any() and not v[0].any()
    assert not vc[1, :group].any() and not vp[1, 0].view(torch.int16).any() and not v[1, :group].any()
    n, p = quantise32(x[:, 0], group)
    assert torch.equal(vc[1, group:], n[1, group:]) and torch.equal(vp[1, 1:], p[1, 1:])
    assert torch.equal(vc[3], n[3]) and torch.equal(vp[3], p[3])
    rest = x[2, 0].float()[:group].nan_to_num(math.inf)
    assert vc[2, 3] == 0 and v[2, 3] == rest.amin().half().to(dtype)
