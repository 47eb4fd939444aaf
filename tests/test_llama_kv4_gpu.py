"""The Llama decoder with a 4-bit KV cache, scaled rotary positions and forked
sequences."""
import dataclasses
import math

import pytest
import torch

from kv4_common import attend64, parts, values
from test_llama_tp_gpu import _cfg, _hf, _rel, _teacher_forced

pytestmark = pytest.mark.gpu


def _decoder(cfg, **kw):
    from directaccesskernel_b200.llama_tp import LlamaShape, TPLlamaDecoder

    return TPLlamaDecoder(LlamaShape.from_config(cfg), batch=kw.pop("batch", 2), max_ctx=kw.pop("max_ctx", 200), **kw)


@pytest.mark.parametrize("kv_host,group", [(0.0, 128), (0.5, 32), (1.0, 64)])
def test_attention_of_every_step_is_that_of_its_4_bit_pages(kv_host, group):
    """Eager steps over a page border; after each, the last layer's attention output is
    the 64-bit attention of its query over its pages, and the graph of a step
    continues with the same bits."""
    from directaccesskernel_b200 import runtime
    from test_kv4_gpu import _bound

    cfg = _cfg()
    dec = _decoder(cfg, kv_bits=4, kv_group=group, kv_host_fraction=kv_host).load_hf(_hf(cfg, seed=5))
    assert dec.kv_bytes()[0] + dec.kv_bytes()[1] == dec.s.kv_bytes_per_rank(1, 2, 200, kv_bits=4, kv_group=group)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, cfg.vocab_size, (2, 70), generator=g).cuda()
    scale = 1 / math.sqrt(128)
    for t in range(70):
        dec.ids.copy_(prompt[:, t])
        dec.set_positions(t)
        with torch.inference_mode():
            dec.forward_step()
        if t not in (0, 1, 63, 64, 69):
            continue
        torch.cuda.synchronize()
        pools = [None if p is None else p[-1].cpu() for p in (dec.kv_dev, dec.kv_host)]
        q = dec.q_buf.cpu()
        ref = attend64(q, pools, 64, group, dec.host_table, [t + 1] * 2, scale)
        used = [p for p in pools if p is not None]
        v_range = 15 * max(torch.nan_to_num(parts(p, 64, group)[3][..., 0].double(), 0, 0, 0).abs().amax() for p in used)
        k_abs = max(torch.nan_to_num(values(*parts(p, 64, group)[:2]), 0, 0, 0).abs().amax() for p in used)
        assert ((dec.attn_out.cpu().double() - ref).abs() <= _bound(ref, q, k_abs, v_range, scale, q.dtype)).all()
    dec.ids.copy_(prompt[:, 69])
    dec.set_positions(69)
    dec.capture()
    dec.step()
    torch.cuda.synchronize()
    graphed = dec.attn_out.clone()
    dec.graph = None
    dec.ids.copy_(prompt[:, 69])
    dec.set_positions(69)
    dec.step()
    assert torch.equal(graphed, dec.attn_out)
    assert runtime.device_status() == 0 and not dec.merge_counters.any()


def test_4_bit_logits_stay_near_16_bit_logits():
    """K and V off by at most half a step, range / 30 of a group, move the logits, but
    not beyond recognition: the step's logits correlate with the 16-bit cache's."""
    cfg = _cfg()
    hf = _hf(cfg, seed=7)
    prompt = torch.randint(0, cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(3)).cuda()
    a = _teacher_forced(_decoder(cfg).load_hf(hf), prompt)
    b = _teacher_forced(_decoder(cfg, kv_bits=4, kv_group=32, kv_host_fraction=0.5).load_hf(hf), prompt)
    a, b = (t - t.mean(-1, keepdim=True) for t in (a.double(), b.double()))
    cos = (a * b).sum(-1) / (a.norm(dim=-1) * b.norm(dim=-1))
    # Half a step is at most 1/30 of a group's range, 4 to 5 standard deviations of 32 values: 1/6 at the very
    # most and 1/12 rms of what attention adds to the stream, beside the embedding and the MLPs: an angle of
    # at most asin(1/6) + asin(1/6).
    assert cos.min() > math.cos(2 * math.asin(1 / 6))


@pytest.mark.parametrize("scaling", [
    dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=64),
    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64), dict(rope_type="linear", factor=4.0)])
def test_scaled_rotary_matches_transformers(scaling):
    cfg = _cfg()
    theta = (getattr(cfg, "rope_parameters", None) or {}).get("rope_theta", 500000.0)
    cfg.rope_parameters = dict(scaling, rope_theta=theta)
    hf = _hf(cfg, seed=5)
    prompt = torch.randint(0, cfg.vocab_size, (2, 90), generator=torch.Generator().manual_seed(2)).cuda()
    dec = _decoder(cfg, kv_host_fraction=0.5).load_hf(hf)
    assert (dec.rope_scale != 1.0) == (scaling["rope_type"] == "yarn")
    assert dec.kernel_launches_per_step() == 2 + 3 * (9 if dec.rope_scale != 1.0 else 8)
    got = _teacher_forced(dec, prompt)
    with torch.inference_mode():
        ref = hf(input_ids=prompt).logits.float()
    assert _rel(got, ref) <= 1e-2  # test_llama_tp_gpu's tolerance


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_fork_continues_like_its_source(kv_bits):
    cfg = _cfg()
    dec = _decoder(cfg, batch=3, kv_bits=kv_bits, kv_host_fraction=0.4).load_hf(_hf(cfg, seed=11))
    prompt = torch.randint(0, cfg.vocab_size, (3, 71), generator=torch.Generator().manual_seed(4)).cuda()
    _teacher_forced(dec, prompt)
    dec.ids.copy_(prompt[:, 70])
    dec.set_positions(70)
    dec.ids[2] += 1
    dec.fork(1, 2, 70)
    for _ in range(4):
        with torch.inference_mode():
            dec.forward_step(keep_logits=True)
            dec.advance()
        assert torch.equal(dec.logits_full[1], dec.logits_full[2])
        assert not torch.equal(dec.logits_full[0], dec.logits_full[1])
    for bad in ((1, 1, 5), (0, 3, 5), (0, 1, 201), (0, 1, -1)):
        with pytest.raises(ValueError):
            dec.fork(*bad)


@pytest.mark.parametrize("kv_bits", [16, 4])
@pytest.mark.parametrize("tokens", [0, 1, 63, 64, 66])
def test_fork_behind_its_source_goes_on_from_there(kv_bits, tokens):
    """A row forked at an earlier token, fed what its source was fed, comes to the
    same logits: nothing past ``tokens`` is read before it is written."""
    cfg = _cfg()
    dec = _decoder(cfg, batch=3, kv_bits=kv_bits, kv_host_fraction=0.4).load_hf(_hf(cfg, seed=11))
    prompt = torch.randint(0, cfg.vocab_size, (3, 70), generator=torch.Generator().manual_seed(5)).cuda()
    _teacher_forced(dec, prompt)
    dec.set_positions(70)
    with torch.inference_mode():
        dec.ids.copy_(prompt[:, 69])
        dec.set_positions(69)
        dec.forward_step(keep_logits=True)
        want = dec.logits_full[1].clone()
        dec.fork(1, 2, tokens)
        assert dec.pos.tolist() == [69, 69, tokens]
        for t in range(tokens, 70):
            dec.ids[2] = prompt[1, t]
            dec.pos[2] = t
            dec.pos[:2] = 69
            dec.forward_step(keep_logits=True)
    assert torch.equal(dec.logits_full[2], want) and torch.equal(dec.logits_full[1], want)


def test_random_4_bit_pages_are_sane_and_steps_run():
    cfg = _cfg()
    from directaccesskernel_b200.llama_tp import LlamaShape, TPLlamaDecoder

    shape = dataclasses.replace(LlamaShape.from_config(cfg), layers=2)
    dec = TPLlamaDecoder(shape, batch=2, max_ctx=150, kv_bits=4, kv_host_fraction=0.5).init_random(seed=1)
    dec.fill_kv_random(130)
    for p in (dec.kv_dev.cpu(), dec.kv_host):
        kc, kp, vc, vp = parts(p, 64, 128)
        assert kc.float().mean() > 7 and vc.float().mean() < 8
        assert values(kc, kp).abs().max() < 2.61 and values(vc, vp).abs().max() < 2.61
    dec.capture()
    for _ in range(3):
        dec.step()
    torch.cuda.synchronize()
    assert torch.isfinite(dec.attn_out).all() and int(dec.pos[0]) == 133
