"""GPU test of the attention block with a 4-bit cache and 4-bit projections: all the
4-bit operators together, over steps of many and of single tokens, against 64 bits."""
import numpy as np
import pytest
import torch

from ai_engine_amd.attn_block import AttnBlock
from ai_engine_amd.conv import AihError, DType
from tests.gpu_util import rel_err
from tests.mx4_util import TORCH, quant_rows, values
from tests.test_gpu_attn_block import BAR

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def make_weights(seed, c, hq, hkv, d):
    r = np.random.default_rng(seed)
    n = lambda *s, scale: (r.standard_normal(s) * scale).astype(np.float32)
    return dict(w_qkv=n((hq + 2 * hkv) * d, c, scale=c ** -0.5), b_qkv=n((hq + 2 * hkv) * d, scale=0.01),
                w_out=n(c, hq * d, scale=(hq * d) ** -0.5), b_out=n(c, scale=0.01), wq=1 + n(d, scale=0.1),
                wk=1 + n(d, scale=0.1))


def in4(x):
    """The values that rows [rows, k] stand for in 4 bits, fp64."""
    return values(*quant_rows(x))[:, :x.shape[1]]


@pytest.mark.parametrize("dt", list(DType))
@pytest.mark.parametrize("proj4", [False, True])
@pytest.mark.parametrize("causal, c, hq, hkv, d, page", [(True, 64, 4, 2, 32, 16), (False, 128, 8, 2, 64, 64), (True, 96, 3, 3, 96, 32)])
def test_block_over_steps(dt, proj4, causal, c, hq, hkv, d, page):
    streams, steps, cap = 3, [45, 1, 1, 20, 1], 80
    g = torch.Generator().manual_seed(7)
    x = torch.randn(streams, sum(steps), c, generator=g).to(TORCH[dt])
    w = make_weights(3, c, hq, hkv, d)
    block = AttnBlock(c, hq, hkv, d, streams, capacity=cap, weights=w, dt=dt, causal=causal, cache4=True, page=page, proj4=proj4)
    W = {k: torch.from_numpy(v).double() for k, v in w.items()}
    if proj4:
        W["w_qkv"], W["w_out"] = in4(torch.from_numpy(w["w_qkv"])), in4(torch.from_numpy(w["w_out"]))
    ang = torch.arange(cap).double()[:, None] * 10000.0 ** (-torch.arange(d // 2).double() / (d // 2))
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def norm_rotate(y, gain, at):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * gain
        a, b = y[..., :d // 2], y[..., d // 2:]
        c_, s_ = cos[at:at + y.shape[1]], sin[at:at + y.shape[1]]
        return torch.cat([a * c_ - b * s_, a * s_ + b * c_], -1)

    at = 0
    for m in steps:
        xs = x[:, at:at + m].contiguous()
        y = block.step(xs.to(DEV)).double().cpu()
        o = block._plans[m]["o"].double().cpu().view(streams, m, hq * d)
        rows = xs.reshape(-1, c)
        rows = in4(rows) if proj4 else rows.double()
        qkv = (rows @ W["w_qkv"].T + W["b_qkv"]).view(streams, m, hq + 2 * hkv, d)
        q = norm_rotate(qkv[:, :, :hq], W["wq"], at)
        new = (norm_rotate(qkv[:, :, hq:hq + hkv], W["wk"], at), qkv[:, :, hq + hkv:])
        # what the cache holds: the new rows within the format's error, which is a quarter of a block's largest
        # magnitude at most (above 6 scales of 8, or half of a step of 2 there)
        held = []
        for i in range(2):
            v = values(block.cache[2 * i].flatten(0, 2), block.cache[2 * i + 1].flatten(0, 2))
            v = v.view(streams, -1, hkv, page, d).transpose(2, 3).reshape(streams, -1, hkv, d)
            top = new[i].reshape(*new[i].shape[:3], -1, 32).abs().amax(-1, keepdim=True)
            off = (v[:, at:at + m] - new[i]).reshape(*new[i].shape[:3], -1, 32).abs()
            assert (off <= (0.25 + BAR[dt]) * top + BAR[dt]).all()
            held.append(v[:, :at + m])
        k, v = (z.repeat_interleave(hq // hkv, 2).transpose(1, 2) for z in held)
        sc = q.transpose(1, 2) @ k.transpose(2, 3) / d ** 0.5
        if causal:
            sc = sc.masked_fill(torch.arange(at + m)[None] > torch.arange(at, at + m)[:, None], float("-inf"))
        want = (torch.softmax(sc, -1) @ v).transpose(1, 2).reshape(streams, m, hq * d)
        assert rel_err(o.numpy(), want.numpy()) < BAR[dt]
        # the projection back, of the rows as the block has them
        rows = in4(o.reshape(-1, hq * d)).view_as(o) if proj4 else o
        out = xs.double() + rows @ W["w_out"].T + W["b_out"]
        assert rel_err(y.numpy(), out.numpy()) < BAR[dt]
        at += m
    with pytest.raises(AihError, match="room for"):
        block.step(torch.zeros(streams, cap - at + 1, c, dtype=TORCH[dt], device=DEV))
    block.reset()
    again = block.step(x[:, :steps[0]].contiguous().to(DEV))
    block.reset()
    assert torch.equal(again, block.step(x[:, :steps[0]].contiguous().to(DEV)))


def test_a_step_is_the_sum_of_its_tokens():
    # whole prompts and single tokens leave the same cache and nearly the same rows
    c, hq, hkv, d = 64, 4, 2, 64
    w = make_weights(5, c, hq, hkv, d)
    x = torch.randn(2, 30, c, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    one, many = (AttnBlock(c, hq, hkv, d, 2, 64, w, DType.BF16, cache4=True, page=16) for _ in range(2))
    whole = one.step(x)
    rows = torch.cat([many.step(x[:, t:t + 1].contiguous()) for t in range(30)], 1)
    assert (whole.float() - rows.float()).abs().max() < BAR[DType.BF16]
    for a, b in zip(one.cache, many.cache):
        assert (a == b).double().mean() > 0.99  # a projection's last bit may fall to the other side of a border
