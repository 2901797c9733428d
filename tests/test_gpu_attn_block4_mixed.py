"""GPU test of the attention block with 4-bit projections over a 16-bit or fp32 cache and
behind a shared context, against 64 bits."""
import pytest
import torch

from ai_engine_amd.attn_block import AttnBlock
from ai_engine_amd.conv import DType
from tests.gpu_util import rel_err
from tests.mx4_util import TORCH
from tests.test_gpu_attn_block import BAR
from tests.test_gpu_attn_block4 import DEV, in4, make_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", list(DType))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shared", [0, 50])
@pytest.mark.parametrize("c, hq, hkv, d", [(64, 4, 2, 32), (96, 3, 3, 40), (128, 8, 2, 64)])
def test_block_over_steps(dt, causal, shared, c, hq, hkv, d):
    streams, steps = 3, [33, 1, 1, 12, 1]
    g = torch.Generator().manual_seed(9)
    x = torch.randn(streams, sum(steps), c, generator=g).to(TORCH[dt])
    front = torch.randn(shared, c, generator=g).to(TORCH[dt])
    w = make_weights(4, c, hq, hkv, d)
    rot = d // 16 * 16
    block = AttnBlock(c, hq, hkv, d, streams, capacity=60, weights=w, dt=dt, causal=causal, rot=rot, prefix=64, proj4=True)
    if shared:
        block.share(front.to(DEV))
    W = {k: torch.from_numpy(v).double() for k, v in w.items()}
    W["w_qkv"], W["w_out"] = in4(torch.from_numpy(w["w_qkv"])), in4(torch.from_numpy(w["w_out"]))
    n = shared + sum(steps)
    full = torch.cat([front.expand(streams, -1, -1), x], 1)
    qkv = (in4(full.reshape(-1, c)) @ W["w_qkv"].T + W["b_qkv"]).view(streams, n, hq + 2 * hkv, d)
    ang = torch.arange(n).double()[:, None] * 10000.0 ** (-torch.arange(rot // 2).double() / (rot // 2))
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def norm_rotate(y, gain):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * gain
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., rot:]], -1)

    q, k = norm_rotate(qkv[:, :, :hq], W["wq"]), norm_rotate(qkv[:, :, hq:hq + hkv], W["wk"])
    k, v = (z.repeat_interleave(hq // hkv, 2).transpose(1, 2) for z in (k, qkv[:, :, hq + hkv:]))
    at = 0
    for m in steps:
        xs = x[:, at:at + m].contiguous()
        y = block.step(xs.to(DEV)).double().cpu()
        o = block._plans[m]["o"].double().cpu().view(streams, m, hq * d)
        end = shared + at + m
        sc = q[:, end - m:end].transpose(1, 2) @ k[:, :, :end].transpose(2, 3) / d ** 0.5
        if causal:
            sc = sc.masked_fill(torch.arange(end)[None] > torch.arange(end - m, end)[:, None], float("-inf"))
        want = (torch.softmax(sc, -1) @ v[:, :, :end]).transpose(1, 2).reshape(streams, m, hq * d)
        assert rel_err(o.numpy(), want.numpy()) < BAR[dt]
        # the projection back, of the rows as the block has them
        out = xs.double() + in4(o.reshape(-1, hq * d)).view_as(o) @ W["w_out"].T + W["b_out"]
        assert rel_err(y.numpy(), out.numpy()) < BAR[dt]
        at += m
    block.reset()
    again = block.step(x[:, :steps[0]].contiguous().to(DEV))
    block.reset()
    assert torch.equal(again, block.step(x[:, :steps[0]].contiguous().to(DEV)))
