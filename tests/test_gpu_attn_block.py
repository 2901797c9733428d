"""GPU test of the attention block: steps of many and of single tokens, behind a
shared context, against the whole computation in 64 bits on the host."""
import numpy as np
import pytest
import torch

from ai_engine_amd.attn_block import AttnBlock
from ai_engine_amd.conv import AihError, DType
from tests.gpu_util import rel_err

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TORCH = {DType.F32: torch.float32, DType.F16: torch.float16, DType.BF16: torch.bfloat16}
# the framework's bars for results against the reference (fp32, 16 bit)
BAR = {DType.F32: 1e-4, DType.F16: 2e-2, DType.BF16: 2e-2}
C, HQ, HKV, D = 64, 4, 2, 32


def make_weights(seed):
    r = np.random.default_rng(seed)
    n = lambda *s, scale: (r.standard_normal(s) * scale).astype(np.float32)
    return dict(w_qkv=n((HQ + 2 * HKV) * D, C, scale=C ** -0.5), b_qkv=n((HQ + 2 * HKV) * D, scale=0.01),
                w_out=n(C, HQ * D, scale=(HQ * D) ** -0.5), b_out=n(C, scale=0.01), wq=1 + n(D, scale=0.1),
                wk=1 + n(D, scale=0.1))


def reference(w, x, shared, causal, steps):
    """x [streams, tokens, C]: the block over the whole stream at once; without
    `causal` a token sees its whole step."""
    w = {k: torch.from_numpy(v).double() for k, v in w.items()}
    s, t, _ = x.shape
    full = torch.cat([shared.expand(s, -1, -1), x], 1).double()
    n, p = full.shape[1], shared.shape[1]
    qkv = (full @ w["w_qkv"].T + w["b_qkv"]).view(s, n, HQ + 2 * HKV, D)

    def norm_rotate(y, g):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * g
        ang = torch.arange(n).double()[:, None] * 10000.0 ** (-torch.arange(D // 2).double() / (D // 2))
        c, sn = ang.cos()[:, None], ang.sin()[:, None]
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat([a * c - b * sn, a * sn + b * c], -1)

    q, k = norm_rotate(qkv[:, :, :HQ], w["wq"]), norm_rotate(qkv[:, :, HQ:HQ + HKV], w["wk"])
    v = qkv[:, :, HQ + HKV:]
    last = torch.empty(n, dtype=torch.long)  # the last token each one sees
    at = p
    for m in steps:
        last[at:at + m] = torch.arange(at, at + m) if causal else at + m - 1
        at += m
    hidden = torch.arange(n)[None] > last[p:, None]
    k, v = (z.repeat_interleave(HQ // HKV, 2).transpose(1, 2) for z in (k, v))
    sc = q[:, p:].transpose(1, 2) @ k.transpose(2, 3) / D ** 0.5
    o = torch.softmax(sc.masked_fill(hidden, float("-inf")), -1) @ v
    return x.double() + o.transpose(1, 2).reshape(s, t, HQ * D) @ w["w_out"].T + w["b_out"]


@pytest.mark.parametrize("dt", list(DType))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shared", [0, 90])
def test_block_over_steps(dt, causal, shared):
    streams, steps = 3, [45, 1, 1, 20, 1]
    g = torch.Generator().manual_seed(7)
    x = torch.randn(streams, sum(steps), C, generator=g).to(TORCH[dt])
    ctx = torch.randn(1, shared, C, generator=g).to(TORCH[dt])
    w = make_weights(3)
    block = AttnBlock(C, HQ, HKV, D, streams, capacity=80, weights=w, dt=dt, causal=causal, prefix=100)
    if shared:
        block.share(ctx[0].to(DEV))
    want = reference(w, x.float(), ctx.float(), causal, steps).numpy()
    for _ in range(2):  # again after a reset
        got, at = [], 0
        for m in steps:
            got.append(block.step(x[:, at:at + m].contiguous().to(DEV)).cpu())
            at += m
        got = torch.cat(got, 1).float().numpy()
        assert rel_err(got, want) <= BAR[dt]
        block.reset()


def test_block_refusals():
    block = AttnBlock(C, HQ, HKV, D, 2, capacity=8, weights=make_weights(1), prefix=4)
    x = torch.zeros(2, 5, C, device=DEV)
    with pytest.raises(AihError, match="room for 4"):
        block.share(x[0])
    block.step(x)
    with pytest.raises(AihError, match="room for 8"):
        block.step(x)
    with pytest.raises(AihError, match="before"):
        block.share(x[0, :2])
    with pytest.raises(AihError, match="takes"):
        block.step(x.half())
    with pytest.raises(AihError, match="takes"):
        block.step(x[:1])
    assert block.step(x[:, :0]).shape == (2, 0, C)
    with pytest.raises(AihError, match="multiple of 8"):
        AttnBlock(12, HQ, HKV, D, 2, 8, make_weights(1))
