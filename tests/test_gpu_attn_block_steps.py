"""GPU test of the attention block's steps whose lengths grow and shrink: their
buffers are shared."""
import pytest
import torch

from ai_engine_amd.attn_block import AttnBlock
from ai_engine_amd.conv import DType
from tests.gpu_util import rel_err
from tests.test_gpu_attn_block import BAR, C, D, DEV, HKV, HQ, TORCH, make_weights, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", list(DType))
@pytest.mark.parametrize("shared", [0, 30])
def test_lengths_that_grow_and_shrink(dt, shared):
    streams, steps = 3, [1, 20, 3, 70, 1, 20, 71, 2]
    g = torch.Generator().manual_seed(9)
    x = torch.randn(streams, sum(steps), C, generator=g).to(TORCH[dt])
    ctx = torch.randn(1, shared, C, generator=g).to(TORCH[dt])
    w = make_weights(4)
    block = AttnBlock(C, HQ, HKV, D, streams, capacity=sum(steps), weights=w, dt=dt, prefix=40)
    block.share(ctx[0].to(DEV))
    want = reference(w, x.float(), ctx.float(), True, steps).numpy()
    got, at = [], 0
    for m in steps:  # results are compared at the end: no step may touch another's
        got.append(block.step(x[:, at:at + m].contiguous().to(DEV)))
        at += m
    assert rel_err(torch.cat(got, 1).cpu().float().numpy(), want) <= BAR[dt]
