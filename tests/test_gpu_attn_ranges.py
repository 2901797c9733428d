"""GPU tests of the attention operators at the ends of the numbers' range.

Norms: scaling a head by a power of two rounds nothing, so the bound is that of
test_gpu_attn.py.
"""
import pytest
import torch

from ai_engine_amd.conv import DType
from tests.test_gpu_attn import ALL, TORCH, Rope

pytestmark = pytest.mark.gpu

# ---------------------------------------------------------------- norms

@pytest.mark.parametrize("dt", [DType.F32, DType.BF16])
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e-38])
@pytest.mark.parametrize("d, rot, pairs", [(64, 64, False), (72, 0, False), (96, 48, True), (256, 252, False)])
def test_norms_of_tiny_and_huge_heads(dt, eps, d, rot, pairs):
    # heads of every magnitude side by side, subnormal values among them
    r = Rope(dt, 24, 3, 2, d, rot, pairs, seed=d, eps=eps, scale=1.0)
    scales = [1e-42, 1e-39, 1e-36, 1e-30, 1e-23, 1e-20, 1e-19, 1e-15, 1.0, 1e15, 1e18, 3e18, 1e19, 1e20, 1e25, 1e30, 1e36,
              5e37]
    x = r.x.float().clamp(-4, 4).double()
    for t in range(24):
        for h in range(7):
            x[t, h] *= scales[(5 * t + h) % len(scales)]
    r.x = x.to(torch.float32).to(TORCH[dt])
    assert torch.isfinite(r.x).all()
    (wq, wk), wv, (eq, ek) = r.exact()
    q, k, v = r.run()
    assert torch.equal(v.double(), wv)
    for got, want, bound in ((q, wq, eq), (k, wk, ek)):
        # a head of zeros (bf16's 1e-42) without eps is 0 / 0
        defined = ~want.isnan()
        assert eps == 0 or defined.all()
        assert ((got.double() - want).abs() <= bound)[defined].all()


@pytest.mark.parametrize("dt", ALL)
def test_norms_of_heads_of_zeros_and_of_one_value(dt):
    r = Rope(dt, 6, 2, 1, 64, 64, seed=7, eps=1e-30 if dt != DType.F16 else 1e-6)
    r.x[0] = 0
    r.x[1] = 0
    r.x[1, :, 9] = torch.finfo(TORCH[dt]).tiny
    r.x[2] = torch.finfo(TORCH[dt]).max
    r.x[3] = 0
    r.x[3, :, 63] = torch.finfo(TORCH[dt]).max
    got = r.run()
    r.check(got)
    assert (got[0][0] == 0).all() and (got[1][0] == 0).all()
