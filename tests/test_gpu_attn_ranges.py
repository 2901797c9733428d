"""GPU tests of the attention operators at the ends of the numbers' range.

Scores: q . k holds whole numbers times powers of two that fp32 products and
sums keep exactly, so equal scores are equal and different ones are so far
apart that only the largest count: the result is the mean of their values,
within the roundings of a probability, the sums, the quotient and the store,
  |o - exact| <= A (w + (2 n + 64) u) + w |exact| + tiny,  A the mean of |v|.

Norms: scaling a head by a power of two rounds nothing, so the bound is that of
test_gpu_attn.py.
"""
import pytest
import torch

from ai_engine_amd import attn
from ai_engine_amd.conv import DType
from tests.test_gpu_attn import ALL, TINY, TORCH, U, W, Rope
from tests.test_gpu_attn_routes import Batch

pytestmark = pytest.mark.gpu

ROWS, KEYS = attn.AttnKernel.ROWS, attn.AttnKernel.KEYS


def check_largest(c, rank, spec=None):
    """q . k = 2^14 rank of the key: the keys of the largest rank that a row sees share it."""
    g = torch.Generator().manual_seed(3)
    dims = torch.randint(0, c.d, (c.hkv,), generator=g)
    c.q, c.k = torch.zeros_like(c.q), torch.zeros_like(c.k)
    ranks = [rank(torch.arange(n)) for n in c.k_lens]
    flat = torch.zeros(c.rows)
    for s, r in zip(c.k_starts, ranks):
        flat[s:s + len(r)] = r.float()
    for h in range(c.hkv):
        c.q[:, h * (c.hq // c.hkv):(h + 1) * (c.hq // c.hkv), dims[h]] = 2.0 ** 7
        c.k[:, h, dims[h]] = (2.0 ** 7 * flat).to(c.k.dtype)
    got = c.run(spec=spec).double()
    for b, (lq, lk) in enumerate(zip(c.q_lens, c.k_lens)):
        v = c.v[c.k_starts[b]:c.k_starts[b] + lk].double().repeat_interleave(c.hq // c.hkv, 1)
        seen = (torch.arange(lq) + 1 + lk - lq).clamp(0, lk)[:, None] if c.causal else torch.full((lq, 1), lk)
        r = ranks[b][None].masked_fill(torch.arange(lk)[None] >= seen, -1 << 40)
        top = ((r == r.amax(-1, keepdim=True)) & (r > -1 << 40)).double()
        top = top / top.sum(-1, keepdim=True).clamp(min=1)  # the share of each key
        want, a = (top @ x.reshape(lk, -1) for x in (v, v.abs()))
        bound = a * (W[c.dt] + (2 * seen + 64) * U) + W[c.dt] * want.abs() + TINY[c.dt]
        off = (got[c.q_starts[b]:c.q_starts[b] + lq].reshape(lq, -1) - want).abs()
        assert (off <= bound).all(), (b, float((off / bound).max()))


RANKS = {"equal": lambda j: 0 * j + 37, "rising": lambda j: j // 4, "falling": lambda j: 90 - j // 4,
         "two": lambda j: 50 - (j * 7 % 64 > 1).long(), "below": lambda j: -1 - (j * 5) % 90}
# scores of 2^14 rank times these; the last is the largest scale there is
SCALES = [2.0 ** 6, 3.1e4, 1.7e6, 9.0e9, 1e20]


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("scale", SCALES)
def test_huge_scores_of_prompts(dt, d, scale):
    f32 = dt == DType.F32
    for name, rank in RANKS.items():
        heads, lens = (224, [333, 260]) if f32 else (100, [333])
        c = Batch(dt, heads, heads, d, lens, lens, scale=scale, seed=d)
        assert c.spec().plan().kernel == (KEYS if f32 and d > 128 else ROWS)
        check_largest(c, rank)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("lens", [[180, 33, 1], [3000, 1030, 257]])
def test_huge_scores_of_caches(dt, d, scale, lens):
    for name, rank in RANKS.items():
        c = Batch(dt, 8, 2, d, [2] * 3, lens, scale=scale, seed=d)
        assert c.spec().plan().kernel == KEYS
        check_largest(c, lambda j, rank=rank: rank(j % 400))


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
