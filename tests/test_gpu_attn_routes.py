"""GPU tests of the attention kernels' less usual routes against plain 64-bit
computations, with the bounds of test_gpu_attn.py: each asserts the plan, so
that it cannot drift to another kernel.

  rows kernel   fp32, more than 64 sequences, more than 8 key heads, a prefix in
                a launch of its own, whole and cut
  keys kernel   workgroups that take several items of cut keys
  softmax       a maximum that is raised in later blocks, or never again
"""
import math

import numpy as np
import pytest
import torch

from ai_engine_amd import attn
from ai_engine_amd.conv import DType
from tests.test_gpu_attn import ALL, DEV, TINY, TORCH, U, W, Case, i32

pytestmark = pytest.mark.gpu

ROWS, KEYS = attn.AttnKernel.ROWS, attn.AttnKernel.KEYS
CUS = 256
HALF = [DType.F16, DType.BF16]


class Batch(Case):
    """A Case whose 64-bit result is computed a sequence and a few heads at a time."""

    def exact(self):
        scale = self.scale if self.scale is not None else 1.0 / math.sqrt(self.d)
        o = torch.zeros(self.tokens, self.hq, self.d, dtype=torch.float64)
        e = torch.zeros_like(o)
        g = self.hq // self.hkv
        for b, (lq, lk) in enumerate(zip(self.q_lens, self.k_lens)):
            n = lk + self.prefix
            if lq == 0 or n == 0:
                continue
            t0, k0 = self.q_starts[b], self.k_starts[b]
            seen = torch.full((lq,), lk)
            if self.causal:
                seen = (torch.arange(lq) + 1 + lk - lq).clamp(0, lk)
            seen = seen + self.prefix
            hidden = (torch.arange(n)[None] >= seen[:, None]).repeat_interleave(g, 0)[None]
            count = seen.repeat_interleave(g).double()[None, :, None]
            step = max(1, (1 << 24) // (lq * g * n))
            for h in range(0, self.hkv, step):
                m = min(step, self.hkv - h)
                q = self.q[t0:t0 + lq, h * g:(h + m) * g].double().view(lq, m, g, self.d)
                q = q.transpose(0, 1).reshape(m, lq * g, self.d)
                kk, vv = (torch.cat([p[:, h:h + m], t[k0:k0 + lk, h:h + m]]).double().transpose(0, 1).contiguous()
                          for p, t in ((self.pk, self.k), (self.pv, self.v)))
                kt = kk.transpose(1, 2).contiguous()
                s = scale * (q @ kt)
                far = (q.abs() @ kt.abs()).masked_fill(hidden, 0).amax(-1, keepdim=True)
                ds = scale * (self.d + 8) * U * far + 4 * U * s.abs().masked_fill(hidden, 0).amax(-1, keepdim=True)
                s = s.masked_fill(hidden, -math.inf)
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
                z = p.sum(-1, keepdim=True)
                p = p / torch.where(z == 0, torch.ones_like(z), z)
                oo, a = p @ vv, p @ vv.abs()
                w = W[self.dt]
                err = (a * (4 * ds + w + (2 * count + 64) * U) + w * oo.abs() + count * 2.0 ** -32 * vv.abs().max()
                       + TINY[self.dt])
                for to, x in ((o, oo), (e, err)):
                    to[t0:t0 + lq, h * g:(h + m) * g] = (x.view(m, lq, g, self.d).transpose(0, 1)
                                                         .reshape(lq, m * g, self.d))
        return o, e


def ragged(n, hi, seed, longest):
    r = np.random.default_rng(seed)
    lens = r.integers(0, hi, n).tolist()
    lens[0], lens[1], lens[n // 2], lens[-1] = 0, 1, longest, 0  # empty ones at both ends
    return lens


def test_the_batched_result_is_the_other_one():
    kw = dict(prefix=9, gap=2, seed=1)
    a, b = (cls(DType.F16, 6, 2, 8, [5, 0, 30, 1], [3, 4, 37, 0], True, **kw).exact() for cls in (Case, Batch))
    assert torch.allclose(a[0], b[0], rtol=1e-12, atol=1e-13)
    assert torch.allclose(a[1], b[1], rtol=1e-3, atol=1e-23)  # max|v| is of a few heads, or of all


# ---------------------------------------------------------------- rows kernel

@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_fp32_prompts_over_the_rows(d, causal):
    lens = ragged(70, 81, d, 300)
    c = Batch(DType.F32, 24, 24, d, lens, lens, causal, seed=d)
    assert c.spec().plan().kernel == ROWS
    c.check()


@pytest.mark.parametrize("d", [64, 128])
def test_fp32_prompts_over_the_rows_after_earlier_keys(d):
    q_lens = ragged(70, 61, d, 200)
    k_lens = [max(0, n + (-3, 0, 50)[i % 3]) for i, n in enumerate(q_lens)]  # some rows see nothing
    c = Batch(DType.F32, 48, 24, d, q_lens, k_lens, True, seed=d + 1, gap=1)
    assert c.spec().plan().kernel == ROWS
    c.check()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("n, hq, hkv", [(70, 12, 12), (130, 18, 9), (65, 40, 20)])
def test_many_sequences_and_heads_over_the_rows(dt, d, n, hq, hkv):
    lens = ragged(n, 90, d + n, 250)
    c = Batch(dt, hq, hkv, d, lens, lens, seed=n)
    assert c.spec().plan().kernel == ROWS
    c.check()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 136, 256])
@pytest.mark.parametrize("prefix, cut", [(70, False), (1300, True)])
def test_a_prefix_of_its_own_launch_behind_prompts(dt, d, prefix, cut):
    # keys of the prefix whole, and cut so that a workgroup's begin inside it
    c = Batch(dt, 4, 2, d, [60, 0, 130], [60, 5, 200], prefix=prefix, seed=d)
    p = c.spec().plan()
    assert (p.kernel, p.prefix_kernel) == (ROWS, ROWS) and (p.prefix_parts > 1) == cut
    c.check()


@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("prefix", [33, 400])
def test_a_prefix_of_its_own_launch_behind_fp32_prompts(d, prefix):
    lens = ragged(70, 81, d, 200)
    c = Batch(DType.F32, 24, 24, d, lens, lens, prefix=prefix, seed=d)
    p = c.spec().plan()
    assert (p.kernel, p.prefix_kernel) == (ROWS, ROWS)
    c.check()


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("d", [64, 96, 128, 136, 256])
def test_a_long_prefix_of_its_own_launch_under_single_tokens(dt, d):
    # much to read for every 32 rows: over the rows, cut, joined with the keys kernel's parts
    c = Batch(dt, 256, 8, d, [1] * 40, [5, 0, 9, 2] * 10, prefix=4200, seed=d)
    p = c.spec().plan()
    assert (p.kernel, p.prefix_kernel) == (KEYS, ROWS) and p.prefix_parts > 1
    c.check()


# ---------------------------------------------------------------- keys kernel, several items a workgroup

# key heads for each size so that items are more than workgroups ever run at once
MANY = [(40, 16), (64, 16), (96, 8), (128, 8), (256, 4)]
PLACES = {40: 4, 64: 4, 96: 2, 128: 2, 256: 1}  # workgroups a CU at most


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d, hkv", MANY)
@pytest.mark.parametrize("lq, prefix", [(1, 0), (3, 0), (1, 150)])
def test_workgroups_that_take_several_items(dt, d, hkv, lq, prefix):
    r = np.random.default_rng(d + lq)
    lens = [(0, 1, 33, 1025, 1300, 40)[i] for i in r.integers(0, 6, 129)] + [3000]
    c = Batch(dt, 2 * hkv, hkv, d, [lq] * 130, lens, prefix=prefix, seed=d + lq, gap=1)
    p = c.spec().plan()
    assert p.kernel == KEYS and p.parts > 1
    items = hkv * sum(max(1, -(-n // p.chunk)) for n in lens)
    assert items > CUS * PLACES[d]
    # what no sequence holds, and with three tokens the last value, which only the last one sees
    for t in (c.k, c.v):
        keep = t.clone()
        t[:] = float("nan")
        for s, n in zip(c.k_starts, c.k_lens):
            t[s:s + n] = keep[s:s + n]
    c.check()
    if lq == 3:
        want = c.run()
        for s, n in zip(c.k_starts, c.k_lens):
            if n:
                c.v[s + n - 1] = float("inf")
        got = c.run()
        first = torch.arange(c.tokens) % 3 < 2
        assert torch.equal(got[first], want[first])
        last = torch.tensor([3 * b + 2 for b, n in enumerate(lens) if n])
        assert not torch.isfinite(got[last]).any()


def test_several_items_give_the_same_bits_every_time():
    lens = [(0, 1, 33, 1025, 1300, 40)[i % 6] for i in range(130)]
    c = Batch(DType.BF16, 16, 8, 128, [1] * 130, lens, seed=5)
    spec = c.spec(max_len=3000)
    assert spec.plan().parts > 1
    want = c.run(spec=spec)
    for _ in range(3):
        assert torch.equal(c.run(spec=spec), want)


# ---------------------------------------------------------------- the running maximum

def along(case, shape, seed):
    """Scores that follow `shape` (of the key's place in its sequence, in 64 bits; the
    exponent's units) along the keys: q . k scale log2(e) = shape + a little."""
    d, g = case.d, torch.Generator().manual_seed(seed)
    u = torch.randn(d, generator=g)
    u = u / u.norm()
    scale = 1.0 / math.sqrt(d) * 1.4426950408889634
    case.q = (8 * u + 0.1 * torch.randn(case.tokens, case.hq, d, generator=g)).to(TORCH[case.dt])
    rows = torch.cat([shape(torch.arange(n).double()) for n in case.k_lens]).float()
    case.k = (rows[:, None, None] * u / (8 * scale)
              + 0.1 * torch.randn(len(rows), case.hkv, d, generator=g)).to(TORCH[case.dt])


SHAPES = {"rising": lambda j: 0.4 * j, "falling": lambda j: -0.4 * j, "steps": lambda j: 40 * (j // 100),
          "waves": lambda j: 30 * torch.sin(j / 20) + 0.1 * j}


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 136, 256])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_the_maximum_along_prompts(dt, d, shape, causal):
    lens = [333, 260] if dt == DType.F32 else [333]
    hkv = 224 if dt == DType.F32 and d <= 128 else 100
    c = Batch(dt, hkv, hkv, d, lens, lens, causal, seed=d)
    rows = d <= 128 or dt != DType.F32
    assert c.spec().plan().kernel == (ROWS if rows else KEYS)
    along(c, SHAPES[shape], d)
    c.check()


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens", [[700], [2500, 333]])
def test_the_maximum_along_caches(dt, d, shape, lens):
    c = Batch(dt, 8, 2, d, [2] * len(lens), lens, seed=d)
    assert c.spec().plan().kernel == KEYS
    along(c, SHAPES[shape], d)
    c.check()
