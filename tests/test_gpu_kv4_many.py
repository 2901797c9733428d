"""GPU tests of attention over the 4-bit cache for very many sequences."""
import pytest
import torch

from ai_engine_amd import mx4
from ai_engine_amd.conv import DType
from tests.test_gpu_kv4 import DEV, Case, i32, noise_cache

pytestmark = pytest.mark.gpu


def run(n, q, lens, cache, **kw):
    heads, d = q.shape[1:]
    at = torch.arange(n, device=DEV) % len(q)
    out = torch.full((n, heads, d), float("nan"), dtype=q.dtype, device=DEV)
    spec = mx4.Kv4AttnSpec(nseq=n, tokens=n, hq=heads, hkv=cache[0].shape[1], d=d, page=16, pages=2, table_width=2,
                           dt=DType.F16, **kw)
    args = q[at], *cache, torch.arange(n + 1, dtype=torch.int32, device=DEV), i32([[1, 0]]).repeat(n, 1), i32(lens)[at], out
    times = []
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        spec.run(*args)
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return out, min(times)


def test_time_grows_with_the_sequences_and_not_with_their_square():
    hkv, d = 8, 32
    cache = noise_cache(1, 2, 16, hkv, d)
    for s in cache[1::2]:
        s.clamp_(120, 130)
    lens = [20, 1, 0, 32, 17, 9, 31, 3]
    q = torch.randn(8, 4 * hkv, d, generator=torch.Generator().manual_seed(2)).half().to(DEV)
    few, _ = run(8, q, lens, cache)
    some, t0 = run(1 << 14, q, lens, cache)
    many, t1 = run(1 << 17, q, lens, cache)
    for out in (some, many):
        assert torch.equal(out, few.repeat(len(out) // 8, 1, 1))
    assert t1 < 24 * t0, (t0, t1)  # 8 times the sequences; 64 times where each item counts them all


@pytest.mark.parametrize("dt", list(DType))
@pytest.mark.parametrize("d", [32, 96, 160])
def test_more_sequences_than_are_counted_at_once(d, dt):
    # 257 and more, some empty, some of several tiles, batches of 64 that hold nothing at all
    n = 300
    q_lens = [(7 * i) % 4 if i % 50 else 37 for i in range(n)]
    q_lens[64:128] = [0] * 64
    k_lens = [max(q, (13 * i) % 90) for i, q in enumerate(q_lens)]
    Case(d, q_lens, k_lens, 4, 2, d, dt).check()
