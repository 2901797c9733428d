"""GPU tests of 4-bit calls with more work items than a launch has workgroups of 256 threads,
2^24 - 1."""
import pytest
import torch

from ai_engine_amd import mx4
from ai_engine_amd.conv import DType
from tests.mx4_util import row_buffers
from tests.test_gpu_kv4 import DEV, i32, noise_cache

pytestmark = pytest.mark.gpu


def test_attention_of_more_items_than_workgroups():
    n, heads, d, page = 4097, 4096, 32, 16
    assert n * heads > (1 << 24) - 1
    cache = noise_cache(1, 2, page, heads, d)
    for s in cache[1::2]:
        s.clamp_(120, 130)
    g = torch.Generator().manual_seed(2)
    q1 = torch.randn(8, heads, d, generator=g).bfloat16().to(DEV)
    lens = [20, 1, 0, 32, 17, 9, 31, 3]
    table = i32([[1, 0]])
    spec = lambda b: mx4.Kv4AttnSpec(nseq=b, tokens=b, hq=heads, hkv=heads, d=d, page=page, pages=2, table_width=2, dt=DType.BF16)
    few, out = torch.empty_like(q1), torch.full((n, heads, d), float("nan"), dtype=torch.bfloat16, device=DEV)
    spec(8).run(q1, *cache, i32(list(range(9))), table.repeat(8, 1), i32(lens), few)
    at = torch.arange(n, device=DEV) % 8
    spec(n).run(q1[at], *cache, torch.arange(n + 1, dtype=torch.int32, device=DEV), table.repeat(n, 1), i32(lens)[at], out)
    assert torch.isfinite(few).all() and (few[0] != 0).any()
    for i in range(8):  # a tile of 16 rows each: the same bits
        assert torch.equal(out[i::8], few[i:i + 1].expand(len(out[i::8]), -1, -1))


def test_product_of_more_pixels_than_workgroups_of_64():
    m, k, cout, dt = (1 << 30) + 37, 32, 4, DType.BF16
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of device memory")
    codes = torch.zeros(m, 64, dtype=torch.uint8, device=DEV)
    scales = torch.zeros(m, 16, dtype=torch.uint8, device=DEV)
    wq = row_buffers(cout, k)
    w = torch.randn(cout, k, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    mx4.Mx4QuantSpec(rows=cout, k=k, dt=dt).run(w, *wq)
    codes[-100:, :16], scales[-100:] = torch.arange(1600, device=DEV).view(100, 16).to(torch.uint8), 127
    scales[:-100] = 127
    y = torch.full((m + 1, cout), 5.0, dtype=torch.bfloat16, device=DEV)
    mx4.Mx4PwSpec(m=m, k=k, cout=cout, dt=dt).run(codes, scales, *wq, None, None, y)
    alone = torch.empty(100, cout, dtype=torch.bfloat16, device=DEV)
    mx4.Mx4PwSpec(m=100, k=k, cout=cout, dt=dt).run(codes[-100:].contiguous(), scales[-100:].contiguous(), *wq, None, None, alone)
    assert not y[:m - 100].any() and (y[m] == 5).all()
    assert torch.equal(y[m - 100:m], alone)  # one block a row: sums of one order
    del codes, scales, y
    torch.cuda.empty_cache()
