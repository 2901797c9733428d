"""CPU tests of the 4-bit cache attention's plan: where its routes change. Nothing here
launches a kernel; the plans are those of 256 CUs."""
import pytest

from ai_engine_amd import mx4
from ai_engine_amd.conv import DType


def plan(nseq, tokens, hq, hkv, d, keys, dt=DType.BF16, **kw):
    width = -(-keys // 64)
    return mx4.Kv4AttnSpec(**{**dict(
        nseq=nseq, tokens=tokens, hq=hq, hkv=hkv, d=d, page=64, pages=nseq * width, table_width=width, dt=dt,
        max_len=keys), **kw}).plan()


@pytest.mark.parametrize("dt", list(DType))
@pytest.mark.parametrize("nseq, tokens, hq, hkv, d, bm", [
    # 16 rows hold a sequence, 32 do, and more
    (128, 128, 32, 8, 128, 16), (128, 128 * 4, 32, 8, 128, 16), (128, 128 * 5, 32, 8, 128, 32),
    (256, 256 * 2, 64, 4, 64, 32), (1024, 1024, 32, 1, 128, 32), (512, 512, 32, 1, 96, 32), (128, 128 * 8, 32, 8, 128, 32),
    (128, 128 * 9, 32, 8, 128, 64), (4, 2224, 32, 8, 128, 64), (1, 4096, 32, 8, 64, 64), (4, 2224, 32, 8, 32, 32),
    (4, 2224, 32, 8, 256, 32), (1, 512, 32, 8, 128, 32)])
def test_rows_of_a_tile(nseq, tokens, hq, hkv, d, bm, dt):
    assert plan(nseq, tokens, hq, hkv, d, 1000, dt).bm == bm


@pytest.mark.parametrize("nseq, hq, hkv, d, keys, parts", [
    # single tokens: cut from 1024 keys on, heads of more than 128 from 512 on unless every CU has one
    (4, 16, 4, 256, 600, 3), (4, 16, 4, 256, 512, 1), (64, 16, 4, 256, 600, 1), (64, 16, 4, 256, 960, 1),
    (64, 8, 2, 192, 960, 4), (4, 16, 4, 128, 960, 1), (1, 16, 4, 128, 131072, 128), (64, 32, 8, 128, 8192, 8)])
def test_parts_of_the_keys(nseq, hq, hkv, d, keys, parts):
    assert plan(nseq, nseq, hq, hkv, d, keys).parts == parts
