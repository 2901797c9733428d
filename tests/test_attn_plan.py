"""CPU tests of the attention plan's figures and of where its routes change.
Nothing here launches a kernel; the plans are those of 256 CUs."""
import pytest

from ai_engine_amd.attn import AttnKernel, AttnSpec
from ai_engine_amd.conv import DType

ROWS, KEYS = AttnKernel.ROWS, AttnKernel.KEYS


def plan(**kw):
    return AttnSpec(**{**dict(nseq=1, tokens=1, rows=100, hq=8, hkv=2, d=64, dt=DType.F16), **kw}).plan()


def test_grid_without_a_prefix():
    # 64 x 720 tokens of 4 heads a group: 128 rows a tile and a tile more a sequence at most
    p = plan(nseq=64, tokens=64 * 720, rows=64 * 720)
    assert p.kernel == ROWS and p.grid == 2 * (64 * 720 * 4 // 128 + 64)
    # cut keys: every part of every sequence's tile
    p = plan(nseq=64, tokens=64, rows=64 * 8192, hq=32, hkv=8, d=128, max_len=8192)
    assert p.kernel == KEYS and p.grid == 8 * (64 * 4 // 32 + 64) * p.parts


def test_grid_with_a_prefix_in_the_same_launch():
    p = plan(nseq=6, tokens=12, rows=6 * 77, prefix=720)
    assert (p.kernel, p.prefix_kernel) == (KEYS, KEYS)
    own, pre = 2 * (12 * 4 // 32 + 6) * p.parts, 2 * 2 * p.prefix_parts  # 48 rows: two tiles
    assert p.grid == own + pre


def test_grid_with_a_prefix_of_its_own_launch():
    p = plan(nseq=3, tokens=190, rows=265, max_len=200, hq=4, prefix=1300)
    assert (p.kernel, p.prefix_kernel) == (ROWS, ROWS)
    assert p.grid == 2 * 3 * p.prefix_parts  # 380 rows: three tiles


def test_nothing_to_do_has_no_grid():
    assert plan(nseq=0).grid == 0 and plan(tokens=0, prefix=9).grid == 0


# ---------------------------------------------------------------- where routes change: the side that measured faster

H = dict(f32=DType.F32, f16=DType.F16, bf16=DType.BF16)


@pytest.mark.parametrize("dt, nseq, keys, hq, hkv, d, parts", [
    ("f16", 1, 512, 32, 8, 128, 1), ("f16", 1, 1024, 32, 8, 128, None), ("bf16", 1, 4096, 32, 8, 128, None),
    ("f16", 16, 1024, 32, 8, 128, 1), ("f16", 16, 2048, 32, 8, 128, 2), ("f16", 4, 600, 16, 4, 256, None),
    ("f16", 16, 600, 16, 4, 256, 1), ("f32", 1, 384, 8, 2, 64, 1), ("f32", 1, 512, 8, 2, 64, None),
    ("f32", 1, 271, 16, 4, 256, None), ("f32", 40, 600, 4, 4, 32, 1), ("f32", 8, 2000, 18, 3, 256, 8),
    ("f32", 16, 2000, 32, 8, 64, 4)])
def test_single_tokens_are_cut_where_it_pays(dt, nseq, keys, hq, hkv, d, parts):
    p = plan(nseq=nseq, tokens=nseq, rows=nseq * keys, max_len=keys, hq=hq, hkv=hkv, d=d, dt=H[dt])
    assert p.kernel == KEYS
    assert p.parts == parts if parts else p.parts > 1


@pytest.mark.parametrize("dt, nseq, n, hq, hkv, d, kernel, cut", [
    ("f16", 1, 1500, 4, 4, 64, KEYS, False), ("f32", 1, 1024, 4, 4, 64, KEYS, True),
    ("f32", 1, 300, 16, 4, 256, KEYS, False), ("f32", 1, 4096, 16, 4, 96, KEYS, False),
    ("f32", 4, 2048, 16, 4, 96, KEYS, False), ("f32", 16, 720, 16, 4, 96, ROWS, False),
    ("f16", 1, 2880, 8, 2, 64, KEYS, False), ("f16", 1, 2880, 16, 4, 128, ROWS, False),
    ("f16", 40, 100, 8, 2, 128, ROWS, False), ("f32", 4, 100, 16, 4, 128, KEYS, False),
    ("f32", 40, 64, 16, 4, 128, ROWS, False), ("f32", 8, 260, 16, 4, 128, KEYS, False),
    ("f32", 20, 300, 16, 4, 128, ROWS, False), ("f32", 3, 700, 16, 4, 128, KEYS, False),
    ("bf16", 1, 520, 8, 4, 256, KEYS, False), ("bf16", 2, 900, 8, 4, 256, KEYS, False),
    ("bf16", 8, 260, 8, 4, 256, ROWS, False), ("bf16", 6, 520, 8, 4, 256, ROWS, False),
    ("bf16", 1, 3000, 8, 4, 256, ROWS, False)])
def test_prompts_take_the_faster_kernel(dt, nseq, n, hq, hkv, d, kernel, cut):
    p = plan(nseq=nseq, tokens=nseq * n, rows=nseq * n, max_len=n, hq=hq, hkv=hkv, d=d, dt=H[dt])
    assert p.kernel == kernel and (p.parts > 1) == cut


@pytest.mark.parametrize("dt, nseq, lq, prefix, hq, hkv, d, kernel, parts", [
    ("bf16", 64, 1, 4096, 32, 8, 128, KEYS, 4), ("bf16", 64, 4, 4096, 12, 2, 128, KEYS, None),
    ("bf16", 64, 4, 8000, 12, 2, 128, KEYS, None), ("bf16", 64, 4, 8000, 8, 2, 64, KEYS, None),
    ("bf16", 64, 4, 24000, 8, 2, 64, ROWS, None), ("bf16", 64, 1, 24000, 32, 8, 128, ROWS, None),
    ("bf16", 16, 4, 24000, 16, 4, 256, ROWS, None), ("bf16", 16, 4, 60000, 16, 4, 256, ROWS, None),
    ("f32", 5, 1, 651, 16, 4, 256, KEYS, 6), ("f32", 64, 4, 24000, 32, 8, 64, KEYS, None)])
def test_a_prefix_takes_the_faster_kernel(dt, nseq, lq, prefix, hq, hkv, d, kernel, parts):
    p = plan(nseq=nseq, tokens=nseq * lq, rows=nseq * 134, max_len=134, hq=hq, hkv=hkv, d=d, dt=H[dt], prefix=prefix)
    assert p.kernel == KEYS and p.prefix_kernel == kernel
    assert p.prefix_parts == parts if parts else True
