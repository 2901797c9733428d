"""CPU tests of the attention plan's figures.
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
