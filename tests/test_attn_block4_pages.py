"""CPU tests of the sizes that an attention block with a 4-bit cache refuses when it is
made, not at its first step. Nothing here launches a kernel."""
import pytest

from ai_engine_amd.conv import AihError
from tests.test_attn_block4 import make_block


@pytest.mark.parametrize("page", [0, 8, 24, 48, 8192, -16, 16.0, True, None])
def test_pages(page):
    with pytest.raises(AihError, match="4-bit cache takes pages"):
        make_block(cache4=True, page=page)
    make_block(page=page)  # of no meaning without that cache


@pytest.mark.parametrize("d", [288, 512])
def test_heads(d):
    with pytest.raises(AihError, match="4-bit cache takes heads"):
        make_block(cache4=True, d=d)


@pytest.mark.parametrize("page", [16, 4096])
def test_ends_of_the_range(page):
    assert make_block(cache4=True, page=page).cache[0].shape[2] == page
