"""CPU tests of what an attention block in 4 bits refuses. Nothing here launches a kernel."""
import numpy as np
import pytest

from ai_engine_amd.attn_block import AttnBlock
from ai_engine_amd.conv import AihError, DType


def make_block(d=32, hq=4, hkv=2, c=64, **kw):
    z = lambda *s: np.zeros(s, np.float32)
    w = dict(w_qkv=z((hq + 2 * hkv) * d, c), b_qkv=z((hq + 2 * hkv) * d), w_out=z(c, hq * d), b_out=z(c), wq=z(d), wk=z(d))
    return AttnBlock(c, hq, hkv, d, streams=3, capacity=40, weights=w, dt=DType.BF16, device="cpu", **kw)


@pytest.mark.parametrize("kw", [dict(d=40), dict(rot=8), dict(rot=24), dict(prefix=4)])
def test_refused(kw):
    with pytest.raises(AihError, match="4-bit cache"):
        make_block(cache4=True, **kw)


def test_pages():
    b = make_block(cache4=True, page=16)
    assert b.table.tolist() == [[0, 1, 2], [3, 4, 5], [6, 7, 8]] and b._first.tolist() == [0, 48, 96]
    assert [tuple(c.shape) for c in b.cache] == [(9, 2, 16, 16), (9, 2, 16, 1)] * 2
