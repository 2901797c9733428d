"""GPU tests of attention over the 4-bit cache in tiles of 64 rows, which take whole prompts
of many heads: every such kernel against the formula in 64 bits, with its plan asserted."""
import pytest
import torch

from tests.mx4_util import DTS, IDS
from tests.test_gpu_kv4 import Case

pytestmark = pytest.mark.gpu

HEADS = [(64, 64), (64, 32), (96, 32), (32, 8)]  # 1, 2, 3 and 4 queries a key head; 3 does not divide 64


def prompts(seed, d, dt, hq, hkv, causal=True, **kw):
    """Sequences of odd lengths, some behind earlier keys, that make two tiles of 64 rows a CU."""
    g = hq // hkv
    q = [70, 1, 0, 131, 64, 3, 97, 40]
    k = [70, 5, 33, 200, 64, 3, 300, 0] if causal else [1, 50, 33, 200, 64, 90, 300, 0]
    while (sum(q) * g // 64 + len(q) // 2) * hkv < 512 or sum(q) * g <= 32 * len(q):
        q.append(37 + 5 * (len(q) % 9))
        k.append(q[-1] + 16 * (len(q) % 3))
    c = Case(seed, q, k, hq, hkv, d, dt, causal=causal, **kw)
    assert c.spec().plan().bm == 64
    return c


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d, heads", [(64, 0), (96, 1), (128, 3), (64, 2), (128, 2)])
def test_prompts(d, heads, causal, dt):
    prompts(d + heads, d, dt, *HEADS[heads], causal=causal, page=16 if causal else 32, pad=8).check()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("d, heads", [(64, 1), (96, 2), (128, 1)])
def test_nan_blocks_and_pages_outside_the_cache(d, heads, dt):
    c = prompts(7 + d, d, dt, *HEADS[heads])
    # of a sequence's keys and values some blocks are NaN: near the end, where few rows see them, and in the middle
    for b, j, head, block, which in [(0, 69, 0, 0, 1), (0, 60, 1, d // 32 - 1, 0), (3, 150, 2, d // 32 - 1, 1),
                                     (3, 199, 0, 1, 1), (6, 299, 3, 0, 0), (6, 280, 0, d // 32 - 1, 1)]:
        c.cache[2 * which + 1][c.table[b, j // 16], head, j % 16, block] = 255
    c.table[4, 1], c.table[4, 3], c.table[6, 2], c.table[6, 17] = -1, c.pages, 1 << 30, -5
    want, _ = c.want()
    assert torch.isnan(want).any() and not torch.isnan(want).all()
    c.check()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("d", [64, 96, 128])
def test_keys_that_were_not_foreseen(d, dt):
    # max_len is a guess: the lengths are the arrays', and the table's end cuts them
    c = prompts(9 + d, d, dt, 64, 32)
    c.check(spec=c.spec(max_len=1))
    c.check(spec=c.spec(max_len=0))


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("d", [64, 96, 128])
def test_the_same_rows_in_tiles_of_32(d, dt):
    # half of the sequences alone are too few for tiles of 64; the same keys in the same order either way
    c = prompts(11 + d, d, dt, 64, 32)
    got = c.run()
    few = Case.__new__(Case)
    few.__dict__ = dict(c.__dict__)
    n = len(c.q_lens) // 4
    few.q_lens, few.k_lens = c.q_lens[:n], c.k_lens[:n]
    few.q_start, few.table = c.q_start[:n + 1], c.table[:n]
    few.tokens, few.q = c.q_start[n], c.q[:c.q_start[n]]
    assert few.spec().plan().bm == 32
    few.check()
    want, tol = c.want()
    a, b = few.run().double(), got[:few.tokens].double()
    assert ((a - b).abs() <= 2 * tol[:few.tokens]).all()
