"""GPU tests of the 4-bit pointwise conv's tiles, each in every type with residual and
activation, partial tiles on both sides, and rows of 8- and 16-byte alignment; and of scales
far from one. The sizes fall to the tiles named beside them on 256 CUs."""
import pytest
import torch

from ai_engine_amd import mx4
from ai_engine_amd.conv import Activation, DType
from tests.mx4_util import DTS, IDS, TORCH, row_buffers, values
from tests.test_gpu_mx4 import DEV, check_pw, make_pw

pytestmark = pytest.mark.gpu

TILES = [
    # whole 128s of k odd and even; channels of 8-byte and of 16-byte rows
    ("256x256", 4000, 2048, 4012), ("256x256", 3900, 2100, 4016),
    ("128x128", 2000, 2176, 2500), ("128x128", 1990, 2048, 2504),
    ("64x128", 1100, 2100, 2100), ("64x128", 1111, 2048, 2104),
    ("64x64", 300, 2100, 300), ("64x64", 333, 2048, 328),
    ("128x128 of short stages", 4000, 1000, 1100), ("128x128 of short stages", 4010, 260, 1104),
    ("64x64 of short stages", 500, 1000, 332), ("64x64 of short stages", 501, 132, 328),
    ("few, 16 wavefronts", 13, 4100, 1004), ("few, 4 wavefronts", 31, 1000, 2004)]


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("tile, m, k, cout", TILES, ids=lambda v: str(v).replace(" ", "_"))
def test_tiles(tile, m, k, cout, dt):
    xq, wq, b, r = make_pw(m + k, m, k, cout, dt, True)
    y = check_pw(xq, wq, b, r, m, k, cout, dt, act=Activation.RELU6)
    assert (y[m] == 5).all()
    y = check_pw(xq, wq, None, None, m, k, cout, dt)
    assert (y[m] == 5).all()


@pytest.mark.parametrize("tile, m, k, cout", TILES, ids=lambda v: str(v).replace(" ", "_"))
def test_nan_blocks(tile, m, k, cout):
    xq, wq, b, _ = make_pw(13, m, k, cout, DType.F16, False)
    good = torch.empty(m, cout, dtype=torch.float16, device=DEV)
    spec = mx4.Mx4PwSpec(m=m, k=k, cout=cout, act=Activation.HARDSWISH, dt=DType.F16)
    spec.run(*xq, *wq, b, None, good)
    last = -(-k // 32) - 1
    xq[1][3, 2], xq[1][m - 1, last], wq[1][1, 0], wq[1][cout - 1, last] = 255, 255, 255, 255
    y = torch.empty_like(good)
    spec.run(*xq, *wq, b, None, y)
    bad = torch.zeros(m, cout, dtype=torch.bool, device=DEV)
    bad[3], bad[m - 1], bad[:, 1], bad[:, cout - 1] = True, True, True, True
    assert torch.equal(torch.isnan(y), bad)
    assert torch.equal(y[~bad], good[~bad])


@pytest.mark.parametrize("tile, m, k, cout", [t for t in TILES if t[2] != 2048], ids=lambda v: str(v).replace(" ", "_"))
def test_scales_of_no_element_do_not_count(tile, m, k, cout):
    xq, wq, b, r = make_pw(17, m, k, cout, DType.F16, True)
    for q in (xq, wq):
        q[1][:, -(-k // 128) * 4:] = 255
    check_pw(xq, wq, b, r, m, k, cout, DType.F16)


# ---------------------------------------------------------------- scales far from one

def moved(rows, by):
    """The scales of rows (codes, scales) moved by a power of two; those of no element stay."""
    scales = rows[1]
    k_blocks = rows[0].shape[1] // 16
    s = scales[:, :k_blocks].int()
    live = s > 0
    s = torch.where(live, s + by, s)
    assert s.min() >= 0 and s.max() <= 252
    scales[:, :k_blocks] = s.to(torch.uint8)
    return rows


@pytest.mark.parametrize("m, k, cout", [(9, 512, 64), (200, 1000, 96), (300, 2100, 300), (1111, 2048, 2104)])
@pytest.mark.parametrize("ex, ew", [(110, -110), (-108, 112), (60, 50), (-40, -50), (0, 100), (-112, 0)])
def test_scales_far_from_one(ex, ew, m, k, cout):
    # blocks of scales near either end of the range: products in the range of fp32 are what they were, times the
    # powers of two
    dt = DType.F32
    xq, wq, _, _ = make_pw(m + cout, m, k, cout, dt, False)
    base = torch.empty(m, cout, device=DEV)
    spec = mx4.Mx4PwSpec(m=m, k=k, cout=cout, dt=dt)
    spec.run(*xq, *wq, None, None, base)
    for q, e in ((xq, ex), (wq, ew)):
        q[1][:, -(-k // 32):] = 0
        moved(q, e)
    y = torch.empty_like(base)
    spec.run(*xq, *wq, None, None, y)
    assert torch.equal(y.double(), base.double() * 2.0 ** (ex + ew))


@pytest.mark.parametrize("m, k, cout", [(9, 512, 64), (200, 1000, 96), (300, 2100, 300), (1111, 2048, 2104)])
@pytest.mark.parametrize("bx, bw", [(0, 252), (252, 0), (1, 251), (120, 240), (3, 124)])
def test_the_ends_of_the_scales(bx, bw, m, k, cout):
    # one scale for all blocks: exact sums of exact products, in whichever order
    g = torch.Generator().manual_seed(m)
    xq, wq = row_buffers(m, k), row_buffers(cout, k)
    for (codes, scales), rows, byte in ((xq, m, bx), (wq, cout, bw)):
        # magnitudes of 2 at most and few of them: multiples of 1/4 whose sums stay far below 2^22
        c = torch.randint(0, 5, (rows, k), generator=g) + 8 * torch.randint(0, 2, (rows, k), generator=g)
        wide = torch.zeros(rows, 2 * codes.shape[1], dtype=torch.long)
        wide[:, :k] = c
        codes.copy_((wide[:, 0::2] | wide[:, 1::2] << 4).to(torch.uint8))
        scales.fill_(0)
        scales[:, :-(-k // 32)] = byte
    y = torch.empty(m, cout, device=DEV)
    mx4.Mx4PwSpec(m=m, k=k, cout=cout).run(*xq, *wq, None, None, y)
    want = values(*xq).to(DEV) @ values(*wq).to(DEV).t().contiguous()
    if (want.abs() < 2.0 ** -126).any():  # below the normal numbers fp32 has multiples of 2^-149
        assert ((y.double() - want).abs() <= 2.0 ** -149 * k).all()
    else:
        assert torch.equal(y.double(), want)
