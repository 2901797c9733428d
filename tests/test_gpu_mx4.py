"""GPU tests of microscaled 4-bit rows and their pointwise conv, against the format
and the product in 64 bits. Codes, scales and values are exact and have to be equal."""
import pytest
import torch

from ai_engine_amd import mx4
from ai_engine_amd.conv import AihError, Activation, DType
from tests.mx4_util import DTS, IDS, TORCH, quant_rows, row_buffers, values

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def some_rows(seed, rows, k, dt):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    return x.to(TORCH[dt])


def check_quant(x, dt, x_stride=0):
    """x [rows, k] on the host; the rows on the GPU `x_stride` apart, NaN in between."""
    rows, k = x.shape
    if x_stride:
        wide = torch.full((rows, x_stride), float("nan"), dtype=x.dtype)
        wide[:, :k] = x
        xd = wide.to(DEV)
    else:
        xd = x.to(DEV)
    codes, scales = row_buffers(rows, k)
    mx4.Mx4QuantSpec(rows=rows, k=k, dt=dt, x_stride=x_stride).run(xd, codes, scales)
    want_c, want_s = quant_rows(x)
    blocks = want_s.shape[1]
    assert torch.equal(codes.cpu(), want_c)
    assert torch.equal(scales.cpu()[:, :blocks], want_s)
    assert (scales.cpu()[:, blocks:] == 0x77).all()  # of no element: left as they were
    return codes, scales


def check_dequant(codes, scales, k, dt, y_stride=0, **strides):
    rows = codes.shape[0]
    y = torch.full((rows, y_stride or k), -77.0, dtype=TORCH[dt], device=DEV)
    mx4.Mx4DequantSpec(rows=rows, k=k, dt=dt, y_stride=y_stride, **strides).run(codes, scales, y)
    want = values(codes, scales)[:, :k].to(TORCH[dt])
    got = y.cpu()
    assert torch.equal(torch.isnan(got[:, :k]), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got[:, :k]), torch.nan_to_num(want))
    assert (got[:, k:] == -77.0).all()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("rows, k, stride", [
    (1, 4, 0), (1, 32, 0), (3, 36, 0), (7, 128, 0), (5, 132, 0), (9, 260, 264), (33, 960, 0), (4, 1000, 1004),
    (2, 4096, 8192), (300, 20, 0), (64, 516, 0), (1, 8196, 0)])
def test_rows(rows, k, stride, dt):
    codes, scales = check_quant(some_rows(rows + k, rows, k, dt), dt, stride)
    check_dequant(codes, scales, k, dt, stride)


@pytest.mark.parametrize("dt", DTS, ids=IDS)
def test_every_border(dt):
    # all values a block can round, at every scale that the type has, one ulp to either side too
    t = TORCH[dt]
    grid = torch.tensor([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.9])
    lo, hi = {DType.F32: (-149, 125), DType.F16: (-24, 12), DType.BF16: (-133, 125)}[dt]
    rows = []
    for e in range(lo, hi):
        v = torch.ldexp(grid.double(), torch.tensor(e)).to(t)
        up = torch.nextafter(v, torch.tensor(float("inf"), dtype=t))
        down = torch.nextafter(v, torch.tensor(0.0, dtype=t))
        for w in (v, up, down, -up, -down):
            block = torch.zeros(64, dtype=t)
            block[:17] = w
            block[32:49] = w * 0.5
            rows.append(block)
    check_quant(torch.stack(rows), dt)


@pytest.mark.parametrize("dt", DTS, ids=IDS)
def test_nan_inf_zero_and_subnormal_blocks(dt):
    t = TORCH[dt]
    x = some_rows(3, 12, 132, dt)
    x[0, 5], x[1, 40], x[2, 131], x[3] = float("nan"), float("inf"), float("-inf"), 0
    x[4] = -0.0
    x[5], x[6, 64:96] = torch.finfo(t).smallest_normal / 4, torch.finfo(t).max
    codes, scales = check_quant(x, dt)
    assert scales[0, 0] == 255 and scales[1, 1] == 255 and scales[2, 4] == 255
    check_dequant(codes, scales, 132, dt)


@pytest.mark.parametrize("dt", DTS, ids=IDS)
def test_every_code_and_scale_reads_back(dt):
    codes = torch.arange(256, dtype=torch.uint8).repeat(2)[None].repeat(253, 1)  # 1024 elements a row
    scales = torch.arange(253, dtype=torch.uint8)[:, None].repeat(1, 32)
    check_dequant(codes.to(DEV), scales.to(DEV), 1024, dt)


def test_rows_of_a_cache_read_back():
    # rows of 96 elements without the padding: 48 bytes of codes, 3 scales
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (50, 48), generator=g, dtype=torch.uint8).to(DEV)
    scales = torch.randint(100, 140, (50, 3), generator=g, dtype=torch.uint8).to(DEV)
    check_dequant(codes, scales, 96, DType.BF16, code_stride=48, scale_stride=3)


# ---------------------------------------------------------------- the product

def make_pw(seed, m, k, cout, dt, residual):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))).to(TORCH[dt]).to(DEV)
    w = (torch.randn(cout, k, generator=g) / k ** 0.5).to(TORCH[dt]).to(DEV)
    b = torch.randn(cout, generator=g).to(TORCH[dt]).to(DEV)
    r = torch.randn(m, cout, generator=g).to(TORCH[dt]).to(DEV) if residual else None
    xq, wq = row_buffers(m, k), row_buffers(cout, k)
    mx4.Mx4QuantSpec(rows=m, k=k, dt=dt).run(x, *xq)
    mx4.Mx4QuantSpec(rows=cout, k=k, dt=dt).run(w, *wq)
    return xq, wq, b, r


ACTS = {Activation.NONE: lambda v: v, Activation.RELU6: lambda v: v.clamp(0, 6),
        Activation.HARDSWISH: lambda v: v * ((v + 3).clamp(0, 6) / 6), Activation.SIGMOID: torch.sigmoid}


def check_pw(xq, wq, b, r, m, k, cout, dt, act=Activation.NONE, y=None, stream=None):
    if y is None:
        y = torch.full((m + 1, cout), float("nan"), dtype=TORCH[dt], device=DEV)
        y[m] = 5  # behind the last pixel
    mx4.Mx4PwSpec(m=m, k=k, cout=cout, act=act, residual=r is not None, dt=dt).run(*xq, *wq, b, r, y, stream=stream)
    torch.cuda.synchronize()
    xv, wv = values(*xq).to(DEV), values(*wq).to(DEV)
    s = xv @ wv.t().contiguous() + (0 if b is None else b.double())
    want = ACTS[act](s) + (0 if r is None else r.double())
    # A product of blocks is exact before its scale (multiples of 1/4 below 2^11). Each of the k / 32 blocks, the
    # joined parts (16) and the bias is added in fp32, an addition off by at most 2^-23 of the terms' magnitudes
    # (twice a rounding: the matrix unit may cut instead). The activations have a slope of at most 1.5 and are off
    # by a few units themselves, the residual is one more addition, the store half a step.
    mag = xv.abs() @ wv.abs().t().contiguous() + (0 if b is None else b.double().abs())
    tol = 1.5 * (k / 32 + 18) * 2.0 ** -23 * mag + 2.0 ** -20 * (ACTS[act](s).abs() + want.abs())
    tol = tol + want.abs() * torch.finfo(TORCH[dt]).eps / 2 + 1e-30
    got = y[:m].double()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()
    return y


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("m, k, cout", [
    (1, 4, 4), (1, 4096, 20), (16, 128, 16), (17, 132, 36), (33, 2048, 100), (64, 960, 160), (65, 260, 68),
    (100, 36, 4), (129, 1000, 132), (500, 516, 260), (1007, 1000, 724), (260, 4160, 64),
    (3, 70000, 8), (70, 70020, 8), (300, 2180, 300)])
def test_product(m, k, cout, dt):
    residual = (m + cout) % 3 == 0
    xq, wq, b, r = make_pw(m * k, m, k, cout, dt, residual)
    y = check_pw(xq, wq, b, r, m, k, cout, dt, act=Activation.HARDSWISH if m % 2 else Activation.RELU6)
    assert (y[m] == 5).all()


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("m", [5, 200])
def test_product_activations(m, act):
    xq, wq, b, r = make_pw(7, m, 512, 64, DType.F32, True)
    check_pw(xq, wq, b, r, m, 512, 64, DType.F32, act=act)
    check_pw(xq, wq, None, None, m, 512, 64, DType.F32, act=act)


@pytest.mark.parametrize("m, k, cout", [(4096, 256, 4100), (8200, 512, 2050 * 4), (33000, 128, 132), (70000, 64, 36)])
def test_product_of_many_tiles(m, k, cout):
    xq, wq, b, r = make_pw(9, m, k, cout, DType.BF16, False)
    check_pw(xq, wq, b, r, m, k, cout, DType.BF16)


@pytest.mark.parametrize("m", [9, 150])
def test_product_in_place_of_the_residual(m):
    xq, wq, b, r = make_pw(11, m, 256, 96, DType.F16, True)
    keep = r.clone()
    spec = mx4.Mx4PwSpec(m=m, k=256, cout=96, residual=True, dt=DType.F16)
    other = torch.empty_like(r)
    spec.run(*xq, *wq, b, keep, other)
    spec.run(*xq, *wq, b, r, r)
    assert torch.equal(r, other)


@pytest.mark.parametrize("m", [9, 150, 3000])
def test_nan_blocks_reach_their_pixels_and_channels_alone(m):
    xq, wq, b, _ = make_pw(13, m, 300, 72, DType.F32, False)
    good = torch.empty(m, 72, device=DEV)
    spec = mx4.Mx4PwSpec(m=m, k=300, cout=72, dt=DType.F32)
    spec.run(*xq, *wq, b, None, good)
    xq[1][3, 2], wq[1][10, 0], wq[1][71, 9] = 255, 255, 255
    y = torch.empty(m, 72, device=DEV)
    spec.run(*xq, *wq, b, None, y)
    bad = torch.zeros(m, 72, dtype=torch.bool, device=DEV)
    bad[3], bad[:, 10], bad[:, 71] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    assert torch.equal(y[~bad], good[~bad])


@pytest.mark.parametrize("m", [8, 400])
def test_captured_and_replayed(m):
    k, cout, dt = 640, 320, DType.BF16
    x = some_rows(1, m, k, dt).to(DEV)
    _, wq, b, _ = make_pw(2, m, k, cout, dt, False)
    xq, y = row_buffers(m, k), torch.empty(m, cout, dtype=TORCH[dt], device=DEV)
    quant, pw = mx4.Mx4QuantSpec(rows=m, k=k, dt=dt), mx4.Mx4PwSpec(m=m, k=k, cout=cout, dt=dt)

    def both():
        quant.run(x, *xq)
        pw.run(*xq, *wq, b, None, y)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for i in range(3):
        x.copy_(some_rows(10 + i, m, k, dt))
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = y.clone()
        both()
        assert torch.equal(y, replayed)


def test_two_streams_at_once():
    xq, wq, b, _ = make_pw(21, 700, 512, 260, DType.F16, False)
    spec = mx4.Mx4PwSpec(m=700, k=512, cout=260, dt=DType.F16)
    want = torch.empty(700, 260, dtype=torch.float16, device=DEV)
    spec.run(*xq, *wq, b, None, want)
    torch.cuda.synchronize()
    streams, ys = [torch.cuda.Stream() for _ in range(2)], [torch.empty_like(want) for _ in range(2)]
    for _ in range(5):
        for s, y in zip(streams, ys):
            spec.run(*xq, *wq, b, None, y, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in ys)


def test_short_strided_and_other_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=torch.float16, device=DEV)
    c, s = row_buffers(4, 64)
    spec = mx4.Mx4QuantSpec(rows=4, k=64, dt=DType.F16)
    spec.run(x, c, s)
    for bad in (x[:3], x.float(), x.t(), x.cpu()):
        with pytest.raises(AihError, match="x must be a dense tensor"):
            spec.run(bad, c, s)
    for bad in (c[:3], c.to(torch.int8), c.cpu()):
        with pytest.raises(AihError, match="codes must be a dense tensor"):
            spec.run(x, bad, s)


@pytest.mark.parametrize("m, k, cout", [
    (1, 100, 40), (20, 2100, 36), (200, 1000, 64), (300, 2100, 300), (1100, 2100, 2100), (2000, 2100, 2500), (4096, 2176, 4096)])
def test_scales_of_no_element_do_not_count(m, k, cout):
    # an odd number of 128s, every size of tile; what is behind a row's scales reads as NaN
    xq, wq, b, r = make_pw(17, m, k, cout, DType.BF16, False)
    for q in (xq, wq):
        q[1][:, -(-k // 128) * 4:] = 255
    check_pw(xq, wq, b, r, m, k, cout, DType.BF16)


def test_a_row_is_its_own():
    # the same pixels among others, in another place and in another number of them: the same tile, the same bits
    xq, wq, b, _ = make_pw(19, 700, 1024, 200, DType.F32, False)
    y = check_pw(xq, wq, b, None, 700, 1024, 200, DType.F32)[:700]
    at = torch.randperm(700, generator=torch.Generator().manual_seed(1)).to(DEV)
    other = torch.empty_like(y)
    mx4.Mx4PwSpec(m=700, k=1024, cout=200).run(xq[0][at].contiguous(), xq[1][at].contiguous(), *wq, b, None, other)
    assert torch.equal(other, y[at])


def test_rows_and_results_beyond_4_gib():
    rows, k, cout, dt = (1 << 21) + 37, 1024, 1024, DType.BF16
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV)
    x[-200:] = some_rows(1, 200, k, dt).to(DEV)
    assert x.numel() * 2 > 1 << 32
    codes, scales = row_buffers(rows, k)
    mx4.Mx4QuantSpec(rows=rows, k=k, dt=dt).run(x, codes, scales)
    want_c, want_s = quant_rows(x[-200:].cpu())
    assert torch.equal(codes[-200:].cpu(), want_c) and torch.equal(scales[-200:].cpu()[:, :want_s.shape[1]], want_s)
    assert not codes[:-200].any()
    x.fill_(7.0)
    mx4.Mx4DequantSpec(rows=rows, k=k, dt=dt).run(codes, scales, x)
    assert torch.equal(x[-200:].cpu(), values(codes[-200:], scales[-200:]).bfloat16()) and not x[:-200].any()
    # the product of the same rows: the last ones among all are the same as alone
    w = some_rows(2, cout, k, dt).to(DEV)
    wq = row_buffers(cout, k)
    mx4.Mx4QuantSpec(rows=cout, k=k, dt=dt).run(w, *wq)
    x.fill_(7.0)
    mx4.Mx4PwSpec(m=rows, k=k, cout=cout, dt=dt).run(codes, scales, *wq, None, None, x)
    assert not x[:-200].any()
    check_pw((codes[-200:].contiguous(), scales[-200:].contiguous()), wq, None, None, 200, k, cout, dt)
    alone = torch.empty(200, cout, dtype=torch.bfloat16, device=DEV)
    mx4.Mx4PwSpec(m=200, k=k, cout=cout, dt=dt).run(codes[-200:].contiguous(), scales[-200:].contiguous(), *wq, None, None, alone)
    # sums of the same blocks in another order: a few roundings of fp32 each, and one of the store
    assert ((x[-200:].float() - alone.float()).abs() <= 2.0 ** -7 * alone.float().abs() + 1e-3 * alone.float().abs().max()).all()
