"""CPU tests of the 4-bit operators' boundary: what is refused and with which
message. Nothing here launches a kernel."""
import ctypes as C

import pytest
import torch

from ai_engine_amd import conv, mx4
from ai_engine_amd.conv import AihError, Activation, DType
from tests.mx4_util import blocks_of, pack, quant_rows, values

FAKE = 1 << 20  # a 16-byte aligned address that no refused call touches
BIG = (1 << 20) + 4


def quant(**kw):
    return mx4.Mx4QuantSpec(**{**dict(rows=4, k=64, dt=DType.F16), **kw})


def dequant(**kw):
    return mx4.Mx4DequantSpec(**{**dict(rows=4, k=64, dt=DType.F16), **kw})


def pw(**kw):
    return mx4.Mx4PwSpec(**{**dict(m=4, k=64, cout=32, dt=DType.F16), **kw})


def run(spec, **kw):
    names = {mx4.Mx4QuantSpec: ("x", "codes", "scales"), mx4.Mx4DequantSpec: ("codes", "scales", "y"),
             mx4.Mx4PwSpec: ("x_codes", "x_scales", "w_codes", "w_scales", "bias", "res", "y")}[type(spec)]
    return spec.run(*(kw.get(n, FAKE) for n in names), stream=0)


@pytest.mark.parametrize("make, kw, msg", [
    (quant, dict(k=0), "k must be"), (quant, dict(k=6), "k must be"), (quant, dict(k=BIG), "k must be"),
    (quant, dict(dt=7), "dtype"), (quant, dict(x_stride=60), "x_stride"), (quant, dict(x_stride=66), "x_stride"),
    (quant, dict(x_stride=1 << 23), "x_stride"), (quant, dict(rows=1 << 31), "2\\^35"),
    (dequant, dict(k=0), "k must be"), (dequant, dict(k=2), "k must be"), (dequant, dict(k=BIG), "k must be"),
    (dequant, dict(dt=-1), "dtype"), (dequant, dict(y_stride=8), "y_stride"), (dequant, dict(code_stride=16), "code_stride"),
    (dequant, dict(code_stride=40), "code_stride"), (dequant, dict(scale_stride=1), "scale_stride"),
    (dequant, dict(rows=1 << 31), "2\\^35"),
    (pw, dict(k=0), "k must be"), (pw, dict(k=30), "k must be"), (pw, dict(cout=0), "cout"), (pw, dict(cout=6), "cout"),
    (pw, dict(cout=BIG), "cout"), (pw, dict(m=1 << 31), "2\\^31"), (pw, dict(act=11), "activation"),
    (pw, dict(act=-1), "activation"), (pw, dict(dt=3), "dtype"),
])
def test_refused_sizes(make, kw, msg):
    with pytest.raises(AihError, match=msg):
        run(make(**kw))


@pytest.mark.parametrize("make", [quant, dequant, pw])
@pytest.mark.parametrize("bad", [-1, 1.0, 1 << 32, True])
def test_sizes_are_whole_numbers(make, bad):
    for name in ("m",) if make is pw else ("rows",):
        with pytest.raises(AihError, match=name):
            make(**{name: bad})


@pytest.mark.parametrize("make, names", [
    (quant, ("x", "codes", "scales")), (dequant, ("codes", "scales", "y")),
    (pw, ("x_codes", "x_scales", "w_codes", "w_scales", "y"))])
def test_null_and_unaligned(make, names):
    for name in names:
        with pytest.raises(AihError, match="NULL"):
            run(make(), **{name: None})
        if (make, name) != (dequant, "scales"):  # bytes, read one by one
            with pytest.raises(AihError, match="aligned"):
                run(make(), **{name: FAKE + 8})
    if make is pw:
        with pytest.raises(AihError, match="residual needs res"):
            run(pw(residual=True), res=None)
        for name in ("bias", "res"):
            with pytest.raises(AihError, match="aligned"):
                run(pw(residual=True), **{name: FAKE + 2})


def test_nothing_to_do():
    run(quant(rows=0), x=None, codes=None, scales=None)
    run(dequant(rows=0), codes=None, scales=None, y=None)
    run(pw(m=0), x_codes=None, x_scales=None, w_codes=None, w_scales=None, y=None)


@pytest.mark.parametrize("make, names", [
    (quant, ("x", "codes", "scales")), (dequant, ("codes", "scales", "y")),
    (pw, ("x_codes", "x_scales", "w_codes", "w_scales", "bias", "res", "y"))])
def test_tensors_on_the_host_are_refused(make, names, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(mx4, "_torch", None)
    kw = dict(residual=True) if make is pw else {}
    for name in names:
        values_of = name in ("x", "y", "bias", "res")
        t = torch.zeros(1 << 12, dtype=torch.float16 if values_of else torch.uint8)
        with pytest.raises(AihError, match=f"{name} must be a dense tensor"):
            run(make(**kw), **{name: t})
    monkeypatch.setattr(mx4, "_torch", None)


def test_null_descriptor():
    L = mx4.lib()
    for fn, n in ((L.aih_mx4_quant, 4), (L.aih_mx4_dequant, 4), (L.aih_mx4_pw, 8)):
        assert fn(None, *[None] * n) == -1
        assert "NULL descriptor" in conv.last_error()


def test_row_sizes():
    assert [mx4.code_bytes(k) for k in (4, 128, 132, 960)] == [64, 64, 128, 512]
    assert [mx4.scale_bytes(k) for k in (4, 512, 516, 960)] == [16, 16, 32, 32]
    assert quant(k=960).code_bytes == 512 and quant(k=960).scale_bytes == 32


def test_the_tests_own_format():
    # one block by hand: the largest is 5 -> 2^(2 - 2) = 1; ties go to the even code
    x = torch.zeros(32)
    x[:9] = torch.tensor([5.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -6.5, 7.9])
    c, s = blocks_of(x)
    assert s.item() == 127 and c[:9].tolist() == [6, 0, 2, 2, 4, 4, 6, 15, 7]
    assert values(pack(c)[None], s.view(1, 1))[0, :9].tolist() == [4, 0, 1, 1, 2, 2, 4, -6, 6]
    assert blocks_of(torch.zeros(32))[1].item() == 0
    assert blocks_of(torch.full((32,), 2.0 ** -127, dtype=torch.float64))[1].item() == 0
    assert blocks_of(torch.tensor([float("inf")] + [1.0] * 31))[1].item() == 255
    c, s = quant_rows(torch.ones(2, 36))
    assert c.shape == (2, 64) and s.shape == (2, 4) and (c[:, 18:] == 0).all()
