"""CPU tests of the 4-bit operators' largest sizes: a launch takes less than 2^32 threads, and
what would need more is refused by a message that says so. Nothing here launches a kernel."""
import pytest

from ai_engine_amd.conv import AihError, DType
from tests.test_kv4 import append, run as run_kv
from tests.test_kv4_plan import plan
from tests.test_mx4 import dequant, pw, quant, run


@pytest.mark.parametrize("make, kw, msg", [
    (quant, dict(rows=(1 << 28) - 1, k=128), "2\\^35 - 2048"), (quant, dict(rows=(1 << 28) - 15, k=4), "2\\^35 - 2048"),
    (dequant, dict(rows=(1 << 32) - 1, k=8), "2\\^35 - 2048"), (dequant, dict(rows=(1 << 32) - 255, k=4), "2\\^35 - 2048"),
    (pw, dict(m=(1 << 31) - 255), "2\\^31 - 256"), (pw, dict(m=(1 << 31) - 1), "2\\^31 - 256")])
def test_rows(make, kw, msg):
    with pytest.raises(AihError, match=msg):
        run(make(**kw))


@pytest.mark.parametrize("make, kw", [
    (quant, dict(rows=(1 << 28) - 16, k=128)), (dequant, dict(rows=(1 << 32) - 256, k=8)), (pw, dict(m=(1 << 31) - 256))])
def test_the_largest_are_asked_further(make, kw):
    with pytest.raises(AihError, match="aligned"):
        run(make(**kw), **{"codes" if make is not pw else "y": (1 << 20) + 4})


@pytest.mark.parametrize("d", [32, 96, 128, 256])
def test_appended_heads(d):
    most = ((1 << 24) - 1) * 4 * (512 // d)
    sizes = dict(hq=0, hkv=1, d=d, rot=0)
    with pytest.raises(AihError, match="tokens \\* \\(hq"):
        run_kv(append(tokens=most // 2 + 1, **sizes))
    with pytest.raises(AihError, match="aligned"):
        run_kv(append(tokens=most // 2, **sizes), x=(1 << 20) + 4)


def test_keys_of_very_many_rows_are_not_cut():
    # what joins the parts takes up to 1024 threads a row
    sizes = dict(hq=32, hkv=8, d=64, keys=16384, dt=DType.F16, pages=1000)
    assert plan(1 << 17, (1 << 17) - 1, **sizes).parts > 1
    p = plan(1 << 17, 1 << 17, **sizes)
    assert p.parts == 1 and p.ws_bytes == 0
