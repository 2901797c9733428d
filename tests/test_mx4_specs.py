"""CPU test that the 4-bit operators' specs copy and pickle. Nothing here launches a kernel."""
import copy
import ctypes as C
import pickle

import pytest

from ai_engine_amd import mx4
from ai_engine_amd.conv import Activation, AihError, DType

SPECS = [
    mx4.Mx4QuantSpec(rows=5, k=96, dt=DType.F16, x_stride=100), mx4.Mx4DequantSpec(rows=5, k=96, code_stride=48, scale_stride=3),
    mx4.Mx4PwSpec(m=7, k=96, cout=40, act=Activation.RELU6, residual=True, dt=DType.BF16),
    mx4.Kv4AppendSpec(tokens=4, hq=4, hkv=2, d=64, page=32, pages=8, rot=64, positions=9, norm=True, eps=1e-5),
    mx4.Kv4AttnSpec(nseq=1, tokens=1, hq=8, hkv=2, d=64, page=64, pages=4096, table_width=4096, scale=0.25, dt=DType.F16)]


@pytest.mark.parametrize("spec", SPECS, ids=lambda s: type(s).__name__)
@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda s: pickle.loads(pickle.dumps(s))], ids=["copy", "deepcopy", "pickle"])
def test_copies(spec, how):
    other = how(spec)
    assert other == spec and other is not spec and type(other) is type(spec)
    assert bytes(other._desc) == bytes(spec._desc) and other._sizes == spec._sizes
    assert C.addressof(other._desc) != C.addressof(spec._desc) and other._ref._obj is other._desc
    n = {"Mx4QuantSpec": 3, "Mx4DequantSpec": 3, "Mx4PwSpec": 7, "Kv4AppendSpec": 12, "Kv4AttnSpec": 9}[type(spec).__name__]
    ws = {"ws": 1 << 20} if isinstance(spec, mx4.Kv4AttnSpec) else {}
    with pytest.raises(AihError, match="aligned"):  # the library reads the copy's descriptor
        other.run(*[(1 << 20) + 2] * n, stream=0, **ws)
    if ws:
        assert other.workspace_bytes() == spec.workspace_bytes() > 0
