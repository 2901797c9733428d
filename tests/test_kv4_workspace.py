"""CPU test of what the 4-bit cache attention asks of its workspace. Nothing here launches
a kernel: what stands for tensors on GPUs has no memory."""
from types import SimpleNamespace

import pytest
import torch

from ai_engine_amd import mx4
from ai_engine_amd.conv import AihError, DType

FAKE = 1 << 20


def on_gpu(device, nbytes, at=FAKE, dense=True):
    return SimpleNamespace(numel=lambda: nbytes // 4, element_size=lambda: 4, is_cuda=True, get_device=lambda: device,
                           is_contiguous=lambda: dense, device=f"cuda:{device}", data_ptr=lambda: at)


def test_a_workspace_on_another_device_is_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(mx4, "_torch", None)
    spec = mx4.Kv4AttnSpec(nseq=1, tokens=1, hq=8, hkv=2, d=64, page=64, pages=4096, table_width=4096, dt=DType.F16)
    n = spec.workspace_bytes()
    assert n > 0
    for ws in (on_gpu(1, n), on_gpu(0, n - 4), on_gpu(0, n, dense=False)):
        with pytest.raises(AihError, match="the workspace needs"):
            spec.run(*[FAKE] * 9, ws=ws, stream=0)
    with pytest.raises(AihError, match="aligned"):  # the current device's is taken, and asked further
        spec.run(*[FAKE] * 9, ws=on_gpu(0, n, at=FAKE + 8), stream=0)
    monkeypatch.setattr(mx4, "_torch", None)
