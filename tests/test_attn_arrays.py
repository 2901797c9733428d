"""CPU tests of the attention bindings' index and table arrays: the kernels read
them as dense values of one type, so any other tensor is refused. Nothing here
launches a kernel."""
import pytest
import torch

from ai_engine_amd import attn
from ai_engine_amd.conv import AihError, DType

FAKE = 1 << 20  # a 16-byte aligned address that no refused call touches
NSEQ, TOKENS, POSITIONS, ROT = 3, 5, 7, 32

I32, F32 = torch.int32, torch.float32
ATTN = {"q_start": (NSEQ + 1, I32), "k_start": (NSEQ, I32), "k_len": (NSEQ, I32)}
ROPE = {"cosines": (POSITIONS * ROT // 2, F32), "sines": (POSITIONS * ROT // 2, F32), "pos": (TOKENS, I32),
        "slots": (TOKENS, I32)}


class OnGpu(torch.Tensor):
    """A host tensor that says it is on the GPU, for the checks behind that one."""

    is_cuda = True


def run_attn(**kw):
    args = {n: FAKE for n in ("q", "k", "v", "q_start", "k_start", "k_len", "out")}
    attn.AttnSpec(nseq=NSEQ, tokens=TOKENS, rows=20, hq=2, hkv=1, d=64).run(**{**args, **kw}, stream=0)


def run_rope(**kw):
    args = {n: FAKE for n in ("x", "wq", "wk", "cosines", "sines", "pos", "slots", "q", "k", "v")}
    attn.QkNormRopeSpec(tokens=TOKENS, hq=2, hkv=1, d=64, rot=ROT, positions=POSITIONS).run(**{**args, **kw}, stream=0)


def others(n, dtype, device="cpu"):
    yield torch.zeros(n, dtype={I32: torch.int64, F32: torch.float64}[dtype], device=device)  # arange's, cumsum's
    yield torch.zeros(n, dtype={I32: torch.int16, F32: torch.float16}[dtype], device=device)
    yield torch.zeros(n - 1, dtype=dtype, device=device)
    yield torch.zeros(2 * n, dtype=dtype, device=device)[::2]
    yield torch.zeros(1, dtype=dtype, device=device).expand(n)


CASES = [(run_attn, name, i, *ATTN[name]) for name in ATTN for i in range(5)]
CASES += [(run_rope, name, i, *ROPE[name]) for name in ROPE for i in range(5)]


@pytest.mark.parametrize("run, name, i, n, dtype", CASES)
def test_other_arrays_are_refused(run, name, i, n, dtype):
    t = list(others(n, dtype))[i].as_subclass(OnGpu)
    with pytest.raises(AihError, match=f"{name} must be a dense tensor of at least {n} {dtype}"):
        run(**{name: t})


@pytest.mark.parametrize("run, name", [(run_attn, n) for n in ATTN] + [(run_rope, n) for n in ROPE])
def test_host_arrays_are_refused(run, name):
    n, dtype = (ATTN | ROPE)[name]
    with pytest.raises(AihError, match=f"{name} must be .* on the GPU, not .* on cpu"):
        run(**{name: torch.zeros(n, dtype=dtype)})
