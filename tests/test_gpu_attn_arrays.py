"""GPU tests of the attention bindings' index and table arrays: what is refused
where the tensors are on the GPU, and that arrays with more values than needed
are taken."""
import pytest
import torch

from ai_engine_amd import attn
from ai_engine_amd.conv import AihError
from tests.test_attn_arrays import CASES, NSEQ, POSITIONS, ROT, TOKENS, others, run_attn, run_rope

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("run, name, i, n, dtype", CASES)
def test_other_arrays_are_refused_on_the_gpu(run, name, i, n, dtype):
    # the others are as they should be: the tensors in the call differ from a good call's in one
    if run is run_attn:
        good = dict(q_start=torch.zeros(NSEQ + 1, **I32), k_start=torch.zeros(NSEQ, **I32),
                    k_len=torch.zeros(NSEQ, **I32))
    else:
        table = torch.zeros(POSITIONS, ROT // 2, device=DEV)
        good = dict(cosines=table, sines=table, pos=torch.zeros(TOKENS, **I32), slots=torch.zeros(TOKENS, **I32))
    t = list(others(n, dtype, DEV))[i]
    with pytest.raises(AihError, match=f"{name} must be a dense tensor of at least {n} {dtype}"):
        run(**{**good, name: t})


def test_arrays_may_hold_more():
    x = torch.randn(TOKENS, 4, 64, device=DEV)
    q, k, v = (torch.empty(TOKENS, h, 64, device=DEV) for h in (2, 1, 1))
    tables = torch.ones(POSITIONS + 2, ROT // 2, device=DEV)
    more = torch.arange(TOKENS + 3, **I32)
    spec = attn.QkNormRopeSpec(tokens=TOKENS, hq=2, hkv=1, d=64, rot=ROT, positions=POSITIONS)
    spec.run(x, None, None, tables, tables, more, more, q, k, v)
    out = torch.full((TOKENS, 2, 64), float("nan"), device=DEV)
    spec = attn.AttnSpec(nseq=1, tokens=TOKENS, rows=TOKENS, hq=2, hkv=1, d=64)
    i32 = lambda *a: torch.tensor(a, **I32)
    spec.run(q, k, v, i32(0, TOKENS, 99), i32(0, 7), i32(TOKENS, 7), out)
    assert torch.equal(v, x[:, 3:]) and torch.isfinite(out).all()
    assert torch.allclose(out[0], v[0].expand(2, -1))  # a causal first token sees its own value alone
