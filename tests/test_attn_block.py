"""CPU tests of the attention block's boundary: what is refused before anything
runs. Nothing here launches a kernel."""
import numpy as np
import pytest
import torch

from ai_engine_amd.attn_block import AttnBlock
from ai_engine_amd.conv import AihError, DType

C, HQ, HKV, D = 64, 4, 2, 32


def make_weights(**kw):
    z = lambda *s: np.zeros(s, np.float32)
    return {**dict(w_qkv=z((HQ + 2 * HKV) * D, C), b_qkv=z((HQ + 2 * HKV) * D), w_out=z(C, HQ * D), b_out=z(C), wq=z(D),
                   wk=z(D)), **kw}


def make_block(dt=DType.F32, weights=None, **kw):
    return AttnBlock(C, HQ, HKV, D, streams=2, capacity=8, weights=weights or make_weights(), dt=dt, prefix=4,
                     device="cpu", **kw)


# ---------------------------------------------------------------- the rows of share and step

BAD_ROWS = [
    ("another type", lambda *s: torch.zeros(*s, C, dtype=torch.float16)),
    ("fewer channels", lambda *s: torch.zeros(*s, C // 2)),
    ("more channels", lambda *s: torch.zeros(*s, C + 8)),
    ("transposed", lambda *s: torch.zeros(*s[:-1], C, s[-1]).transpose(-1, -2)),
    ("a slice", lambda *s: torch.zeros(*s, 2 * C)[..., :C]),
    ("one dim more", lambda *s: torch.zeros(*s, C, 1)),
    ("one dim less", lambda *s: torch.zeros(s[-1] * C)),
    ("another device", lambda *s: torch.zeros(*s, C, device="meta")),
]


@pytest.mark.parametrize("what, make", BAD_ROWS, ids=[w for w, _ in BAD_ROWS])
def test_share_refuses_other_rows(what, make, monkeypatch):
    block = make_block()
    monkeypatch.setattr(block, "_project", lambda *a: pytest.fail("the projection was called"))
    with pytest.raises(AihError, match="share takes"):
        block.share(make(3))
    assert block.shared == 0


@pytest.mark.parametrize("what, make", BAD_ROWS, ids=[w for w, _ in BAD_ROWS])
def test_step_refuses_other_rows(what, make, monkeypatch):
    block = make_block()
    monkeypatch.setattr(block, "_project", lambda *a: pytest.fail("the projection was called"))
    with pytest.raises(AihError, match="step takes"):
        block.step(make(2, 3))
    assert block.length == 0


def test_sharing_no_tokens_leaves_no_context(monkeypatch):
    block = make_block()
    monkeypatch.setattr(block, "_project", lambda *a: pytest.fail("the projection was called"))
    block.shared = 3
    block.share(torch.zeros(0, C))
    assert block.shared == 0


# ---------------------------------------------------------------- weights

@pytest.mark.parametrize("name", ["w_qkv", "b_qkv", "w_out", "b_out", "wq", "wk"])
@pytest.mark.parametrize("more", [-1, 1])
def test_weights_of_another_size_are_refused(name, more):
    w = make_weights()
    w[name] = np.zeros(w[name].size + more, np.float32)
    with pytest.raises(AihError, match=f"{name} must hold"):
        make_block(weights=w)


def test_norm_weights_are_stored_dense():
    w = make_weights(wq=torch.arange(2.0 * D)[::2], wk=torch.arange(4.0 * D)[::4])
    block = make_block(weights=w)
    assert block.wq.is_contiguous() and block.wk.is_contiguous()
    assert torch.equal(block.wq, w["wq"]) and torch.equal(block.wk, w["wk"])


# ---------------------------------------------------------------- what a block keeps

def held(block):
    """Bytes of the distinct buffers that a block's steps keep."""
    tensors = [t for p in block._plans.values() for t in p.values() if isinstance(t, torch.Tensor)]
    tensors += [t for t in vars(block).values() if isinstance(t, torch.Tensor)]
    return sum({t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in tensors}.values())


@pytest.mark.parametrize("shared", [0, 40])
def test_steps_of_many_lengths_hold_one_set_of_buffers(shared):
    make = lambda: AttnBlock(C, HQ, HKV, D, streams=16, capacity=200, weights=make_weights(), prefix=40, device="cpu")
    one, many = make(), make()
    one.shared = many.shared = shared
    one._plan(200)
    for tokens in [*range(1, 201, 7), 200, *range(200, 0, -7)]:
        p = many._plan(tokens)
        assert p["q"].shape == p["o"].shape == (16 * tokens, HQ, D) and p["at"].shape == (tokens,)
        assert p["q"].data_ptr() != p["o"].data_ptr() and p["q"].is_contiguous() and p["o"].is_contiguous()
        need = p["attn"].workspace_bytes()
        assert (p["ws"] is None) == (need == 0) and (need == 0 or 4 * p["ws"].numel() >= need)
    # the rest is a starts array of each length
    assert held(many) <= held(one) + 80 * 4 * 17
    # no length keeps buffers that have been outgrown
    assert len({p["q"].untyped_storage().data_ptr() for p in many._plans.values()}) == 1
