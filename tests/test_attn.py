"""CPU tests of the attention operators' boundary: what is refused and with
which message, and what the plan says. Nothing here launches a kernel."""
import ctypes as C
import dataclasses

import pytest

from ai_engine_amd import attn, conv
from ai_engine_amd.conv import AihError, DType

FAKE = 1 << 20  # a 16-byte aligned address that no refused call touches


def attn_spec(**kw):
    base = dict(nseq=2, tokens=10, rows=20, hq=8, hkv=2, d=64, dt=DType.F16)
    return attn.AttnSpec(**{**base, **kw})


def call_attn(spec, **kw):
    names = ("q", "k", "v", "q_start", "k_start", "k_len", "out")
    args = {n: kw.get(n, FAKE) for n in names}
    spec.run(*args.values(), prefix_k=kw.get("prefix_k"), prefix_v=kw.get("prefix_v"), ws=kw.get("ws"), stream=0)


def rope_spec(**kw):
    base = dict(tokens=4, hq=4, hkv=2, d=64, rot=64, positions=16, dt=DType.F16)
    return attn.QkNormRopeSpec(**{**base, **kw})


def call_rope(spec, **kw):
    names = ("x", "wq", "wk", "cosines", "sines", "pos", "slots", "q", "k", "v")
    spec.run(*(kw.get(n, FAKE) for n in names), stream=0)


@pytest.mark.parametrize("kw, msg", [
    (dict(d=0), "d must be"), (dict(d=12), "d must be"), (dict(d=264), "d must be"),
    (dict(hq=0), "heads"), (dict(hq=5000), "heads"), (dict(hkv=0), "multiple of hkv"), (dict(hkv=3), "multiple of hkv"),
    (dict(dt=7), "dtype"), (dict(scale=1e30), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q_stride=500), "q_stride"), (dict(q_stride=516), "16-byte"), (dict(k_stride=64), "k_stride"),
    (dict(v_stride=1 << 23), "v_stride"), (dict(o_stride=8), "o_stride"), (dict(pk_stride=1), "pk_stride"),
    (dict(pv_stride=130), "16-byte"), (dict(tokens=1 << 31), "2^31"), (dict(rows=1 << 31), "2^31"),
    (dict(nseq=1 << 31), "2^31"), (dict(prefix=1 << 31), "2^31"), (dict(tokens=1 << 29), "tokens \\* hq"),
])
def test_attn_refuses(kw, msg):
    with pytest.raises(AihError, match=msg.replace("^", "\\^")):
        attn_spec(**kw).plan()
    with pytest.raises(AihError, match=msg.replace("^", "\\^")):
        call_attn(attn_spec(**kw))


@pytest.mark.parametrize("kw", [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(tokens=-1),
                                dict(tokens=1.0), dict(rows=1 << 32), dict(d=True), dict(max_len=-5)])
def test_attn_spec_refuses(kw):
    with pytest.raises(AihError):
        attn_spec(**kw)


@pytest.mark.parametrize("name", ["q", "k", "v", "q_start", "k_start", "k_len", "out"])
def test_attn_null_tensor(name):
    with pytest.raises(AihError, match="NULL"):
        call_attn(attn_spec(), **{name: None})


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_attn_unaligned(name):
    with pytest.raises(AihError, match="aligned"):
        call_attn(attn_spec(), **{name: FAKE + 8})


def test_attn_prefix_needs_tensors():
    with pytest.raises(AihError, match="prefix_k"):
        call_attn(attn_spec(prefix=5), ws=FAKE)
    with pytest.raises(AihError, match="aligned"):
        call_attn(attn_spec(prefix=5), ws=FAKE, prefix_k=FAKE + 2, prefix_v=FAKE)


def test_attn_workspace_too_small():
    spec = attn_spec(prefix=5)
    n = spec.workspace_bytes()
    assert n > 0
    L = attn.lib()
    rc = L.aih_attn(C.byref(spec._desc), *[FAKE] * 10, n - 1, 0)
    assert rc == -1 and "workspace needs %d bytes, not %d" % (n, n - 1) in conv.last_error()
    rc = L.aih_attn(C.byref(spec._desc), *[FAKE] * 9, None, n, 0)
    assert rc == -1 and "workspace" in conv.last_error()


def test_attn_workspace_tensor_too_small():
    import torch

    spec = attn_spec(prefix=5)
    with pytest.raises(AihError, match="workspace"):
        call_attn(spec, prefix_k=FAKE, prefix_v=FAKE, ws=torch.zeros(8))


def test_null_descriptors():
    L = attn.lib()
    assert L.aih_attn_plan(None, None) == -1 and "NULL" in conv.last_error()
    assert L.aih_attn_plan(C.byref(attn_spec()._desc), None) == -1
    assert L.aih_attn(None, *[FAKE] * 10, 0, 0) == -1
    assert L.aih_qk_norm_rope(None, *[FAKE] * 11) == -1


def test_nothing_to_do_is_accepted():
    call_attn(attn_spec(nseq=0))
    call_attn(attn_spec(tokens=0))
    call_rope(rope_spec(tokens=0))


@pytest.mark.parametrize("kw, msg", [
    (dict(d=4), "d must be"), (dict(d=512), "d must be"), (dict(hq=0), "heads"), (dict(dt=3), "dtype"),
    (dict(rot=6), "rot"), (dict(rot=68), "rot"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(positions=0), "tables"), (dict(x_stride=256), "x_stride"),
    (dict(x_stride=516), "16-byte"), (dict(q_stride=100), "q_stride"), (dict(k_stride=100), "k_stride"),
    (dict(v_stride=1 << 30), "v_stride"), (dict(tokens=1 << 31), "2^31"), (dict(rows=1 << 31), "2^31"),
])
def test_rope_refuses(kw, msg):
    with pytest.raises(AihError, match=msg.replace("^", "\\^")):
        call_rope(rope_spec(**kw))


@pytest.mark.parametrize("name", ["x", "q", "k", "cosines", "sines"])
def test_rope_null_tensor(name):
    with pytest.raises(AihError, match="NULL|cosines"):
        call_rope(rope_spec(), **{name: None})


@pytest.mark.parametrize("name", ["x", "wq", "wk", "cosines", "sines", "q", "k", "v"])
def test_rope_unaligned(name):
    with pytest.raises(AihError, match="aligned"):
        call_rope(rope_spec(), **{name: FAKE + 4})


def test_plan_routes():
    # one token a sequence: 32 rows a tile, the keys over the wavefronts
    p = attn_spec(nseq=64, tokens=64, rows=64 * 8192, hq=32, hkv=8, d=128, max_len=8192).plan()
    assert p.kernel == attn.AttnKernel.KEYS and p.bm == 32 and p.parts > 1 and p.chunk % 32 == 0
    assert p.ws_bytes == p.parts * 64 * 32 * (128 + 2) * 4
    # whole prompts: tiles of rows, no workspace
    p = attn_spec(nseq=64, tokens=64 * 720, rows=64 * 720).plan()
    assert p.kernel == attn.AttnKernel.ROWS and p.parts == 1 and p.ws_bytes == 0
    # a prefix always leaves two parts to join
    p = attn_spec(nseq=6, tokens=12, rows=6 * 77, prefix=720).plan()
    assert p.prefix_kernel and p.prefix_parts >= 1 and p.ws_bytes > 0


def test_specs_are_frozen():
    with pytest.raises(dataclasses.FrozenInstanceError):
        attn_spec().d = 32
    assert dataclasses.replace(attn_spec(), d=32)._desc.d == 32
