"""CPU tests of the 4-bit cache operators' boundary: what is refused and with which
message, and what the plan says. Nothing here launches a kernel."""
import ctypes as C

import pytest
import torch

from ai_engine_amd import conv, mx4
from ai_engine_amd.conv import AihError, DType

FAKE = 1 << 20
APPEND = ("x", "wq", "wk", "cosines", "sines", "pos", "slots", "q", "k_codes", "k_scales", "v_codes", "v_scales")
ATTN = ("q", "k_codes", "k_scales", "v_codes", "v_scales", "q_start", "table", "k_len", "out")


def append(**kw):
    return mx4.Kv4AppendSpec(**{**dict(tokens=4, hq=4, hkv=2, d=64, page=32, pages=8, rot=64, positions=9, dt=DType.F16), **kw})


def attn(**kw):
    return mx4.Kv4AttnSpec(**{**dict(nseq=2, tokens=10, hq=8, hkv=2, d=64, page=32, pages=8, table_width=4, dt=DType.F16), **kw})


def run(spec, **kw):
    names = APPEND if isinstance(spec, mx4.Kv4AppendSpec) else ATTN
    more = {"ws": kw.pop("ws")} if "ws" in kw else {}
    return spec.run(*(kw.get(n, FAKE) for n in names), stream=0, **more)


@pytest.mark.parametrize("make", [append, attn])
@pytest.mark.parametrize("kw, msg", [
    (dict(d=0), "d must be"), (dict(d=48), "d must be"), (dict(d=288), "d must be"), (dict(dt=7), "dtype"),
    (dict(hkv=0), "hkv"), (dict(hkv=5000), "hkv"), (dict(hq=5000), "hq"), (dict(page=8), "page must"),
    (dict(page=48), "page must"), (dict(page=8192), "page must"), (dict(pages=1 << 26), "pages \\* page"),
    (dict(q_stride=8), "q_stride"), (dict(q_stride=260 + 512), "q_stride"), (dict(q_stride=1 << 23), "q_stride")])
def test_cache_sizes(make, kw, msg):
    with pytest.raises(AihError, match=msg):
        run(make(**kw))


@pytest.mark.parametrize("kw, msg", [
    (dict(rot=8), "rot must"), (dict(rot=24), "rot must"), (dict(rot=80), "rot must"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(positions=0), "tables"),
    (dict(positions=1 << 31), "tables"), (dict(tokens=1 << 29), "tokens"), (dict(x_stride=500), "x_stride"),
    (dict(x_stride=516), "x_stride")])
def test_append_sizes(kw, msg):
    with pytest.raises(AihError, match=msg):
        run(append(**kw))


@pytest.mark.parametrize("kw, msg", [
    (dict(hq=0), "multiple of hkv"), (dict(hq=3), "multiple of hkv"), (dict(nseq=1 << 31), "2\\^31"),
    (dict(tokens=1 << 31), "2\\^31"), (dict(tokens=1 << 29), "tokens \\* hq"), (dict(table_width=1 << 27), "table_width"),
    (dict(scale=1e30), "scale"), (dict(scale=float("inf")), "scale"), (dict(o_stride=8), "o_stride"),
    (dict(o_stride=514), "o_stride"), (dict(hq=4096, hkv=4096, tokens=1 << 18, nseq=1 << 30, max_len=0), "tiles")])
def test_attn_sizes(kw, msg):
    with pytest.raises(AihError, match=msg):
        attn(**kw).plan()
    with pytest.raises(AihError, match=msg):
        run(attn(**kw))


@pytest.mark.parametrize("kw", [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(tokens=-1),
                                dict(tokens=1.0), dict(table_width=1 << 32), dict(page=True), dict(max_len=-5)])
def test_attn_spec_refuses(kw):
    with pytest.raises(AihError):
        attn(**kw)


def test_null_and_unaligned():
    for name in ("x", "slots", "q", "k_codes", "k_scales", "v_codes", "v_scales"):
        with pytest.raises(AihError, match="NULL"):
            run(append(), **{name: None})
    for name in ("cosines", "sines"):
        with pytest.raises(AihError, match="needs cosines and sines"):
            run(append(), **{name: None})
    for name in set(APPEND) - {"pos", "slots"}:
        with pytest.raises(AihError, match="aligned"):
            run(append(), **{name: FAKE + 8})
    for name in ("q", "q_start", "k_len", "out"):
        with pytest.raises(AihError, match="NULL"):
            run(attn(), **{name: None})
    for name in ("k_codes", "k_scales", "v_codes", "v_scales", "table"):
        with pytest.raises(AihError, match="must not be NULL"):
            run(attn(), **{name: None})
    for name in ("q", "k_codes", "k_scales", "v_codes", "v_scales", "out"):
        with pytest.raises(AihError, match="aligned"):
            run(attn(), **{name: FAKE + 4})


def test_nothing_to_do():
    run(append(tokens=0), **{n: None for n in APPEND})
    run(attn(nseq=0, tokens=0), **{n: None for n in ATTN})
    run(attn(nseq=3, tokens=0), **{n: None for n in ATTN})
    assert attn(nseq=0, tokens=0).plan().ws_bytes == 0


def test_plan():
    p = attn().plan()  # 128 keys at most
    assert (p.bm, p.parts, p.chunk, p.ws_bytes) == (32, 1, 0, 0) and attn(tokens=2).plan().bm == 16
    p = attn(nseq=1, tokens=1, pages=4096, table_width=4096, page=64, hq=16, hkv=4, d=128).plan()
    assert p.parts > 1 and p.parts * p.chunk >= 4096 * 64 and p.ws_bytes == p.parts * 16 * 130 * 4
    assert p.grid == 4 * p.parts


def test_workspace():
    spec = attn(nseq=1, tokens=1, pages=4096, table_width=4096, page=64)
    n = spec.workspace_bytes()
    with pytest.raises(AihError, match="aligned"):
        run(spec, ws=FAKE + 8)
    for ws in (torch.empty(n // 4), torch.empty(n // 4 - 1), torch.empty(n // 4, 2)[:, 0]):  # on the host, all of them
        with pytest.raises(AihError, match="the workspace needs"):
            run(spec, ws=ws)
    d = spec._desc
    rc = mx4.lib().aih_kv4_attn(C.byref(d), *[FAKE] * 9, FAKE, n - 4, None)
    assert rc == -1 and "workspace needs" in conv.last_error()
    rc = mx4.lib().aih_kv4_attn(C.byref(d), *[FAKE] * 9, None, n, None)
    assert rc == -1 and "workspace needs" in conv.last_error()


def test_null_descriptor():
    L = mx4.lib()
    assert L.aih_kv4_append(None, *[None] * 13) == -1 and "NULL descriptor" in conv.last_error()
    assert L.aih_kv4_attn(None, *[None] * 10, 0, None) == -1 and "NULL descriptor" in conv.last_error()
    assert L.aih_kv4_attn_plan(None, None) == -1 and "NULL descriptor" in conv.last_error()
