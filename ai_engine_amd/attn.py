"""Host side of the attention operators (include/aih_attn.h): what runs between
the two pointwise convs of an attention block.

* `QkNormRopeSpec` -> aih_qk_norm_rope: head norms and position rotation of the
  projection's rows, keys and values to their cache rows
* `AttnSpec`       -> aih_attn: attention of packed sequences, whole prompts or
  single tokens over a cache, optionally behind a shared prefix

As in `conv`, buffers are device tensors or raw device addresses, every call is
asynchronous on the given stream (default: torch's current stream), and there
is no CPU fallback.  The specs are frozen: their C descriptor is built once.
"""
from __future__ import annotations

import ctypes as C
import enum
from dataclasses import dataclass

from . import conv
from .conv import AihError, DType  # noqa: F401  (AihError is what a refused call raises)


class AttnKernel(enum.IntEnum):
    """Which kernel runs (enum aih_attn_kernel)."""

    ROWS = 1
    KEYS = 2


class _QkDesc(C.Structure):
    _fields_ = [("tokens", C.c_uint32), ("hq", C.c_uint32), ("hkv", C.c_uint32), ("d", C.c_uint32),
                ("rot", C.c_uint32), ("pairs", C.c_int32), ("eps", C.c_float), ("dt", C.c_int32),
                ("positions", C.c_uint32), ("rows", C.c_uint32), ("x_stride", C.c_uint64), ("q_stride", C.c_uint64),
                ("k_stride", C.c_uint64), ("v_stride", C.c_uint64)]


class _AttnDesc(C.Structure):
    _fields_ = [("nseq", C.c_uint32), ("tokens", C.c_uint32), ("rows", C.c_uint32), ("hq", C.c_uint32),
                ("hkv", C.c_uint32), ("d", C.c_uint32), ("causal", C.c_int32), ("scale", C.c_float),
                ("dt", C.c_int32), ("max_len", C.c_uint32), ("prefix", C.c_uint32), ("q_stride", C.c_uint64),
                ("k_stride", C.c_uint64), ("v_stride", C.c_uint64), ("o_stride", C.c_uint64),
                ("pk_stride", C.c_uint64), ("pv_stride", C.c_uint64)]


class AttnPlan(C.Structure):
    _fields_ = [("kernel", C.c_int32), ("bm", C.c_uint32), ("parts", C.c_uint32), ("chunk", C.c_uint32),
                ("prefix_kernel", C.c_int32), ("prefix_bm", C.c_uint32), ("prefix_parts", C.c_uint32),
                ("prefix_chunk", C.c_uint32), ("grid", C.c_uint32), ("ws_bytes", C.c_size_t)]


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        L = conv.lib()
        P = C.c_void_p
        sigs = {
            "aih_qk_norm_rope": [C.POINTER(_QkDesc)] + [P] * 11,
            "aih_attn_plan": [C.POINTER(_AttnDesc), C.POINTER(AttnPlan)],
            "aih_attn": [C.POINTER(_AttnDesc)] + [P] * 10 + [C.c_size_t, P],
        }
        for name, args in sigs.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = C.c_int, args
        _lib = L
    return _lib


def _u32(name, v, lo=0):
    if type(v) is not int or not lo <= v < 1 << 32:
        raise AihError(f"{name} must be an integer from {lo} to 2^32 - 1, not {v!r}")
    return v


def _workspace_on(nbytes, device, stream):
    """Device memory of the stream it is used on: torch gives a freed block to that stream's next allocation only."""
    device = device or "cuda"  # a raw address has none
    if stream is None:
        return conv._workspace(nbytes, None, device)
    import torch

    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device) if isinstance(stream, int) else stream):
        return conv._workspace(nbytes, None, device)


@dataclass(frozen=True)
class QkNormRopeSpec:
    """Head norms and rotation; fields of aih_qk_norm_rope_desc (strides in elements, 0 = dense)."""

    tokens: int
    hq: int
    hkv: int
    d: int
    rot: int = 0
    pairs: bool = False
    eps: float = 1e-6
    dt: DType = DType.F32
    positions: int = 0
    rows: int | None = None  # of k and v; None: tokens
    x_stride: int = 0
    q_stride: int = 0
    k_stride: int = 0
    v_stride: int = 0

    def __post_init__(self):
        rows = self.tokens if self.rows is None else self.rows
        object.__setattr__(self, "_desc", _QkDesc(
            *(_u32(n, getattr(self, n)) for n in ("tokens", "hq", "hkv", "d", "rot")), int(bool(self.pairs)),
            self.eps, int(self.dt), _u32("positions", self.positions), _u32("rows", rows),
            *(_u32(n, getattr(self, n)) for n in ("x_stride", "q_stride", "k_stride", "v_stride"))))

    def run(self, x, wq, wk, cosines, sines, pos, slots, q, k, v, stream=None):
        """x [tokens, x_stride]; wq, wk [d] or None; cosines, sines [positions, rot/2] fp32; pos, slots int32
        [tokens] or None; q [tokens, hq, d]; k, v [rows, hkv, d] (v None: the values stay in x)."""
        p = conv._ptr
        if (_lib or lib()).aih_qk_norm_rope(C.byref(self._desc), p(x), p(wq), p(wk), p(cosines), p(sines), p(pos), p(slots),
                                            p(q), p(k), p(v), conv._stream(stream)):
            raise AihError(conv.last_error())
        return q, k, v


@dataclass(frozen=True)
class AttnSpec:
    """Attention; fields of aih_attn_desc (strides in elements, 0 = dense; scale None = 1 / sqrt(d))."""

    nseq: int
    tokens: int
    rows: int
    hq: int
    hkv: int
    d: int
    causal: bool = True
    scale: float | None = None
    dt: DType = DType.F32
    max_len: int = 0
    prefix: int = 0
    q_stride: int = 0
    k_stride: int = 0
    v_stride: int = 0
    o_stride: int = 0
    pk_stride: int = 0
    pv_stride: int = 0

    def __post_init__(self):
        if self.scale is not None and not self.scale > 0:
            raise AihError(f"scale must be positive, not {self.scale!r}")
        object.__setattr__(self, "_desc", _AttnDesc(
            *(_u32(n, getattr(self, n)) for n in ("nseq", "tokens", "rows", "hq", "hkv", "d")),
            int(bool(self.causal)), self.scale or 0.0, int(self.dt), _u32("max_len", self.max_len),
            _u32("prefix", self.prefix),
            *(_u32(n, getattr(self, n)) for n in ("q_stride", "k_stride", "v_stride", "o_stride", "pk_stride",
                                                  "pv_stride"))))
        object.__setattr__(self, "_ws", None)

    def plan(self) -> AttnPlan:
        p = AttnPlan()
        conv._check(lib().aih_attn_plan(C.byref(self._desc), C.byref(p)))
        return p

    def workspace_bytes(self) -> int:
        if self._ws is None:
            object.__setattr__(self, "_ws", self.plan().ws_bytes)
        return self._ws

    def run(self, q, k, v, q_start, k_start, k_len, out, prefix_k=None, prefix_v=None, ws=None, stream=None):
        """q, out [tokens, hq, d]; k, v [rows, hkv, d]; q_start [nseq + 1], k_start, k_len [nseq] int32;
        prefix_k, prefix_v [prefix, hkv, d]; ws: workspace_bytes() of device memory, made here if None."""
        n = self._ws if self._ws is not None else self.workspace_bytes()
        if n:
            if ws is None:
                ws = _workspace_on(n, conv._device_of(out), stream)
            if not isinstance(ws, int) and ws.numel() * ws.element_size() < n:
                raise AihError(f"the workspace needs {n} bytes, not {ws.numel() * ws.element_size()}")
        p = conv._ptr
        if (_lib or lib()).aih_attn(C.byref(self._desc), p(q), p(k), p(v), p(q_start), p(k_start), p(k_len), p(prefix_k),
                                    p(prefix_v), p(out), p(ws) if n else None, n, conv._stream(stream)):
            raise AihError(conv.last_error())
        return out
