"""Host side of the attention operators (include/aih_attn.h): what runs between
the two pointwise convs of an attention block.

* `QkNormRopeSpec` -> aih_qk_norm_rope: head norms and position rotation of the
  projection's rows, keys and values to their cache rows
* `AttnSpec`       -> aih_attn: attention of packed sequences, whole prompts or
  single tokens over a cache, optionally behind a shared prefix

As in `conv`, buffers are device tensors or raw device addresses, every call is
asynchronous on the given stream (default: torch's current stream), and there
is no CPU fallback.  The specs are frozen: their C descriptor is built once.
Index arrays (starts, lengths, positions, slots) are int32 and tables fp32:
tensors of another type or length, strided ones and ones on the host are refused.
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


_torch = None  # torch's Tensor, int32 and float32


def _torch_types():
    global _torch
    import torch

    _torch = torch.Tensor, torch.int32, torch.float32
    return _torch


def _arrays(**arrays):
    """Device addresses of index and table arrays, name = (tensor, values read, type). Refuses tensors that the
    kernels would read as other values or past their end; None and raw addresses are the caller's, as everywhere.
    `run` asks the same in line first, at half the time: a call costs as much as its launch."""
    for name, (t, n, dtype) in arrays.items():
        if t is not None and not isinstance(t, int) and (
                t.dtype is not dtype or not t.is_contiguous() or t.numel() < n or not t.is_cuda):
            raise AihError(f"{name} must be a dense tensor of at least {n} {dtype} on the GPU, not {tuple(t.shape)} "
                           f"{t.dtype} on {t.device}" + ("" if t.is_contiguous() else ", not dense"))
    return [conv._ptr(t) for t, _, _ in arrays.values()]


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
        object.__setattr__(self, "_half", self.positions * (self.rot // 2))  # values of a table

    def run(self, x, wq, wk, cosines, sines, pos, slots, q, k, v, stream=None):
        """x [tokens, x_stride]; wq, wk [d] or None; cosines, sines [positions, rot/2] fp32; pos, slots int32
        [tokens] or None; q [tokens, hq, d]; k, v [rows, hkv, d] (v None: the values stay in x)."""
        T, i32, f32 = _torch or _torch_types()
        p, n, half = conv._ptr, self.tokens, self._half
        if (pos.__class__ is T and pos.dtype is i32 and pos.is_cuda and pos.is_contiguous() and pos.numel() >= n
                and (slots is None or slots.__class__ is T and slots.dtype is i32 and slots.is_cuda
                     and slots.is_contiguous() and slots.numel() >= n)
                and cosines.__class__ is T and cosines.dtype is f32 and cosines.is_cuda and cosines.is_contiguous()
                and cosines.numel() >= half and sines.__class__ is T and sines.dtype is f32 and sines.is_cuda
                and sines.is_contiguous() and sines.numel() >= half):
            arrays = cosines.data_ptr(), sines.data_ptr(), pos.data_ptr(), p(slots)
        else:
            arrays = _arrays(cosines=(cosines, half, f32), sines=(sines, half, f32), pos=(pos, n, i32),
                             slots=(slots, n, i32))
        if (_lib or lib()).aih_qk_norm_rope(
                C.byref(self._desc), x.data_ptr() if x.__class__ is T else p(x), p(wq), p(wk), *arrays,
                q.data_ptr() if q.__class__ is T else p(q), k.data_ptr() if k.__class__ is T else p(k),
                v.data_ptr() if v.__class__ is T else p(v), conv._stream(stream)):
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
        T, i32, _ = _torch or _torch_types()
        b = self.nseq
        if (q_start.__class__ is T and q_start.dtype is i32 and q_start.is_cuda and q_start.is_contiguous()
                and q_start.numel() > b and k_start.__class__ is T and k_start.dtype is i32 and k_start.is_cuda
                and k_start.is_contiguous() and k_start.numel() >= b and k_len.__class__ is T and k_len.dtype is i32
                and k_len.is_cuda and k_len.is_contiguous() and k_len.numel() >= b):
            arrays = q_start.data_ptr(), k_start.data_ptr(), k_len.data_ptr()
        else:
            arrays = _arrays(q_start=(q_start, b + 1, i32), k_start=(k_start, b, i32), k_len=(k_len, b, i32))
        n = self._ws if self._ws is not None else self.workspace_bytes()
        if n:
            if ws is None:
                ws = _workspace_on(n, conv._device_of(out), stream)
            if not isinstance(ws, int) and ws.numel() * ws.element_size() < n:
                raise AihError(f"the workspace needs {n} bytes, not {ws.numel() * ws.element_size()}")
        p = conv._ptr
        if (_lib or lib()).aih_attn(
                C.byref(self._desc), q.data_ptr() if q.__class__ is T else p(q),
                k.data_ptr() if k.__class__ is T else p(k), v.data_ptr() if v.__class__ is T else p(v), *arrays,
                p(prefix_k), p(prefix_v), out.data_ptr() if out.__class__ is T else p(out), p(ws) if n else None, n,
                conv._stream(stream)):
            raise AihError(conv.last_error())
        return out
