"""Host side of the operators on microscaled 4-bit rows (include/aih_mx4.h).

* `Mx4QuantSpec`   -> aih_mx4_quant: rows of a storage type to 4 bits
* `Mx4DequantSpec` -> aih_mx4_dequant: the values that 4-bit rows stand for
* `Mx4PwSpec`      -> aih_mx4_pw: the 1x1 conv of 4-bit rows and 4-bit weights
* `Kv4AppendSpec`  -> aih_kv4_append: rotation of queries and keys, new keys and
  values into the pages of a 4-bit cache
* `Kv4AttnSpec`    -> aih_kv4_attn: attention over such a cache

As in `conv`, buffers are device tensors or raw device addresses, every call is
asynchronous on the given stream (default: torch's current stream), and there is no
CPU fallback.  The specs are frozen: their C descriptor is built once.  Tensors
that are strided, too short, of another type or not on the current device are
refused; raw addresses are the caller's own.

    quant = Mx4QuantSpec(rows=cout, k=cin, dt=DType.F16)   # weights, once: [cout, cin]
    quant.run(w, w_codes, w_scales)                        # quant.code_bytes, quant.scale_bytes
    pw = Mx4PwSpec(m=pixels, k=cin, cout=cout, act=Activation.RELU6, dt=DType.F16)
    Mx4QuantSpec(rows=pixels, k=cin, dt=DType.F16).run(x, x_codes, x_scales)
    pw.run(x_codes, x_scales, w_codes, w_scales, bias, None, y)
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, fields

from . import conv
from .attn import _u32, _workspace_on
from .conv import Activation, AihError, DType


class _QuantDesc(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("k", C.c_uint32), ("dt", C.c_int32), ("x_stride", C.c_uint64)]


class _DequantDesc(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("k", C.c_uint32), ("dt", C.c_int32), ("code_stride", C.c_uint32),
                ("scale_stride", C.c_uint32), ("y_stride", C.c_uint64)]


class _PwDesc(C.Structure):
    _fields_ = [("m", C.c_uint32), ("k", C.c_uint32), ("cout", C.c_uint32), ("act", C.c_int32),
                ("residual", C.c_int32), ("dt", C.c_int32)]


class _AppendDesc(C.Structure):
    _fields_ = [("tokens", C.c_uint32), ("hq", C.c_uint32), ("hkv", C.c_uint32), ("d", C.c_uint32),
                ("rot", C.c_uint32), ("pairs", C.c_int32), ("norm", C.c_int32), ("eps", C.c_float), ("dt", C.c_int32),
                ("positions", C.c_uint32), ("page", C.c_uint32), ("pages", C.c_uint32), ("x_stride", C.c_uint64),
                ("q_stride", C.c_uint64)]


class _AttnDesc(C.Structure):
    _fields_ = [("nseq", C.c_uint32), ("tokens", C.c_uint32), ("hq", C.c_uint32), ("hkv", C.c_uint32),
                ("d", C.c_uint32), ("page", C.c_uint32), ("pages", C.c_uint32), ("table_width", C.c_uint32),
                ("causal", C.c_int32), ("scale", C.c_float), ("dt", C.c_int32), ("max_len", C.c_uint32),
                ("q_stride", C.c_uint64), ("o_stride", C.c_uint64)]


class Kv4AttnPlan(C.Structure):
    _fields_ = [("bm", C.c_uint32), ("parts", C.c_uint32), ("chunk", C.c_uint32), ("grid", C.c_uint32),
                ("ws_bytes", C.c_size_t)]


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        L = conv.lib()
        P = C.c_void_p
        sigs = {
            "aih_mx4_quant": [C.POINTER(_QuantDesc)] + [P] * 4,
            "aih_mx4_dequant": [C.POINTER(_DequantDesc)] + [P] * 4,
            "aih_mx4_pw": [C.POINTER(_PwDesc)] + [P] * 8,
            "aih_kv4_append": [C.POINTER(_AppendDesc)] + [P] * 13,
            "aih_kv4_attn_plan": [C.POINTER(_AttnDesc), C.POINTER(Kv4AttnPlan)],
            "aih_kv4_attn": [C.POINTER(_AttnDesc)] + [P] * 10 + [C.c_size_t, P],
        }
        for name, args in sigs.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = C.c_int, args
        _lib = L
    return _lib


_torch = None  # torch's Tensor, current device and its current stream, and the types of DType, codes and index arrays


def _torch_types():
    global _torch
    import torch

    _torch = (torch.Tensor, torch.cuda.current_device, torch._C._cuda_getCurrentRawStream,
              {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}, torch.uint8, torch.int32)
    return _torch


def _take(name, t, n, dtype):
    """The device address of `n` values; refuses a tensor that the kernels would read as other values, past its end
    or on another device. None and raw addresses are the caller's, as everywhere. `run` asks the same in line
    first, at half the time: a call costs as much as its launch."""
    if t is None or t.__class__ is int:
        return t
    if t.dtype is dtype and t.is_cuda and t.get_device() == _torch[1]() and t.is_contiguous() and t.numel() >= n:
        return t.data_ptr()
    raise AihError(f"{name} must be a dense tensor of at least {n} {dtype} on the current device, not {tuple(t.shape)} "
                   f"{t.dtype} on {t.device}" + ("" if t.is_contiguous() else ", not dense"))


def code_bytes(k: int) -> int:
    """Bytes of a row's codes, as Mx4QuantSpec writes them."""
    return -(-k // 128) * 64


def scale_bytes(k: int) -> int:
    """Bytes of a row's scales, as Mx4QuantSpec writes them."""
    return -(-k // 512) * 16


def _keep(spec, desc, sizes):
    """The descriptor, a reference to it for the calls, and how many values each tensor has to hold."""
    for name, v in (("_desc", desc), ("_ref", C.byref(desc)), ("_sizes", sizes)):
        object.__setattr__(spec, name, v)


class _Spec:
    """Copies and pickles of a spec are made of its fields, with a descriptor of their own."""

    def __reduce__(self):
        return type(self), tuple(getattr(self, f.name) for f in fields(self))


def _span(rows, stride, last):
    """Values that rows `stride` apart reach over, the last one `last` long."""
    return (rows - 1) * stride + last if rows else 0


@dataclass(frozen=True)
class Mx4QuantSpec(_Spec):
    """Rows to 4 bits; fields of aih_mx4_quant_desc (x_stride in elements, 0 = dense)."""

    rows: int
    k: int
    dt: DType = DType.F32
    x_stride: int = 0

    def __post_init__(self):
        desc = _QuantDesc(_u32("rows", self.rows), _u32("k", self.k), int(self.dt), _u32("x_stride", self.x_stride))
        _keep(self, desc, (_span(self.rows, self.x_stride or self.k, self.k), self.rows * self.code_bytes,
                           self.rows * self.scale_bytes))

    @property
    def code_bytes(self) -> int:
        return code_bytes(self.k)

    @property
    def scale_bytes(self) -> int:
        return scale_bytes(self.k)

    def run(self, x, codes, scales, stream=None):
        """x [rows, x_stride]; codes [rows, code_bytes], scales [rows, scale_bytes] uint8."""
        T, device, raw, types, u8, _ = _torch or _torch_types()
        (nx, nc, ns), t = self._sizes, types.get(self.dt)
        if (x.__class__ is T and x.is_cuda and x.get_device() == (dev := device()) and x.dtype is t
                and x.is_contiguous() and x.numel() >= nx
                and codes.__class__ is T and codes.get_device() == dev and codes.dtype is u8
                and codes.is_contiguous() and codes.numel() >= nc
                and scales.__class__ is T and scales.get_device() == dev and scales.dtype is u8
                and scales.is_contiguous() and scales.numel() >= ns):
            at = x.data_ptr(), codes.data_ptr(), scales.data_ptr(), raw(dev) if stream is None else conv._stream(stream)
        else:
            at = (_take("x", x, nx, t), _take("codes", codes, nc, u8), _take("scales", scales, ns, u8),
                  conv._stream(stream))
        if (_lib or lib()).aih_mx4_quant(self._ref, *at):
            raise AihError(conv.last_error())
        return codes, scales


@dataclass(frozen=True)
class Mx4DequantSpec(_Spec):
    """4-bit rows to values; fields of aih_mx4_dequant_desc (strides: bytes of codes and scales, elements of y)."""

    rows: int
    k: int
    dt: DType = DType.F32
    code_stride: int = 0
    scale_stride: int = 0
    y_stride: int = 0

    def __post_init__(self):
        desc = _DequantDesc(
            _u32("rows", self.rows), _u32("k", self.k), int(self.dt), _u32("code_stride", self.code_stride),
            _u32("scale_stride", self.scale_stride), _u32("y_stride", self.y_stride))
        blocks = -(-self.k // 32)
        _keep(self, desc, (
            _span(self.rows, self.code_stride or code_bytes(self.k), blocks * 16),
            _span(self.rows, self.scale_stride or scale_bytes(self.k), blocks),
            _span(self.rows, self.y_stride or self.k, self.k)))

    def run(self, codes, scales, y, stream=None):
        """codes, scales uint8; y [rows, y_stride]."""
        T, device, raw, types, u8, _ = _torch or _torch_types()
        (nc, ns, ny), t = self._sizes, types.get(self.dt)
        if (codes.__class__ is T and codes.is_cuda and codes.get_device() == (dev := device()) and codes.dtype is u8
                and codes.is_contiguous() and codes.numel() >= nc
                and scales.__class__ is T and scales.get_device() == dev and scales.dtype is u8
                and scales.is_contiguous() and scales.numel() >= ns
                and y.__class__ is T and y.get_device() == dev and y.dtype is t and y.is_contiguous()
                and y.numel() >= ny):
            at = codes.data_ptr(), scales.data_ptr(), y.data_ptr(), raw(dev) if stream is None else conv._stream(stream)
        else:
            at = (_take("codes", codes, nc, u8), _take("scales", scales, ns, u8), _take("y", y, ny, t),
                  conv._stream(stream))
        if (_lib or lib()).aih_mx4_dequant(self._ref, *at):
            raise AihError(conv.last_error())
        return y


@dataclass(frozen=True)
class Mx4PwSpec(_Spec):
    """The 1x1 conv of 4-bit rows; fields of aih_mx4_pw_desc."""

    m: int
    k: int
    cout: int
    act: Activation = Activation.NONE
    residual: bool = False
    dt: DType = DType.F32

    def __post_init__(self):
        desc = _PwDesc(
            *(_u32(n, getattr(self, n)) for n in ("m", "k", "cout")), int(self.act), int(bool(self.residual)),
            int(self.dt))
        cb, sb = code_bytes(self.k), scale_bytes(self.k)
        _keep(self, desc, (self.m * cb, self.m * sb, self.cout * cb, self.cout * sb, self.m * self.cout))

    def run(self, x_codes, x_scales, w_codes, w_scales, bias, res, y, stream=None):
        """Codes and scales as Mx4QuantSpec makes them, of x [m, k] and of the weights [cout, k]; bias [cout] or None;
        res (with `residual`) and y [m, cout]."""
        T, device, raw, types, u8, _ = _torch or _torch_types()
        (nxc, nxs, nwc, nws, ny), t = self._sizes, types.get(self.dt)
        if (y.__class__ is T and y.is_cuda and y.get_device() == (dev := device()) and y.dtype is t
                and y.is_contiguous() and y.numel() >= ny
                and x_codes.__class__ is T and x_codes.get_device() == dev and x_codes.dtype is u8
                and x_codes.is_contiguous() and x_codes.numel() >= nxc
                and x_scales.__class__ is T and x_scales.get_device() == dev and x_scales.dtype is u8
                and x_scales.is_contiguous() and x_scales.numel() >= nxs
                and w_codes.__class__ is T and w_codes.get_device() == dev and w_codes.dtype is u8
                and w_codes.is_contiguous() and w_codes.numel() >= nwc
                and w_scales.__class__ is T and w_scales.get_device() == dev and w_scales.dtype is u8
                and w_scales.is_contiguous() and w_scales.numel() >= nws
                and (bias is None or bias.__class__ is T and bias.get_device() == dev and bias.dtype is t
                     and bias.is_contiguous() and bias.numel() >= self.cout)
                and (res is None or res.__class__ is T and res.get_device() == dev and res.dtype is t
                     and res.is_contiguous() and res.numel() >= (ny if self.residual else 0))):
            at = (x_codes.data_ptr(), x_scales.data_ptr(), w_codes.data_ptr(), w_scales.data_ptr(),
                  None if bias is None else bias.data_ptr(), None if res is None else res.data_ptr(), y.data_ptr(),
                  raw(dev) if stream is None else conv._stream(stream))
        else:
            at = (_take("x_codes", x_codes, nxc, u8), _take("x_scales", x_scales, nxs, u8),
                  _take("w_codes", w_codes, nwc, u8), _take("w_scales", w_scales, nws, u8),
                  _take("bias", bias, self.cout, t), _take("res", res, ny if self.residual else 0, t),
                  _take("y", y, ny, t), conv._stream(stream))
        if (_lib or lib()).aih_mx4_pw(self._ref, *at):
            raise AihError(conv.last_error())
        return y


def kv4_cache(pages, page, hkv, d, device="cuda:0"):
    """(k_codes, k_scales, v_codes, v_scales) of an empty 4-bit cache: [pages, hkv, page, d / 2] and [..., d / 32]."""
    import torch

    return tuple(torch.zeros(pages, hkv, page, n, dtype=torch.uint8, device=device) for n in (d // 2, d // 32) * 2)


@dataclass(frozen=True)
class Kv4AppendSpec(_Spec):
    """New tokens into a 4-bit cache; fields of aih_kv4_append_desc (strides in elements, 0 = dense)."""

    tokens: int
    hq: int
    hkv: int
    d: int
    page: int
    pages: int
    rot: int = 0
    pairs: bool = False
    norm: bool = False
    eps: float = 1e-6
    dt: DType = DType.F32
    positions: int = 0
    x_stride: int = 0
    q_stride: int = 0

    def __post_init__(self):
        u = {n: _u32(n, getattr(self, n)) for n in ("tokens", "hq", "hkv", "d", "rot", "positions", "page", "pages",
                                                    "x_stride", "q_stride")}
        desc = _AppendDesc(
            u["tokens"], u["hq"], u["hkv"], u["d"], u["rot"], int(bool(self.pairs)), int(bool(self.norm)), self.eps,
            int(self.dt), u["positions"], u["page"], u["pages"], u["x_stride"], u["q_stride"])
        row, rows = (self.hq + 2 * self.hkv) * self.d, self.pages * self.hkv * self.page
        _keep(self, desc, (
            _span(self.tokens, self.x_stride or row, row),
            _span(self.tokens, self.q_stride or self.hq * self.d, self.hq * self.d) if self.hq else 0,
            self.positions * (self.rot // 2), rows * (self.d // 2), rows * (self.d // 32)))

    def run(self, x, wq, wk, cosines, sines, pos, slots, q, k_codes, k_scales, v_codes, v_scales, stream=None):
        """x [tokens, x_stride]; wq, wk [d] or None; cosines, sines [positions, rot/2] fp32; pos int32 [tokens] or None;
        slots int32 [tokens]; q [tokens, hq, d]; the cache as kv4_cache makes it."""
        T, device, raw, types, u8, i32 = _torch or _torch_types()
        t, f32, n = types.get(self.dt), types[0], self.tokens
        nx, nq, nt, nc, ns = self._sizes
        if (x.__class__ is T and x.is_cuda and x.get_device() == (dev := device()) and x.dtype is t
                and x.is_contiguous() and x.numel() >= nx
                and slots.__class__ is T and slots.get_device() == dev and slots.dtype is i32
                and slots.is_contiguous() and slots.numel() >= n
                and (cosines is None or cosines.__class__ is T and cosines.get_device() == dev and cosines.dtype is f32
                     and cosines.is_contiguous() and cosines.numel() >= nt)
                and (sines is None or sines.__class__ is T and sines.get_device() == dev and sines.dtype is f32
                     and sines.is_contiguous() and sines.numel() >= nt)
                and (pos is None or pos.__class__ is T and pos.get_device() == dev and pos.dtype is i32
                     and pos.is_contiguous() and pos.numel() >= n)
                and q.__class__ is T and q.get_device() == dev and q.dtype is t and q.is_contiguous()
                and q.numel() >= nq
                and k_codes.__class__ is T and k_codes.get_device() == dev and k_codes.dtype is u8
                and k_codes.is_contiguous() and k_codes.numel() >= nc
                and k_scales.__class__ is T and k_scales.get_device() == dev and k_scales.dtype is u8
                and k_scales.is_contiguous() and k_scales.numel() >= ns
                and v_codes.__class__ is T and v_codes.get_device() == dev and v_codes.dtype is u8
                and v_codes.is_contiguous() and v_codes.numel() >= nc
                and v_scales.__class__ is T and v_scales.get_device() == dev and v_scales.dtype is u8
                and v_scales.is_contiguous() and v_scales.numel() >= ns):
            end = (q.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
                   raw(dev) if stream is None else conv._stream(stream))
            first = x.data_ptr()
            index = (None if cosines is None else cosines.data_ptr(), None if sines is None else sines.data_ptr(),
                     None if pos is None else pos.data_ptr(), slots.data_ptr())
        else:
            end = (_take("q", q, nq, t), _take("k_codes", k_codes, nc, u8), _take("k_scales", k_scales, ns, u8),
                   _take("v_codes", v_codes, nc, u8), _take("v_scales", v_scales, ns, u8), conv._stream(stream))
            first = _take("x", x, nx, t)
            index = (_take("cosines", cosines, nt, f32), _take("sines", sines, nt, f32), _take("pos", pos, n, i32),
                     _take("slots", slots, n, i32))
        if (_lib or lib()).aih_kv4_append(
                self._ref, first, wq if wq is None else _take("wq", wq, self.d, t),
                wk if wk is None else _take("wk", wk, self.d, t), *index, *end):
            raise AihError(conv.last_error())
        return q


@dataclass(frozen=True)
class Kv4AttnSpec(_Spec):
    """Attention over a 4-bit cache; fields of aih_kv4_attn_desc (strides in elements, 0 = dense; scale None =
    1 / sqrt(d))."""

    nseq: int
    tokens: int
    hq: int
    hkv: int
    d: int
    page: int
    pages: int
    table_width: int
    causal: bool = True
    scale: float | None = None
    dt: DType = DType.F32
    max_len: int = 0
    q_stride: int = 0
    o_stride: int = 0

    def __post_init__(self):
        if self.scale is not None and not self.scale > 0:
            raise AihError(f"scale must be positive, not {self.scale!r}")
        desc = _AttnDesc(
            *(_u32(n, getattr(self, n)) for n in ("nseq", "tokens", "hq", "hkv", "d", "page", "pages", "table_width")),
            int(bool(self.causal)), self.scale or 0.0, int(self.dt), _u32("max_len", self.max_len),
            _u32("q_stride", self.q_stride), _u32("o_stride", self.o_stride))
        row, rows = self.hq * self.d, self.pages * self.hkv * self.page
        _keep(self, desc, (
            _span(self.tokens, self.q_stride or row, row), _span(self.tokens, self.o_stride or row, row),
            rows * (self.d // 2), rows * (self.d // 32), self.nseq * self.table_width))
        object.__setattr__(self, "_ws", None)

    def plan(self) -> Kv4AttnPlan:
        p = Kv4AttnPlan()
        conv._check(lib().aih_kv4_attn_plan(C.byref(self._desc), C.byref(p)))
        return p

    def workspace_bytes(self) -> int:
        if self._ws is None:
            object.__setattr__(self, "_ws", self.plan().ws_bytes)
        return self._ws

    def run(self, q, k_codes, k_scales, v_codes, v_scales, q_start, table, k_len, out, ws=None, stream=None):
        """q, out [tokens, hq, d]; the cache as kv4_cache makes it; q_start [nseq + 1], table [nseq, table_width], k_len
        [nseq] int32; ws: workspace_bytes() of device memory, made here if None."""
        T, device, raw, types, u8, i32 = _torch or _torch_types()
        t, b = types.get(self.dt), self.nseq
        nq, no, nc, ns, nt = self._sizes
        n = self._ws if self._ws is not None else self.workspace_bytes()
        if n:
            if ws is None:
                ws = _workspace_on(n, conv._device_of(out), stream)
            if ws.__class__ is not int and (ws.numel() * ws.element_size() < n or not ws.is_cuda
                                            or ws.get_device() != device() or not ws.is_contiguous()):
                raise AihError(f"the workspace needs {n} bytes, dense and on the current device, not "
                               f"{ws.numel() * ws.element_size()} on {ws.device}")
        if (out.__class__ is T and out.is_cuda and out.get_device() == (dev := device()) and out.dtype is t
                and out.is_contiguous() and out.numel() >= no
                and q.__class__ is T and q.get_device() == dev and q.dtype is t and q.is_contiguous()
                and q.numel() >= nq
                and k_codes.__class__ is T and k_codes.get_device() == dev and k_codes.dtype is u8
                and k_codes.is_contiguous() and k_codes.numel() >= nc
                and k_scales.__class__ is T and k_scales.get_device() == dev and k_scales.dtype is u8
                and k_scales.is_contiguous() and k_scales.numel() >= ns
                and v_codes.__class__ is T and v_codes.get_device() == dev and v_codes.dtype is u8
                and v_codes.is_contiguous() and v_codes.numel() >= nc
                and v_scales.__class__ is T and v_scales.get_device() == dev and v_scales.dtype is u8
                and v_scales.is_contiguous() and v_scales.numel() >= ns
                and q_start.__class__ is T and q_start.get_device() == dev and q_start.dtype is i32
                and q_start.is_contiguous() and q_start.numel() > b
                and table.__class__ is T and table.get_device() == dev and table.dtype is i32
                and table.is_contiguous() and table.numel() >= nt
                and k_len.__class__ is T and k_len.get_device() == dev and k_len.dtype is i32
                and k_len.is_contiguous() and k_len.numel() >= b):
            at = (q.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
                  q_start.data_ptr(), table.data_ptr(), k_len.data_ptr(), out.data_ptr(), conv._ptr(ws) if n else None, n,
                  raw(dev) if stream is None else conv._stream(stream))
        else:
            at = (_take("q", q, nq, t), _take("k_codes", k_codes, nc, u8), _take("k_scales", k_scales, ns, u8),
                  _take("v_codes", v_codes, nc, u8), _take("v_scales", v_scales, ns, u8),
                  _take("q_start", q_start, b + 1, i32), _take("table", table, nt, i32), _take("k_len", k_len, b, i32),
                  _take("out", out, no, t), conv._ptr(ws) if n else None, n, conv._stream(stream))
        if (_lib or lib()).aih_kv4_attn(self._ref, *at):
            raise AihError(conv.last_error())
        return out
