"""Host side of the operators on microscaled 4-bit rows (include/aih_mx4.h).

* `Mx4QuantSpec`   -> aih_mx4_quant: rows of a storage type to 4 bits
* `Mx4DequantSpec` -> aih_mx4_dequant: the values that 4-bit rows stand for
* `Mx4PwSpec`      -> aih_mx4_pw: the 1x1 conv of 4-bit rows and 4-bit weights

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
from dataclasses import dataclass

from . import conv
from .attn import _u32
from .conv import Activation, AihError, DType


class _QuantDesc(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("k", C.c_uint32), ("dt", C.c_int32), ("x_stride", C.c_uint64)]


class _DequantDesc(C.Structure):
    _fields_ = [("rows", C.c_uint32), ("k", C.c_uint32), ("dt", C.c_int32), ("code_stride", C.c_uint32),
                ("scale_stride", C.c_uint32), ("y_stride", C.c_uint64)]


class _PwDesc(C.Structure):
    _fields_ = [("m", C.c_uint32), ("k", C.c_uint32), ("cout", C.c_uint32), ("act", C.c_int32),
                ("residual", C.c_int32), ("dt", C.c_int32)]


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
        }
        for name, args in sigs.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = C.c_int, args
        _lib = L
    return _lib


_torch = None  # torch's Tensor, current device, and the types of DType, codes and index arrays


def _torch_types():
    global _torch
    import torch

    _torch = (torch.Tensor, torch.cuda.current_device, {0: torch.float32, 1: torch.float16, 2: torch.bfloat16},
              torch.uint8, torch.int32)
    return _torch


def _take(name, t, n, dtype, device):
    """The device address of `n` values; refuses a tensor that the kernels would read as other values, past its end
    or on another device. None and raw addresses are the caller's, as everywhere."""
    if t is None or t.__class__ is int:
        return t
    if device is None:  # the call's other tensors are raw addresses
        device = _torch[1]()
    if t.dtype is dtype and t.get_device() == device and t.is_contiguous() and t.numel() >= n:
        return t.data_ptr()
    raise AihError(f"{name} must be a dense tensor of at least {n} {dtype} on the current device, not {tuple(t.shape)} "
                   f"{t.dtype} on {t.device}" + ("" if t.is_contiguous() else ", not dense"))


def code_bytes(k: int) -> int:
    """Bytes of a row's codes, as Mx4QuantSpec writes them."""
    return -(-k // 128) * 64


def scale_bytes(k: int) -> int:
    """Bytes of a row's scales, as Mx4QuantSpec writes them."""
    return -(-k // 512) * 16


def _span(rows, stride, last):
    """Values that rows `stride` apart reach over, the last one `last` long."""
    return (rows - 1) * stride + last if rows else 0


@dataclass(frozen=True)
class Mx4QuantSpec:
    """Rows to 4 bits; fields of aih_mx4_quant_desc (x_stride in elements, 0 = dense)."""

    rows: int
    k: int
    dt: DType = DType.F32
    x_stride: int = 0

    def __post_init__(self):
        object.__setattr__(self, "_desc", _QuantDesc(_u32("rows", self.rows), _u32("k", self.k), int(self.dt),
                                                     _u32("x_stride", self.x_stride)))
        object.__setattr__(self, "_sizes", (_span(self.rows, self.x_stride or self.k, self.k),
                                            self.rows * self.code_bytes, self.rows * self.scale_bytes))

    @property
    def code_bytes(self) -> int:
        return code_bytes(self.k)

    @property
    def scale_bytes(self) -> int:
        return scale_bytes(self.k)

    def run(self, x, codes, scales, stream=None):
        """x [rows, x_stride]; codes [rows, code_bytes], scales [rows, scale_bytes] uint8."""
        T, device, types, u8, _ = _torch or _torch_types()
        dev, (nx, nc, ns) = device() if x.__class__ is T else None, self._sizes
        if (_lib or lib()).aih_mx4_quant(
                C.byref(self._desc), _take("x", x, nx, types.get(self.dt), dev), _take("codes", codes, nc, u8, dev),
                _take("scales", scales, ns, u8, dev), conv._stream(stream)):
            raise AihError(conv.last_error())
        return codes, scales


@dataclass(frozen=True)
class Mx4DequantSpec:
    """4-bit rows to values; fields of aih_mx4_dequant_desc (strides: bytes of codes and scales, elements of y)."""

    rows: int
    k: int
    dt: DType = DType.F32
    code_stride: int = 0
    scale_stride: int = 0
    y_stride: int = 0

    def __post_init__(self):
        object.__setattr__(self, "_desc", _DequantDesc(
            _u32("rows", self.rows), _u32("k", self.k), int(self.dt), _u32("code_stride", self.code_stride),
            _u32("scale_stride", self.scale_stride), _u32("y_stride", self.y_stride)))
        blocks = -(-self.k // 32)
        object.__setattr__(self, "_sizes", (
            _span(self.rows, self.code_stride or code_bytes(self.k), blocks * 16),
            _span(self.rows, self.scale_stride or scale_bytes(self.k), blocks),
            _span(self.rows, self.y_stride or self.k, self.k)))

    def run(self, codes, scales, y, stream=None):
        """codes, scales uint8; y [rows, y_stride]."""
        T, device, types, u8, _ = _torch or _torch_types()
        dev, (nc, ns, ny) = device() if y.__class__ is T else None, self._sizes
        if (_lib or lib()).aih_mx4_dequant(
                C.byref(self._desc), _take("codes", codes, nc, u8, dev), _take("scales", scales, ns, u8, dev),
                _take("y", y, ny, types.get(self.dt), dev), conv._stream(stream)):
            raise AihError(conv.last_error())
        return y


@dataclass(frozen=True)
class Mx4PwSpec:
    """The 1x1 conv of 4-bit rows; fields of aih_mx4_pw_desc."""

    m: int
    k: int
    cout: int
    act: Activation = Activation.NONE
    residual: bool = False
    dt: DType = DType.F32

    def __post_init__(self):
        object.__setattr__(self, "_desc", _PwDesc(
            *(_u32(n, getattr(self, n)) for n in ("m", "k", "cout")), int(self.act), int(bool(self.residual)),
            int(self.dt)))
        cb, sb = code_bytes(self.k), scale_bytes(self.k)
        object.__setattr__(self, "_sizes", (self.m * cb, self.m * sb, self.cout * cb, self.cout * sb, self.m * self.cout))

    def run(self, x_codes, x_scales, w_codes, w_scales, bias, res, y, stream=None):
        """Codes and scales as Mx4QuantSpec makes them, of x [m, k] and of the weights [cout, k]; bias [cout] or None;
        res (with `residual`) and y [m, cout]."""
        T, device, types, u8, _ = _torch or _torch_types()
        dev, (nxc, nxs, nwc, nws, ny), t = device() if y.__class__ is T else None, self._sizes, types.get(self.dt)
        if (_lib or lib()).aih_mx4_pw(
                C.byref(self._desc), _take("x_codes", x_codes, nxc, u8, dev), _take("x_scales", x_scales, nxs, u8, dev),
                _take("w_codes", w_codes, nwc, u8, dev), _take("w_scales", w_scales, nws, u8, dev),
                _take("bias", bias, self.cout, t, dev), _take("res", res, ny if self.residual else 0, t, dev),
                _take("y", y, ny, t, dev), conv._stream(stream)):
            raise AihError(conv.last_error())
        return y
