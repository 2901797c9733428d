"""MI355X (gfx950) backend for ai_engine's conv-as-GEMM path.

The product is the HIP library libaih_conv.so (sources in csrc/, C ABI in
include/aih_conv.h); `conv` is its host-side mirror of the reference's op
interface (GemmPwSpec / ConvIgemmSpec / ConvDwSpec / lower_op's Conv arm).
`attn` (include/aih_attn.h) adds the attention operators of hybrid networks,
`attn_block` an attention block that runs them between two pointwise convs.
`mx4` (include/aih_mx4.h) adds microscaled 4-bit rows and their pointwise conv.
"""
from . import attn, conv, mx4  # noqa: F401

__all__ = ["attn", "conv", "mx4"]
