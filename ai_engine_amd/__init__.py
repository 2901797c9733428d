"""MI355X (gfx950) backend for ai_engine's conv-as-GEMM path.

The product is the HIP library libaih_conv.so (sources in csrc/, C ABI in
include/aih_conv.h); `conv` is its host-side mirror of the reference's op
interface (GemmPwSpec / ConvIgemmSpec / ConvDwSpec / lower_op's Conv arm).
`attn` (include/aih_attn.h) adds the attention operators of hybrid networks,
`attn_block` an attention block that runs them between two pointwise convs.
"""
from . import attn, conv  # noqa: F401

__all__ = ["attn", "conv"]
