"""The microscaled 4-bit format written out in 64 bits, for the tests: a block of 32
elements has the scale 2^e, e = max(floor(log2 max|x|) - 2, -127), and an element is
the nearest of 0 .5 1 1.5 2 3 4 6 scales, ties to the even code, above 6 scales 6."""
from __future__ import annotations

import torch

from ai_engine_amd.conv import DType
from ai_engine_amd.mx4 import code_bytes, scale_bytes

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
TORCH = {DType.F32: torch.float32, DType.F16: torch.float16, DType.BF16: torch.bfloat16}
DTS = [DType.F32, DType.F16, DType.BF16]
IDS = ["f32", "f16", "bf16"]


def blocks_of(x):
    """(codes, scale bytes) of x [..., 32], any float type: whole numbers."""
    x = x.double().cpu()
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    top = torch.where(bad, 1.0, top)
    e = torch.frexp(top)[1].long() - 1 - 2  # frexp: top = f 2^e, f in [1/2, 1)
    e = torch.where(top == 0, -127, e.clamp(min=-127))
    a = torch.ldexp(torch.where(bad[..., None], 0.0, x.abs()), -e[..., None])
    dist = (a[..., None] - GRID).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best
    even = torch.arange(8) % 2 == 0
    # of two as near the even code
    code = torch.where((near & even).any(-1), (near & even).long().argmax(-1), near.long().argmax(-1))
    code = code + 8 * torch.signbit(x).long()
    return torch.where(bad[..., None], 0, code).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def quant_rows(x):
    """codes [rows, code_bytes(k)] and the scales of whole 128s [rows, code_bytes(k) / 16]."""
    rows, k = x.shape
    kp = 2 * code_bytes(k)
    wide = torch.zeros(rows, kp, dtype=torch.float64)
    wide[:, :k] = x.double().cpu()
    codes, scales = blocks_of(wide.view(rows, -1, 32))
    return pack(codes).view(rows, -1), scales


def values(codes, scales):
    """fp64 values [rows, 32 blocks] of codes [rows, 16 blocks] and scales [rows, at least blocks]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).cpu().long()
    v = GRID[c & 7] * torch.where(c >= 8, -1.0, 1.0)
    s = scales[:, :codes.shape[1] // 16].cpu().long()
    size = torch.where(s == 255, float("nan"), torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s - 127))
    return v * size.repeat_interleave(32, -1)


def row_buffers(rows, k, device="cuda:0"):
    return (torch.full((rows, code_bytes(k)), 0x77, dtype=torch.uint8, device=device),
            torch.full((rows, scale_bytes(k)), 0x77, dtype=torch.uint8, device=device))
