"""The 8-bit codes of AdamW's moments, in torch operations (any device).

The GPU step (csrc/kernels/adamw.hip, which explains the format) encodes and decodes by itself;
this is the same format for optimizer states on the CPU and for moments that come from outside (a
checkpoint of a 32-bit state).  64 neighbouring elements share a scale byte s, the unit 2**(s-127)
of their codes; a code is a float with 4 exponent bits, linear below its first binade.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

BLOCK = 64
M_BITS, ROOT_BITS = 3, 4  # mantissa bits: first moment (with a sign bit), root of the second
_HASH_STEP, _HASH_HIGH, _HASH_1, _HASH_2 = 0x632BE5AB, 0x27D4A62F, 0x6E7A3B15, 0x35D2C1A7
_MASK = 0xFFFFFFFF


def dither(numel: int, step: int, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The 16 + 16 bits that round the codes of step number ``step``, for every place of the state."""
    i = torch.arange(numel, device=device, dtype=torch.int64)
    x = ((i & _MASK) + (i >> 32) * _HASH_HIGH + int(step) * _HASH_STEP) & _MASK
    x = ((x ^ (x >> 16)) * _HASH_1) & _MASK
    x = ((x ^ (x >> 15)) * _HASH_2) & _MASK
    x = x ^ (x >> 16)
    return (x & 0xFFFF).int(), (x >> 16).int()


def encode(x: torch.Tensor, mantissa: int, bits16: Optional[torch.Tensor] = None):
    """``(codes, scale bytes)`` of fp32 values (a multiple of 64 of them); ``bits16``: 16 random bits
    each, None rounds to the nearest.  A root that is not zero keeps a code that is not zero."""
    one, drop = 1 << mantissa, 23 - mantissa
    a = x.abs().view(-1, BLOCK)
    top = a.amax(1)
    bad = ~torch.isfinite(top)
    a = torch.where(bad[:, None], torch.zeros_like(a), a)
    last = ((2 * one - 1) << drop) - (1 << 23)
    scale = (((top.view(torch.int32) + (0x7FFFFF - last)) >> 23) - (14 + mantissa)).clamp(min=1)
    scale = torch.where(bad, torch.full_like(scale, 255), scale)
    unit = (254 - torch.where(bad, torch.full_like(scale, 127), scale)) << 23
    y = (a * unit.view(torch.float32)[:, None]).view(-1)
    low = y < one  # adding `one` puts the linear part into that binade
    part = torch.where(low, y + one, y).view(torch.int32) - (low.int() << 23) - ((126 + mantissa) << 23)
    half = 1 << 15 if bits16 is None else bits16
    code = (part + (half << (drop - 16)) + (1 << (drop - 17))) >> drop
    if mantissa == ROOT_BITS:
        code = torch.maximum(code, (a.view(-1) > 0).int())
    else:
        # the sign bit, of zeros too, as the kernel keeps it: a value that rounded to -0 is code 0x80
        code = code | (torch.signbit(x) & ~bad.repeat_interleave(BLOCK)).int() << 7
    return code.to(torch.uint8), scale.to(torch.uint8)


def decode(codes: torch.Tensor, scales: torch.Tensor, mantissa: int) -> torch.Tensor:
    """The fp32 values of codes; NaN in a block whose scale byte is 255."""
    one = 1 << mantissa
    c = codes.int()
    sign = 1.0
    if mantissa == M_BITS:
        sign, c = 1.0 - 2.0 * (c >> 7), c & 127
    low = c < one
    value = ((c << (23 - mantissa)) + (low.int() << 23) + ((126 + mantissa) << 23)).view(torch.float32)
    value = (value - low * float(one)) * sign
    s = scales.int()
    unit = (torch.where(s == 255, torch.zeros_like(s), s) << 23).view(torch.float32)
    unit = torch.where(s == 255, torch.full_like(unit, float("nan")), unit)
    return (value.view(-1, BLOCK) * unit[:, None]).view(-1)
