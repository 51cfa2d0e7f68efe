"""4-bit weights with group scales: quantisation and the storage format of ``ops.linear_w4``.

No counterpart in the reference, whose projections are bf16 ``nn.Linear`` layers
(src/helios/runtime/qwen3/layers.py:13-27,109-146).

A weight ``[n, k]`` is cut along k into groups; a group's values are ``(q - z) * s`` with codes
q in 0..15, a bf16 scale s and a zero point z (8 for symmetric weights, which store none).

``packed`` int32 ``[n, k / 8]``: word c of a row holds k = 8c .. 8c + 7, the even k's in its low 16
bits and the odd k's in its high 16 bits, four bits each in ascending k. So
``(word >> 4i) & 0x000F000F`` is the pair k = 8c + 2i, 8c + 2i + 1, which is what the kernel unpacks.
``scales`` and ``zeros`` are ``[k / group, n]``: neighbouring rows' values are neighbours in memory.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn

from helios_b200 import ops

GROUPS = (32, 64, 128)
NIBBLE_SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)  # bit position of k = 8c + i in word c


class W4Weight(NamedTuple):
    packed: torch.Tensor         # int32 [n, k / 8]
    scales: torch.Tensor         # bf16 [k / group, n]
    zeros: torch.Tensor | None   # uint8 [k / group, n]; None: 8

    @property
    def out_features(self) -> int:
        return self.packed.shape[0]

    @property
    def in_features(self) -> int:
        return self.packed.shape[1] * 8


def pack_w4(codes: torch.Tensor) -> torch.Tensor:
    """Codes 0..15 ``[n, k]`` (any integer type) to int32 words ``[n, k / 8]``."""
    if codes.dim() != 2 or codes.shape[1] % 8:
        raise ValueError("codes must be [n, k] with k a multiple of 8")
    codes = codes.to(torch.int32).reshape(codes.shape[0], -1, 8)
    packed = torch.zeros(codes.shape[:2], dtype=torch.int32, device=codes.device)
    for i, shift in enumerate(NIBBLE_SHIFTS):
        packed |= (codes[:, :, i] & 15) << shift
    return packed


def unpack_w4(packed: torch.Tensor) -> torch.Tensor:
    """int32 words ``[n, k / 8]`` to codes ``[n, k]`` (int32)."""
    shifts = torch.tensor(NIBBLE_SHIFTS, dtype=torch.int32, device=packed.device)
    return ((packed.unsqueeze(-1) >> shifts) & 15).reshape(packed.shape[0], -1)


def quantize_w4(weight: torch.Tensor, group_size: int = 128, *, symmetric: bool = True) -> W4Weight:
    """Round ``weight [n, k]`` to 4-bit codes, nearest value per element.

    Symmetric: ``s = max|w| / 7`` per group, codes ``8 + round(w / s)`` in 1..15. Otherwise
    ``s = (max - min) / 15`` over the group's values and 0, ``z = round(-min / s)``. Scales are
    rounded to bf16 first, so the codes belong to the scales that are stored; a group of zeros
    has scale 0."""
    if weight.dim() != 2:
        raise ValueError("weight must be [n, k]")
    n, k = weight.shape
    if group_size not in GROUPS or k % group_size:
        raise ValueError(f"group_size must be one of {GROUPS} and divide k = {k}")
    w = weight.detach().float().reshape(n, k // group_size, group_size)
    if not bool(torch.isfinite(w).all()):
        raise ValueError("weight has values that are not finite")
    if symmetric:
        scale = (w.abs().amax(-1) / 7).to(torch.bfloat16)
        zero = torch.full_like(scale, 8, dtype=torch.float32)
    else:
        low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        if not bool(torch.isfinite(high - low).all()):
            raise ValueError("weight has a group whose values span more than fp32 holds")
        scale = ((high - low) / 15).to(torch.bfloat16)
        zero = torch.where(scale > 0, (-low / scale.float()).round(), torch.zeros_like(low)).clamp(0, 15)
    s = scale.float().unsqueeze(-1)
    codes = torch.where(s > 0, (w / s).round(), torch.zeros_like(w)) + zero.unsqueeze(-1)
    packed = pack_w4(codes.clamp(0, 15).to(torch.int32).reshape(n, k))
    return W4Weight(packed, scale.t().contiguous(), None if symmetric else zero.t().to(torch.uint8).contiguous())


def dequantize_w4(weight: W4Weight, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The ``[n, k]`` values a W4Weight stands for."""
    groups, n = weight.scales.shape
    codes = unpack_w4(weight.packed).view(n, groups, -1).to(torch.float64)
    zeros = 8.0 if weight.zeros is None else (weight.zeros & 15).t().unsqueeze(-1).to(torch.float64)
    return ((codes - zeros) * weight.scales.t().unsqueeze(-1).to(torch.float64)).reshape(n, -1).to(dtype)


class W4Linear(nn.Module):
    """A bias-free Linear whose weight is held in 4 bits (``ops.linear_w4``). The tensors are
    buffers, so they move with the model; they are not part of its state dict."""

    def __init__(self, weight: W4Weight) -> None:
        super().__init__()
        for name in W4Weight._fields:
            self.register_buffer(name, getattr(weight, name), persistent=False)

    @property
    def weight(self) -> W4Weight:
        return W4Weight(self.packed, self.scales, self.zeros)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return ops.linear_w4(x, self.packed, self.scales, self.zeros)
