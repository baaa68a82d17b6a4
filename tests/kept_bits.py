"""How linear_act keeps h in bfloat16 before an activation's slope: the upper 16 bits of the fp32 value in `h`,
the next 4 of 8 adjacent channels in one word of `low`, lowest channel first."""
from __future__ import annotations

import torch

HALF = 2.0 ** -12  # half a step of the 12 significant bits that 20 hold, relative to the value


def pack(values: torch.Tensor, parts: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(h, low) of float32 values [rows, parts * outer], cut to 20 bits."""
    bits = values.contiguous().view(torch.int32).cpu().to(torch.int64) & 0xffffffff
    rows, outer = values.shape[0], values.shape[1] // parts
    h = ((bits >> 16) - ((bits >> 31) << 16)).to(torch.int16).view(torch.bfloat16)
    nibbles = torch.zeros(rows, parts, (outer + 7) // 8 * 8, dtype=torch.int64)
    nibbles[:, :, :outer] = (bits.reshape(rows, parts, outer) >> 12) & 15
    words = (nibbles.reshape(rows, parts, -1, 8) << (4 * torch.arange(8))).sum(-1)
    return h.to(values.device), (words - ((words >> 31) << 32)).to(torch.int32).to(values.device)


def unpack(h: torch.Tensor, low: torch.Tensor) -> torch.Tensor:
    """float32 values [rows, parts * outer] from h like that and low [rows, parts, words]."""
    rows, parts = low.shape[:2]
    nibbles = ((low.cpu().to(torch.int64)[..., None] >> (4 * torch.arange(8))) & 15).reshape(rows, parts, -1)
    outer = h.shape[1] // parts
    bits = (h.contiguous().view(torch.int16).cpu().to(torch.int64) & 0xffff) << 16
    bits = bits | (nibbles[:, :, :outer].reshape(rows, -1) << 12)
    return (bits - ((bits >> 31) << 32)).to(torch.int32).view(torch.float32).to(h.device)
