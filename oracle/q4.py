"""The 4-bit cache row in 64-bit arithmetic (values, and a row's bytes).

A row holds one head's 128 values of one token in 72 bytes; the layout and the
rounding rules are those of ``include/retree_b200.h`` (RT_Q4_ROW_BYTES).  The
reference has no cache below 16 bits, so this follows the format's definition.
"""

from __future__ import annotations

import torch

ROW_BYTES = 72
GROUP = 32


def quantise(x: torch.Tensor):
    """``(u, z, s)`` of rows ``[..., 128]``: codes ``[..., 4, 32]``, zero points and scales ``[..., 4, 1]`` (float64)."""
    g = x.double().unflatten(-1, (4, GROUP))
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    lo = torch.minimum(g.amin(-1, keepdim=True), zero)
    hi = torch.maximum(g.amax(-1, keepdim=True), zero)
    mant, expo = torch.frexp((hi - lo) / 15)
    s = torch.ldexp(torch.ceil(mant * 16) / 16, expo)
    # (hi - lo may have lost its small end even in 64 bits; 15 s less the large end loses nothing)
    short = 15 * s - torch.maximum(hi, -lo) < torch.minimum(hi, -lo)
    s = torch.where(short, s + torch.ldexp(torch.full_like(s, 1 / 16), torch.frexp(s)[1]), s)
    s = torch.where(s < 2.0 ** -126, zero, s)
    d = torch.where(s == 0, 1.0, s)
    z = torch.round(-lo / d)
    u = torch.clamp(torch.round(g / d) + z, 0, 15)
    flat = s == 0
    bad = ~torch.isfinite(x).all(-1, keepdim=True).unsqueeze(-1).expand_as(s)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    z = torch.where(flat | bad, zero, z)
    u = torch.where(flat | bad, zero, u)
    return u, z, s


def values(x: torch.Tensor) -> torch.Tensor:
    """What rows ``[..., 128]`` read as once they are in the cache (float64)."""
    u, z, s = quantise(x)
    return ((u - z) * s).flatten(-2)


def pack(x: torch.Tensor) -> torch.Tensor:
    """The bytes ``[..., 72]`` of rows ``[..., 128]``."""
    u, z, s = quantise(x)
    codes = u.flatten(-2).to(torch.int64).unflatten(-1, (16, 8))
    word = torch.zeros(codes.shape[:-1], dtype=torch.int64, device=x.device)
    for d in range(8):
        word |= codes[..., d] << (4 * (d // 2 + 4 * (d % 2)))
    sbits = (s.float().view(torch.int32).to(torch.int64) >> 16) & 0x7FF0
    sbits = torch.where(torch.isnan(s), torch.full_like(sbits, 0x7FF0), sbits)
    meta = (sbits | z.nan_to_num().to(torch.int64)).squeeze(-1)
    b = [(word >> (8 * i)) & 255 for i in range(4)]
    m = [(meta >> (8 * i)) & 255 for i in range(2)]
    return torch.cat([torch.stack(b, -1).flatten(-2), torch.stack(m, -1).flatten(-2)], -1).to(torch.uint8)


def unpack(rows: torch.Tensor) -> torch.Tensor:
    """float64 values ``[..., 128]`` of the bytes ``[..., 72]``."""
    r = rows.to(torch.int64)
    word = sum(r[..., i:64:4] << (8 * i) for i in range(4))
    meta = r[..., 64::2] | (r[..., 65::2] << 8)
    s = ((meta & 0x7FF0) << 16).to(torch.int32).view(torch.float32).double()
    s = torch.where((meta & 0x7F80) == 0, torch.zeros_like(s), s)
    out = torch.stack([(word >> (4 * (d // 2 + 4 * (d % 2)))) & 15 for d in range(8)], -1).flatten(-2).double()
    out = out.unflatten(-1, (4, GROUP))
    return ((out - (meta & 15).double().unsqueeze(-1)) * s.unsqueeze(-1)).flatten(-2)
