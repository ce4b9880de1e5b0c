"""Plain 64-bit forms of the MXFP4 and expert operators, from their definitions."""
from __future__ import annotations

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def blocks_of(k: int) -> int:
    return (k + 31) // 32


def quantize(x: torch.Tensor):
    """(codes, scales) of x [rows, k] on the CPU: the nearest of the eight magnitudes by trying them all."""
    rows, k = x.shape
    nb = blocks_of(k)
    v = torch.zeros(rows, nb * 32, dtype=torch.float64)
    v[:, :k] = x.cpu().double()
    v = v.view(rows, nb, 32)
    top = v.abs().amax(dim=2)
    finite = torch.isfinite(top)
    safe = torch.where(finite & (top > 0), top, torch.ones_like(top))
    e = torch.frexp(safe).exponent.double() - 1  # floor(log2), exact
    e = torch.where(top > 0, e - 2, torch.full_like(e, -127.0)).clamp(min=-127)
    a = torch.where(finite.unsqueeze(2), v, torch.zeros_like(v)) / torch.exp2(e).unsqueeze(2)
    far = (a.abs().unsqueeze(-1) - VALUES).abs()
    least = far.min(dim=-1, keepdim=True).values
    code = torch.arange(8).expand_as(far)
    tied = far == least
    even = torch.where(tied & (code % 2 == 0), code, 8).min(dim=-1).values  # of two nearest ones the even code
    odd = torch.where(tied, code, 8).min(dim=-1).values
    code = torch.where(even < 8, even, odd) + 8 * torch.signbit(v).long()
    code = torch.where(finite.unsqueeze(2), code, torch.zeros_like(code)).view(rows, -1)
    scales = torch.where(finite, e + 127, torch.full_like(e, 255.0)).to(torch.uint8)
    return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8), scales


def dequantize(codes: torch.Tensor, scales: torch.Tensor, k: int) -> torch.Tensor:
    """The values [..., k] in 64 bits."""
    c = codes.long()
    nibble = torch.stack([c % 16, c // 16], dim=-1).reshape(*scales.shape, 32)
    v = VALUES.to(codes.device)[nibble % 8]
    v = torch.where(nibble >= 8, -v, v)
    s = torch.exp2(scales.double() - 127.0)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (v * s.unsqueeze(-1)).reshape(*scales.shape[:-1], -1)[..., :k]


def random_weight(g: torch.Generator, shape, k: int, device, lo: int = 118, hi: int = 128):
    """Random codes and scales of a weight [*shape, k], zero past column k."""
    nb = blocks_of(k)
    codes = torch.randint(0, 256, (*shape, nb * 16), generator=g, device=device, dtype=torch.uint8)
    if k % 32:
        col = torch.arange(nb * 16, device=device) * 2
        codes = torch.where(col + 1 < k, codes, torch.where(col < k, codes & 15, torch.zeros_like(codes)))
    scales = torch.randint(lo, hi, (*shape, nb), generator=g, device=device, dtype=torch.uint8)
    return codes.contiguous(), scales


def sort(ids: torch.Tensor, experts: int):
    """(order, positions, offsets) with a stable sort on the CPU."""
    flat = ids.cpu().long().reshape(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True).indices
    kept = int((key < experts).sum())
    positions = torch.full_like(flat, -1)
    positions[order[:kept]] = torch.arange(kept)
    offsets = torch.tensor([int((key < e).sum()) for e in range(experts + 1)])
    return order, positions.view(ids.shape), offsets


#: The unit roundoff of each output type: a rounding is off by at most this times the value.
ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def close(y: torch.Tensor, want: torch.Tensor, size: torch.Tensor, adds: int) -> None:
    """y (of any type) against the exact sum ``want`` of ``adds`` terms whose magnitudes add up to ``size``:
    each FP32 addition (rounded or cut off) is off by at most 2^-23 of a partial sum, which is at most
    ``size``; the output's own rounding adds its unit roundoff, in FP16 at least half its smallest step.
    What FP16 rounds to infinity (65520 and more) is infinite, of the sum's sign."""
    u = ROUNDOFF[y.dtype]
    bound = (want.abs() + adds * 2.0 ** -23 * size) * u + adds * 2.0 ** -23 * size
    if y.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    off = (y.double() - want).abs()
    if y.dtype == torch.float16:
        off = torch.where(torch.isinf(y) & (y.sign() == want.sign()), 65520 - want.abs(), off)
    bad = ~(off <= bound)
    assert not bool(bad.any()), (int(bad.sum()), float(off[bad].max()), bad.nonzero()[:4].tolist())
