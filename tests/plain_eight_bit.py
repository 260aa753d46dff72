"""Numbers in 8 bits from their definitions, in 64 bits: what the tests hold the kernels to."""

from __future__ import annotations

import torch

F64 = torch.float64
TOP = 448.0  # the largest e4m3 number


def grid(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number, ties to the even one; NaN for what is not finite."""
    x = x.to(F64)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6, max=2.0**10))) - 3.0)
    return torch.where(x.isfinite(), torch.round(x / step) * step, torch.nan)


def exponents(top: torch.Tensor) -> torch.Tensor:
    """The smallest e >= -126 with ``top <= 448 * 2^e``; 0 where top is 0."""
    e = torch.full(top.shape, -126, dtype=torch.int64, device=top.device)
    for k in range(-126, 121):
        e = torch.where(top > TOP * 2.0**k, k + 1, e)
    return torch.where(top > 0, e, 0)


def finite_top(x: torch.Tensor, dim) -> torch.Tensor:
    return torch.where(x.isfinite(), x.abs(), 0.0).amax(dim)


def quantize(x: torch.Tensor, rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values, scales)``, block by block."""
    x = x.to(F64)
    m, k = x.shape
    values, scales = torch.empty_like(x), torch.empty((-(-m // rows), -(-k // 128)), dtype=F64, device=x.device)
    for j, k0 in enumerate(range(0, k, 128)):
        piece = x[:, k0 : k0 + 128]
        tops = torch.stack([t.max() for t in finite_top(piece, 1).split(rows)])
        scales[:, j] = torch.exp2(exponents(tops).to(F64))
        values[:, k0 : k0 + 128] = grid(piece / scales[:, j].repeat_interleave(rows)[:m, None])
    return values, scales


def spread(scales: torch.Tensor, rows: int, m: int, k: int) -> torch.Tensor:
    return scales.to(F64).repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def linear(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The product, and the sum of its terms' sizes (what the roundings of its 32-bit sums are relative to)."""
    values, scales = quantize(x)
    left, right = values * spread(scales, 1, *x.shape), w.to(F64) * spread(w_scales, 128, *w.shape)
    return left @ right.t(), left.abs() @ right.abs().t()


def turn(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Heads ``[n, heads, D]`` rotated (pairs ``(j, j + D/2)``) as 32-bit numbers: two products and a sum, each rounded."""
    d = x.shape[-1]
    row = table[positions.long().clamp(0, table.shape[0] - 1)][:, None]
    c, s, a, b = row[..., : d // 2], row[..., d // 2 :], x[..., : d // 2].float(), x[..., d // 2 :].float()
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def attention(q, keys, values, first_position: int, scale: float, window: int | None) -> torch.Tensor:
    """One request: ``q [n, H, D]`` at positions ``first_position ..``, ``keys`` / ``values [len, KV, D]``; rows without a key are zeros."""
    n, heads, d = q.shape
    group = heads // keys.shape[1]
    out = torch.zeros((n, heads, d), dtype=F64, device=q.device)
    for i in range(n):
        p = first_position + i
        lo, hi = (0 if window is None else max(0, p - window + 1)), min(p + 1, keys.shape[0])
        if hi <= lo:
            continue
        k, v = (x[lo:hi].to(F64).repeat_interleave(group, 1) for x in (keys, values))
        s = torch.einsum("hd,jhd->hj", q[i].to(F64), k) * scale
        out[i] = torch.einsum("hj,jhd->hd", torch.softmax(s, 1), v)
    return out
