"""The 8-bit rows, their norm and their products in 64 bits, from the definition: what the tests hold the kernels to."""

from __future__ import annotations

import torch

from .attention_oracle import e4m3, scale_of

BLOCK = 128


def rounded(x: torch.Tensor) -> torch.Tensor:
    """Rows ``[m, k]`` in 8 bits, as the values they stand for; what is not finite becomes NaN."""
    x = x.double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at:at + BLOCK]
        finite = part.isfinite()
        scale = scale_of(torch.where(finite, part, 0.0).abs().amax(1))[:, None]
        out[:, at:at + BLOCK] = torch.where(finite, e4m3(torch.where(finite, part, 0.0) / scale) * scale, torch.nan)
    return out


def weight(w: torch.Tensor, gate_up: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``(values, scales)`` of a weight in 8 bits, with a scale per 128 x 128 of each half."""
    w = w.double()
    values, scales = [], []
    for half in w.chunk(2) if gate_up else (w,):
        of = torch.empty(-(-half.shape[0] // BLOCK), -(-half.shape[1] // BLOCK), dtype=torch.float64)
        got = torch.empty_like(half)
        for i in range(of.shape[0]):
            for j in range(of.shape[1]):
                at = slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK)
                part = half[at]
                finite = part.isfinite()
                of[i, j] = scale_of(torch.where(finite, part, 0.0).abs().amax())
                got[at] = torch.where(finite, e4m3(torch.where(finite, part, 0.0) / of[i, j]) * of[i, j], torch.nan)
        values.append(got)
        scales.append(of)
    return torch.cat(values), torch.cat(scales)


def norm(x: torch.Tensor, of: torch.Tensor | None, eps: float, residual: torch.Tensor | None = None):
    """``(norm in 64 bits, sum in x's type)``."""
    t = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    y = t.double()
    y = y / (y.square().mean(1, keepdim=True) + eps).sqrt()
    return (y if of is None else y * of.double()), t


def places(rows: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Where codes and scales of ``[rows, k]`` lie in their buffers."""
    frags = -(-rows // 16)
    r, c = torch.arange(rows)[:, None], torch.arange(k)
    codes = (((c // 128 * frags + r // 16) * 2 + c // 64 % 2) * 4 + c // 8 % 4) * 256 + r % 16 * 16 + c // 32 % 2 * 8 + c % 8
    b = torch.arange(-(-k // 128))
    return codes, ((b // 4 * frags + r // 16) * 16 + r % 16) * 4 + b % 4


def order(n: int, gate_up: bool) -> torch.Tensor:
    """The row of its fragments that each row of a weight lies in."""
    if not gate_up:
        return torch.arange(n)
    i = torch.arange(n // 2)
    gate = i // 16 * 32 + i % 16
    return torch.cat((gate, gate + 16))
