"""The paged cache and its attention in 64 bits, token by token from the definition: what the tests hold the
kernels to. Values are found by their places in the buffers, and a sequence is taken at a time."""

from __future__ import annotations

import math

import torch

E4M3_TOP = 448.0
LEAST_EXPONENT = -64


def place(name: str, e4m3: bool, token: torch.Tensor, dim: torch.Tensor) -> torch.Tensor:
    """Element of a 16 x 64 unit that holds (token % 16, dim % 64)."""
    n, e = token % 16, dim % 64
    if e4m3:
        return e // 16 * 256 + n * 16 + e % 16 if name == "k" else n // 4 * 256 + e // 4 * 16 + e % 4 * 4 + n % 4
    if name == "k":
        return e // 8 % 2 * 512 + e // 16 * 128 + n * 8 + e % 8
    return e // 2 % 2 * 512 + n // 4 * 128 + e // 4 * 8 + e % 2 * 4 + n % 4


def _flat(x: torch.Tensor, page: int, heads: int, size: int, dim: int, name: str) -> torch.Tensor:
    """Index into the flattened buffer of page ``page``: [size, heads, dim]."""
    chunks = -(-dim // 64)
    n, h, d = torch.arange(size)[:, None, None], torch.arange(heads)[None, :, None], torch.arange(dim)
    unit = ((page * heads + h) * (size // 16) + n // 16) * chunks + d // 64
    return unit * 1024 + place(name, x.dtype == torch.float8_e4m3fn, n, d)


def _bits(x: torch.Tensor) -> torch.Tensor:
    return x.view(torch.uint8 if x.dtype == torch.float8_e4m3fn else torch.int16).flatten()


def get_page(x: torch.Tensor, scale: torch.Tensor | None, page: int, heads: int, size: int, dim: int, name: str) -> torch.Tensor:
    """Values of one page, [size, heads, dim] float64 on the CPU."""
    at = _flat(x, page, heads, size, dim, name).to(x.device)
    got = _bits(x)[at].view(x.dtype).cpu().to(torch.float32).double()
    return got if scale is None else got * scale[page].cpu().double()[None, :, None]


def put_page(x: torch.Tensor, page: int, values: torch.Tensor, name: str) -> None:
    """Writes [size, heads, dim] elements of x's type into one page."""
    size, heads, dim = values.shape
    at = _flat(x, page, heads, size, dim, name).to(x.device)
    _bits(x)[at.flatten()] = _bits(values.contiguous().to(x.device))


def scale_of(largest: torch.Tensor) -> torch.Tensor:
    """Least power of two s >= 2^-64 with largest <= 448 s."""
    s = torch.full_like(largest.double(), 2.0 ** LEAST_EXPONENT)
    while bool((low := largest.double() > E4M3_TOP * s).any()):
        s = torch.where(low, 2 * s, s)
    return s


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value of |x| <= 448, ties to even, in 64 bits."""
    grid = torch.tensor([math.ldexp(c, -9) if c < 8 else math.ldexp(8 + c % 8, c // 8 - 10) for c in range(127)],
                        dtype=torch.float64)
    a = x.abs().clamp(max=E4M3_TOP).contiguous()
    hi = torch.searchsorted(grid, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), grid[hi], grid[lo]) * torch.sign(x)


def rotate(x: torch.Tensor, turn: torch.Tensor | None, side_by_side: bool) -> torch.Tensor:
    """[rows, heads, dim] turned by [rows, rotary] cosines and sines, in 64 bits."""
    x = x.double().clone()
    if turn is None:
        return x
    half = turn.shape[1] // 2
    c, s = turn[:, None, :half].double(), turn[:, None, half:].double()
    i = torch.arange(half)
    first, second = (2 * i, 2 * i + 1) if side_by_side else (i, i + half)
    a, b = x[..., first], x[..., second]
    x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    return x


def round_rows(k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """A round's rows: [rows, rows] what each sees among them, and their places after the context."""
    rows = k + k * k
    see, places = torch.zeros((rows, rows), dtype=torch.bool), torch.zeros(rows, dtype=torch.int64)
    for i in range(k):
        see[i, : i + 1] = True
        places[i] = i
        for j in range(k):
            r = k + i * k + j
            see[r, : i + 1] = True
            see[r, k + i * k: r + 1] = True
            places[r] = i + 1 + j
    return see, places


def seen(context: int, rows: int, tokens: int, window: int | None, sinks: int, see: torch.Tensor | None,
         places: torch.Tensor | None) -> torch.Tensor:
    """[rows, tokens]: what each row of a sequence sees. ``places`` are absolute positions."""
    t, r = torch.arange(tokens)[None, :], torch.arange(rows)[:, None]
    out = t <= context + r
    if see is not None:
        among = torch.zeros((rows, tokens), dtype=torch.bool)
        most = min(rows, tokens - context)
        if most > 0:
            among[:, context:context + most] = see[:rows, :most]
        out = (t < context) | among
    if window is not None:
        at = (places if places is not None else context + torch.arange(rows))[:, None]
        near = (t > at - window) | (t < sinks)
        out = out & (near | (t >= context) if see is not None else near)
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, visible: torch.Tensor, scale: float):
    """q [rows, heads, dim], k and v [tokens, kv_heads, dim], visible [rows, tokens]: the output, the same of
    |values|, and the largest sum of |q k| scale of a visible pair; all in 64 bits. Rows that see nothing are 0."""
    q, k, v = q.double(), k.double(), v.double()
    group = q.shape[1] // k.shape[1]
    out, size, most = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for h in range(q.shape[1]):
        kh, vh = k[:, h // group], v[:, h // group]
        s = (q[:, h] @ kh.T * scale).masked_fill(~visible, -math.inf)
        p = torch.softmax(s, -1).masked_fill(~visible, 0.0).nan_to_num(0.0)
        out[:, h], size[:, h] = p @ vh, p @ vh.abs()
        if visible.any():
            most = max(most, float((q[:, h].abs() @ kh.abs().T * scale)[visible].max()))
    return out, size, most
