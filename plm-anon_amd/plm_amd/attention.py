"""Attention over a paged cache of keys and values on the HIP library: what runs between a round's QKV
and attn-out linears.

* ``PagedCache`` — the handle on a cache's tensors, in the model's 16 bits or as e4m3 codes with a
  power-of-two scale per page and head (half the bytes that a decoding step reads);
* ``append_kv`` — rotates a call's queries and keys by their positions and stores keys and values;
* ``attend`` — attention of the rows over the cache: causal or with a round's own mask, whole or through a
  sliding window with the first tokens kept (sinks);
* ``read_kv`` — cached tokens back as values;
* ``round_mask`` — mask and places of a round's k + k*k rows.

Rows are packed: ``total`` rows of ``seqs`` sequences one after the other, sequence b's in
``[row_starts[b], row_starts[b + 1])`` (``None``: the same number each). They follow ``lengths[b]``
cached tokens; token t of sequence b lies in page ``table[b, t // page]``. ``lengths``, ``row_starts`` and
``positions`` are int64 tensors on the GPU and are never read on the host, so every call can be captured
in a HIP graph and replayed as the sequences grow; only ``max_rows`` (the longest sequence's rows) and the
tensors' shapes size a launch. Table entries outside the cache are pages that are not there.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

PAGES = (16, 32, 64, 128)
MAX_HEAD_DIM = 256
MAX_ROPE_ROWS = 1 << 30
_TYPES = {torch.bfloat16: _lib.PLM_CACHE_BF16, torch.float16: _lib.PLM_CACHE_F16, torch.float8_e4m3fn: _lib.PLM_CACHE_E4M3}
LEAST_SCALE = 2.0 ** -64   # of an 8-bit page that holds nothing but zeros


def _shapes(pages: int, kv_heads: int, page: int, head_dim: int, e4m3: bool) -> tuple[tuple, tuple]:
    lead = (pages, kv_heads, page // 16, -(-head_dim // 64))
    return (lead + (4, 16, 16), lead + (4, 16, 4, 4)) if e4m3 else (lead + (2, 4, 16, 8), lead + (2, 4, 16, 2, 4))


class PagedCache:
    """Keys and values of ``kv_heads`` heads in pages of 16, 32, 64 or 128 tokens. The tensors are used as they
    are, in the order the matrix instructions read (``include/plm_amd.h`` states it): 16-bit
    ``k [pages, kv_heads, page / 16, ceil(head_dim / 64), 2, 4, 16, 8]`` and ``v [.., 2, 4, 16, 2, 4]``, or e4m3
    ``k [.., 4, 16, 16]`` and ``v [.., 4, 16, 4, 4]`` with float32 ``k_scale`` and ``v_scale``
    ``[pages, kv_heads]``, powers of two. Dimensions past ``head_dim`` hold zeros. ``PagedCache.empty``
    allocates one."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, *, head_dim: int):
        if k.dtype not in _TYPES or v.dtype != k.dtype:
            raise TypeError(f"a cache is bf16, fp16 or float8_e4m3fn, keys and values alike, got {k.dtype} and {v.dtype}")
        if not 8 <= head_dim <= MAX_HEAD_DIM or head_dim % 8:
            raise ValueError(f"head_dim must be a multiple of 8 in [8, {MAX_HEAD_DIM}], got {head_dim}")
        if k.dim() < 4 or k.shape[0] < 1 or k.shape[1] < 1 or 16 * k.shape[2] not in PAGES:
            raise ValueError(f"keys must be [pages, kv_heads, page / 16, ...] with pages of {PAGES} tokens, got {tuple(k.shape)}")
        e4m3 = k.dtype == torch.float8_e4m3fn
        pages, heads, page = k.shape[0], k.shape[1], 16 * k.shape[2]
        wanted = _shapes(pages, heads, page, head_dim, e4m3)
        if (tuple(k.shape), tuple(v.shape)) != wanted:
            raise ValueError(f"keys and values of {pages} pages of {page} tokens, {heads} heads of {head_dim} must be "
                             f"{wanted[0]} and {wanted[1]}, got {tuple(k.shape)} and {tuple(v.shape)}")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("a cache's keys and values must be contiguous")
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            if e4m3 != (s is not None):
                raise ValueError(f"{name} goes with an e4m3 cache, and with no other")
            if s is not None and (s.shape != (pages, heads) or s.dtype != torch.float32 or not s.is_contiguous()
                                  or s.device != k.device):
                raise ValueError(f"{name} must be a contiguous float32 [{pages}, {heads}] tensor on {k.device}")
        if not k.is_cuda or v.device != k.device:
            raise RuntimeError(f"a cache lives on one GPU; got {k.device} and {v.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page, self.head_dim, self.dtype = pages, heads, page, head_dim, k.dtype
        self.device = k.device
        self._handle = _lib.KvCache(k.data_ptr(), v.data_ptr(), 0 if k_scale is None else k_scale.data_ptr(),
                                    0 if v_scale is None else v_scale.data_ptr(), pages, heads, page, head_dim,
                                    _TYPES[k.dtype])
        self._ref = ctypes.byref(self._handle)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, *, page: int = 64,
              dtype: torch.dtype = torch.float8_e4m3fn, device: torch.device | str = "cuda") -> "PagedCache":
        """A cache of ``pages`` zeroed pages; ``dtype`` float8_e4m3fn (8 bits), bfloat16 or float16."""
        if dtype not in _TYPES:
            raise TypeError(f"a cache is bf16, fp16 or float8_e4m3fn, got {dtype}")
        if page not in PAGES or pages < 1 or kv_heads < 1 or head_dim < 1:
            raise ValueError(f"pages of {PAGES} tokens, at least one page and head required, got page={page}, "
                             f"pages={pages}, kv_heads={kv_heads}, head_dim={head_dim}")
        e4m3 = dtype == torch.float8_e4m3fn
        shapes = _shapes(pages, kv_heads, page, head_dim, e4m3)
        if e4m3:
            k, v = (torch.zeros(s, dtype=torch.uint8, device=device).view(dtype) for s in shapes)
            scales = [torch.full((pages, kv_heads), LEAST_SCALE, device=k.device) for _ in range(2)]
        else:
            k, v = (torch.zeros(s, dtype=dtype, device=device) for s in shapes)
            scales = [None, None]
        return cls(k, v, *scales, head_dim=head_dim)


def _index(t: torch.Tensor, name: str, shape: tuple, dev: torch.device) -> int:
    if t.dtype != torch.int64 or t.shape != shape or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int64 {list(shape)} tensor on {dev}, got {t.dtype} "
                         f"{list(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, total: int, heads: int | None, dim: int,
          dev: torch.device) -> torch.Tensor:
    """``t`` as [rows, heads, dim] rows that a kernel can read: dimensions contiguous, rows and heads on 16 bytes."""
    if t.dim() != 3 or t.shape[0] != total or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [{total}, {'heads' if heads is None else heads}, {dim}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != dev:
        raise RuntimeError(f"{name} must be on the cache's GPU {dev}, got {t.device}")
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _call(cache: PagedCache, total: int, table: torch.Tensor, lengths: torch.Tensor, row_starts: torch.Tensor | None,
          max_rows: int | None) -> tuple[int, tuple]:
    """``(max_rows, arguments)`` of a call's rows, from ``total`` to ``row_starts`` of the C entries."""
    dev = cache.device
    if table.dim() != 2 or table.dtype != torch.int32 or table.device != dev or table.shape[1] < 1 or table.stride(1) != 1:
        raise ValueError(f"table must be an int32 [seqs, pages] tensor with contiguous rows on {dev}, got {table.dtype} "
                         f"{tuple(table.shape)} on {table.device}")
    seqs, width = table.shape
    if row_starts is None:
        if seqs < 1 or total % seqs:
            raise ValueError(f"{total} rows are no whole number for each of {seqs} sequences: row_starts is needed")
        each = total // seqs
        if max_rows is not None and max_rows != each:
            raise ValueError(f"max_rows must be {each} for {total} rows of {seqs} sequences, got {max_rows}")
        max_rows, starts = each, None
    else:
        starts = _index(row_starts, "row_starts", (seqs + 1,), dev)
        if max_rows is None:
            max_rows = total
        elif not 1 <= max_rows <= total:
            raise ValueError(f"max_rows must be in [1, {total}], got {max_rows}")
    stride = table.stride(0) if seqs > 1 else width
    if stride < width:
        raise ValueError("the table's rows must not overlap")
    return max_rows, (total, seqs, max_rows, table.data_ptr(), stride, width, _index(lengths, "lengths", (seqs,), dev), starts)


def _model_dtype(cache: PagedCache, dtype: torch.dtype) -> int:
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None:
        raise TypeError(f"rows must be bf16 or fp16, got {dtype}")
    if cache.dtype != dtype and cache.dtype != torch.float8_e4m3fn:
        raise TypeError(f"rows of a {cache.dtype} cache must be of its type, got {dtype}")
    return code


def append_kv(cache: PagedCache, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
              lengths: torch.Tensor, *, rope: torch.Tensor | None = None, interleaved: bool = False,
              positions: torch.Tensor | None = None, row_starts: torch.Tensor | None = None,
              max_rows: int | None = None) -> torch.Tensor | None:
    """Stores the rows' keys and values ``[total, kv_heads, head_dim]`` (views into a QKV product are read in
    place) as tokens ``lengths[b] + i`` and returns the queries ``[total, heads, head_dim]``, rotated.

    ``rope [positions, rotary]`` (float32) holds a position's rotary / 2 cosines, then its sines; pairs are
    ``(i, i + rotary / 2)``, or ``(2 i, 2 i + 1)`` with ``interleaved``; dimensions past ``rotary`` and, without
    ``rope``, all of them stay as they are. A row's position is ``positions[row]``, or its token number; one that
    ``rope`` does not hold gives NaN. In an 8-bit cache a page's scale is the least power of two that its rows
    need: it grows with them (rows that stay are rounded again) and starts anew with the page's first row.
    ``lengths`` stays as it is. Two sequences may share pages, but not the ones this call appends to."""
    total = k.shape[0] if k.dim() == 3 else 0
    if total < 1:
        raise ValueError(f"k must be [rows, {cache.kv_heads}, {cache.head_dim}] with at least one row, got {tuple(k.shape)}")
    dev, dim, dtype = cache.device, cache.head_dim, k.dtype
    code = _model_dtype(cache, dtype)
    k = _rows(k, "k", dtype, total, cache.kv_heads, dim, dev)
    v = _rows(v, "v", dtype, total, cache.kv_heads, dim, dev)
    out, heads, q_args = None, 0, (0, 0, 0, 0, 0)
    if q is not None:
        q = _rows(q, "q", dtype, total, None, dim, dev)
        heads = q.shape[1]
        out = torch.empty((total, heads, dim), dtype=dtype, device=dev)
        q_args = (q.data_ptr(), q.stride(0), q.stride(1), heads, out.data_ptr())
    _, rows = _call(cache, total, table, lengths, row_starts, max_rows)
    rope_args = (0, 0, 0)
    if rope is not None:
        if rope.dim() != 2 or rope.dtype != torch.float32 or rope.device != dev or not rope.is_contiguous():
            raise ValueError(f"rope must be a contiguous float32 [positions, rotary] tensor on {dev}")
        if rope.shape[0] < 1 or rope.shape[1] < 2 or rope.shape[1] % 2 or rope.shape[1] > dim:
            raise ValueError(f"rope must hold an even number of entries up to {dim} per position, got {tuple(rope.shape)}")
        if rope.data_ptr() % 16:
            rope = rope.clone()
        rope_args = (rope.data_ptr(), rope.shape[0], rope.shape[1])
    at = None if positions is None else _index(positions, "positions", (total,), dev)
    status = _lib.lib().plm_kv_append(code, cache._ref, *q_args, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                                      v.stride(0), v.stride(1), *rows, *rope_args, bool(interleaved), at,
                                      _lib.stream_handle(dev))
    if status:
        _lib.check(status, f"plm_kv_append({total} rows, {rows[1]} sequences, heads {heads}/{cache.kv_heads} of {dim})")
    return out


def read_kv(cache: PagedCache, table: torch.Tensor, first: torch.Tensor, ends: torch.Tensor, most: int,
            dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of tokens ``[first[b], min(first[b] + most, ends[b]))`` as ``dtype``
    ``[seqs, most, kv_heads, head_dim]``, zeros after them."""
    code = _model_dtype(cache, dtype)
    dev = cache.device
    if table.dim() != 2 or table.dtype != torch.int32 or table.device != dev or table.shape[0] < 1 or table.shape[1] < 1 \
            or table.stride(1) != 1:
        raise ValueError(f"table must be an int32 [seqs, pages] tensor with contiguous rows on {dev}, got {table.dtype} "
                         f"{tuple(table.shape)} on {table.device}")
    if most < 1:
        raise ValueError(f"most must be at least 1, got {most}")
    seqs, width = table.shape
    k, v = (torch.empty((seqs, most, cache.kv_heads, cache.head_dim), dtype=dtype, device=dev) for _ in range(2))
    status = _lib.lib().plm_kv_read(code, cache._ref, table.data_ptr(), table.stride(0) if seqs > 1 else width, width,
                                    _index(first, "first", (seqs,), dev), _index(ends, "ends", (seqs,), dev), seqs, most,
                                    k.data_ptr(), v.data_ptr(), _lib.stream_handle(dev))
    if status:
        _lib.check(status, f"plm_kv_read({seqs} sequences, most {most})")
    return k, v


def attend(cache: PagedCache, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
           row_starts: torch.Tensor | None = None, max_rows: int | None = None, window: int | None = None, sinks: int = 0,
           mask: torch.Tensor | None = None, positions: torch.Tensor | None = None,
           scale: float | None = None) -> torch.Tensor:
    """Attention ``[total, heads, head_dim]`` of rotated queries over the cache, which holds the rows' own keys and
    values already (``append_kv``); query head h reads key head ``h // (heads // kv_heads)``.

    Row i of a sequence sees tokens up to its own, ``lengths[b] + i``. With ``mask`` (int32 ``[rows, words]``, bit
    j % 32 of word j // 32 set where row i sees row j; the same for every sequence) it sees the context and those
    rows. With ``window`` it sees of these the tokens after ``position - window`` and the first ``sinks``, the
    position being ``positions[row]`` or the row's token number; under a mask the window holds for the context
    alone. A row that sees nothing is zero. ``scale`` is 1 / sqrt(head_dim) unless given."""
    if q.dim() != 3 or q.shape[0] < 1:
        raise ValueError(f"q must be [rows, heads, {cache.head_dim}] with at least one row, got {tuple(q.shape)}")
    dev, dim, dtype, total, heads = cache.device, cache.head_dim, q.dtype, q.shape[0], q.shape[1]
    code = _model_dtype(cache, dtype)
    q = _rows(q, "q", dtype, total, None, dim, dev)
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"the query heads must be a multiple of the cache's {cache.kv_heads}, got {heads}")
    most, rows = _call(cache, total, table, lengths, row_starts, max_rows)
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 token, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    mask_args = (None, 0, 0)
    if mask is not None:
        if mask.dim() != 2 or mask.dtype != torch.int32 or mask.device != dev or not mask.is_contiguous() \
                or mask.shape[0] < most or mask.shape[1] * 32 < most:
            raise ValueError(f"mask must be a contiguous int32 [rows, words] tensor on {dev} with a bit for each of {most} "
                             f"rows, got {mask.dtype} {tuple(mask.shape)} on {mask.device}")
        mask_args = (mask.data_ptr(), mask.shape[0], mask.shape[1])
    at = None if positions is None else _index(positions, "positions", (total,), dev)
    out = torch.empty((total, heads, dim), dtype=dtype, device=dev)
    stream = _lib.stream_handle(dev)
    size = _lib.lib().plm_attend_workspace_bytes(cache.kv_heads, cache.page, dim, heads, total, rows[1], most, rows[5])
    space = torch.empty(size, dtype=torch.uint8, device=dev) if size else None   # partial results: this call's alone
    status = _lib.lib().plm_attend(code, cache._ref, q.data_ptr(), q.stride(0), q.stride(1), heads, out.data_ptr(), *rows,
                                   0 if window is None else window, sinks, *mask_args, at,
                                   1 / math.sqrt(dim) if scale is None else scale,
                                   None if space is None else space.data_ptr(), size, stream)
    if status:
        _lib.check(status, f"plm_attend({total} rows, {rows[1]} sequences, heads {heads}/{cache.kv_heads} of {dim})")
    return out


def round_mask(k: int, device: torch.device | str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """``(mask, places)`` of a round's k + k*k rows: k verify rows, each seeing those up to itself, then k blocks
    of k proposals, block i seeing verify rows 0..i and itself up to the row. ``places`` (int64) are the rows'
    positions after the context: ``positions = (lengths[:, None] + places).flatten()``."""
    if k < 1:
        raise ValueError(f"k must be at least 1, got {k}")
    rows = k + k * k
    words = -(-rows // 32)
    seen = [[r for r in range(i + 1)] for i in range(k)]
    seen += [[*range(i + 1), *range(k + i * k, k + i * k + j + 1)] for i in range(k) for j in range(k)]
    places = list(range(k)) + [i + 1 + j for i in range(k) for j in range(k)]
    bits = torch.zeros((rows, words), dtype=torch.int64)
    for i, own in enumerate(seen):
        for r in own:
            bits[i, r // 32] |= 1 << (r % 32)
    bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits)
    return bits.to(torch.int32).to(device), torch.tensor(places, device=device)
