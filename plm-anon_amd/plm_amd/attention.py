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
``[row_starts[b], row_starts[b + 1])`` (``None``: the same number each). Rows that no sequence holds (before
the first start, past the last one, past ``max_rows`` of a sequence) are not stored and come back as zeros, so a
captured batch can be padded. A sequence's rows follow ``lengths[b]`` cached tokens; token t of sequence b lies
in page ``table[b, t // page]``. ``lengths``, ``row_starts`` (which do not fall) and ``positions`` are int64
tensors on the GPU and are never read on the host, so every call can be captured in a HIP graph and replayed as
the sequences grow; only ``max_rows`` (the longest sequence's rows) and the tensors' shapes size a launch. Table
entries outside the cache are pages that are not there. Nothing here has a derivative: rows that require a
gradient are refused while gradients are recorded, and so are those that carry a forward-mode tangent.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _lib

PAGES = (16, 32, 64, 128)
MAX_HEAD_DIM = 256
_TYPES = {torch.bfloat16: _lib.PLM_CACHE_BF16, torch.float16: _lib.PLM_CACHE_F16, torch.float8_e4m3fn: _lib.PLM_CACHE_E4M3}
LEAST_SCALE = 2.0 ** -64   # of an 8-bit page that holds nothing but zeros
_SCALES = (2.0 ** -62, 2.0 ** 126)   # of the scores: times log2 e and a page's scale neither zero nor infinite in fp32


def _shapes(pages: int, kv_heads: int, page: int, head_dim: int, e4m3: bool) -> tuple[tuple, tuple]:
    lead = (pages, kv_heads, page // 16, -(-head_dim // 64))
    return (lead + (4, 16, 16), lead + (4, 16, 4, 4)) if e4m3 else (lead + (2, 4, 16, 8), lead + (2, 4, 16, 2, 4))


class PagedCache:
    """Keys and values of ``kv_heads`` heads in pages of 16, 32, 64 or 128 tokens. The tensors, which stay the
    handle's, are used as they are, in the order the matrix instructions read (``include/plm_amd.h`` states it): 16-bit
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
        self._index = k.get_device()
        self._handle = _lib.KvCache(k.data_ptr(), v.data_ptr(), 0 if k_scale is None else k_scale.data_ptr(),
                                    0 if v_scale is None else v_scale.data_ptr(), pages, heads, page, head_dim,
                                    _TYPES[k.dtype])
        self._ref = ctypes.addressof(self._handle)

    # What the kernels were told once stays: another tensor in a cache's place would leave them its freed memory, another
    # size a shape that the checks of a call and the kernels see differently.
    def __setattr__(self, name: str, value) -> None:
        if name in self.__dict__:
            raise AttributeError(f"a cache's {name} stays as it is; make another PagedCache")
        object.__setattr__(self, name, value)

    def __delattr__(self, name: str) -> None:
        raise AttributeError(f"a cache keeps its {name}")

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


# The checks below are on every call's path, where the host's time counts: one look at each property, strides only of
# tensors that are not contiguous, messages formed for refusals alone.


def _numbers(t: torch.Tensor, name: str, n: int, cache: PagedCache) -> int:
    """Device pointer of ``n`` int64 numbers."""
    if t.dtype is not torch.int64 or t.shape != (n,) or t.get_device() != cache._index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int64 [{n}] tensor on {cache.device}, got {t.dtype} "
                         f"{list(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, cache: PagedCache) -> tuple[torch.Tensor, int, int, int]:
    """``t`` [rows, heads, dim] as a kernel can read it (dimensions contiguous, rows and heads on 16 bytes), its pointer
    and the strides of its rows and heads."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != cache._index:
        raise RuntimeError(f"{name} must be on the cache's GPU {cache.device}, got {t.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, and the cache's calls have none: detach it, or call under no_grad")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} carries a forward-mode tangent, and the cache's calls have none: detach it")
    at = t.data_ptr()
    if at % 16 == 0:
        if t.is_contiguous():
            return t, at, shape[1] * shape[2], shape[2]
        row, head, one = t.stride()
        if one == 1 and row % 8 == 0 and head % 8 == 0:
            return t, at, row, head
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), shape[1] * shape[2], shape[2]


def _table(t: torch.Tensor, cache: PagedCache) -> tuple[int, int, int, int]:
    """Sequences, pointer, row stride and width of a page table."""
    if t.dim() == 2 and t.dtype is torch.int32 and t.get_device() == cache._index:
        seqs, width = t.shape
        if seqs and width:
            if t.is_contiguous():
                return seqs, t.data_ptr(), width, width
            row, one = t.stride()
            if (one == 1 or width == 1) and (row >= width or seqs == 1):
                return seqs, t.data_ptr(), max(row, width), width
    raise ValueError(f"table must be an int32 [seqs, pages] tensor with contiguous rows on {cache.device}, got {t.dtype} "
                     f"{list(t.shape)} on {t.device}")


def _call(cache: PagedCache, total: int, table: torch.Tensor, lengths: torch.Tensor, row_starts: torch.Tensor | None,
          max_rows: int | None) -> tuple:
    """plm_kv_rows of a call."""
    seqs, at, stride, width = _table(table, cache)
    if row_starts is None:
        if total % seqs:
            raise ValueError(f"{total} rows are no whole number for each of {seqs} sequences: row_starts is needed")
        each = total // seqs
        if max_rows is not None and max_rows != each:
            raise ValueError(f"max_rows must be {each} for {total} rows of {seqs} sequences, got {max_rows}")
        return total, seqs, each, at, stride, width, _numbers(lengths, "lengths", seqs, cache), 0
    starts = _numbers(row_starts, "row_starts", seqs + 1, cache)
    if max_rows is None:
        max_rows = total
    elif not 1 <= max_rows <= total:
        raise ValueError(f"max_rows must be in [1, {total}], got {max_rows}")
    return total, seqs, max_rows, at, stride, width, _numbers(lengths, "lengths", seqs, cache), starts


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
    if k.dim() != 3 or k.shape[0] < 1:
        raise ValueError(f"k must be [rows, {cache.kv_heads}, {cache.head_dim}] with at least one row, got {list(k.shape)}")
    dim, dtype, total = cache.head_dim, k.dtype, k.shape[0]
    code = _model_dtype(cache, dtype)
    shape = (total, cache.kv_heads, dim)
    k, k_at, k_row, k_head = _rows(k, "k", dtype, shape, cache)
    v, v_at, v_row, v_head = _rows(v, "v", dtype, shape, cache)
    out, q_at, q_row, q_head, heads, out_at = None, 0, 0, 0, 0, 0
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        q, q_at, q_row, q_head = _rows(q, "q", dtype, (total, heads, dim), cache)
        if heads < 1:
            raise ValueError("q must have at least one head")
        out = q.new_empty((total, heads, dim))
        out_at = out.data_ptr()
    rows = _call(cache, total, table, lengths, row_starts, max_rows)
    rope_at, rope_rows, rotary = 0, 0, 0
    if rope is not None:
        if rope.dim() != 2 or rope.dtype is not torch.float32 or rope.get_device() != cache._index or not rope.is_contiguous():
            raise ValueError(f"rope must be a contiguous float32 [positions, rotary] tensor on {cache.device}")
        rope_rows, rotary = rope.shape
        if rope_rows < 1 or rotary < 2 or rotary % 2 or rotary > dim:
            raise ValueError(f"rope must hold an even number of entries up to {dim} per position, got {list(rope.shape)}")
        rope_at = rope.data_ptr()
        if rope_at % 16:
            rope = rope.clone()
            rope_at = rope.data_ptr()
    at = 0 if positions is None else _numbers(positions, "positions", total, cache)
    status = _lib.lib().plm_kv_append(
        _lib.pack_append(code, cache._ref, *rows, q_at, q_row, q_head, heads, out_at, k_at, k_row, k_head, v_at, v_row, v_head,
                         rope_at, rope_rows, rotary, bool(interleaved), at),
        _lib.stream_handle(cache.device))
    if status:
        _lib.check(status, f"plm_kv_append({total} rows, {rows[1]} sequences, heads {heads}/{cache.kv_heads} of {dim})")
    return out


def read_kv(cache: PagedCache, table: torch.Tensor, first: torch.Tensor, ends: torch.Tensor, most: int,
            dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of tokens ``[first[b], min(first[b] + most, ends[b]))`` as ``dtype``
    ``[seqs, most, kv_heads, head_dim]``, zeros after them."""
    code = _model_dtype(cache, dtype)
    if most < 1:
        raise ValueError(f"most must be at least 1, got {most}")
    seqs, table_at, stride, width = _table(table, cache)
    first_at, ends_at = _numbers(first, "first", seqs, cache), _numbers(ends, "ends", seqs, cache)
    k, v = torch.empty((2, seqs, most, cache.kv_heads, cache.head_dim), dtype=dtype, device=cache.device).unbind(0)
    status = _lib.lib().plm_kv_read(
        _lib.pack_read(code, cache._ref, table_at, stride, width, first_at, ends_at, seqs, most, k.data_ptr(), v.data_ptr()),
        _lib.stream_handle(cache.device))
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
    alone. A row that sees nothing is zero. ``scale`` is 1 / sqrt(head_dim) unless given, in [2^-62, 2^126]."""
    if q.dim() != 3 or q.shape[0] < 1:
        raise ValueError(f"q must be [rows, heads, {cache.head_dim}] with at least one row, got {list(q.shape)}")
    dim, dtype = cache.head_dim, q.dtype
    total, heads, _ = shape = q.shape
    code = _model_dtype(cache, dtype)
    q, q_at, q_row, q_head = _rows(q, "q", dtype, (total, heads, dim), cache)
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"the query heads must be a multiple of the cache's {cache.kv_heads}, got {heads}")
    rows = _call(cache, total, table, lengths, row_starts, max_rows)
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 token, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    if scale is not None and not _SCALES[0] <= scale <= _SCALES[1]:
        raise ValueError(f"scale must be in [2^-62, 2^126], got {scale}")
    mask_at, mask_rows, mask_words = 0, 0, 0
    if mask is not None:
        most = rows[2]
        if mask.dim() != 2 or mask.dtype is not torch.int32 or mask.get_device() != cache._index or not mask.is_contiguous() \
                or mask.shape[0] < most or mask.shape[1] * 32 < most:
            raise ValueError(f"mask must be a contiguous int32 [rows, words] tensor on {cache.device} with a bit for each of "
                             f"{most} rows, got {mask.dtype} {list(mask.shape)} on {mask.device}")
        mask_at, (mask_rows, mask_words) = mask.data_ptr(), mask.shape
    at = 0 if positions is None else _numbers(positions, "positions", total, cache)
    out = q.new_empty(shape)
    call = _lib.pack_attend(code, cache._ref, *rows, q_at, q_row, q_head, heads, out.data_ptr(), window or 0, sinks, mask_at,
                            mask_rows, mask_words, at, 1 / math.sqrt(dim) if scale is None else scale)
    lib = _lib.lib()
    space, size = 0, lib.plm_attend_workspace_bytes(call)
    if size:
        work = torch.empty(size, dtype=torch.uint8, device=cache.device)   # partial results: this call's alone
        space = work.data_ptr()
    status = lib.plm_attend(call, space, size, _lib.stream_handle(cache.device))
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
