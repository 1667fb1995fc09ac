"""A decoder layer's attention, put together from this package's calls: the norm before it, the QKV product, the append with
the position rotation, the attention over the paged cache, and the attn-out product; and the whole layer with its gated MLP.

``AttentionLayer`` is the attention for any batch of rows, ``DecoderLayer`` the layer, with weights in 16 bits or in 8
(``fp8.Weight``); ``PageTable`` hands out a cache's pages to sequences. Run as

    python -m plm_amd.attention_layer [--hidden 1024 --heads 8 --kv-heads 2 --prompt 2000 --k 7 --rounds 20 --cache e4m3
                                       --weights e4m3 --mlp 2816]

it reads a prompt in chunks, then replays one captured round of k + k*k rows while the sequence grows, as a decoder
does, and prints the time of a chunk and of a round (random weights; a layer alone). ``--mlp`` makes it the whole layer, of
that intermediate size.
"""

from __future__ import annotations

import argparse

import torch

from . import attention, fp8
from .fast_gemm import default_config, hip_linear, llama_mlp

CACHES = {"e4m3": torch.float8_e4m3fn, "model": torch.bfloat16}


def _linear(x: torch.Tensor | fp8.Rows, w: torch.Tensor | fp8.Weight, dtype: torch.dtype) -> torch.Tensor:
    if isinstance(w, fp8.Weight):
        return fp8.linear(x, w, out_dtype=dtype)
    return hip_linear(x, w, default_config(x.shape[0], w.shape[0], w.shape[1]))


def _norm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None, w: torch.Tensor | fp8.Weight):
    """(what a product with ``w`` takes, the sum) of x and the residual."""
    rows = fp8.rms_norm(x, weight, eps, residual=residual, dtype=fp8.E4M3 if isinstance(w, fp8.Weight) else None)
    return (rows, x) if residual is None else rows


def rope_table(positions: int, rotary: int, theta: float = 10000.0, device: torch.device | str = "cuda") -> torch.Tensor:
    """``[positions, rotary]`` float32: cosines, then sines, of position * theta^(-2 i / rotary)."""
    half = rotary // 2
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat((angle.cos(), angle.sin()), 1).float().to(device)


class PageTable:
    """The pages of one cache, handed out to ``seqs`` sequences of up to ``tokens`` tokens as they grow. ``table`` is
    what the calls read; a page is a sequence's until ``free``."""

    def __init__(self, cache: attention.PagedCache, seqs: int, tokens: int):
        self.page = cache.page
        self.table = torch.full((seqs, -(-tokens // cache.page)), -1, dtype=torch.int32, device=cache.device)
        self._held: list[list[int]] = [[] for _ in range(seqs)]
        self._free = list(range(cache.pages))

    def reserve(self, seq: int, tokens: int) -> None:
        """Pages for the first ``tokens`` tokens of sequence ``seq``."""
        need = -(-tokens // self.page)
        if need > self.table.shape[1]:
            raise ValueError(f"sequence {seq} holds up to {self.table.shape[1] * self.page} tokens, {tokens} asked for")
        held = self._held[seq]
        if need - len(held) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {need - len(held)} are needed")
        if need > len(held):
            new = [self._free.pop() for _ in range(need - len(held))]
            self.table[seq, len(held):need] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
            held += new

    def free(self, seq: int) -> None:
        self.table[seq] = -1
        self._free += self._held[seq]
        self._held[seq] = []


class AttentionLayer:
    """``qkv_weight [(heads + 2 kv_heads) head_dim, hidden]`` (queries, keys, values), ``out_weight [hidden, heads head_dim]``,
    each in 16 bits or an ``fp8.Weight``, a cache and its rotation table. Called with rows ``x [total, hidden]`` and the batch's
    arguments of ``attention.append_kv`` and ``attention.attend``, it stores the rows' keys and values and returns ``[total,
    hidden]``; the sequences' lengths stay the caller's. With ``norm [hidden]`` the rows are normed first (``fp8.rms_norm``, with
    ``residual`` added to them), and it returns ``(rows, x + residual)``."""

    def __init__(self, qkv_weight: torch.Tensor | fp8.Weight, out_weight: torch.Tensor | fp8.Weight, cache: attention.PagedCache,
                 heads: int, rope: torch.Tensor | None = None, *, interleaved: bool = False, window: int | None = None,
                 sinks: int = 0, norm: torch.Tensor | None = None, eps: float = 1e-6):
        width = (heads + 2 * cache.kv_heads) * cache.head_dim
        if qkv_weight.shape[0] != width or out_weight.shape[1] != heads * cache.head_dim:
            raise ValueError(f"{heads} query heads and {cache.kv_heads} key heads of {cache.head_dim} need weights of {width} "
                             f"rows and {heads * cache.head_dim} columns, got {list(qkv_weight.shape)} and {list(out_weight.shape)}")
        self.qkv_weight, self.out_weight, self.cache, self.heads, self.rope = qkv_weight, out_weight, cache, heads, rope
        self.interleaved, self.window, self.sinks, self.norm, self.eps = interleaved, window, sinks, norm, eps

    def __call__(self, x: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, row_starts: torch.Tensor | None = None,
                 max_rows: int | None = None, mask: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
        cache, rows = self.cache, dict(row_starts=row_starts, max_rows=max_rows, positions=positions)
        if self.norm is None and residual is not None:
            raise ValueError("a residual is added in the norm, which this layer has none of")
        normed, total = (x, x) if self.norm is None else _norm(x, self.norm, self.eps, residual, self.qkv_weight)
        qkv = _linear(normed, self.qkv_weight, x.dtype).view(x.shape[0], -1, cache.head_dim)
        keys, values = self.heads, self.heads + cache.kv_heads
        q = attention.append_kv(cache, qkv[:, :keys], qkv[:, keys:values], qkv[:, values:], table, lengths, rope=self.rope,
                                interleaved=self.interleaved, **rows)
        y = attention.attend(cache, q, table, lengths, window=self.window, sinks=self.sinks, mask=mask, **rows)
        y = _linear(y.view(x.shape[0], -1), self.out_weight, x.dtype)
        return y if self.norm is None else (y, total)


class DecoderLayer:
    """``attention``, an ``AttentionLayer`` with a norm, then ``norm [hidden]`` and the gated MLP: ``gate_up [2 I, hidden]`` (gate
    rows first) and ``down [hidden, I]`` in 16 bits or as ``fp8.Weight`` (gate_up made with ``gate_up=True``). Called as the
    attention, it returns ``(rows, x + residual so far)``, which are the next layer's ``x`` and ``residual``."""

    def __init__(self, attention: AttentionLayer, norm: torch.Tensor, gate_up: torch.Tensor | fp8.Weight,
                 down: torch.Tensor | fp8.Weight, eps: float = 1e-6):
        if attention.norm is None:
            raise ValueError("a decoder layer's attention needs its norm")
        if isinstance(gate_up, fp8.Weight) is not isinstance(down, fp8.Weight):
            raise TypeError("gate_up and down are both tensors or both an fp8.Weight")
        self.attention, self.norm, self.gate_up, self.down, self.eps = attention, norm, gate_up, down, eps

    def __call__(self, x: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, residual: torch.Tensor | None = None,
                 **rows) -> tuple[torch.Tensor, torch.Tensor]:
        y, total = self.attention(x, table, lengths, residual=residual, **rows)
        normed, total = _norm(y, self.norm, self.eps, total, self.gate_up)
        if isinstance(self.gate_up, fp8.Weight):
            return fp8.llama_mlp(normed, self.gate_up, self.down, out_dtype=x.dtype), total
        return llama_mlp(normed, self.gate_up, self.down), total


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--heads", type=int, default=8)
    ap.add_argument("--kv-heads", type=int, default=2)
    ap.add_argument("--prompt", type=int, default=2000)
    ap.add_argument("--chunk", type=int, default=512)
    ap.add_argument("--k", type=int, default=7)
    ap.add_argument("--rounds", type=int, default=20)
    ap.add_argument("--cache", choices=CACHES, default="e4m3")
    ap.add_argument("--weights", choices=("e4m3", "model"), default="model")
    ap.add_argument("--mlp", type=int, default=0, help="the gated MLP's intermediate size: the whole layer, with its norms")
    a = ap.parse_args()
    dev, dim = torch.device("cuda", torch.cuda.current_device()), a.hidden // a.heads
    g = torch.Generator(device=dev).manual_seed(0)

    def weight(n: int, k: int, gate_up: bool = False) -> torch.Tensor | fp8.Weight:
        w = (0.02 * torch.randn(n, k, generator=g, device=dev)).bfloat16()
        return fp8.Weight.quantize(w, gate_up=gate_up) if a.weights == "e4m3" else w

    rows = a.k + a.k * a.k
    tokens = a.prompt + rows + (a.rounds + 1) * a.k
    cache = attention.PagedCache.empty(-(-tokens // 64), a.kv_heads, dim, dtype=CACHES[a.cache], device=dev)
    pages = PageTable(cache, 1, tokens)
    ones = torch.ones(a.hidden, dtype=torch.bfloat16, device=dev) if a.mlp else None
    layer = AttentionLayer(weight((a.heads + 2 * a.kv_heads) * dim, a.hidden), weight(a.hidden, a.heads * dim), cache, a.heads,
                           rope_table(tokens, dim, device=dev), norm=ones)
    if a.mlp:
        layer = DecoderLayer(layer, ones, weight(2 * a.mlp, a.hidden, gate_up=True), weight(a.hidden, a.mlp))
    length = torch.zeros(1, dtype=torch.int64, device=dev)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for first in range(0, a.prompt, a.chunk):
        x = torch.randn(min(a.chunk, a.prompt - first), a.hidden, generator=g, device=dev).bfloat16()
        pages.reserve(0, first + x.shape[0])
        begin.record()
        layer(x, pages.table, length)
        end.record()
        length += x.shape[0]
    torch.cuda.synchronize()
    if a.prompt:
        print(f"prompt of {a.prompt} tokens: its last chunk {1e3 * begin.elapsed_time(end):.1f} us")

    mask, places = attention.round_mask(a.k, device=dev)
    x = torch.randn(rows, a.hidden, generator=g, device=dev).bfloat16()

    def step() -> torch.Tensor:
        y = layer(x, pages.table, length, mask=mask, positions=length + places)
        return y[0] if a.mlp else y

    pages.reserve(0, a.prompt + rows)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()                       # packs the weights and sizes the products' workspace
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    total = 0.0
    for r in range(a.rounds):
        pages.reserve(0, a.prompt + rows + r * a.k)
        x.copy_(torch.randn(x.shape, generator=g, device=dev))
        begin.record()
        graph.replay()
        end.record()
        length += 1 + r % a.k        # what the round accepted
        torch.cuda.synchronize()
        total += begin.elapsed_time(end)
    print(f"{a.rounds} rounds of {rows} rows from {a.prompt} tokens on ({a.cache} cache of {cache.pages} pages): "
          f"{1e3 * total / max(a.rounds, 1):.1f} us each, {int(length)} tokens held, finite {bool(torch.isfinite(out).all())}")


if __name__ == "__main__":
    main()
