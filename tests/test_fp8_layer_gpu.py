"""A decoder layer with its weights in 8 bits (``plm_amd.attention_layer``): a prompt, then captured rounds, against the same
layer over the weights' values in 16 bits; and its command.

Tolerance: both layers have the same weights, exactly. The 8-bit one rounds the rows before each product to 8 bits, half a
step of e4m3 (2^-4) of each value, independent of one another; the 16-bit one rounds to bf16 what it does not. A product's
error is then 2^-4 / sqrt(3) of the root mean square of its terms, times sqrt(K), against values of the same size: 4% of
a product's typical size for each of the four in a row, 8% for their sum, and six times that at the most.
"""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from plm_amd import attention, fp8
from plm_amd.attention_layer import AttentionLayer, DecoderLayer, PageTable, rope_table

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HIDDEN, HEADS, KV_HEADS, DIM, INNER, TOKENS = 256, 8, 2, 32, 384, 400


def _layer(device, eight, kind=BF16):
    g = torch.Generator().manual_seed(3)

    def weight(n, k, gate_up=False):
        w = fp8.Weight.quantize((k ** -0.5 * torch.randn(n, k, generator=g)).bfloat16().to(device), gate_up=gate_up)
        return w if eight else w.values(BF16)

    cache = attention.PagedCache.empty(-(-TOKENS // 16) + 1, KV_HEADS, DIM, page=16, dtype=kind, device=device)
    norms = [(1 + 0.1 * torch.randn(HIDDEN, generator=g)).bfloat16().to(device) for _ in range(2)]
    layer = AttentionLayer(weight((HEADS + 2 * KV_HEADS) * DIM, HIDDEN), weight(HIDDEN, HEADS * DIM), cache, HEADS,
                           rope_table(TOKENS, DIM, device=device), norm=norms[0])
    return DecoderLayer(layer, norms[1], weight(2 * INNER, HIDDEN, True), weight(HIDDEN, INNER)), PageTable(cache, 1, TOKENS)


def _rows(n, seed, device):
    return torch.randn(n, HIDDEN, generator=torch.Generator().manual_seed(seed)).bfloat16().to(device)


@pytest.mark.parametrize("parts", [[200], [70, 1, 129]])
def test_against_its_values_in_16_bits(device, parts):
    outs = []
    for eight in (True, False):
        layer, pages = _layer(device, eight)
        length, got = 0, []
        for i, n in enumerate(parts):
            pages.reserve(0, length + n)
            x, r = _rows(n, 10 + i, device), _rows(n, 20 + i, device)
            y, total = layer(x, pages.table, torch.tensor([length], device=device), residual=r)
            assert y.shape == total.shape == (n, HIDDEN) and y.dtype is total.dtype is BF16
            got.append(torch.cat((y, total)).float())
            length += n
        outs.append(torch.cat(got))
    size = outs[1].square().mean().sqrt()
    off = outs[0] - outs[1]
    assert float(off.square().mean().sqrt()) <= 0.08 * float(size)
    assert float(off.abs().max()) <= 6 * 0.08 * float(outs[1].abs().max())


def test_captured_rounds_are_eager_ones(device):
    """Rounds of k + k*k rows over a growing sequence, replayed, bit for bit the eager calls'."""
    k = 4
    rows = k + k * k
    mask, places = attention.round_mask(k, device=device)
    graphed, pages = _layer(device, True, torch.float8_e4m3fn)
    eager, theirs = _layer(device, True, torch.float8_e4m3fn)
    length = torch.zeros(1, dtype=torch.int64, device=device)
    for layer, table in ((graphed, pages), (eager, theirs)):
        table.reserve(0, 300)
        layer(_rows(50, 0, device), table.table, length, residual=_rows(50, 1, device))
    length += 50
    x, r = _rows(rows, 2, device), _rows(rows, 3, device)
    step = lambda layer, table: layer(x, table.table, length, residual=r, mask=mask, positions=length + places)
    step(graphed, pages)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed, pages)
    for i in range(4):
        x.copy_(_rows(rows, 30 + i, device)), r.copy_(_rows(rows, 40 + i, device))
        graph.replay()
        want = step(eager, theirs)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        length += 1 + i


def test_refusals(device):
    layer, pages = _layer(device, True)
    pages.reserve(0, 10)
    bare = AttentionLayer(layer.attention.qkv_weight, layer.attention.out_weight, layer.attention.cache, HEADS)
    with pytest.raises(ValueError):
        DecoderLayer(bare, layer.norm, layer.gate_up, layer.down)
    with pytest.raises(ValueError):
        bare(_rows(2, 0, device), pages.table, torch.zeros(1, dtype=torch.int64, device=device), residual=_rows(2, 0, device))
    with pytest.raises(ValueError):
        AttentionLayer(layer.attention.out_weight, layer.attention.out_weight, layer.attention.cache, HEADS)


def test_weights_of_two_kinds_are_refused(device):
    layer, _ = _layer(device, True)
    plain = torch.zeros(layer.down.shape, dtype=torch.bfloat16, device=device)
    with pytest.raises(TypeError):
        DecoderLayer(layer.attention, layer.norm, layer.gate_up, plain)


@pytest.mark.parametrize("weights,mlp", [("e4m3", "0"), ("e4m3", "384"), ("model", "384")])
def test_the_command_runs(device, weights, mlp):
    root = Path(__file__).resolve().parents[1]
    got = subprocess.run([sys.executable, "-m", "plm_amd.attention_layer", "--hidden", "256", "--heads", "4", "--kv-heads", "2", "--prompt",
                          "300", "--chunk", "128", "--k", "3", "--rounds", "4", "--weights", weights, "--mlp", mlp],
                         cwd=root / "plm-anon_amd", capture_output=True, text=True, timeout=100)
    assert got.returncode == 0, got.stderr
    assert "4 rounds of 12 rows" in got.stdout and "finite True" in got.stdout
