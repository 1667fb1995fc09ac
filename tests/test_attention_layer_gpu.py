"""The attention layer of ``plm_amd.attention_layer``: a prompt in one go and in chunks, rounds that are partly taken
back, single tokens, and its command."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from oracle import attention_oracle as oracle
from plm_amd import attention
from plm_amd.attention_layer import AttentionLayer, PageTable, rope_table

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, DIM = 256, 8, 2, 32


def _layer(device, kind, tokens, **more):
    g = torch.Generator().manual_seed(1)
    qkv = (0.06 * torch.randn((HEADS + 2 * KV_HEADS) * DIM, HIDDEN, generator=g)).bfloat16().to(device)
    out = (0.06 * torch.randn(HIDDEN, HEADS * DIM, generator=g)).bfloat16().to(device)
    cache = attention.PagedCache.empty(-(-tokens // 16) + 1, KV_HEADS, DIM, page=16, dtype=kind, device=device)
    pages = PageTable(cache, 1, tokens)
    return AttentionLayer(qkv, out, cache, HEADS, rope_table(tokens, DIM, device=device), **more), pages


def _run(device, kind, parts, x, **more):
    layer, pages = _layer(device, kind, 400, **more)
    outs, length = [], 0
    for n in parts:
        pages.reserve(0, length + n)
        outs.append(layer(x[length:length + n], pages.table, torch.tensor([length], device=device)))
        length += n
    return layer, pages, torch.cat(outs)


def test_a_prompt_in_chunks_is_the_prompt(device):
    """16-bit pages: the same cached tokens however the prompt is cut, to the QKV product's one rounding, and outputs to
    within the roundings of two orders of one softmax."""
    x = torch.randn(300, HIDDEN, generator=torch.Generator().manual_seed(2)).bfloat16().to(device)
    layer, pages, whole = _run(device, torch.bfloat16, [300], x)
    for parts in ([100, 200], [129, 171], [150, 149, 1]):
        other, theirs, got = _run(device, torch.bfloat16, parts, x)
        ends, zero = torch.tensor([300], device=device), torch.zeros(1, dtype=torch.int64, device=device)
        a = attention.read_kv(layer.cache, pages.table, zero, ends, 300, torch.bfloat16)
        b = attention.read_kv(other.cache, theirs.table, zero, ends, 300, torch.bfloat16)
        for p, q in zip(a, b):
            # One rounding of the QKV product apart at most (its K order may go by the number of rows).
            assert ((p.float() - q.float()).abs() <= 2.0 ** -7 * p.float().abs() + 2.0 ** -7 * 0.1).all()
        # Probabilities, the attention and the product each round once per side, on values of about 1.
        assert ((got.float() - whole.float()).abs().max()) <= 8 * 2.0 ** -8 * float(whole.float().abs().max())


@pytest.mark.parametrize("window", [None, 40])
def test_against_64_bits(device, window):
    """The layer on 16-bit pages against products and attention in 64 bits: every stage rounds its result once
    (2^-8 of it), four stages in a row, each on sums of terms no larger than a few times the result's size."""
    x = torch.randn(90, HIDDEN, generator=torch.Generator().manual_seed(3)).bfloat16().to(device)
    layer, _, got = _run(device, torch.bfloat16, [60, 29, 1], x, window=window, sinks=2)
    qkv = F.linear(x.cpu().double(), layer.qkv_weight.cpu().double()).view(90, -1, DIM)
    turn = layer.rope.cpu()[:90]
    q = oracle.rotate(qkv[:, :HEADS], turn, False)
    k = oracle.rotate(qkv[:, HEADS:HEADS + KV_HEADS], turn, False)
    y, _, _ = oracle.attention(q, k, qkv[:, HEADS + KV_HEADS:], oracle.seen(0, 90, 90, window, 2, None, None), DIM ** -0.5)
    want = F.linear(y.view(90, -1), layer.out_weight.cpu().double())
    off = (got.cpu().double() - want).norm() / want.norm()
    assert float(off) <= 4 * 2.0 ** -8


def test_rounds_that_are_partly_taken_back(device):
    """Tokens a round accepted stay, the rest are overwritten: after it the cache is that of a plain append."""
    k, rows = 3, 12
    x = torch.randn(60, HIDDEN, generator=torch.Generator().manual_seed(4)).bfloat16().to(device)
    layer, pages = _layer(device, torch.bfloat16, 400)
    plain, theirs = _layer(device, torch.bfloat16, 400)
    mask, places = attention.round_mask(k, device=device)
    pages.reserve(0, 100)
    theirs.reserve(0, 100)
    length = torch.zeros(1, dtype=torch.int64, device=device)
    layer(x[:40], pages.table, length)
    plain(x[:40], theirs.table, length)
    length += 40
    for accepted in (2, 3, 1):
        at = int(length)
        block = torch.cat((x[at:at + k], torch.randn(k * k, HIDDEN, device=device).bfloat16()))
        out = layer(block, pages.table, length, mask=mask, positions=length + places)
        # Verify rows see what a plain chunk's rows see.
        want = plain(x[at:at + k], theirs.table, length)
        assert float((out[:k].float() - want.float()).abs().max()) <= 8 * 2.0 ** -8 * float(want.float().abs().max())
        length += accepted
    zero, n = torch.zeros(1, dtype=torch.int64, device=device), int(length)
    a = attention.read_kv(layer.cache, pages.table, zero, length, n, torch.bfloat16)
    b = attention.read_kv(plain.cache, theirs.table, zero, length, n, torch.bfloat16)
    for p, q in zip(a, b):
        assert ((p.float() - q.float()).abs() <= 2.0 ** -7 * p.float().abs() + 2.0 ** -7 * 0.1).all()


def test_the_command(device):
    package = Path(__file__).resolve().parents[1] / "plm-anon_amd"
    done = subprocess.run([sys.executable, "-m", "plm_amd.attention_layer", "--prompt", "300", "--chunk", "200", "--rounds", "3"],
                          cwd=package, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stderr[-2000:]
    assert "3 rounds of 56 rows from 300 tokens on" in done.stdout and "finite True" in done.stdout
