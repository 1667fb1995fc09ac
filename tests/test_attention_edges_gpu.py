"""The paged cache and its attention at the ends of what they are given: page scales far apart, positions and windows past
any cache, rows that no sequence holds, pages that several sequences read, keys that need no rounding.

Tolerances are those of test_attention_gpu.py, whose cases these are."""

from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from oracle import attention_oracle as oracle
from plm_amd import attention
from test_attention_gpu import BF16, E4M3, FP16, WIDE, Case, check

pytestmark = pytest.mark.gpu


def _quiet_but(c, loud, by=2.0 ** -20):
    """8-bit value pages of ``c`` get the scale ``by``, those of sequence 0 whose numbers are in ``loud`` 2^5."""
    c.cache.v_scale.fill_(by)
    for n in loud:
        c.cache.v_scale[int(c.table[0, n])] = 2.0 ** 5


@pytest.mark.parametrize("heads, wider", [(4, 0), (64, WIDE)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_loud_pages_that_rows_do_not_see(device, heads, wider, dtype, page):
    """Values of 2^5 * 448 in pages past a row, or between its first tokens and its window, are nothing to its own of 2^-20."""
    c = Case(device, [3 * page + 2], [page + 9], heads, 1, 64, page, dtype=dtype, seed=60, wider=wider)
    _quiet_but(c, [4])
    want, tol = c.expected()
    got = c.attend()
    blind = slice(0, page - 2)           # rows of page 3
    check(got[blind], want[blind], tol[blind], "rows before the page")
    check(got, want, tol)
    c = Case(device, [5 * page], [3], heads, 1, 64, page, dtype=dtype, seed=61, wider=wider)
    _quiet_but(c, [1, 2])
    check(c.attend(window=page, sinks=3), *c.expected(window=page, sinks=3))


@pytest.mark.parametrize("heads, wider", [(4, 0), (64, WIDE)])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_loud_pages_of_no_weight(device, heads, wider, page):
    """Loud tokens that a row sees with a probability of about 2^-90, before, among and after quiet ones."""
    for loud in ([0], [2], [1, 3], [5]):
        c = Case(device, [6 * page - 3], [3], heads, 1, 64, page, dtype=FP16, seed=62, wider=wider)
        c.q = torch.ones_like(c.q)
        _quiet_but(c, loud, 2.0 ** -24)
        c.cache.k_scale.fill_(1.0)
        for n in range(6):
            at = int(c.table[0, n])
            values = torch.full((page, 1, 64), -8.0 if n in loud else 0.0)
            oracle.put_page(c.cache.k, at, values.to(E4M3), "k")
        check(c.attend(), *c.expected(), what=f"loud {loud}")


@pytest.mark.parametrize("heads, wider", [(4, 0), (64, WIDE)])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_quiet_and_loud_pages_in_turn(device, heads, wider, page):
    c = Case(device, [8 * page - 5], [40], heads, 1, 72, page, dtype=FP16, seed=63, wider=wider)
    for i, s in enumerate([2.0 ** -18, 2.0 ** 4, 2.0 ** -18, 2.0 ** -64, 2.0 ** -8, 2.0 ** -22, 2.0 ** 7, 2.0 ** -30]):
        c.cache.v_scale[int(c.table[0, i])] = s
    check(c.attend(), *c.expected())
    check(c.attend(window=page + 5, sinks=3), *c.expected(window=page + 5, sinks=3))


@pytest.mark.parametrize("heads, wider", [(4, 0), (64, WIDE)])
@pytest.mark.parametrize("page", [16, 32])
def test_nan_among_pages_of_unlike_scales(device, heads, wider, page):
    """Also of a page whose scale is the least: nothing but zeros and NaN was appended to it."""
    c = Case(device, [5 * page - 2], [9], heads, 1, 64, page, dtype=FP16, seed=71, wider=wider)
    for i, s in enumerate([2.0 ** 4, 2.0 ** -20, 2.0 ** -6, 2.0 ** -64, 2.0 ** 5, 2.0 ** -6]):
        c.cache.v_scale[int(c.table[0, i])] = s
    want, tol = c.expected()
    for number, token in ((3, 3), (5, 1)):     # in every row's sight; in those after the row that holds it
        at = int(c.table[0, number])
        values = oracle.get_page(c.cache.v, None, at, 1, page, 64, "v")
        values[token, 0, 7 * number] = math.nan
        oracle.put_page(c.cache.v, at, values.float().to(E4M3), "v")
    got = c.attend()
    first = 5 * page + 1 - (5 * page - 2)
    assert got[:, :, 21].isnan().all() and got[first:, :, 35].isnan().all()
    fine = [e for e in range(64) if e not in (21, 35)]
    check(got[:, :, fine], want[:, :, fine], tol[:, :, fine])
    check(got[:first, :, 35], want[:first, :, 35], tol[:first, :, 35])


@pytest.mark.parametrize("heads, wider", [(4, 0), (32, WIDE)])
@pytest.mark.parametrize("mask", [False, True])
def test_windows_and_positions_past_any_cache(device, heads, wider, mask):
    """A window is as long as it says, and a position as far, whatever a cache can hold."""
    c = Case(device, [60, 7], [9, 9], heads, 2, 64, 16, seed=64, wider=wider)
    see = torch.ones(9, 9, dtype=torch.bool).tril() if mask else None
    bits = torch.tensor([[(1 << (i + 1)) - 1] for i in range(9)], dtype=torch.int32).to(device) if mask else None
    row = torch.arange(18)
    for window, far in ((2 ** 30 - 1, 2 ** 30 + row), (2 ** 30, 2 ** 30 + 3 * row), (2 ** 29 + 5, 2 ** 31 + row),
                        (10 ** 12, 10 ** 12 + 20 + row % 9), (10 ** 12, 10 ** 15 + row), (2 ** 62, 2 ** 62 + 2 * row),
                        (2 ** 62, -(2 ** 63) + row), (5, -(2 ** 63) + row), (2 ** 63 - 1, 2 ** 63 - 1 - row)):
        # The same visibility in small numbers: the window's first token, held to what a sequence has.
        first = [max(int(p) - window + 1, 0) for p in far]
        places = torch.tensor([min(f, 10 ** 6) + 99 for f in first])
        want, tol = c.expected(window=100, sinks=2, see=see, places=places)
        check(c.attend(window=window, sinks=2, positions=far.to(device), mask=bits), want, tol, f"window {window} at {int(far[0])}")


@pytest.mark.parametrize("heads, wider", [(4, 0), (32, WIDE)])
def test_least_scale(device, heads, wider):
    """Masked tokens of pages of zeros, whose scale is the least there is, at the least scale of the scores."""
    c = Case(device, [45], [12], heads, 1, 64, 16, seed=72, wider=wider)
    c.cache.k_scale.fill_(attention.LEAST_SCALE)
    check(c.attend(scale=2.0 ** -62), *c.expected(scale=2.0 ** -62))


def _spoil(device, shape, dtype):
    """Leaves memory of ``shape`` full of NaN to the next allocation."""
    x = torch.full(shape, math.nan, dtype=dtype, device=device)
    torch.cuda.synchronize()
    del x


# Rows of three sequences (the second without any) among rows that are no one's: before the first, past max_rows of the
# third, after the last.
PLACES, STARTS, MOST = [2, 3, 4, 5, 6, 7], [2, 5, 5, 9], 3


@pytest.mark.parametrize("heads, dim, wider", [(4, 64, 0), (32, 64, WIDE), (4, 256, 0), (64, 80, WIDE)])
@pytest.mark.parametrize("context", [40, 5000])
@pytest.mark.parametrize("total", [12, 1500])
def test_rows_of_no_sequence_are_zero(device, heads, dim, wider, context, total):
    c = Case(device, [context, 5, 90], [3, 0, 3], heads, 1, dim, 64, seed=65, wider=wider)
    q = torch.randn(total, heads, dim).to(BF16)
    q[PLACES] = c.q
    q = q.to(device)
    want, tol = c.expected()
    rest = [r for r in range(total) if r not in PLACES]
    starts = torch.tensor(STARTS, device=device)
    for window in (None, 10 ** 6):
        _spoil(device, q.shape, BF16)
        got = attention.attend(c.cache, q, c.calls["table"], c.calls["lengths"], row_starts=starts, max_rows=MOST, window=window)
        check(got[PLACES], want, tol)
        assert torch.equal(got[rest].cpu(), torch.zeros(len(rest), heads, dim, dtype=BF16))


@pytest.mark.parametrize("kind", [E4M3, FP16])
@pytest.mark.parametrize("total", [12, 1500])
@pytest.mark.parametrize("side", [False, True])
def test_appended_rows_of_no_sequence_are_zero(device, kind, total, side):
    a, b = (Case(device, [40, 5, 90], [3, 0, 3], 4, 2, 80, 16, dtype=FP16, kind=kind, seed=66) for _ in range(2))
    angle = torch.arange(200, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    rope = torch.cat((angle.cos(), angle.sin()), 1).float().to(device)
    want = attention.append_kv(a.cache, a.q.to(device), a.k.to(device), a.v.to(device), **a.calls, rope=rope, interleaved=side)
    rows = []
    for x in (b.q, b.k, b.v):
        y = torch.randn(total, *x.shape[1:]).to(FP16)
        y[PLACES] = x
        rows.append(y.to(device))
    _spoil(device, rows[0].shape, FP16)
    got = attention.append_kv(b.cache, *rows, b.calls["table"], b.calls["lengths"], rope=rope, interleaved=side,
                              row_starts=torch.tensor(STARTS, device=device), max_rows=MOST)
    assert torch.equal(got[PLACES], want)
    rest = [r for r in range(total) if r not in PLACES]
    assert torch.equal(got[rest].cpu(), torch.zeros(len(rest), 4, 80, dtype=FP16))
    for x, y in ((a.cache.k, b.cache.k), (a.cache.v, b.cache.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("heads, wider", [(4, 0), (32, WIDE)])
def test_many_sequences_among_rows_of_none(device, heads, wider):
    """Gaps after every sequence of more than a wavefront's lanes of them."""
    n = 150
    c = Case(device, [(31 * b) % 190 for b in range(n)], [2] * n, heads, 1, 16, 16, seed=67, wider=wider)
    starts = [1]
    for b in range(n):
        starts.append(starts[-1] + 2 + (b % 3 == 0))     # a row past max_rows
    held = [s + i for s in starts[:-1] for i in (0, 1)]
    total = starts[-1] + 3
    q = torch.randn(total, heads, 16).to(BF16)
    q[held] = c.q
    q = q.to(device)
    want, tol = c.expected()
    _spoil(device, q.shape, BF16)
    got = attention.attend(c.cache, q, c.calls["table"], c.calls["lengths"], row_starts=torch.tensor(starts, device=device), max_rows=2)
    check(got[held], want, tol)
    rest = [r for r in range(total) if r not in held]
    assert rest and got[rest].abs().max() == 0


@pytest.mark.parametrize("kind", [E4M3, BF16])
def test_ragged_rows_without_their_most(device, kind):
    """row_starts alone: launches go by the rows in all."""
    a, b = (Case(device, [33, 250, 1000, 4], [3, 1, 65, 0], 8, 2, 64, 32, kind=kind, seed=68) for _ in range(2))
    calls = {k: x for k, x in a.calls.items() if k != "max_rows"}
    check(attention.attend(a.cache, a.q.to(device), **calls), *a.expected())
    q1 = attention.append_kv(a.cache, a.q.to(device), a.k.to(device), a.v.to(device), **calls)
    q2 = attention.append_kv(b.cache, b.q.to(device), b.k.to(device), b.v.to(device), **b.calls)
    assert torch.equal(q1, q2)
    for x, y in ((a.cache.k, b.cache.k), (a.cache.v, b.cache.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("contexts, rows, heads, kv_heads, dim, kind, window", [
    ([1800, 700, 33] * 13, [1] * 39, 8, 8, 128, BF16, 1797),     # 312 groups of up to 59 steps
    ([900, 640], [110, 110], 20, 4, 64, E4M3, 529),              # 280
    ([1000] * 65, [1] * 65, 4, 4, 16, E4M3, None),               # 260, without a window
])
def test_groups_past_the_cus(device, contexts, rows, heads, kv_heads, dim, kind, window):
    """A few more groups of middling length than CUs."""
    c = Case(device, contexts, rows, heads, kv_heads, dim, 128, kind=kind, seed=69)
    check(c.attend(window=window, sinks=2 if window else 0), *c.expected(window, 2 if window else 0))


def _append_us(cache, k, v, table, lengths, rope, interleaved):
    def times(n):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(n):
            attention.append_kv(cache, None, k, v, table, lengths, rope=rope, interleaved=interleaved)
        end.record()
        torch.cuda.synchronize()
        return begin.elapsed_time(end) * 1e3 / n

    times(5)
    return min(times(20) for _ in range(5))


@pytest.mark.parametrize("side", [False, True])
def test_keys_that_need_no_rounding_cost_no_more(device, side):
    """Zero rows (padding), and rows at position 0, are turned exactly in fp32: they do not go one by one through fp64, which
    takes 128 turns per thread here. The factor is far from both: about 1, and about 10."""
    cache = attention.PagedCache.empty(16, 4, 256, page=128, device=device)
    table = torch.arange(16, dtype=torch.int32, device=device)[None]
    zero = torch.zeros(1, dtype=torch.int64, device=device)
    k, v = (torch.randn(2048, 4, 256, device=device).bfloat16() for _ in range(2))
    angle = torch.arange(2048, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(128, dtype=torch.float64) / 128)
    rope = torch.cat((angle.cos(), angle.sin()), 1).float().to(device)
    still = torch.cat((torch.ones(2048, 128), torch.zeros(2048, 128)), 1).to(device)
    usual = _append_us(cache, k, v, table, zero, rope, side)
    zeros = _append_us(cache, torch.zeros_like(k), v, table, zero, rope, side)
    first = _append_us(cache, k, v, table, zero, still, side)
    assert zeros < 3 * usual and first < 3 * usual, (usual, zeros, first)


@pytest.mark.parametrize("kind", [E4M3, BF16])
@pytest.mark.parametrize("rows, heads", [(1, 8), (12, 8), (40, 32)])
def test_sequences_that_share_pages(device, kind, rows, heads):
    """Five sequences whose first pages are the same ones, each with a last page of its own."""
    c = Case(device, [200, 150, 2000, 130, 199], [rows] * 5, heads, 2, 64, 64, kind=kind, seed=70)
    for b in (0, 1, 3, 4):
        c.table[b, :2] = c.table[2, :2]
    c.calls["table"] = c.table.to(device)
    check(c.attend(), *c.expected())
    check(c.attend(window=100, sinks=70), *c.expected(window=100, sinks=70))


def test_the_command_without_a_prompt(device):
    package = Path(__file__).resolve().parents[1] / "plm-anon_amd"
    done = subprocess.run([sys.executable, "-m", "plm_amd.attention_layer", "--prompt", "0", "--rounds", "3", "--cache", "model"],
                          cwd=package, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stderr[-2000:]
    assert "3 rounds of 56 rows from 0 tokens on" in done.stdout and "finite True" in done.stdout


@pytest.mark.parametrize("dtype, kind", [(BF16, E4M3), (FP16, E4M3), (BF16, BF16), (FP16, FP16)])
@pytest.mark.parametrize("shape, wider", [
    (([7], [1], 8, 2, 64, 64), 0),
    (([30, 8, 0], [1] * 3, 4, 4, 128, 16), 0),
    (([300, 40], [5, 2], 20, 4, 80, 32), 0),
    (([130], [56], 4, 1, 256, 64), 0),
    (([20, 0, 3], [3, 1, 2], 10, 1, 64, 16), WIDE),      # 32 columns
    (([3000], [2], 16, 2, 128, 64), 0),                  # cut and joined
])
def test_probabilities_are_not_rounded_to_the_models_type(device, shape, wider, dtype, kind):
    """Up to 32 columns the output's rounding is the only one of the type's: probabilities come in two parts, each off by half
    a step of what is left, 2^-16 in bf16 and 2^-22 in fp16 of a probability, or half of fp16's least, 2^-25 / 2^8."""
    c = Case(device, *shape, dtype=dtype, kind=kind, seed=73, wider=wider)
    want, tol = c.expected()
    half = torch.finfo(dtype).eps / 2
    sizes, most = [], 0.0
    for b, (n, r) in enumerate(zip(c.contexts, c.rows)):
        k, v = c.tokens("k", b, n + r), c.tokens("v", b, n + r)
        q = c.q[c.starts[b]:c.starts[b + 1]]
        _, size, score = oracle.attention(q, k, v, oracle.seen(n, r, n + r, None, 0, None, None), 1 / math.sqrt(c.dim))
        off = 2 * (2.0 ** -24 * (c.dim + 12) * score + 2.0 ** -20) + (n + r) * 2.0 ** -24 + half * half
        sizes.append(off * size + (n + r) * 2.0 ** -33 * float(v.abs().max()))
    off = torch.cat(sizes)
    check(c.attend(), want, off * (1 + half) + half * want.abs() + (2.0 ** -25 if dtype == FP16 else 0.0))
