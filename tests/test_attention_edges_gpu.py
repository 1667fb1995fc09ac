"""The paged cache and its attention at the ends of what they are given: page scales far apart, positions and windows past
any cache, rows that no sequence holds, pages that several sequences read, keys that need no rounding.

Tolerances are those of test_attention_gpu.py, whose cases these are."""

from __future__ import annotations

import math

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
