"""The paged cache's append and read and the attention over it, against the definition in 64 bits.

Tolerances. Half a step of a type is ``finfo(t).eps / 2`` of the value (e4m3: 2^-4, and 2^-10 scales below its
smallest normal). Append: a 16-bit value is rounded once from fp32 arithmetic of two products (3 * 2^-24 of
|a| + |b|); an 8-bit one once to its page's scale. Attention, with A the attention of |values|: probabilities
are rounded once to the model's type and the output once; scores carry fp32 products and sums (dim + 8 roundings
of sum |q k| scale, and four of the exponent's argument), the exponential 2^-20, the sums over n tokens n 2^-24.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import attention_oracle as oracle
from plm_amd import attention

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


class Case:
    """A cache with random pages, a shuffled table and packed rows."""

    def __init__(self, device, contexts, rows, heads, kv_heads, dim, page, dtype=BF16, kind=E4M3, seed=0, spare=2,
                 wider=0, loud=1.0):
        g = torch.Generator().manual_seed(seed)
        need = [max(1, -(-(c + r) // page)) for c, r in zip(contexts, rows)]
        pages = sum(need) + spare
        self.cache = cache = attention.PagedCache.empty(pages, kv_heads, dim, page=page, dtype=kind, device=device)
        ids = torch.randperm(pages, generator=g)[: sum(need)].to(torch.int32)
        self.table = torch.full((len(need), max(need) + wider), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        for p in range(pages):
            for name, x, s in (("k", cache.k, cache.k_scale), ("v", cache.v, cache.v_scale)):
                values = torch.randn(page, kv_heads, dim, generator=g).double() * loud
                if kind == E4M3:
                    scale = oracle.scale_of(values.abs().amax((0, 2)))
                    s[p] = scale.float()
                    values = oracle.e4m3(values / scale[None, :, None]).float().to(E4M3)
                else:
                    values = values.to(kind)
                oracle.put_page(x, p, values, name)
        self.contexts, self.rows, self.dim, self.page, self.dtype, self.kind = contexts, rows, dim, page, dtype, kind
        self.heads, self.kv_heads, self.device, self.g = heads, kv_heads, device, g
        total = sum(rows)
        self.q = torch.randn(total, heads, dim, generator=g).to(dtype)
        self.k = (torch.randn(total, kv_heads, dim, generator=g) * loud).to(dtype)
        self.v = (torch.randn(total, kv_heads, dim, generator=g) * loud).to(dtype)
        self.starts = [sum(rows[:b]) for b in range(len(rows) + 1)]
        same = len(set(rows)) == 1
        self.calls = dict(table=self.table.to(device), lengths=torch.tensor(contexts, device=device),
                          row_starts=None if same else torch.tensor(self.starts, device=device), max_rows=max(rows))

    def tokens(self, name, b, n):
        """The first n cached tokens of sequence b in 64 bits; pages that are not there read as zeros."""
        c = self.cache
        x, s = (c.k, c.k_scale) if name == "k" else (c.v, c.v_scale)
        parts = [torch.zeros(0, self.kv_heads, self.dim, dtype=torch.float64)]
        for i in range(-(-n // self.page)):
            p = int(self.table[b, i]) if i < self.table.shape[1] else -1
            parts.append(oracle.get_page(x, s, p, self.kv_heads, self.page, self.dim, name) if 0 <= p < c.pages else
                         torch.zeros(self.page, self.kv_heads, self.dim, dtype=torch.float64))
        return torch.cat(parts)[:n]

    def expected(self, window=None, sinks=0, see=None, places=None, scale=None, hidden=None):
        """(output, tolerance) of the whole call. ``hidden[b]``: tokens of sequence b that no row sees."""
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        outs, tols = [], []
        for b, (c, r) in enumerate(zip(self.contexts, self.rows)):
            n = c + r
            mine = None if places is None else places[self.starts[b]:self.starts[b + 1]]
            vis = oracle.seen(c, r, n, window, sinks, see, mine)
            if hidden is not None:
                vis[:, hidden[b]] = False
            k, v = self.tokens("k", b, n), self.tokens("v", b, n)
            out, size, most = oracle.attention(self.q[self.starts[b]:self.starts[b + 1]], k, v, vis, scale)
            half = torch.finfo(self.dtype).eps / 2
            off = 2 * (2.0 ** -24 * (self.dim + 8 + 4) * most + 2.0 ** -20) + n * 2.0 ** -24
            outs.append(out)
            tols.append((half + off) * size * (1 + 2 * half) + half * out.abs() + 1e-30 + (2.0 ** -25 if self.dtype == FP16 else 0))
        return torch.cat(outs), torch.cat(tols)

    def attend(self, q=None, **more):
        return attention.attend(self.cache, (self.q if q is None else q).to(self.device), **{**self.calls, **more})


def check(got, want, tol, what=""):
    got = got.cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol).nan_to_num(9e9).max()):.3g} tolerances"


# contexts, rows, heads, kv_heads, dim, page
SHAPES = [
    ([0], [1], 1, 1, 8, 16),                           # one token and nothing before it
    ([499], [1], 8, 2, 64, 64),
    ([0, 1, 15, 16, 17, 700], [1] * 6, 8, 1, 128, 16),  # lengths around a unit, a table of very unlike rows
    ([33, 250, 1000], [3, 1, 5], 20, 4, 80, 32),       # ragged, heads of 80, groups of five
    ([100, 3], [40, 7], 4, 4, 96, 128),
    ([130], [70], 8, 1, 128, 64),                      # several tiles of columns, the last part full
    ([61, 0], [33, 33], 2, 2, 256, 16),
    ([90], [21], 6, 2, 192, 64),
    ([5000], [2], 16, 2, 128, 64),                     # one sequence cut into many ranges
    ([2100, 40], [17, 17], 64, 1, 72, 32),             # one key head for 64, the last 16 dimensions half full
]


@pytest.mark.parametrize("dtype, kind", [(BF16, E4M3), (FP16, E4M3), (BF16, BF16), (FP16, FP16)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_causal(device, shape, dtype, kind):
    c = Case(device, *SHAPES[shape], dtype=dtype, kind=kind, seed=shape)
    check(c.attend(), *c.expected())


# A table wide enough that the sizes alone speak for much work: the 32-, 64- and 128-column kernels on small inputs,
# and sequences cut into ranges.
WIDE = 12000
WIDE_SHAPES = [
    ([70, 0, 3], [3, 1, 2], 10, 1, 64, 16),              # 32 columns, in part
    ([901, 17], [5, 8], 8, 2, 128, 32),                  # 32 columns, two chunks
    ([130, 5], [21, 40], 8, 2, 64, 16),                  # 64 columns, the last tile in part
    ([1100], [56], 16, 4, 128, 64),                      # 64 columns, cut
    ([75, 300], [33, 7], 6, 2, 80, 16),
    ([200], [30], 4, 2, 192, 128),
    ([40, 333], [25, 12], 4, 1, 256, 16),                # 64 columns of four chunks, one set in LDS
    ([90], [520], 64, 1, 16, 64),                        # 128 columns
    ([600, 10], [1040, 600], 20, 1, 72, 32),             # 128 columns, two chunks, the second in part
]


@pytest.mark.parametrize("dtype, kind", [(BF16, E4M3), (FP16, E4M3), (BF16, BF16), (FP16, FP16)])
@pytest.mark.parametrize("shape", range(len(WIDE_SHAPES)))
def test_wide_tables(device, shape, dtype, kind):
    c = Case(device, *WIDE_SHAPES[shape], dtype=dtype, kind=kind, seed=50 + shape, wider=WIDE)
    check(c.attend(), *c.expected())


# Groups of 17 to 100 steps of 32 tokens that all find a CU: workgroups of as many wavefronts as it holds.
MIDDLING_SHAPES = [
    ([600], [1], 4, 2, 64, 64),                          # 19 steps over 16 wavefronts (in 8 bits)
    ([1000, 3, 544, 0], [1] * 4, 8, 2, 128, 16),         # 12 wavefronts, some without a step
    ([3100], [9], 16, 4, 128, 64),                       # three tiles, the last in part
    ([800, 70], [6, 33], 6, 2, 80, 32),
    ([580], [5], 8, 2, 192, 16),
    ([900, 31], [5, 4], 12, 3, 256, 128),
    ([1500], [40], 3, 3, 8, 32),
]


@pytest.mark.parametrize("dtype, kind", [(BF16, E4M3), (FP16, E4M3), (BF16, BF16), (FP16, FP16)])
@pytest.mark.parametrize("shape", range(len(MIDDLING_SHAPES)))
@pytest.mark.parametrize("window, sinks", [(None, 0), (577, 40)])
def test_middling_contexts(device, shape, dtype, kind, window, sinks):
    c = Case(device, *MIDDLING_SHAPES[shape], dtype=dtype, kind=kind, seed=70 + shape)
    check(c.attend(window=window, sinks=sinks), *c.expected(window, sinks))


@pytest.mark.parametrize("k, heads, kv_heads, dim, dtype, kind", [(6, 20, 20, 80, FP16, E4M3), (7, 16, 4, 128, BF16, E4M3),
                                                                (5, 8, 2, 64, BF16, BF16)])
@pytest.mark.parametrize("window", [None, 600])
def test_round_after_middling_contexts(device, k, heads, kv_heads, dim, dtype, kind, window):
    c = Case(device, [1100, 605], [k + k * k] * 2, heads, kv_heads, dim, 32, dtype=dtype, kind=kind, seed=k)
    bits, places = attention.round_mask(k, device=device)
    see, want = oracle.round_rows(k)
    at = (torch.tensor(c.contexts)[:, None] + want).flatten()
    got = c.attend(mask=bits, positions=at.to(device), window=window, sinks=3)
    check(got, *c.expected(window, 3, see, at))


@pytest.mark.parametrize("kind", [E4M3, BF16])
def test_nan_after_a_middling_context_stays_with_its_row(device, kind):
    c = Case(device, [700], [3], 4, 2, 128, 64, kind=kind, seed=5)
    want, tol = c.expected()
    values = oracle.get_page(c.cache.v, c.cache.v_scale, int(c.table[0, 702 // 64]), 2, 64, 128, "v")
    scale = 1.0 if kind == BF16 else c.cache.v_scale[int(c.table[0, 702 // 64])].cpu().double()[None, :, None]
    values = values / scale
    values[702 % 64] = math.nan
    oracle.put_page(c.cache.v, int(c.table[0, 702 // 64]), values.float().to(kind), "v")
    got = c.attend()
    check(got[:2], want[:2], tol[:2])
    assert got[2].isnan().all()


@pytest.mark.parametrize("window, sinks", [(16, 4), (100, 40), (777, 19)])
@pytest.mark.parametrize("dtype, kind", [(BF16, E4M3), (FP16, FP16)])
def test_window_of_many_columns(device, window, sinks, dtype, kind):
    """Heads enough that a window's short walks are work for the 64-column (and, through 777, the 128-column) kernel."""
    c = Case(device, [30], [760], 128, 128, 8, 16, dtype=dtype, kind=kind, seed=window)
    check(c.attend(window=window, sinks=sinks), *c.expected(window, sinks))


@pytest.mark.parametrize("k, heads, kv_heads, dim, dtype, kind", [(6, 20, 20, 80, FP16, E4M3), (7, 16, 4, 128, BF16, E4M3),
                                                                (10, 8, 1, 64, FP16, FP16), (7, 8, 2, 256, BF16, BF16)])
@pytest.mark.parametrize("window", [None, 50])
def test_round_of_many_columns(device, k, heads, kv_heads, dim, dtype, kind, window):
    rows = k + k * k
    c = Case(device, [300, 0, 77], [rows] * 3, heads, kv_heads, dim, 32, dtype=dtype, kind=kind, seed=k, wider=WIDE)
    bits, places = attention.round_mask(k, device=device)
    see, want = oracle.round_rows(k)
    at = (torch.tensor(c.contexts)[:, None] + want).flatten()
    got = c.attend(mask=bits, positions=at.to(device), window=window, sinks=3)
    check(got, *c.expected(window, 3, see, at))


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (100, 40), (777, 19), (10 ** 12, 5)])
@pytest.mark.parametrize("kind", [E4M3, BF16])
def test_window(device, window, sinks, kind):
    c = Case(device, [1500, 0, 60], [9, 130, 1], 8, 2, 64, 32, kind=kind, seed=window % 97)
    check(c.attend(window=window, sinks=sinks), *c.expected(window, sinks))


@pytest.mark.parametrize("k, heads, kv_heads, dim", [(1, 2, 2, 64), (6, 20, 20, 80), (7, 16, 4, 128), (10, 8, 1, 64)])
@pytest.mark.parametrize("window", [None, 50])
def test_round(device, k, heads, kv_heads, dim, window):
    rows = k + k * k
    c = Case(device, [300, 0, 77], [rows] * 3, heads, kv_heads, dim, 32, seed=k)
    bits, places = attention.round_mask(k, device=device)
    see, want = oracle.round_rows(k)
    at = (torch.tensor(c.contexts)[:, None] + want).flatten()
    got = c.attend(mask=bits, positions=at.to(device), window=window, sinks=3)
    check(got, *c.expected(window, 3, see, at))


@pytest.mark.parametrize("heads, wider", [(4, 0), (8, WIDE), (32, WIDE)])
def test_rows_that_see_nothing_are_zero(device, heads, wider):
    c = Case(device, [0, 40], [5, 5], heads, 2, 64, 16, seed=3, wider=wider)
    bits = torch.tensor([[0], [0b10], [0], [0b11111], [0]], dtype=torch.int32)
    see = torch.tensor([[(int(w) >> j) & 1 for j in range(5)] for w in bits[:, 0]], dtype=torch.bool)
    got = c.attend(mask=bits.to(device))
    want, tol = c.expected(see=see)
    check(got, want, tol)
    assert got[[0, 2, 4]].abs().max() == 0 and got[[1, 3]].abs().min() > 0
    # A window whose place is far past every token, and one far before: nothing left, and nothing but the sinks.
    far = torch.full((10,), 10 ** 15, device=device)
    assert c.attend(window=8, positions=far).abs().max() == 0
    check(c.attend(window=8, sinks=2, positions=far), *c.expected(window=8, sinks=2, places=far.cpu()))
    check(c.attend(window=8, positions=-far), *c.expected(window=8, places=-far.cpu()))


@pytest.mark.parametrize("heads, wider", [(4, 0), (1, WIDE), (4, WIDE)])
@pytest.mark.parametrize("kind", [E4M3, FP16])
def test_what_is_masked_does_not_reach_the_rows(device, kind, heads, wider):
    """NaN and infinities in tokens past the end, outside the window, and ahead of a row in its own tile."""
    c = Case(device, [70], [20], heads, 1, 64, 32, dtype=FP16, kind=kind, seed=5, wider=wider)
    window = None if wider else 30        # 16-column tiles; the wider ones, without a window
    want, tol = c.expected(window=window, sinks=1)
    bad = {0x7F, 0xFF} if kind == E4M3 else {0x7C00, 0xFC00, 0x7E00}
    places = [75, 89, 90, 93, 95] if wider else [5, 41, 75, 89, 90, 93, 95]
    for name, x in (("k", c.cache.k), ("v", c.cache.v)):
        flat = oracle._bits(x)
        for t in places:    # left of every window, in row 0's alone, own rows 5 and 19, past the end
            at = oracle._flat(x, int(c.table[0, t // 32]), 1, 32, 64, name)[t % 32].flatten().to(device)
            for i, code in enumerate(sorted(bad)):
                flat[at[i::len(bad)]] = torch.tensor(code, dtype=torch.int32, device=device).to(flat.dtype)
    got = c.attend(window=window, sinks=1).cpu()
    rows = torch.tensor([r for r in range(20) if not any((wider or 70 + r - 30 < t) and t <= 70 + r for t in places)])
    clean = [0, 1, 2, 3, 4] if wider else [1, 2, 3, 4]
    assert rows.tolist() == clean
    dirty = [r for r in range(20) if r not in clean]
    check(got[rows], want[rows], tol[rows])
    assert not torch.isfinite(got[dirty].float()).all(-1).any()


def test_extreme_scores(device):
    """Scores far apart, all alike, and of the model type's largest values."""
    for loud, dtype in ((30.0, BF16), (0.0, BF16), (30.0, FP16)):
        c = Case(device, [200], [3], 2, 1, 64, 16, dtype=dtype, kind=dtype, seed=7, loud=loud)
        check(c.attend(), *c.expected(), what=f"loud {loud}")
    c = Case(device, [64], [1], 1, 1, 64, 16, kind=BF16, seed=8)
    c.cache.v.fill_(2.0 ** 100)
    check(c.attend(), *c.expected(), what="values of 2^100")


@pytest.mark.parametrize("heads, wider", [(4, 0), (64, WIDE)])
def test_pages_of_very_unlike_scales(device, heads, wider):
    """8-bit pages of fp16 rows: values of 2^8 and of 2^-14 next to each other, and pages of zeros."""
    c = Case(device, [150], [2], heads, 1, 64, 16, dtype=FP16, seed=9, wider=wider)
    for i, s in enumerate([2.0 ** 5, 2.0 ** -20, 2.0 ** -9, 2.0 ** -64, 2.0 ** 3, 2.0 ** -6, 1.0, 2.0 ** -30, 2.0 ** -12, 2.0 ** -8]):
        c.cache.v_scale[int(c.table[0, i])] = s
        c.cache.k_scale[int(c.table[0, i])] = 2.0 ** -8 if i % 2 else 2.0 ** -9
    check(c.attend(), *c.expected())


@pytest.mark.parametrize("heads, wider", [(4, 0), (8, WIDE), (32, WIDE)])
def test_pages_that_are_not_there(device, heads, wider):
    c = Case(device, [100, 30], [4, 4], heads, 2, 64, 16, seed=10, wider=wider)
    missing = {0: [1, 3], 1: [0]}
    for b, numbers in missing.items():
        for n in numbers:
            c.table[b, n] = -1 if n % 2 else c.cache.pages
    c.calls["table"] = c.table.to(device)
    hidden = [[t for n in missing[b] for t in range(16 * n, 16 * n + 16)] for b in (0, 1)]
    check(c.attend(), *c.expected(hidden=hidden))
    k, v = attention.read_kv(c.cache, c.calls["table"], torch.tensor([10, 0], device=device),
                             torch.tensor([104, 34], device=device), 94, BF16)
    for b, first in ((0, 10), (1, 0)):
        n = (104, 34)[b] - first
        assert torch.equal(k[b, :n].cpu().double(), c.tokens("k", b, first + n)[first:]) and not k[b, n:].any()
        assert torch.equal(v[b, :n].cpu().double(), c.tokens("v", b, first + n)[first:])
    before = (c.cache.k.view(torch.uint8).clone(), c.cache.v.view(torch.uint8).clone())
    c.calls["table"][:] = -1
    attention.append_kv(c.cache, None, c.k.to(device), c.v.to(device), **c.calls)   # nothing to store the rows in
    assert torch.equal(c.cache.k.view(torch.uint8), before[0]) and torch.equal(c.cache.v.view(torch.uint8), before[1])
    assert c.attend().abs().max() == 0


@pytest.mark.parametrize("heads, wider", [(4, 0), (32, WIDE)])
def test_numbers_out_of_range_shorten_a_sequence(device, heads, wider):
    """Lengths past the table, negative ones, and starts past the rows: no access leaves a buffer, the others hold."""
    c = Case(device, [50, 20], [4, 4], heads, 2, 64, 16, seed=11, wider=wider)
    want, tol = c.expected()
    lengths = torch.tensor([10 ** 14, 20], device=device)
    got = c.attend(lengths=lengths)
    check(got[4:], want[4:], tol[4:])
    got = c.attend(lengths=torch.tensor([-5, 20], device=device))
    check(got[4:], want[4:], tol[4:])
    got = c.attend(row_starts=torch.tensor([-3, 4, 10 ** 12], device=device), max_rows=4)
    check(got[4:], want[4:], tol[4:])
    attention.append_kv(c.cache, c.q.to(device), c.k.to(device), c.v.to(device),
                        **{**c.calls, "lengths": torch.tensor([10 ** 14, -2], device=device)})
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", [E4M3, BF16])
def test_strided_queries_and_wide_tables(device, kind):
    c = Case(device, [500, 20], [6, 6], 8, 2, 64, 32, kind=kind, seed=12, wider=3000)
    want = c.attend()
    check(want, *c.expected())
    qkv = torch.randn(12, 8 + 2 + 2, 64).to(BF16).to(device)
    qkv[:, :8] = c.q.to(device)
    assert torch.equal(c.attend(q=qkv[:, :8]), want)
    narrow = c.calls["table"][:, : c.table.shape[1] - 3000]        # rows of a wider tensor
    assert narrow.stride(0) > narrow.shape[1]
    check(c.attend(table=narrow), *c.expected())
    odd = torch.empty(12 * 8 * 64 + 1, dtype=BF16, device=device)[1:].view(12, 8, 64)
    odd.copy_(c.q)
    assert torch.equal(c.attend(q=odd), want)


@pytest.mark.parametrize("heads, wider", [(4, 0), (64, WIDE)])
def test_sequences_without_rows(device, heads, wider):
    c = Case(device, [50, 0, 20, 7], [0, 3, 0, 2], heads, 1, 64, 16, seed=15, wider=wider)
    check(c.attend(), *c.expected())
    before = c.cache.k.view(torch.uint8).clone()
    attention.append_kv(c.cache, None, c.k.to(device), c.v.to(device), **c.calls)
    for b in (0, 2):
        held = [p for p in c.table[b].tolist() if p >= 0]
        assert torch.equal(before[held], c.cache.k.view(torch.uint8)[held])


def test_many_sequences(device):
    contexts = [(37 * b) % 211 for b in range(150)]
    c = Case(device, contexts, [1 + b % 3 for b in range(150)], 4, 1, 16, 16, seed=13)
    check(c.attend(), *c.expected())
    contexts[77] = 6000    # one that is cut, past the first 64
    c = Case(device, contexts, [1 + b % 3 for b in range(150)], 4, 1, 16, 128, seed=14)
    check(c.attend(), *c.expected())


def test_caches_past_32_bits(device):
    """Pages whose bytes begin past 2^32, and element numbers past 2^31."""
    pages = 140000     # x 4 heads x 64 tokens x 128 dimensions: 4.6e9 bytes each
    cache = attention.PagedCache.empty(pages, 4, 128, page=64, device=device)
    ids = torch.tensor([[pages - 1, 7, pages - 2]], dtype=torch.int32, device=device)
    k, v = (torch.randn(150, 4, 128, device=device).bfloat16() for _ in range(2))
    q = torch.randn(150, 8, 128, device=device).bfloat16()
    zero = torch.zeros(1, dtype=torch.int64, device=device)
    attention.append_kv(cache, None, k, v, ids, zero)
    small = attention.PagedCache.empty(3, 4, 128, page=64, device=device)
    near = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=device)
    attention.append_kv(small, None, k, v, near, zero)
    for far_x, near_x in ((cache.k, small.k), (cache.v, small.v)):
        for i in range(3):
            assert torch.equal(far_x[int(ids[0, i])].view(torch.uint8), near_x[int(near[0, i])].view(torch.uint8))
    assert torch.equal(attention.attend(cache, q, ids, zero), attention.attend(small, q, near, zero))
    ends = torch.tensor([150], device=device)
    far, close = attention.read_kv(cache, ids, zero, ends, 150, BF16), attention.read_kv(small, near, zero, ends, 150, BF16)
    assert torch.equal(far[0], close[0]) and torch.equal(far[1], close[1])


def _turn(dim, rotary, n, device):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(rotary // 2, dtype=torch.float64) / (rotary // 2))
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _expected_append(c, rope, side_by_side, positions):
    """Per sequence: rotated queries, and per touched page (keys, values): (values in 64 bits before the last
    rounding, scale, which tokens are new)."""
    queries, pages = [], {}
    for b, (ctx, r) in enumerate(zip(c.contexts, c.rows)):
        rows = slice(c.starts[b], c.starts[b + 1])
        at = torch.arange(ctx, ctx + r) if positions is None else positions[rows]
        turn = None if rope is None else rope[at]
        queries.append(oracle.rotate(c.q[rows], turn, side_by_side))
        for name, new in (("k", oracle.rotate(c.k[rows], turn, side_by_side)), ("v", c.v[rows].double())):
            x, s = (c.cache.k, c.cache.k_scale) if name == "k" else (c.cache.v, c.cache.v_scale)
            for p in range(ctx // c.page, -(-(ctx + r) // c.page)):
                base, page = p * c.page, int(c.table[b, p])
                value = torch.zeros(c.page, c.kv_heads, c.dim, dtype=torch.float64)
                stay = max(0, ctx - base)
                held = oracle.get_page(x, s, page, c.kv_heads, c.page, c.dim, name)
                value[:stay] = held[:stay]
                lo, hi = max(ctx, base), min(ctx + r, base + c.page)
                value[lo - base:hi - base] = new[lo - ctx:hi - ctx]
                scale = None
                if s is not None:
                    scale = oracle.scale_of(value[lo - base:hi - base].abs().amax((0, 2)))
                    if stay:
                        scale = torch.maximum(scale, s[page].cpu().double())
                pages[name, page] = (value, scale, lo - base, hi - base)
    return torch.cat(queries), pages


APPENDS = [
    # contexts, rows, heads, kv_heads, dim, page, rotary, side by side
    ([0], [1], 1, 1, 8, 16, 8, False),
    ([0, 5, 64, 127], [1, 1, 1, 1], 4, 2, 128, 64, 128, False),
    ([371], [56], 8, 2, 64, 32, 64, False),
    ([1001, 0, 63], [100, 33, 1], 8, 8, 80, 128, 40, True),
    ([10, 3], [21, 90], 2, 1, 80, 16, 40, False),            # halves of 20: no multiple of 8
    ([7], [40], 2, 1, 72, 16, 36, True),                     # 36 dimensions turn: the last group in part
    ([100, 1], [300, 2], 4, 2, 256, 128, 256, False),
    ([13], [50], 4, 1, 96, 32, 2, True),
    ([13], [50], 4, 1, 96, 32, 0, False),                    # no rotation
]


@pytest.mark.parametrize("dtype, kind", [(BF16, E4M3), (FP16, E4M3), (BF16, BF16), (FP16, FP16)])
@pytest.mark.parametrize("shape", range(len(APPENDS)))
def test_append(device, shape, dtype, kind):
    *sizes, rotary, side = APPENDS[shape]
    # Louder new rows than the pages hold: the scales of pages with rows from before grow.
    c = Case(device, *sizes, dtype=dtype, kind=kind, seed=20 + shape)
    c.k, c.v = (c.k * 5).to(dtype), (c.v / 3).to(dtype)
    rope = _turn(c.dim, rotary, 1200, device) if rotary else None
    positions = None if shape % 2 else torch.randint(0, 1200, (sum(c.rows),), generator=c.g)
    want_q, pages = _expected_append(c, rope, side, positions)
    others = [p for p in range(c.cache.pages) if ("k", p) not in pages]
    before = [x.view(torch.uint8)[others].clone() for x in (c.cache.k, c.cache.v)]
    got_q = attention.append_kv(c.cache, c.q.to(device), c.k.to(device), c.v.to(device), c.calls["table"], c.calls["lengths"],
                                rope=None if rope is None else rope.to(device), interleaved=side,
                                positions=None if positions is None else positions.to(device),
                                row_starts=c.calls["row_starts"], max_rows=c.calls["max_rows"])
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == FP16 else 0.0
    arithmetic = 6 * 2.0 ** -24 * float(c.q.double().abs().max())
    check(got_q, want_q, half * want_q.abs() + 2 * arithmetic + tiny, "queries")
    assert torch.equal(before[0], c.cache.k.view(torch.uint8)[others]) and torch.equal(before[1], c.cache.v.view(torch.uint8)[others])
    arithmetic = 6 * 2.0 ** -24 * float(c.k.double().abs().max())
    for (name, page), (value, scale, lo, hi) in pages.items():
        x, s = (c.cache.k, c.cache.k_scale) if name == "k" else (c.cache.v, c.cache.v_scale)
        got = oracle.get_page(x, s, page, c.kv_heads, c.page, c.dim, name)
        if scale is None:
            assert torch.equal(got[:lo], value[:lo])
            check(got[lo:hi], value[lo:hi], half * value[lo:hi].abs() + 2 * arithmetic + tiny, f"{name} of page {page}")
            continue
        assert torch.equal(s[page].cpu().double(), scale), (name, page)
        # Rows that stay: the page's rounding alone, and where its scale stays they are not touched.
        assert torch.equal(got[:lo], oracle.e4m3(value[:lo] / scale[:, None]) * scale[:, None])
        tol = (2.0 ** -4 * value[lo:hi].abs()).maximum(2.0 ** -10 * scale[None, :, None]) + 2 * arithmetic
        check(got[lo:hi], value[lo:hi], tol, f"{name} of page {page}")


@pytest.mark.parametrize("dim, rotary, side", [(128, 128, False), (64, 64, True), (80, 40, False), (80, 40, True)])
@pytest.mark.parametrize("cosine", [1.0625, 1.1875])
def test_turned_keys_round_once(device, dim, rotary, side, cosine):
    """Turned keys 2^-30 to either side of the middle between two codes: beyond fp32's reach, and rounded the right way."""
    c = Case(device, [0, 3], [40, 30], 2, 2, dim, 32, seed=3)
    c.k = torch.where(torch.randn(c.k.shape, generator=c.g) < 0, -1.0, 1.0).to(BF16)
    c.k[::2] *= 256   # pages' scales are 1
    half = rotary // 2
    sine = torch.where(torch.randn(100, half, generator=c.g) < 0, -2.0 ** -30, 2.0 ** -30)
    rope = torch.cat((torch.full((100, half), cosine), sine), 1)
    _, pages = _expected_append(c, rope, side, None)
    attention.append_kv(c.cache, None, c.k.to(device), c.v.to(device), c.calls["table"], c.calls["lengths"],
                        rope=rope.to(device), interleaved=side, row_starts=c.calls["row_starts"], max_rows=c.calls["max_rows"])
    for (name, page), (value, scale, lo, hi) in pages.items():
        if name == "k":
            assert torch.equal(c.cache.k_scale[page].cpu().double(), scale)
            got = oracle.get_page(c.cache.k, c.cache.k_scale, page, c.kv_heads, c.page, c.dim, "k")
            assert torch.equal(got[lo:hi], (oracle.e4m3(value / scale[:, None]) * scale[:, None])[lo:hi])


def test_append_in_steps_is_what_was_appended(device):
    """A prompt, then tokens one by one and in rounds that are partly taken back, through a page's life."""
    cache = attention.PagedCache.empty(9, 2, 64, page=16, device=device)
    table = torch.randperm(9, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None].to(device)
    g = torch.Generator().manual_seed(2)
    kept = []
    length = 0
    for rows, keep in ((21, 21), (1, 1), (12, 3), (12, 1), (1, 1), (30, 30), (1, 1), (40, 5), (17, 17)):
        k, v = (torch.randn(rows, 2, 64, generator=g).bfloat16() for _ in range(2))
        attention.append_kv(cache, None, k.to(device), v.to(device), table, torch.tensor([length], device=device))
        kept.append((k[:keep], v[:keep]))
        length += keep
        want = [torch.cat([x[i] for x in kept]).double() for i in (0, 1)]
        got = attention.read_kv(cache, table, torch.zeros(1, dtype=torch.int64, device=device),
                                torch.tensor([length], device=device), length + 3, BF16)
        for x, w in zip(got, want):
            x = x[0].cpu().double()
            assert x[length:].abs().max() == 0
            # A scale grows a few times here; each rounding of a value of up to 5 is within 2^-4 of it.
            assert ((x[:length] - w).abs() <= 3 * 2.0 ** -4 * w.abs() + 3 * 2.0 ** -10 * 2.0 ** -6).all()


@pytest.mark.parametrize("kind", [E4M3, BF16])
def test_append_of_what_is_not_finite(device, kind):
    c = Case(device, [5], [6], 2, 1, 64, 16, kind=kind, seed=30)
    c.k[1, 0, 3], c.k[2, 0, 9], c.v[3, 0, 5], c.v[4, 0, 63] = math.inf, math.nan, -math.inf, math.nan
    c.k[5] = 0
    attention.append_kv(c.cache, None, c.k.to(device), c.v.to(device), **c.calls)
    for name, new in (("k", c.k), ("v", c.v)):
        got = c.tokens(name, 0, 11)[5:]
        assert torch.equal(torch.isfinite(got), torch.isfinite(new.double())), name
        fine = torch.isfinite(new)
        step = 2.0 ** -4 if kind == E4M3 else 0.0
        assert ((got - new.double())[fine].abs() <= step * new.double()[fine].abs() + (2.0 ** -10 * 2.0 ** -6 if step else 0)).all()


def test_positions_outside_the_table_are_nan(device):
    c = Case(device, [0], [4], 2, 1, 64, 16, kind=BF16, seed=31)
    rope = _turn(64, 32, 10, device).to(device)
    at = torch.tensor([0, -1, 10, 10 ** 15], device=device)
    q = attention.append_kv(c.cache, c.q.to(device), c.k.to(device), c.v.to(device), **c.calls, rope=rope, positions=at)
    assert torch.isfinite(q[0]).all() and torch.isnan(q[1:, :, :32]).all()
    assert torch.equal(q[1:, :, 32:].cpu(), c.q[1:, :, 32:])
    k = c.tokens("k", 0, 4)
    assert torch.isfinite(k[0]).all() and torch.isnan(k[1:, :, :32]).all()


def test_append_reads_views_of_the_qkv_product(device):
    sizes = ([9, 40], [3, 3], 4, 2, 64, 32)
    a, b = Case(device, *sizes, seed=32), Case(device, *sizes, seed=32)
    rope = _turn(64, 64, 100, device).to(device)
    qkv = torch.cat((a.q, a.k, a.v), 1).to(device)
    q1 = attention.append_kv(a.cache, qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], **a.calls, rope=rope)
    q2 = attention.append_kv(b.cache, b.q.to(device), b.k.to(device), b.v.to(device), **b.calls, rope=rope)
    assert torch.equal(q1, q2)
    for x, y in ((a.cache.k, b.cache.k), (a.cache.v, b.cache.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert torch.equal(a.cache.k_scale, b.cache.k_scale) and torch.equal(a.cache.v_scale, b.cache.v_scale)


def test_read_from_inside_a_page(device):
    c = Case(device, [70, 9], [1, 1], 2, 2, 80, 16, seed=33)
    for first, ends, most in (([3, 1], [70, 9], 67), ([0, 0], [1, 0], 1), ([69, 70], [200, 9], 5), ([14, 6], [19, 9], 4)):
        k, v = attention.read_kv(c.cache, c.calls["table"], torch.tensor(first, device=device),
                                 torch.tensor(ends, device=device), most, BF16)
        for b in (0, 1):
            for name, got in (("k", k), ("v", v)):
                want = torch.zeros(most, 2, 80, dtype=torch.float64)
                stop = min(ends[b], first[b] + most, c.page * c.table.shape[1])
                if stop > first[b]:
                    want[: stop - first[b]] = c.tokens(name, b, stop)[first[b]:]
                assert torch.equal(got[b].cpu().double(), want), (first, name, b)


def test_results_repeat_and_streams_do_not_meet(device):
    """The same bits every time; calls on two streams at once, each with ranges to join."""
    c = Case(device, [4000, 2500], [2, 2], 8, 2, 64, 64, seed=40)
    want = c.attend()
    check(want, *c.expected())
    q = c.q.to(device)
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    torch.cuda.synchronize()
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(device))
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(attention.attend(c.cache, q, **c.calls))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_graph_of_a_layer_step(device):
    """Append and attention captured once and replayed as the sequences grow, with eager calls between."""
    a = Case(device, [600, 1300], [1, 1], 8, 2, 64, 64, seed=41)
    b = Case(device, [600, 1300], [1, 1], 8, 2, 64, 64, seed=41)
    # Room for the tokens to come.
    for c in (a, b):
        spare = torch.tensor([p for p in range(c.cache.pages) if p not in c.table.flatten().tolist()], dtype=torch.int32)
        c.table = torch.cat((c.table, torch.full((2, 1), -1, dtype=torch.int32)), 1)
        for s, n in enumerate((10, 21)):
            c.table[s, n] = spare[s]
        c.calls["table"] = c.table.to(device)
    rope = _turn(64, 64, 2000, device).to(device)
    qkv = torch.cat((a.q, a.k, a.v), 1).to(device)

    def step(c, qkv):
        q = attention.append_kv(c.cache, qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], **c.calls, rope=rope)
        out = attention.attend(c.cache, q, **c.calls)
        c.calls["lengths"] += 1
        return out

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        warm = step(a, qkv)
    torch.cuda.current_stream(device).wait_stream(side)
    assert torch.equal(warm, step(b, qkv))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, qkv)
    for i in range(45):
        qkv.copy_(torch.randn(qkv.shape, generator=a.g).bfloat16())
        graph.replay()
        want = step(b, qkv)
        assert torch.equal(out, want), i
    assert torch.equal(a.calls["lengths"], b.calls["lengths"])
