"""CPU checks of the paged attention's host side: what its calls refuse, before any kernel is launched; the
round's mask; the layout's places; the 64-bit oracle against closed forms."""

from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

from oracle import attention_oracle as oracle
from plm_amd import _lib, attention

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _stub(pages=4, heads=2, dim=64, page=32, dtype=E4M3):
    """A handle whose tensors are on the CPU: every refusal comes before a pointer is used."""
    c = object.__new__(attention.PagedCache)
    c.pages, c.kv_heads, c.page, c.head_dim, c.dtype, c.device = pages, heads, page, dim, dtype, torch.device("cpu")
    kind = {BF16: 0, FP16: 1, E4M3: 2}[dtype]
    c._handle = _lib.KvCache(1 << 20, 1 << 20, 1 << 20, 1 << 20, pages, heads, page, dim, kind)
    c._ref, c._index = ctypes.addressof(c._handle), -1
    return c


def _call(seqs=2, rows=3, heads=4, kv=2, dim=64, dtype=BF16):
    return dict(q=torch.zeros(seqs * rows, heads, dim, dtype=dtype), k=torch.zeros(seqs * rows, kv, dim, dtype=dtype),
                v=torch.zeros(seqs * rows, kv, dim, dtype=dtype), table=torch.zeros(seqs, 3, dtype=torch.int32),
                lengths=torch.zeros(seqs, dtype=torch.int64))


def test_cache_refuses():
    make = attention._shapes(3, 2, 32, 80, True)
    k, v = (torch.zeros(s, dtype=torch.uint8).view(E4M3) for s in make)
    s = torch.ones(3, 2)
    with pytest.raises(TypeError):
        attention.PagedCache(k.float(), v.float(), head_dim=80)
    with pytest.raises(TypeError):
        attention.PagedCache(k, v.view(torch.uint8).to(BF16), s, s, head_dim=80)
    for dim in (0, 7, 12, 264):
        with pytest.raises(ValueError):
            attention.PagedCache(k, v, s, s, head_dim=dim)
    with pytest.raises(ValueError):   # 40 dimensions are one chunk, not two
        attention.PagedCache(k, v, s, s, head_dim=40)
    with pytest.raises(ValueError):
        attention.PagedCache(v, k, s, s, head_dim=80)
    with pytest.raises(ValueError):
        attention.PagedCache(k, v, head_dim=80)
    with pytest.raises(ValueError):
        attention.PagedCache(k, v, s, s.double(), head_dim=80)
    with pytest.raises(ValueError):
        attention.PagedCache(k, v, s, s[:, :1], head_dim=80)
    with pytest.raises(ValueError):
        attention.PagedCache(k.transpose(0, 1), v, s, s, head_dim=80)
    with pytest.raises(RuntimeError):   # all in order, but on the CPU
        attention.PagedCache(k, v, s, s, head_dim=80)
    with pytest.raises(ValueError):
        attention.PagedCache.empty(3, 2, 80, page=48, device="cpu")
    with pytest.raises(TypeError):
        attention.PagedCache.empty(3, 2, 80, dtype=torch.float32, device="cpu")


@pytest.mark.parametrize("change, error", [
    (dict(q=torch.zeros(6, 3, 64, dtype=BF16)), ValueError),            # 3 heads over 2
    (dict(q=torch.zeros(6, 4, 32, dtype=BF16)), ValueError),
    (dict(q=torch.zeros(6, 256, dtype=BF16)), ValueError),
    (dict(q=torch.zeros(0, 4, 64, dtype=BF16)), ValueError),
    (dict(q=torch.zeros(5, 4, 64, dtype=BF16)), ValueError),            # 5 rows of 2 sequences
    (dict(q=torch.zeros(6, 4, 64)), TypeError),
    (dict(table=torch.zeros(2, 3)), ValueError),
    (dict(table=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError),
    (dict(table=torch.zeros(2, 0, dtype=torch.int32)), ValueError),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(lengths=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(row_starts=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(row_starts=torch.zeros(3, dtype=torch.int64), max_rows=7), ValueError),
    (dict(row_starts=torch.zeros(3, dtype=torch.int64), max_rows=0), ValueError),
    (dict(max_rows=2), ValueError),
    (dict(window=0), ValueError),
    (dict(sinks=-1), ValueError),
    (dict(mask=torch.zeros(2, 1, dtype=torch.int32)), ValueError),      # 2 of 3 rows
    (dict(mask=torch.zeros(3, 1, dtype=torch.int64)), ValueError),
    (dict(mask=torch.zeros(3, 0, dtype=torch.int32)), ValueError),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(scale=math.nan), ValueError),
])
def test_attend_refuses(change, error):
    c = _call()
    args = {"q": c["q"], "table": c["table"], "lengths": c["lengths"], **change}
    with pytest.raises(error):
        attention.attend(_stub(), args.pop("q"), args.pop("table"), args.pop("lengths"), **args)


@pytest.mark.parametrize("change, error", [
    (dict(k=torch.zeros(6, 3, 64, dtype=BF16)), ValueError),
    (dict(k=torch.zeros(0, 2, 64, dtype=BF16)), ValueError),
    (dict(v=torch.zeros(5, 2, 64, dtype=BF16)), ValueError),
    (dict(v=torch.zeros(6, 2, 64, dtype=FP16)), TypeError),
    (dict(q=torch.zeros(6, 4, 64, dtype=FP16)), TypeError),
    (dict(rope=torch.zeros(9, 66)), ValueError),
    (dict(rope=torch.zeros(9, 7)), ValueError),
    (dict(rope=torch.zeros(0, 8)), ValueError),
    (dict(rope=torch.zeros(9, 8, dtype=torch.float64)), ValueError),
    (dict(rope=torch.zeros(9, 16)[:, ::2]), ValueError),
    (dict(positions=torch.zeros(6, dtype=torch.int32)), ValueError),
    (dict(lengths=torch.zeros(1, dtype=torch.int64)), ValueError),
])
def test_append_refuses(change, error):
    args = {**_call(), **change}
    with pytest.raises(error):
        attention.append_kv(_stub(), args.pop("q"), args.pop("k"), args.pop("v"), args.pop("table"), args.pop("lengths"), **args)


def test_types_of_rows_and_cache_go_together():
    c = _call(dtype=FP16)
    with pytest.raises(TypeError):
        attention.attend(_stub(dtype=BF16), c["q"], c["table"], c["lengths"])
    with pytest.raises(TypeError):
        attention.read_kv(_stub(), c["table"], c["lengths"], c["lengths"], 4, torch.float32)
    with pytest.raises(ValueError):
        attention.read_kv(_stub(), c["table"], c["lengths"], c["lengths"], 0, BF16)
    with pytest.raises(ValueError):
        attention.read_kv(_stub(), c["table"].long(), c["lengths"], c["lengths"], 4, BF16)


def test_structs_are_the_headers():
    """The packed structs have the header's fields, in its order."""
    text = (Path(__file__).resolve().parents[1] / "include" / "plm_amd.h").read_text()

    def fields(name):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        found = []
        for line in body.strip().split(";"):
            words = line.replace("*", " ").replace(",", " ").split()
            words = [w for w in words if w not in ("const", "void", "int64_t", "int32_t", "uint32_t", "float", "double")]
            if words[:1] == ["plm_kv_rows"]:
                words = list(fields("plm_kv_rows"))
            elif words[:1] == ["plm_kv_cache"]:
                words = words[1:]
            found += words
        return tuple(found)

    assert fields("plm_kv_rows") == _lib.KV_ROWS
    assert fields("plm_append_call") == _lib.APPEND_FIELDS
    assert fields("plm_read_call") == _lib.READ_FIELDS
    assert fields("plm_attend_call") == _lib.ATTEND_FIELDS
    assert fields("plm_kv_cache") == tuple(name for name, _ in _lib.KvCache._fields_)


def test_c_entries_refuse_before_a_launch():
    lib, f = _lib.lib(), 1 << 20   # never dereferenced
    kept = []

    def cache(**more):
        fields = dict(k=f, v=f, k_scale=f, v_scale=f, pages=4, kv_heads=2, page=32, head_dim=64, type=2)
        kept.append(_lib.KvCache(**{**fields, **more}))
        return ctypes.addressof(kept[-1])

    rows = dict(total=6, seqs=2, max_rows=3, table=f, table_stride=3, table_width=3, lengths=f, row_starts=0)

    def attend(space=f, size=1 << 30, **more):
        call = dict(dtype=0, cache=cache(), **rows, q=f, q_row=256, q_head=64, heads=4, out=f, window=0, sinks=0, mask=0,
                    mask_rows=0, mask_words=0, positions=0, scale=0.125)
        assert set(more) <= set(call)
        packed = _lib.pack_attend(*{**call, **more}.values())
        return lib.plm_attend(packed, space, size, None), lib.plm_attend_workspace_bytes(packed)

    assert lib.plm_attend(None, f, 1 << 30, None) == -1 and lib.plm_attend_workspace_bytes(None) == 0
    for bad in (dict(k=None), dict(pages=0), dict(kv_heads=0), dict(page=48), dict(head_dim=60), dict(head_dim=264),
                dict(type=3), dict(k_scale=None), dict(type=1)):
        assert attend(cache=cache(**bad)) == (-1, 0), bad
    for bad in (dict(cache=0), dict(dtype=2), dict(heads=3), dict(heads=0), dict(total=0), dict(total=5), dict(seqs=0),
                dict(max_rows=0), dict(max_rows=7, row_starts=f), dict(table=0), dict(lengths=0), dict(table_width=0),
                dict(table_stride=2), dict(window=-1), dict(sinks=-1), dict(mask=f), dict(mask=f, mask_rows=3), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)):
        assert attend(**bad) == (-1, 0), bad
    for bad in (dict(q=0), dict(out=0)):
        assert attend(**bad)[0] == -1, bad
    for bad in (dict(q=f + 2), dict(out=f + 8), dict(q_row=100), dict(q_head=4)):
        assert attend(**bad)[0] == -2, bad
    wide = dict(table_stride=64, table_width=64)
    need = attend(space=None, **wide)[1]
    assert need > 0 and attend(size=need - 1, **wide) == (-4, need) and attend(space=None, **wide) == (-4, need)
    assert attend(q=0)[1] == 0   # short tables are never cut

    def append(**more):
        call = dict(dtype=0, cache=cache(), **rows, q=f, q_row=256, q_head=64, heads=4, q_out=f, k=f, k_row=128, k_head=64, v=f,
                    v_row=128, v_head=64, rope=f, rope_rows=9, rotary=64, side_by_side=0, positions=0)
        assert set(more) <= set(call)
        return lib.plm_kv_append(_lib.pack_append(*{**call, **more}.values()), None)

    assert lib.plm_kv_append(None, None) == -1
    for bad in (dict(dtype=5), dict(heads=0), dict(q_out=0), dict(k=0), dict(v=0), dict(total=7), dict(rotary=66), dict(rotary=3),
                dict(rope_rows=0), dict(cache=cache(head_dim=0))):
        assert append(**bad) == -1, bad
    for bad in (dict(k=f + 4), dict(rope=f + 4), dict(k_row=132), dict(q_out=f + 2)):
        assert append(**bad) == -2, bad

    def read(**more):
        call = dict(dtype=0, cache=cache(), table=f, table_stride=3, table_width=3, first=f, ends=f, seqs=2, most=4, k=f, v=f)
        assert set(more) <= set(call)
        return lib.plm_kv_read(_lib.pack_read(*{**call, **more}.values()), None)

    assert lib.plm_kv_read(None, None) == -1
    for bad in (dict(first=0), dict(ends=0), dict(most=0), dict(seqs=0), dict(table_width=0), dict(table_width=4), dict(k=0)):
        assert read(**bad) == -1, bad
    assert read(k=f + 2) == -2


@pytest.mark.parametrize("k", [1, 2, 6, 7, 10])
def test_round_mask_is_the_rounds(k):
    bits, places = attention.round_mask(k, device="cpu")
    see, want = oracle.round_rows(k)
    rows = k + k * k
    got = torch.stack([(bits[:, r // 32].long() >> (r % 32)) & 1 for r in range(rows)], 1).bool()
    assert torch.equal(got, see) and torch.equal(places, want)
    assert bits.shape == (rows, -(-rows // 32)) and bits.dtype == torch.int32 and places.dtype == torch.int64
    # By hand: proposal j of block i is i + 1 + j places on and sees i + 1 verify rows and j + 1 of its own.
    for i in range(k):
        for j in range(k):
            assert int(see[k + i * k + j].sum()) == i + 1 + j + 1


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("name", ["k", "v"])
def test_every_place_of_a_unit_is_taken_once(e4m3, name):
    n, e = torch.meshgrid(torch.arange(16), torch.arange(64), indexing="ij")
    assert torch.equal(oracle.place(name, e4m3, n, e).flatten().sort().values, torch.arange(1024))


def test_oracle_pieces():
    codes = torch.arange(256, dtype=torch.uint8).view(E4M3).float().double()
    finite = codes[~codes.isnan()]
    assert torch.equal(oracle.e4m3(finite), finite)
    x = torch.linspace(-448, 448, 4001, dtype=torch.float64)
    assert torch.equal(oracle.e4m3(x), x.float().to(E4M3).float().double())
    assert oracle.scale_of(torch.tensor([0.0, 448.0, 449.0, 1.75, 1.7501])).tolist() == [2.0 ** -64, 1.0, 2.0, 2.0 ** -8, 2.0 ** -7]
    turn = torch.tensor([[0.0, 1.0, 1.0, 0.0]])   # pair 0 by a quarter turn, pair 1 not at all
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]]])
    assert oracle.rotate(x, turn, False).tolist() == [[[-3.0, 2.0, 1.0, 4.0, 5.0, 6.0]]]
    assert oracle.rotate(x, turn, True).tolist() == [[[-2.0, 1.0, 3.0, 4.0, 5.0, 6.0]]]
    # Equal scores: the mean of what is seen; nothing seen: zero.
    v = torch.arange(12, dtype=torch.float64).reshape(6, 1, 2)
    see = oracle.seen(4, 2, 6, 2, 1, None, None)
    assert see.tolist() == [[True, False, False, True, True, False], [True, False, False, False, True, True]]
    out, size, _ = oracle.attention(torch.zeros(2, 1, 2), torch.zeros(6, 1, 2), v, see, 1.0)
    assert torch.allclose(out[0, 0], v[[0, 3, 4], 0].mean(0)) and torch.allclose(size, out)
    out, _, _ = oracle.attention(torch.zeros(1, 1, 2), torch.zeros(6, 1, 2), v, torch.zeros(1, 6, dtype=torch.bool), 1.0)
    assert out.abs().max() == 0
    assert math.isclose(float(oracle.attention(torch.ones(1, 1, 2), torch.ones(6, 1, 2), v, see[:1], 0.5)[2]), 1.0)


def test_pages_are_handed_out_and_taken_back():
    from plm_amd.attention_layer import PageTable

    cache = _stub(pages=5, page=16)
    pages = PageTable(cache, 2, 64)
    assert pages.table.tolist() == [[-1] * 4] * 2
    pages.reserve(0, 17)
    pages.reserve(1, 33)
    held = [t for t in pages.table.flatten().tolist() if t >= 0]
    assert len(held) == 5 and sorted(held) == [0, 1, 2, 3, 4]
    pages.reserve(0, 32)   # already there
    with pytest.raises(RuntimeError):
        pages.reserve(0, 33)
    with pytest.raises(ValueError):
        pages.reserve(1, 65)
    pages.free(1)
    assert pages.table[1].tolist() == [-1] * 4
    pages.reserve(0, 64)
    assert sorted(pages.table[0].tolist()) == sorted({*pages.table[0].tolist()})
