"""CPU checks of the 8-bit calls' host side: what they refuse before any kernel is launched, the structs, the sizes and
places of the layout, and the 64-bit oracle against closed forms."""

from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

from oracle import fp8_oracle as oracle
from plm_amd import _lib, fp8

BF16, FP16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def test_calls_refuse():
    x = torch.zeros(3, 64, dtype=BF16)
    for bad in (x[0], x[None]):
        with pytest.raises(ValueError):
            fp8.quantize(bad)
    for bad in (x.float(), x.to(E4M3), x.int()):
        with pytest.raises(TypeError):
            fp8.quantize(bad)
    for k in (0, 4, 12, 65):
        with pytest.raises(ValueError):
            fp8.quantize(torch.zeros(3, k, dtype=BF16))
    with pytest.raises(RuntimeError):   # a gradient is refused before the device is looked at
        fp8.quantize(x.float().requires_grad_().bfloat16())
    with pytest.raises(RuntimeError):   # all in order, but on the CPU
        fp8.quantize(x)
    for call in (fp8.linear, fp8.gate_up_silu):
        with pytest.raises(TypeError):
            call(x, x)
    with pytest.raises(RuntimeError):
        fp8.rms_norm(x, None)
    for gate_up in (False, True):
        with pytest.raises(ValueError):
            fp8.Weight.from_blocks(x.to(E4M3), torch.ones(1, 1), gate_up=gate_up)


def test_made_rows_refuse():
    need = fp8_bytes(3, 64)
    codes, scales = torch.zeros(need[0], dtype=torch.uint8).view(E4M3), torch.zeros(need[1], dtype=torch.uint8)
    for c, s, rows, k in ((codes[:-1], scales, 3, 64), (codes, scales[1:], 3, 64), (codes.view(torch.uint8), scales, 3, 64),
                          (codes, scales.view(torch.int32), 3, 64), (codes, scales, 17, 64), (codes, scales, 0, 64),
                          (codes, scales, 3, 60)):
        with pytest.raises(ValueError):
            fp8.Rows(c, s, rows, k)
    with pytest.raises(ValueError):
        fp8.Weight(codes, scales, 3, 64, gate_up=True)
    with pytest.raises(RuntimeError):
        fp8.Rows(codes, scales, 3, 64)


def fp8_bytes(rows, k):
    lib = _lib.lib()
    return int(lib.plm_fp8_codes_bytes(rows, k)), int(lib.plm_fp8_scales_bytes(rows, k))


@pytest.mark.parametrize("rows,k", [(1, 8), (16, 128), (17, 136), (33, 640), (100, 1032)])
def test_every_place_is_taken_once(rows, k):
    frags, blocks = -(-rows // 16), -(-k // 128)
    assert fp8_bytes(rows, k) == (frags * blocks * 2048, frags * -(-blocks // 4) * 64)
    codes, scales = oracle.places(16 * frags, 128 * blocks)
    assert torch.equal(codes.flatten().sort().values, torch.arange(frags * blocks * 2048))
    assert scales.flatten().unique().numel() == scales.numel() and int(scales.max()) < frags * -(-blocks // 4) * 64
    assert torch.equal(oracle.order(96, True).sort().values, torch.arange(96))
    assert oracle.order(96, True)[[0, 15, 16, 48, 63, 64]].tolist() == [0, 15, 32, 16, 31, 48]


def test_sizes_of_no_rows():
    for rows, k in ((0, 64), (-1, 64), (1 << 24, 64), (4, 0), (4, 4), (4, 12), (4, (1 << 24) + 8), (4, -8)):
        assert fp8_bytes(rows, k) == (0, 0)


def test_structs_are_the_headers():
    text = (Path(__file__).resolve().parents[1] / "include" / "plm_amd.h").read_text()

    def fields(name):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        words = re.sub(r"[*,;]", " ", body).split()
        return tuple(w for w in words if w not in ("const", "void", "int64_t", "float", "double"))

    assert fields("plm_fp8_rows_call") == _lib.FP8_ROWS_FIELDS
    assert fields("plm_fp8_weight_call") == _lib.FP8_WEIGHT_FIELDS
    assert fields("plm_fp8_linear_call") == _lib.FP8_LINEAR_FIELDS
    for name, packed in (("plm_fp8_rows_call", _lib.pack_fp8_rows), ("plm_fp8_weight_call", _lib.pack_fp8_weight),
                         ("plm_fp8_linear_call", _lib.pack_fp8_linear)):
        assert len(packed(*[1] * len(fields(name)))) == 8 * len(fields(name))


def test_c_entries_refuse_before_a_launch():
    lib, f = _lib.lib(), 1 << 20   # never dereferenced

    def caller(entry, pack, call):
        def run(**more):
            assert set(more) <= set(call)
            return entry(pack(*{**call, **more}.values()), None)

        assert entry(None, None) == -1
        return run

    rows = caller(lib.plm_fp8_rows, _lib.pack_fp8_rows,
                  dict(dtype=0, rows=3, k=64, x=f, x_row=64, norm=1, residual=f, residual_row=64, sum=f, weight=f, eps=1e-6, y=0,
                       codes=f, scales=f))
    for bad in (dict(dtype=2), dict(rows=0), dict(rows=1 << 24), dict(k=60), dict(k=0), dict(x=0), dict(x_row=-8), dict(sum=0),
                dict(residual=0), dict(codes=0), dict(scales=0), dict(norm=0), dict(norm=0, residual=0, sum=0),
                dict(norm=0, residual=0, sum=0, weight=0, y=f), dict(eps=0.0), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf)):
        assert rows(**bad) == -1, bad
    for bad in (dict(x=f + 2), dict(residual=f + 8), dict(sum=f + 4), dict(weight=f + 2), dict(y=f + 8), dict(codes=f + 8),
                dict(scales=f + 4), dict(x_row=68), dict(residual_row=4)):
        assert rows(**bad) == -2, bad

    weight = caller(lib.plm_fp8_weight, _lib.pack_fp8_weight,
                    dict(dtype=0, n=64, k=64, w=f, ld=64, blocks=0, gate_up=0, codes=f, scales=f))
    for bad in (dict(dtype=3), dict(n=0), dict(k=12), dict(w=0), dict(ld=56), dict(gate_up=1, n=48), dict(codes=0), dict(scales=0)):
        assert weight(**bad) == -1, bad
    for bad in (dict(w=f + 8), dict(w=f + 4, blocks=f), dict(ld=68), dict(codes=f + 2), dict(scales=f + 8)):
        assert weight(**bad) == -2, bad

    def product(call, stream):
        return lib.plm_fp8_linear(call, f, 1 << 40, stream)

    assert lib.plm_fp8_linear_workspace_bytes(None) == 0
    linear = caller(product, _lib.pack_fp8_linear,
                    dict(m=3, n=64, k=64, x_type=0, x=f, x_scales=f, x_row=0, w=f, w_scales=f, y=f, ldy=64, out=0, act=0))
    for bad in (dict(m=0), dict(m=(1 << 21) + 1), dict(n=0), dict(k=4), dict(x=0), dict(x_scales=0), dict(w=0), dict(w_scales=0),
                dict(y=0), dict(ldy=63), dict(out=3), dict(out=-1), dict(act=1, n=48), dict(act=1, ldy=31), dict(x_type=3),
                dict(x_type=-1), dict(x_type=2, x_row=-8), dict(n=(1 << 21) + 1, ldy=1 << 22)):
        assert linear(**bad) == -1, bad
    for bad in (dict(x=f + 8), dict(x_scales=f + 4), dict(w=f + 2), dict(w_scales=f + 8), dict(y=f + 1), dict(y=f + 2, out=2),
                dict(x_type=1, x_row=4), dict(x_type=1, x=f + 8)):
        assert linear(**bad) == -2, bad

    # Few columns over a long K: K is cut, and the partial sums need a workspace.
    call = _lib.pack_fp8_linear(64, 2048, 8192, 0, f, f, 0, f, f, f, 2048, 0, 0)
    need = lib.plm_fp8_linear_workspace_bytes(call)
    assert need > 0 and need % 1024 == 0
    assert lib.plm_fp8_linear(call, None, 0, None) == -4 and lib.plm_fp8_linear(call, f, need - 1, None) == -4
    assert lib.plm_fp8_linear(call, f + 8, need, None) == -2
    rows = _lib.pack_fp8_linear(64, 2048, 8192, 1, f, 0, 8192, f, f, f, 2048, 0, 0)   # rounded first, into the workspace
    assert lib.plm_fp8_linear_workspace_bytes(rows) == need + sum(fp8_bytes(64, 8192))
    assert lib.plm_fp8_linear(rows, f, need, None) == -4
    assert lib.plm_fp8_linear_workspace_bytes(_lib.pack_fp8_linear(64, 2048, 8196, 0, f, f, 0, f, f, f, 2048, 0, 0)) == 0

    for bad in ((0, f, 3, 64, 0, 0, f), (f, 0, 3, 64, 0, 0, f), (f, f, 0, 64, 0, 0, f), (f, f, 3, 60, 0, 0, f), (f, f, 48, 64, 1, 0, f),
                (f, f, 3, 64, 0, 3, f), (f, f, 3, 64, 0, 0, 0)):
        assert lib.plm_fp8_values(*bad, None) == -1, bad
    assert lib.plm_fp8_values(f + 8, f, 3, 64, 0, 0, f, None) == -2


def test_oracle_pieces():
    x = torch.zeros(2, 200, dtype=BF16)
    x[0, :3] = torch.tensor([448.0, 1.0625, 17.0])     # 1.0625 lies between 1 and 1.125, ties to even
    x[0, 130] = 449.0                                   # bf16 keeps 448; a block of its own
    x[1, 199] = float("inf")
    got = oracle.rounded(x)
    assert got[0, :3].tolist() == [448.0, 1.0, 16.0] and float(got[0, 130]) == 448.0
    assert got[1].isnan().nonzero().tolist() == [[199]]
    y, t = oracle.norm(torch.tensor([[3.0, 4.0]], dtype=BF16), torch.tensor([2.0, 1.0], dtype=BF16), 0.0,
                       torch.tensor([[0.0, 0.0]], dtype=BF16))
    assert torch.allclose(y, torch.tensor([[6.0, 4.0]], dtype=torch.float64) / math.sqrt(12.5)) and t.dtype is BF16
    w = torch.ones(32, 8, dtype=BF16)
    w[16:] = 512
    values, scales = oracle.weight(w, gate_up=True)
    assert torch.equal(values, w.double()) and scales.flatten().tolist() == [2.0 ** -8, 2.0]


def test_sizes_have_a_largest():
    """2^25 fragments: more threads than a launch has would be needed for more."""
    most = 1 << 25
    assert fp8_bytes(16 * 2, 128 * (1 << 17)) == (2048 << 18, 64 << 16)
    assert fp8_bytes((1 << 24) - 1, 128 * 32)[0] == most * 2048
    assert fp8_bytes((1 << 24) - 1, 128 * 32 + 8) == (0, 0)
    assert fp8_bytes(16 * (most >> 17) + 1, 128 << 17) == (0, 0)


def test_overlap():
    """Against a map of the bytes."""
    for rows in (1, 2, 3):
        for a_row in (0, 8, 12):
            for b_row in (8, 12):
                for a_width in (2, 4, 8):
                    for b_width in (2, 6):
                        for b in range(0, 60):
                            def held(at, row, width):
                                return {at + r * row + i for r in range(rows) for i in range(width)}
                            meet = bool(held(20, a_row, a_width) & held(b, b_row, b_width))
                            got = fp8._overlap(20, a_row, a_width, b, b_row, b_width, rows)
                            assert got or not meet
                            if a_row == b_row and a_row >= max(a_width, b_width) and abs(b - 20) < a_row:
                                assert got == meet   # columns of one matrix
