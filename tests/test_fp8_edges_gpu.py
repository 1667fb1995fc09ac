"""The 8-bit calls where they could go wrong without a word: derivatives that they would drop, values at the ends of fp32's
range, sums that lose their small terms, results that lie on what is read."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from oracle import fp8_oracle as oracle
from plm_amd import fp8

pytestmark = pytest.mark.gpu

BF16, FP16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def test_derivatives_of_every_argument_are_refused(device):
    x, ones = torch.ones(3, 64, dtype=BF16, device=device), torch.ones(64, dtype=BF16, device=device)
    w = fp8.Weight.quantize(torch.ones(32, 64, dtype=BF16, device=device))
    codes, scales = torch.ones(32, 64, device=device).to(E4M3), torch.ones(1, 1, device=device)
    out = torch.empty(3, 32, dtype=BF16, device=device)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: fp8.rms_norm(dual(x), ones), lambda: fp8.rms_norm(x, dual(ones)),
                     lambda: fp8.rms_norm(x, ones, residual=dual(x)), lambda: fp8.linear(dual(x), w),
                     lambda: fp8.linear(x, w, out=dual(out)), lambda: fp8.Weight.from_blocks(codes, dual(scales))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        assert torch.equal(fp8.linear(x, w), torch.full_like(out, 64))   # no tangent, no refusal
        assert torch.equal(fp8.rms_norm(x, ones, 2.0 ** -100), x)
    for call in (lambda: fp8.linear(x, w, out=out.clone().requires_grad_()),
                 lambda: fp8.Weight.from_blocks(codes, scales.clone().requires_grad_()),
                 lambda: fp8.Weight.from_blocks(codes.clone().requires_grad_(), scales)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()


def test_a_weight_without_memory_is_refused(device):
    """It is not a norm without weights, whose pointer is null."""
    from torch._subclasses import FakeTensorMode

    x = torch.ones(3, 64, dtype=BF16, device=device)
    with FakeTensorMode():
        weight = torch.empty(64, dtype=BF16, device="cuda")
    for dtype in (BF16, E4M3):
        with pytest.raises(RuntimeError, match="no memory"):
            fp8.rms_norm(x, weight, dtype=dtype)


def _same(got, want):
    got, want = got.cpu().double(), want.to(got.dtype).double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


# A row to a workgroup, sixteen to a fragment's workgroup.
@pytest.mark.parametrize("m,k", [(5, 1416), (130, 512), (4096, 264)])
@pytest.mark.parametrize("size", [2.0 ** 3, 2.0 ** 10, 2.0 ** 60, 2.0 ** 120])
def test_norm_of_rows_wider_than_fp32(device, m, k, size):
    """A value so far below its row's size that their quotient is subnormal in fp32, or zero, until the weight multiplies it.
    The tolerance in 16 bits is that of any norm: half a step and 2^-21 of the value, half of the least subnormal."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(m, k, generator=g)
    x[:, 1::2] *= 2.0 ** -86
    x[:, 2::7] *= 2.0 ** -120
    x[:, 5::11] = 0
    x[:, :128] = 0
    x[:, 0] = 2.0 ** 60
    x[m // 2] *= 2.0 ** -20
    x = x.to(BF16)
    w = (size * (1 + 0.3 * torch.randn(k, generator=g))).to(BF16)
    for r in (None, x.flip(0)):
        want, total = oracle.norm(x, w, 1e-5, r)
        on = None if r is None else r.to(device)
        eight, sixteen = (fp8.rms_norm(x.to(device), w.to(device), 1e-5, residual=on, dtype=kind) for kind in (E4M3, None))
        if r is not None:
            assert torch.equal(eight[1].cpu(), total) and torch.equal(sixteen[1].cpu(), total)
            eight, sixteen = eight[0], sixteen[0]
        _same(eight.values(), oracle.rounded(want))
        off = (sixteen.cpu().double() - want).abs()
        assert (off <= want.abs() * (2.0 ** -8 + 2.0 ** -21) + 2.0 ** -134).all()


# In place, after a launch that rounds, K in ranges, tiles.
RANGES = [(3, 40, 264), (20, 40, 264), (42, 512, 10240), (700, 2056, 1032)]


@pytest.mark.parametrize("m,n,k", RANGES)
@pytest.mark.parametrize("out", [F32, BF16])
def test_codes_of_two_to_the_128th(device, m, n, k, out):
    """bf16's largest values round up to 2^128, which fp32 does not hold but a product with a small weight does. Each row of the
    result is the sum of one such product and one of ordinary size that it swallows, so that the result is the product."""
    x = torch.zeros(m, k, dtype=BF16)
    x[:, k - 3] = torch.finfo(BF16).max
    x[1::2, k - 3] = torch.finfo(BF16).min
    x[:, 2] = 1
    w = torch.zeros(n, k, dtype=BF16)
    w[:, k - 3] = 2.0 ** -(10 + torch.arange(n) % 5)
    w[3::4, k - 3] = 0
    w[:, 2] = 1
    want = x[:, k - 3].sign().double()[:, None] * 2.0 ** 128 * w[:, k - 3].double()
    want = torch.where(want == 0, 1.0, want)
    got = fp8.linear(x.to(device), fp8.Weight.quantize(w.to(device)), out_dtype=out)
    assert torch.equal(got.cpu().double(), want)
    # The same of a weight's, and of both, which is past the range of any type.
    got = fp8.linear(w.to(device), fp8.Weight.quantize(x.to(device)), out_dtype=out)
    assert torch.equal(got.cpu().double(), want.T)
    got = fp8.linear(x.to(device), fp8.Weight.quantize(x[:2].to(device)), out_dtype=out)
    assert torch.equal(got.cpu().double(), x[:, k - 3:k - 2].sign().double() * x[:2, k - 3].sign().double() * float("inf"))


@pytest.mark.parametrize("m", [3, 20, 600])
def test_gates_past_fp32(device, m):
    """The activation in fp32 with such a code in the up row, and one in the gate row."""
    half, k = 2048, 264
    w = torch.zeros(2 * half, k, dtype=BF16)
    w[:half, 0], w[half:, 1] = 1, torch.finfo(BF16).max
    w[half // 2:half, 0], w[half + half // 2:, 1] = torch.finfo(BF16).max, 1
    x = torch.zeros(m, k, dtype=BF16)
    x[:, 0], x[:, 1] = 2.0 ** -30, 2.0 ** -40
    x[:, 130] = 1
    got = fp8.gate_up_silu(x.to(device), fp8.Weight.quantize(w.to(device), gate_up=True), out_dtype=F32).cpu().double()
    g = torch.tensor([2.0 ** -30, 2.0 ** 98], dtype=torch.float64).repeat_interleave(half // 2)
    u = torch.tensor([2.0 ** 88, 2.0 ** -40], dtype=torch.float64).repeat_interleave(half // 2)
    want = (g * torch.sigmoid(g) * u).expand(m, half)
    assert ((got - want).abs() <= want * (2.0 ** -20 + 2.0 ** -24)).all()


@pytest.mark.parametrize("m", [1, 70, 600])
@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("up", [2.0 ** 20, -2.0 ** 60, 2.0 ** 100])
def test_low_gates_beside_large_values(device, m, out, up):
    """Gates whose activation is below fp32's normal range while its product with the up value is not. The exponential e^(-|g| / 2)
    is normal down to -174."""
    half, k = 2048, 128
    gates = torch.cat([torch.linspace(-174, -80, half // 2), torch.linspace(-104, -87, half // 2)])
    w = torch.zeros(2 * half, k, dtype=BF16)
    w[:half, 0], w[half:, 2] = gates.to(BF16), up
    x = torch.zeros(m, k, dtype=BF16)
    x[:, 0] = x[:, 2] = 1
    weight = fp8.Weight.quantize(w.to(device), gate_up=True)
    gate = oracle.weight(w, True)[0][:half, 0].double().clamp(min=-174)
    got = fp8.gate_up_silu(x.to(device), weight, out_dtype=out).cpu().double()
    within = oracle.weight(w, True)[0][:half, 0] >= -174
    want = gate * torch.sigmoid(gate) * up
    off = want.abs() * 2.0 ** -20 + 2.0 ** -149
    info = torch.finfo(out)
    bad = (got - want).abs() > off + (want.abs() + off) * info.eps / 2 + info.smallest_normal * info.eps / 2
    assert not (bad & within).any()


# Narrow in place, its ranges of K, an LM head, tiles of either size, all with a long K.
LONG = [(1, 2048, 2048), (16, 50257, 2048), (42, 512, 10240), (64, 2048, 8192), (110, 2048, 2048), (700, 2056, 2056), (513, 640, 8192)]


@pytest.mark.parametrize("m,n,k", LONG)
def test_fp32_results_keep_small_terms(device, m, n, k):
    """In every eight of K two large products cancel and the others are so small that an instruction which cuts an eight's
    products at 2^-14 of the largest loses them. The sums are whole numbers of 2^-2 below 2^22, whatever their order, so
    fp32 holds them exactly."""
    g = torch.Generator().manual_seed(m)
    x = torch.randint(-2, 3, (m, k), generator=g).float() / 2
    w = torch.randint(-2, 3, (n, k), generator=g).float() / 2
    x[:, 0::8], x[:, 5::8] = 256, 256
    w[:, 0::8], w[:, 5::8] = 256, -256
    weight = fp8.Weight.quantize(w.to(BF16).to(device))
    want = (x.to(device).double() @ w.to(device).double().T.contiguous()).float()
    for rows in (x.to(BF16).to(device), fp8.quantize(x.to(BF16).to(device))):
        assert torch.equal(fp8.linear(rows, weight, out_dtype=F32), want)
    # The 8-bit instruction would not: its 16-bit results have lost what they were made for.
    if m <= 64:
        assert not torch.equal(fp8.linear(x.to(BF16).to(device), weight), want.to(BF16))


@pytest.mark.parametrize("m,n,k", [(1, 2048, 2048), (42, 512, 10240), (56, 6144, 2048), (517, 2048, 1416), (1100, 8200, 640)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_the_cut_has_no_sign(device, m, n, k, dtype):
    """Products are cut toward zero, whatever their sign: negative rows have the negative results, bit for bit."""
    g = torch.Generator(device=device).manual_seed(k)
    x = torch.randn(m, k, generator=g, device=device) * (1 + 15 * (torch.rand(k, generator=g, device=device) < 0.01))
    weight = fp8.Weight.quantize((0.05 * torch.randn(n, k, generator=g, device=device)).to(dtype))
    x = x.to(dtype)
    assert torch.equal(fp8.linear(-x, weight), -fp8.linear(x, weight))


def test_out_on_an_operand_is_refused(device):
    """A result may not lie on 8-bit rows or weights either, on their codes or their scales; beside them it may."""
    ones = torch.ones(64, 256, dtype=BF16, device=device)
    w = fp8.Weight.quantize(ones)
    x = fp8.quantize(ones)
    size, after = x.codes.numel(), x.codes.numel() + 64 * 64 * 2
    store = torch.zeros(1 << 16, dtype=torch.uint8, device=device)
    store[:size], store[after:after + x.scales.numel()] = x.codes.view(torch.uint8), x.scales
    codes, scales = store[:size].view(E4M3), store[after:after + x.scales.numel()]

    def out(begin):
        return store[begin:begin + 64 * 64 * 2].view(BF16).view(64, 64)

    for rows, weight in ((fp8.Rows(codes, scales, 64, 256), w), (x, fp8.Weight(codes, scales, 64, 256))):
        for begin in (0, size - 16, size + 16, after, after + x.scales.numel() - 16):
            with pytest.raises(ValueError, match="overlaps an operand"):
                fp8.linear(rows, weight, out=out(begin))
        for begin in (size, after + x.scales.numel()):
            assert bool((fp8.linear(rows, weight, out=out(begin)) == 256).all())
    with pytest.raises(ValueError, match="overlaps an operand"):
        fp8.linear(ones, fp8.Weight(codes, scales, 64, 256), out=out(0))


@pytest.mark.parametrize("a,b,unit", [(256, 256, 3), (448, 448, 3), (240, 256, 2), (240, 240, 1), (1, 1, -13), (2.0 ** -6, 256, -11),
                                      (2.0 ** -9, 256, -11), (7 * 2.0 ** -9, 448, -11)])
def test_where_an_eight_is_cut(device, a, b, unit):
    """At 2^-13 of two to the largest sum of two factors' exponents, a subnormal code's being -6: what is below goes, toward
    zero, in its own eight alone, and fp32 results keep it."""
    def one(small, out, at=2):
        x, w = torch.zeros(2, 256, dtype=BF16), torch.zeros(16, 256, dtype=BF16)
        x[:, 126::128], w[:, 125::128] = 448, 448          # scales of 1, and products of zero in an eight of their own
        x[0, 0], x[0, 1], w[:, 0], w[:, 1] = a, a, b, -b
        half = max(-9, min(8, unit))          # factors that are codes: the other one normal
        x[0, at], w[:, at] = 2.0 ** half, small * 2.0 ** -half
        x[1] = -x[0]
        w8 = fp8.Weight.quantize(w.to(device))
        assert torch.equal(w8.values().cpu(), w.float())
        got = fp8.linear(x.to(device), w8, out_dtype=out).cpu()
        assert torch.equal(got[0], -got[1])
        return float(got[0, 0])

    for small, kept in ((2.0 ** unit, 2.0 ** unit), (1.875 * 2.0 ** unit, 2.0 ** unit), (2.0 ** (unit - 1), 0.0), (1.5 * 2.0 ** (unit - 1), 0.0)):
        assert one(small, BF16) == kept
        assert one(small, BF16, at=8) == small
        assert one(small, F32) == small
