"""CPU checks of what the 8-bit calls refuse because they have no derivative and nothing a tracer could record."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from plm_amd import _lib, fp8

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _weight():
    """A weight as far as a refused call looks at it."""
    w = fp8.Weight.__new__(fp8.Weight)
    w.__dict__.update(rows=32, k=64, _index=0, codes_at=0, scales_at=0)
    return w


@pytest.mark.parametrize("call", [fp8.quantize, fp8.Weight.quantize, lambda t: fp8.rms_norm(t, None),
                                  lambda t: fp8.linear(t, _weight())])
def test_tangents_are_refused(call):
    x = torch.zeros(3, 64, dtype=BF16)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for t in (dual, dual[:, :64], dual[1:]):
            with pytest.raises(RuntimeError, match="tangent"):
                call(t)
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):   # which leaves forward mode as it is
                call(t)
        with pytest.raises(RuntimeError, match="GPU|cuda"):   # no tangent: all in order, but on the CPU
            call(x)
    with pytest.raises(RuntimeError, match="tangent"):
        torch.func.jvp(call, (x,), (x,))
    with pytest.raises(RuntimeError, match="gradient"):
        torch.func.vjp(call, x)


def test_codes_with_a_gradient_are_refused():
    lib = _lib.lib()
    codes = torch.zeros(int(lib.plm_fp8_codes_bytes(32, 64)), dtype=torch.uint8).view(E4M3).requires_grad_()
    scales = torch.zeros(int(lib.plm_fp8_scales_bytes(32, 64)), dtype=torch.uint8)
    for make in (fp8.Rows, fp8.Weight):
        with pytest.raises(RuntimeError, match="gradient"):
            make(codes, scales, 32, 64)
        with pytest.raises(RuntimeError, match="one GPU"):
            make(codes.detach(), scales, 32, 64)


def test_tracers_are_refused():
    """Before the library is reached: a trace would hold an allocation in the place of a result."""
    called = []

    def entry(*args):
        called.append(args)
        return 0

    def traced(x):
        fp8._run(entry, 0)
        return x

    with pytest.raises(RuntimeError, match="tracer"):
        torch.jit.trace(traced, torch.zeros(3))
    assert not called


def test_tensors_without_memory_are_refused():
    from torch._subclasses import FakeTensorMode

    mode = FakeTensorMode()
    with mode:
        x, codes, scales = (torch.empty(3, 64, device="cuda", dtype=dtype) for dtype in (BF16, E4M3, torch.float32))
    for call in (fp8.quantize, fp8.Weight.quantize, lambda t: fp8.rms_norm(t, None), lambda t: fp8.linear(t, _weight()),
                 lambda t: fp8.Weight.from_blocks(codes, scales[:1, :1])):
        with pytest.raises(RuntimeError, match="no memory"):
            call(x)
