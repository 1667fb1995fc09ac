"""The 8-bit calls where they could go wrong without a word: derivatives that they would drop, values at the ends of fp32's
range, sums that lose their small terms, results that lie on what is read."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

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
