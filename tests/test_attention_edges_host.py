"""CPU checks of what the paged attention's calls refuse or hold to, at the ends of what they are given."""

from __future__ import annotations

import ctypes

import pytest
import torch

from plm_amd import _lib, attention
from test_attention_host import _call, _stub

LEAST, MOST = 2.0 ** -62, 2.0 ** 126


@pytest.mark.parametrize("scale, fine", [(LEAST, True), (MOST, True), (1e-9, True), (1e9, True), (LEAST * (1 - 2 ** -20), False),
                                         (MOST * (1 + 2 ** -20), False), (1e-30, False), (5e-324, False), (2.5e38, False)])
def test_scales_that_single_precision_cannot_hold(scale, fine):
    """A scale that fp32 turns into zero or infinity, by itself or times a page's, would make what is masked NaN."""
    f = 1 << 20
    handle = _lib.KvCache(f, f, f, f, 4, 2, 32, 64, _lib.PLM_CACHE_E4M3)
    call = _lib.pack_attend(0, ctypes.addressof(handle), 6, 2, 3, f, 64, 64, f, 0, f, 256, 64, 4, f, 0, 0, 0, 0, 0, 0, scale)
    lib = _lib.lib()
    # A wide table needs a workspace: what is right is refused for want of it, before any launch.
    assert lib.plm_attend(call, None, 0, None) == (-4 if fine else -1)
    assert (lib.plm_attend_workspace_bytes(call) > 0) == fine
    if not fine:
        c = _call()
        with pytest.raises(ValueError):
            attention.attend(_stub(), c["q"], c["table"], c["lengths"], scale=scale)


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale", "pages", "kv_heads", "page", "head_dim", "dtype", "device"])
def test_a_cache_stays_what_it_was_made_of(name):
    """The handle holds addresses and sizes: another tensor in their place would leave it with freed memory."""
    cache = _stub()
    if not hasattr(cache, name):
        setattr(cache, name, torch.zeros(1))
    held = getattr(cache, name)
    with pytest.raises(AttributeError):
        setattr(cache, name, held)
    with pytest.raises(AttributeError):
        delattr(cache, name)
    assert getattr(cache, name) is held


def test_gradients_are_refused():
    """There is no backward: an output without a graph would lose a gradient in silence."""
    for name in ("q", "k", "v"):
        c = _call()
        c[name].requires_grad_()
        with pytest.raises(RuntimeError, match="gradient"):
            attention.append_kv(_stub(), c["q"], c["k"], c["v"], c["table"], c["lengths"])
        if name == "q":
            with pytest.raises(RuntimeError, match="gradient"):
                attention.attend(_stub(), c["q"], c["table"], c["lengths"])
    with torch.no_grad():      # past the refusal: 5 rows of 2 sequences
        q = torch.zeros(5, 4, 64, dtype=torch.bfloat16, requires_grad=True)
        with pytest.raises(ValueError, match="row_starts"):
            attention.attend(_stub(), q, c["table"], c["lengths"])
