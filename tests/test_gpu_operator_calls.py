"""Calls of the training-step operators (csrc/group_norm.hip, csrc/lookup.hip, csrc/orthogonalize.hip and their Python entries) that the
tests by operator leave out: other derivatives, sizes past 32 bits, special values, hooks, caches, optimiser options and states."""
import copy

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from openpcdet_amd import backbones, optim, scatter, vfe
from openpcdet_amd.spconv import pytorch as spconv
from openpcdet_amd.spconv.pytorch import norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# ---- sizes past 32 bits ----------------------------------------------------------------------------------------------------
def test_lookup_refuses_counts_past_32_bits(cuda_device):
    """2^32 + 5 is 5 in 32 bits.  The tensors are expanded from one element: refused before anything of that size is made"""
    big = 2 ** 32 + 5
    one, zero = torch.zeros(1, 1, dtype=torch.bfloat16, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for call in (lambda: scatter.lookup_rows(one.expand(big, 1), zero), lambda: scatter.lookup_rows(one, zero.expand(big)),
                 lambda: scatter.lookup_rows(one.expand(2, big), zero), lambda: scatter.sort_index(zero, big),
                 lambda: scatter.sort_index(zero.expand(big), 4)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


def test_group_norm_refuses_counts_past_32_bits(cuda_device):
    big = 2 ** 32 + 5
    one, off = torch.zeros(1, 1, dtype=torch.bfloat16, device=cuda_device), torch.zeros(2, dtype=torch.int32, device=cuda_device)
    for call in (lambda: norm.group_norm_act(one.expand(big, 1), 1, offsets=off), lambda: norm.group_norm_act(one.expand(big, 1), 1),
                 lambda: norm.group_norm_act(one.expand(1, big), 1), lambda: norm.group_norm_act(one.unsqueeze(0).expand(1, big, 1), 1),
                 lambda: norm.group_norm_act(one, 1, offsets=off[:1].expand(big))):
        with pytest.raises(ValueError, match="32 bits"):
            call()


# ---- forward-mode derivatives ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(cuda_device, grad):
    """no forward-mode derivative is defined: refused, not taken for zero"""
    x, w, r = (torch.randn(s, device=cuda_device) for s in ((6, 8), (8,), (6, 8)))
    index = torch.tensor([0, 5, 2], device=cuda_device)
    plain = norm.group_norm_act(x, 2, w, act="relu", residual=r), scatter.lookup_rows(x, index)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: norm.group_norm_act(dual(x), 2, w), lambda: norm.group_norm_act(x, 2, dual(w)),
                     lambda: norm.group_norm_act(x, 2, w, dual(w)), lambda: norm.group_norm_act(x, 2, residual=dual(r)),
                     lambda: scatter.lookup_rows(dual(x), index)):
            with pytest.raises(RuntimeError):
                call()
        assert torch.equal(norm.group_norm_act(x, 2, w, act="relu", residual=r), plain[0])      # nothing dual: as ever
        assert torch.equal(scatter.lookup_rows(x, index), plain[1])
    with torch.set_grad_enabled(grad):
        for f in (lambda t: norm.group_norm_act(t, 2, w), lambda t: scatter.lookup_rows(t, index)):
            with pytest.raises(RuntimeError):
                torch.func.jvp(f, (x,), (torch.ones_like(x),))
            with pytest.raises(RuntimeError):
                torch.func.vmap(f)(x.expand(3, 6, 8))


# ---- the largest sizes of the norm -----------------------------------------------------------------------------------------
def test_norm_of_more_than_2_30_samples(cuda_device):
    """the rows are those of the last sample: the search for it adds up sample numbers past 2^31"""
    samples, n = 2 ** 30 + 1000, 700
    off = torch.zeros(samples + 1, dtype=torch.int32, device=cuda_device)
    off[-1] = n
    x = torch.randn(n, 1, device=cuda_device)
    y = norm.group_norm_act(x, 1, offsets=off)
    want = norm.group_norm_act(x, 1, offsets=torch.tensor([0, n], dtype=torch.int32, device=cuda_device))
    assert float((y - want).abs().max()) <= 8 * U * float(want.abs().max() + 1)
