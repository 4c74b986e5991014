"""The modulation of a gated half: frozen, and never silently without a gradient that was asked for."""

import pytest
import torch

from ksanadit_b200 import _lib
from ksanadit_b200.gated_block import B200GatedFeedForward, gated_stack
from ksanadit_b200.w4 import B200W4Linear


def test_an_embedding_that_is_trained_is_refused():
    m = B200GatedFeedForward(64, 40, group=64)
    temb = torch.zeros(1, 64, dtype=torch.bfloat16, requires_grad=True)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: m.vectors(temb), lambda: m(x, temb), lambda: gated_stack([m], x, temb)):
        with pytest.raises(_lib.KsanaB200Error, match="no backward pass"):
            call()


@pytest.mark.gpu
def test_detached_or_another_linear():
    m = B200GatedFeedForward(64, 40, group=64, device="cuda")
    lin = torch.nn.Linear(64, 192, device="cuda")
    m.modulation = B200W4Linear.from_float(lin, 64)
    temb = torch.randn(2, 64, device="cuda").bfloat16().requires_grad_(True)
    with pytest.raises(_lib.KsanaB200Error, match="no backward pass"):
        m.vectors(temb)
    detached = m.vectors(temb.detach())
    with torch.no_grad():
        plain = m.vectors(temb)
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(detached, plain))
    m.modulation = lin.bfloat16()  # one that has a backward pass trains
    shift, scale, gate = m.vectors(temb)
    assert [v.shape for v in (shift, scale, gate)] == [(2, 1, 64)] * 3 and gate.requires_grad
    assert bool(torch.autograd.grad(gate.float().sum(), temb)[0].isfinite().all())
