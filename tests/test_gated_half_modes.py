"""CPU tests: modes of torch that the operators of a gated half cannot follow are errors of the call, not results without a part."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from ksanadit_b200 import _lib, ops, w4


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def calls():
    """name -> (function of its tensors, the tensors that a derivative could be asked of)"""
    packed, scale, _ = w4.quantize_w4(torch.randn(16, 64), 64)
    return {
        "gated": (lambda *t: ops.gated_linear(*t), (_t(2, 16), _t(8, 16), _t(8, 16), _t(8), _t(8))),
        "norms": (lambda x, y, g, sc, sh, wp, wn: ops.sandwich_norm(x, y, gate=g, scale=sc, shift=sh, post_weight=wp, pre_weight=wn),
                  (_t(2, 16), _t(2, 16), _t(16), _t(16), _t(16), torch.ones(16), torch.ones(16))),
        "w4": (lambda x, s, b: ops.w4_linear(x, packed, s, None, b), (_t(2, 64), scale, _t(16))),
    }


@pytest.mark.parametrize("name", ["gated", "norms", "w4"])
def test_forward_mode_is_refused(name):
    f, tensors = calls()[name]
    for i, t in enumerate(tensors):
        with fwd.dual_level():
            dual = fwd.make_dual(t, torch.ones_like(t))
            with pytest.raises(_lib.KsanaB200Error, match="forward-mode"):
                f(*tensors[:i], dual, *tensors[i + 1:])


@pytest.mark.parametrize("name", ["gated", "norms", "w4"])
def test_recording_is_refused(name):
    """What records a call sees its output's allocation and no kernel that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, tensors = calls()[name]
    with pytest.raises(_lib.KsanaB200Error, match="torch.ops.ksana_b200"):
        torch.jit.trace(f, tensors, check_trace=False)
    with pytest.raises(_lib.KsanaB200Error, match="torch.ops.ksana_b200"):
        make_fx(f)(*tensors)
