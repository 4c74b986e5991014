"""CPU tests of what ops.sandwich_norm and its C entries refuse."""

import ctypes

import pytest
import torch

from ksanadit_b200 import _lib, native, ops


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,kw", [
    ((_t(2, 12),), {}), ((_t(2, 8200),), {}), ((_t(2, 0),), {}), ((_t(2, 16), _t(3, 16)), {}), ((_t(2, 16), _t(2, 16, dtype=torch.float16)), {}),
    ((_t(2, 16),), dict(gate=_t(16))), ((_t(2, 16),), dict(post_weight=torch.ones(16))), ((_t(2, 16),), dict(pre=False)), ((_t(2, 16), _t(2, 16)), dict(pre=False, scale=_t(16))),
    ((_t(2, 16), _t(2, 16)), dict(kind="batch")), ((_t(2, 16), _t(2, 16)), dict(gate=_t(3, 16))), ((_t(2, 16), _t(2, 16)), dict(gate=_t(8))),
    ((_t(2, 16), _t(2, 16)), dict(gate=_t(16, dtype=torch.float16))), ((_t(2, 3, 16), _t(2, 3, 16)), dict(gate=_t(3, 16))), ((_t(2, 3, 16), _t(2, 3, 16)), dict(gate=_t(1, 3, 16))),
    ((_t(4, 3, 16), _t(4, 3, 16)), dict(gate=_t(4, 1, 16), scale=_t(4, 3, 16))), ((_t(2, 16), _t(2, 16)), dict(pre_weight=_t(16))), ((_t(2, 16), _t(2, 16)), dict(pre_weight=torch.ones(8))),
    ((_t(2, 16), _t(2, 16)), dict(pre_weight=torch.ones(32)[::2])), ((_t(2, 16), _t(2, 16)), dict(pre_weight=torch.ones(17)[1:])), ((_t(2, 16), _t(2, 16)), {})])
def test_refusals(args, kw):
    with pytest.raises(_lib.KsanaB200Error):  # the last one: everything fits, but on the CPU
        ops.sandwich_norm(*args, **kw)


def test_refused_types():
    with pytest.raises(TypeError):
        ops.sandwich_norm(torch.zeros(2, 16))


P = 0x1000  # never read


def _args(**kw):
    a = native.NormArgs(P, P, P, P, P, P, P, P, 6, 16, 2, 16, 16, 16, 16, 16, 0, 0, 1e-6, 1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()

    def forward(r=P, h=P, **kw):
        return lib.ksb_sandwich_norm(ctypes.byref(_args(**kw)), r, h, None)

    def backward(grads=(P, P, P, P, P, P, P, P, P, 16, 16), ws=P, **kw):
        return lib.ksb_sandwich_norm_backward(ctypes.byref(_args(**kw)), ctypes.byref(native.NormGrads(*grads)), ws, None)

    assert forward(M=0) == 0
    bad = (dict(dtype=2), dict(C=12), dict(C=0), dict(M=-1), dict(mod_rows=0), dict(mod_rows=4), dict(x=P + 2), dict(y=P + 4), dict(gate=P + 8), dict(ldx=8), dict(ldy=20),
           dict(gate_stride=4), dict(scale_stride=12), dict(shift_stride=2), dict(post_w=P + 4), dict(x=None))
    for kw in bad + (dict(y=None), dict(r=None), dict(y=None, gate=None, post_w=None, h=None), dict(h=None), dict(r=P + 4), dict(h=P + 2)):
        assert forward(**kw) == -1, kw
    for kw in bad + (dict(stats=None), dict(ws=None), dict(grads=(None, None) + (P,) * 7 + (16, 16)), dict(grads=(P,) * 9 + (8, 16)), dict(grads=(P,) * 9 + (16, 20)),
                     dict(grads=(P, P, P + 2) + (P,) * 6 + (16, 16)), dict(grads=(P, None) + (P,) * 7 + (16, 16)), dict(y=None, gate=None, post_w=None)):
        assert backward(**kw) == -1, kw
    assert forward(C=8200, ldx=8200, ldy=8200) == -3
    assert lib.ksb_sandwich_norm(None, P, P, None) == -1 and lib.ksb_sandwich_norm_workspace(0, 16, 1) == 0 and lib.ksb_sandwich_norm_workspace(6, 16, 4) == 0
    assert lib.ksb_sandwich_norm_workspace(6, 16, 2) > 0
