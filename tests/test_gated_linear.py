"""CPU tests of what ops.gated_linear and its C entries refuse."""

import ctypes

import pytest
import torch

from ksanadit_b200 import _lib, native, ops


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,kw", [
    ((_t(2, 16), _t(8, 24), _t(8, 24)), {}), ((_t(2, 16), _t(8, 16), _t(16, 16)), {}), ((_t(2, 12), _t(8, 12), _t(8, 12)), {}), ((_t(2, 16), _t(12, 16), _t(12, 16)), {}),
    ((_t(2, 0), _t(8, 0), _t(8, 0)), {}), ((_t(2, 16), _t(8, 16, dtype=torch.float16), _t(8, 16)), {}), ((_t(2, 16), _t(8, 16), _t(8, 16)), dict(act="relu")),
    ((_t(2, 16), _t(8, 16), _t(8, 16), _t(16)), {}), ((_t(2, 16), _t(8, 16), _t(8, 16), torch.zeros(8)), {}), ((_t(2, 16), _t(8, 16), _t(8, 16), None, _t(9)[1:]), {}),
    ((_t(2, 16), _t(8, 16), _t(8, 16), _t(16)[::2]), {}), ((_t(2, 16), _t(16), _t(16)), {}), ((_t(2, 16), _t(8, 16), _t(8, 16)), {})])
def test_refusals(args, kw):
    with pytest.raises(_lib.KsanaB200Error):  # the last one: everything fits, but on the CPU
        ops.gated_linear(*args, **kw)


def test_refused_types():
    with pytest.raises(TypeError):
        ops.gated_linear(torch.zeros(2, 16), torch.zeros(8, 16), torch.zeros(8, 16))


P = 0x1000  # never read


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()

    def forward(x=P, ldx=16, wg=P, ldg=16, wu=P, ldu=16, bg=None, bu=None, dtype=0, M=4, F=8, K=16, act=0, h=P, saved=None):
        return lib.ksb_gated_linear(x, ldx, wg, ldg, wu, ldu, bg, bu, dtype, M, F, K, act, h, saved, None)

    assert forward(M=0) == 0
    for kw in (dict(x=None), dict(wg=None), dict(wu=None), dict(h=None), dict(x=P + 2), dict(wg=P + 8), dict(wu=P + 4), dict(bg=P + 2), dict(bu=P + 2), dict(h=P + 2), dict(ldx=8),
               dict(ldx=20), dict(ldg=8), dict(ldu=18), dict(dtype=2), dict(M=-1), dict(F=12), dict(K=20), dict(F=0), dict(K=0), dict(act=2), dict(saved=P + 2)):
        assert forward(**kw) == -1, kw

    def backward(ws=P, **kw):
        a = native.GatedGrads(P, P, P, P, P, P, P, P, P, P, 4, 8, 16, 16, 16, 16, 8, 0, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.ksb_gated_linear_backward(ctypes.byref(a), ws, None)

    for kw in (dict(x=None), dict(w_gate=None), dict(w_up=None), dict(saved=None), dict(saved=P + 2), dict(dh=None), dict(ws=None), dict(dx=P + 2), dict(dw_gate=P + 2), dict(dw_up=P + 8),
               dict(lddh=4), dict(ldx=12), dict(ldg=8), dict(ldu=17), dict(M=-1), dict(F=4), dict(K=4), dict(dtype=3), dict(act=-1)):
        assert backward(**kw) == -1, kw
    assert lib.ksb_gated_linear_backward(None, P, None) == -1
    assert lib.ksb_gated_linear_workspace(0, 8, 8) == 0 and lib.ksb_gated_linear_workspace(4, 12, 8) == 0 and lib.ksb_gated_linear_workspace(4, 8, 12) == 0
    assert lib.ksb_gated_linear_workspace(4, 8, 8) > 0
    # few tiles and a long sum: room for its parts besides dg, du and the bias sums
    assert lib.ksb_gated_linear_workspace(75600, 128, 256) > 4 * 75600 * 128 + 4 * 128 * 256 * 8
    assert lib.ksb_gated_linear_saved(4, 8) > 0 and lib.ksb_gated_linear_saved(0, 8) == 0 and lib.ksb_gated_linear_saved(4, 9) == 0


def test_registered_operators_have_shape_inference():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import ksanadit_b200.torch_ops  # noqa: F401
    t = torch.ops.ksana_b200
    with FakeTensorMode():
        x, w = torch.empty(2, 7, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(48, 64, dtype=torch.bfloat16, device="cuda")
        h = t.gated_linear(x, w, w)
        assert h.shape == (2, 7, 48) and h.dtype == torch.bfloat16
        r, h = t.sandwich_norm(x, x)
        assert r.shape == h.shape == x.shape and r.dtype == h.dtype == x.dtype
        o = t.w4_linear(x, torch.empty(3, 1, 512, dtype=torch.uint8, device="cuda"), torch.empty(3, 1, 16, dtype=torch.bfloat16, device="cuda"), None, None, 40)
        assert o.shape == (2, 7, 40) and o.dtype == torch.bfloat16
    with pytest.raises(Exception):
        t.gated_linear(_t(2, 16), _t(8, 16), _t(8, 16))


def test_module_refuses_what_it_does_not_have():
    from ksanadit_b200.gated_block import B200GatedFeedForward, gated_stack
    m = B200GatedFeedForward(128, 264, bias=True)
    assert set(dict(m.named_parameters())) == {"w_gate", "w_up", "b_gate", "b_up", "down.weight", "down.bias", "pre_norm", "post_norm", "modulation.weight",
                                               "modulation.weight_scale", "modulation.bias"}
    assert [n for n, p in m.named_parameters() if not p.requires_grad] == ["modulation.weight", "modulation.weight_scale", "modulation.bias"]
    x = _t(1, 2, 128)
    assert gated_stack([], x) is x
    with pytest.raises(_lib.KsanaB200Error):
        gated_stack([m], x, vectors=[])
    with pytest.raises(_lib.KsanaB200Error):
        B200GatedFeedForward(128, 264, act="relu")
    with pytest.raises(_lib.KsanaB200Error):
        B200GatedFeedForward(100, 264)  # its modulation's groups
    with pytest.raises(_lib.KsanaB200Error):
        B200GatedFeedForward(128, 264, modulation=False)(x, x[:, 0])
