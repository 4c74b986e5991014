"""Modes of torch that the operators of a gated half cannot follow are errors of the call, and what they can follow is not refused."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from ksanadit_b200 import _lib, ops, w4

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"], autouse=True)
def way(request, monkeypatch):
    """Every test both ways: plain calls through the extension, and all calls through Python."""
    from ksanadit_b200 import native
    if request.param == "python":
        monkeypatch.setattr(native, "host_ops", lambda: False)
    else:
        assert native.host_ops()
    return request.param


def _n(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def calls():
    """name -> (function of its tensors, the tensors that a derivative could be asked of)"""
    packed, scale, _ = w4.quantize_w4(_n(48, 64, dtype=torch.float32), 64)
    return {
        "gated": (lambda *t: ops.gated_linear(*t), (_n(20, 16), _n(24, 16, seed=1), _n(24, 16, seed=2), _n(24), _n(24))),
        "norms": (lambda x, y, g, sc, sh, wp, wn: ops.sandwich_norm(x, y, gate=g, scale=sc, shift=sh, post_weight=wp, pre_weight=wn),
                  (_n(20, 16), _n(20, 16), _n(16), _n(16), _n(16), _n(16, dtype=torch.float32), _n(16, dtype=torch.float32))),
        "w4": (lambda x, s, b: ops.w4_linear(x, packed, s, None, b), (_n(2, 64), scale, _n(48))),
    }


@pytest.mark.parametrize("name", ["gated", "norms", "w4"])
def test_forward_mode_is_refused(name):
    f, tensors = calls()[name]
    for i, t in enumerate(tensors):
        with fwd.dual_level():
            for needs in (False, True) if name != "w4" else (False,):
                dual = fwd.make_dual(t.detach().clone().requires_grad_(needs), torch.ones_like(t))
                with pytest.raises(_lib.KsanaB200Error, match="forward-mode"):
                    f(*tensors[:i], dual, *tensors[i + 1:])
            f(*tensors)  # without a dual tensor a level changes nothing


@pytest.mark.parametrize("name", ["gated", "norms"])
def test_forward_over_reverse_is_refused(name):
    f, tensors = calls()[name]
    leaves = [t.detach().clone().requires_grad_(True) for t in tensors]
    out = f(*leaves)
    out = out if name == "gated" else out[0]
    with fwd.dual_level():
        d = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, leaves[:2], d)


def test_registered_operators_refuse_forward_mode():
    import ksanadit_b200.torch_ops  # noqa: F401
    x, w = _n(20, 16), _n(24, 16)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: torch.ops.ksana_b200.gated_linear(dual, w, w), lambda: torch.ops.ksana_b200.sandwich_norm(dual, x)):
            with pytest.raises(RuntimeError):
                call()


@pytest.mark.parametrize("name", ["gated", "norms", "w4"])
def test_recording_is_refused(name):
    """What records a call sees its output's allocation and no kernel that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, tensors = calls()[name]
    with torch.no_grad():
        with pytest.raises(_lib.KsanaB200Error, match="torch.ops.ksana_b200"):
            torch.jit.trace(f, tensors, check_trace=False)
        with pytest.raises(_lib.KsanaB200Error, match="torch.ops.ksana_b200"):
            make_fx(f)(*tensors)
        f(*tensors)


def test_registered_operators_are_recorded():
    from torch.fx.experimental.proxy_tensor import make_fx

    import ksanadit_b200.torch_ops  # noqa: F401
    t = torch.ops.ksana_b200
    packed, scale, _ = w4.quantize_w4(_n(48, 64, dtype=torch.float32), 64)
    w = _n(64, 16, seed=1)

    def f(x, y):
        r, h = t.sandwich_norm(x, y, x[0], None, None, None, None, 0.5, "rms", 1e-6)
        return r, t.w4_linear(t.gated_linear(h, w, w, None, None, "silu"), packed, scale, None, None, 48)

    with torch.no_grad():
        for recorded in (torch.jit.trace(f, (_n(20, 16), _n(20, 16, seed=2))), make_fx(f)(_n(20, 16), _n(20, 16, seed=2))):
            x, y = _n(20, 16, seed=3), _n(20, 16, seed=4)
            assert all(torch.equal(a, b) for a, b in zip(recorded(x, y), f(x, y)))
            assert torch.equal(f(x, y)[0], ops.sandwich_norm(x, y, gate=x[0], residual_scale=0.5)[0])


def _captured(step):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    return out


def test_capture_beside_an_eager_graph_of_other_leaves():
    """An eager graph of a weight lives; a captured backward pass that does not ask for the weight's gradient has nothing to do with it."""
    x = _n(20, 16).requires_grad_(True)
    w = [_n(24, 16, seed=i).requires_grad_(True) for i in (1, 2)]
    p = _n(16, dtype=torch.float32).requires_grad_(True)
    plain = lambda: torch.autograd.grad(ops.gated_linear(x, *w).sum(), [x])  # noqa: E731
    normed = lambda: torch.autograd.grad(ops.sandwich_norm(x, pre_weight=p)[1].sum(), [x])  # noqa: E731
    want = [plain()[0], normed()[0]]
    eager = ops.gated_linear(x.detach(), *w), ops.sandwich_norm(x.detach(), pre_weight=p)[1]
    got = [_captured(plain)[0], _captured(normed)[0]]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(t.grad_fn is not None for t in eager)
    with pytest.raises(RuntimeError, match="release its outputs"):
        _captured(lambda: torch.autograd.grad(ops.gated_linear(x, *w).sum(), w))
    _lib.assert_device_ok()
