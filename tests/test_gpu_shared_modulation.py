"""Gradients of a modulation tensor with one row beside others that tell rows apart: one fp32 sum over all rows, rounded once."""

import pytest
import torch
from test_gpu_sandwich_norm import NAMES, _compare, _inputs, _reference

from ksanadit_b200 import _lib, ops

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


def _grads(t, names, residual_scale=1.0, kind="rms", use_r=True, use_h=True):
    leaves = [t[k].requires_grad_(True) for k in names]
    r, h = ops.sandwich_norm(t["x"], t["y"], residual_scale=residual_scale, kind=kind, **{k: t[k] for k in NAMES[2:]})
    pick = [(v, t[d]) for v, d, use in ((r, "dr", use_r), (h, "dh", use_h)) if use]
    return dict(zip(names, torch.autograd.grad([v for v, _ in pick], leaves, [d for _, d in pick])))


# few samples of many rows, some samples, a modulation row for a few rows, a row each; one and four chunks a thread
SHAPES = [((3, 20, 136), (3, 1)), ((40, 7, 520), (40, 1)), ((400, 3, 72), (400, 1)), ((2, 300, 264), (2, 300)), ((2, 5, 8192), (2, 1)), ((200, 2, 5200), (200, 1)),
          ((2, 2100, 1544), (2, 2100))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shared", [("gate",), ("scale",), ("shift",), ("gate", "shift"), ("scale", "shift"), ("gate", "scale")])
@pytest.mark.parametrize("shape,mods", SHAPES)
def test_one_rounding(shape, mods, shared, dtype):
    kind = "layer" if len(shared) == 2 else "rms"
    t = _inputs(shape, mods, True, dtype, sum(shape))
    for i, name in enumerate(shared):
        t[name] = t[name].reshape(-1, shape[-1])[0].clone().view(*((1,) * i), -1)  # [C] and [1, C]
    ref, size = _reference(t, 0.5, kind == "layer", 1e-6)
    got = _grads(t, NAMES, 0.5, kind)
    _lib.assert_device_ok()
    rows = torch.Size(shape[:-1]).numel()
    for name, g in got.items():
        assert g.shape == t[name].shape and g.dtype == t[name].dtype
        _compare(name, g, ref[name], size[name], rows if name not in ("x", "y") else 0)
    for name in NAMES:  # the same bits whatever is asked for
        assert torch.equal(_grads(t, (name,), 0.5, kind)[name], got[name]), name


@pytest.mark.parametrize("samples,tokens", [(1, 32760), (8, 4095)])
def test_terms_below_the_types_least_number(samples, tokens):
    """A gate for all beside a scale per token, in fp16: 32760 terms of 2^-26 each, a quarter of the least fp16 number."""
    C = 64
    t = {k: None for k in NAMES}
    t["x"], t["y"] = (torch.ones(samples, tokens, C, device="cuda").half() for _ in range(2))
    t["gate"], t["scale"] = torch.ones(C, device="cuda").half(), torch.zeros(samples, tokens, C, device="cuda").half()
    t["dr"] = t["dh"] = torch.full((samples, tokens, C), 2.0 ** -24, device="cuda").half()
    # N(y) = 1 to within eps: dgate = 2^-2 sum(dr)
    got = _grads(t, ("gate",), 0.25, use_h=False)["gate"]
    assert torch.allclose(got.double(), torch.full((C,), samples * tokens * 2.0 ** -26, device="cuda").double(), rtol=2.0 ** -11 + 1e-5)


@pytest.mark.parametrize("samples,tokens", [(2, 64), (200, 2)])
def test_parts_above_the_types_largest_number(samples, tokens):
    """The first half of the samples sums to more than fp16 holds, the whole does not."""
    C = 64
    t = _inputs((samples, tokens, C), (samples, 1), False, torch.float16, 5)
    t["shift"] = t["shift"][0, 0].clone()
    t["dh"] = torch.full((samples, tokens, C), 60000.0, device="cuda").half()
    t["dh"][samples // 2:] = -60000.0
    t["dh"][-1, -1] = -59968.0
    assert torch.equal(_grads(t, ("shift",))["shift"], torch.full((C,), 32.0, device="cuda").half())


def test_expanded_rows_have_gradients_of_their_own():
    """One row that is expanded ahead of the call has a gradient per row, as any expanded tensor."""
    t = _inputs((3, 20, 136), (3, 1), True, torch.bfloat16, 7)
    one = t["gate"][:1].clone()
    t["gate"] = one.expand(3, 1, 136)
    ref, size = _reference({**t, "gate": one.repeat(3, 1, 1)}, 1.0, False, 1e-6)
    t["gate"].requires_grad_(True)
    r, h = ops.sandwich_norm(t["x"], t["y"], **{k: t[k] for k in NAMES[2:]})
    (g,) = torch.autograd.grad((r, h), [t["gate"]], (t["dr"], t["dh"]))
    assert g.shape == (3, 1, 136)
    _compare("gate", g, ref["gate"], size["gate"], 60)


def test_no_rows():
    x = torch.empty(2, 0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    gate, scale = (torch.ones(*s, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True) for s in ((), (2, 1)))
    r, h = ops.sandwich_norm(x, x, gate=gate, scale=scale)
    a, b = torch.autograd.grad((r, h), (gate, scale), (torch.empty_like(r), torch.empty_like(h)))
    assert a.shape == (64,) and b.shape == (2, 1, 64) and not bool(a.any()) and not bool(b.any())
