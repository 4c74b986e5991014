"""sandwich_norm of one row, or none, out of tensors whose rows are any number of elements apart."""

import pytest
import torch

from ksanadit_b200 import ops

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


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("shape", [(), (1,)])
def test_a_row_of_a_wide_tensor(rows, shape):
    C = 64
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = [torch.randn(2, 77, device="cuda", generator=g).bfloat16() for _ in range(5)]
    x, y, gate, dr, dh = (w[:rows, :C].view(*shape, rows, C) for w in wide)
    gate = wide[2][:1, :C]
    want = [t.clone(memory_format=torch.contiguous_format) for t in (x, y, gate, dr, dh)]

    def run(x, y, gate, dr, dh):
        x, y, gate = (t.detach().requires_grad_(True) for t in (x, y, gate))
        r, h = ops.sandwich_norm(x, y, gate=gate, residual_scale=1)
        with torch.no_grad():
            r2, h2 = ops.sandwich_norm(x, y, gate=gate)
        assert torch.equal(r, r2) and torch.equal(h, h2)
        return [r, h, *torch.autograd.grad((r, h), (x, y, gate), (dr, dh))]

    assert all(torch.equal(a, b) for a, b in zip(run(x, y, gate, dr, dh), run(*want)))
