"""ops.w4_linear and B200W4Linear against 64-bit products of the dequantised weight."""

import pytest
import torch

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


def _case(M, N, K, group, zeros, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(N, K, device="cuda", generator=g) * 0.02
    x = torch.randn(M, K, device="cuda", generator=g)
    x[:, ::50] *= 20
    packed, scale, zero = w4.quantize_w4(w, group, zeros, dtype)
    return x.to(dtype), packed, scale, zero, (torch.randn(N, device="cuda", generator=g) * 0.1).to(dtype)


def _check(out, x, packed, scale, zero, bias, N, K):
    w = w4.dequantize_w4(packed, scale, zero, N, K).double()  # (q - z) * s is exact in fp32: 4 + 11 bits
    xd = x.double().reshape(-1, K)
    ref = xd @ w.T
    size = xd.abs() @ w.abs().T
    if bias is not None:
        ref, size = ref + bias.double(), size + bias.double().abs()
    # one rounding of the result (a half step of the smallest number where it is tiny); the sum's roundings, each at most 2^-22 of the
    # terms' sizes (a step and a half of truncation): 16 products each, over the groups, the warps and the bias
    t = x.dtype
    room = torch.finfo(t).eps / 2 * ref.abs() + (K / 16 + 48) * 2.0 ** -22 * size * (1 + torch.finfo(t).eps) + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    err = (out.double().reshape(ref.shape) - ref).abs()
    assert bool((err <= room).all()), float((err / room).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K,group,zeros", [
    (1, 16, 32, 32, False), (1, 1, 64, 64, True), (2, 17, 96, 32, True), (3, 100, 128, 128, False), (8, 48, 2048, 64, True), (9, 33, 2176, 128, True),
    (16, 4000, 256, 32, False), (7, 2500, 4160, 32, True), (17, 50, 512, 64, False), (35, 24, 128, 64, True), (1, 9216, 1536, 128, False), (12, 40, 13824, 128, True),
    (16, 64, 8960, 64, False), (5, 16, 32768, 32, True)])
def test_products(dtype, M, N, K, group, zeros):
    x, packed, scale, zero, bias = _case(M, N, K, group, zeros, dtype, M + N + K)
    for b in (None, bias):
        out = ops.w4_linear(x, packed, scale, zero, b, out_features=N)
        _lib.assert_device_ok()
        assert out.shape == (M, N) and out.dtype == dtype
        _check(out, x, packed, scale, zero, b, N, K)


def test_every_nibble_zero_point_and_place():
    """Integers throughout: exact, whatever the place of a weight."""
    N, K, group = 48, 192, 32
    g = torch.Generator().manual_seed(1)
    q = torch.randint(0, 16, (N, K), dtype=torch.uint8, generator=g)
    z = torch.randint(0, 16, (N, K // group), dtype=torch.uint8, generator=g)
    x = torch.zeros(K, K)
    x[torch.arange(K), torch.randperm(K, generator=g)] = 1  # each row picks one column
    ref = ((q.float().view(N, -1, group) - z.float()[..., None]).view(N, K) @ x.T).T
    for dtype in (torch.bfloat16, torch.float16):
        out = ops.w4_linear(x.to("cuda", dtype), w4.pack_w4(q).cuda(), w4.tile_groups(torch.ones(N, K // group, dtype=dtype)).cuda(), w4.tile_groups(z).cuda(), out_features=N)
        assert torch.equal(out.float().cpu(), ref)


def test_strides_leading_axes_and_empty():
    x, packed, scale, zero, bias = _case(6, 40, 128, 64, True, torch.bfloat16)
    whole = ops.w4_linear(x, packed, scale, zero, bias, out_features=40)
    for v in (x.view(2, 3, 128), x.view(1, 6, 1, 128)):
        assert torch.equal(ops.w4_linear(v, packed, scale, zero, bias).reshape(6, -1), whole)
    wide = torch.full((6, 300), float("nan"), dtype=torch.bfloat16, device="cuda")
    for at in (0, 8, 5):  # rows apart, on a 16-byte boundary and off it
        wide[:, at:at + 128] = x
        assert torch.equal(ops.w4_linear(wide[:, at:at + 128], packed, scale, zero, bias), whole)
    assert torch.equal(ops.w4_linear(x.T.contiguous().T, packed, scale, zero, bias), whole)
    assert torch.equal(ops.w4_linear(x[:1].expand(6, 128), packed, scale, zero, bias), whole[:1].expand(6, 40))
    assert ops.w4_linear(x[:0], packed, scale, zero, bias).shape == (0, 40)


def test_rows_do_not_touch_one_another():
    """A row of NaN or infinities leaves the others as they are, and the result does not depend on the rows beside it."""
    x, packed, scale, zero, bias = _case(16, 200, 640, 128, True, torch.float16)
    whole = ops.w4_linear(x, packed, scale, zero, bias)
    bad = x.clone()
    bad[3], bad[9] = float("nan"), float("inf")
    out = ops.w4_linear(bad, packed, scale, zero, bias)
    keep = [i for i in range(16) if i not in (3, 9)]
    assert torch.equal(out[keep], whole[keep]) and bool(out[3].isnan().all()) and not bool(out[9].isfinite().any())
    for i in (0, 7, 8, 15):
        assert torch.equal(ops.w4_linear(x[i:i + 1], packed, scale, zero, bias), whole[i:i + 1])


def test_module_stream_and_graph():
    lin = torch.nn.Linear(256, 100, device="cuda")
    m = w4.B200W4Linear.from_float(lin, 64, True)
    x = torch.randn(2, 256, device="cuda").bfloat16()
    ref = m(x)
    _check(ref, x, m.weight, m.weight_scale, m.weight_zero, m.bias, 100, 256)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = m(x)
    side.synchronize()
    assert torch.equal(y, ref)
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        y = m(static)
    static.copy_(2 * x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, m(2 * x))
    _lib.assert_device_ok()
