"""ops.gated_linear and its gradients against the formulas in 64 bits and against differences."""

import math

import pytest
import torch

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


def _inputs(M, K, F, dtype, bias, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*s, std):
        return (torch.randn(*s, device="cuda", generator=g) * std).to(dtype)

    t = {"x": n(M, K, std=1.0), "w_gate": n(F, K, std=K ** -0.5), "w_up": n(F, K, std=K ** -0.5)}
    t["b_gate"], t["b_up"] = (n(F, std=0.5), n(F, std=0.5)) if bias else (None, None)
    t["dh"] = n(M, F, std=0.1)
    return t


def _act(v, act):
    """act, its slope."""
    if act == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + th), 0.5 * (1 + th) + 0.5 * v * (1 - th * th) * c * (1 + 3 * 0.044715 * v * v)


def _reference(t, act, grads):
    """Results and gradients in 64 bits, and how far roundings may put each off, by arithmetic:
    a sum of n products in fp32 by (n / 16 + 16) 2^-22 of the terms' sizes (the tensor core adds 16 products at a time, a step and a half of
    truncation each); the activation by 2^-20 of its value; a value kept in the half type by half a step.  Both activations'
    slopes are below 1.13 and second derivatives below 1."""
    d = {k: None if v is None else v.detach().double() for k, v in t.items()}
    step = torch.finfo(t["x"].dtype).eps / 2
    tiny = torch.finfo(t["x"].dtype).smallest_normal * step
    x, wg, wu = d["x"], d["w_gate"], d["w_up"]
    M, K = x.shape
    F = wg.shape[0]

    def acc(n):
        return (n / 16 + 16) * 2.0 ** -22

    g, u = x @ wg.T, x @ wu.T
    og, ou = (acc(K) * (x.abs() @ w.abs().T) for w in (wg, wu))
    if d["b_gate"] is not None:
        g, og = g + d["b_gate"], og + 2.0 ** -23 * d["b_gate"].abs()
    if d["b_up"] is not None:
        u, ou = u + d["b_up"], ou + 2.0 ** -23 * d["b_up"].abs()
    a, s = _act(g, act)
    oa = 1.13 * og + 2.0 ** -20 * a.abs() + 2.0 ** -40
    h = a * u
    out, off = {"h": h}, {"h": oa * u.abs() + a.abs() * ou + oa * ou}
    if grads:
        dh = d["dh"]
        og, ou = og + 2.0 ** -16 * g.abs() + 2.0 ** -130, ou + 2.0 ** -16 * u.abs() + 2.0 ** -130  # as they are kept: 24 bits, half a step 2^-17
        dg, du = dh * u * s, dh * a
        os_ = og + 2.0 ** -19
        odg = dh.abs() * (ou * s.abs() + u.abs() * os_ + ou * os_)
        odu = dh.abs() * (1.13 * og + 2.0 ** -20 * a.abs() + 2.0 ** -40)
        bias = {"b_gate": (dg.sum(0), odg.sum(0) + (M + 16) * 2.0 ** -24 * dg.abs().sum(0)), "b_up": (du.sum(0), odu.sum(0) + (M + 16) * 2.0 ** -24 * du.abs().sum(0))}
        for n, (v, o) in bias.items():
            if d[n] is not None:
                out[n], off[n] = v, o
        odg, odu = odg + step * (dg.abs() + odg) + tiny, odu + step * (du.abs() + odu) + tiny
        out["x"] = dg @ wg + du @ wu
        off["x"] = odg @ wg.abs() + odu @ wu.abs() + acc(2 * F) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
        for n, v, o in (("w_gate", dg, odg), ("w_up", du, odu)):
            out[n], off[n] = v.T @ x, o.T @ x.abs() + acc(M) * (v.abs().T @ x.abs())
    return out, off


def _compare(name, got, ref, off):
    f = torch.finfo(got.dtype)
    room = f.eps / 2 * (ref.abs() + off) + off + f.smallest_normal * f.eps / 2
    err = (got.detach().double().reshape(ref.shape) - ref).abs()
    assert bool((err <= room).all()), (name, float((err / room).max()))
    # and as a whole: the bounds above are for the worst case of every rounding; in the mean they go by their squares
    assert float((err * err).sum().sqrt()) <= 4 * f.eps * float((ref * ref).sum().sqrt()) + 1e-6, name


def _call(t, act):
    return ops.gated_linear(t["x"], t["w_gate"], t["w_up"], t["b_gate"], t["b_up"], act=act)


# (rows, K, F): one row, the forms for few rows with ragged columns, one tile and its edges, single and paired tiles, odd sizes
FORWARD = [(1, 8, 8), (1, 1536, 8960), (2, 72, 24), (31, 520, 136), (32, 64, 16), (33, 128, 264), (77, 1032, 1000), (128, 256, 64), (129, 64, 128), (200, 200, 1544),
           (257, 328, 136), (1, 5120, 13824), (5, 13824, 72), (16, 5120, 1504), (8, 1536, 1208), (9, 16400, 208), (1101, 136, 392), (1500, 264, 4616), (5000, 72, 1160), (3, 8200, 40)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,bias", [("silu", False), ("gelu_tanh", True)])
@pytest.mark.parametrize("M,K,F", FORWARD)
def test_forward(M, K, F, act, bias, dtype):
    t = _inputs(M, K, F, dtype, bias, M + K + F)
    h = _call(t, act)
    _lib.assert_device_ok()
    assert h.shape == (M, F) and h.dtype == dtype
    ref, off = _reference(t, act, False)
    _compare("h", h, ref["h"], off["h"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu_tanh", False)])
@pytest.mark.parametrize("M,K,F", [(1, 8, 8), (2, 72, 24), (33, 64, 128), (64, 128, 64), (65, 200, 72), (130, 520, 264), (257, 136, 1000), (300, 1536, 392), (1101, 264, 520),
                                   (2500, 1160, 1288), (40, 8200, 16), (9000, 24, 40), (100, 72, 13832), (100, 20008, 64), (300, 72, 20008), (20000, 136, 72),
                                   (6001, 264, 520), (513, 72, 9000), (7000, 8, 8)])
def test_gradients(M, K, F, act, bias, dtype):
    t = _inputs(M, K, F, dtype, bias, M + K + F + 1)
    leaves = {k: t[k].requires_grad_(True) for k in ("x", "w_gate", "w_up", "b_gate", "b_up") if t[k] is not None}
    h = _call(t, act)
    grads = torch.autograd.grad(h, list(leaves.values()), t["dh"])
    _lib.assert_device_ok()
    ref, off = _reference(t, act, True)
    _compare("h", h, ref["h"], off["h"])
    with torch.no_grad():
        alone = _call(t, act)
    _compare("h", alone, ref["h"], off["h"])
    assert M <= 16 or torch.equal(alone, h)  # the same kernel with and without what the backward pass keeps, but for few rows
    for name, g in zip(leaves, grads):
        assert g.shape == t[name].shape and g.dtype == dtype
        _compare(name, g, ref[name], off[name])


def test_each_gradient_alone(way):
    t = _inputs(300, 136, 264, torch.bfloat16, True, 5)
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    for n in names:
        t[n].requires_grad_(True)
    whole = dict(zip(names, torch.autograd.grad(_call(t, "silu"), [t[n] for n in names], t["dh"])))
    launches = {}
    for n in names:  # asked for alone
        h = _call(t, "silu")
        before = ops.STATS.kernels
        (g,) = torch.autograd.grad(h, [t[n]], t["dh"])
        launches[n] = ops.STATS.kernels - before
        assert torch.equal(g, whole[n]), n
    # the elements' gradients, and one product or sum; from Python a function does not hear which of its gradients are asked for
    assert way == "python" or launches == {"x": 2, "w_gate": 2, "w_up": 2, "b_gate": 2, "b_up": 2}
    for n in names:  # the only one that has one
        for k in names:
            t[k].requires_grad_(k == n)
        (g,) = torch.autograd.grad(_call(t, "silu"), [t[n]], t["dh"])
        assert torch.equal(g, whole[n]), n


def test_gradient_against_differences():
    """Along a direction, by differences of the formula in 64 bits."""
    t = _inputs(40, 64, 72, torch.float16, True, 9)
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    for n in names:
        t[n].requires_grad_(True)
    for act in ("silu", "gelu_tanh"):
        grads = dict(zip(names, torch.autograd.grad(_call(t, act), [t[n] for n in names], t["dh"])))
        for n in names:
            u = torch.randn(t[n].shape, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(3))

            def f(s):
                v = {k: t[k].detach().double() + (s * u if k == n else 0) for k in names}
                g, up = v["x"] @ v["w_gate"].T + v["b_gate"], v["x"] @ v["w_up"].T + v["b_up"]
                return float((_act(g, act)[0] * up * t["dh"].double()).sum())

            diff = (f(1e-4) - f(-1e-4)) / 2e-4
            terms = (grads[n].double() * u)
            # four half steps per term (twice the projections' gradients, and the result); the differences are off by the order of 1e-8
            assert abs(float(terms.sum()) - diff) <= 4 * torch.finfo(torch.float16).eps / 2 * float(terms.abs().sum()) + 1e-4 * (1 + abs(diff)), (n, act)


def test_strides_leading_axes_and_empty():
    t = _inputs(24, 136, 264, torch.bfloat16, True, 11)
    whole = _call(t, "silu")
    assert torch.equal(_call({**t, "x": t["x"].view(2, 3, 4, 136)}, "silu").reshape(24, -1), whole)
    fused = torch.cat([t["w_gate"], t["w_up"]])  # the two halves of one weight
    a, b = fused.chunk(2)
    assert torch.equal(_call({**t, "w_gate": a, "w_up": b}, "silu"), whole)
    wide = torch.full((264, 400), float("nan"), device="cuda").bfloat16()
    xw = torch.full((24, 400), float("nan"), device="cuda").bfloat16()
    for at in (8, 3):  # rows apart, on a 16-byte boundary and off it
        wide[:, at:at + 136], xw[:, at:at + 136] = t["w_gate"], t["x"]
        assert torch.equal(_call({**t, "w_gate": wide[:, at:at + 136], "x": xw[:, at:at + 136]}, "silu"), whole)
    assert torch.equal(_call({**t, "w_up": t["w_up"].T.contiguous().T}, "silu"), whole)
    for n in ("x", "w_gate", "w_up", "b_gate", "b_up"):
        t[n].requires_grad_(True)
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    h = _call(t, "silu")
    grads = torch.autograd.grad(h, [t[n] for n in names], t["dh"], retain_graph=True)
    dw = torch.zeros(24, 300, device="cuda").bfloat16()
    dw[:, 8:272] = t["dh"]
    again = torch.autograd.grad(h, [t[n] for n in names], dw[:, 8:272])
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    h = _call(t, "silu")
    expanded = torch.autograd.grad(h, [t[n] for n in names], t["dh"][:1, :1].expand(24, 264))
    same = torch.autograd.grad(_call(t, "silu"), [t[n] for n in names], t["dh"][:1, :1].expand(24, 264).contiguous())
    assert all(torch.equal(p, q) for p, q in zip(expanded, same))
    empty = _call({**t, "x": t["x"][:0]}, "silu")
    assert empty.shape == (0, 264)
    got = torch.autograd.grad(empty, [t["w_gate"], t["b_up"]], torch.empty_like(empty))
    assert not bool(got[0].any()) and not bool(got[1].any())


def test_rows_are_apart():
    """A row of NaN or infinities stays its own, in the form for few rows too; rows behind the last one are not written."""
    for M in (20, 300):
        t = _inputs(M, 264, 200, torch.float16, False, 13)
        whole = _call(t, "silu")
        x = t["x"].clone()
        x[3], x[17] = float("nan"), float("inf")
        h = _call({**t, "x": x}, "silu")
        keep = [i for i in range(M) if i not in (3, 17)]
        assert torch.equal(h[keep], whole[keep]) and bool(h[3].isnan().all())
        lib, buf = _lib.load(), torch.full((M + 40, 200), 7.0, device="cuda").half()
        rc = lib.ksb_gated_linear(t["x"].data_ptr(), 264, t["w_gate"].data_ptr(), 264, t["w_up"].data_ptr(), 264, None, None, 1, M, 200, 264, 0, buf.data_ptr(), None,
                                  torch.cuda.current_stream().cuda_stream)
        assert rc == 1
        assert torch.equal(buf[:M], whole) and bool((buf[M:] == 7).all())


def test_far_out_activations():
    """Values whose exponentials leave fp32's range."""
    for act in ("silu", "gelu_tanh"):
        v = torch.tensor([-60000.0, -300.0, -100.0, -88.5, -20.0, 0.0, 20.0, 89.0, 300.0, 60000.0], device="cuda")
        x = torch.zeros(10, 8, device="cuda")
        x[:, 0], x[:, 1] = v, 1
        w_gate, w_up = torch.zeros(8, 8, device="cuda"), torch.zeros(8, 8, device="cuda")
        w_gate[:, 0], w_up[:, 1] = 1, 1
        t = {"x": x.bfloat16().requires_grad_(True), "w_gate": w_gate.bfloat16(), "w_up": w_up.bfloat16(), "b_gate": None, "b_up": None}
        h = _call(t, act)
        a, s = _act(t["x"].detach().double()[:, :1], act)
        assert torch.allclose(h.double(), a.expand(10, 8), rtol=2.0 ** -8, atol=1e-37)
        (dx,) = torch.autograd.grad(h, [t["x"]], torch.ones_like(h))
        # eight columns' dg, each half a step off, and half a step of the sum
        assert torch.allclose(dx.double()[:, :1], 8 * s, rtol=2.0 ** -7, atol=1e-30)


def test_repeats_streams_and_graph():
    t = _inputs(700, 264, 520, torch.bfloat16, True, 17)
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    leaves = [t[n].requires_grad_(True) for n in names]

    def step():
        h = _call(t, "silu")
        return [h.detach(), *torch.autograd.grad(h, leaves, t["dh"])]

    ref = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), ref))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        t["x"].copy_(t["x"] * 0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))
    _lib.assert_device_ok()


def test_no_second_derivatives():
    """With create_graph the gradients are the same ones; to differentiate them again is an error, not a constant."""
    t = _inputs(40, 72, 136, torch.bfloat16, True, 21)
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    leaves = [t[n].requires_grad_(True) for n in names]
    step = lambda: _call(t, "silu")  # noqa: E731
    whole = torch.autograd.grad(step().float().sum(), leaves)
    again = torch.autograd.grad(step().float().sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(whole, again))
    for g in again:
        with pytest.raises(RuntimeError, match="no second derivatives"):
            torch.autograd.grad(g.float().square().sum(), leaves[0], allow_unused=True)


def test_capture_with_eager_leaves_alive():
    """A leaf's accumulation node of the default stream cannot take part in a capture: an error of the call, and nothing is lost."""
    t = _inputs(40, 72, 136, torch.bfloat16, True, 21)
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    leaves = [t[n].requires_grad_(True) for n in names]
    step = lambda: _call(t, "silu")  # noqa: E731
    eager = step()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="release its outputs"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(step().sum(), leaves)
    whole = torch.autograd.grad(eager.sum(), leaves)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(step().sum(), leaves)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, whole))
    _lib.assert_device_ok()
