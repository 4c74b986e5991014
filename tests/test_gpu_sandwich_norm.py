"""ops.sandwich_norm and its gradients against the formulas in 64 bits and against differences."""

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

NAMES = ("x", "y", "gate", "scale", "shift", "post_weight", "pre_weight")


def _inputs(shape, mods, weights, dtype, seed=0, without=()):
    """mods: shape of the modulation's leading axes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    C = shape[-1]

    def n(*s, std=1.0):
        return torch.randn(*s, device="cuda", generator=g) * std

    t = {"x": n(*shape).to(dtype), "y": (3 * n(*shape) + 0.5).to(dtype)}
    for name in ("gate", "scale", "shift"):
        t[name] = n(*mods, C, std=0.3).to(dtype)
    t["post_weight"], t["pre_weight"] = (1 + n(C, std=0.2), 1 + n(C, std=0.2)) if weights else (None, None)
    for name in without:
        t[name] = None
    t["dr"], t["dh"] = n(*shape).to(dtype), n(*shape).to(dtype)
    return t


def _norm(v, layer, eps):
    d = v - v.mean(-1, keepdim=True) if layer else v
    return d * torch.rsqrt((d * d).mean(-1, keepdim=True) + eps)


def _rows_of(t, shape):
    """A modulation tensor as rows that broadcast against [M, C]."""
    M, C = torch.Size(shape[:-1]).numel(), shape[-1]
    t2 = t.reshape(-1, C)
    return t2.repeat_interleave(M // t2.shape[0], 0)


def _reference(t, a, layer, eps, use_r=True, use_h=True, grads=True):
    """Results and gradients in 64 bits, by the formulas, and for each the size of the terms that its fp32 roundings go by."""
    d = {k: None if v is None else v.detach().double() for k, v in t.items()}
    shape = d["x"].shape
    C = shape[-1]
    x = d["x"].reshape(-1, C)
    mod = {k: None if d[k] is None else _rows_of(d[k], shape) for k in ("gate", "scale", "shift")}
    one = torch.ones((), dtype=torch.float64, device="cuda")
    gate, scale = (one if mod["gate"] is None else mod["gate"]), (0 * one if mod["scale"] is None else mod["scale"])
    shift = 0 * one if mod["shift"] is None else mod["shift"]
    wp, wn = (one if d[k] is None else d[k] for k in ("post_weight", "pre_weight"))
    out, size = {}, {}

    def stats(v):
        mean = v.mean(-1, keepdim=True) if layer else 0 * one
        c = v - mean
        rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
        return c * rstd, rstd, (v.abs() + abs(mean)) * rstd  # last: what the normed value's roundings go by

    A, B = a * gate * wp, (1 + scale) * wn
    B_size = (1 + scale.abs()) * wn.abs()
    if d["y"] is not None:
        yh, y_rstd, yh_size = stats(d["y"].reshape(-1, C))
        r = x + A * yh
        r_size = x.abs() + A.abs() * yh_size
    else:
        r, r_size, yh = x, x.abs(), None
    out["r"], size["r"] = r, r_size
    if use_h:
        rh, r_rstd, _ = stats(r)
        mean_abs = r_size.mean(-1, keepdim=True) if layer else 0
        rh_size = (r_size + mean_abs) * r_rstd + rh.abs()
        out["h"], size["h"] = rh * B + shift, rh_size * B_size + shift.abs()
    if grads:
        D = d["dr"].reshape(-1, C) if use_r else torch.zeros_like(x)
        D_size = D.abs()
        if use_h:
            dh = d["dh"].reshape(-1, C)
            tt, t_size = dh * B, dh.abs() * B_size
            m1, m1_size = (tt * rh).mean(-1, keepdim=True), (t_size * rh_size).mean(-1, keepdim=True)
            m0, m0_size = (tt.mean(-1, keepdim=True), t_size.mean(-1, keepdim=True)) if layer else (0, 0)
            D = D + r_rstd * (tt - rh * m1 - m0)
            D_size = D_size + r_rstd * (t_size + rh_size * m1_size + m0_size)
        out["x"], size["x"] = D, D_size
        if yh is not None:
            e, e_size = D * A, D_size * A.abs()
            n1, n1_size = (e * yh).mean(-1, keepdim=True), (e_size * yh_size).mean(-1, keepdim=True)
            n0, n0_size = (e.mean(-1, keepdim=True), e_size.mean(-1, keepdim=True)) if layer else (0, 0)
            out["y"], size["y"] = y_rstd * (e - yh * n1 - n0), y_rstd * (e_size + yh_size * n1_size + n0_size)

        def total(name, v, s):
            ref = d[name]
            rows = 1 if ref.dim() == 1 or ref.numel() == C else ref.numel() // C
            out[name] = v.reshape(rows, -1, C).sum(1)
            size[name] = s.reshape(rows, -1, C).sum(1)

        full = torch.ones_like(x)
        if yh is not None:
            if d["gate"] is not None:
                total("gate", a * wp * D * yh, abs(a) * wp.abs() * D_size * yh_size * full)
            if d["post_weight"] is not None:
                total("post_weight", a * gate * D * yh, abs(a) * gate.abs() * D_size * yh_size * full)
        if use_h:
            if d["scale"] is not None:
                total("scale", dh * rh * wn, dh.abs() * rh_size * wn.abs() * full)
            if d["pre_weight"] is not None:
                total("pre_weight", dh * rh * (1 + scale), dh.abs() * rh_size * (1 + scale.abs()) * full)
            if d["shift"] is not None:
                total("shift", dh * full, dh.abs())
    return out, size


def _compare(name, got, ref, size, rows=0):
    """Half a step of the result's type, and of the fp32 sums: at most 64 roundings on the way to a value (a row's sums are trees of a few
    dozen), one more for each row that a sum over rows runs over, each 2^-24 of the terms' sizes; half the least number of the type."""
    f = torch.finfo(got.dtype)
    room = f.eps / 2 * ref.abs() * (got.dtype != torch.float32) + (64 + rows) * 2.0 ** -24 * (1 + f.eps) * size + f.smallest_normal * f.eps / 2
    err = (got.detach().double().reshape(ref.shape) - ref).abs()
    assert bool((err <= room).all()), (name, float((err / room).max()))


SHAPES = [
    ((1, 8), (1,), True), ((5, 64), (5,), True), ((3, 7, 40), (3, 1), False), ((2, 33, 1536), (2, 1), True), ((2, 65, 1544), (), True), ((1, 130, 5120), (1, 1), True),
    ((2, 5, 8192), (2, 5), False), ((400, 3, 72), (400, 1), True), ((2, 300, 264), (2, 300), True), ((600, 2056), (300,), False), ((3, 777, 520), (3,), True),
    ((2, 3, 4, 136), (2, 3, 1), True), ((40000, 16), (2,), True), ((16500, 528), (1,), True), ((4100, 264), (4100,), True), ((2, 2100, 1544), (2, 2100), False), ((200, 2, 5200), (200, 1), True)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("shape,mods,weights", SHAPES)
def test_results_and_gradients(shape, mods, weights, kind, dtype):
    t = _inputs(shape, mods, weights, dtype, sum(shape))
    ref, size = _reference(t, 0.5, kind == "layer", 1e-6)
    leaves = {k: t[k].requires_grad_(True) for k in NAMES if t[k] is not None}
    kw = {k: t[k] for k in NAMES[2:]}
    with torch.no_grad():
        r, h = ops.sandwich_norm(t["x"], t["y"], residual_scale=0.5, kind=kind, **kw)
    r2, h2 = ops.sandwich_norm(t["x"], t["y"], residual_scale=0.5, kind=kind, **kw)
    assert torch.equal(r, r2) and torch.equal(h, h2) and r.shape == h.shape == torch.Size(shape)
    grads = torch.autograd.grad((r2, h2), list(leaves.values()), (t["dr"], t["dh"]))
    _lib.assert_device_ok()
    _compare("r", r, ref["r"], size["r"])
    _compare("h", h, ref["h"], size["h"])
    rows = torch.Size(shape[:-1]).numel()
    for name, g in zip(leaves, grads):
        assert g.shape == t[name].shape and g.dtype == t[name].dtype
        _compare(name, g, ref[name], size[name], rows if name not in ("x", "y") else 0)


@pytest.mark.parametrize("without", [("gate",), ("scale", "shift"), ("gate", "scale", "shift", "post_weight", "pre_weight"), ("shift", "post_weight")])
@pytest.mark.parametrize("use_r,use_h", [(True, True), (True, False), (False, True)])
def test_optional_parts(without, use_r, use_h):
    t = _inputs((2, 50, 264), (2, 1), True, torch.bfloat16, 3, without)
    ref, size = _reference(t, 1.0, True, 1e-5, use_r, use_h)
    leaves = {k: t[k].requires_grad_(True) for k in NAMES if t[k] is not None}
    r, h = ops.sandwich_norm(t["x"], t["y"], kind="layer", eps=1e-5, **{k: t[k] for k in NAMES[2:]})
    pick = [v for v, u in ((r, use_r), (h, use_h)) if u]
    grads = torch.autograd.grad(pick, list(leaves.values()), [v for v, u in ((t["dr"], use_r), (t["dh"], use_h)) if u], allow_unused=True)
    for name, g in zip(leaves, grads):
        if name in ref:
            _compare(name, g, ref[name], size[name], 100 if name not in ("x", "y") else 0)
        else:
            assert g is None, name


def test_each_gradient_alone(way):
    t = _inputs((2, 40, 264), (2, 1), True, torch.bfloat16, 19)
    leaves = {k: t[k].requires_grad_(True) for k in NAMES}

    def call():
        return ops.sandwich_norm(t["x"], t["y"], **{k: t[k] for k in NAMES[2:]})

    whole = dict(zip(leaves, torch.autograd.grad(call(), list(leaves.values()), (t["dr"], t["dh"]))))
    for n in NAMES:
        out = call()
        before = ops.STATS.kernels
        (g,) = torch.autograd.grad(out, [t[n]], (t["dr"], t["dh"]))
        assert torch.equal(g, whole[n]), n
        # sums over rows only where they are asked for (from Python a function does not hear which are)
        assert way == "python" or ops.STATS.kernels - before == (1 if n in ("x", "y") else 2), n
    for n in NAMES:
        for k in NAMES:
            t[k].requires_grad_(k == n)
        (g,) = torch.autograd.grad(call(), [t[n]], (t["dr"], t["dh"]))
        assert torch.equal(g, whole[n]), n


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_one_sided_forms(kind):
    t = _inputs((3, 20, 136), (3, 1), True, torch.float16, 5)
    layer = kind == "layer"
    # only the norm ahead: x itself comes back
    ahead = {**t, "y": None, "gate": None, "post_weight": None}
    ref, size = _reference(ahead, 1.0, layer, 1e-6)
    leaves = {k: t[k].requires_grad_(True) for k in ("x", "scale", "shift", "pre_weight")}
    r, h = ops.sandwich_norm(t["x"], scale=t["scale"], shift=t["shift"], pre_weight=t["pre_weight"], kind=kind)
    assert r is t["x"]
    _compare("h", h, ref["h"], size["h"])
    _, size_g = ref, size
    ref0, size0 = _reference(ahead, 1.0, layer, 1e-6, use_r=False)
    for name, g in zip(leaves, torch.autograd.grad(h, list(leaves.values()), t["dh"])):
        _compare(name, g, ref0[name], size0[name], 60)
    # only the norm behind
    behind = {**t, "scale": None, "shift": None, "pre_weight": None}
    ref, size = _reference(behind, 2.0, layer, 1e-6, use_h=False)
    leaves = {k: t[k].requires_grad_(True) for k in ("x", "y", "gate", "post_weight")}
    r, h = ops.sandwich_norm(t["x"], t["y"], gate=t["gate"], post_weight=t["post_weight"], residual_scale=2.0, pre=False, kind=kind)
    assert h is None
    _compare("r", r, ref["r"], size["r"])
    for name, g in zip(leaves, torch.autograd.grad(r, list(leaves.values()), t["dr"])):
        _compare(name, g, ref[name], size[name], 60)


def test_modulation_of_different_rows_and_views():
    """A gate shared by all beside scales per sample; chunks of one modulation tensor (rows apart); columns off a 16-byte boundary."""
    t = _inputs((3, 20, 136), (3, 1), True, torch.bfloat16, 7)
    t["gate"] = t["gate"][0, 0].clone()
    ref, size = _reference(t, 1.0, False, 1e-6)
    leaves = {k: t[k].requires_grad_(True) for k in NAMES}
    r, h = ops.sandwich_norm(t["x"], t["y"], **{k: t[k] for k in NAMES[2:]})
    for name, g in zip(leaves, torch.autograd.grad((r, h), list(leaves.values()), (t["dr"], t["dh"]))):
        if name == "gate":  # three samples' gradients, each rounded to bf16 on its way
            size[name] = size[name] + 3 * torch.finfo(torch.bfloat16).eps / 2 * 2 ** 24 / 124 * size[name]
        _compare(name, g, ref[name], size[name], 60 if name not in ("x", "y") else 0)
    with torch.no_grad():
        for C, pad in ((136, 0), (136, 4)):
            mods = torch.randn(3, 1, 3 * C + pad, device="cuda").bfloat16()
            gate, scale, shift = mods[..., pad:].chunk(3, -1)
            a = ops.sandwich_norm(t["x"], t["y"], gate=gate, scale=scale, shift=shift)
            b = ops.sandwich_norm(t["x"], t["y"], gate=gate.contiguous(), scale=scale.contiguous(), shift=shift.contiguous())
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        wide = torch.randn(3, 20, 300, device="cuda").bfloat16()
        for at in (8, 3):
            v = wide[..., at:at + 136]
            a, b = ops.sandwich_norm(v, v), ops.sandwich_norm(v.contiguous(), v.contiguous())
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        v = t["x"][:, :1].expand(3, 20, 136)
        a, b = ops.sandwich_norm(v, t["y"]), ops.sandwich_norm(v.contiguous(), t["y"])
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_gradient_against_differences():
    """The derivative along a direction, by differences of the forward pass in 64 bits: (f(v + s u) - f(v - s u)) / 2 s, off by s^2."""
    t = _inputs((2, 9, 72), (2, 1), True, torch.float16, 11)
    leaves = {k: t[k].requires_grad_(True) for k in NAMES}
    r, h = ops.sandwich_norm(t["x"], t["y"], kind="layer", **{k: t[k] for k in NAMES[2:]})
    grads = torch.autograd.grad((r, h), list(leaves.values()), (t["dr"], t["dh"]))
    g = torch.Generator(device="cuda").manual_seed(1)

    def f(v):
        out, _ = _reference({**t, **v}, 1.0, True, 1e-6, grads=False)
        return float((out["r"] * t["dr"].double().reshape(out["r"].shape)).sum() + (out["h"] * t["dh"].double().reshape(out["r"].shape)).sum())

    for name, grad in zip(leaves, grads):
        u = torch.randn(t[name].shape, device="cuda", dtype=torch.float64, generator=g)
        s = 1e-4
        diff = (f({name: t[name].detach().double() + s * u}) - f({name: t[name].detach().double() - s * u})) / (2 * s)
        dot = float((grad.double() * u).sum())
        # half a step per term of the dot product; the differences' own error is of the order s^2 = 1e-8 of the third derivatives
        room = float((grad.double() * u).abs().sum()) * torch.finfo(torch.float16).eps + 1e-4 * (1 + abs(diff))
        assert abs(dot - diff) <= room, (name, dot, diff, room)


def test_rows_are_apart_and_specials():
    t = _inputs((6, 200), (6,), True, torch.bfloat16, 13)
    clean = ops.sandwich_norm(t["x"], t["y"], **{k: t[k] for k in NAMES[2:]})
    x, y = t["x"].clone(), t["y"].clone()
    x[1, 3], y[2, 5], y[4] = float("nan"), float("inf"), 0
    x[5], y[5] = 0, 0
    r, h = ops.sandwich_norm(x, y, **{k: t[k] for k in NAMES[2:]})
    for i in (0, 3):
        assert torch.equal(r[i], clean[0][i]) and torch.equal(h[i], clean[1][i])
    assert bool(h[1].isnan().all()) and bool(r[1, 3].isnan()) and int(r[1].isnan().sum()) == 1
    assert torch.equal(r[4], x[4])  # the norm of zeros is zeros
    assert torch.equal(r[5], x[5]) and torch.equal(h[5], t["shift"][5])


def test_empty():
    x = torch.empty(2, 0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    gate = torch.ones(2, 1, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    r, h = ops.sandwich_norm(x, x, gate=gate, scale=gate, post_weight=w)
    assert r.shape == h.shape == (2, 0, 64)
    gx, gg, gw = torch.autograd.grad((r, h), (x, gate, w), (torch.empty_like(r), torch.empty_like(h)))
    assert gx.shape == x.shape and not bool(gg.any()) and not bool(gw.any())


def test_repeats_streams_and_graph():
    t = _inputs((2, 700, 1032), (2, 1), True, torch.bfloat16, 17)
    leaves = [t[k].requires_grad_(True) for k in NAMES]

    def step():
        r, h = ops.sandwich_norm(t["x"], t["y"], **{k: t[k] for k in NAMES[2:]})
        return [r.detach(), h.detach(), *torch.autograd.grad((r, h), leaves, (t["dr"], t["dh"]))]

    ref = step()
    for a, b in zip(step(), ref):
        assert torch.equal(a, b)  # the order of the sums is fixed
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
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_no_second_derivatives():
    """With create_graph the gradients are the same ones; to differentiate them again is an error, not a constant."""
    t = _inputs((2, 20, 72), (2, 1), True, torch.bfloat16, 21)
    leaves = [t[n].requires_grad_(True) for n in NAMES]
    step = lambda: torch.cat(ops.sandwich_norm(t["x"], **{n: t[n] for n in NAMES[1:]}))  # noqa: E731
    whole = torch.autograd.grad(step().float().sum(), leaves)
    again = torch.autograd.grad(step().float().sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(whole, again))
    for g in again:
        with pytest.raises(RuntimeError, match="no second derivatives"):
            torch.autograd.grad(g.float().square().sum(), leaves[0], allow_unused=True)


def test_capture_with_eager_leaves_alive():
    """A leaf's accumulation node of the default stream cannot take part in a capture: an error of the call, and nothing is lost."""
    t = _inputs((2, 20, 72), (2, 1), True, torch.bfloat16, 21)
    leaves = [t[n].requires_grad_(True) for n in NAMES]
    step = lambda: torch.cat(ops.sandwich_norm(t["x"], **{n: t[n] for n in NAMES[1:]}))  # noqa: E731
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
