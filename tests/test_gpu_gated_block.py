"""The operators together, as a stack of gated halves uses them: against the formulas in 64 bits, trained, served, captured."""

import pytest
import torch

from ksanadit_b200 import _lib, ops
from ksanadit_b200.gated_block import B200GatedFeedForward, gated_stack
from ksanadit_b200.linear import B200Fp8Linear
from ksanadit_b200.w4 import B200W4Linear

pytestmark = pytest.mark.gpu


def _halves(n, dim, hidden, dtype, kind, seed, **kw):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i in range(n):
        m = B200GatedFeedForward(dim, hidden, bias=True, act=("silu", "gelu_tanh")[i % 2], kind=kind, residual_scale=0.5, group=64, device="cuda", dtype=dtype, **kw)
        for name, p in m.named_parameters():
            if p.dtype == torch.uint8 or name.startswith("modulation"):
                continue
            std = dim ** -0.5 if p.dim() == 2 else 0.2
            with torch.no_grad():
                p.copy_((1 if name.endswith("norm") else 0) + std * torch.randn(p.shape, device="cuda", generator=g))
        lin = torch.nn.Linear(dim, 3 * dim, device="cuda")
        with torch.no_grad():
            lin.weight.copy_(0.3 * dim ** -0.5 * torch.randn(lin.weight.shape, device="cuda", generator=g))
            lin.bias.copy_(0.3 * torch.randn(lin.bias.shape, device="cuda", generator=g))
        if m.modulation is not None:
            m.modulation = B200W4Linear.from_float(lin, 64, dtype=dtype)
        out.append(m)
    x = torch.randn(2, 75, dim, device="cuda", generator=g).to(dtype)
    temb = torch.randn(2, dim, device="cuda", generator=g).to(dtype)
    return out, x, temb


def _formula(halves, x, vectors, p):
    """The stack in 64 bits; p: parameters by (half, name)."""
    def norm(v, w, m):
        c = v - v.mean(-1, keepdim=True) if m.kind == "layer" else v
        return c * torch.rsqrt((c * c).mean(-1, keepdim=True) + m.eps) * w

    for i, (m, (shift, scale, gate)) in enumerate(zip(halves, vectors)):
        h = norm(x, p[i, "pre_norm"], m) * (1 + scale) + shift
        g, u = h @ p[i, "w_gate"].T + p[i, "b_gate"], h @ p[i, "w_up"].T + p[i, "b_up"]
        a = torch.nn.functional.silu(g) if m.act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
        y = (a * u) @ p[i, "down.weight"].T + p[i, "down.bias"]
        x = x + m.residual_scale * gate * norm(y, p[i, "post_norm"], m)
    return x


def _off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_stack_and_its_gradients(dtype, kind):
    halves, x, temb = _halves(3, 256, 520, dtype, kind, 1)
    vectors = [m.vectors(temb) for m in halves]
    for m, v in zip(halves, vectors):  # the 4-bit product, one rounding of it and of the SiLU ahead of it
        exact = torch.nn.functional.linear(torch.nn.functional.silu(temb.double()), m.modulation.dequantized().double(), m.modulation.bias.double())
        assert _off(torch.cat(v, -1)[:, 0], exact) <= 2 * torch.finfo(dtype).eps
    params = {(i, n): q.detach().double().requires_grad_(True) for i, m in enumerate(halves) for n, q in m.named_parameters() if not n.startswith("modulation")}
    xd = x.double().requires_grad_(True)
    ref = _formula(halves, xd, [[v.double() for v in vs] for vs in vectors], params)
    x.requires_grad_(True)
    out = gated_stack(halves, x, temb)
    dy = torch.randn(out.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    mine = [(i, n) for i, m in enumerate(halves) for n, _ in m.named_parameters() if not n.startswith("modulation")]
    got = torch.autograd.grad(out, [x] + [dict(halves[i].named_parameters())[n] for i, n in mine], dy)
    want = torch.autograd.grad(ref, [xd] + [params[k] for k in mine], dy.double())
    _lib.assert_device_ok()
    # a handful of roundings per half, each half a step and independent of the others: in the mean they add up by their squares, and a few
    # dozen of them (three halves, forward and back) stay below eight steps
    step = torch.finfo(dtype).eps
    assert _off(out.detach(), ref.detach()) <= 4 * step
    for k, a, b in zip(["x"] + mine, got, want):
        assert _off(a, b) <= 8 * step, (k, _off(a, b) / step)


def test_one_half_alone_and_vectors_of_the_caller():
    halves, x, temb = _halves(2, 128, 264, torch.bfloat16, "rms", 3)
    with torch.no_grad():
        whole = gated_stack(halves, x, temb)
        vectors = [m.vectors(temb) for m in halves]
        assert torch.equal(gated_stack(halves, x, vectors=vectors), whole)
        one = halves[1](halves[0](x, temb), vectors=vectors[1])
        # the shared pass norms the unrounded sum, the halves apart a rounded one
        assert _off(one, whole.double()) <= 4 * torch.finfo(torch.bfloat16).eps
        assert gated_stack([], x, temb) is x
    with pytest.raises(_lib.KsanaB200Error):
        gated_stack(halves, x, vectors=vectors[:1])
    bare = B200GatedFeedForward(128, 264, modulation=False, device="cuda")
    with pytest.raises(_lib.KsanaB200Error):
        bare(x, temb)
    with pytest.raises(_lib.KsanaB200Error):
        B200GatedFeedForward(128, 264, act="relu")
    layer = B200GatedFeedForward(128, 264, kind="layer", device="cuda")
    with pytest.raises(_lib.KsanaB200Error):
        gated_stack([halves[0], layer], x, vectors=vectors)


def test_served_with_an_fp8_down_projection_and_as_a_graph():
    halves, x, temb = _halves(2, 128, 272, torch.bfloat16, "rms", 5)
    with torch.no_grad():
        plain = gated_stack(halves, x, temb)
        for m in halves:
            m.down = B200Fp8Linear.from_float(m.down)
        ref = gated_stack(halves, x, temb)
        assert _off(ref, plain.double()) <= 0.05  # e4m3: half a step of 2^-3 per operand, over 272 products and a quarter of the residual sum
        for tokens in (1, 7):  # single tokens
            assert gated_stack(halves, x[:, :tokens].contiguous(), temb).shape == (2, tokens, 128)
        for m in halves:
            m.eval()
        graph, static = torch.cuda.CUDAGraph(), x.clone()
        gated_stack(halves, static, temb)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = gated_stack(halves, static, temb)
        static.copy_(2 * x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gated_stack(halves, 2 * x, temb))


def test_launches_are_counted_and_registered_operators_agree():
    import ksanadit_b200.torch_ops  # noqa: F401
    halves, x, temb = _halves(1, 128, 264, torch.bfloat16, "layer", 7)
    m = halves[0]
    with torch.no_grad():
        before = ops.STATS.kernels
        m(x, temb)
        assert ops.STATS.kernels == before + 4  # the modulation, two norms, the projections
        t = torch.ops.ksana_b200
        shift, scale, gate = m.vectors(temb)
        h = ops.gated_linear(x, m.w_gate, m.w_up, m.b_gate, m.b_up)
        assert torch.equal(t.gated_linear(x, m.w_gate, m.w_up, m.b_gate, m.b_up, "silu"), h)
        a = t.sandwich_norm(x, x, gate, scale, shift, m.post_norm, m.pre_norm, 0.5, "layer", 1e-6)
        b = ops.sandwich_norm(x, x, gate=gate, scale=scale, shift=shift, post_weight=m.post_norm, pre_weight=m.pre_norm, residual_scale=0.5, kind="layer")
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        w = m.modulation
        assert torch.equal(t.w4_linear(temb, w.weight, w.weight_scale, None, w.bias, 384), w(temb))


def test_the_same_tensor_twice():
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = (torch.randn(*s, device="cuda", generator=g).bfloat16() for s in ((70, 72), (136, 72)))
    x2, w2 = x.clone(), w.clone()
    for t in (x, w, x2, w2):
        t.requires_grad_(True)
    dh = torch.randn(70, 136, device="cuda", generator=g).bfloat16()
    h = ops.gated_linear(x, w, w)
    assert torch.equal(h, ops.gated_linear(x, w, w2))
    both = torch.autograd.grad(ops.gated_linear(x, w, w2), [x, w, w2], dh)
    one = torch.autograd.grad(h, [x, w], dh)
    assert torch.equal(one[0], both[0]) and torch.equal(one[1], both[1] + both[2])
    d = torch.randn(70, 72, device="cuda", generator=g).bfloat16()
    r, n = ops.sandwich_norm(x, x, gate=x[0], scale=x[0])
    r2, n2 = ops.sandwich_norm(x, x2, gate=x2[0], scale=x2[0])
    assert torch.equal(r, r2) and torch.equal(n, n2)
    one, two = torch.autograd.grad((r, n), [x], (d, d)), torch.autograd.grad((r2, n2), [x, x2], (d, d))
    # the parts are rounded sums in either order: a few half steps of the largest
    assert torch.allclose(one[0].float(), two[0].float() + two[1].float(), rtol=0, atol=4 * 2.0 ** -8 * float(two[1].abs().max() + two[0].abs().max()))


def test_threads_and_streams_at_once():
    """Calls of all three operators from several threads, each on its own stream, at the same time: nothing is shared between them."""
    import threading
    g = torch.Generator(device="cuda").manual_seed(6)
    w = [(torch.randn(520, 264, device="cuda", generator=g) * 0.1).bfloat16() for _ in range(2)]
    lin = B200W4Linear.from_float(torch.nn.Linear(264 - 264 % 32, 777, device="cuda"), 32)
    xs = [torch.randn(m, 264, device="cuda", generator=g).bfloat16() for m in (3, 33, 300, 900)]

    def run(x):
        x = x.detach().requires_grad_(True)
        h = ops.gated_linear(x, *w)
        r, n = ops.sandwich_norm(x, x * 0.5)
        with torch.no_grad():
            small = lin(x[:9, :256].contiguous())
        return [h.detach(), small, *torch.autograd.grad((h, r, n), [x], (h.detach(), r.detach(), n.detach()))]

    want = [run(x) for x in xs]
    torch.cuda.synchronize()
    got, failed = [None] * len(xs), []

    def worker(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = run(xs[i])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert all(torch.equal(a, b) for p, q in zip(want, got) for a, b in zip(p, q))
    _lib.assert_device_ok()


def test_checkpoint_hooks_and_transforms():
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(50, 72, device="cuda", generator=g).bfloat16().requires_grad_(True)
    w = [(torch.randn(136, 72, device="cuda", generator=g) * 0.1).bfloat16().requires_grad_(True) for _ in range(2)]

    def half(x, a, b):
        return ops.sandwich_norm(ops.gated_linear(x, a, b), kind="layer")[1]

    dh = torch.randn(50, 136, device="cuda", generator=g).bfloat16()
    want = torch.autograd.grad(half(x, *w), [x, *w], dh)
    got = torch.autograd.grad(checkpoint(half, x, *w, use_reentrant=False), [x, *w], dh)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.autograd.graph.save_on_cpu(pin_memory=False):
        h = half(x, *w)
    got = torch.autograd.grad(h, [x, *w], dh)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # transforms see no kernel they could follow: refused, in either pass
    h = half(x, *w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(h, [x], torch.stack([dh, dh]), is_grads_batched=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: half(v, *w))(torch.stack([x, x]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: half(v, *w).float().sum())(x)
    h = half(x, *w)
    with torch.no_grad():
        w[0].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, [x], dh)
    with torch.inference_mode():
        assert half(x, *w).shape == (50, 136)
