"""Scales of 4-bit weights at the ends of the half types' ranges."""

import pytest
import torch

from ksanadit_b200 import _lib, ops, w4


def _weight(std, seed=0):
    return torch.randn(48, 256, generator=torch.Generator().manual_seed(seed)) * std


def _error(w, group, zeros, dtype):
    packed, scale, zero = w4.quantize_w4(w, group, zeros, dtype)
    assert bool(scale.isfinite().all()) and bool((scale > 0).all())
    return w4.dequantize_w4(packed, scale, zero, *w.shape) - w, scale


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("std", [1e-2, 1e-3, 1e-4, 3e-5, 1e-5, 1e-6, 2e-7])
def test_small_weights_keep_their_four_bits(std, zeros):
    w = _weight(std)
    least = 2.0 ** -24  # of fp16
    for group in (32, 128):
        err, scale = _error(w, group, zeros, torch.float16)
        g = w.view(48, -1, group)
        span = g.amax(-1).clamp(min=0) - g.amin(-1).clamp(max=0) if zeros else g.abs().amax(-1)
        # at most a step of fp16 above the exact scale; half a level off, and with a zero point its own half step as well
        step = span / (15 if zeros else 7) * (1 + 2.0 ** -11) + least
        room = (1.0 if zeros else 0.5) * step * (1 + 2.0 ** -20)
        assert bool((err.view_as(g).abs() <= room[..., None]).all())
        if std >= 1e-5:  # a scale of 50 of the least steps or more: the type's rounding is a hundredth
            wide, _ = _error(w, group, zeros, torch.bfloat16)
            assert float(err.norm()) <= 1.05 * float(wide.norm())


def test_zeros_and_lost_groups():
    w = _weight(0.02)
    w[3], w[7, :64] = 0, 1e-9  # a group that no fp16 scale holds, and that is nothing beside the others
    for zeros in (False, True):
        err, _ = _error(w, 64, zeros, torch.float16)
        assert bool((err[3] == 0).all()) and float(err[7, :64].abs().max()) <= 1e-9 + 2.0 ** -25
        with pytest.raises(_lib.KsanaB200Error, match="bfloat16"):
            w4.quantize_w4(_weight(1e-8), 64, zeros, torch.float16)
        with pytest.raises(_lib.KsanaB200Error, match="finite"):
            w4.quantize_w4(_weight(1e6), 64, zeros, torch.float16)
        for bad in (float("inf"), float("nan")):
            v = _weight(0.02)
            v[1, 1] = bad
            with pytest.raises(_lib.KsanaB200Error, match="finite"):
                w4.quantize_w4(v, 64, zeros)
        _error(_weight(1e-8), 64, zeros, torch.bfloat16)
    with pytest.raises(_lib.KsanaB200Error, match="bfloat16"):
        lin = torch.nn.Linear(64, 16)
        with torch.no_grad():
            lin.weight.mul_(1e-8)
        w4.B200W4Linear.from_float(lin, 64, dtype=torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("std,dtype", [(1e-5, torch.float16), (1e-6, torch.float16), (1e-30, torch.bfloat16)])
@pytest.mark.parametrize("zeros", [False, True])
def test_products_with_small_scales(std, dtype, zeros):
    w = _weight(std).cuda()
    packed, scale, zero = w4.quantize_w4(w, 64, zeros, dtype)
    x = (torch.randn(5, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 100).to(dtype)
    out = ops.w4_linear(x, packed, scale, zero, out_features=48)
    back = w4.dequantize_w4(packed, scale, zero, 48, 256).double()
    ref, size = x.double() @ back.T, x.double().abs() @ back.T.abs()
    # one rounding of the result, half a step of the type's least number where it is tiny, and the sum's (256 / 16 + 48 of 2^-22)
    f = torch.finfo(dtype)
    assert bool(((out.double() - ref).abs() <= f.eps / 2 * ref.abs() + f.smallest_normal * f.eps / 2 + 64 * 2.0 ** -22 * (1 + f.eps) * size).all())


def test_a_parameter_is_quantised_without_a_graph():
    lin = torch.nn.Linear(64, 16)
    for zeros in (False, True):
        parts = w4.quantize_w4(lin.weight, 64, zeros)
        assert not any(t is not None and t.requires_grad for t in parts)
        assert all(a is b or torch.equal(a, b) for a, b in zip(parts, w4.quantize_w4(lin.weight.detach(), 64, zeros)))


def test_values_of_more_than_four_bits_are_refused():
    q = torch.randint(0, 16, (17, 64), dtype=torch.uint8, generator=torch.Generator().manual_seed(0))
    q[16, 63] = 15
    w4.pack_w4(q)
    for bad in (16, 255):
        q[16, 63] = bad
        with pytest.raises(_lib.KsanaB200Error, match="15"):
            w4.pack_w4(q)
