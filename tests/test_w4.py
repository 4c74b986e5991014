"""CPU tests of the 4-bit weight format, the B200W4Linear contract and what ops.w4_linear and its C entry refuse."""

import pytest
import torch

from ksanadit_b200 import _lib, ops, w4


@pytest.mark.parametrize("N,K", [(1, 32), (16, 64), (37, 96), (45, 640)])
def test_packing_is_undone_and_places_are_those_of_the_format(N, K):
    q = torch.randint(0, 16, (N, K), dtype=torch.uint8, generator=torch.Generator().manual_seed(N + K))
    p = w4.pack_w4(q)
    assert p.shape == ((N + 15) // 16, (K + 63) // 64, 512) and torch.equal(w4.unpack_w4(p, N, K), q)
    for n, k in ((0, 0), (N - 1, K - 1), (N // 2, K // 3), (N - 1, 5), (N // 2, 7)):
        h, r, b, t, c = n % 16 // 8, n % 8, k % 64 // 32, k % 32 // 8, k % 8
        high = c in (2, 3, 6, 7)
        i = [0, 4, 1, 5].index(c - 2 if high else c)
        byte = int(p[n // 16, k // 64, (r * 4 + t) * 16 + 8 * b + 4 * h + i])
        assert (byte >> 4 if high else byte & 15) == int(q[n, k])


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantiser_is_off_by_half_a_step(zeros, group, dtype):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(40, 256, generator=g) * 0.02
    w[3] = 0
    w[5, :group] = w[5, :group].abs()
    packed, scale, zero = w4.quantize_w4(w, group, zeros, dtype)
    assert scale.dtype == dtype and (zero is not None) == zeros
    back = w4.dequantize_w4(packed, scale, zero, 40, 256)
    step = w4.untile_groups(scale, 40).double().repeat_interleave(group, 1)
    # half a step; at a group's ends half a rounding of the scale more, seven (fifteen) times, and with a zero point its own half step
    room = step * ((1.0 if zeros else 0.5) + 15 * torch.finfo(dtype).eps / 2) + 1e-9
    assert bool(((back.double() - w.double()).abs() <= room).all())
    assert bool((back[3] == 0).all())


def test_module_contract():
    m = w4.B200W4Linear(128, 40, group=64, zeros=True, dtype=torch.float16)
    assert set(m.state_dict()) == {"weight", "weight_scale", "weight_zero", "bias"}
    assert not any(p.requires_grad for p in m.parameters()) and m.reset_parameters() is None
    lin = torch.nn.Linear(128, 40)
    q = w4.B200W4Linear.from_float(lin, 64, True, torch.float16)
    m.load_state_dict(q.state_dict())
    assert torch.equal(m.dequantized(), q.dequantized())
    assert float((m.dequantized() - lin.weight).detach().abs().max()) < 0.02
    with pytest.raises(_lib.KsanaB200Error):
        m(torch.zeros(1, 128, dtype=torch.float16))  # CPU
    with pytest.raises(_lib.KsanaB200Error):
        w4.B200W4Linear(100, 40)
    with pytest.raises(TypeError):
        w4.B200W4Linear(128, 40, dtype=torch.float32)


def _args(M=2, N=40, K=128, group=64, dtype=torch.bfloat16):
    packed, scale, zero = w4.quantize_w4(torch.randn(N, K), group, True, dtype)
    return dict(x=torch.zeros(M, K, dtype=dtype), weight=packed, weight_scale=scale, weight_zero=zero, bias=torch.zeros(N, dtype=dtype), out_features=N)


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(2, 64, dtype=torch.bfloat16)), dict(x=torch.zeros(2, 128, dtype=torch.float16)), dict(out_features=33 + 16), dict(out_features=0),
    dict(weight=torch.zeros(3, 2, 256, dtype=torch.uint8)), dict(weight=torch.zeros(3, 2, 512, dtype=torch.int8)),
    dict(weight=torch.zeros(3, 2, 1024, dtype=torch.uint8)[..., ::2]),
    dict(weight_scale=torch.zeros(3, 2, 16)), dict(weight_scale=torch.zeros(3, 16, 16, dtype=torch.bfloat16)), dict(weight_scale=torch.zeros(3, 3, 16, dtype=torch.bfloat16)),
    dict(weight_zero=torch.zeros(3, 2, 16, dtype=torch.int32)), dict(weight_zero=torch.zeros(3, 1, 16, dtype=torch.uint8)),
    dict(bias=torch.zeros(41, dtype=torch.bfloat16)), dict(bias=torch.zeros(40)), dict(bias=torch.zeros(80, dtype=torch.bfloat16)[::2]),
    dict(x=torch.zeros(2, 128, dtype=torch.bfloat16, requires_grad=True)), dict()])
def test_refusals(change):
    with pytest.raises(_lib.KsanaB200Error):  # the last one: everything fits, but on the CPU
        ops.w4_linear(**{**_args(), **change})


def test_refused_types():
    with pytest.raises(TypeError):
        ops.w4_linear(**{**_args(), "x": torch.zeros(2, 128)})


def test_c_entry_refuses_before_any_launch():
    lib = _lib.load()
    p = 0x1000  # never read

    def call(x=p, dtype=0, M=1, K=128, ldx=128, w=p, s=p, z=None, group=64, N=16, out=p, ldo=16):
        return lib.ksb_w4_linear(x, dtype, M, K, ldx, w, s, z, group, None, N, out, ldo, None)

    assert call(M=0) == 0
    for bad in (dict(x=None), dict(w=None), dict(s=None), dict(out=None), dict(dtype=2), dict(group=16), dict(group=0), dict(K=100), dict(K=0), dict(N=0), dict(M=-1),
                dict(x=p + 2), dict(w=p + 8), dict(z=p + 4), dict(M=2, ldx=64), dict(M=2, ldx=132), dict(M=2, ldo=8)):
        assert call(**bad) == -1, bad
    assert call(K=32768 + 64) == -3
