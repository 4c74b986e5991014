"""CPU tests of the C entry's checks of modulation tensors with one row."""

import ctypes

import pytest

from ksanadit_b200 import _lib, native

P = 0x1000  # never read


@pytest.mark.parametrize("args,one_row", [(dict(gate_stride=16), 1), (dict(scale_stride=16), 2), (dict(shift_stride=16), 4), (dict(gate=None), 1), (dict(scale=None), 3),
                                          (dict(shift=None), 4), (dict(), 8), (dict(), -1)])
def test_one_row_belongs_to_a_tensor_with_one_row(args, one_row):
    a = native.NormArgs(P, P, P, P, P, P, P, P, 6, 16, 2, 16, 16, 0, 0, 0, 0, 0, 1e-6, 1.0)
    for k, v in args.items():
        setattr(a, k, v)
    g = native.NormGrads(P, P, P, P, P, P, P, P, P, 16, 16, one_row)
    assert _lib.load().ksb_sandwich_norm_backward(ctypes.byref(a), ctypes.byref(g), P, None) == -1
    assert b"one_row" in _lib.load().ksb_last_error()


def test_struct_is_the_headers():
    assert ctypes.sizeof(native.NormGrads) == 9 * 8 + 2 * 8 + 8
