"""How rows of ops.w4_linear are shared out over passes of the weight, and results where passes differ."""

import pytest
import torch
from test_gpu_w4 import _case, _check

from ksanadit_b200 import _lib, ops

pytestmark = pytest.mark.gpu


# (rows, N, K, group, zeros, passes): few row tiles and the longest K; many row tiles, whose sums take room in shared memory; passes of different sizes
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K,group,zeros,passes", [
    (16, 64, 32768, 128, False, 2), (16, 40, 32768, 32, True, 2), (9, 16, 30016, 32, True, 1), (35, 24, 32768, 64, True, 3), (16, 30720, 13824, 128, False, 2),
    (16, 30720, 13824, 32, True, 2), (16, 30720, 5120, 128, False, 1), (33, 9216, 1536, 64, True, 3), (13, 2000, 26112, 128, False, 1)])
def test_passes(M, N, K, group, zeros, passes, dtype):
    if N > 10000 and dtype == torch.float16:
        pytest.skip("one type is enough of the large ones")
    x, packed, scale, zero, bias = _case(M, N, K, group, zeros, dtype, M + N + K)
    before = ops.STATS.kernels
    out = ops.w4_linear(x, packed, scale, zero, bias, out_features=N)
    assert ops.STATS.kernels - before == passes
    _lib.assert_device_ok()
    _check(out, x, packed, scale, zero, bias, N, K)
    assert torch.equal(ops.w4_linear(x, packed, scale, zero, bias, out_features=N), out)
    # rows by themselves are the same to within the sums' roundings (the plan of the sums goes by the number of rows)
    _check(ops.w4_linear(x[3:5], packed, scale, zero, bias, out_features=N), x[3:5], packed, scale, zero, bias, N, K)
