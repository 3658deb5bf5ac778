"""Rows to 8-bit integers where the kernels change: lengths around what stays in registers (1024 for a wave, 8192 for a workgroup) and
around the numbers of rows and elements that choose between them, and ties at the ends of each type's range."""
import pytest
import torch

import clblas_amd as cb
from ffn_util import DTYPES, normal
from test_ffn_gpu import quantize

pytestmark = pytest.mark.gpu


def check(x, type_, off=0, pad=0):
    X, q, s = quantize(x, type_, off, pad)
    a = X.abs().amax(1, keepdim=True)
    assert torch.equal(q.double(), torch.where(a > 0, torch.round(127 * X / a), torch.zeros_like(X)))
    assert bool(((s.double() - a[:, 0] / 127).abs() <= 2.0 ** -24 * a[:, 0] / 127 + 2.0 ** -150).all())


@pytest.mark.parametrize("type_", list(cb.Type))
@pytest.mark.parametrize("M", [2047, 2048, 2050])
@pytest.mark.parametrize("K,pad", [(8, 0), (511, 1), (512, 0), (519, 0), (1016, 0), (1023, 2), (1024, 0), (1024, 3), (1025, 0), (1032, 0)])
def test_a_wave_or_a_workgroup_a_row(type_, M, K, pad):
    x = normal(M, K, M + K)
    x[::50, -1] = 9.0  # (the last element the largest)
    x[3], x[-1, 1:] = 0, 0
    check(x, type_, pad, pad)


@pytest.mark.parametrize("type_", list(cb.Type))
@pytest.mark.parametrize("K", [8184, 8191, 8192, 8193, 8200, 12288, 16391])
@pytest.mark.parametrize("place", [0, 0.5, 1])
def test_rows_longer_than_registers_hold(type_, K, place):
    x = normal(5, K, K)
    x[:, int((K - 1) * place)] = 7.0
    check(x, type_)


@pytest.mark.parametrize("type_", list(cb.Type))
def test_half_of_the_largest_number_is_a_tie(type_):
    """127 x / a = 63.5 exactly: halving is exact in every type, and the even neighbour is 64."""
    f = torch.finfo(DTYPES[type_])
    for a in (f.max, f.smallest_normal, 1.0, f.smallest_normal * f.eps * 2):
        x = torch.tensor([[a, a / 2, -a, -a / 2, 0.0]], dtype=torch.float64).to(DTYPES[type_])
        assert float(x[0, 1]) == a / 2
        _, q, _ = quantize(x, type_)
        assert q[0].tolist() == [127, 64, -127, -64, 0]
