"""Which calls take ROUND_TERMS, and what else may be added to a gate: nothing (no GPU: every call fails a check)."""
import pytest

import clblas_amd as cb
from test_ffn_api import gated, gated_grad, gated_i8


@pytest.mark.parametrize("fn", [gated, gated_i8])
@pytest.mark.parametrize("gate", list(cb.Gate))
def test_products_without_terms_refuse_it(fn, gate):
    assert fn(gate=gate + cb.ROUND_TERMS) == cb.Status.InvalidValue


@pytest.mark.parametrize("gate", [cb.ROUND_TERMS + 3, 0x200, 2 * cb.ROUND_TERMS + cb.ROUND_TERMS, -1, -1 - cb.ROUND_TERMS, 0x101000])
def test_gradients_refuse_gates_that_do_not_exist(gate):
    assert gated_grad(gate=gate) == cb.Status.InvalidValue


@pytest.mark.parametrize("gate", list(cb.Gate))
def test_gradients_check_the_rest_with_it_as_without(gate):
    for add in (0, cb.ROUND_TERMS):
        assert gated_grad(gate=gate + add, M=0) == cb.Status.InvalidDim
        assert gated_grad(gate=gate + add, lddx=6) == cb.Status.InvalidLeadDimC
        assert gated_grad(gate=gate + add, N=2 ** 20, lddh=2 ** 20, ldg=2 ** 20, ldu=2 ** 20) == cb.Status.NotImplemented
