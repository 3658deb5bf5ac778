"""The debug switches of the feed-forward products: values that name no form leave the choice to the rule."""
import pytest
import torch

import clblas_amd as cb
import test_ffn_gpu as products
from ffn_util import normal, scales, whole
from gpu_util import debug_env

pytestmark = pytest.mark.gpu


def outputs():
    M, N, K, d = 70, 90, 200, torch.bfloat16
    X, Wg, Wu, dH, G, U = (normal(r, c, i).to(d).cuda() for i, (r, c) in enumerate(((M, K), (N, K), (N, K), (M, N), (M, N), (M, N))))
    H, dX, dWg, dWu = (torch.full_like(t, 7) for t in (G, X, Wg, Wu))
    C = torch.full((M, N), 7.0, device="cuda")
    got = []
    assert cb.gated(cb.Type.BF16, cb.Gate.Silu, M, N, K, X, 0, K, Wg, 0, K, Wu, 0, K, H, 0, N) == 0
    got.append(cb.last_dispatch())
    assert cb.i8gemm(cb.Type.F32, M, N, K, whole(M, K, 1).cuda(), 0, K, scales(M, 3).cuda(), whole(N, K, 2).cuda(), 0, K, scales(N, 4).cuda(), C, 0, N) == 0
    got.append(cb.last_dispatch())
    for flags in (0, cb.ROUND_TERMS):
        assert cb.gated_grad(cb.Type.BF16, cb.Gate.Silu + flags, M, N, K, dH, 0, N, X, 0, K, Wg, 0, K, Wu, 0, K, G, 0, N, U, 0, N, dX, 0, K, dWg, 0, K,
                             dWu, 0, K) == 0
        got.append(cb.last_dispatch())
        got += [dX.clone(), dWg.clone(), dWu.clone()]
    torch.cuda.synchronize()
    return got + [H, C]


def same(a, b):
    return torch.equal(a, b) if torch.is_tensor(a) else a[0] == b[0]  # (what was launched; the count goes on)


@pytest.mark.parametrize("form", [9, 10, 100, 2 ** 31 - 1, -2, -100])
def test_a_form_that_does_not_exist_is_not_asked_for(form):
    want = outputs()
    with debug_env(CLBLAS_AMD_FFN_FORM=form):
        got = outputs()
    assert all(same(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("splits", [-1, 1, 1000, 2 ** 31 - 1])
def test_more_ranges_than_steps_are_one_a_step(splits):
    with debug_env(CLBLAS_AMD_FFN_SPLITS=splits):
        products.test_i8gemm(cb.Type.F32, 70, 90, 400, 0, 0)
        products.test_gated(cb.Type.F16, True, 70, 90, 200, 0, 0)
        products.test_gated_grad(cb.Type.BF16, 70, 90, 200, 0, 0)
        products.test_gated_grad(cb.Type.F16, 70, 90, 200, 0, 0)
