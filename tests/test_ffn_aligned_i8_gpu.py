"""8-bit operands that the tiles load from where they are (rows of whole dwords), with depths that end inside a 16-byte slot: what
lies behind a row - 127 in the gaps of both operands - must not reach a sum.  Compared with the exact integers."""
import math

import pytest
import torch

import clblas_amd as cb
from ffn_util import DTYPES, Buf, close, gated_want, scales, whole
from gpu_util import debug_env

pytestmark = pytest.mark.gpu

# M, N, K, leading dimension (a multiple of 4 beyond K)
SHAPES = [(70, 90, 129, 132), (33, 140, 450, 452), (130, 70, 97, 100), (257, 300, 127, 128), (64, 128, 1, 4), (5, 60, 15, 16), (300, 520, 911, 1000),
          (1000, 620, 130, 132), (128, 256, 255, 260)]


def operands(M, N, K, ld, n):
    return [Buf(r, K, torch.int8, 4, ld - K, whole(r, K, i), fill=127) for i, r in enumerate((M,) + (N,) * n)]


def launches_since(before):
    return cb.last_dispatch()[1] - before


@pytest.mark.parametrize("form", list(range(9)))
@pytest.mark.parametrize("splits", [0, 3])
def test_every_form(form, splits):
    with debug_env(CLBLAS_AMD_FFN_FORM=form, CLBLAS_AMD_FFN_SPLITS=splits):
        for M, N, K, ld in SHAPES:
            A, B, B2 = operands(M, N, K, ld, 2)
            one = torch.ones(max(M, N), device="cuda")
            sums, sums2 = A.mat.double() @ B.mat.double().t(), A.mat.double() @ B2.mat.double().t()
            C = Buf(M, N, torch.float32, 1, 3)
            before = cb.last_dispatch()[1]
            assert cb.i8gemm(cb.Type.F32, M, N, K, *A.args(), one, *B.args(), one, *C.args()) == 0
            # one launch, and one more that adds ranges up: no copy
            assert launches_since(before) == (2 if "join" in cb.last_dispatch()[0] else 1)
            torch.cuda.synchronize()
            assert torch.equal(C.mat.double(), sums) and C.surroundings_untouched()
            for type_ in cb.Type:
                sx, sg, su = scales(M, 3).cuda(), (scales(N, 4) / math.sqrt(K)).cuda(), (scales(N, 5) / math.sqrt(K)).cuda()
                H = Buf(M, N, DTYPES[type_], 1, 3)
                assert cb.gated_i8(type_, cb.Gate.Gelu, M, N, K, *A.args(), sx, *B.args(), sg, *B2.args(), su, *H.args()) == 0
                torch.cuda.synchronize()
                g, u = sums * sx.double()[:, None] * sg.double()[None, :], sums2 * sx.double()[:, None] * su.double()[None, :]
                h, eh = gated_want(cb.Gate.Gelu, g, u, g.abs() * 3 * 2.0 ** -24, u.abs() * 3 * 2.0 ** -24)
                close(H.mat, h, eh, DTYPES[type_])
                assert H.surroundings_untouched()


@pytest.mark.parametrize("form", [4, 5, 6, 7, 8])
def test_more_tiles_than_workgroups(form):
    M, N = (4300, 4500) if form == 4 else (3000, 3100)
    with debug_env(CLBLAS_AMD_FFN_FORM=form):
        for K, ld in ((97, 100), (259, 260)):
            A, B, B2 = operands(M, N, K, ld, 2)
            one = torch.ones(max(M, N), device="cuda")
            C = Buf(M, N, torch.float32)
            assert cb.i8gemm(cb.Type.F32, M, N, K, *A.args(), one, *B.args(), one, *C.args()) == 0
            sums, sums2 = A.mat.double() @ B.mat.double().t(), A.mat.double() @ B2.mat.double().t()
            torch.cuda.synchronize()
            assert torch.equal(C.mat.double(), sums)
            H, small = Buf(M, N, torch.float16), torch.full((max(M, N),), 2.0 ** -8, device="cuda")
            assert cb.gated_i8(cb.Type.F16, cb.Gate.Silu, M, N, K, *A.args(), one, *B.args(), small, *B2.args(), small, *H.args()) == 0
            torch.cuda.synchronize()
            g, u = sums * 2.0 ** -8, sums2 * 2.0 ** -8
            h, eh = gated_want(cb.Gate.Silu, g, u, torch.zeros_like(g), torch.zeros_like(u))
            close(H.mat, h, eh, torch.float16)


@pytest.mark.parametrize("M,N,K,ld", [(2048, 1000, 4096, 4096), (1000, 5003, 2501, 2508), (256, 1024, 4097, 4100), (16, 12288, 4096, 4096), (8192, 640, 130, 132)])
def test_as_the_rule_chooses(M, N, K, ld):
    A, B, B2 = operands(M, N, K, ld, 2)
    one = torch.ones(max(M, N), device="cuda")
    C = Buf(M, N, torch.float32)
    assert cb.i8gemm(cb.Type.F32, M, N, K, *A.args(), one, *B.args(), one, *C.args()) == 0
    assert "copy" not in cb.last_dispatch()[0]
    torch.cuda.synchronize()
    sums = A.mat.double() @ B.mat.double().t()
    assert torch.equal(C.mat, sums.float())
    sx, sg = scales(M, 3).cuda(), (scales(N, 4) / math.sqrt(K)).cuda()
    H = Buf(M, N, torch.bfloat16)
    assert cb.gated_i8(cb.Type.BF16, cb.Gate.GeluTanh, M, N, K, *A.args(), sx, *B.args(), sg, *B2.args(), sg, *H.args()) == 0
    torch.cuda.synchronize()
    s = sx.double()[:, None] * sg.double()[None, :]
    g, u = sums * s, (A.mat.double() @ B2.mat.double().t()) * s
    h, eh = gated_want(cb.Gate.GeluTanh, g, u, g.abs() * 3 * 2.0 ** -24, u.abs() * 3 * 2.0 ** -24)
    close(H.mat, h, eh, torch.bfloat16)
