"""The forms that work from registers, where their loops over the depth turn: wave w of W takes every W-th piece of 128 bytes, loads
D pieces ahead and goes on in rounds of D, so a wave's share of the whole pieces is taken below D, at D, at 2 D - 1 and 2 D, at 3 D + 1
(W is 8 and D up to 4), each with nothing, a part and almost a whole piece behind the last one.  Operands whose rows start on
dwords and ones that have to be shifted; 8-bit sums are compared exactly, what lies between rows is poisoned."""
import math

import pytest
import torch

import clblas_amd as cb
from ffn_util import DTYPES, SUM, Buf, close, gated_want, normal, scales, whole
from gpu_util import debug_env

pytestmark = pytest.mark.gpu

PIECES = [1, 7, 8, 9, 24, 31, 32, 33, 56, 63, 64, 65, 96, 104]  # whole pieces of 128 bytes; a wave has 0 ... 13 of them
REST = [0, 1, 16, 33, 63]  # elements behind them (16 bits: of 64; 8 bits: twice that)


def aligned(K, size):
    """Padding up to rows of whole dwords, one dword between them."""
    return (-K * size % 4) // size + 4 // size


def shifted(K, size):
    """Padding that leaves rows off the dword grid, one byte (8 bits) or two (16 bits) further each."""
    return (1 - K) % 4 + 4 if size == 1 else (1 - K) % 2 + 2


def exact_sums(A, B):
    return A.mat.double() @ B.mat.double().t()


def i8_case(M, N, K, pad):
    A, B, C = (Buf(n, K, torch.int8, 0, pad(K, 1), whole(n, K, i), fill=127) for i, n in enumerate((M, N, N)))
    one = torch.ones(max(M, N), device="cuda")
    out = Buf(M, N, torch.float32)
    assert cb.i8gemm(cb.Type.F32, M, N, K, *A.args(), one, *B.args(), one, *out.args()) == 0
    want = exact_sums(A, B)
    assert float(want.abs().max()) < 2 ** 31
    torch.cuda.synchronize()
    assert torch.equal(out.mat, want.float()) and out.surroundings_untouched()  # (the sum, rounded to a float)
    # the gated product on them
    sx, sg, su = scales(M, 3).cuda(), (scales(N, 4) / math.sqrt(K)).cuda(), (scales(N, 5) / math.sqrt(K)).cuda()
    H = Buf(M, N, torch.bfloat16)
    assert cb.gated_i8(cb.Type.BF16, cb.Gate.Silu, M, N, K, *A.args(), sx, *B.args(), sg, *C.args(), su, *H.args()) == 0
    torch.cuda.synchronize()
    g = want * sx.double()[:, None] * sg.double()[None, :]
    u = exact_sums(A, C) * sx.double()[:, None] * su.double()[None, :]
    h, eh = gated_want(cb.Gate.Silu, g, u, g.abs() * 3 * 2.0 ** -24, u.abs() * 3 * 2.0 ** -24)
    close(H.mat, h, eh, torch.bfloat16)


def gated_case(type_, M, N, K, pad):
    d = DTYPES[type_]
    X = Buf(M, K, d, 0, pad(K, 2), normal(M, K, 1), fill=math.nan)
    Wg, Wu = (Buf(N, K, d, 0, pad(K, 2), normal(N, K, i, 1 / math.sqrt(K)), fill=math.nan) for i in (2, 3))
    H, G, U = (Buf(M, N, d) for _ in range(3))
    assert cb.gated(type_, cb.Gate.Silu, M, N, K, *X.args(), *Wg.args(), *Wu.args(), *H.args(), *G.args(), *U.args()) == 0
    torch.cuda.synchronize()
    x, wg, wu = X.mat.double(), Wg.mat.double(), Wu.mat.double()
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = K * SUM * (x.abs() @ wg.abs().t()), K * SUM * (x.abs() @ wu.abs().t())
    close(G.mat, g, eg, d)
    close(U.mat, u, eu, d)
    h, eh = gated_want(cb.Gate.Silu, g, u, eg, eu)
    close(H.mat, h, eh, d)


@pytest.mark.parametrize("pad", [aligned, shifted], ids=["aligned", "shifted"])
@pytest.mark.parametrize("form", [0, 1, 2, 3])
@pytest.mark.parametrize("M", [1, 17, 70])
def test_every_turn_of_the_loops(form, M, pad):
    N = 70
    with debug_env(CLBLAS_AMD_FFN_FORM=form):
        for i, pieces in enumerate(PIECES):
            rest = REST[(i + M) % len(REST)]
            i8_case(M, N, 128 * pieces + 2 * rest + (rest & 1), pad)
            gated_case(cb.Type.BF16 if i % 2 else cb.Type.F16, M, N, 64 * pieces + rest, pad)
            assert "rows_kernel" in cb.last_dispatch()[0]


@pytest.mark.parametrize("form", [0, 1, 2, 3])
def test_one_element_out_of_place_shows(form):
    """Each piece of the depth counts once: operands that are zero but for one 64-byte run, moved through all of it."""
    M, N, K = 5, 40, 64 * 67 + 11
    X, W = torch.zeros(M, K, dtype=torch.float16, device="cuda"), torch.ones(N, K, dtype=torch.float16, device="cuda")
    W *= torch.arange(1, N + 1, device="cuda").half()[:, None]
    H, G, U = (torch.empty(M, N, dtype=torch.float16, device="cuda") for _ in range(3))
    with debug_env(CLBLAS_AMD_FFN_FORM=form):
        for at in range(0, K, 32):
            X.zero_()
            X[:, at:at + 32] = 1.0
            n = min(32, K - at)
            assert cb.gated(cb.Type.F16, cb.Gate.Silu, M, N, K, X, 0, K, W, 0, K, W, 0, K, H, 0, N, G, 0, N, U, 0, N) == 0
            assert torch.equal(G, (n * torch.arange(1, N + 1, device="cuda")).half().expand(M, N))


@pytest.mark.parametrize("M,N,K", [(1, 12288, 4096), (1, 4096, 12288), (16, 1536, 4096), (8, 2048, 12345), (3, 1000, 6200)])
@pytest.mark.parametrize("pad", [lambda K, size: 0, aligned, shifted], ids=["none", "aligned", "shifted"])
def test_decoding_sizes_as_the_rule_chooses(M, N, K, pad):
    gated_case(cb.Type.BF16, M, N, K, pad)
    gated_case(cb.Type.F16, M, N, K, pad)
    i8_case(M, N, K, pad)
