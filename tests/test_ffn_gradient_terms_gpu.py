"""The terms that the gated product's gradients sum, dG = dH o U o act'(G) and dU = dH o act(G): no rounding or range of theirs
that a float would not have.  Every bound here leaves the terms themselves a relative error of 2^-15 in bf16 and 2^-20 in f16 (two 16-bit
numbers hold 16 and 21 bits, and the gate's functions are good to 2^-20) and, in f16, the last bit of the smaller number, 2^-38
of the largest term of the call; one 16-bit number is off by 2^-8 and 2^-11 (ROUND_TERMS, which asks for that)."""
import math

import pytest
import torch

import clblas_amd as cb
from ffn_util import DTYPES, FUNC, SUM, act, close, normal, slope

pytestmark = pytest.mark.gpu

GATES = list(cb.Gate)
HALVES = [cb.Type.BF16, cb.Type.F16]
TERM = {cb.Type.BF16: 2.0 ** -15, cb.Type.F16: 2.0 ** -20}


def gradients(type_, gate, dH, X, Wg, Wu, G, U, flags=0):
    M, N, K = X.shape[0], G.shape[1], X.shape[1]
    dX, dWg, dWu = (torch.full_like(t, 7) for t in (X, Wg, Wu))
    assert cb.gated_grad(type_, gate + flags, M, N, K, dH, 0, N, X, 0, K, Wg, 0, K, Wu, 0, K, G, 0, N, U, 0, N, dX, 0, K, dWg, 0, K, dWu, 0, K) == 0
    torch.cuda.synchronize()
    return dX, dWg, dWu


def check(type_, gate, dH, X, Wg, Wu, G, U, flags=0):
    """The call against the definitions in 64 bits; returns the largest term."""
    d = DTYPES[type_]
    dh, x, wg, wu, g, u = (t.double() for t in (dH, X, Wg, Wu, G, U))
    M, N = G.shape
    dg, du = dh * u * slope(gate, g), dh * act(gate, g)
    top = float(torch.maximum(dg.abs().max(), du.abs().max()))
    last = 2.0 ** -38 * top if type_ == cb.Type.F16 else 0.0
    rounded = (torch.finfo(d).eps / 2 * 1.01 if flags else TERM[type_]) + FUNC
    edg = dg.abs() * rounded + (dh * u).abs() * 2.0 ** -20 + last
    edu = du.abs() * rounded + dh.abs() * 2.0 ** -22 + last
    dX, dWg, dWu = gradients(type_, gate, dH, X, Wg, Wu, G, U, flags)
    # sums of 2 N (M) values, each of two products: the additions' steps, as in the other sums' bounds
    mags = (dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()
    close(dX, dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + 4 * N * SUM * mags, d)
    for got, v, e in ((dWg, dg, edg), (dWu, du, edu)):
        close(got, v.t() @ x, e.t() @ x.abs() + 2 * M * SUM * ((v.abs() + e).t() @ x.abs()), d)
    return top


def layer(type_, M, N, K, seed, dh=1.0, x=1.0, w=1.0, g=1.0, u=1.0):
    d = DTYPES[type_]
    sizes = ((M, N, dh), (M, K, x), (N, K, w), (N, K, w), (M, N, g), (M, N, u))
    return [(normal(r, c, seed + i) * s).to(d).cuda() for i, (r, c, s) in enumerate(sizes)]


SHAPES = [(1, 1, 1), (1, 700, 300), (3, 33, 31), (31, 64, 40), (32, 31, 64), (33, 96, 130), (65, 257, 70), (130, 129, 257), (300, 520, 190), (70, 1100, 2060)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("type_", HALVES)
def test_terms_are_not_rounded_to_sixteen_bits(type_, gate, M, N, K):
    check(type_, gate, *layer(type_, M, N, K, 10 * M + N))


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("type_", HALVES)
def test_terms_rounded_on_request(type_, M, N, K):
    gate = GATES[(M + N + K) % 3]
    case = layer(type_, M, N, K, 10 * M + N)
    check(type_, gate, *case, flags=cb.ROUND_TERMS)
    if M * N > 2000:  # (another computation: some last bits differ)
        assert any(not torch.equal(a, b) for a, b in zip(gradients(type_, gate, *case), gradients(type_, gate, *case, flags=cb.ROUND_TERMS)))


@pytest.mark.parametrize("form", [4, 5, 6, 7, 8])
@pytest.mark.parametrize("splits", [0, 2, 5])
@pytest.mark.parametrize("type_", HALVES)
def test_every_tile_and_ranges_of_depth_with_rounded_terms(type_, form, splits):
    from gpu_util import debug_env
    with debug_env(CLBLAS_AMD_FFN_FORM=form, CLBLAS_AMD_FFN_SPLITS=splits):
        for M, N, K in ((33, 160, 70), (200, 96, 130), (290, 330, 520)):
            check(type_, GATES[(form + splits) % 3], *layer(type_, M, N, K, form), flags=cb.ROUND_TERMS)


def test_f16_range_with_rounded_terms():
    for dh, u, x, w, g in ((200.0, 200.0, 1e-3, 1e-3, 4.0), (1e-5, 0.1, 100.0, 100.0, 0.5), (1e-6, 1e-3, 1e4, 1e4, 1e-3)):
        check(cb.Type.F16, cb.Gate.Silu, *layer(cb.Type.F16, 300, 90, 50, 3, dh=dh, u=u, x=x, w=w, g=g), flags=cb.ROUND_TERMS)


@pytest.mark.parametrize("type_", HALVES)
@pytest.mark.parametrize("side", ["dX", "dWg", "dWu"])
def test_what_is_left_of_sums_that_cancel(type_, side):
    """Pairs of terms (1 + h)^2 and -(1 + 2 h), of which 16 bits hold the second only: rounded to them the two would cancel."""
    d, h, n, K = DTYPES[type_], 2.0 ** -5 if type_ == cb.Type.BF16 else 2.0 ** -6, 64, 5
    dH, U, sign = (torch.ones(n, dtype=d, device="cuda") for _ in range(3))
    dH[::2], U[::2], U[1::2], sign[1::2] = 1 + h, 1 + h, 1 + 2 * h, -1
    # G = 64 U: far above zero act(G) = G and act'(G) = 1
    shape = (1, n) if side == "dX" else (n, 1)
    dH, U = dH.view(shape), U.view(shape)
    M, N = shape
    X, Wg, Wu = (torch.zeros(r, K, dtype=d, device="cuda") for r in (M, N, N))
    (Wg if side == "dX" else X)[:] = sign[:, None]
    dX, dWg, dWu = gradients(type_, cb.Gate.Silu, dH, X, Wg, Wu, 64 * U, U)
    dg, du = dH.double() * U.double(), dH.double() * 64 * U.double()
    got, want = {"dX": (dX, dg @ Wg.double()), "dWg": (dWg, dg.t() @ X.double()), "dWu": (dWu, du.t() @ X.double())}[side]
    size = n * (1 + h) ** 2 * (64 if side == "dWu" else 1)
    err = size * (TERM[type_] + FUNC + 2 * n * SUM)
    assert float(want.abs().min()) > 2 * err  # (zero is not within the bound)
    close(got, want, torch.full_like(want, err), d)


# ---- the range of f16: terms beyond 65504 and below 2^-24 whose sums are in range ----

@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (70, 90, 50), (300, 520, 190)])
def test_f16_terms_above_the_largest_number(gate, M, N, K):
    top = check(cb.Type.F16, gate, *layer(cb.Type.F16, M, N, K, 3, dh=200.0, u=200.0, x=1e-3, w=1e-3, g=4.0))
    assert top > 65504 or M == 1


def test_f16_one_term_above_the_largest_number():
    f = lambda v: torch.full((1, 1), v, dtype=torch.float16, device="cuda")  # noqa: E731
    dX, dWg, dWu = gradients(cb.Type.F16, cb.Gate.Silu, f(300.0), f(0.01), f(0.01), f(0.0), f(4.0), f(300.0))
    g = torch.tensor(4.0, dtype=torch.float64)
    x = float(f(0.01))
    want = 90000 * float(slope(cb.Gate.Silu, g)) * x
    for got in (dX, dWg):
        assert abs(float(got) - want) <= want * (2.0 ** -11 + 2.0 ** -18)
    want = 300 * float(act(cb.Gate.Silu, g)) * x
    assert abs(float(dWu) - want) <= want * (2.0 ** -11 + 2.0 ** -18)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (70, 90, 50), (2000, 70, 60)])
def test_f16_terms_below_the_smallest_number(gate, M, N, K):
    top = check(cb.Type.F16, gate, *layer(cb.Type.F16, M, N, K, 4, dh=1e-5, u=0.1, x=100.0, w=100.0, g=0.5))
    assert top < 2.0 ** -13
    top = check(cb.Type.F16, gate, *layer(cb.Type.F16, M, N, K, 5, dh=1e-6, u=1e-3, x=1e4, w=1e4, g=1e-3))
    assert top < 2.0 ** -25


def test_f16_tokens_of_very_different_size():
    dH, X, Wg, Wu, G, U = layer(cb.Type.F16, 200, 130, 90, 6, w=0.1)
    dH *= torch.logspace(-6, 3, 200, dtype=torch.float64).half().cuda()[:, None]
    dH[7], dH[11:90] = 0, 0
    check(cb.Type.F16, cb.Gate.Gelu, dH, X, Wg, Wu, G, U)


@pytest.mark.parametrize("type_", HALVES)
def test_gradients_of_nothing_are_zero(type_):
    dH, X, Wg, Wu, G, U = layer(type_, 40, 50, 30, 7)
    for t in gradients(type_, cb.Gate.GeluTanh, dH.zero_(), X, Wg, Wu, G, U):
        assert not t.any()


# ---- values that are not finite ----

@pytest.mark.parametrize("type_", HALVES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_one_token_that_is_not_finite_leaves_the_others(type_, bad):
    dH, X, Wg, Wu, G, U = layer(type_, 70, 90, 50, 8)
    clean, _, _ = gradients(type_, cb.Gate.Silu, dH, X, Wg, Wu, G, U)
    dH[5, 3] = bad
    dX, dWg, dWu = gradients(type_, cb.Gate.Silu, dH, X, Wg, Wu, G, U)
    assert not torch.isfinite(dX[5]).any()
    rest = [i for i in range(70) if i != 5]
    # (without that token's terms f16's common power of two may be another one: a last bit then)
    assert bool(((dX[rest] - clean[rest]).abs() <= clean[rest].abs() * torch.finfo(DTYPES[type_]).eps + 1e-4).all())
    for t in (dWg, dWu):
        assert not torch.isfinite(t[3]).any()
        assert bool(torch.isfinite(torch.cat([t[:3], t[4:]])).all())


@pytest.mark.parametrize("type_", HALVES)
def test_infinite_operands_give_infinities_where_a_float_would(type_):
    """A term times infinity is infinite with the term's sign, and no NaN, whether or not 16 bits hold the term."""
    d = DTYPES[type_]
    dH, U = torch.tensor([[1.0, 1.25, -3.0, 1 + 2.0 ** -7]], dtype=d, device="cuda").t(), torch.tensor([[1.0, 2.0, 1.0, 1 + 2.0 ** -6]], dtype=d, device="cuda").t()
    for m in range(4):
        X = torch.ones(1, 3, dtype=d, device="cuda")
        X[0, 1] = math.inf
        W = torch.full((1, 3), 0.5, dtype=d, device="cuda")
        one = torch.full((1, 1), 64.0, dtype=d, device="cuda")
        dX, dWg, dWu = gradients(type_, cb.Gate.Silu, dH[m:m + 1].contiguous(), X, W, W, one, U[m:m + 1].contiguous())
        sign = -1.0 if m == 2 else 1.0
        for t in (dWg, dWu):
            assert float(t[0, 1]) == sign * math.inf and bool(torch.isfinite(t[0, [0, 2]]).all())
        assert bool(torch.isfinite(dX).all())


# ---- strides, streams and graphs ----

def test_f16_scale_does_not_look_between_the_rows():
    """Infinities, NaN and large numbers in the gaps of dH, G and U; the common power of two comes from the rows alone."""
    from ffn_util import Buf
    M, N, K, d = 37, 45, 60, torch.float16
    dH, X, Wg, Wu, G, U = layer(cb.Type.F16, M, N, K, 9, dh=1e-5, u=0.1, x=100.0, w=100.0)
    want = gradients(cb.Type.F16, cb.Gate.Silu, dH, X, Wg, Wu, G, U)
    for fill in (math.nan, math.inf, 60000.0):
        b = [Buf(M, N, d, 3, 5, t, fill=fill) for t in (dH, G, U)]
        got = [torch.full_like(t, 7) for t in (X, Wg, Wu)]
        dx, dwg, dwu = got
        assert cb.gated_grad(cb.Type.F16, cb.Gate.Silu, M, N, K, *b[0].args(), X, 0, K, Wg, 0, K, Wu, 0, K, *b[1].args(), *b[2].args(),
                             dx, 0, K, dwg, 0, K, dwu, 0, K) == 0
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))


@pytest.mark.parametrize("type_", HALVES)
@pytest.mark.parametrize("M,N,K,flags", [(3, 5003, 1030, 0), (130, 300, 200, 0), (520, 700, 640, 0), (130, 300, 200, cb.ROUND_TERMS)])
def test_a_replayed_graph_follows_its_inputs(type_, M, N, K, flags):
    """Replays on other data of another size (f16: another power of two), eager work of the same stream between them."""
    dH, X, Wg, Wu, G, U = layer(type_, M, N, K, 12, w=0.05)
    keep = dH.clone()
    dX, dWg, dWu = (torch.empty_like(t) for t in (X, Wg, Wu))
    stream = torch.cuda.Stream()

    def run():
        assert cb.gated_grad(type_, cb.Gate.Gelu + flags, M, N, K, dH, 0, N, X, 0, K, Wg, 0, K, Wu, 0, K, G, 0, N, U, 0, N, dX, 0, K, dWg, 0, K, dWu, 0, K) == 0

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run()
    for size in (1.0, 2.0 ** -9, 2.0 ** 4, 0.0, 1.0):
        dH.copy_(keep * size)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            run()
        stream.synchronize()
        want = [t.clone() for t in (dX, dWg, dWu)]
        for t in (dX, dWg, dWu):
            t.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((dX, dWg, dWu), want))


@pytest.mark.parametrize("form", [4, 5, 6, 7, 8])
@pytest.mark.parametrize("splits", [0, 1, 2, 5])
@pytest.mark.parametrize("type_", HALVES)
def test_every_tile_and_ranges_of_depth(type_, form, splits):
    """Ranges that end inside dG's part and inside dU's, on the border between them, and one step long."""
    from gpu_util import debug_env
    with debug_env(CLBLAS_AMD_FFN_FORM=form, CLBLAS_AMD_FFN_SPLITS=splits):
        for M, N, K in ((33, 160, 70), (200, 96, 130), (290, 330, 520)):
            check(type_, GATES[(form + splits) % 3], *layer(type_, M, N, K, form))


@pytest.mark.parametrize("which", ["x", "w"])
@pytest.mark.parametrize("type_", HALVES)
@pytest.mark.parametrize("M,N,K", [(1, 3000, 1030), (40, 2100, 1500), (1100, 1300, 900), (2100, 600, 2300)])
def test_one_side_alone_equals_a_float_sum_too(type_, which, M, N, K):
    d = DTYPES[type_]
    dH, X, Wg, Wu, G, U = layer(type_, M, N, K, 13, w=0.05)
    dX, dWg, dWu = (torch.full_like(t, 7) for t in (X, Wg, Wu))
    none = (None, 0, 0)
    assert cb.gated_grad(type_, cb.Gate.Silu, M, N, K, dH, 0, N, X, 0, K, Wg, 0, K, Wu, 0, K, G, 0, N, U, 0, N,
                         *((dX, 0, K) if which == "x" else none), *((dWg, 0, K, dWu, 0, K) if which == "w" else none + none)) == 0
    torch.cuda.synchronize()
    dh, x, wg, wu, g, u = (t.double() for t in (dH, X, Wg, Wu, G, U))
    dg, du = dh * u * slope(cb.Gate.Silu, g), dh * act(cb.Gate.Silu, g)
    e = TERM[type_] + FUNC
    if which == "x":
        mags = dg.abs() @ wg.abs() + du.abs() @ wu.abs()
        extra = ((dh * u).abs() @ wg.abs()) * 2.0 ** -20 + (dh.abs() @ wu.abs()) * 2.0 ** -22
        close(dX, dg @ wg + du @ wu, mags * (e + 4 * N * SUM) + extra, d)
    for t, v, r in ((dWg, dg, (dh * u).abs() * 2.0 ** -20), (dWu, du, dh.abs() * 2.0 ** -22)):
        if which == "w":
            close(t, v.t() @ x, (v.abs().t() @ x.abs()) * (e + 2 * M * SUM) + r.t() @ x.abs(), d)
        else:
            assert bool((t == 7).all())
    assert which == "x" or bool((dX == 7).all())


@pytest.mark.parametrize("type_", HALVES)
@pytest.mark.parametrize("flags", [0, cb.ROUND_TERMS])
def test_the_workspace_that_the_header_states_is_enough_and_needed(type_, flags):
    """Sums in one piece: the gemm buffer holds the terms alone."""
    from gpu_util import debug_env
    M, N, K = 2000, 1000, 64
    need = (4 * M * 1024 if flags else 8 * M * 1024) + 5 * 1024
    dH, X, Wg, Wu, G, U = layer(type_, M, N, K, 14, w=0.05)
    dX, dWg, dWu = (torch.full_like(t, 7) for t in (X, Wg, Wu))
    for bytes_, want in ((need - 16384, cb.Status.InvalidOperation), (need, 0)):
        stream = torch.cuda.Stream()
        assert cb.release_stream(stream) == 0
        assert cb.reserve_workspace(gemm_bytes=bytes_, stream=stream) == 0
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with debug_env(CLBLAS_AMD_FFN_SPLITS=1), torch.cuda.graph(graph, stream=stream):
            st = cb.gated_grad(type_, cb.Gate.Silu + flags, M, N, K, dH, 0, N, X, 0, K, Wg, 0, K, Wu, 0, K, G, 0, N, U, 0, N, dX, 0, K, dWg, 0, K, dWu, 0, K)
        assert st == want
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool((t == 7).all()) == (want != 0) for t in (dX, dWg, dWu))
        del graph
        assert cb.release_stream(stream) == 0
    for got, again in zip((dX, dWg, dWu), gradients(type_, cb.Gate.Silu, dH, X, Wg, Wu, G, U, flags)):
        assert bool(((got.double() - again.double()).abs() <= again.double().abs() * 2.0 ** -7 + 1e-2).all())


@pytest.mark.parametrize("size", [2.0 ** 14, 1.0, 2.0 ** -10, 2.0 ** -17, 2.0 ** -26, 2.0 ** -37])
def test_f16_terms_that_sixteen_bits_hold_stay_exact(size):
    """One token of a call whose terms are short and `size`, the largest being 2^15, in sums that are short: nothing is added to them.
    (They are multiplied by 1/2, so from 2^-23 on the smallest f16 holds them; below that they are off by 2^-38 of the largest.)"""
    d = torch.float16
    M, N, K = 3, 4, 6
    f = lambda r, c, v: torch.full((r, c), v, dtype=d, device="cuda")  # noqa: E731
    dH, U, G = f(M, N, 2.0 ** 8), f(M, N, 2.0 ** 7), f(M, N, 64.0)
    half = 2.0 ** (math.floor(math.log2(size)) // 2)
    dH[1], U[1] = half, size / half
    X, Wg, Wu = f(M, K, 1.0), f(N, K, 0.0), f(N, K, 0.0)
    Wg[0], Wg[1], Wg[2] = 2.0 ** 13, 2.0 ** 12, 2.0 ** 4
    dX, _, _ = gradients(cb.Type.F16, cb.Gate.Silu, dH, X, Wg, Wu, G, U)
    want = size * (2.0 ** 13 + 2.0 ** 12 + 2.0 ** 4)
    exact = float(torch.tensor(want, dtype=torch.float64).half())
    off = 0.0 if size >= 2.0 ** -23 else 2.0 ** -38 * 2.0 ** 15 * want / size
    assert want > 65504 or all(abs(x - exact) <= off for x in dX[1].tolist())
