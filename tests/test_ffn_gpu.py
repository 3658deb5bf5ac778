"""The products of a gated feed-forward layer against their definitions in 64 bits, through the C ABI."""
import math

import pytest
import torch

import clblas_amd as cb
from ffn_util import (DTYPES, FUNC, SUM, Buf, act, close, gated_want, half_step, normal, scales, slope, whole)

pytestmark = pytest.mark.gpu

GATES = list(cb.Gate)
HALVES = [cb.Type.BF16, cb.Type.F16]
# M, N, K, offset, padding: single tokens and elements, edges of tiles and of their 16-byte pieces, odd sizes and strides
SHAPES = [
    (1, 1, 1, 0, 0), (1, 16, 16, 0, 0), (1, 40, 64, 0, 8), (2, 3, 5, 1, 3), (5, 129, 17, 3, 0), (8, 1000, 512, 0, 0), (16, 256, 2048, 0, 16),
    (17, 33, 130, 0, 2), (31, 65, 1024, 2, 6), (33, 300, 96, 0, 0), (64, 64, 64, 0, 0), (65, 200, 4096, 0, 0), (100, 90, 8200, 0, 0),
    (128, 128, 128, 0, 0), (127, 255, 144, 4, 4), (129, 257, 333, 1, 1), (256, 512, 256, 0, 0), (300, 1100, 520, 0, 8), (513, 771, 1030, 0, 0),
    (1030, 2052, 72, 0, 0), (2100, 4200, 200, 8, 8),
]
IDS = ["%dx%dx%d+%d+%d" % s for s in SHAPES]


def cuda64(x):
    return x.cuda().double()


# ---- rows to 8-bit integers ----

def quantize(x, type_, off=0, pad=0):
    X = Buf(*x.shape, DTYPES[type_], off, pad, x)
    Q = Buf(*x.shape, torch.int8, off + 1, pad + 2)
    s = torch.full((x.shape[0] + 1,), -5.0, device="cuda")
    assert cb.quantize_rows(type_, *x.shape, *X.args(), *Q.args(), s) == 0
    torch.cuda.synchronize()
    assert Q.surroundings_untouched() and float(s[-1]) == -5.0
    return X.mat.double(), Q.mat, s[:-1]


@pytest.mark.parametrize("type_", list(cb.Type))
@pytest.mark.parametrize("M,K,off,pad", [(1, 1, 0, 0), (3, 7, 1, 2), (5, 8, 0, 0), (2, 511, 3, 1), (64, 1024, 0, 0), (9, 8191, 0, 5), (4, 8200, 0, 0),
                                         (3, 20011, 1, 0), (300, 130, 0, 6)])
def test_quantize_rows(type_, M, K, off, pad):
    x = normal(M, K, 11 * M + K)
    x[:, ::3] *= 9
    if M > 2:
        x[1] = 0
    X, q, s = quantize(x, type_, off, pad)
    a = X.abs().amax(1, keepdim=True)
    # the quotient in 64 bits never lands on a half that is none: halves differ from others by more than 2^-33 of them
    want = torch.where(a > 0, torch.round(127 * X / a), torch.zeros_like(X))
    assert torch.equal(q.double(), want)
    assert bool(((s.double() - a[:, 0] / 127).abs() <= 2.0 ** -24 * a[:, 0] / 127 + 2.0 ** -150).all())


@pytest.mark.parametrize("type_", list(cb.Type))
@pytest.mark.parametrize("M,K,off,pad", [(2048, 1, 0, 0), (5003, 130, 1, 3), (2051, 1024, 0, 0), (4099, 1023, 1, 0), (4098, 7, 0, 1)])
def test_quantize_many_short_rows(type_, M, K, off, pad):
    x = normal(M, K, 7 * M + K)
    x[5::97] = 0
    X, q, s = quantize(x, type_, off, pad)
    a = X.abs().amax(1, keepdim=True)
    assert torch.equal(q.double(), torch.where(a > 0, torch.round(127 * X / a), torch.zeros_like(X)))
    assert bool(((s.double() - a[:, 0] / 127).abs() <= 2.0 ** -24 * a[:, 0] / 127 + 2.0 ** -150).all())


@pytest.mark.parametrize("type_", list(cb.Type))
def test_quantize_rows_ties_go_to_even(type_):
    # a = 127 / 8: every x = (n + 1/2) / 8 is a tie; a = 96 and 250: only a / 2 is one (63.5 -> 64)
    n = torch.arange(-127, 127, dtype=torch.float32)
    rows = torch.zeros(3, 256)
    rows[0, :254], rows[0, 255] = (n + 0.5) / 8, 127 / 8
    rows[1, :4] = torch.tensor([96.0, 48.0, -48.0, 47.75])
    rows[2, :4] = torch.tensor([-250.0, 125.0, -125.0, 124.0])
    _, q, _ = quantize(rows, type_)
    assert torch.equal(q[0, :254].cpu().double(), torch.round(n.double() + 0.5)) and int(q[0, 255]) == 127
    assert q[1, :4].tolist() == [127, 64, -64, 63] and q[2, :4].tolist() == [-127, 64, -64, 63]


@pytest.mark.parametrize("type_", list(cb.Type))
def test_quantize_rows_of_extremes(type_):
    f = torch.finfo(DTYPES[type_])
    tiny = f.smallest_normal * f.eps
    rows = torch.tensor([[f.max, f.max / 2, -f.max, 0.0], [tiny, 0.0, -tiny, 0.0], [2 * tiny, tiny, -tiny, 0.0], [f.smallest_normal, tiny, 0.0, -0.0],
                         [1.0, math.inf, 2.0, 3.0], [1.0, math.nan, 2.0, 3.0], [math.nan, math.inf, -math.inf, 0.0], [1.0, -math.inf, 0.0, 0.0]],
                        dtype=torch.float64).to(DTYPES[type_])
    _, q, s = quantize(rows.cpu(), type_)
    assert q[0].tolist() == [127, 64, -127, 0] or q[0].tolist() == [127, 63, -127, 0]  # (max / 2 rounds to either side in its type)
    assert q[1].tolist() == [127, 0, -127, 0] and q[2].tolist() == [127, 64, -64, 0]
    assert q[3].tolist() == [127, int(torch.round(torch.tensor(127 * f.eps, dtype=torch.float64))), 0, 0]
    assert not q[4:].any()
    assert math.isinf(s[4]) and math.isnan(s[5]) and math.isnan(s[6]) and math.isinf(s[7])


# ---- 8-bit product ----

@pytest.mark.parametrize("M,N,K,off,pad", SHAPES, ids=IDS)
@pytest.mark.parametrize("type_", list(cb.Type))
def test_i8gemm(type_, M, N, K, off, pad):
    A, B = Buf(M, K, torch.int8, off, pad, whole(M, K, 1)), Buf(N, K, torch.int8, off, pad, whole(N, K, 2))
    sa, sb = scales(M, 3).cuda(), scales(N, 4).cuda()
    C = Buf(M, N, DTYPES[type_], off, pad)
    assert cb.i8gemm(type_, M, N, K, *A.args(), sa, *B.args(), sb, *C.args()) == 0
    torch.cuda.synchronize()
    want = (A.mat.double() @ B.mat.double().t()) * sa.double()[:, None] * sb.double()[None, :]
    close(C.mat, want, want.abs() * 3 * 2.0 ** -24, DTYPES[type_])  # int32 -> float and two products
    assert C.surroundings_untouched()


def test_i8gemm_deepest_sum_of_the_largest_products():
    K = 131071
    A, B = torch.full((3, K), -128, dtype=torch.int8, device="cuda"), torch.full((20, K), -128, dtype=torch.int8, device="cuda")
    B[7] = 127
    one = torch.ones(20, device="cuda")
    C = torch.empty(3, 20, device="cuda")
    assert cb.i8gemm(cb.Type.F32, 3, 20, K, A, 0, K, one, B, 0, K, one, C, 0, 20) == 0
    want = torch.full((3, 20), float(2 ** 14 * K), dtype=torch.float64, device="cuda")
    want[:, 7] = -128.0 * 127 * K
    assert torch.equal(C.double(), want.float().double())
    assert cb.i8gemm(cb.Type.F32, 3, 20, K + 1, A, 0, K + 1, one, B, 0, K + 1, one, C, 0, 20) == cb.Status.NotImplemented


def test_i8gemm_passes_scales_that_are_not_finite_on():
    A, B = whole(4, 64, 1).cuda(), whole(6, 64, 2).cuda()
    sa, sb = scales(4, 3).cuda(), scales(6, 4).cuda()
    sa[1], sa[2] = math.nan, 0.0
    C = torch.empty(4, 6, device="cuda")
    assert cb.i8gemm(cb.Type.F32, 4, 6, 64, A, 0, 64, sa, B, 0, 64, sb, C, 0, 6) == 0
    assert bool(torch.isnan(C[1]).all()) and bool((C[2] == 0).all()) and bool(torch.isfinite(C[[0, 3]]).all())


# ---- gated product ----

def layer(type_, M, N, K, off, pad, seed=5):
    d = DTYPES[type_]
    X = Buf(M, K, d, off, pad, normal(M, K, seed))
    Wg = Buf(N, K, d, off, pad, normal(N, K, seed + 1, 1.5 / math.sqrt(K)))
    Wu = Buf(N, K, d, off + 1, pad + 1, normal(N, K, seed + 2, 1.0 / math.sqrt(K)))
    return X, Wg, Wu


@pytest.mark.parametrize("M,N,K,off,pad", SHAPES, ids=IDS)
@pytest.mark.parametrize("type_,save", [(cb.Type.BF16, False), (cb.Type.BF16, True), (cb.Type.F16, True)])
def test_gated(type_, save, M, N, K, off, pad):
    d, gate = DTYPES[type_], GATES[(M + N + K) % 3]
    X, Wg, Wu = layer(type_, M, N, K, off, pad)
    if (off, pad) == (0, 0):
        Wu = Buf(N, K, d, 0, 0, Wu.mat)  # every operand where the kernels can load it from
    H, G, U = (Buf(M, N, d, off, pad) for _ in range(3))
    st = cb.gated(type_, gate, M, N, K, *X.args(), *Wg.args(), *Wu.args(), *H.args(), *((*G.args(), *U.args()) if save else ()))
    assert st == 0
    torch.cuda.synchronize()
    x, wg, wu = X.mat.double(), Wg.mat.double(), Wu.mat.double()
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = K * SUM * (x.abs() @ wg.abs().t()), K * SUM * (x.abs() @ wu.abs().t())
    if save:
        close(G.mat, g, eg, d)
        close(U.mat, u, eu, d)
    h, eh = gated_want(gate, g, u, eg, eu)
    close(H.mat, h, eh, d)
    for b in (H, G, U):
        assert b.surroundings_untouched()


@pytest.mark.parametrize("gate", GATES)
def test_gated_over_the_gates_range(gate):
    """G runs from far below to far above zero, where the functions saturate (one term per sum)."""
    g = torch.cat([torch.linspace(-30, 30, 601), torch.tensor([-3e38, -1e30, -200.0, -100.0, -88.5, 88.5, 100.0, 1e30, 3e38])]).bfloat16()
    M = g.numel()
    X = torch.zeros(M, 32, dtype=torch.bfloat16)
    X[:, 0], X[:, 1] = g, 1.0
    Wg, Wu = torch.zeros(16, 32, dtype=torch.bfloat16), torch.zeros(16, 32, dtype=torch.bfloat16)
    Wg[:, 0], Wu[:, 1] = 1.0, 1.0
    X, Wg, Wu = X.cuda(), Wg.cuda(), Wu.cuda()
    H = torch.empty(M, 16, dtype=torch.bfloat16, device="cuda")
    assert cb.gated(cb.Type.BF16, gate, M, 16, 32, X, 0, 32, Wg, 0, 32, Wu, 0, 32, H, 0, 16) == 0
    x = g.cuda().double()
    want = act(gate, x)
    # in float an argument of the exponential is off by 3 units in its last place, and the value by that times its size
    arg = x.abs() if gate == cb.Gate.Silu else (x * x if gate == cb.Gate.Gelu else 1.6 * (x.abs() + 0.0448 * x.abs() ** 3))
    rel = FUNC + 2.0 ** -22 * torch.clamp(arg, max=110.0)
    err = want.abs() * rel + 1e-36 * x.abs().clamp(max=1e3)  # below 2^-126 the reciprocal of the exponential gives zero
    for c in (0, 15):
        close(H[:, c], want, err, torch.bfloat16)


def test_gated_passes_nan_on_to_its_rows_and_columns_only():
    X, Wg, Wu = (t.bfloat16().cuda() for t in (normal(70, 200, 1), normal(90, 200, 2), normal(90, 200, 3)))
    X[5, 199], Wu[7, 0] = math.nan, math.inf
    H = torch.empty(70, 90, dtype=torch.bfloat16, device="cuda")
    assert cb.gated(cb.Type.BF16, cb.Gate.Silu, 70, 90, 200, X, 0, 200, Wg, 0, 200, Wu, 0, 200, H, 0, 90) == 0
    ok = torch.isfinite(H)
    assert not ok[5].any() and not ok[:, 7].any()
    ok[5], ok[:, 7] = True, True
    assert bool(ok.all())


@pytest.mark.parametrize("M,N,K,off,pad", SHAPES, ids=IDS)
@pytest.mark.parametrize("type_", list(cb.Type))
def test_gated_i8(type_, M, N, K, off, pad):
    gate = GATES[(M + N + K + int(type_)) % 3]
    X, Wg, Wu = (Buf(n, K, torch.int8, off, pad, whole(n, K, i)) for i, n in enumerate((M, N, N)))
    sx, sg, su = scales(M, 3).cuda(), (scales(N, 4) / math.sqrt(K)).cuda(), (scales(N, 5) / math.sqrt(K)).cuda()
    H = Buf(M, N, DTYPES[type_], off, pad)
    assert cb.gated_i8(type_, gate, M, N, K, *X.args(), sx, *Wg.args(), sg, *Wu.args(), su, *H.args()) == 0
    torch.cuda.synchronize()
    g = (X.mat.double() @ Wg.mat.double().t()) * sx.double()[:, None] * sg.double()[None, :]
    u = (X.mat.double() @ Wu.mat.double().t()) * sx.double()[:, None] * su.double()[None, :]
    h, eh = gated_want(gate, g, u, g.abs() * 3 * 2.0 ** -24, u.abs() * 3 * 2.0 ** -24)
    close(H.mat, h, eh, DTYPES[type_])
    assert H.surroundings_untouched()


# ---- gradients ----

def grad_case(type_, gate, M, N, K, off, pad, which="xw", seed=5):
    d = DTYPES[type_]
    X, Wg, Wu = layer(type_, M, N, K, off, pad, seed)
    G, U, dH = (Buf(M, N, d, off, pad, normal(M, N, seed + 3 + i, s)) for i, s in enumerate((1.5, 1.0, 1.0)))
    dX, dWg, dWu = Buf(M, K, d, off, pad), Buf(N, K, d, off, pad), Buf(N, K, d, off, pad)
    none = (None, 0, 0)
    st = cb.gated_grad(type_, gate, M, N, K, *dH.args(), *X.args(), *Wg.args(), *Wu.args(), *G.args(), *U.args(),
                       *(dX.args() if "x" in which else none), *((*dWg.args(), *dWu.args()) if "w" in which else none + none))
    assert st == 0
    torch.cuda.synchronize()
    return X, Wg, Wu, G, U, dH, dX, dWg, dWu


def grad_check(type_, gate, M, N, X, Wg, Wu, G, U, dH, dX, dWg, dWu, which="xw"):
    d = DTYPES[type_]
    x, wg, wu, g, u, dh = (b.mat.double() for b in (X, Wg, Wu, G, U, dH))
    du, dg = dh * act(gate, g), dh * u * slope(gate, g)
    # values on their way: two or three roundings in float, the functions', then one to the type
    edu = half_step(d, du) * 1.01 + du.abs() * FUNC + dh.abs() * 2.0 ** -22
    edg = half_step(d, dg) * 1.01 + dg.abs() * FUNC + (dh * u).abs() * 2.0 ** -20
    if "x" in which:
        mags = (dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()
        close(dX.mat, dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + 2 * N * SUM * mags, d)
    if "w" in which:
        for got, v, e in ((dWg, dg, edg), (dWu, du, edu)):
            close(got.mat, v.t() @ x, e.t() @ x.abs() + M * SUM * ((v.abs() + e).t() @ x.abs()), d)
    for b, w in ((dX, "x"), (dWg, "w"), (dWu, "w")):
        assert b.surroundings_untouched()
        if w not in which:
            assert bool((b.flat == b.fill).all())


@pytest.mark.parametrize("M,N,K,off,pad", SHAPES, ids=IDS)
@pytest.mark.parametrize("type_", HALVES)
def test_gated_grad(type_, M, N, K, off, pad):
    gate = GATES[(M + N + K) % 3]
    grad_check(type_, gate, M, N, *grad_case(type_, gate, M, N, K, off, pad))


@pytest.mark.parametrize("type_", HALVES)
@pytest.mark.parametrize("M,N,K,off,pad", [(1, 6000, 2100, 0, 0), (3, 5003, 1030, 0, 6), (40, 3000, 4100, 2, 8), (17, 9000, 203, 1, 0)])
def test_gated_grad_of_few_tokens_and_wide_layers(type_, M, N, K, off, pad):
    """Sizes at which the two products may go in a launch each; the same call again, captured, gives the same bits."""
    gate = GATES[(M + N) % 3]
    bufs = grad_case(type_, gate, M, N, K, off, pad)
    grad_check(type_, gate, M, N, *bufs)
    X, Wg, Wu, G, U, dH, dX, dWg, dWu = bufs
    keep = [b.mat.clone() for b in (dX, dWg, dWu)]

    def run():
        assert cb.gated_grad(type_, gate, M, N, K, *dH.args(), *X.args(), *Wg.args(), *Wu.args(), *G.args(), *U.args(), *dX.args(), *dWg.args(),
                             *dWu.args()) == 0

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run()
    for _ in range(3):
        for b in (dX, dWg, dWu):
            b.mat.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(b.mat, k) for b, k in zip((dX, dWg, dWu), keep))
        assert all(b.surroundings_untouched() for b in (dX, dWg, dWu))


@pytest.mark.parametrize("which", ["x", "w"])
@pytest.mark.parametrize("M,N,K,off,pad", [(1, 1, 1, 0, 0), (70, 130, 200, 0, 0), (33, 65, 17, 1, 3)])
def test_gated_grad_of_one_side_alone(which, M, N, K, off, pad):
    bufs = grad_case(cb.Type.BF16, cb.Gate.Gelu, M, N, K, off, pad, which)
    grad_check(cb.Type.BF16, cb.Gate.Gelu, M, N, *bufs, which=which)


@pytest.mark.parametrize("gate", GATES)
def test_gated_grad_where_the_gate_saturates(gate):
    g = torch.cat([torch.linspace(-30, 30, 241), torch.tensor([-1e30, -200.0, -100.0, 100.0, 1e30])]).bfloat16()
    M = g.numel()
    G = g[:, None].contiguous().cuda()
    one, X = torch.ones(M, 1, dtype=torch.bfloat16, device="cuda"), torch.zeros(M, 1, dtype=torch.bfloat16, device="cuda")
    Wg, Wu = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda")
    dX = torch.empty(M, 1, dtype=torch.bfloat16, device="cuda")
    none = (None, 0, 0)
    assert cb.gated_grad(cb.Type.BF16, gate, M, 1, 1, one, 0, 1, X, 0, 1, Wg, 0, 1, Wu, 0, 1, G, 0, 1, one, 0, 1, dX, 0, 1, *none, *none) == 0
    want = slope(gate, G.double().clamp(-150, 150))
    close(dX, want, half_step(torch.bfloat16, want) * 1.01 + 2.0 ** -18, torch.bfloat16)


@pytest.mark.parametrize("gate", GATES)
def test_gated_grad_against_differences(gate):
    """dX and dW from the call against central differences of sum(H dH) in 64 bits along random directions."""
    M, N, K = 40, 72, 56
    X, Wg, Wu = (t.cuda() for t in (normal(M, K, 1).half(), (normal(N, K, 2) / 7).half(), (normal(N, K, 3) / 7).half()))
    dH = normal(M, N, 4).half().cuda()
    H, G, U = (torch.empty(M, N, dtype=torch.float16, device="cuda") for _ in range(3))
    dX, dWg, dWu = torch.empty_like(X), torch.empty_like(Wg), torch.empty_like(Wu)
    assert cb.gated(cb.Type.F16, gate, M, N, K, X, 0, K, Wg, 0, K, Wu, 0, K, H, 0, N, G, 0, N, U, 0, N) == 0
    assert cb.gated_grad(cb.Type.F16, gate, M, N, K, dH, 0, N, X, 0, K, Wg, 0, K, Wu, 0, K, G, 0, N, U, 0, N, dX, 0, K, dWg, 0, K, dWu, 0, K) == 0
    x, wg, wu, dh = X.double(), Wg.double(), Wu.double(), dH.double()

    def loss(x, wg, wu):
        return float((act(gate, x @ wg.t()) * (x @ wu.t()) * dh).sum())

    h = 1e-5
    for i, (got, at) in enumerate(((dX, x), (dWg, wg), (dWu, wu))):
        v = normal(*at.shape, 20 + i).cuda().double()
        step = [a + h * v if j == i else a for j, a in enumerate((x, wg, wu))]
        back = [a - h * v if j == i else a for j, a in enumerate((x, wg, wu))]
        slope_fd = (loss(*step) - loss(*back)) / (2 * h)
        # G and U (rounded, 2^-11), dG and dU and the result each off by half a step at most, no cancellation assumed
        g, u = x @ wg.t(), x @ wu.t()
        size = (dh.abs() * (g.abs() + 1) * (u.abs() + 1)).sum(0 if i else 1)
        bound = 6 * 2.0 ** -11 * float((v.abs() * ((size[:, None] * x.abs().amax(0)) if i else
                                                   (dh.abs() * (g.abs() + 1) * (u.abs() + 1)) @ (wg.abs() + wu.abs()))).sum())
        assert abs(float((got.double() * v).sum()) - slope_fd) <= bound
        assert bound < 0.5 * float((got.double().abs() * v.abs()).sum())  # (the comparison says something)


# ---- as they are used ----

def test_a_serving_layer_in_eight_bits():
    """quantise -> gated -> quantise -> product, each step against its definition on what the step before gave."""
    M, K, N = 37, 256, 640
    x = normal(M, K, 1).bfloat16().cuda()
    weights = [(normal(n, k, 2 + i) / math.sqrt(k)).cuda() for i, (n, k) in enumerate(((N, K), (N, K), (K, N)))]
    bf, f32 = cb.Type.BF16, cb.Type.F32
    q = [torch.empty(w.shape, dtype=torch.int8, device="cuda") for w in weights]
    s = [torch.empty(w.shape[0], device="cuda") for w in weights]
    for w, qi, si in zip(weights, q, s):
        assert cb.quantize_rows(f32, *w.shape, w, 0, w.shape[1], qi, 0, w.shape[1], si) == 0
    qx, sx = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    h, qh, sh = torch.empty(M, N, dtype=torch.bfloat16, device="cuda"), torch.empty(M, N, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    y = torch.empty(M, K, dtype=torch.bfloat16, device="cuda")

    def run():
        assert cb.quantize_rows(bf, M, K, x, 0, K, qx, 0, K, sx) == 0
        assert cb.gated_i8(bf, cb.Gate.Silu, M, N, K, qx, 0, K, sx, q[0], 0, K, s[0], q[1], 0, K, s[1], h, 0, N) == 0
        assert cb.quantize_rows(bf, M, N, h, 0, N, qh, 0, N, sh) == 0
        assert cb.i8gemm(bf, M, K, N, qh, 0, N, sh, q[2], 0, N, s[2], y, 0, K) == 0

    run()

    def scaled(a, sa, b, sb):  # the integer sums exactly (they may cancel), then the scales
        return (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None, :]

    g, u = scaled(qx, sx, q[0], s[0]), scaled(qx, sx, q[1], s[1])
    want, err = gated_want(cb.Gate.Silu, g, u, g.abs() * 2.0 ** -22, u.abs() * 2.0 ** -22)
    close(h, want, err, torch.bfloat16)
    assert torch.equal(qh.double(), torch.round(127 * h.double() / h.double().abs().amax(1, keepdim=True)))
    want = scaled(qh, sh, q[2], s[2])
    close(y, want, want.abs() * 2.0 ** -22, torch.bfloat16)
    # and the whole stays near the layer in full precision: three quantisations to steps of a / 127
    full = (act(cb.Gate.Silu, x.double() @ weights[0].double().t()) * (x.double() @ weights[1].double().t())) @ weights[2].double().t()
    assert float((y.double() - full).norm() / full.norm()) < 0.05

    # the same from a captured graph, several times, with other work between
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run()
    stream.synchronize()
    keep = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run()
    for _ in range(3):
        for t in (qx, sx, h, qh, sh, y):
            t.zero_()
        run()
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, keep)


def test_a_training_step_forward_and_backward_replays_from_a_graph():
    M, N, K = 130, 300, 200
    d = torch.bfloat16
    X, Wg, Wu, dH = normal(M, K, 1).to(d).cuda(), (normal(N, K, 2) / 14).to(d).cuda(), (normal(N, K, 3) / 14).to(d).cuda(), normal(M, N, 4).to(d).cuda()
    H, G, U = (torch.empty(M, N, dtype=d, device="cuda") for _ in range(3))
    dX, dWg, dWu = torch.empty_like(X), torch.empty_like(Wg), torch.empty_like(Wu)
    outs = (H, G, U, dX, dWg, dWu)

    def run():
        assert cb.gated(cb.Type.BF16, cb.Gate.Gelu, M, N, K, X, 0, K, Wg, 0, K, Wu, 0, K, H, 0, N, G, 0, N, U, 0, N) == 0
        assert cb.gated_grad(cb.Type.BF16, cb.Gate.Gelu, M, N, K, dH, 0, N, X, 0, K, Wg, 0, K, Wu, 0, K, G, 0, N, U, 0, N, dX, 0, K, dWg, 0, K,
                             dWu, 0, K) == 0

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    stream.synchronize()
    keep = [t.clone() for t in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run()
    for _ in range(3):
        for t in outs:
            t.fill_(math.nan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, keep))
    # gradients through autograd of the plain layer in 64 bits, from the same G and U
    g, u = G.double().requires_grad_(), U.double().requires_grad_()
    (act(cb.Gate.Gelu, g) * u * dH.double()).sum().backward()
    want = g.grad @ Wg.double() + u.grad @ Wu.double()
    assert float((dX.double() - want).norm() / want.norm()) < 2 * 2.0 ** -8


def test_capture_without_buffers_is_refused_and_touches_nothing():
    M, N, K = 64, 96, 72
    d = torch.bfloat16
    X, W, G = torch.ones(M, K, dtype=d, device="cuda"), torch.ones(N, K, dtype=d, device="cuda"), torch.ones(M, N, dtype=d, device="cuda")
    dX, dWg, dWu = torch.full_like(X, 3), torch.full_like(W, 3), torch.full_like(W, 3)
    stream = torch.cuda.Stream()
    cb.release_stream(stream)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        st = cb.gated_grad(cb.Type.BF16, cb.Gate.Silu, M, N, K, G, 0, N, X, 0, K, W, 0, K, W, 0, K, G, 0, N, G, 0, N, dX, 0, K, dWg, 0, K, dWu, 0, K)
    assert st == cb.Status.InvalidOperation
    graph.replay()
    torch.cuda.synchronize()
    assert all(bool((t == 3).all()) for t in (dX, dWg, dWu))


def test_on_a_side_stream_beside_the_default_one():
    """Two streams at once, each with its own scratch: results equal those of one after the other."""
    M, N, K = 96, 512, 4096
    A, B = whole(M, K, 1).cuda(), whole(N, K, 2).cuda()
    sa, sb = scales(M, 3).cuda(), scales(N, 4).cuda()
    outs = [torch.empty(M, N, device="cuda") for _ in range(9)]
    torch.cuda.synchronize()
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    for i, C in enumerate(outs):
        assert cb.i8gemm(cb.Type.F32, M, N, K, A, 0, K, sa, B, 0, K, sb, C, 0, N, stream=streams[i % 3]) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], C) for C in outs[1:])


# ---- every form of the kernels, and what the choice of a form leaves to larger calls ----

FORMS = list(range(9))  # four from registers, five tiled
# tails of every length in a step's 16-byte slots and in its two halves; more tiles than workgroups; few steps per tile
FORM_SHAPES = [(70, 90, 8, 0), (70, 90, 63, 1), (33, 140, 65, 1), (130, 70, 97, 3), (257, 300, 127, 1), (64, 128, 129, 3), (300, 520, 450, 2), (1500, 1600, 40, 0)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("splits", [0, 3])
def test_every_form(form, splits):
    from gpu_util import debug_env
    with debug_env(CLBLAS_AMD_FFN_FORM=form, CLBLAS_AMD_FFN_SPLITS=splits):
        for M, N, K, pad in FORM_SHAPES:
            test_i8gemm(cb.Type.BF16, M, N, K, 0, pad + 3)
            test_gated(cb.Type.F16, True, M, N, K, 0, pad)
            test_gated_i8(cb.Type.F32, M, N, K, 0, 4 - (K + 1) % 4)
            if form >= 4:  # (the gradients are tiled)
                test_gated_grad(cb.Type.BF16, M, N, K, 0, pad)
                test_gated_grad(cb.Type.F16, K, M, N, 0, 0)


@pytest.mark.parametrize("form", [4, 5, 6, 7, 8])
@pytest.mark.parametrize("K", [100, 260])
def test_more_tiles_than_workgroups(form, K):
    """One or a few steps per tile, and workgroups that walk several tiles: the loads of later tiles run ahead."""
    from gpu_util import debug_env
    M, N = (4300, 4500) if form == 4 else (3000, 3100)
    with debug_env(CLBLAS_AMD_FFN_FORM=form):
        test_i8gemm(cb.Type.F16, M, N, K, 0, 0)
        test_gated(cb.Type.BF16, False, M, N // 2 + 7, K, 0, 0)
        if K == 100:
            n = 2700 if form == 4 else 1500
            test_gated_grad(cb.Type.BF16, n, n + 30, n + 8, 0, 0)


@pytest.mark.parametrize("form", FORMS)
def test_what_lies_between_rows_does_not_matter(form):
    """NaN in the gaps between the rows of every operand, where loads of whole pieces of a row reach."""
    from gpu_util import debug_env
    M, N, d = 70, 200, torch.bfloat16
    for K, pad in ((57, 1), (64, 2), (101, 3), (200, 8)):
        X, Wg, Wu = (Buf(n, K, d, 0, pad, normal(n, K, i), fill=math.nan) for i, n in enumerate((M, N, N)))
        G, U, dH = (Buf(M, N, d, 0, pad, normal(M, N, 3 + i), fill=math.nan) for i in range(3))
        H, dX, dWg, dWu = Buf(M, N, d, 0, pad), Buf(M, K, d, 0, pad), Buf(N, K, d, 0, pad), Buf(N, K, d, 0, pad)
        with debug_env(CLBLAS_AMD_FFN_FORM=form):
            assert cb.gated(cb.Type.BF16, cb.Gate.Silu, M, N, K, *X.args(), *Wg.args(), *Wu.args(), *H.args()) == 0
            assert cb.gated_grad(cb.Type.BF16, cb.Gate.Silu, M, N, K, *dH.args(), *X.args(), *Wg.args(), *Wu.args(), *G.args(), *U.args(), *dX.args(),
                                 *dWg.args(), *dWu.args()) == 0
        torch.cuda.synchronize()
        for b in (H, dX, dWg, dWu):
            assert bool(torch.isfinite(b.mat).all()) and b.surroundings_untouched()


def test_results_and_operands_beyond_32_bits():
    """Element offsets past 2^31 and byte offsets past 2^32, in operands and results; rows from both ends are checked."""
    M, N, K = 33000, 66000, 64
    A, B = whole(M, K, 1).cuda(), whole(N, K, 2).cuda()
    sa, sb = scales(M, 3).cuda(), scales(N, 4).cuda()
    C = torch.full((M, N), 7.0, dtype=torch.bfloat16, device="cuda")
    assert cb.i8gemm(cb.Type.BF16, M, N, K, A, 0, K, sa, B, 0, K, sb, C, 0, N) == 0
    torch.cuda.synchronize()
    for r in (slice(0, 40), slice(16400, 16440), slice(M - 40, M)):
        want = (A[r].double() @ B.double().t()) * sa[r].double()[:, None] * sb.double()[None, :]
        close(C[r], want, want.abs() * 3 * 2.0 ** -24, torch.bfloat16)
    # the result as an operand: rows 132 000 bytes apart
    ld, m, k, n = N, M, 72, 48
    Wg, Wu = normal(n, k, 5).bfloat16().cuda(), normal(n, k, 6).bfloat16().cuda()
    H = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    assert cb.gated(cb.Type.BF16, cb.Gate.Gelu, m, n, k, C, 0, ld, Wg, 0, k, Wu, 0, k, H, 0, n) == 0
    dX, dWg, dWu = torch.empty(m, k, dtype=torch.bfloat16, device="cuda"), torch.empty_like(Wg), torch.empty_like(Wu)
    dH, G, U = (normal(m, n, 7 + i).bfloat16().cuda() for i in range(3))
    assert cb.gated_grad(cb.Type.BF16, cb.Gate.Gelu, m, n, k, dH, 0, n, C, 0, ld, Wg, 0, k, Wu, 0, k, G, 0, n, U, 0, n, dX, 0, k, dWg, 0, k, dWu, 0, k) == 0
    Q, s = torch.empty(m, k, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    assert cb.quantize_rows(cb.Type.BF16, m, k, C, 0, ld, Q, 0, k, s) == 0
    torch.cuda.synchronize()
    x = C[:, :k].double()
    g, u = x @ Wg.double().t(), x @ Wu.double().t()
    eg, eu = k * SUM * (x.abs() @ Wg.double().abs().t()), k * SUM * (x.abs() @ Wu.double().abs().t())
    h, eh = gated_want(cb.Gate.Gelu, g, u, eg, eu)
    close(H, h, eh, torch.bfloat16)
    a = x.abs().amax(1, keepdim=True)
    assert torch.equal(Q.double(), torch.where(a > 0, torch.round(127 * x / a), torch.zeros_like(x)))
    du, dg = dH.double() * act(cb.Gate.Gelu, G.double()), dH.double() * U.double() * slope(cb.Gate.Gelu, G.double())
    for got, v in ((dWg, dg), (dWu, du)):
        e = half_step(torch.bfloat16, v) * 1.01 + (dH * U).double().abs() * 2.0 ** -19 + dH.double().abs() * 2.0 ** -19
        close(got, v.t() @ x, e.t() @ x.abs() + m * SUM * (v.abs().t() @ x.abs()), torch.bfloat16)


def test_same_weights_twice_and_no_copy_of_results():
    """Wg and Wu the same matrix: H = act(G) o G."""
    M, N, K = 50, 60, 70
    X, W = normal(M, K, 1).half().cuda(), (normal(N, K, 2) / 8).half().cuda()
    H, G, U = (torch.empty(M, N, dtype=torch.float16, device="cuda") for _ in range(3))
    assert cb.gated(cb.Type.F16, cb.Gate.Silu, M, N, K, X, 0, K, W, 0, K, W, 0, K, H, 0, N, G, 0, N, U, 0, N) == 0
    assert torch.equal(G, U)
    g = X.double() @ W.double().t()
    e = K * SUM * (X.double().abs() @ W.double().abs().t())
    h, eh = gated_want(cb.Gate.Silu, g, g, e, e)
    close(H, h, eh, torch.float16)


def test_repeated_calls_give_the_same_bits():
    for M, N, K in ((16, 700, 4096), (100, 90, 8200), (513, 771, 1030)):
        a = [t.clone() for t in _outs(M, N, K)]
        for _ in range(3):
            assert all(torch.equal(x, y) for x, y in zip(a, _outs(M, N, K)))


def _outs(M, N, K):
    bufs = grad_case(cb.Type.BF16, cb.Gate.Gelu, M, N, K, 0, 0)
    H = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    assert cb.gated(cb.Type.BF16, cb.Gate.Gelu, M, N, K, *bufs[0].args(), *bufs[1].args(), *bufs[2].args(), H, 0, N) == 0
    torch.cuda.synchronize()
    return [H] + [b.mat for b in bufs[6:]]


def test_reserved_workspace_lets_the_first_call_be_captured():
    """The sizes that the header gives are enough."""
    M, N, K = 100, 90, 8201  # copies (rows of an odd number of 16-bit elements) and partial sums
    d = torch.bfloat16
    X, Wg, Wu = (normal(n, K, i).to(d).cuda() for i, n in enumerate((M, N, N)))
    G, U, dH = (normal(M, N, 3 + i).to(d).cuda() for i in range(3))
    H, dX, dWg, dWu = torch.empty(M, N, dtype=d, device="cuda"), torch.empty_like(X), torch.empty_like(Wg), torch.empty_like(Wu)
    row = (2 * K + 127) // 128 * 128
    copies = row * (M + 2 * N) + 3 * 256
    grads = 4 * M * ((N + 63) // 64 * 64) + copies + 256
    sums = 32 * 4 * max(2 * M * (N + 3), M * (K + 3) + 2 * N * (K + 3)) + 256
    stream = torch.cuda.Stream()
    assert cb.reserve_workspace(gemm_bytes=sums, trmm_bytes=max(copies, grads), stream=stream) == 0
    torch.cuda.synchronize()

    def run():
        a = cb.gated(cb.Type.BF16, cb.Gate.Silu, M, N, K, X, 0, K, Wg, 0, K, Wu, 0, K, H, 0, N)
        b = cb.gated_grad(cb.Type.BF16, cb.Gate.Silu, M, N, K, dH, 0, N, X, 0, K, Wg, 0, K, Wu, 0, K, G, 0, N, U, 0, N, dX, 0, K, dWg, 0, K, dWu, 0, K)
        return a, b

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert run() == (0, 0)
    graph.replay()
    torch.cuda.synchronize()
    first = [t.clone() for t in (H, dX, dWg, dWu)]
    assert run() == (0, 0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, (H, dX, dWg, dWu)))


def test_memory_check_covers_the_scales():
    from gpu_util import debug_env
    A, B, C = torch.zeros(4, 16, dtype=torch.int8, device="cuda"), torch.zeros(600, 16, dtype=torch.int8, device="cuda"), torch.zeros(4, 600, device="cuda")
    big = torch.ones(1 << 20, device="cuda")
    end = big[-2:]  # (allocations are rounded up: only the end of one is known to be an end)
    with debug_env(CLBLAS_AMD_CHECK_MEM=1):
        assert cb.i8gemm(cb.Type.F32, 4, 600, 16, A, 0, 16, big, B, 0, 16, big, C, 0, 600) == 0
        ok = cb.i8gemm(cb.Type.F32, 1, 600, 16, A, 0, 16, end, B, 0, 16, big, C, 0, 600)
        assert ok == 0
        far = big.data_ptr() + (1 << 40)
        assert cb.i8gemm(cb.Type.F32, 4, 600, 16, A, 0, 16, far, B, 0, 16, big, C, 0, 600) == cb.Status.InvalidVecX
        assert cb.i8gemm(cb.Type.F32, 4, 600, 16, A, 0, 16, big, B, 0, 16, far, C, 0, 600) == cb.Status.InvalidVecY
    torch.cuda.synchronize()


def test_quantize_rows_more_rows_than_31_bits_can_step_over():
    """Rows numbered up to almost 2^31: the step from a workgroup's row to its next one passes 31 bits."""
    M = 2 ** 31 - 600
    X = torch.full((M,), 2.0, dtype=torch.bfloat16, device="cuda")
    X[-3:] = torch.tensor([0.0, -4.0, 8.0], device="cuda")
    Q, s = torch.zeros(M + 8, dtype=torch.int8, device="cuda"), torch.zeros(M, device="cuda")
    assert cb.quantize_rows(cb.Type.BF16, M, 1, X, 0, 1, Q, 0, 1, s) == 0
    torch.cuda.synchronize()
    assert Q[-11:].tolist() == [0, -127, 127] + [0] * 8 and s[-4:].tolist() == [torch.tensor(v / 127).float().item() for v in (2.0, 0.0, 4.0, 8.0)]
    assert bool((Q[:M - 3] == 127).all()) and bool((s[:M - 3] == s[0]).all())


def test_more_rows_than_one_launch_of_the_smallest_products_holds():
    """2^29 tokens, one channel: a register form's grid would pass 2^32 threads."""
    M = 2 ** 29 + 77
    A = torch.ones(M, 4, dtype=torch.int8, device="cuda")
    A[::1000003, 2] = 3
    sa = torch.full((M,), 0.5, device="cuda")
    B, sb = torch.ones(1, 4, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda")
    C = torch.zeros(M + 4, dtype=torch.float16, device="cuda")
    assert cb.i8gemm(cb.Type.F16, M, 1, 4, A, 0, 4, sa, B, 0, 4, sb, C, 0, 1) == 0
    torch.cuda.synchronize()
    want = torch.full((M,), 2.0, dtype=torch.float16, device="cuda")
    want[::1000003] = 3.0
    assert torch.equal(C[:M], want) and not C[M:].any()
