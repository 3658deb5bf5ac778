"""Refusals of the feed-forward products (no GPU: every call fails a check before anything is launched)."""
import pytest

import clblas_amd as cb

FAKE = 0x1000
S = cb.Status
M, N, K = 5, 6, 7


def quantize(**kw):
    a = dict(type_=cb.Type.BF16, M=M, K=K, X=FAKE, offX=0, ldx=K, Q=FAKE, offQ=0, ldq=K, scale=FAKE)
    a.update(kw)
    return cb.quantize_rows(**a, stream=0)


def i8gemm(**kw):
    a = dict(typeC=cb.Type.F32, M=M, N=N, K=K, A=FAKE, offA=0, lda=K, scaleA=FAKE, B=FAKE, offB=0, ldb=K, scaleB=FAKE, C=FAKE, offC=0, ldc=N)
    a.update(kw)
    return cb.i8gemm(**a, stream=0)


def gated(**kw):
    a = dict(type_=cb.Type.BF16, gate=cb.Gate.Silu, M=M, N=N, K=K, X=FAKE, offX=0, ldx=K, Wg=FAKE, offWg=0, ldwg=K, Wu=FAKE, offWu=0, ldwu=K,
             H=FAKE, offH=0, ldh=N, G=FAKE, offG=0, ldg=N, U=FAKE, offU=0, ldu=N)
    a.update(kw)
    return cb.gated(**a, stream=0)


def gated_i8(**kw):
    a = dict(typeH=cb.Type.BF16, gate=cb.Gate.Silu, M=M, N=N, K=K, X=FAKE, offX=0, ldx=K, scaleX=FAKE, Wg=FAKE, offWg=0, ldwg=K, scaleWg=FAKE,
             Wu=FAKE, offWu=0, ldwu=K, scaleWu=FAKE, H=FAKE, offH=0, ldh=N)
    a.update(kw)
    return cb.gated_i8(**a, stream=0)


def gated_grad(**kw):
    a = dict(type_=cb.Type.F16, gate=cb.Gate.Gelu, M=M, N=N, K=K, dH=FAKE, offdH=0, lddh=N, X=FAKE, offX=0, ldx=K, Wg=FAKE, offWg=0, ldwg=K,
             Wu=FAKE, offWu=0, ldwu=K, G=FAKE, offG=0, ldg=N, U=FAKE, offU=0, ldu=N, dX=FAKE, offdX=0, lddx=K, dWg=FAKE, offdWg=0, lddwg=K,
             dWu=FAKE, offdWu=0, lddwu=K)
    a.update(kw)
    return cb.gated_grad(**a, stream=0)


CASES = [
    (quantize, dict(X=None, Q=None), S.InvalidMatA), (quantize, dict(Q=None, scale=None), S.InvalidMatC), (quantize, dict(scale=None, type_=9), S.InvalidVecX),
    (quantize, dict(type_=3, M=0), S.InvalidValue), (quantize, dict(type_=-1), S.InvalidValue), (quantize, dict(M=0), S.InvalidDim),
    (quantize, dict(K=0), S.InvalidDim), (quantize, dict(ldx=K - 1, ldq=0), S.InvalidLeadDimA), (quantize, dict(ldq=K - 1), S.InvalidLeadDimC),
    (quantize, dict(M=2 ** 31), S.NotImplemented),
    (i8gemm, dict(A=None, B=None), S.InvalidMatA), (i8gemm, dict(B=None, C=None), S.InvalidMatB), (i8gemm, dict(C=None, scaleA=None), S.InvalidMatC),
    (i8gemm, dict(scaleA=None, scaleB=None), S.InvalidVecX), (i8gemm, dict(scaleB=None, typeC=7), S.InvalidVecY), (i8gemm, dict(typeC=3), S.InvalidValue),
    (i8gemm, dict(M=0), S.InvalidDim), (i8gemm, dict(N=0), S.InvalidDim), (i8gemm, dict(K=0), S.InvalidDim), (i8gemm, dict(lda=K - 1, ldb=0), S.InvalidLeadDimA),
    (i8gemm, dict(ldb=K - 1, ldc=0), S.InvalidLeadDimB), (i8gemm, dict(ldc=N - 1), S.InvalidLeadDimC),
    (i8gemm, dict(K=131072, lda=131072, ldb=131072), S.NotImplemented), (i8gemm, dict(N=2 ** 31, ldc=2 ** 31), S.NotImplemented),
    (gated, dict(X=None), S.InvalidMatA), (gated, dict(Wg=None), S.InvalidMatB), (gated, dict(Wu=None, H=None), S.InvalidMatB), (gated, dict(H=None), S.InvalidMatC),
    (gated, dict(G=None), S.InvalidMatC), (gated, dict(U=None, type_=0), S.InvalidMatC), (gated, dict(type_=cb.Type.F32), S.InvalidValue),
    (gated, dict(gate=3, M=0), S.InvalidValue), (gated, dict(gate=-1), S.InvalidValue), (gated, dict(M=0), S.InvalidDim), (gated, dict(N=0), S.InvalidDim),
    (gated, dict(K=0), S.InvalidDim), (gated, dict(ldx=K - 1), S.InvalidLeadDimA), (gated, dict(ldwg=K - 1), S.InvalidLeadDimB),
    (gated, dict(ldwu=K - 1, ldh=0), S.InvalidLeadDimB), (gated, dict(ldh=N - 1), S.InvalidLeadDimC), (gated, dict(ldg=N - 1), S.InvalidLeadDimC),
    (gated, dict(ldu=N - 1), S.InvalidLeadDimC), (gated, dict(ldx=2 ** 32), S.NotImplemented),
    (gated_i8, dict(X=None), S.InvalidMatA), (gated_i8, dict(Wg=None), S.InvalidMatB), (gated_i8, dict(Wu=None), S.InvalidMatB), (gated_i8, dict(H=None), S.InvalidMatC),
    (gated_i8, dict(scaleX=None, scaleWg=None), S.InvalidVecX), (gated_i8, dict(scaleWg=None), S.InvalidVecY), (gated_i8, dict(scaleWu=None), S.InvalidVecY),
    (gated_i8, dict(typeH=5), S.InvalidValue), (gated_i8, dict(gate=5), S.InvalidValue), (gated_i8, dict(K=0), S.InvalidDim),
    (gated_i8, dict(ldx=K - 1), S.InvalidLeadDimA), (gated_i8, dict(ldwu=K - 1), S.InvalidLeadDimB), (gated_i8, dict(ldh=N - 1), S.InvalidLeadDimC),
    (gated_i8, dict(K=131072, ldx=131072, ldwg=131072, ldwu=131072), S.NotImplemented),
    (gated_grad, dict(X=None, dH=None), S.InvalidMatA), (gated_grad, dict(dH=None), S.InvalidMatB), (gated_grad, dict(G=None), S.InvalidMatB),
    (gated_grad, dict(U=None), S.InvalidMatB), (gated_grad, dict(Wg=None), S.InvalidMatB), (gated_grad, dict(Wu=None), S.InvalidMatB),
    (gated_grad, dict(dX=None, dWg=None, dWu=None), S.InvalidMatC), (gated_grad, dict(dWg=None), S.InvalidMatC), (gated_grad, dict(dX=None, dWu=None), S.InvalidMatC),
    (gated_grad, dict(type_=cb.Type.F32), S.InvalidValue), (gated_grad, dict(gate=4), S.InvalidValue), (gated_grad, dict(M=0), S.InvalidDim),
    (gated_grad, dict(lddh=N - 1, ldx=0), S.InvalidLeadDimB), (gated_grad, dict(ldx=K - 1), S.InvalidLeadDimA), (gated_grad, dict(ldwg=K - 1), S.InvalidLeadDimB),
    (gated_grad, dict(ldu=N - 1), S.InvalidLeadDimB), (gated_grad, dict(lddx=K - 1), S.InvalidLeadDimC), (gated_grad, dict(lddwg=K - 1), S.InvalidLeadDimC),
    (gated_grad, dict(lddwu=K - 1), S.InvalidLeadDimC), (gated_grad, dict(dX=None, lddwu=K - 1), S.InvalidLeadDimC),
]


@pytest.mark.parametrize("fn,change,want", CASES, ids=["%s-%s" % (f.__name__, "-".join("%s=%s" % kv for kv in c.items())) for f, c, _ in CASES])
def test_refused(fn, change, want):
    assert fn(**change) == want
