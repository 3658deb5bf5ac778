// C ABI of the feed-forward products: argument checks and dispatch.
#include "../../include/clblas_amd.h"
#include "api_checks.hpp"
#include "ffn.hpp"
#include "internal.h"

#include <hip/hip_runtime_api.h>

#include <initializer_list>

namespace {

using cba::ffn::Mat;
using cba::ffn::OutMat;

bool valid_type(clblasAmdType t) { return t == clblasAmdF32 || t == clblasAmdF16 || t == clblasAmdBf16; }
bool valid_gate(clblasAmdGate g) { return g == clblasAmdSilu || g == clblasAmdGelu || g == clblasAmdGeluTanh; }
size_t size_of(clblasAmdType t) { return t == clblasAmdF32 ? 4 : 2; }

clblasStatus check_rows(size_t rows, size_t cols, size_t ld, MatId which, const void *base, size_t off, size_t tsize) {
    return check_matrix_sizes(clblasRowMajor, clblasNoTrans, rows, cols, ld, which, base, off, tsize);
}

// A vector of n floats (one per token: VecX, one per channel: VecY): with CLBLAS_AMD_CHECK_MEM=1 it has to fit behind its pointer.
clblasStatus check_scales(const float *scale, size_t n, bool tokens) {
    if (!cba::knobs().check_mem) return clblasSuccess;
    const size_t mem = cba::mem_behind(scale);
    if (mem == 0) return tokens ? clblasInvalidVecX : clblasInvalidVecY;
    if (mem / sizeof(float) < n) return tokens ? clblasInsufficientMemVecX : clblasInsufficientMemVecY;
    return clblasSuccess;
}

// Offsets in elements, rows * ld, stay below 2^63 (and no memory is as large as that: whatever passes this only has to be
// addressed correctly).
bool strides_in_range(std::initializer_list<size_t> lds) {
    for (size_t ld : lds)
        if (ld > ((size_t)1 << 31)) return false;
    return true;
}

Mat mat(const void *p, size_t off, size_t ld, size_t tsize) {
    Mat m;
    m.ptr = p ? static_cast<const char *>(p) + off * tsize : nullptr;
    m.ld = (int64_t)ld;
    return m;
}
OutMat out_mat(void *p, size_t off, size_t ld, size_t tsize) {
    OutMat m;
    m.ptr = p ? static_cast<char *>(p) + off * tsize : nullptr;
    m.ld = (int64_t)ld;
    return m;
}

// Depth up to which sums of products of two 8-bit integers, (-128)^2 = 2^14 at most, stay below 2^31.
const size_t kMaxDepthI8 = ((size_t)1 << 17) - 1;

#define CBA_CHECK(expr)                                   \
    do {                                                  \
        const clblasStatus st_ = (expr);                  \
        if (st_ != clblasSuccess) return st_;             \
    } while (0)

}  // namespace

extern "C" {

clblasStatus clblasAmdQuantizeRows(clblasAmdType type, size_t M, size_t K, const void *X, size_t offX, size_t ldx,
                                   signed char *Q, size_t offQ, size_t ldq, float *scale, hipStream_t stream) {
    if (!X) return clblasInvalidMatA;
    if (!Q) return clblasInvalidMatC;
    if (!scale) return clblasInvalidVecX;
    if (!valid_type(type)) return clblasInvalidValue;
    CBA_CHECK(check_rows(M, K, ldx, MAT_A, X, offX, size_of(type)));
    CBA_CHECK(check_rows(M, K, ldq, MAT_C, Q, offQ, 1));
    CBA_CHECK(check_scales(scale, M, true));
    if (M > kMaxDim || K > kMaxDim || !strides_in_range({ldx, ldq})) return clblasNotImplemented;
    return map_hip_error(cba::ffn::quantize_rows(type, (int)M, (int)K, mat(X, offX, ldx, size_of(type)), reinterpret_cast<int8_t *>(Q) + offQ,
                                                 (int64_t)ldq, scale, stream));
}

clblasStatus clblasAmdI8gemm(clblasAmdType typeC, size_t M, size_t N, size_t K, const signed char *A, size_t offA, size_t lda,
                             const float *scaleA, const signed char *B, size_t offB, size_t ldb, const float *scaleB, void *C,
                             size_t offC, size_t ldc, hipStream_t stream) {
    cba::CallLease lease;  // scratch handed out during this call stays ours until it returns
    if (!A) return clblasInvalidMatA;
    if (!B) return clblasInvalidMatB;
    if (!C) return clblasInvalidMatC;
    if (!scaleA) return clblasInvalidVecX;
    if (!scaleB) return clblasInvalidVecY;
    if (!valid_type(typeC)) return clblasInvalidValue;
    CBA_CHECK(check_rows(M, K, lda, MAT_A, A, offA, 1));
    CBA_CHECK(check_rows(N, K, ldb, MAT_B, B, offB, 1));
    CBA_CHECK(check_rows(M, N, ldc, MAT_C, C, offC, size_of(typeC)));
    CBA_CHECK(check_scales(scaleA, M, true));
    CBA_CHECK(check_scales(scaleB, N, false));
    if (M > kMaxDim || N > kMaxDim || K > kMaxDepthI8 || !strides_in_range({lda, ldb, ldc})) return clblasNotImplemented;
    return map_hip_error(cba::with_workspaces_secured(stream, [&] {
        return cba::ffn::product_i8(typeC, 0, (int)M, (int)N, (int)K, mat(A, offA, lda, 1), scaleA, mat(B, offB, ldb, 1), scaleB, Mat(),
                                    nullptr, out_mat(C, offC, ldc, size_of(typeC)), stream);
    }));
}

clblasStatus clblasAmdGated(clblasAmdType type, clblasAmdGate gate, size_t M, size_t N, size_t K, const void *X, size_t offX, size_t ldx,
                            const void *Wg, size_t offWg, size_t ldwg, const void *Wu, size_t offWu, size_t ldwu, void *H, size_t offH,
                            size_t ldh, void *G, size_t offG, size_t ldg, void *U, size_t offU, size_t ldu, hipStream_t stream) {
    cba::CallLease lease;
    if (!X) return clblasInvalidMatA;
    if (!Wg || !Wu) return clblasInvalidMatB;
    if (!H || !G != !U) return clblasInvalidMatC;
    if ((type != clblasAmdF16 && type != clblasAmdBf16) || !valid_gate(gate)) return clblasInvalidValue;
    CBA_CHECK(check_rows(M, K, ldx, MAT_A, X, offX, 2));
    CBA_CHECK(check_rows(N, K, ldwg, MAT_B, Wg, offWg, 2));
    CBA_CHECK(check_rows(N, K, ldwu, MAT_B, Wu, offWu, 2));
    CBA_CHECK(check_rows(M, N, ldh, MAT_C, H, offH, 2));
    if (G) {
        CBA_CHECK(check_rows(M, N, ldg, MAT_C, G, offG, 2));
        CBA_CHECK(check_rows(M, N, ldu, MAT_C, U, offU, 2));
    }
    if (M > kMaxDim || N > kMaxDim || K > kMaxDim || !strides_in_range({ldx, ldwg, ldwu, ldh, G ? ldg : 0, G ? ldu : 0}))
        return clblasNotImplemented;
    return map_hip_error(cba::with_workspaces_secured(stream, [&] {
        return cba::ffn::gated(type, gate, (int)M, (int)N, (int)K, mat(X, offX, ldx, 2), mat(Wg, offWg, ldwg, 2), mat(Wu, offWu, ldwu, 2),
                               out_mat(H, offH, ldh, 2), out_mat(G, offG, ldg, 2), out_mat(U, offU, ldu, 2), stream);
    }));
}

clblasStatus clblasAmdGatedI8(clblasAmdType typeH, clblasAmdGate gate, size_t M, size_t N, size_t K, const signed char *X, size_t offX,
                              size_t ldx, const float *scaleX, const signed char *Wg, size_t offWg, size_t ldwg, const float *scaleWg,
                              const signed char *Wu, size_t offWu, size_t ldwu, const float *scaleWu, void *H, size_t offH, size_t ldh,
                              hipStream_t stream) {
    cba::CallLease lease;
    if (!X) return clblasInvalidMatA;
    if (!Wg || !Wu) return clblasInvalidMatB;
    if (!H) return clblasInvalidMatC;
    if (!scaleX) return clblasInvalidVecX;
    if (!scaleWg || !scaleWu) return clblasInvalidVecY;
    if (!valid_type(typeH) || !valid_gate(gate)) return clblasInvalidValue;
    CBA_CHECK(check_rows(M, K, ldx, MAT_A, X, offX, 1));
    CBA_CHECK(check_rows(N, K, ldwg, MAT_B, Wg, offWg, 1));
    CBA_CHECK(check_rows(N, K, ldwu, MAT_B, Wu, offWu, 1));
    CBA_CHECK(check_rows(M, N, ldh, MAT_C, H, offH, size_of(typeH)));
    CBA_CHECK(check_scales(scaleX, M, true));
    CBA_CHECK(check_scales(scaleWg, N, false));
    CBA_CHECK(check_scales(scaleWu, N, false));
    if (M > kMaxDim || N > kMaxDim || K > kMaxDepthI8 || !strides_in_range({ldx, ldwg, ldwu, ldh})) return clblasNotImplemented;
    return map_hip_error(cba::with_workspaces_secured(stream, [&] {
        return cba::ffn::product_i8(typeH, gate, (int)M, (int)N, (int)K, mat(X, offX, ldx, 1), scaleX, mat(Wg, offWg, ldwg, 1), scaleWg,
                                    mat(Wu, offWu, ldwu, 1), scaleWu, out_mat(H, offH, ldh, size_of(typeH)), stream);
    }));
}

clblasStatus clblasAmdGatedGrad(clblasAmdType type, clblasAmdGate gate, size_t M, size_t N, size_t K, const void *dH, size_t offdH,
                                size_t lddh, const void *X, size_t offX, size_t ldx, const void *Wg, size_t offWg, size_t ldwg,
                                const void *Wu, size_t offWu, size_t ldwu, const void *G, size_t offG, size_t ldg, const void *U,
                                size_t offU, size_t ldu, void *dX, size_t offdX, size_t lddx, void *dWg, size_t offdWg, size_t lddwg,
                                void *dWu, size_t offdWu, size_t lddwu, hipStream_t stream) {
    cba::CallLease lease;
    if (!X) return clblasInvalidMatA;
    if (!dH || !Wg || !Wu || !G || !U) return clblasInvalidMatB;
    if ((!dX && !dWg) || !dWg != !dWu) return clblasInvalidMatC;
    if ((type != clblasAmdF16 && type != clblasAmdBf16) || !valid_gate((clblasAmdGate)(gate & ~clblasAmdRoundTerms))) return clblasInvalidValue;
    CBA_CHECK(check_rows(M, N, lddh, MAT_B, dH, offdH, 2));
    CBA_CHECK(check_rows(M, K, ldx, MAT_A, X, offX, 2));
    CBA_CHECK(check_rows(N, K, ldwg, MAT_B, Wg, offWg, 2));
    CBA_CHECK(check_rows(N, K, ldwu, MAT_B, Wu, offWu, 2));
    CBA_CHECK(check_rows(M, N, ldg, MAT_B, G, offG, 2));
    CBA_CHECK(check_rows(M, N, ldu, MAT_B, U, offU, 2));
    if (dX) CBA_CHECK(check_rows(M, K, lddx, MAT_C, dX, offdX, 2));
    if (dWg) {
        CBA_CHECK(check_rows(N, K, lddwg, MAT_C, dWg, offdWg, 2));
        CBA_CHECK(check_rows(N, K, lddwu, MAT_C, dWu, offdWu, 2));
    }
    if (M > kMaxDim || N > kMaxDim || K > kMaxDim ||
        4 * (N + 63) > (size_t)cba::ffn::kMaxRowBytes || 2 * K + 127 > (size_t)cba::ffn::kMaxRowBytes ||  // rows of dG and dU, and of copies
        !strides_in_range({lddh, ldx, ldwg, ldwu, ldg, ldu, dX ? lddx : 0, dWg ? lddwg : 0, dWg ? lddwu : 0}))
        return clblasNotImplemented;
    return map_hip_error(cba::with_workspaces_secured(stream, [&] {
        return cba::ffn::gated_grad(type, gate, (int)M, (int)N, (int)K, mat(dH, offdH, lddh, 2), mat(X, offX, ldx, 2),
                                    mat(Wg, offWg, ldwg, 2), mat(Wu, offWu, ldwu, 2), mat(G, offG, ldg, 2), mat(U, offU, ldu, 2),
                                    out_mat(dX, offdX, lddx, 2), out_mat(dWg, offdWg, lddwg, 2), out_mat(dWu, offdWu, lddwu, 2), stream);
    }));
}

}  // extern "C"
