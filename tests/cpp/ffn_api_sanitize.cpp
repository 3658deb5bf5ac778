// Drives the argument checks of the feed-forward products in a CPU build of clblas_amd/csrc/ffn_api.cpp with AddressSanitizer
// / UBSan.  What it hands valid problems to is replaced by stubs that count: a call that gets past the checks is seen.
#include <cstdio>
#include <cstdlib>
#include <limits>

#include "../../clblas_amd/csrc/ffn.hpp"
#include "../../clblas_amd/csrc/internal.h"
#include "../../include/clblas_amd.h"

namespace cba {
static DebugKnobs g_knobs;
static size_t g_behind = 0;
const DebugKnobs &knobs() { return g_knobs; }
size_t mem_behind(const void *) { return g_behind; }
DryRun *&dry_run_slot() {
    static DryRun *none = nullptr;
    return none;
}
DispatchRecord &dispatch_record() {
    static DispatchRecord r;
    return r;
}
hipError_t workspace_get(hipStream_t, size_t, int, void **) { return hipErrorOutOfMemory; }
CallLease::CallLease() {}
CallLease::~CallLease() {}
static int g_calls = 0;
namespace ffn {
hipError_t quantize_rows(int, int, int, Mat, int8_t *, int64_t, float *, hipStream_t) { ++g_calls; return hipSuccess; }
hipError_t product_i8(int, int, int, int, int, Mat, const float *, Mat, const float *, Mat, const float *, OutMat, hipStream_t) {
    ++g_calls;
    return hipErrorOutOfMemory;
}
hipError_t gated(int, int, int, int, int, Mat, Mat, Mat, OutMat, OutMat, OutMat, hipStream_t) { ++g_calls; return hipErrorNotSupported; }
hipError_t gated_grad(int, int, int, int, int, Mat, Mat, Mat, Mat, Mat, Mat, OutMat, OutMat, OutMat, hipStream_t) {
    ++g_calls;
    return hipErrorStreamCaptureUnsupported;
}
}  // namespace ffn
}  // namespace cba

static int failures = 0;
static void expect(const char *what, clblasStatus got, clblasStatus want, int calls) {
    if (got == want && cba::g_calls == calls) return;
    std::fprintf(stderr, "%s: %d, expected %d (%d calls, expected %d)\n", what, (int)got, (int)want, cba::g_calls, calls);
    ++failures;
}

int main() {
    static float f[4];
    static signed char q[4];
    const size_t top = std::numeric_limits<size_t>::max();
    auto quant = [&](clblasAmdType t, size_t M, size_t K, size_t ldx, size_t ldq) {
        return clblasAmdQuantizeRows(t, M, K, f, 0, ldx, q, 0, ldq, f, nullptr);
    };
    auto gemm = [&](size_t M, size_t N, size_t K, size_t ld, size_t ldc) {
        return clblasAmdI8gemm(clblasAmdF16, M, N, K, q, 0, ld, f, q, 0, ld, f, f, 0, ldc, nullptr);
    };
    auto gated = [&](size_t M, size_t N, size_t K, size_t ld, size_t ldh, void *G, void *U) {
        return clblasAmdGated(clblasAmdF16, clblasAmdGelu, M, N, K, f, 0, ld, f, 0, ld, f, 0, ld, f, 0, ldh, G, 0, ldh, U, 0, ldh, nullptr);
    };
    auto grad = [&](size_t M, size_t N, size_t K, void *dX, void *dWg, void *dWu) {
        return clblasAmdGatedGrad(clblasAmdBf16, clblasAmdSilu, M, N, K, f, 0, N, f, 0, K, f, 0, K, f, 0, K, f, 0, N, f, 0, N, dX, 0, K, dWg, 0, K, dWu, 0, K,
                                  nullptr);
    };
    // past every check: the launcher's status comes back in the library's codes
    expect("quant", quant(clblasAmdF32, 2, 3, 3, 3), clblasSuccess, 1);
    expect("gemm", gemm(2, 3, 4, 4, 3), clblasOutOfResources, 2);
    expect("gated", gated(2, 3, 4, 4, 3, f, f), clblasNotImplemented, 3);
    expect("grad", grad(2, 3, 4, f, f, f), clblasInvalidOperation, 4);
    expect("grad, one side", grad(2, 3, 4, nullptr, f, f), clblasInvalidOperation, 5);
    // sizes and strides at and beyond what is indexed
    expect("rows", quant(clblasAmdF32, top, 3, 3, 3), clblasNotImplemented, 5);
    expect("columns", quant(clblasAmdBf16, 2, top, top, top), clblasNotImplemented, 5);
    expect("stride", quant(clblasAmdBf16, 2, 3, top, 3), clblasNotImplemented, 5);
    expect("depth", gemm(2, 3, (size_t)1 << 17, (size_t)1 << 17, 3), clblasNotImplemented, 5);
    expect("gated columns", gated(2, (size_t)1 << 31, 4, 4, (size_t)1 << 31, nullptr, nullptr), clblasNotImplemented, 5);
    expect("channels of a gradient", grad(2, (size_t)1 << 20, 4, f, f, f), clblasNotImplemented, 5);
    expect("depth of a gradient", grad(2, 3, (size_t)1 << 21, f, f, f), clblasNotImplemented, 5);
    expect("most channels of a gradient", grad(2, ((size_t)1 << 20) - 320, 4, f, f, f), clblasInvalidOperation, 6);
    // values outside the enumerations
    for (int t : {-1, 3, std::numeric_limits<int>::max(), std::numeric_limits<int>::min()}) {
        expect("type", quant((clblasAmdType)t, 2, 3, 3, 3), clblasInvalidValue, 6);
        expect("gate", clblasAmdGated(clblasAmdF16, (clblasAmdGate)t, 2, 3, 4, f, 0, 4, f, 0, 4, f, 0, 4, f, 0, 3, nullptr, 0, 0, nullptr, 0, 0, nullptr),
               clblasInvalidValue, 6);
    }
    // CLBLAS_AMD_CHECK_MEM: footprints that leave 64 bits
    cba::g_knobs.check_mem = 1;
    cba::g_behind = 16;
    expect("fits", quant(clblasAmdF32, 1, 4, 4, 4), clblasSuccess, 7);
    expect("does not fit", quant(clblasAmdF32, 1, 5, 5, 5), clblasInsufficientMemMatA, 7);
    expect("wraps", quant(clblasAmdF32, top / 2, 4, top / 2, 4), clblasInsufficientMemMatA, 7);
    expect("scales", clblasAmdI8gemm(clblasAmdF16, 5, 1, 1, q, 0, 1, f, q, 0, 1, f, f, 0, 1, nullptr), clblasInsufficientMemVecX, 7);
    expect("scales of channels", clblasAmdI8gemm(clblasAmdF16, 1, 5, 1, q, 0, 1, f, q, 0, 1, f, f, 0, 5, nullptr), clblasInsufficientMemVecY, 7);
    if (failures) return 1;
    std::puts("ok");
    return 0;
}
