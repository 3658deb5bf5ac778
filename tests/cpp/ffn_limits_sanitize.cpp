// The largest sizes that the feed-forward products take and the smallest that they refuse, as the header states them, in a
// CPU build of clblas_amd/csrc/ffn_api.cpp with AddressSanitizer / UBSan.  What valid problems are handed to counts them.
#include <cstdio>

#include "../../clblas_amd/csrc/ffn.hpp"
#include "../../clblas_amd/csrc/internal.h"
#include "../../include/clblas_amd.h"

namespace cba {
static DebugKnobs g_knobs;
const DebugKnobs &knobs() { return g_knobs; }
size_t mem_behind(const void *) { return 0; }
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
static int g_calls = 0, g_gate = 0;
namespace ffn {
hipError_t quantize_rows(int, int, int, Mat, int8_t *, int64_t, float *, hipStream_t) { ++g_calls; return hipSuccess; }
hipError_t product_i8(int, int, int, int, int, Mat, const float *, Mat, const float *, Mat, const float *, OutMat, hipStream_t) {
    ++g_calls;
    return hipSuccess;
}
hipError_t gated(int, int, int, int, int, Mat, Mat, Mat, OutMat, OutMat, OutMat, hipStream_t) { ++g_calls; return hipSuccess; }
hipError_t gated_grad(int, int gate, int, int, int, Mat, Mat, Mat, Mat, Mat, Mat, OutMat, OutMat, OutMat, hipStream_t) {
    ++g_calls;
    g_gate = gate;
    return hipSuccess;
}
}  // namespace ffn
}  // namespace cba

static int failures = 0, calls = 0;
static void expect(const char *what, clblasStatus got, bool taken) {
    calls += taken;
    if (got == (taken ? clblasSuccess : clblasNotImplemented) && cba::g_calls == calls) return;
    std::fprintf(stderr, "%s: %d (%d calls, expected %d)\n", what, (int)got, cba::g_calls, calls);
    calls = cba::g_calls;
    ++failures;
}

int main() {
    static float f[4];
    static signed char q[4];
    const size_t dim = ((size_t)1 << 31) - 513, ld = (size_t)1 << 31, n = ((size_t)1 << 20) - 319, k = ((size_t)1 << 21) - 576, i8 = 131071;
    auto grad = [&](int flags, size_t M, size_t N, size_t K) {
        return clblasAmdGatedGrad(clblasAmdF16, (clblasAmdGate)(clblasAmdGelu + flags), M, N, K, f, 0, N, f, 0, K, f, 0, K, f, 0, K, f, 0, N, f, 0, N, f, 0, K, f,
                                  0, K, f, 0, K, nullptr);
    };
    for (int flags : {0, (int)clblasAmdRoundTerms}) {
        expect("most channels of a gradient", grad(flags, 2, n, 4), true);
        expect("one more", grad(flags, 2, n + 1, 4), false);
        expect("deepest rows of a gradient", grad(flags, 2, 3, k), true);
        expect("one more", grad(flags, 2, 3, k + 1), false);
        expect("most tokens of a gradient", grad(flags, dim, 3, 4), true);
        expect("one more", grad(flags, dim + 1, 3, 4), false);
        if (cba::g_gate != (int)clblasAmdGelu + flags) {
            std::fprintf(stderr, "gate %d arrived for %d\n", cba::g_gate, (int)clblasAmdGelu + flags);
            ++failures;
        }
    }
    // the terms' rows, 4 bytes a channel in whole lines of 128, stay within what the tiles address
    if ((int64_t)((n * 4 + 127) / 128 * 128) > cba::ffn::kMaxRowBytes) ++failures, std::fprintf(stderr, "rows of terms are too long\n");
    auto quant = [&](size_t M, size_t K, size_t ldx) { return clblasAmdQuantizeRows(clblasAmdF32, M, K, f, 0, ldx, q, 0, K, f, nullptr); };
    expect("most rows", quant(dim, 1, 1), true);
    expect("one more", quant(dim + 1, 1, 1), false);
    expect("longest row", quant(1, dim, dim), true);
    expect("one more", quant(1, dim + 1, dim + 1), false);
    expect("widest stride", quant(2, 1, ld), true);
    expect("one more", quant(2, 1, ld + 1), false);
    auto gemm = [&](size_t M, size_t N, size_t K) { return clblasAmdI8gemm(clblasAmdF16, M, N, K, q, 0, K, f, q, 0, K, f, f, 0, N, nullptr); };
    expect("deepest 8-bit sum", gemm(1, 1, i8), true);
    expect("one more", gemm(1, 1, i8 + 1), false);
    expect("most tokens", gemm(dim, 1, 1), true);
    expect("one more", gemm(dim + 1, 1, 1), false);
    expect("most channels", gemm(1, dim, 1), true);
    expect("one more", gemm(1, dim + 1, 1), false);
    auto gated = [&](size_t M, size_t N, size_t K, size_t ldh) {
        return clblasAmdGated(clblasAmdF16, clblasAmdSilu, M, N, K, f, 0, K, f, 0, K, f, 0, K, f, 0, ldh, nullptr, 0, 0, nullptr, 0, 0, nullptr);
    };
    expect("deepest sum", gated(1, 1, dim, 1), true);
    expect("one more", gated(1, 1, dim + 1, 1), false);
    expect("widest result", gated(1, 1, 1, ld), true);
    expect("one more", gated(1, 1, 1, ld + 1), false);
    if (failures) return 1;
    std::puts("ok");
    return 0;
}
