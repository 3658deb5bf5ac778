// The feed-forward products' launchers, and what is shared by their host and device code.  Not part of the C ABI.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

namespace cba {
namespace ffn {

enum ElemKind { ET_I8 = 0, ET_F16 = 1, ET_BF16 = 2 };                    // operands of a product
enum OutKind { OT_F32 = 0, OT_F16 = 1, OT_BF16 = 2 };                    // results (numbered as clblasAmdType)
enum GateKind { GATE_SILU = 0, GATE_GELU = 1, GATE_GELU_TANH = 2 };      // numbered as clblasAmdGate
enum { ROUND_TERMS = 0x100 };                                            // added to the gate of gated_grad()

// One product, as the kernels take it.  Strides and lengths of the operands count bytes, those of results elements.
struct Product {
    const void *A[2];       // [batch entry]
    const void *B[2];       // gate's and other weight
    int64_t lda, ldb[2];
    int64_t a_bytes, b_bytes[2];  // from the first element to behind the last one
    int64_t k_bytes;        // depth (two bytes per index also where an operand's rows run across it)
    int part_steps;         // steps of depth after which B[1] takes B[0]'s place (GATED has both at once: unused)
    int64_t a_jump;         // and by how much more than a step A's place moves on then
    const float *unscale;   // f16 gradients: what the sums are multiplied by
    const float *scale_a;   // 8-bit operands: one scale per row of A / B
    const float *scale_b[2];
    void *C[2];             // [batch entry]
    int64_t ldc[2];
    void *save[2];          // the gate's two products, if they are wanted
    int64_t ld_save[2];
    int M, N;               // rows of A / rows of one B: C is M x N
    int batch;              // 1, or 2: two products A[z] B^T -> C[z]
    int out_type, gate;
    int tiles_m, tiles_n, group_m;
    int splits, steps_per_split;  // depth ranges, and their length in steps of 128 bytes
    uint32_t *ws;           // partial sums of a split product
    int64_t ws_ld, ws_plane, ws_split;
};

struct ProductPair {
    Product p[2];
};

// A matrix as the caller gave it: rows of `ld` elements.
struct Mat {
    const void *ptr = nullptr;
    int64_t ld = 0;
};
struct OutMat {
    void *ptr = nullptr;
    int64_t ld = 0;
};

// Rows of a tiled operand are addressed across a tile with 32-bit offsets: at most this many bytes from row to row.
constexpr int64_t kMaxRowBytes = ((int64_t)1 << 22) - 1024;

hipError_t quantize_rows(int type, int M, int K, Mat X, int8_t *Q, int64_t ldq, float *scale, hipStream_t stream);
// C = A B^T (8-bit, scaled), or with Bu: act(A Bg^T) o (A Bu^T).
hipError_t product_i8(int out_type, int gate, int M, int N, int K, Mat A, const float *sA, Mat Bg, const float *sBg, Mat Bu,
                      const float *sBu, OutMat C, hipStream_t stream);
hipError_t gated(int type, int gate, int M, int N, int K, Mat X, Mat Wg, Mat Wu, OutMat H, OutMat G, OutMat U, hipStream_t stream);
// dX = dG Wg + dU Wu, dWg = dG^T X, dWu = dU^T X; gate + ROUND_TERMS: dG and dU rounded to one 16-bit number each.
hipError_t gated_grad(int type, int gate, int M, int N, int K, Mat dH, Mat X, Mat Wg, Mat Wu, Mat G, Mat U, OutMat dX, OutMat dWg,
                      OutMat dWu, hipStream_t stream);

}  // namespace ffn
}  // namespace cba
