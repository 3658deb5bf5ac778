// Argument checks and status mapping shared by the files that implement the C ABI.
#pragma once

#include <hip/hip_runtime_api.h>

#include "../../include/clblas_amd.h"
#include "internal.h"

enum MatId { MAT_A = 0, MAT_B = 1, MAT_C = 2 };

static inline clblasStatus lead_dim_error(MatId m) {
    return m == MAT_A ? clblasInvalidLeadDimA : (m == MAT_B ? clblasInvalidLeadDimB : clblasInvalidLeadDimC);
}

static inline clblasStatus mem_error(MatId m, bool insufficient) {
    if (insufficient)
        return m == MAT_A ? clblasInsufficientMemMatA : (m == MAT_B ? clblasInsufficientMemMatB : clblasInsufficientMemMatC);
    return m == MAT_A ? clblasInvalidMatA : (m == MAT_B ? clblasInvalidMatB : clblasInvalidMatC);
}

// Restates checkMatrixSizes (generic/common.c:585-688) for a rows x cols logical matrix:
// zero dimension -> InvalidDim; ld below the number of elements that are contiguous in
// memory -> InvalidLeadDim{A,B,C}.  The reference's third outcome, InsufficientMemMat*
// (common.c:644-684), compares offset + footprint against CL_MEM_SIZE of the cl_mem.  A raw
// device pointer carries no size, so by default that code cannot arise; with the debug switch
// CLBLAS_AMD_CHECK_MEM=1 the allocation behind `base` is looked up and the same rule applied:
// (off + (lines - 1) ld + run) sizeof(T) beyond the memory behind the pointer ->
// InsufficientMemMat{A,B,C}; a pointer that no allocation holds -> InvalidMat{A,B,C} (the
// reference's answer when clGetMemObjectInfo fails).
static inline clblasStatus check_matrix_sizes(clblasOrder order, clblasTranspose trans, size_t rows, size_t cols, size_t ld,
                                MatId which, const void *base, size_t off, size_t tsize) {
    if (rows == 0 || cols == 0) return clblasInvalidDim;
    const bool rows_contiguous = (order == clblasRowMajor && trans != clblasNoTrans) ||
                                 (order == clblasColumnMajor && trans == clblasNoTrans);
    if (rows_contiguous ? (ld < rows) : (ld < cols)) return lead_dim_error(which);
    if (cba::knobs().check_mem) {
        const size_t mem = cba::mem_behind(base);
        if (mem == 0) return mem_error(which, false);
        const size_t run = rows_contiguous ? rows : cols, lines = rows_contiguous ? cols : rows;
        // ((lines - 1) ld + run + off) tsize, refusing anything that leaves 64 bits on the way
        unsigned __int128 used = (unsigned __int128)(lines - 1) * ld + run + off;
        used *= tsize;
        if (used > (unsigned __int128)mem) return mem_error(which, true);
    }
    return clblasSuccess;
}

static inline bool valid_order(clblasOrder o) { return o == clblasRowMajor || o == clblasColumnMajor; }
static inline bool valid_trans(clblasTranspose t) { return t == clblasNoTrans || t == clblasTrans || t == clblasConjTrans; }

static inline clblasStatus map_hip_error(hipError_t e) {
    if (e == hipSuccess) return clblasSuccess;
    (void)hipGetLastError();
    if (e == hipErrorOutOfMemory) return clblasOutOfResources;
    if (e == hipErrorInvalidValue) return clblasInvalidValue;
    if (e == hipErrorNotSupported) return clblasNotImplemented;
    if (e == hipErrorStreamCaptureUnsupported) return clblasInvalidOperation;  // would have had to allocate under capture
    return clblasOutOfResources;
}

// Kernels index rows and columns with 32-bit ints (reference: cl_uint, xgemm.cc:362-372); the largest
// index they form is a dimension rounded up to a whole tile (edge 256) plus one vector, so dimensions
// stop one tile short of 2^31.
static const size_t kMaxDim = 0x7fffffff - 512;
