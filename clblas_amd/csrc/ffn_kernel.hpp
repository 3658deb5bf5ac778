// Device code of the feed-forward products: 16-bit and 8-bit MFMA products of two matrices whose rows run along
// the depth, with the gate or the scales applied before the result is stored.
//
//     acc(m, n) = sum_k A(m, k) B(n, k)          A: one row per token, B: one row per channel
//
// A row of either operand is a plain run of bytes along k, and 16 of them are what one lane feeds an MFMA with,
// whatever the type (8 x 16 bits or 16 x 8 bits).  So the whole data path counts bytes: a workgroup steps through
// the depth 128 bytes at a time, and only the MFMA itself and the accumulator (float / int32) know the type.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ffn.hpp"
#include "internal.h"

namespace cba {
namespace ffn {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void_t;

template <int ET> struct ElemOf;
template <> struct ElemOf<ET_I8> { typedef int8_t type; typedef int Acc; };
template <> struct ElemOf<ET_F16> { typedef _Float16 type; typedef float Acc; };
template <> struct ElemOf<ET_BF16> { typedef __bf16 type; typedef float Acc; };

// One MFMA on MB x MB blocks.  Lane l holds row l % MB of either operand, the 16 bytes that start at byte
// 16 (l / MB) of the instruction's depth (MB = 16: 64 bytes deep, MB = 32: 32 bytes).  Of the result it holds column
// l % MB and, for every group q of four elements, rows 4 (64 / MB q + l / MB) .. + 3.
template <int ET, int MB> struct Mfma;
#define CBA_FFN_MFMA(ET, MB, ACC, OPND, BUILTIN)                                                              \
    template <> struct Mfma<ET, MB> {                                                                         \
        typedef ACC Acc;                                                                                      \
        static __device__ __forceinline__ Acc run(u32x4 a, u32x4 b, Acc c) {                                  \
            return BUILTIN(__builtin_bit_cast(OPND, a), __builtin_bit_cast(OPND, b), c, 0, 0, 0);             \
        }                                                                                                     \
    };
CBA_FFN_MFMA(ET_I8, 16, i32x4, i32x4, __builtin_amdgcn_mfma_i32_16x16x64_i8)
CBA_FFN_MFMA(ET_F16, 16, f32x4, f16x8, __builtin_amdgcn_mfma_f32_16x16x32_f16)
CBA_FFN_MFMA(ET_BF16, 16, f32x4, bf16x8, __builtin_amdgcn_mfma_f32_16x16x32_bf16)
CBA_FFN_MFMA(ET_I8, 32, i32x16, i32x4, __builtin_amdgcn_mfma_i32_32x32x32_i8)
CBA_FFN_MFMA(ET_F16, 32, f32x16, f16x8, __builtin_amdgcn_mfma_f32_32x32x16_f16)
CBA_FFN_MFMA(ET_BF16, 32, f32x16, bf16x8, __builtin_amdgcn_mfma_f32_32x32x16_bf16)
#undef CBA_FFN_MFMA

// ---- elements of the result ----

static __device__ __forceinline__ float gate_value(int gate, float g) {
    if (gate == GATE_GELU) return g * 0.5f * erfcf(-0.70710678f * g);
    // SiLU is g sigmoid(g); the tanh form of GELU is g sigmoid(2 z), z = sqrt(2 / pi) (g + 0.044715 g^3)
    const float x = gate == GATE_SILU ? g : 1.59576912f * (g + 0.044715f * g * g * g);
    return g * __builtin_amdgcn_rcpf(1.f + __expf(-x));
}

// act(g) and act'(g).  The slope is flat (0 or 1 to the last bit) far from zero; |g| is cut off there, so that the
// products in it cannot turn into 0 * inf.  NaN passes through the comparisons.
static __device__ __forceinline__ void gate_value_and_slope(int gate, float g, float &value, float &slope) {
    value = gate_value(gate, g);
    const float c = g > 128.f ? 128.f : (g < -128.f ? -128.f : g);
    if (gate == GATE_GELU) {
        slope = 0.5f * erfcf(-0.70710678f * c) + c * 0.39894228f * __expf(-0.5f * c * c);
        return;
    }
    float x = c, dx = 1.f;
    if (gate == GATE_GELU_TANH) {
        x = 1.59576912f * (c + 0.044715f * c * c * c);
        dx = 1.59576912f * (1.f + 0.134145f * c * c);
    }
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-x)), t = __builtin_amdgcn_rcpf(1.f + __expf(x));  // t = 1 - s
    slope = s + c * s * t * dx;
}

// Rounds to the storage type (to nearest, ties to even); the only rounding below 32 bits on the way to a result.
template <int OT> struct Store;
template <> struct Store<OT_F32> {
    typedef float type;
    static __device__ __forceinline__ float of(float x) { return x; }
};
template <> struct Store<OT_F16> {
    typedef _Float16 type;
    static __device__ __forceinline__ _Float16 of(float x) { return (_Float16)x; }
};
template <> struct Store<OT_BF16> {
    typedef __bf16 type;
    static __device__ __forceinline__ __bf16 of(float x) { return (__bf16)x; }
};

// x[0 .. valid) to p (element-aligned), valid <= 4.
template <int OT> static __device__ __forceinline__ void store4_as(void *base, int64_t at, const float *x, int valid) {
    typedef typename Store<OT>::type T;
    T *p = static_cast<T *>(base) + at;
    T v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = Store<OT>::of(x[e]);
    if (valid >= 4) {
        __builtin_memcpy(p, v, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < valid) p[e] = v[e];
    }
}
static __device__ __forceinline__ void store4(int ot, void *base, int64_t at, const float *x, int valid) {
    if (ot == OT_BF16) store4_as<OT_BF16>(base, at, x, valid);
    else if (ot == OT_F16) store4_as<OT_F16>(base, at, x, valid);
    else store4_as<OT_F32>(base, at, x, valid);
}

// Four neighbouring results (m, n .. n + 3) from their accumulators; `first` is the plain product or the gate's.
template <int ET, bool GATED>
static __device__ __forceinline__ void finish4(const Product &p, int z, int m, int n, const float *first, const float *second) {
    float x[4], u[4];
    const int valid = p.N - n;
    float sa = 1.f;
    if (ET == ET_I8) sa = p.scale_a[m];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = first[e];
        if (GATED) u[e] = second[e];
        if (ET == ET_I8 && e < valid) {
            x[e] = x[e] * sa * p.scale_b[0][n + e];
            if (GATED) u[e] = u[e] * sa * p.scale_b[1][n + e];
        }
    }
    if (GATED) {
        if (p.save[0]) {
            store4(p.out_type, p.save[0], (int64_t)m * p.ld_save[0] + n, x, valid);
            store4(p.out_type, p.save[1], (int64_t)m * p.ld_save[1] + n, u, valid);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = gate_value(p.gate, x[e]) * u[e];
    }
    store4(p.out_type, p.C[z], (int64_t)m * p.ldc[z] + n, x, valid);
}

static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void *p, int64_t bytes_left) {
    // An access reaches at most 2 GiB from its descriptor's base (the host sees to the row strides); what lies
    // beyond the operand's last byte reads as zero.  The length is rounded up to whole dwords: a 16-bit operand may
    // end in the middle of one.
    const int64_t n = bytes_left <= 0 ? 0 : (bytes_left > 0x7ffffffcLL ? 0x7ffffffcLL : ((bytes_left + 3) & ~3LL));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)n, 0x00020000);
}

// Workgroup id -> entry of the tile list: ids are handed to the 8 XCDs in turn, and each XCD has an L2 of its own, so
// every XCD gets a contiguous piece of the list.
static __device__ __forceinline__ int xcd_contiguous(int id, int total) {
    const int per = total >> 3, rem = total & 7, xcd = id & 7, q = id >> 3;
    return xcd * per + (xcd < rem ? xcd : rem) + q;
}

// ---- the tiled product ----
//
// A workgroup computes a BM x BN tile of accumulators with waves of WM x WN.  Both operands travel HBM -> LDS without
// passing through registers (buffer_load ... lds, 16 bytes per lane), 128 bytes of depth at a time, as rows of eight
// 16-byte slots; slot s of row r is kept in place s ^ (r % 8), so that the eight rows that one pass of a fragment read
// touches lie in different banks.  GATED: the BN rows are BN / 2 channels of either weight, arranged per wave (WN / 2
// of the gate's, then the same WN / 2 channels of the other's), so that both factors of a result sit in the same lane.
template <int ET_, int MB_, int BM_, int BN_, int WM_, int WN_, bool GATED_> struct TileCfg {
    static constexpr int ET = ET_, MB = MB_, BM = BM_, BN = BN_, WM = WM_, WN = WN_;
    static constexpr bool GATED = GATED_;
    static constexpr int WAVES_M = BM / WM, WAVES_N = BN / WN, WAVES = WAVES_M * WAVES_N, THREADS = 64 * WAVES;
    static constexpr int CHANNELS = GATED ? BN / 2 : BN;  // columns of the result per tile
    static constexpr int TM = WM / MB, TN = WN / MB;
    static constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // wave-wide loads per step (8 rows each)
    static constexpr int STAGE = (BM + BN) * 128;
    static constexpr int LDS = 2 * STAGE;
    static constexpr int KSTEPS = MB == 16 ? 2 : 4;  // MFMAs that take up 128 bytes of depth
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "rows divide over the waves");
    static_assert(!GATED || (WN / 2) % MB == 0, "the halves of a wave's columns are whole blocks");
    static_assert(!GATED || (WN / 2) % 8 == 0, "one load stays inside one weight");
};

template <typename Cfg> __global__ __launch_bounds__(Cfg::THREADS, 1) void tile_kernel(Product p) {
    extern __shared__ __attribute__((aligned(128))) char lds[];
    constexpr int MB = Cfg::MB, BM = Cfg::BM;
    typedef Mfma<Cfg::ET, MB> Op;
    typedef typename Op::Acc Acc;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / Cfg::WAVES_N, wn = wave % Cfg::WAVES_N;

    // tile, split and batch entry of this workgroup
    const int tiles = p.tiles_m * p.tiles_n;
    int id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int split = id / (tiles * p.batch);
    id -= split * tiles * p.batch;
    const int z = id / tiles;
    id -= z * tiles;
    const int per_group = p.group_m * p.tiles_n, grp = id / per_group, first_m = grp * p.group_m;
    const int gm = p.tiles_m - first_m < p.group_m ? p.tiles_m - first_m : p.group_m;
    const int r_in = id - grp * per_group;
    const int m0 = (first_m + r_in % gm) * BM, n0 = r_in / gm * Cfg::CHANNELS;

    const int64_t k0 = (int64_t)split * p.steps_per_split * 128;  // bytes
    const int64_t k_left = p.k_bytes - k0;
    const int steps_all = (int)((k_left + 127) >> 7);
    const int steps = steps_all < p.steps_per_split ? steps_all : p.steps_per_split;

    // Operands from this tile's first element on, and this lane's place in the rows it loads.
    const char *a_base = static_cast<const char *>(p.A[z]) + (int64_t)m0 * p.lda + k0;
    int64_t a_left = p.a_bytes - (int64_t)m0 * p.lda - k0;
    const char *b_base[2];
    int64_t b_left[2];
#pragma unroll
    for (int h = 0; h < (Cfg::GATED ? 2 : 1); ++h) {
        b_base[h] = static_cast<const char *>(p.B[h]) + (int64_t)n0 * p.ldb[h] + k0;
        b_left[h] = p.b_bytes[h] - (int64_t)n0 * p.ldb[h] - k0;
    }
    const int row8 = lane >> 3, slot = (lane & 7) ^ row8;
    // (in the last step the slots beyond the depth are sent out of range and read as zero)
    const int last_slots = (int)((k_left - (int64_t)(steps - 1) * 128) >> 4);
    constexpr uint32_t kOutside = 0x80000000u;

    auto issue = [&](int step, int stage) {
        char *dst = lds + stage * Cfg::STAGE;
        const bool out = step == steps - 1 && slot >= last_slots;
        const int64_t at = (int64_t)step * 128;
        const __amdgpu_buffer_rsrc_t ra = rsrc_of(a_base + at, a_left - at);
#pragma unroll
        for (int i = 0; i < Cfg::LA; ++i) {
            const int row = (wave + i * Cfg::WAVES) * 8;
            const uint32_t off = (uint32_t)((row + row8) * (int)p.lda + slot * 16);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void_t *)(dst + row * 128), 16, (int)(out ? kOutside : off), 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < Cfg::LB; ++i) {
            const int row = (wave + i * Cfg::WAVES) * 8;
            const int h = Cfg::GATED ? (row % Cfg::WN) / (Cfg::WN / 2) : 0;
            const int ch = Cfg::GATED ? row / Cfg::WN * (Cfg::WN / 2) + row % (Cfg::WN / 2) : row;
            const __amdgpu_buffer_rsrc_t rb = rsrc_of((h ? b_base[1] : b_base[0]) + at, (h ? b_left[1] : b_left[0]) - at);
            const uint32_t off = (uint32_t)((ch + row8) * (int)(h ? p.ldb[1] : p.ldb[0]) + slot * 16);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void_t *)(dst + (BM + row) * 128), 16, (int)(out ? kOutside : off), 0, 0, 0);
        }
    };

    Acc acc[Cfg::TM][Cfg::TN];
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i)
#pragma unroll
        for (int j = 0; j < Cfg::TN; ++j) acc[i][j] = Acc{};

    const int r = lane % MB, g = lane / MB;
    const int frag0 = r * 128 + ((g ^ (r & 7)) << 4);
    if (steps > 0) issue(0, 0);
    for (int s = 0; s < steps; ++s) {
        __builtin_amdgcn_s_waitcnt(0xf70);  // vmcnt(0)
        __syncthreads();
        if (s + 1 < steps) issue(s + 1, (s + 1) & 1);
        const char *as = lds + (s & 1) * Cfg::STAGE + wm * Cfg::WM * 128;
        const char *bs = lds + (s & 1) * Cfg::STAGE + (BM + wn * Cfg::WN) * 128;
#pragma unroll
        for (int kk = 0; kk < Cfg::KSTEPS; ++kk) {
            const int off = frag0 ^ (kk * (128 / Cfg::KSTEPS));
            u32x4 a[Cfg::TM], b[Cfg::TN];
#pragma unroll
            for (int i = 0; i < Cfg::TM; ++i) a[i] = *reinterpret_cast<const u32x4 *>(as + i * MB * 128 + off);
#pragma unroll
            for (int j = 0; j < Cfg::TN; ++j) b[j] = *reinterpret_cast<const u32x4 *>(bs + j * MB * 128 + off);
            // the weights are the instruction's first operand: a lane then holds one token's neighbouring channels
#pragma unroll
            for (int i = 0; i < Cfg::TM; ++i)
#pragma unroll
                for (int j = 0; j < Cfg::TN; ++j) acc[i][j] = Op::run(b[j], a[i], acc[i][j]);
        }
    }

    constexpr int HALF = Cfg::GATED ? Cfg::TN / 2 : Cfg::TN, QUADS = MB * MB / 64 / 4;
#pragma unroll
    for (int i = 0; i < Cfg::TM; ++i) {
        const int m = m0 + wm * Cfg::WM + i * MB + r;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < HALF; ++j)
#pragma unroll
            for (int q = 0; q < QUADS; ++q) {
                const int n = n0 + wn * (HALF * MB) + j * MB + 4 * (64 / MB * q + g);
                if (n >= p.N) continue;
                constexpr int J2 = Cfg::GATED ? HALF : 0;
                if (p.splits > 1) {
                    typedef typename ElemOf<Cfg::ET>::Acc S;
                    typedef S sx4 __attribute__((ext_vector_type(4)));
                    S *w = reinterpret_cast<S *>(p.ws) + (int64_t)split * p.ws_split + (int64_t)z * p.ws_plane + (int64_t)m * p.ws_ld + n;
                    sx4 v, v2;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = acc[i][j][4 * q + e];
                        v2[e] = acc[i][j + J2][4 * q + e];
                    }
                    *reinterpret_cast<sx4 *>(w) = v;
                    if (Cfg::GATED) *reinterpret_cast<sx4 *>(w + p.ws_plane) = v2;
                } else {
                    float x[4], u[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = (float)acc[i][j][4 * q + e];
                        u[e] = (float)acc[i][j + J2][4 * q + e];
                    }
                    finish4<Cfg::ET, Cfg::GATED>(p, z, m, n, x, u);
                }
            }
    }
}

// Adds up the depth ranges of a split product (in their order, whatever finished first) and finishes the results.
// Partial sums: [range][plane][row][column], rows of ws_ld (a multiple of 4) 32-bit sums; planes are the batch's
// entries or the gate's two products.
template <int ET, bool GATED> __global__ __launch_bounds__(256) void join_kernel(Product p) {
    const int64_t per_row = p.ws_ld >> 2, per_plane = per_row * p.M, total = per_plane * p.batch;
    typedef typename ElemOf<ET>::Acc S;
    typedef S sx4 __attribute__((ext_vector_type(4)));
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int z = (int)(t / per_plane);
        const int64_t u = t - (int64_t)z * per_plane;
        const int m = (int)(u / per_row), n = (int)(u - (int64_t)m * per_row) * 4;
        const uint32_t *w = p.ws + (int64_t)z * p.ws_plane + (int64_t)m * p.ws_ld + n;
        sx4 a = {}, b = {};
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s, w += p.ws_split) {
            a += *reinterpret_cast<const sx4 *>(w);
            if (GATED) b += *reinterpret_cast<const sx4 *>(w + p.ws_plane);
        }
        float x[4] = {(float)a[0], (float)a[1], (float)a[2], (float)a[3]};
        float y[4] = {(float)b[0], (float)b[1], (float)b[2], (float)b[3]};
        finish4<ET, GATED>(p, z, m, n, x, y);
    }
}

}  // namespace ffn
}  // namespace cba
