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
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void_t;

template <int ET> struct ElemOf;
template <> struct ElemOf<ET_I8> { typedef int8_t type; typedef int Acc; };
template <> struct ElemOf<ET_F16> { typedef _Float16 type; typedef float Acc; };
template <> struct ElemOf<ET_BF16> { typedef __bf16 type; typedef float Acc; };

// One MFMA on 16 x 16 blocks, 64 bytes deep.  Lane l holds row l % 16 of either operand, the 16 bytes from byte
// 16 (l / 16) of the depth on; of the result it holds column l % 16, rows 4 (l / 16) .. + 3.
template <int ET> struct Mfma;
#define CBA_FFN_MFMA(ET, ACC, OPND, BUILTIN)                                                            \
    template <> struct Mfma<ET> {                                                                       \
        typedef ACC Acc;                                                                                \
        static __device__ __forceinline__ Acc run(u32x4 a, u32x4 b, Acc c) {                            \
            return BUILTIN(__builtin_bit_cast(OPND, a), __builtin_bit_cast(OPND, b), c, 0, 0, 0);       \
        }                                                                                               \
    };
CBA_FFN_MFMA(ET_I8, i32x4, i32x4, __builtin_amdgcn_mfma_i32_16x16x64_i8)
CBA_FFN_MFMA(ET_F16, f32x4, f16x8, __builtin_amdgcn_mfma_f32_16x16x32_f16)
CBA_FFN_MFMA(ET_BF16, f32x4, bf16x8, __builtin_amdgcn_mfma_f32_16x16x32_bf16)
#undef CBA_FFN_MFMA

// A kernel's Product where the launch left it.  What is needed once per tile is read from there when it is needed, through a
// pointer that the compiler cannot see through: it would keep some sixty scalar registers alive across the inner loop.
typedef const __attribute__((address_space(4))) Product Args;
static __device__ __forceinline__ Args *kernel_args() { return (Args *)__builtin_amdgcn_kernarg_segment_ptr(); }
static __device__ __forceinline__ Args &fresh(Args *p) {
    asm volatile("" : "+s"(p));
    return *p;
}

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
    const float c = g > 128.f ? 128.f : (g < -128.f ? -128.f : g);
    if (gate == GATE_GELU) {
        const float p = 0.5f * erfcf(-0.70710678f * c);
        value = g * p;
        slope = p + c * 0.39894228f * __expf(-0.5f * c * c);
        return;
    }
    float x = c, dx = 1.f;
    if (gate == GATE_GELU_TANH) {
        x = 1.59576912f * (c + 0.044715f * c * c * c);
        dx = 1.59576912f * (1.f + 0.134145f * c * c);
    }
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-x)), t = __builtin_amdgcn_rcpf(1.f + __expf(x));  // t = 1 - s
    value = g * s;
    slope = s + c * s * t * dx;
}

// Rounds to the storage type (to nearest, ties to even): the one rounding of a result.
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
static __device__ __forceinline__ void finish4(Args &p, int z, int m, int n, const float *first, const float *second) {
    float x[4], u[4];
    const int valid = p.N - n;
    float sa = 1.f;
    if (ET == ET_I8) sa = p.scale_a[m];
    if (ET == ET_F16 && !GATED) sa = *p.unscale;  // (the gradients)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = first[e];
        if (GATED) u[e] = second[e];
        if (ET == ET_F16 && !GATED) x[e] *= sa;
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
    // end in the middle of one.  (In 32-bit scalar steps: the compiler compares 64 bits on the vector unit.)
    const int high = (int)(bytes_left >> 31);
    uint32_t n = ((uint32_t)bytes_left + 3) & ~3u;
    n = high > 0 ? 0x7ffffffcu : n;
    n = high < 0 ? 0u : n;
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
// A workgroup computes BM x BN tiles of accumulators with waves of WM x WN.  Both operands travel HBM -> LDS without
// passing through registers (buffer_load ... lds, 16 bytes per lane), one step of 128 bytes (64 or 128 elements, two MFMAs
// deep) at a time, through a ring of S stages.  (Steps of 64 bytes allow a finer ring, but fetch half cache lines: 8192 x
// 12288 x 4096 gated in 1370-1450 us against 1320.)  Workgroups stay: each walks its part of the list of tiles, and the ring
// runs on across the borders, so that the next tile's first steps are on their way while results are stored.
//
// An operand lies in memory either with its rows along the depth (ALONG_K: the forward products) or across it
// (ACROSS_K, 16-bit types: a row per depth index, as the gradients meet weights and activations).
// TERMS (B across the depth): every value of A is the sum of two 16-bit numbers, first terms and second ones of 32 values
// side by side (64 bytes each).  A step is then 32 deep: its first MFMAs take the first terms, its second ones the others, and
// both meet the same operands of B, which are read once.
//   ALONG_K   LDS image: a row of eight 16-byte slots per tile row, slot s of row r in place s ^ (r % 8), so that the
//             eight rows that one pass of a fragment read touches lie in different banks.
//   ACROSS_K  LDS image: 64 rows of depth (TERMS: 32, of A for either term), each the tile's edge long.  A lane reads V neighbouring columns (8 or 4 bytes) of
//             its 8 rows of depth and swaps 16-bit halves between row pairs (v_perm_b32): that gives it the operands
//             of V MFMA blocks, block e holding columns e, V + e, 2 V + e ...  (The transposing LDS reads would do
//             this without the swaps, but the compiler makes each of them wait for every load into LDS that is in
//             flight: 2048 x 4096 x 4096, both operands across, 231 us.)
// GATED: the BN rows of weights are BN / 2 channels of either weight, arranged per wave (WN / 2 of the gate's, then the
// same WN / 2 channels of the other's), so that both factors of a result end up in the same lane.
enum Lay { ALONG_K = 0, ACROSS_K = 1 };

template <int ET_, int BM_, int BN_, int WM_, int WN_, int S_, bool GATED_, Lay LAYA_ = ALONG_K, Lay LAYB_ = ALONG_K, bool TERMS_ = false> struct TileCfg {
    static constexpr int ET = ET_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_;
    static constexpr bool GATED = GATED_;
    static constexpr Lay LAYA = LAYA_, LAYB = LAYB_;
    static constexpr bool SPLITS = BM * BN < 65536;    // the depth may be cut into ranges
    static constexpr int WAVES_M = BM / WM, WAVES_N = BN / WN, WAVES = WAVES_M * WAVES_N, THREADS = 64 * WAVES;
    static constexpr int CHANNELS = GATED ? BN / 2 : BN;  // columns of the result per tile
    // B in two parts, one after the other along the depth (the gradient of the input: both weights)
    static constexpr bool PARTS = LAYA == ALONG_K && LAYB == ACROSS_K;
    static constexpr bool TERMS = TERMS_;
    static constexpr int DEPTH = TERMS ? 32 : 64;  // of a step, 16-bit types
    static constexpr int TM = WM / 16, TN = WN / 16;
    static constexpr int A_BYTES = BM * 128, B_BYTES = BN * (TERMS ? 64 : 128);
    static constexpr int LA = A_BYTES / 1024 / WAVES, LB = B_BYTES / 1024 / WAVES;  // wave-wide loads per step (1 KiB each)
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int LDS = S * STAGE;
    static_assert(A_BYTES % (1024 * WAVES) == 0 && B_BYTES % (1024 * WAVES) == 0, "an operand's loads divide over the waves");
    static_assert(!TERMS || LAYB == ACROSS_K, "");
    static_assert(!GATED || (WN / 2) % 16 == 0, "the halves of a wave's columns are whole blocks, and whole loads");
    static_assert(!GATED || LAYB == ALONG_K, "");
    static_assert(ET != ET_I8 || (LAYA == ALONG_K && LAYB == ALONG_K), "half swaps are for 16-bit types");
    static_assert(LDS <= 160 * 1024 && S >= 2 && (S - 1) * (LA + LB) < 64, "");
};

// How one wave-wide load fills its 1 KiB of an operand's LDS image.  X: tile edge.
template <int X, Lay LAY> struct Image {
    static constexpr int PER_ROW = LAY == ALONG_K ? 8 : X / 8;  // 16-byte slots
    static constexpr int ROW = PER_ROW * 16;                    // bytes
    static constexpr int ROWS_PER_LOAD = 64 / PER_ROW;
    static __device__ __forceinline__ int swizzle(int row) {
        if (LAY == ALONG_K) return row & 7;
        return PER_ROW >= 16 ? ((row >> 3) & 1) << 3 : 0;  // (lane groups of a read are eight rows apart)
    }
    // Row and 16-byte slot (of memory) that this lane fetches in wave-wide load `q`.
    static __device__ __forceinline__ int row_of(int q, int lane) { return q * ROWS_PER_LOAD + lane / PER_ROW; }
    static __device__ __forceinline__ int slot_of(int q, int lane) { return (lane % PER_ROW) ^ swizzle(row_of(q, lane)); }
};

// MFMA operands of NBLK blocks of 16 rows, from tile row x0 of the image on, for either MFMA (kk) of a step.  read() fetches
// as many registers as one block takes; ready() turns the V blocks of a group, read in raw form, into operands.
template <int X, Lay LAY, int NBLK> struct Fragments {
    typedef Image<X, LAY> Im;
    static constexpr int V = LAY == ALONG_K ? 1 : NBLK % 4 == 0 ? 4 : 2;  // blocks per group
    static_assert(NBLK % V == 0, "");
    int off[LAY == ALONG_K ? 2 : NBLK / V];
    __device__ __forceinline__ void init(int lane, int x0) {
        const int r = lane & 15, g = lane >> 4;
        if constexpr (LAY == ALONG_K) {
            off[0] = (x0 + r) * Im::ROW + ((g ^ (r & 7)) << 4);
            off[1] = off[0] ^ 64;
        } else {
#pragma unroll
            for (int u = 0; u < NBLK / V; ++u) {
                const int at = (x0 + u * 16 * V + V * r) * 2;
                off[u] = 8 * g * Im::ROW + (((at >> 4) ^ Im::swizzle(8 * g)) << 4) + (at & 15);
            }
        }
    }
    __device__ __forceinline__ u32x4 read(const char *base, int j, int kk) const {
        if constexpr (LAY == ALONG_K) {
            return *reinterpret_cast<const u32x4 *>(base + off[kk] + j * 16 * Im::ROW);
        } else if constexpr (V == 4) {
            const char *at = base + off[j / 4] + (32 * kk + 2 * (j % 4)) * Im::ROW;
            const u32x2 x = *reinterpret_cast<const u32x2 *>(at), y = *reinterpret_cast<const u32x2 *>(at + Im::ROW);
            return u32x4{x[0], x[1], y[0], y[1]};
        } else {
            const char *at = base + off[j / 2] + (32 * kk + 4 * (j % 2)) * Im::ROW;
            return u32x4{*reinterpret_cast<const uint32_t *>(at), *reinterpret_cast<const uint32_t *>(at + Im::ROW),
                         *reinterpret_cast<const uint32_t *>(at + 2 * Im::ROW), *reinterpret_cast<const uint32_t *>(at + 3 * Im::ROW)};
        }
    }
    static __device__ __forceinline__ uint32_t halves(uint32_t row, uint32_t next_row, int e) {
        return __builtin_amdgcn_perm(next_row, row, e & 1 ? 0x07060302u : 0x05040100u);
    }
    // f: the V quadruples of registers of one group
    static __device__ __forceinline__ void ready(u32x4 *f) {
        if constexpr (V == 4) {
            u32x4 o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int q = 0; q < 4; ++q) o[e][q] = halves(f[q][e >> 1], f[q][2 + (e >> 1)], e);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = o[e];
        } else if constexpr (V == 2) {
            u32x4 o[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int q = 0; q < 4; ++q) o[e][q] = halves(f[q >> 1][2 * (q & 1)], f[q >> 1][2 * (q & 1) + 1], e);
#pragma unroll
            for (int e = 0; e < 2; ++e) f[e] = o[e];
        }
    }
    // Row (within the wave's) that lane place r of block j stands for.
    static __device__ __forceinline__ int row(int j, int r) { return V == 1 ? 16 * j + r : j / V * (16 * V) + V * r + j % V; }
};

// s_waitcnt immediates (gfx9: vmcnt in bits 3:0 and 15:14, expcnt 6:4, lgkmcnt 11:8)
#define CBA_FFN_WAIT_VM(n) __builtin_amdgcn_s_waitcnt((((n) & 0xf) | (((n) >> 4) << 14) | (0x7 << 4) | (0xf << 8)))
#define CBA_FFN_WAIT_LDS() __builtin_amdgcn_s_waitcnt((0xf | (3 << 14) | (0x7 << 4)))

// Where entry `id` of the list of tiles, batch entries and depth ranges lies.
struct TileAt {
    int m0, n0, z, split, first_step;
    int steps;        // of the tile
    int whole, rest;  // steps of 128 bytes from first_step to the end of the depth, and the bytes behind them
    // Bytes of the depth in step s.
    __device__ __forceinline__ int bytes(int s) const {
        const int behind = s == whole ? rest : 0;
        return s < whole ? 128 : behind;
    }
};
template <typename Cfg> static __device__ __forceinline__ TileAt tile_at(Args &p, int id) {
    TileAt t;
    const int tiles = p.tiles_m * p.tiles_n;
    t.split = 0;
    if (Cfg::SPLITS) {
        t.split = id / (tiles * p.batch);
        id -= t.split * tiles * p.batch;
    }
    t.z = id / tiles;
    id -= t.z * tiles;
    // groups of group_m tile rows, column by column: tiles that run together share both operands' rows in an L2
    const int per_group = p.group_m * p.tiles_n, grp = id / per_group, first_m = grp * p.group_m;
    const int gm = p.tiles_m - first_m < p.group_m ? p.tiles_m - first_m : p.group_m;
    const int in_group = id - grp * per_group;
    t.m0 = (first_m + in_group % gm) * Cfg::BM;
    t.n0 = in_group / gm * Cfg::CHANNELS;
    t.first_step = Cfg::SPLITS ? t.split * p.steps_per_split : 0;
    t.whole = (int)(p.k_bytes >> 7) - t.first_step;
    t.rest = (int)(p.k_bytes & 127);
    const int all = t.whole + (t.rest > 0);
    t.steps = Cfg::SPLITS && all > p.steps_per_split ? p.steps_per_split : all;
    return t;
}

// From a wave's accumulators to memory.  A lane has four neighbouring columns of a row per quad; two quads make 16 bytes of a
// 16-bit result.  ALONG_K: quad j holds columns 16 j + 4 g on; lanes 16 apart exchange halves (v_permlane16_swap), after which
// an even lane group g has columns 4 g .. 4 g + 7 of block j and its odd neighbour those of block j + 1, and a store writes
// 64 bytes of each of 16 rows.  (8 bytes per lane: 32 bytes a row, 16 x more often half a cache line; gated 8192 x
// 12288 x 4096 with G and U stored 1330 us, this 1273.)  ACROSS_K: element e of a quad comes from the e-th block of a group, and two quads
// are neighbours anyway.
template <typename Cfg> struct Results {
    typedef Fragments<Cfg::BM, Cfg::LAYA, Cfg::TM> FragA;
    static constexpr int V = Fragments<Cfg::BN, Cfg::LAYB, Cfg::TN>::V;
    static constexpr int QUADS = Cfg::GATED ? Cfg::TN / 2 : Cfg::TN, COLUMNS = 16 * QUADS;  // of a wave
    typedef typename Mfma<Cfg::ET>::Acc Acc;
    static __device__ __forceinline__ int column(int j, int g) {
        return V == 1 ? 16 * j + 4 * g : V == 4 ? j / 4 * 64 + 16 * g + 4 * (j % 4) : j / 2 * 32 + 8 * g + 4 * (j % 2);
    }
    static __device__ __forceinline__ Acc quad(const Acc (&acc)[Cfg::TN], int j) {
        Acc x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = V == 1 ? acc[j][e] : V == 4 ? acc[j / 4 * 4 + e][j % 4] : acc[j / 2 * 2 + (e & 1)][2 * (j % 2) + (e >> 1)];
        return x;
    }
    // Row m's quads to `base` (rows of ld elements, N columns), from column n on.
    template <int OT> static __device__ __forceinline__ void row(void *base, int64_t ld, int N, int m, int n, int g, const float (&x)[QUADS][4]) {
        typedef typename Store<OT>::type T;
        T *to = static_cast<T *>(base) + (int64_t)m * ld;
        if constexpr (OT != OT_F32 && QUADS % 2 == 0) {
#pragma unroll
            for (int j = 0; j < QUADS; j += 2) {
                union {
                    T v[8];
                    uint32_t d[4];
                } u;
#pragma unroll
                for (int e = 0; e < 8; ++e) u.v[e] = Store<OT>::of(x[j + e / 4][e % 4]);
                int at = n + column(j, g);
                if (V == 1) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const auto s = __builtin_amdgcn_permlane16_swap(u.d[h], u.d[2 + h], false, false);
                        u.d[h] = s[0];
                        u.d[2 + h] = s[1];
                    }
                    at = n + 16 * (j + (g & 1)) + 4 * (g & 2);
                }
                if (at + 8 <= N) {
                    __builtin_memcpy(to + at, u.v, 16);
                } else {
#pragma unroll
                    for (int e = 0; e < 7; ++e)
                        if (at + e < N) to[at + e] = u.v[e];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < QUADS; ++j)
                if (n + column(j, g) < N) store4_as<OT>(to, n + column(j, g), x[j], N - n - column(j, g));
        }
    }
    template <int OT>
    static __device__ __forceinline__ void store(Args &p, const TileAt &t, const Acc (&acc)[Cfg::TM][Cfg::TN], int wm, int wn, int r, int g) {
        const int N = p.N, n = t.n0 + wn * COLUMNS;
        constexpr bool SCALED = Cfg::LAYB == ACROSS_K && Cfg::ET == ET_F16;  // (the gradients)
        const float unscale = SCALED ? *p.unscale : 1.f;
        constexpr int FACTORS = Cfg::GATED ? 2 : 1;
        float scale[FACTORS][QUADS][4];  // of the channels
        if (Cfg::ET == ET_I8) {
#pragma unroll
            for (int h = 0; h < FACTORS; ++h)
#pragma unroll
                for (int j = 0; j < QUADS; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = n + column(j, g) + e;
                        scale[h][j][e] = p.scale_b[h][c < N ? c : N - 1];
                    }
        }
#pragma unroll
        for (int i = 0; i < Cfg::TM; ++i) {
            const int m = t.m0 + wm * Cfg::WM + FragA::row(i, r);
            const bool there = m < p.M;  // (lanes stay together for the exchange)
            float x[QUADS][4], u[QUADS][4];
            float sa = 1.f;
            if (Cfg::ET == ET_I8) sa = p.scale_a[there ? m : p.M - 1];
#pragma unroll
            for (int j = 0; j < QUADS; ++j) {
                const Acc q = quad(acc[i], j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[j][e] = (float)q[e];
                    if (SCALED) x[j][e] *= unscale;
                    if (Cfg::ET == ET_I8) x[j][e] = x[j][e] * sa * scale[0][j][e];
                    if (Cfg::GATED) {
                        u[j][e] = (float)acc[i][j + Cfg::TN / 2][e];
                        if (Cfg::ET == ET_I8) u[j][e] = u[j][e] * sa * scale[FACTORS - 1][j][e];
                    }
                }
            }
            const int last = there ? N : 0;  // (a row that is not there has no columns)
            if (Cfg::GATED) {
                if (p.save[0]) {
                    row<OT>(p.save[0], p.ld_save[0], last, m, n, g, x);
                    row<OT>(p.save[1], p.ld_save[1], last, m, n, g, u);
                }
#pragma unroll
                for (int j = 0; j < QUADS; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[j][e] = gate_value(p.gate, x[j][e]) * u[j][e];
            }
            row<OT>(p.C[t.z], p.ldc[t.z], last, m, n, g, x);
        }
    }
};

// Tiles id, id + stride, ... below `end`.
template <typename Cfg> static __device__ __forceinline__ void walk_tiles(Args *args, int id, int stride, int end, char *lds) {
    constexpr int BM = Cfg::BM, BN = Cfg::BN, TM = Cfg::TM, TN = Cfg::TN, S = Cfg::S, LA = Cfg::LA, LB = Cfg::LB;
    typedef Mfma<Cfg::ET> Op;
    typedef typename Op::Acc Acc;
    typedef Image<BM, Cfg::LAYA> ImA;
    typedef Image<BN, Cfg::LAYB> ImB;
    typedef Fragments<BM, Cfg::LAYA, TM> FragA;
    typedef Fragments<BN, Cfg::LAYB, TN> FragB;
    typedef Results<Cfg> Res;
    if (id >= end) return;
    Args &p = *args;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / Cfg::WAVES_N, wn = wave % Cfg::WAVES_N;

    // The lane's place in what it loads.  (The swizzle repeats after as many rows as lie between two loads of a wave.)
    static_assert(Cfg::LAYA == ALONG_K || Cfg::WAVES * ImA::ROWS_PER_LOAD % 16 == 0, "");
    static_assert(Cfg::LAYB == ALONG_K || Cfg::WAVES * ImB::ROWS_PER_LOAD % 16 == 0, "");
    // (TERMS, A's columns across the depth: after 32 first terms their second ones)
    constexpr bool PAIRS = Cfg::TERMS && Cfg::LAYA == ACROSS_K;
    const int a_col = ImA::slot_of(wave, lane);
    const int a_slot = PAIRS ? (a_col >> 2) * 128 + (a_col & 3) * 16 : a_col * 16, b_slot = ImB::slot_of(wave, lane) * 16;
    const int lda = (int)p.lda, ldb[2] = {(int)p.ldb[0], (int)p.ldb[1]};
    const int a_off = ImA::row_of(0, lane) * lda + a_slot;
    const int b_off[2] = {ImB::row_of(0, lane) * ldb[0] + b_slot, ImB::row_of(0, lane) * ldb[1] + b_slot};
    const int64_t a_step = Cfg::LAYA == ALONG_K ? 128 : Cfg::DEPTH * p.lda;
    const int64_t b_step[2] = {Cfg::LAYB == ALONG_K ? 128 : Cfg::DEPTH * p.ldb[0], Cfg::LAYB == ALONG_K ? 128 : Cfg::DEPTH * p.ldb[1]};
    const char *b_from[2] = {static_cast<const char *>(p.B[0]), static_cast<const char *>(p.B[1])};
    const int64_t b_len[2] = {p.b_bytes[0], p.b_bytes[1]};
    constexpr int kOutside = (int)0x80000000u;

    // The feeding side runs S steps ahead of the multiplying one: the next step to load, and its place in memory.
    // (While a step is within a tile the places only move on; no branch chooses between them.)
    const int part_steps = Cfg::PARTS ? p.part_steps : 0;
    const int64_t a_jump = Cfg::PARTS ? p.a_jump : 0;
    TileAt feed = tile_at<Cfg>(fresh(args), id);
    int feed_id = id, feed_step = 0;
    const char *a_ptr, *b_ptr[2];
    int64_t a_left, b_left[2];
    int part = 0;
    auto aim_a = [&] {
        Args &p = fresh(args);
        const int64_t jump = Cfg::PARTS && feed.first_step >= part_steps ? a_jump : 0;
        const int64_t skip = (Cfg::LAYA == ALONG_K ? feed.m0 * p.lda : (int64_t)feed.m0 * (PAIRS ? 4 : 2)) + feed.first_step * a_step + jump;
        a_ptr = static_cast<const char *>(p.A[feed.z]) + skip;
        a_left = p.a_bytes - skip;
    };
    auto aim_parts = [&] {  // PARTS: anew for every step
        const int step = feed.first_step + feed_step;
        part = step >= part_steps;
        const int64_t skip = (int64_t)feed.n0 * 2 + (int64_t)(part ? step - part_steps : step) * (part ? b_step[1] : b_step[0]);
        b_ptr[0] = (part ? b_from[1] : b_from[0]) + skip;
        b_left[0] = (part ? b_len[1] : b_len[0]) - skip;
    };
    auto aim_b = [&] {
        if constexpr (Cfg::PARTS) {
            aim_parts();
        } else {
            Args &p = fresh(args);
#pragma unroll
            for (int h = 0; h < (Cfg::GATED ? 2 : 1); ++h) {
                const int64_t skip = (Cfg::LAYB == ALONG_K ? feed.n0 * p.ldb[h] : (int64_t)feed.n0 * 2) + feed.first_step * b_step[h];
                b_ptr[h] = static_cast<const char *>(p.B[h]) + skip;
                b_left[h] = p.b_bytes[h] - skip;
            }
        }
    };
    aim_a();
    aim_b();
    // One of the loads of an operand's next step.  ALONG_K: slots behind the depth's end, and everything once the last tile has
    // been fed, go out of range, where loads give zeros.  (ACROSS_K: rows behind it lie behind the operand's last byte.)
    auto load_a = [&](char *dst, int i) {
        const int q = wave + i * Cfg::WAVES;
        const bool out = (Cfg::LAYA == ALONG_K ? a_slot : 0) >= feed.bytes(feed_step);
        const int row = q * ImA::ROWS_PER_LOAD;
        const int off = a_off + (PAIRS ? (row & 31) * lda + (row >> 5) * 64 : row * lda);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(a_ptr, a_left), (lds_void_t *)(dst + q * 1024), 16, out ? kOutside : off, 0, 0, 0);
    };
    auto load_b = [&](char *dst, int i) {
        const int q = wave + i * Cfg::WAVES, row = q * ImB::ROWS_PER_LOAD;
        const int h = Cfg::GATED ? (row % Cfg::WN) / (Cfg::WN / 2) : 0;
        const int ch = Cfg::GATED ? row / Cfg::WN * (Cfg::WN / 2) + row % (Cfg::WN / 2) : row;
        const bool out = (Cfg::LAYB == ALONG_K ? b_slot : 0) >= feed.bytes(feed_step);
        const bool second = Cfg::GATED ? h : Cfg::PARTS ? part : 0;
        const int off = (second ? b_off[1] : b_off[0]) + ch * (second ? ldb[1] : ldb[0]);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_of(h ? b_ptr[1] : b_ptr[0], h ? b_left[1] : b_left[0]), (lds_void_t *)(dst + q * 1024), 16,
                                                 out ? kOutside : off, 0, 0, 0);
    };
    auto feed_on = [&] {
        if (++feed_step < feed.steps) {
            const int64_t on = a_step + (Cfg::PARTS && feed.first_step + feed_step == part_steps ? a_jump : 0);
            a_ptr += on;
            a_left -= on;
            if constexpr (Cfg::PARTS) {
                aim_parts();
            } else {
#pragma unroll
                for (int h = 0; h < (Cfg::GATED ? 2 : 1); ++h) {
                    b_ptr[h] += b_step[h];
                    b_left[h] -= b_step[h];
                }
            }
            return;
        }
        feed_step = 0;
        feed_id += stride;
        if (feed_id < end) {
            feed = tile_at<Cfg>(fresh(args), feed_id);
            aim_a();
            aim_b();
        } else {
            feed.whole = -1;
        }
    };
    // A slot that the depth ends in (its last bytes are real memory: the next row) is cut off in LDS once it is there - for
    // both operands, as zero times NaN is no zero.
    auto cut = [&](char *dst, int q, int slot, int bytes) {
        if (slot != (bytes & ~15)) return;
        u32x4 *at = reinterpret_cast<u32x4 *>(dst + q * 1024 + lane * 16);
        u32x4 v = *at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int keep = (bytes & 15) - 4 * e;  // bytes of this dword
            v[e] = keep >= 4 ? v[e] : keep <= 0 ? 0u : v[e] & ((1u << (8 * keep)) - 1);
        }
        *at = v;
    };
    // What this wave loaded of a step (that holds so many bytes of the depth) is in LDS: make it fit to be read, then wait
    // for the other waves.
    auto publish = [&](char *at, int bytes) {
        if (bytes & 15) {
            if (Cfg::LAYA == ALONG_K)
#pragma unroll
                for (int i = 0; i < LA; ++i) cut(at, wave + i * Cfg::WAVES, a_slot, bytes);
            if (Cfg::LAYB == ALONG_K)
#pragma unroll
                for (int i = 0; i < LB; ++i) cut(at + Cfg::A_BYTES, wave + i * Cfg::WAVES, b_slot, bytes);
        }
        CBA_FFN_WAIT_LDS();  // also: this wave's fragment reads of the stage that is loaded into next have completed
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    FragA ra;
    FragB rb;
    ra.init(lane, wm * Cfg::WM);
    rb.init(lane, wn * Cfg::WN);
    // operands of a step's two MFMAs (TERMS: fb[0] those of both, fb[1] the next step's as they were read)
    u32x4 fa[2][TM], fb[2][TN];
    auto read_one = [&](const char *at, int kk, int i) {
        const int b = Cfg::TERMS && kk ? 0 : TN;
        if (i < b) fb[Cfg::TERMS ? 1 : kk][i] = rb.read(at + Cfg::A_BYTES, i, kk);
        else fa[kk][i - b] = ra.read(at, i - b, kk);
    };
    Acc acc[TM][TN];

    char *stage = lds;
    auto after = [&](char *at) { return at + Cfg::STAGE == lds + Cfg::LDS ? lds : at + Cfg::STAGE; };
#pragma nounroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int i = 0; i < LA; ++i) load_a(lds + s * Cfg::STAGE, i);
#pragma unroll
        for (int i = 0; i < LB; ++i) load_b(lds + s * Cfg::STAGE + Cfg::A_BYTES, i);
        feed_on();
    }
    TileAt t = tile_at<Cfg>(fresh(args), id);
    CBA_FFN_WAIT_VM((S - 1) * (LA + LB));
    publish(lds, t.bytes(0));
    auto read_first = [&](const char *at) {
#pragma unroll
        for (int i = 0; i < TM + TN; ++i) read_one(at, 0, i);
    };
    read_first(lds);

    // MFMAs kk of a step.  Loads and reads are spread between their rows: behind the first, whose operands are there, and
    // none behind the last.
    auto multiply = [&](int kk, int loads, int reads, auto &&load, auto &&read) {
        constexpr int ROWS = TM > 1 ? TM - 1 : 1;
#pragma unroll
        for (int j = 0; j < TN; j += FragB::V) {
            if (Cfg::TERMS && kk) break;
#pragma unroll
            for (int e = 0; e < FragB::V && Cfg::TERMS; ++e) fb[0][j + e] = fb[1][j + e];
            rb.ready(&fb[kk][j]);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            if (i % FragA::V == 0) ra.ready(&fa[kk][i]);
            // the weights are the instruction's first operand: a lane then holds one token's neighbouring channels
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = Op::run(fb[Cfg::TERMS ? 0 : kk][j], fa[kk][i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
            if (i >= ROWS) continue;
#pragma unroll
            for (int o = loads * i / ROWS; o < loads * (i + 1) / ROWS; ++o) load(o);
#pragma unroll
            for (int o = reads * i / ROWS; o < reads * (i + 1) / ROWS; ++o) read(o);
        }
    };
    // One step: multiply its first half while the second's operands are read; publish the next step; multiply the second
    // half while the next step's first operands are read and the loads of the step S later start into the stage that is free.
    auto step = [&](int next_bytes) {
        char *const next = after(stage), *const free = stage;
        multiply(0, 0, Cfg::TERMS ? TM : TM + TN, [&](int) {}, [&](int o) { read_one(free, 1, o); });
        CBA_FFN_WAIT_VM((S - 2) * (LA + LB));
        publish(next, next_bytes);
        multiply(1, LA + LB, TM + TN, [&](int o) { o < LA ? load_a(free, o) : load_b(free + Cfg::A_BYTES, o - LA); },
                 [&](int o) { read_one(next, 0, o); });
        feed_on();
        stage = next;
    };

    const int r = lane & 15, g = lane >> 4;
    for (;;) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = Acc{};
        const int next_id = id + stride;
        const int next_tile_bytes = next_id < end ? tile_at<Cfg>(fresh(args), next_id).bytes(0) : 0;
        for (int s = 1; s <= t.steps; ++s) step(s < t.steps ? t.bytes(s) : next_tile_bytes);

        Args &out = fresh(args);
        if (out.splits > 1) {
            // partial sums, four neighbouring columns of a row at a time
            typedef typename ElemOf<Cfg::ET>::Acc Sum;
            Sum *const ws = reinterpret_cast<Sum *>(out.ws) + (int64_t)t.split * out.ws_split + (int64_t)t.z * out.ws_plane;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int m = t.m0 + wm * Cfg::WM + FragA::row(i, r);
#pragma unroll
                for (int j = 0; j < Res::QUADS; ++j) {
                    const int n = t.n0 + wn * Res::COLUMNS + Res::column(j, g);
                    if (m >= out.M || n >= out.N) continue;
                    Sum *w = ws + (int64_t)m * out.ws_ld + n;
                    *reinterpret_cast<Acc *>(w) = Res::quad(acc[i], j);
                    if (Cfg::GATED) *reinterpret_cast<Acc *>(w + out.ws_plane) = acc[i][j + TN / 2];
                }
            }
        } else if (Cfg::ET == ET_F16 || (Cfg::ET == ET_I8 && out.out_type == OT_F16)) {
            if (Cfg::ET != ET_BF16) Res::template store<OT_F16>(out, t, acc, wm, wn, r, g);
        } else if (Cfg::ET == ET_BF16 || out.out_type == OT_BF16) {
            if (Cfg::ET != ET_F16) Res::template store<OT_BF16>(out, t, acc, wm, wn, r, g);
        } else {
            if (Cfg::ET == ET_I8) Res::template store<OT_F32>(out, t, acc, wm, wn, r, g);
        }
        if (next_id >= end) break;
        id = next_id;
        t = tile_at<Cfg>(fresh(args), id);
        read_first(stage);  // (once more: kept over the stores, these registers would be spilled)
    }
    CBA_FFN_WAIT_VM(0);  // (nothing may be on its way into LDS when the workgroup ends)
}

// Workgroups are handed to the 8 XCDs in turn, and each XCD has an L2 of its own: every XCD walks a contiguous piece of the
// list, its workgroups side by side.  This is workgroup `block` of the `blocks` that walk this list.
template <typename Cfg> static __device__ __forceinline__ void walk_list(Args *p, int block, int blocks, char *lds) {
    const int total = p->tiles_m * p->tiles_n * p->batch * p->splits;
    const int xcds = blocks < 8 ? blocks : 8, xcd = block % xcds, place = block / xcds;
    const int per = total / xcds, rem = total % xcds;
    const int first = xcd * per + (xcd < rem ? xcd : rem), end = first + per + (xcd < rem ? 1 : 0);
    const int stride = (blocks - xcd + xcds - 1) / xcds;  // workgroups on this XCD
    walk_tiles<Cfg>(p, first + place, stride, end, lds);
}
template <typename Cfg> __global__ __launch_bounds__(Cfg::THREADS, 2) void tile_kernel(Product) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    walk_list<Cfg>(kernel_args(), blockIdx.x, gridDim.x, lds);
}
// Two products in one launch (both sides of the gradient): the first `blocks` workgroups walk the first one's tiles.
template <typename Cfg0, typename Cfg1> __global__ __launch_bounds__(Cfg0::THREADS, 2) void two_tiles_kernel(ProductPair, int blocks) {
    static_assert(Cfg0::THREADS == Cfg1::THREADS && Cfg0::LDS == Cfg1::LDS, "");
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    if ((int)blockIdx.x < blocks) walk_list<Cfg0>(kernel_args(), blockIdx.x, blocks, lds);
    else walk_list<Cfg1>(kernel_args() + 1, blockIdx.x - blocks, gridDim.x - blocks, lds);
}

// ---- the product from registers ----
//
// For products too small to fill the card with large tiles, or to pay for a round trip through LDS: a workgroup computes
// a tile of 16 TM x 16 TN (GATED: 16 TN channels of both weights), and its W waves share the DEPTH, wave w taking every
// W-th piece of 128 bytes.  So no wave needs what another has loaded: each reads its rows from memory straight into the
// MFMAs' registers, DEEP pieces ahead, without a barrier, and the W partial tiles are added up in LDS once at the end
// (in wave order).  Rows behind the last one are read as the last one, and not stored.
// SHIFT: rows that do not all start on a dword.  Unaligned 16-byte loads take 2.5 times as long (6 x 536 x 7503 gated in 51 us), so
// each is made from aligned dwords, one more than the four, and shifted into place by bytes (v_alignbyte_b32).
template <int ET_, int TM_, int TN_, int W_, int DEEP_, bool GATED_, bool SHIFT_> struct RowsCfg {
    static constexpr int ET = ET_, TM = TM_, TN = TN_, W = W_, DEEP = DEEP_;
    static constexpr bool GATED = GATED_, SHIFT = SHIFT_;
    static constexpr int NB = GATED ? 2 * TN : TN;  // blocks of weights' rows
    static constexpr int THREADS = 64 * W;
    static constexpr int PITCH = 16 * NB + 4;        // of a partial tile's row in LDS, 32-bit sums
    static constexpr int LDS = W * 16 * TM * PITCH * 4;
};

// The 16 bytes of a row from byte `at` on, as far as they lie before `end` (zeros behind).
template <int ES> static __device__ __forceinline__ u32x4 load16_tail(const char *row, int64_t at, int64_t end) {
    u32x4 v = {};
    if (at + 16 <= end) {
        __builtin_memcpy(&v, row + at, 16);
        return v;
    }
#pragma unroll
    for (int e = 0; e < 16; e += ES)
        if (at + e < end) {
            uint32_t x;
            if (ES == 2) {
                uint16_t y;
                __builtin_memcpy(&y, row + at + e, 2);
                x = y;
            } else {
                x = *reinterpret_cast<const uint8_t *>(row + at + e);
            }
            v[e / 4] |= x << (8 * (e % 4));
        }
    return v;
}

template <typename Cfg> __global__ __launch_bounds__(Cfg::THREADS, 2) void rows_kernel(Product p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int TM = Cfg::TM, TN = Cfg::TN, NB = Cfg::NB, W = Cfg::W, D = Cfg::DEEP, ES = Cfg::ET == ET_I8 ? 1 : 2;
    typedef Mfma<Cfg::ET> Op;
    typedef typename ElemOf<Cfg::ET>::Acc S;
    typedef S sx4 __attribute__((ext_vector_type(4)));
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // neighbours in the list share the weights' rows, and an XCD gets a contiguous piece of it
    const int id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int m0 = id % p.tiles_m * (16 * TM), n0 = id / p.tiles_m * (16 * TN);

    const char *a[TM], *b[NB];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int m = m0 + 16 * i + r;
        a[i] = static_cast<const char *>(p.A[0]) + (int64_t)(m < p.M ? m : p.M - 1) * p.lda;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int h = Cfg::GATED && j >= TN ? 1 : 0;
        const int n = n0 + 16 * (j - h * TN) + r;
        b[j] = static_cast<const char *>(p.B[h]) + (int64_t)(n < p.N ? n : p.N - 1) * p.ldb[h];
    }
    sx4 acc[TM][NB] = {};
    // 16 bytes as they come: four dwords, and with SHIFT the one behind them - or the fourth again where the row is aligned and the
    // fifth need not exist.
    struct Raw {
        u32x4 v;
        uint32_t more;
    };
    Raw fa[D][TM][2], fb[D][NB][2];
    // (off: where in a dword the row starts, and so every piece of it)
    auto fetch = [&](const char *row, int64_t at) {
        Raw f;
        if constexpr (Cfg::SHIFT) {
            const uint32_t off = (uint32_t)(uintptr_t)row & 3;
            const char *from = static_cast<const char *>(__builtin_assume_aligned(row - off, 4)) + at;
            __builtin_memcpy(&f.v, __builtin_assume_aligned(from, 4), 16);
            __builtin_memcpy(&f.more, __builtin_assume_aligned(from + (off ? 16 : 12), 4), 4);
        } else {
            __builtin_memcpy(&f.v, __builtin_assume_aligned(row + at, 4), 16);
        }
        return f;
    };
    auto operand = [&](const Raw &f, const char *row) {
        if constexpr (!Cfg::SHIFT) return f.v;
        const uint32_t off = (uint32_t)(uintptr_t)row & 3;
        return u32x4{__builtin_amdgcn_alignbyte(f.v[1], f.v[0], off), __builtin_amdgcn_alignbyte(f.v[2], f.v[1], off),
                     __builtin_amdgcn_alignbyte(f.v[3], f.v[2], off), __builtin_amdgcn_alignbyte(f.more, f.v[3], off)};
    };
    auto load = [&](int d, int piece) {
        const int64_t at = (int64_t)piece * 128 + g * 16;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
            for (int j = 0; j < NB; ++j) fb[d][j][kk] = fetch(b[j], at + 64 * kk);
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[d][i][kk] = fetch(a[i], at + 64 * kk);
        }
    };
    auto use = [&](int d) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 vb[NB];
#pragma unroll
            for (int j = 0; j < NB; ++j) vb[j] = operand(fb[d][j][kk], b[j]);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const u32x4 va = operand(fa[d][i][kk], a[i]);
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[i][j] = Op::run(vb[j], va, acc[i][j]);
            }
        }
    };
    // pieces wave, wave + W, ... of the whole ones are this wave's
    const int whole = (int)(p.k_bytes >> 7), mine = whole > wave ? (whole - wave + W - 1) / W : 0;
    int i0 = 0;
    if (mine >= D) {
#pragma unroll
        for (int d = 0; d < D; ++d) load(d, wave + d * W);
        for (; i0 + 2 * D <= mine; i0 += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                use(d);
                load(d, wave + (i0 + D + d) * W);
            }
        }
#pragma unroll
        for (int d = 0; d < D; ++d) use(d);
        i0 += D;
    }
    if (i0 < mine) {
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (i0 + d < mine) load(d, wave + (i0 + d) * W);
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (i0 + d < mine) use(d);
    }
    if ((p.k_bytes & 127) && whole % W == wave) {
        const int64_t at = (int64_t)whole * 128 + g * 16;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            if (kk && (p.k_bytes & 127) <= 64) continue;
            u32x4 ta[TM], tb[NB];
#pragma unroll
            for (int i = 0; i < TM; ++i) ta[i] = load16_tail<ES>(a[i], at + 64 * kk, p.k_bytes);
#pragma unroll
            for (int j = 0; j < NB; ++j) tb[j] = load16_tail<ES>(b[j], at + 64 * kk, p.k_bytes);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) acc[i][j] = Op::run(tb[j], ta[i], acc[i][j]);
        }
    }

    // partial tiles [wave][m][n] -> sums -> results
    S *part = reinterpret_cast<S *>(lds);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
            *reinterpret_cast<sx4 *>(part + ((wave * TM + i) * 16 + r) * Cfg::PITCH + 16 * j + 4 * g) = acc[i][j];
    __syncthreads();
    constexpr int QUADS = 16 * TM * 4 * TN;
#pragma unroll
    for (int q0 = 0; q0 < QUADS; q0 += Cfg::THREADS) {
        const int q = q0 + tid, ml = q / (4 * TN), nl = q % (4 * TN) * 4;
        const int m = m0 + ml, n = n0 + nl;
        if ((QUADS % Cfg::THREADS && q >= QUADS) || m >= p.M || n >= p.N) continue;
        sx4 x = {}, y = {};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const S *at = part + (w * TM * 16 + ml) * Cfg::PITCH + nl;
            x += *reinterpret_cast<const sx4 *>(at);
            if (Cfg::GATED) y += *reinterpret_cast<const sx4 *>(at + 16 * TN);
        }
        const float fx[4] = {(float)x[0], (float)x[1], (float)x[2], (float)x[3]}, fy[4] = {(float)y[0], (float)y[1], (float)y[2], (float)y[3]};
        finish4<Cfg::ET, Cfg::GATED>(*kernel_args(), 0, m, n, fx, fy);
    }
}

// Adds up the depth ranges of a split product (in their order, whatever finished first) and finishes the results.
// Partial sums: [range][plane][row][column], rows of ws_ld (a multiple of 4) 32-bit sums; planes are the batch's
// entries or the gate's two products.
template <int ET, bool GATED> static __device__ __forceinline__ void join(Args *args) {
    Args &p = *args;
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
        const float x[4] = {(float)a[0], (float)a[1], (float)a[2], (float)a[3]};
        const float y[4] = {(float)b[0], (float)b[1], (float)b[2], (float)b[3]};
        finish4<ET, GATED>(p, z, m, n, x, y);
    }
}
template <int ET, bool GATED> __global__ __launch_bounds__(256) void join_kernel(Product) { join<ET, GATED>(kernel_args()); }
template <int ET> __global__ __launch_bounds__(256) void join_two_kernel(ProductPair) {
    Args *p = kernel_args() + blockIdx.y;
    if (p->splits > 1) join<ET, false>(p);
}

}  // namespace ffn
}  // namespace cba
