// The products of a gated feed-forward layer: rows to 8-bit integers, the 8-bit product with scales, the gated
// product in 16 and 8 bits, and its gradients.  Kernels that are not the product itself, and the launch logic.
#include <hip/hip_runtime.h>

#include <cstdio>

#include "ffn_kernel.hpp"
#include "workspace.hpp"

namespace cba {
namespace ffn {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// ---- rows to 8-bit integers ----
//
// q = round_half_even(127 x / a), a the row's largest magnitude, exactly: the quotient is formed in float (off by at
// most 127 (2^-24 + 2^-24) < 1.6e-5), and where that lands nearer to a half than it can be off, 254 |x| and
// (2 n + 1) a are compared in double, where both are exact.  (Halves are no rarity: x = a / 2 is one in every format.)
// One workgroup per row (no loop over rows: 16384 x 8192 bf16 in 75.5 us without, 87.5 with one); up to 8192 elements stay in
// registers between the two passes, what is behind them is read twice.  WAVE: one wave per row, of kWaveRow elements at most.
const int kWaveRow = 1024;
static __device__ __forceinline__ float quantized(float x, float a, float inv) {
    const float t = fabsf(x) * inv;
    float n = rintf(t);
    if (__builtin_expect(fabsf(t - n) > 0.49998f, 0)) {
        n = floorf(t);
        const double over = 254.0 * fabsf(x) - (2.0 * n + 1.0) * a;
        if (over > 0.0 || (over == 0.0 && ((int)n & 1))) n += 1.f;
    }
    return copysignf(n, x);
}

template <typename T, bool WAVE> __global__ __launch_bounds__(256) void quantize_kernel(const T *X, int64_t ldx, int8_t *Q, int64_t ldq, float *scale, int M, int K) {
    constexpr int LANES = WAVE ? 64 : 256, ROWS = 256 / LANES, KEEP = WAVE ? kWaveRow / (8 * LANES) : 4;
    const int lane = threadIdx.x % LANES;
    struct Vec8 { T v[8]; };
    __shared__ uint32_t part[4];
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + threadIdx.x / LANES;
    if (row >= M) return;
    const T *x = X + row * ldx;
    int8_t *q = Q + row * ldq;
    const int vecs = K / 8;
    Vec8 kept[KEEP];
    // magnitudes compare as integers, and a NaN's is the largest
    uint32_t top = 0;
    auto take = [&](T v) {
        const uint32_t b = __builtin_bit_cast(uint32_t, (float)v) & 0x7fffffffu;
        top = b > top ? b : top;
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const int c = lane + i * LANES;
        if (c < vecs) {
            __builtin_memcpy(&kept[i], x + (int64_t)c * 8, sizeof(Vec8));
#pragma unroll
            for (int e = 0; e < 8; ++e) take(kept[i].v[e]);
        }
    }
    for (int c = lane + KEEP * LANES; !WAVE && c < vecs; c += LANES) {
        Vec8 v;
        __builtin_memcpy(&v, x + (int64_t)c * 8, sizeof(Vec8));
#pragma unroll
        for (int e = 0; e < 8; ++e) take(v.v[e]);
    }
    const int tail = vecs * 8 + lane;
    if (tail < K) take(x[tail]);
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint32_t o = __shfl_xor(top, d);
        top = o > top ? o : top;
    }
    if (!WAVE) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) top = part[w] > top ? part[w] : top;
    }
    float a = __builtin_bit_cast(float, top);
    if (lane == 0) scale[row] = a / 127.f;
    // tiny rows are scaled up first (exact), so that 127 / a stays finite; a row without a finite, positive a is zero
    const float up = a < 0x1p-100f ? 0x1p100f : 1.f;
    a *= up;
    const bool usable = top > 0 && top < 0x7f800000u;
    const float inv = usable ? 127.f / a : 0.f;
    auto one = [&](T v) -> int8_t { return usable ? (int8_t)quantized((float)v * up, a, inv) : (int8_t)0; };
    auto eight = [&](const Vec8 &v, int c) {
        int8_t o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = one(v.v[e]);
        __builtin_memcpy(q + (int64_t)c * 8, o, 8);
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        const int c = lane + i * LANES;
        if (c < vecs) eight(kept[i], c);
    }
    for (int c = lane + KEEP * LANES; !WAVE && c < vecs; c += LANES) {
        Vec8 v;
        __builtin_memcpy(&v, x + (int64_t)c * 8, sizeof(Vec8));
        eight(v, c);
    }
    if (tail < K) q[tail] = one(x[tail]);
}

// ---- copies that make an operand fit the tiled product ----

// Rows of `bytes` bytes, `ld` apart and aligned to nothing -> rows `ld_to` apart (a multiple of 16), zeros behind.  One launch
// for all operands of a product.
struct Copy {
    const char *from;
    char *to;
    int64_t ld, bytes, ld_to, rows;
};
struct CopyList {
    Copy c[3];
};
__global__ __launch_bounds__(256) void copy_rows_kernel(CopyList list) {
    const Copy &c = list.c[blockIdx.y];
    const int64_t per = c.ld_to >> 4, total = per * c.rows;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int64_t row = t / per, at = (t - row * per) * 16;
        const char *src = c.from + row * c.ld + at;
        char v[16] = {};
        if (at + 16 <= c.bytes) {
            __builtin_memcpy(v, src, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (at + e < c.bytes) v[e] = src[e];
        }
        __builtin_memcpy(__builtin_assume_aligned(c.to + row * c.ld_to + at, 16), v, 16);
    }
}

// ---- gradients of the gate ----
//
// dG = dH o U o act'(G), dU = dH o act(G).  The two products that follow take 16-bit operands.  Rounded to one such number these
// values would carry its error into every result (2.3e-3 of it instead of 1.7e-3 in bf16, 2.9e-4 for 2.1e-4 in f16), so each is kept
// as the sum of two (TWO): the first truncated, the second what is left, rounded - 16 bits of bf16, 21 of f16.
// Truncation gives both the same sign, and neither is left zero: a term times an infinity is then infinite, and no NaN.
// Twice the matrix work: 8192 x 12288 x 4096 bf16 5.6 ms, with one number 3.0.  A caller may choose that (clblasAmdRoundTerms).
// f16 would also lose its range (dH U reaches 2^32): all of a call's values are multiplied by one power of two that brings the
// largest to 2^14 ... 2^15 (exact; what it pushes below 2^-24 is less than 2^-38 of the largest), and the results by its reciprocal.
template <int OT, bool TWO> struct Terms {
    uint16_t first[8], second[8];
    static __device__ __forceinline__ float value(uint16_t bits) {
        return OT == OT_BF16 ? __builtin_bit_cast(float, (uint32_t)bits << 16) : (float)__builtin_bit_cast(_Float16, bits);
    }
    static __device__ __forceinline__ uint16_t rounded(float x) {
        const auto r = Store<OT>::of(x);
        return __builtin_bit_cast(uint16_t, r);
    }
    static __device__ __forceinline__ uint16_t truncated(float x) {
        if (OT == OT_BF16) return (uint16_t)(__builtin_bit_cast(uint32_t, x) >> 16);
        const _Float16 r = (_Float16)__builtin_amdgcn_cvt_pkrtz(x, 0.f)[0];
        return __builtin_bit_cast(uint16_t, r);
    }
    __device__ __forceinline__ void set(int e, float x, float scale) {
        if (OT == OT_F16) x *= scale;
        if (!TWO) {
            first[e] = rounded(x);
            return;
        }
        uint16_t hi = truncated(x), lo = rounded(x - value(hi));
        if (!(fabsf(x) < __builtin_inff())) {
            lo = hi;
        } else if ((lo & 0x7fff) == 0 && (hi & 0x7fff) > 1) {  // one step of the first goes to the second
            --hi;
            lo = rounded(x - value(hi));
        }
        first[e] = hi;
        second[e] = lo;
    }
};

// The values lie as [dG], then [dU]: a row per token, padded with zeros to whole lines of 128 bytes; TWO: 32 first terms and their
// 32 second ones a line.
struct GateGrad {
    const void *dH, *G, *U;
    int64_t lddh, ldg, ldu;
    int M, N, gate;
    char *out;
    int64_t row, plane;  // bytes from token to token, and from dG to dU
    uint32_t *top;       // f16: the largest magnitude that each workgroup of the first pass met
    int tops;
    float *unscale;      // f16: the reciprocal of the common power of two
};

// dG and dU of channels n .. n + 7 of token m; zeros behind the last channel.
template <int OT> static __device__ __forceinline__ void gate_grad8(const GateGrad &p, int64_t m, int n, float (&dg)[8], float (&du)[8]) {
    typedef typename Store<OT>::type T;
    struct Vec8 { T v[8]; };
    const T *h = static_cast<const T *>(p.dH) + m * p.lddh + n, *g = static_cast<const T *>(p.G) + m * p.ldg + n,
            *u = static_cast<const T *>(p.U) + m * p.ldu + n;
    Vec8 vh = {}, vg = {}, vu = {};
    if (n + 8 <= p.N) {
        __builtin_memcpy(&vh, h, 16);
        __builtin_memcpy(&vg, g, 16);
        __builtin_memcpy(&vu, u, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (n + e < p.N) {
                vh.v[e] = h[e];
                vg.v[e] = g[e];
                vu.v[e] = u[e];
            }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float act, slope;
        gate_value_and_slope(p.gate, (float)vg.v[e], act, slope);
        const float dh = (float)vh.v[e];
        dg[e] = dh * (float)vu.v[e] * slope;
        du[e] = dh * act;
    }
}

// The largest of the workgroup's 256 values, in every thread.
static __device__ __forceinline__ uint32_t largest_of_all(uint32_t top) {
    __shared__ uint32_t part[4];
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint32_t o = __shfl_xor(top, d);
        top = o > top ? o : top;
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) top = part[w] > top ? part[w] : top;
    return top;
}

// f16, first pass: the largest finite magnitude (as bits, which compare like it).
__global__ __launch_bounds__(256) void gate_grad_top_kernel(GateGrad p) {
    const int64_t per_row = (p.N + 7) >> 3, total = per_row * p.M;
    uint32_t top = 0;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int64_t m = t / per_row;
        float dg[8], du[8];
        gate_grad8<OT_F16>(p, m, (int)(t - m * per_row) * 8, dg, du);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            for (const float x : {dg[e], du[e]}) {
                const uint32_t b = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
                if (b < 0x7f800000u && b > top) top = b;
            }
    }
    top = largest_of_all(top);
    if (threadIdx.x == 0) p.top[blockIdx.x] = top;
}

template <int OT, bool TWO> __global__ __launch_bounds__(256) void gate_grad_kernel(GateGrad p) {
    float scale = 1.f;
    if (OT == OT_F16) {
        uint32_t top = 0;
        for (int i = threadIdx.x; i < p.tops; i += 256) top = p.top[i] > top ? p.top[i] : top;
        top = largest_of_all(top);
        int e = 0;
        (void)frexpf(__builtin_bit_cast(float, top), &e);  // top = f 2^e, 1/2 <= f < 1
        e = top == 0 ? 0 : 15 - e > 100 ? 100 : 15 - e;
        scale = ldexpf(1.f, e);
        if (blockIdx.x == 0 && threadIdx.x == 0) *p.unscale = ldexpf(1.f, -e);
    }
    const int64_t per_row = p.row >> (TWO ? 5 : 4), total = per_row * p.M;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int64_t m = t / per_row;
        const int n = (int)(t - m * per_row) * 8;
        float dg[8], du[8];
        gate_grad8<OT>(p, m, n, dg, du);
        Terms<OT, TWO> g, u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            g.set(e, dg[e], scale);
            u.set(e, du[e], scale);
        }
        char *to = p.out + m * p.row + (TWO ? (n >> 5) * 128 + (n & 31) * 2 : (int64_t)n * 2);
        __builtin_memcpy(__builtin_assume_aligned(to, 16), g.first, 16);
        __builtin_memcpy(__builtin_assume_aligned(to + p.plane, 16), u.first, 16);
        if (TWO) {
            __builtin_memcpy(__builtin_assume_aligned(to + 64, 16), g.second, 16);
            __builtin_memcpy(__builtin_assume_aligned(to + p.plane + 64, 16), u.second, 16);
        }
    }
}

// ---- launching ----

hipError_t launched(const char *kernel, char type, int bm, int bn, int threads, int M, int N, int K, unsigned gx, unsigned gy, int splits, hipError_t e) {
    if (e != hipSuccess || dry_run_slot()) return e;
    DispatchRecord &r = dispatch_record();
    r.type = type;
    r.bm = bm;
    r.bn = bn;
    r.bk = 128;
    r.threads = threads;
    r.trans_a = 0;
    r.trans_b = 1;
    r.M = M;
    r.N = N;
    r.K = K;
    r.splits = splits;
    r.tail_slices = 1;
    r.tri = 0;
    r.grid_x = gx;
    r.grid_y = gy;
    r.kernel = kernel;
    r.launches++;
    if (knobs().log)
        fprintf(stderr, "clblas_amd: %s<%c,%dx%d,%d threads> M=%d N=%d K=%d grid=(%u,%u) splits=%d\n", kernel, type, bm, bn, threads, M, N, K, gx,
                gy, splits);
    return e;
}

char type_letter(int et) { return et == ET_I8 ? 'i' : et == ET_F16 ? 'h' : 'b'; }

// The forms of a product: those that run from registers (workgroups of 16 TM x 16 TN results - gated: of either factor - on
// W waves), then the tiled ones.
struct RowsShape { int tm, tn; };
const RowsShape kRows[] = {{1, 1}, {2, 1}, {2, 2}, {4, 2}};
enum { ROWS_FORMS = 4, TILE_FORMS = 5 };
// The form that the debug switch asks for; -1 if it names none.
int forced_form() {
    const int form = knobs().ffn_form;
    return form >= 0 && form < ROWS_FORMS + TILE_FORMS ? form : -1;
}
// step: us per step of 128 bytes of depth, alone on a CU / per tile where more tiles than CUs keep it busy.  Measured on products of 128 ... 8192 rows, 1024 ... 12288 channels, 1024 ... 8192 deep (alone: e.g. 64 x 64
// at 256 x 1024 x 4096 8-bit, 32 steps in 14.9 us; busy: 64 x 128 at 1024 x 4096 x 4096 gated, 4 x 64 steps per CU in 102 us).
struct TileShape { int log_bm, log_bn; double step_alone, step_busy; };
const TileShape kTiles[TILE_FORMS] = {
    {8, 8, 1.50, 1.62}, {8, 7, 0.87, 0.97}, {7, 7, 0.97, 0.57}, {6, 7, 0.50, 0.375}, {6, 6, 0.36, 0.27}};  // (edges: powers of two)

// The gradients' with two numbers for each term (both sides alone, 16 x 16 and 32 x 32 tiles, 1024 ... 4096 channels or tokens).
const TileShape kTermTiles[TILE_FORMS] = {{8, 8, 1.50, 1.51}, {8, 7, 0.85, 0.92}, {7, 7, 0.55, 0.455}, {6, 7, 0.46, 0.315}, {6, 6, 0.39, 0.25}};

template <int ET, bool GATED, typename F> hipError_t with_tile(int tile, F &&f) {
    switch (tile) {
    case 0: return f(TileCfg<ET, 256, 256, 128, 64, 2, GATED>());
    case 1: return f(TileCfg<ET, 256, 128, 64, 64, 3, GATED>());
    case 2: return f(TileCfg<ET, 128, 128, 64, 64, 2, GATED>());
    case 3: return f(TileCfg<ET, 64, 128, 32, 64, 3, GATED>());
    default: return f(TileCfg<ET, 64, 64, 32, 32, 5, GATED>());
    }
}
// The gradients'.  (TWO terms: a stage is a quarter or a third smaller, 32 rows of B to 64 bytes of either term of A.)
template <int ET, bool TWO, typename F> hipError_t with_grad_tile(int tile, F &&f) {
    switch (tile) {
    case 0: return f(TileCfg<ET, 256, 256, 128, 64, TWO ? 3 : 2, false, ALONG_K, ACROSS_K, TWO>());
    case 1: return f(TileCfg<ET, 256, 128, 64, 64, 3, false, ALONG_K, ACROSS_K, TWO>());
    case 2: return f(TileCfg<ET, 128, 128, 64, 64, TWO ? 3 : 2, false, ALONG_K, ACROSS_K, TWO>());
    case 3: return f(TileCfg<ET, 64, 128, 32, 64, TWO ? 5 : 3, false, ALONG_K, ACROSS_K, TWO>());
    default: return f(TileCfg<ET, 64, 64, 32, 32, TWO ? 6 : 5, false, ALONG_K, ACROSS_K, TWO>());
    }
}

// How one product is tiled.
struct Tiling {
    int tiles_m = 0, tiles_n = 0, batch = 1, splits = 1, steps_per_split = 0;
    int64_t ws_ld = 0, ws_plane = 0, ws_split = 0;
    size_t ws_bytes = 0;
    int64_t count() const { return (int64_t)tiles_m * tiles_n * batch * splits; }
};
uint32_t blocks_of(uint32_t n, int shift) { return (n + (1u << shift) - 1) >> shift; }
// (This and what follows runs in every call: powers of two and 32-bit quotients.)
Tiling tiling(int tile, bool gated, int M, int N, int batch, int64_t k_bytes) {
    Tiling c;
    const TileShape &t = kTiles[tile];
    c.tiles_m = (int)blocks_of(M, t.log_bm);
    c.tiles_n = (int)blocks_of(N, gated ? t.log_bn - 1 : t.log_bn);
    c.batch = batch;
    c.steps_per_split = (int)((k_bytes + 127) >> 7);
    return c;
}
// Cuts the depth into `splits` ranges at most.  (The largest tiles do not split: TileCfg::SPLITS.)
Tiling cut_depth(Tiling c, int tile, bool gated, int M, int N, int splits) {
    const uint32_t steps = (uint32_t)c.steps_per_split;
    if (splits <= 1 || steps <= 1 || tile == 0) return c;
    if ((uint32_t)splits > steps) splits = (int)steps;
    c.steps_per_split = (int)((steps + splits - 1) / (uint32_t)splits);
    c.splits = (int)((steps + c.steps_per_split - 1) / (uint32_t)c.steps_per_split);
    if (c.splits == 1) return c;
    c.ws_ld = ((int64_t)N + 3) & ~(int64_t)3;
    c.ws_plane = c.ws_ld * M;
    c.ws_split = c.ws_plane * (gated ? 2 : c.batch);
    c.ws_bytes = (size_t)c.ws_split * 4 * c.splits;
    return c;
}

// How `grid` workgroups are shared out between two lists of tiles: so that the busiest has the fewest steps to do.
struct Share {
    int blocks = 0;     // for the first list
    int64_t steps = 0;  // of the busiest workgroup
};
Share share_out(const Tiling *c, int grid) {
    Share best;
    const uint32_t n0 = (uint32_t)c[0].count(), n1 = (uint32_t)c[1].count();
    if (n0 == 0 || n1 == 0 || n0 + n1 <= (uint32_t)grid) {
        const uint32_t n = n0 ? n0 : n1;
        best.blocks = (int)(n0 < (uint32_t)grid ? n0 : (uint32_t)grid);
        const int64_t s0 = n0 ? c[0].steps_per_split : 0, s1 = n1 ? c[1].steps_per_split : 0;
        best.steps = n0 && n1 ? (s0 > s1 ? s0 : s1) : (int64_t)((n + grid - 1) / (uint32_t)grid) * (n0 ? s0 : s1);
        return best;
    }
    for (uint32_t rounds = (n0 + grid - 2) / (uint32_t)(grid - 1), tries = 0; rounds <= n0 && tries < 64; ++rounds, ++tries) {
        const uint32_t blocks = (n0 + rounds - 1) / rounds, others = grid - blocks;
        const int64_t s0 = (int64_t)rounds * c[0].steps_per_split, s1 = (int64_t)((n1 + others - 1) / others) * c[1].steps_per_split;
        const int64_t steps = s0 > s1 ? s0 : s1;
        if (best.steps && steps >= best.steps && s0 > s1) break;
        if (!best.steps || steps < best.steps) {
            best.blocks = (int)blocks;
            best.steps = steps;
        }
    }
    return best;
}

// Time (us) of a launch over the tiles of one product (n = 1) or two: the steps that the busiest workgroup goes through, 4.5 us
// for the launch, the first loads and the results, and for sums in pieces a second launch (3 us) and the partial sums, written
// and read again, at 0.6 us per MB (256 x 4096 x 4096 gated in two ranges of 64 x 128 tiles: 16.8 MB, 43.5 us; in one, 36.7).
// memory: us that the operands take from memory.
double tiled_cost(const TileShape &t, const Tiling *c, int n, double memory) {
    const int64_t count = c[0].count() + (n > 1 ? c[1].count() : 0);
    const int per_cu = t.log_bm + t.log_bn <= 14 ? 2 : 1;
    int64_t steps;
    if (n > 1) steps = share_out(c, 256 * per_cu).steps;
    else steps = count <= 256 ? c[0].steps_per_split : ((count + 255) >> 8) * c[0].steps_per_split;
    // (a workgroup that shares its CU goes through a step in the time of two)
    double time = steps * (count <= 256 ? t.step_alone : n > 1 ? per_cu * t.step_busy : t.step_busy);
    if (time < memory) time = memory;
    const double partial = (double)c[0].ws_bytes + (n > 1 ? (double)c[1].ws_bytes : 0.0);
    return 4.5 + time + (partial > 0 ? 3.0 + partial * 0.6e-6 : 0.0);
}

const int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};

// A form for a whole product, and its time by the model.
struct Choice {
    int form = 0;
    Tiling tiling;
    double cost = 1e30;
};

// From registers: what the busiest CU reads, at 33 bytes per ns (measured for workgroups of 16 x 16 ... 64 x 32 results,
// gated and 8-bit, 16 ... 256 rows; within 10 %; 20 where rows have to be shifted into place), or the weights from memory at 5.4 TB/s; 2.8 us for the launch.
double rows_cost(const RowsShape &s, bool gated, int M, int N, int64_t k_bytes, double memory, bool shift) {
    const int64_t groups = (int64_t)((uint32_t)(M + 16 * s.tm - 1) / (16u * s.tm)) * ((uint32_t)(N + 16 * s.tn - 1) / (16u * s.tn));
    if (groups >= 1 << 23) return 1e29;  // (of 512 threads: more than one launch holds)
    const int64_t rows = (M < 16 * s.tm ? M : 16 * s.tm) + 16 * s.tn * (gated ? 2 : 1);
    const double cu = (double)((groups + 255) >> 8) * rows * k_bytes / (shift ? 20e3 : 33e3);
    return 2.8 + (cu > memory ? cu : memory);
}

// copied: bytes that a tiled form would have to copy first (0.4 us per MB and a launch), where the registers form reads
// anything as it is.  tiled: whether the rows are short enough for the tiled forms.
Choice choose(bool gated, int M, int N, int64_t k_bytes, int64_t copied, bool tiled, bool shift) {
    Choice best;
    const double memory = ((double)M + (double)N * (gated ? 2 : 1)) * k_bytes / 5.4e6;
    const int forced = forced_form();
    for (int i = 0; i < ROWS_FORMS; ++i) {
        const double cost = rows_cost(kRows[i], gated, M, N, k_bytes, memory, shift);
        if (forced >= 0 ? forced == i || (!tiled && i == 0) : cost < best.cost) {
            best.form = i;
            best.cost = cost;
        }
    }
    if (!tiled) return best;
    for (int i = 0; i < TILE_FORMS; ++i) {
        if (forced >= 0 && forced != ROWS_FORMS + i) continue;
        const Tiling whole = tiling(i, gated, M, N, 1, k_bytes);
        for (int splits : kSplits) {
            const int fs = knobs().ffn_splits;
            if (splits > 1 && (fs || whole.count() * splits > 512)) break;  // (more only costs)
            const Tiling t = cut_depth(whole, i, gated, M, N, fs ? fs : splits);
            if (!fs && t.splits != splits) break;
            const double cost = tiled_cost(kTiles[i], &t, 1, memory) + (copied ? 3.0 + copied * 0.4e-6 : 0.0);
            if (cost < best.cost || (forced >= 0 && best.form != forced)) {
                best.form = ROWS_FORMS + i;
                best.tiling = t;
                best.cost = cost;
            }
        }
    }
    return best;
}

Product tiled_product(Product p, const Tiling &c, uint32_t *ws) {
    p.tiles_m = c.tiles_m;
    p.tiles_n = c.tiles_n;
    p.batch = c.batch;
    p.group_m = 4;  // (8192 x 12288 x 4096 gated, us: 4 1287, 6 1365, 8 1308, 16 1342; 8-bit 8192^3 424, 424, 431, 444)
    p.splits = c.splits;
    p.steps_per_split = c.steps_per_split;
    p.ws = ws;
    p.ws_ld = c.ws_ld;
    p.ws_plane = c.ws_plane;
    p.ws_split = c.ws_split;
    return p;
}

// Workgroups that the card holds at once.
template <typename Cfg> constexpr int resident() {
    constexpr int by_lds = 160 * 1024 / Cfg::LDS, by_waves = 8 / Cfg::WAVES;
    return 256 * (by_lds < by_waves ? by_lds : by_waves);
}

unsigned join_grid(const Product &p) {
    const int64_t work = (p.ws_ld >> 2) * p.M * p.batch;
    return (unsigned)(ceil_div(work, 256) < 2048 ? ceil_div(work, 256) : 2048);
}

template <int ET, bool GATED> hipError_t run_tiles(const Product &p, int tile, int K, hipStream_t stream) {
    hipError_t e = with_tile<ET, GATED>(tile, [&](auto cfg) {
        typedef decltype(cfg) Cfg;
        const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.batch * p.splits;
        if (tiles > 0x7fffffff - 65536) return hipErrorNotSupported;
        const unsigned grid = (unsigned)(tiles < resident<Cfg>() ? tiles : resident<Cfg>());
        hipError_t e = ensure_dynamic_lds((const void *)tile_kernel<Cfg>, Cfg::LDS);
        if (e == hipSuccess) e = launch_kernel(tile_kernel<Cfg>, dim3(grid), dim3(Cfg::THREADS), Cfg::LDS, stream, p);
        return launched("ffn_tile_kernel", type_letter(ET), Cfg::BM, Cfg::CHANNELS, Cfg::THREADS, p.M, p.N, K, grid, 1, p.splits, e);
    });
    if (e != hipSuccess || p.splits == 1) return e;
    const unsigned grid = join_grid(p);
    e = launch_kernel(join_kernel<ET, GATED>, dim3(grid), dim3(256), 0, stream, p);
    return launched("ffn_join_kernel", type_letter(ET), 1, 4, 256, p.M, p.N, K, grid, 1, p.splits, e);
}

template <typename Cfg> hipError_t launch_rows(Product p, int K, hipStream_t stream) {
    p.tiles_m = (int)ceil_div(p.M, 16 * Cfg::TM);
    p.tiles_n = (int)ceil_div(p.N, 16 * Cfg::TN);
    p.batch = p.splits = 1;
    const int64_t grid = (int64_t)p.tiles_m * p.tiles_n;
    if (grid * Cfg::THREADS > 0xffffffffLL) return hipErrorNotSupported;
    if (Cfg::LDS > 65536) {
        hipError_t e = ensure_dynamic_lds((const void *)rows_kernel<Cfg>, Cfg::LDS);
        if (e != hipSuccess) return e;
    }
    hipError_t e = launch_kernel(rows_kernel<Cfg>, dim3((unsigned)grid), dim3(Cfg::THREADS), Cfg::LDS, stream, p);
    return launched("ffn_rows_kernel", type_letter(Cfg::ET), 16 * Cfg::TM, 16 * Cfg::TN, Cfg::THREADS, p.M, p.N, K, (unsigned)grid, 1, 1, e);
}

template <int ET, bool GATED, bool SHIFT> hipError_t run_rows(const Product &p, int form, int K, hipStream_t stream) {
    switch (form) {
    case 0: return launch_rows<RowsCfg<ET, 1, 1, 8, SHIFT ? 3 : 4, GATED, SHIFT>>(p, K, stream);
    case 1: return launch_rows<RowsCfg<ET, 2, 1, 8, SHIFT ? 2 : 4, GATED, SHIFT>>(p, K, stream);
    case 2: return launch_rows<RowsCfg<ET, 2, 2, 8, SHIFT ? 1 : 2, GATED, SHIFT>>(p, K, stream);
    default: return launch_rows<RowsCfg<ET, 4, 2, 4, SHIFT ? 1 : 2, GATED, SHIFT>>(p, K, stream);
    }
}

// Layout of one call's copies in the stream's buffer.
struct Copies {
    size_t used = 0;
    size_t add(size_t bytes) {
        const size_t at = used;
        used += (size_t)round_up((int64_t)bytes, 256);
        return at;
    }
};

// Whether the tiled product can load an operand from where it is: dword-aligned rows, near enough to each other for 32-bit
// offsets across a tile.
bool fits(const void *ptr, int64_t ld_bytes) {
    return (reinterpret_cast<uintptr_t>(ptr) & 3) == 0 && (ld_bytes & 3) == 0 && ld_bytes <= kMaxRowBytes;
}

hipError_t copy_rows(const CopyList &list, int n, hipStream_t stream) {
    if (n == 0) return hipSuccess;
    int64_t work = 0;
    for (int i = 0; i < n; ++i) work = list.c[i].rows * (list.c[i].ld_to >> 4) > work ? list.c[i].rows * (list.c[i].ld_to >> 4) : work;
    const dim3 grid((unsigned)(ceil_div(work, 256) < 4096 ? ceil_div(work, 256) : 4096), (unsigned)n);
    hipError_t e = launch_kernel(copy_rows_kernel, grid, dim3(256), 0, stream, list);
    return launched("ffn_copy_rows_kernel", 'p', 1, 16, 256, (int)list.c[0].rows, (int)list.c[0].bytes, 0, grid.x, grid.y, 1, e);
}

// A product whose operands are the caller's: chooses its form, copies what that form cannot load, and runs it.
template <int ET, bool GATED>
hipError_t product_from(int es, int M, int N, int K, Mat A, Mat B0, Mat B1, Product p, hipStream_t stream) {
    constexpr int OPERANDS = GATED ? 3 : 2;
    const int64_t kb = (int64_t)K * es, kp = round_up(kb, 128);  // (copies: rows of whole cache lines)
    const Mat in[3] = {A, B0, B1};
    const int64_t rows[3] = {M, N, N};
    const void *ptr[3] = {};
    int64_t ld[3] = {};
    size_t at[3] = {};
    bool copy[3] = {};
    Copies copies;
    for (int i = 0; i < OPERANDS; ++i) {
        ptr[i] = in[i].ptr;
        ld[i] = in[i].ld * es;
        copy[i] = !fits(ptr[i], ld[i]);
        if (copy[i]) at[i] = copies.add((size_t)kp * rows[i]);
    }
    bool shift = false;  // some row does not start on a dword
    for (int i = 0; i < OPERANDS; ++i) shift |= ((reinterpret_cast<uintptr_t>(ptr[i]) | (uintptr_t)ld[i]) & 3) != 0;
    const Choice c = choose(GATED, M, N, kb, (int64_t)copies.used, kp <= kMaxRowBytes, shift);
    const bool tiled = c.form >= ROWS_FORMS;
    char *buf = nullptr;
    uint32_t *ws = nullptr;
    hipError_t e = hipSuccess;
    if (tiled && copies.used) e = workspace_get(stream, copies.used, WS_TRMM, (void **)&buf);
    if (e == hipSuccess && tiled && c.tiling.ws_bytes) e = workspace_get(stream, c.tiling.ws_bytes, WS_GEMM, (void **)&ws);
    if (e != hipSuccess) return e;
    CopyList list = {};
    int n = 0;
    for (int i = 0; i < OPERANDS; ++i) {
        if (!tiled || !copy[i]) continue;
        list.c[n++] = Copy{static_cast<const char *>(ptr[i]), buf + at[i], ld[i], kb, kp, rows[i]};
        ptr[i] = buf + at[i];
        ld[i] = kp;
    }
    if ((e = copy_rows(list, n, stream)) != hipSuccess) return e;
    p.A[0] = p.A[1] = ptr[0];
    p.lda = ld[0];
    p.a_bytes = (M - 1) * ld[0] + kb;
    for (int h = 0; h < 2; ++h) {
        const int i = GATED ? 1 + h : 1;
        p.B[h] = ptr[i];
        p.ldb[h] = ld[i];
        p.b_bytes[h] = (N - 1) * ld[i] + kb;
    }
    p.k_bytes = kb;
    p.M = M;
    p.N = N;
    if (!tiled) return shift ? run_rows<ET, GATED, true>(p, c.form, K, stream) : run_rows<ET, GATED, false>(p, c.form, K, stream);
    return run_tiles<ET, GATED>(tiled_product(p, c.tiling, ws), c.form - ROWS_FORMS, K, stream);
}

// The two products of the gradient in one launch.  A product that is not wanted, or not here, has no tiles.
template <int ET, bool TWO> hipError_t run_two(const Product &px, const Product &pw, const Tiling *c, int tile, int M, int N, int K, hipStream_t stream) {
    const int64_t nx = c[0].count(), nw = c[1].count();
    if (nx > 0x3fffffff || nw > 0x3fffffff) return hipErrorNotSupported;
    hipError_t e = with_grad_tile<ET, TWO>(tile, [&](auto cfg) {
        typedef decltype(cfg) Cfg0;
        typedef TileCfg<ET, Cfg0::BM, Cfg0::BN, Cfg0::WM, Cfg0::WN, Cfg0::S, false, ACROSS_K, ACROSS_K, TWO> Cfg1;
        int64_t grid = nx + nw < resident<Cfg0>() ? nx + nw : resident<Cfg0>();
        const int64_t blocks = share_out(c, (int)grid).blocks;
        if (grid - blocks > nw) grid = blocks + nw;
        auto kernel = two_tiles_kernel<Cfg0, Cfg1>;
        hipError_t e = ensure_dynamic_lds((const void *)kernel, Cfg0::LDS);
        if (e == hipSuccess) e = launch_kernel(kernel, dim3((unsigned)grid), dim3(Cfg0::THREADS), Cfg0::LDS, stream, ProductPair{{px, pw}}, (int)blocks);
        return launched("ffn_two_tiles_kernel", type_letter(ET), Cfg0::BM, Cfg0::BN, Cfg0::THREADS, M, N, K, (unsigned)grid, 1, c[0].splits, e);
    });
    if (e != hipSuccess || (px.splits <= 1 && pw.splits <= 1)) return e;
    const unsigned gx = px.splits > 1 ? join_grid(px) : 0, gw = pw.splits > 1 ? join_grid(pw) : 0;
    const dim3 grid(gx > gw ? gx : gw, 2);
    e = launch_kernel(join_two_kernel<ET>, grid, dim3(256), 0, stream, ProductPair{{px, pw}});
    return launched("ffn_join_two_kernel", type_letter(ET), 1, 4, 256, M, N, K, grid.x, 2, px.splits > pw.splits ? px.splits : pw.splits, e);
}

// Tiles and ranges of depth for one launch over dX's product (M x K, x_bytes deep), the weights' (N x K twice, w_bytes deep) or
// both; one tile, and ranges of about the same length for both.
struct GradTiling {
    Tiling c[2];
    int tile[2] = {0, 0};
    double cost = 1e30;
};
GradTiling grad_tiling(const TileShape *tiles, int M, int N, int K, int64_t x_bytes, int64_t w_bytes, bool want_x, bool want_w) {
    GradTiling best;
    for (int i = 0; i < TILE_FORMS; ++i) {
        if (forced_form() >= ROWS_FORMS && forced_form() != ROWS_FORMS + i) continue;
        Tiling whole[2];
        if (want_x) whole[0] = tiling(i, false, M, K, 1, x_bytes);
        if (want_w) whole[1] = tiling(i, false, N, K, 2, w_bytes);
        const int longest = whole[0].steps_per_split > whole[1].steps_per_split ? whole[0].steps_per_split : whole[1].steps_per_split;
        for (int cut : kSplits) {
            const int fs = knobs().ffn_splits;
            if (cut > 1 && (fs || cut > longest || whole[0].count() + whole[1].count() > 2048)) break;
            const uint32_t range = (uint32_t)(longest + cut - 1) / (uint32_t)cut;
            Tiling t[2];
            for (int j = 0; j < 2; ++j) t[j] = cut_depth(whole[j], i, false, j ? N : M, K, fs ? fs : (int)((whole[j].steps_per_split + range - 1) / range));
            if (cut > 1 && t[0].count() + t[1].count() > 2048) break;
            const double cost = tiled_cost(tiles[i], t, 2, 0.0);
            if (cost < best.cost) {
                best.cost = cost;
                for (int j = 0; j < 2; ++j) {
                    best.c[j] = t[j];
                    best.tile[j] = i;
                }
            }
        }
    }
    return best;
}

const int kTops = 1024;  // workgroups of the pass that finds f16's largest term: what every one of the next pass reads
template <int ET, int OT, bool TWO>
hipError_t grad_of(int gate, int M, int N, int K, Mat dH, Mat X, Mat Wg, Mat Wu, Mat G, Mat U, OutMat dX, OutMat dWg, OutMat dWu,
                   hipStream_t stream) {
    // [dG], [dU]: bytes from token to token, and from one to the other
    const int64_t row = round_up((int64_t)N * (TWO ? 4 : 2), 128), plane = M * row, w_bytes = (int64_t)M * (TWO ? 4 : 2);
    const bool want_x = dX.ptr, want_w = dWg.ptr;
    // operands that the tiles load as they are, or copies
    Mat in[3] = {X, Wg, Wu};
    const int64_t rows[3] = {M, N, N}, ld_copy = round_up((int64_t)K * 2, 128);
    const bool used[3] = {want_w, want_x, want_x};
    Copies copies;
    size_t at[3] = {0, 0, 0};
    bool copy[3];
    for (int i = 0; i < 3; ++i) {
        copy[i] = used[i] && !fits(in[i].ptr, in[i].ld * 2);
        if (copy[i]) at[i] = copies.add((size_t)rows[i] * ld_copy);
    }
    // Both products in one launch, or each in its own where their sizes ask for different tiles and ranges (few tokens: dX is all
    // depth, the weights' gradients all results; us, one number a term, together / apart: 1 x 12288 x 4096 191 / 112, 8 x 4096 x 4096 66 / 42, 64 x
    // 12288 x 4096 237 / 119; but 200 x 4096 x 4096 64 / 69, 509 x 1367 x 770 30 / 36).
    const TileShape *tiles = TWO ? kTermTiles : kTiles;
    GradTiling both = grad_tiling(tiles, M, N, K, 2 * row, w_bytes, want_x, want_w);
    bool apart = false;
    if (want_x && want_w) {
        const GradTiling x = grad_tiling(tiles, M, N, K, 2 * row, w_bytes, true, false), w = grad_tiling(tiles, M, N, K, 2 * row, w_bytes, false, true);
        apart = x.cost + w.cost < both.cost;
        if (apart) {
            both.c[0] = x.c[0];
            both.c[1] = w.c[1];
            both.tile[0] = x.tile[0];
            both.tile[1] = w.tile[1];
        }
    }
    const Tiling *c = both.c;
    // the gemm buffer: partial sums of either product, the terms, and for f16 what their scale comes from
    const int64_t work = M * (row >> (TWO ? 5 : 4));
    const int tops = OT == OT_F16 ? (int)(ceil_div(work, 256) < kTops ? ceil_div(work, 256) : kTops) : 0;
    Copies scratch;
    const size_t at_x = scratch.add(c[0].ws_bytes), at_w = scratch.add(c[1].ws_bytes), at_terms = scratch.add((size_t)(2 * plane));
    const size_t at_tops = scratch.add((size_t)tops * 4 + 4);
    char *buf = nullptr, *ws = nullptr;
    hipError_t e = copies.used ? workspace_get(stream, copies.used, WS_TRMM, (void **)&buf) : hipSuccess;
    if (e == hipSuccess) e = workspace_get(stream, scratch.used, WS_GEMM, (void **)&ws);
    if (e != hipSuccess) return e;
    const void *ptr[3];
    int64_t ld[3];
    CopyList list = {};
    int n = 0;
    for (int i = 0; i < 3; ++i) {
        ptr[i] = copy[i] ? buf + at[i] : in[i].ptr;
        ld[i] = copy[i] ? ld_copy : in[i].ld * 2;
        if (copy[i]) list.c[n++] = Copy{static_cast<const char *>(in[i].ptr), buf + at[i], in[i].ld * 2, (int64_t)K * 2, ld_copy, rows[i]};
    }
    if ((e = copy_rows(list, n, stream)) != hipSuccess) return e;
    GateGrad gate_grad = {dH.ptr, G.ptr, U.ptr, dH.ld, G.ld, U.ld, M, N, gate, ws + at_terms, row, plane, (uint32_t *)(ws + at_tops), tops,
                          (float *)(ws + at_tops) + tops};
    if (OT == OT_F16) {
        e = launch_kernel(gate_grad_top_kernel, dim3((unsigned)tops), dim3(256), 0, stream, gate_grad);
        if ((e = launched("ffn_gate_grad_top_kernel", type_letter(ET), 1, 8, 256, M, N, K, (unsigned)tops, 1, 1, e)) != hipSuccess) return e;
    }
    const unsigned grid = (unsigned)(ceil_div(work, 256) < 8192 ? ceil_div(work, 256) : 8192);
    e = launch_kernel(gate_grad_kernel<OT, TWO>, dim3(grid), dim3(256), 0, stream, gate_grad);
    if ((e = launched("ffn_gate_grad_kernel", type_letter(ET), 1, 8, 256, M, N, K, grid, 1, 1, e)) != hipSuccess) return e;
    Product p[2] = {};  // [dG | dU] times [Wg; Wu]: the depth runs through dG's row and Wg's rows, then through dU's and Wu's
    p[0].A[0] = p[0].A[1] = gate_grad.out;
    p[0].a_bytes = 2 * plane;
    p[0].a_jump = plane - row;
    for (int h = 0; h < 2; ++h) {
        p[0].B[h] = ptr[1 + h];
        p[0].ldb[h] = ld[1 + h];
        p[0].b_bytes[h] = (N - 1) * ld[1 + h] + (int64_t)K * 2;
    }
    p[0].k_bytes = 2 * row;
    p[0].part_steps = (int)(row >> 7);
    p[0].C[0] = p[0].C[1] = dX.ptr;
    p[0].ldc[0] = p[0].ldc[1] = dX.ld;
    p[0].M = M;
    // dG^T X and dU^T X: the depth runs through the tokens
    for (int z = 0; z < 2; ++z) {
        p[1].A[z] = gate_grad.out + z * plane;
        p[1].B[z] = ptr[0];
        p[1].ldb[z] = ld[0];
        p[1].b_bytes[z] = (M - 1) * ld[0] + (int64_t)K * 2;
    }
    p[1].a_bytes = plane;
    p[1].k_bytes = w_bytes;
    p[1].C[0] = dWg.ptr;
    p[1].C[1] = dWu.ptr;
    p[1].ldc[0] = dWg.ld;
    p[1].ldc[1] = dWu.ld;
    p[1].M = N;
    for (int i = 0; i < 2; ++i) {
        p[i].out_type = OT;
        p[i].lda = row;
        p[i].N = K;
        p[i].unscale = gate_grad.unscale;
        p[i] = tiled_product(p[i], c[i], (uint32_t *)(ws + (i ? at_w : at_x)));
    }
    if (!apart) return run_two<ET, TWO>(p[0], p[1], c, both.tile[0], M, N, K, stream);
    const Tiling only_x[2] = {c[0], Tiling()}, only_w[2] = {Tiling(), c[1]};
    e = run_two<ET, TWO>(p[0], Product(), only_x, both.tile[0], M, N, K, stream);
    return e != hipSuccess ? e : run_two<ET, TWO>(Product(), p[1], only_w, both.tile[1], M, N, K, stream);
}

}  // namespace

template <typename T, bool WAVE>
static hipError_t run_quantize(int M, int K, const void *X, int64_t ldx, int8_t *Q, int64_t ldq, float *scale, char type, hipStream_t stream) {
    const int64_t groups = WAVE ? ceil_div(M, 4) : M;
    const dim3 grid((unsigned)(groups < (1 << 20) ? groups : 1 << 20), (unsigned)ceil_div(groups, 1 << 20));
    const hipError_t e = launch_kernel(quantize_kernel<T, WAVE>, grid, dim3(256), 0, stream, static_cast<const T *>(X), ldx, Q, ldq, scale, M, K);
    return launched("ffn_quantize_kernel", type, WAVE ? 4 : 1, K, 256, M, 1, K, grid.x, grid.y, 1, e);
}
template <typename T> static hipError_t quantize_as(int M, int K, Mat X, int8_t *Q, int64_t ldq, float *scale, char type, hipStream_t stream) {
    // Short rows in great number get a wave each instead of a workgroup: the launch of the workgroups is the time (bf16, us, a
    // workgroup / a wave a row: 16384 x 64 14.0 / 6.6, x 1000 18.4 / 12.6, x 2048 22.4 / 23.1, x 4096 34.7 / 47.5; 4096 x 1000 6.5 /
    // 5.5, x 2048 7.9 / 9.3; of 1024 rows no difference up to 1000, 4.7 / 7.1 at 2048).
    if (K <= kWaveRow && M >= 2048) return run_quantize<T, true>(M, K, X.ptr, X.ld, Q, ldq, scale, type, stream);
    return run_quantize<T, false>(M, K, X.ptr, X.ld, Q, ldq, scale, type, stream);
}
hipError_t quantize_rows(int type, int M, int K, Mat X, int8_t *Q, int64_t ldq, float *scale, hipStream_t stream) {
    if (type == OT_F32) return quantize_as<float>(M, K, X, Q, ldq, scale, 's', stream);
    if (type == OT_F16) return quantize_as<_Float16>(M, K, X, Q, ldq, scale, 'h', stream);
    return quantize_as<__bf16>(M, K, X, Q, ldq, scale, 'b', stream);
}

hipError_t product_i8(int out_type, int gate, int M, int N, int K, Mat A, const float *sA, Mat Bg, const float *sBg, Mat Bu,
                      const float *sBu, OutMat C, hipStream_t stream) {
    Product p = {};
    p.scale_a = sA;
    p.scale_b[0] = sBg;
    p.scale_b[1] = sBu;
    p.C[0] = p.C[1] = C.ptr;
    p.ldc[0] = p.ldc[1] = C.ld;
    p.out_type = out_type;
    p.gate = gate;
    if (Bu.ptr) return product_from<ET_I8, true>(1, M, N, K, A, Bg, Bu, p, stream);
    return product_from<ET_I8, false>(1, M, N, K, A, Bg, Bu, p, stream);
}

hipError_t gated(int type, int gate, int M, int N, int K, Mat X, Mat Wg, Mat Wu, OutMat H, OutMat G, OutMat U, hipStream_t stream) {
    Product p = {};
    p.C[0] = p.C[1] = H.ptr;
    p.ldc[0] = p.ldc[1] = H.ld;
    p.save[0] = G.ptr;
    p.save[1] = U.ptr;
    p.ld_save[0] = G.ld;
    p.ld_save[1] = U.ld;
    p.out_type = type;
    p.gate = gate;
    if (type == OT_F16) return product_from<ET_F16, true>(2, M, N, K, X, Wg, Wu, p, stream);
    return product_from<ET_BF16, true>(2, M, N, K, X, Wg, Wu, p, stream);
}

hipError_t gated_grad(int type, int gate, int M, int N, int K, Mat dH, Mat X, Mat Wg, Mat Wu, Mat G, Mat U, OutMat dX, OutMat dWg,
                      OutMat dWu, hipStream_t stream) {
    const bool two = !(gate & ROUND_TERMS);
    const auto run = type == OT_F16 ? (two ? grad_of<ET_F16, OT_F16, true> : grad_of<ET_F16, OT_F16, false>)
                                    : (two ? grad_of<ET_BF16, OT_BF16, true> : grad_of<ET_BF16, OT_BF16, false>);
    return run(gate & ~ROUND_TERMS, M, N, K, dH, X, Wg, Wu, G, U, dX, dWg, dWu, stream);
}

}  // namespace ffn
}  // namespace cba
