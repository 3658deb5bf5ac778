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
// One workgroup per row; a row of up to 8192 elements stays in registers between the two passes.
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

template <typename T> __global__ __launch_bounds__(256) void quantize_kernel(const T *X, int64_t ldx, int8_t *Q, int64_t ldq, float *scale, int M, int K) {
    constexpr int KEEP = 4;
    struct Vec8 { T v[8]; };
    __shared__ uint32_t part[4];
    for (int row = blockIdx.x; row < M; row += gridDim.x) {
        const T *x = X + (int64_t)row * ldx;
        int8_t *q = Q + (int64_t)row * ldq;
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
            const int c = threadIdx.x + i * 256;
            if (c < vecs) {
                __builtin_memcpy(&kept[i], x + (int64_t)c * 8, sizeof(Vec8));
#pragma unroll
                for (int e = 0; e < 8; ++e) take(kept[i].v[e]);
            }
        }
        for (int c = threadIdx.x + KEEP * 256; c < vecs; c += 256) {
            Vec8 v;
            __builtin_memcpy(&v, x + (int64_t)c * 8, sizeof(Vec8));
#pragma unroll
            for (int e = 0; e < 8; ++e) take(v.v[e]);
        }
        const int tail = vecs * 8 + threadIdx.x;
        if (tail < K) take(x[tail]);
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            const uint32_t o = __shfl_xor(top, d);
            top = o > top ? o : top;
        }
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) top = part[w] > top ? part[w] : top;
        float a = __builtin_bit_cast(float, top);
        if (threadIdx.x == 0) scale[row] = a / 127.f;
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
            const int c = threadIdx.x + i * 256;
            if (c < vecs) eight(kept[i], c);
        }
        for (int c = threadIdx.x + KEEP * 256; c < vecs; c += 256) {
            Vec8 v;
            __builtin_memcpy(&v, x + (int64_t)c * 8, sizeof(Vec8));
            eight(v, c);
        }
        if (tail < K) q[tail] = one(x[tail]);
        __syncthreads();  // (the next row's parts)
    }
}

// ---- copies that make an operand fit the tiled product ----

// Rows of `bytes` bytes, `ld` apart and aligned to nothing -> rows `ld_to` apart (a multiple of 16), zeros behind.
__global__ __launch_bounds__(256) void pack_rows_kernel(const char *from, int64_t ld, int64_t bytes, char *to, int64_t ld_to, int64_t rows) {
    const int64_t per = ld_to >> 4, total = per * rows;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int64_t row = t / per, at = (t - row * per) * 16;
        const char *src = from + row * ld + at;
        char v[16] = {};
        if (at + 16 <= bytes) {
            __builtin_memcpy(v, src, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (at + e < bytes) v[e] = src[e];
        }
        __builtin_memcpy(__builtin_assume_aligned(to + row * ld_to + at, 16), v, 16);
    }
}

// ---- gradients of the gate ----
//
// dG = dH o U o act'(G), dU = dH o act(G), rounded to the operands' 16 bits as the two products that follow take
// them (each result below sums many of them: the roundings, independent and unbiased, add up to about one more
// rounding of the result).  A row per token, [dG | dU], either half padded with zeros to a multiple of 64.
template <int OT> __global__ __launch_bounds__(256) void gate_grad_kernel(const void *dH_, int64_t lddh, const void *G_, int64_t ldg, const void *U_,
                                                                          int64_t ldu, int M, int N, int gate, void *out_, int64_t half) {
    typedef typename Store<OT>::type T;
    struct Vec8 { T v[8]; };
    const T *dH = static_cast<const T *>(dH_), *G = static_cast<const T *>(G_), *U = static_cast<const T *>(U_);
    T *out = static_cast<T *>(out_);
    const int64_t per_row = half >> 3, total = per_row * M;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        const int64_t m = t / per_row;
        const int n = (int)(t - m * per_row) * 8;
        const T *h = dH + m * lddh + n, *g = G + m * ldg + n, *u = U + m * ldu + n;
        Vec8 vh = {}, vg = {}, vu = {}, dg, du;
        if (n + 8 <= N) {
            __builtin_memcpy(&vh, h, 16);
            __builtin_memcpy(&vg, g, 16);
            __builtin_memcpy(&vu, u, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < N) {
                    vh.v[e] = h[e];
                    vg.v[e] = g[e];
                    vu.v[e] = u[e];
                }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float act, slope;
            gate_value_and_slope(gate, (float)vg.v[e], act, slope);
            const float dh = (float)vh.v[e];
            dg.v[e] = Store<OT>::of(dh * (float)vu.v[e] * slope);
            du.v[e] = Store<OT>::of(dh * act);
        }
        T *to = out + m * 2 * half + n;
        __builtin_memcpy(__builtin_assume_aligned(to, 16), &dg, 16);
        __builtin_memcpy(__builtin_assume_aligned(to + half, 16), &du, 16);
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

template <typename Cfg> hipError_t launch_tiles(const Product &p, int K, hipStream_t stream) {
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.batch * p.splits;
    if (tiles > 0x7fffffff - 65536) return hipErrorNotSupported;
    // as many workgroups as the card holds at once
    const int per_cu = 160 * 1024 / Cfg::LDS < 8 / Cfg::WAVES ? 160 * 1024 / Cfg::LDS : 8 / Cfg::WAVES;
    const unsigned grid = (unsigned)(tiles < 256 * per_cu ? tiles : 256 * per_cu);
    hipError_t e = ensure_dynamic_lds((const void *)tile_kernel<Cfg>, Cfg::LDS);
    if (e != hipSuccess) return e;
    e = launch_kernel(tile_kernel<Cfg>, dim3(grid), dim3(Cfg::THREADS), Cfg::LDS, stream, p);
    return launched("ffn_tile_kernel", type_letter(Cfg::ET), Cfg::BM, Cfg::CHANNELS, Cfg::THREADS, p.M, p.N, K, grid, 1, p.splits, e);
}

// The tiled forms: edges, and the index by which a form is known (the forms that run from registers come first).
enum { ROWS_FORMS = 6 };
struct TileShape { int bm, bn; };
const TileShape kTiles[] = {{256, 256}, {256, 128}, {128, 128}, {128, 128}, {64, 128}, {64, 128}, {64, 64}, {128, 64}};

template <int ET, bool GATED, Lay LA, Lay LB, typename F> hipError_t with_tile(int tile, F &&f) {
    switch (tile) {
    case 0: return f(TileCfg<ET, 256, 256, 128, 64, 2, GATED, LA, LB>());
    case 1: return f(TileCfg<ET, 256, 128, 64, 64, 3, GATED, LA, LB>());
    case 2: return f(TileCfg<ET, 128, 128, 64, 64, 5, GATED, LA, LB>());
    case 3: return f(TileCfg<ET, 128, 128, 64, 64, 2, GATED, LA, LB>());
    case 4: return f(TileCfg<ET, 64, 128, 32, 64, 3, GATED, LA, LB>());
    case 5: return f(TileCfg<ET, 64, 128, 32, 64, 6, GATED, LA, LB>());
    case 6: return f(TileCfg<ET, 64, 64, 32, 32, 5, GATED, LA, LB>());
    default: return f(TileCfg<ET, 128, 64, 64, 32, 3, GATED, LA, LB>());
    }
}

struct TileChoice {
    int tile = 0, tiles_m = 0, tiles_n = 0, splits = 1, steps_per_split = 0;
    int64_t ws_ld = 0, ws_plane = 0, ws_split = 0;
    size_t ws_bytes = 0;
};

// The 256 x 256 tile where its tiles fill the 256 CUs, else 128 x 128, with the depth cut into ranges (of at least four
// steps) until they do.
TileChoice choose(bool gated, int M, int N, int batch, int64_t k_bytes) {
    TileChoice c;
    const int64_t steps = ceil_div(k_bytes, 128);
    auto tiles = [&](int bm, int bn) { return ceil_div(M, bm) * ceil_div(N, gated ? bn / 2 : bn) * batch; };
    c.tile = tiles(256, 256) >= 256 ? 0 : 2;
    if (knobs().ffn_form >= ROWS_FORMS) c.tile = knobs().ffn_form - ROWS_FORMS;
    const TileShape t = kTiles[c.tile];
    c.tiles_m = (int)ceil_div(M, t.bm);
    c.tiles_n = (int)ceil_div(N, gated ? t.bn / 2 : t.bn);
    int64_t splits = 1;
    if (t.bm * t.bn < 65536) {
        splits = 512 / tiles(t.bm, t.bn);
        if (splits > steps / 4) splits = steps / 4;
        if (splits > 64) splits = 64;
    }
    if (knobs().ffn_splits) splits = knobs().ffn_splits < steps ? knobs().ffn_splits : steps;
    if (splits < 1 || t.bm * t.bn >= 65536) splits = 1;  // (the largest tiles do not split: TileCfg::SPLITS)
    c.steps_per_split = (int)ceil_div(steps, splits);
    c.splits = (int)ceil_div(steps, c.steps_per_split);
    if (c.splits > 1) {
        c.ws_ld = round_up(N, 4);
        c.ws_plane = c.ws_ld * M;
        c.ws_split = c.ws_plane * (gated ? 2 : batch);
        c.ws_bytes = (size_t)c.ws_split * 4 * c.splits;
    }
    return c;
}

template <int ET, bool GATED, Lay LA, Lay LB> hipError_t run_product(Product p, const TileChoice &c, uint32_t *ws, int K, hipStream_t stream) {
    p.tiles_m = c.tiles_m;
    p.tiles_n = c.tiles_n;
    p.group_m = 8;
    p.splits = c.splits;
    p.steps_per_split = c.steps_per_split;
    p.ws = ws;
    p.ws_ld = c.ws_ld;
    p.ws_plane = c.ws_plane;
    p.ws_split = c.ws_split;
    hipError_t e = with_tile<ET, GATED, LA, LB>(c.tile, [&](auto cfg) { return launch_tiles<decltype(cfg)>(p, K, stream); });
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t work = (c.ws_ld >> 2) * p.M * p.batch;
    const unsigned grid = (unsigned)(ceil_div(work, 256) < 2048 ? ceil_div(work, 256) : 2048);
    e = launch_kernel(join_kernel<ET, GATED>, dim3(grid), dim3(256), 0, stream, p);
    return launched("ffn_join_kernel", type_letter(ET), 1, 4, 256, p.M, p.N, K, grid, 1, p.splits, e);
}

template <typename Cfg> hipError_t launch_rows(Product p, int K, hipStream_t stream) {
    p.tiles_m = (int)ceil_div(p.M, 16 * Cfg::TM);
    p.tiles_n = (int)ceil_div(p.N, 16 * Cfg::TN);
    const int64_t grid = (int64_t)p.tiles_m * p.tiles_n;
    if (grid * Cfg::THREADS > 0xffffffffLL) return hipErrorNotSupported;
    if (Cfg::LDS > 65536) {
        hipError_t e = ensure_dynamic_lds((const void *)rows_kernel<Cfg>, Cfg::LDS);
        if (e != hipSuccess) return e;
    }
    hipError_t e = launch_kernel(rows_kernel<Cfg>, dim3((unsigned)grid), dim3(Cfg::THREADS), Cfg::LDS, stream, p);
    return launched("ffn_rows_kernel", type_letter(Cfg::ET), 16 * Cfg::TM, 16 * Cfg::TN, Cfg::THREADS, p.M, p.N, K, (unsigned)grid, 1, 1, e);
}

template <int ET, bool GATED> hipError_t run_rows(const Product &p, int form, int K, hipStream_t stream) {
    switch (form) {
    case 0: return launch_rows<RowsCfg<ET, 1, 1, 8, 4, GATED>>(p, K, stream);
    case 1: return launch_rows<RowsCfg<ET, 2, 1, 8, 4, GATED>>(p, K, stream);
    case 2: return launch_rows<RowsCfg<ET, 2, 2, 8, 2, GATED>>(p, K, stream);
    case 3: return launch_rows<RowsCfg<ET, 4, 1, 8, 2, GATED>>(p, K, stream);
    case 4: return launch_rows<RowsCfg<ET, 4, 2, 4, 2, GATED>>(p, K, stream);
    default: return launch_rows<RowsCfg<ET, 4, GATED ? 2 : 4, 4, 2, GATED>>(p, K, stream);
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
    return (reinterpret_cast<uintptr_t>(ptr) & 3) == 0 && (ld_bytes & 3) == 0 && ld_bytes < ((int64_t)1 << 22);
}

hipError_t pack_rows(const void *from, int64_t ld, int64_t bytes, char *to, int64_t ld_to, int64_t rows, hipStream_t stream) {
    const int64_t work = (ld_to >> 4) * rows;
    const unsigned grid = (unsigned)(ceil_div(work, 256) < 4096 ? ceil_div(work, 256) : 4096);
    hipError_t e = launch_kernel(pack_rows_kernel, dim3(grid), dim3(256), 0, stream, (const char *)from, ld, bytes, to, ld_to, rows);
    return launched("ffn_pack_rows_kernel", 'p', 1, 16, 256, (int)rows, (int)bytes, 0, grid, 1, 1, e);
}

// A product whose operands are the caller's: copies the ones that do not fit, then runs it.
template <int ET, bool GATED>
hipError_t product_from(int es, int M, int N, int K, Mat A, Mat B0, Mat B1, Product p, hipStream_t stream) {
    const int64_t kb = (int64_t)K * es, kp = round_up(kb, 16);
    Mat in[3] = {A, B0, B1};
    const int form = knobs().ffn_form;
    if (form >= 0 && form < ROWS_FORMS) {
        p.A[0] = A.ptr;
        p.lda = A.ld * es;
        p.B[0] = B0.ptr;
        p.B[1] = B1.ptr;
        p.ldb[0] = B0.ld * es;
        p.ldb[1] = B1.ld * es;
        p.k_bytes = kb;
        p.M = M;
        p.N = N;
        p.batch = 1;
        return run_rows<ET, GATED>(p, form, K, stream);
    }
    const int64_t rows[3] = {M, N, N};
    size_t at[3] = {0, 0, 0};
    bool copy[3] = {false, false, false};
    Copies copies;
    for (int i = 0; i < (GATED ? 3 : 2); ++i) {
        copy[i] = !fits(in[i].ptr, in[i].ld * es);
        if (copy[i]) at[i] = copies.add((size_t)kp * rows[i]);
    }
    char *buf = nullptr;
    hipError_t e;
    if (copies.used && (e = workspace_get(stream, copies.used, WS_TRMM, (void **)&buf)) != hipSuccess) return e;
    const TileChoice c = choose(GATED, M, N, 1, kb);
    uint32_t *ws = nullptr;
    if (c.ws_bytes && (e = workspace_get(stream, c.ws_bytes, WS_GEMM, (void **)&ws)) != hipSuccess) return e;
    const void *ptr[3];
    int64_t ld[3], bytes[3];
    for (int i = 0; i < (GATED ? 3 : 2); ++i) {
        ptr[i] = in[i].ptr;
        ld[i] = in[i].ld * es;
        if (copy[i]) {
            if ((e = pack_rows(in[i].ptr, ld[i], kb, buf + at[i], kp, rows[i], stream)) != hipSuccess) return e;
            ptr[i] = buf + at[i];
            ld[i] = kp;
        }
        bytes[i] = (rows[i] - 1) * ld[i] + kb;
    }
    p.A[0] = p.A[1] = ptr[0];
    p.lda = ld[0];
    p.a_bytes = bytes[0];
    for (int h = 0; h < 2; ++h) {
        const int i = GATED ? 1 + h : 1;
        p.B[h] = ptr[i];
        p.ldb[h] = ld[i];
        p.b_bytes[h] = bytes[i];
    }
    p.k_bytes = kb;
    p.M = M;
    p.N = N;
    p.batch = 1;
    p.part_steps = 0x7fffffff;
    return run_product<ET, GATED, ALONG_K, ALONG_K>(p, c, ws, K, stream);
}

template <int ET, int OT>
hipError_t grad_of(int gate, int M, int N, int K, Mat dH, Mat X, Mat Wg, Mat Wu, Mat G, Mat U, OutMat dX, OutMat dWg, OutMat dWu,
                   hipStream_t stream) {
    const int64_t half = round_up(N, 64), row = 2 * half * 2;  // [dG | dU]: elements to dU, bytes to the next token
    const bool want_x = dX.ptr, want_w = dWg.ptr;
    // operands that the tiles load as they are, or copies
    Mat in[3] = {X, Wg, Wu};
    const int64_t rows[3] = {M, N, N}, ld_copy = round_up((int64_t)K * 2, 16);
    const bool used[3] = {want_w, want_x, want_x};
    Copies copies;
    const size_t at_grads = copies.add((size_t)M * row);
    size_t at[3] = {0, 0, 0};
    bool copy[3];
    for (int i = 0; i < 3; ++i) {
        copy[i] = used[i] && !fits(in[i].ptr, in[i].ld * 2);
        if (copy[i]) at[i] = copies.add((size_t)rows[i] * ld_copy);
    }
    const TileChoice cx = choose(false, M, K, 1, row), cw = choose(false, N, K, 2, (int64_t)M * 2);
    size_t sums = want_x ? cx.ws_bytes : 0;
    if (want_w && cw.ws_bytes > sums) sums = cw.ws_bytes;
    char *buf = nullptr;
    uint32_t *ws = nullptr;
    hipError_t e = workspace_get(stream, copies.used, WS_TRMM, (void **)&buf);
    if (e == hipSuccess && sums) e = workspace_get(stream, sums, WS_GEMM, (void **)&ws);
    if (e != hipSuccess) return e;
    char *grads = buf + at_grads;
    const void *ptr[3];
    int64_t ld[3];
    for (int i = 0; i < 3; ++i) {
        ptr[i] = copy[i] ? buf + at[i] : in[i].ptr;
        ld[i] = copy[i] ? ld_copy : in[i].ld * 2;
        if (copy[i] && (e = pack_rows(in[i].ptr, in[i].ld * 2, (int64_t)K * 2, buf + at[i], ld_copy, rows[i], stream)) != hipSuccess) return e;
    }
    const int64_t work = M * (half / 8);
    const unsigned grid = (unsigned)(ceil_div(work, 256) < 8192 ? ceil_div(work, 256) : 8192);
    e = launch_kernel(gate_grad_kernel<OT>, dim3(grid), dim3(256), 0, stream, dH.ptr, dH.ld, G.ptr, G.ld, U.ptr, U.ld, M, N, gate, (void *)grads, half);
    if ((e = launched("ffn_gate_grad_kernel", type_letter(ET), 1, 8, 256, M, N, K, grid, 1, 1, e)) != hipSuccess) return e;
    Product p = {};
    p.out_type = OT;
    p.lda = row;
    if (want_x) {  // [dG | dU] (M x 2 half) times [Wg; Wu]: the depth runs through Wg's rows, then through Wu's
        p.A[0] = p.A[1] = grads;
        p.a_bytes = M * row;
        for (int h = 0; h < 2; ++h) {
            p.B[h] = ptr[1 + h];
            p.ldb[h] = ld[1 + h];
            p.b_bytes[h] = (N - 1) * ld[1 + h] + (int64_t)K * 2;
        }
        p.k_bytes = row;
        p.part_steps = (int)(half / 64);
        p.C[0] = p.C[1] = dX.ptr;
        p.ldc[0] = p.ldc[1] = dX.ld;
        p.M = M;
        p.N = K;
        p.batch = 1;
        if ((e = run_product<ET, false, ALONG_K, ACROSS_K>(p, cx, ws, (int)(2 * half), stream)) != hipSuccess) return e;
    }
    if (want_w) {  // dG^T X and dU^T X: the depth runs through the tokens
        for (int z = 0; z < 2; ++z) {
            p.A[z] = grads + z * half * 2;
            p.B[z] = ptr[0];
            p.ldb[z] = ld[0];
            p.b_bytes[z] = (M - 1) * ld[0] + (int64_t)K * 2;
        }
        p.a_bytes = M * row - half * 2;
        p.k_bytes = (int64_t)M * 2;
        p.part_steps = 0x7fffffff;
        p.C[0] = dWg.ptr;
        p.C[1] = dWu.ptr;
        p.ldc[0] = dWg.ld;
        p.ldc[1] = dWu.ld;
        p.M = N;
        p.N = K;
        p.batch = 2;
        if ((e = run_product<ET, false, ACROSS_K, ACROSS_K>(p, cw, ws, M, stream)) != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t quantize_rows(int type, int M, int K, Mat X, int8_t *Q, int64_t ldq, float *scale, hipStream_t stream) {
    hipError_t e;
    const dim3 grid((unsigned)(M < (1 << 20) ? M : 1 << 20)), block(256);
    if (type == OT_F32) e = launch_kernel(quantize_kernel<float>, grid, block, 0, stream, (const float *)X.ptr, X.ld, Q, ldq, scale, M, K);
    else if (type == OT_F16) e = launch_kernel(quantize_kernel<_Float16>, grid, block, 0, stream, (const _Float16 *)X.ptr, X.ld, Q, ldq, scale, M, K);
    else e = launch_kernel(quantize_kernel<__bf16>, grid, block, 0, stream, (const __bf16 *)X.ptr, X.ld, Q, ldq, scale, M, K);
    return launched("ffn_quantize_kernel", type == OT_F32 ? 's' : type == OT_F16 ? 'h' : 'b', 1, K, 256, M, 1, K, grid.x, 1, 1, e);
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
    if (type == OT_F16) return grad_of<ET_F16, OT_F16>(gate, M, N, K, dH, X, Wg, Wu, G, U, dX, dWg, dWu, stream);
    return grad_of<ET_BF16, OT_BF16>(gate, M, N, K, dH, X, Wg, Wu, G, U, dX, dWg, dWu, stream);
}

}  // namespace ffn
}  // namespace cba
