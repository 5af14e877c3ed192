// Gated linear block, both projections, the activation and the product in one kernel, with its backward pass:
//
//     g = x Wg^T + bg     u = x Wu^T + bu     y = act(g) * u            x [M][K], W [F][K] (the layout of a Linear's weight), y [M][F]
//
// The backward pass needs g and u once more, and writes what its products need,
//     dg = dy u act'(g)      du = dy act(g)        (one [M][2F] buffer, dg | du, in the inputs' type)
// In bf16 it forms g and u again tile by tile (rounded to bf16 they would cost the gradients a third of their precision, and in float32 their way
// through memory takes as long as the products: M 8192, K 1024, F 4096, 165 us against 150).  In float32, whose products run at a tenth of that
// rate, the forward pass keeps them (K >= 128; M 1999, K 1000, F 1365: 110 us of products against 22 of traffic).
// then  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x;  the bias gradients are column sums of the unrounded dg, du, per row tile into a
// slab that a last pass adds in order (no atomics: the same bits every time).
#include "gated_linear_tile.h"

namespace {

// both projections of TI rows x TJ/2 hidden units, and y, or dg and du
template <typename T, int TI, int TJ, bool BWD>
__global__ __launch_bounds__(256, 2) void gl_gate_kernel(GlArgs p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int G = TJ / 16, RP = 256 / G < TI ? 256 / G : TI;      // 8-column groups of a row, rows of a pass
    const long nt = (p.F + TJ / 2 - 1) / (TJ / 2), mt = (p.M + TI - 1) / TI;
    long row_tile, col_tile;
    gl_tile_at(blockIdx.x, mt, nt, row_tile, col_tile);
    const long m0 = row_tile * TI, f0 = col_tile * (TJ / 2);
    f32x4 acc[TI / 32][TJ / 32];
    const int chunks = (int)((p.K + GlNum<T>::BK - 1) / GlNum<T>::BK);
    gl_loop<T, TI, TJ, GL_KC, GL_DUAL>(lds, acc, p.x, m0, p.w, f0, p.K, chunks, 0, chunks);
    float* t = reinterpret_cast<float*>(lds);
    gl_dump<TI, TJ>(t, acc);
    const int cg = threadIdx.x % G, row0 = threadIdx.x / G;
    const int col = (cg >> 1) * 32 + (cg & 1) * 8;                    // of the gate; the up projection lies 16 columns on
    const long f = f0 + cg * 8, left = p.F - f;
    float bg[8], bu[8], sg[8], su[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        bg[e] = p.bg && e < left ? gl_ld((const T*)p.bg + f + e) : 0.f;
        bu[e] = p.bu && e < left ? gl_ld((const T*)p.bu + f + e) : 0.f;
        sg[e] = su[e] = 0.f;
    }
#pragma unroll
    for (int ps = 0; ps < TI / RP; ++ps) {
        const int row = row0 + ps * RP;
        const long m = m0 + row;
        if (m < p.M && left > 0 && (RP * G == 256 || row < TI)) {
            float g[8], u[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 tg = *reinterpret_cast<const f32x4*>(t + row * (TJ + 4) + col + 4 * h);
                const f32x4 tu = *reinterpret_cast<const f32x4*>(t + row * (TJ + 4) + col + 16 + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) { g[4 * h + e] = tg[e] + bg[4 * h + e]; u[4 * h + e] = tu[e] + bu[4 * h + e]; }
            }
            if constexpr (!BWD) {
                if (sizeof(T) == 4 && p.kept) {
                    gl_store8(p.kept + m * 2 * p.Fp + f, g, true, 8);
                    gl_store8(p.kept + m * 2 * p.Fp + p.Fp + f, u, true, 8);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float a, slope;
                    gl_act<sizeof(T) == 4>(g[e], p.act, a, slope);
                    g[e] = a * u[e];
                }
                gl_store8((T*)p.y + m * p.F + f, g, p.y_vec, left);
            } else {
                float d[8];
                gl_load8((const T*)p.dy + m * p.ldd + f, d, p.dy_vec, left);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float a, slope;
                    gl_act<sizeof(T) == 4>(g[e], p.act, a, slope);
                    g[e] = d[e] * u[e] * slope;
                    u[e] = d[e] * a;
                    sg[e] += g[e];
                    su[e] += u[e];
                }
                if (left < 8) {                               // the products read the columns up to Fp: 0, also where a row of x is infinite
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e >= left) g[e] = u[e] = 0.f;
                }
                gl_store8((T*)p.dgu + m * 2 * p.Fp + f, g, true, 8);
                gl_store8((T*)p.dgu + m * 2 * p.Fp + p.Fp + f, u, true, 8);
            }
        }
    }
    if (BWD && p.slab) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (RP * G == 256 || row0 < RP) {
                t[row0 * (TJ + 1) + cg * 8 + e] = sg[e];
                t[row0 * (TJ + 1) + TJ / 2 + cg * 8 + e] = su[e];
            }
        __syncthreads();
        if (threadIdx.x < TJ) {
            const int c = threadIdx.x % (TJ / 2), up = threadIdx.x / (TJ / 2);
            float sum = 0.f;
            for (int r = 0; r < RP; ++r) sum += t[r * (TJ + 1) + up * (TJ / 2) + c];
            if (f0 + c < p.F) p.slab[(m0 / TI) * 2 * p.F + up * p.F + f0 + c] = sum;
        }
    }
}

// dg | du from the kept g | u: 64 rows x 64 hidden units a workgroup, bound by its 5 float32 transfers an element
__global__ __launch_bounds__(256) void gl_slope_kernel(GlArgs p)
{
    __shared__ float sums[32][129];
    const long nt = (p.F + 63) / 64, m0 = blockIdx.x / nt * 64, f0 = blockIdx.x % nt * 64;
    const int cg = threadIdx.x & 7, row0 = threadIdx.x >> 3;
    const long f = f0 + cg * 8, left = p.F - f;
    float sg[8], su[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sg[e] = su[e] = 0.f;
#pragma unroll
    for (int ps = 0; ps < 2; ++ps) {
        const long m = m0 + row0 + 32 * ps;
        if (m < p.M && left > 0) {
            float g[8], u[8], d[8];
            gl_load8((const float*)p.kept + m * 2 * p.Fp + f, g, left >= 8, left);
            gl_load8((const float*)p.kept + m * 2 * p.Fp + p.Fp + f, u, left >= 8, left);
            gl_load8((const float*)p.dy + m * p.ldd + f, d, p.dy_vec, left);
#pragma unroll
            for (int e = 0; e < 8; ++e) {                             // (past F: all three are 0)
                float a, slope;
                gl_act<true>(g[e], p.act, a, slope);
                g[e] = d[e] * u[e] * slope;
                u[e] = d[e] * a;
                sg[e] += g[e];
                su[e] += u[e];
            }
            gl_store8((float*)p.dgu + m * 2 * p.Fp + f, g, true, 8);
            gl_store8((float*)p.dgu + m * 2 * p.Fp + p.Fp + f, u, true, 8);
        }
    }
    if (p.slab) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { sums[row0][cg * 8 + e] = sg[e]; sums[row0][64 + cg * 8 + e] = su[e]; }
        __syncthreads();
        if (threadIdx.x < 128) {
            const int c = threadIdx.x & 63, up = threadIdx.x >> 6;
            float sum = 0.f;
            for (int r = 0; r < 32; ++r) sum += sums[r][threadIdx.x];
            if (f0 + c < p.F) p.slab[m0 / 64 * 2 * p.F + up * p.F + f0 + c] = sum;
        }
    }
}

// Few rows (M <= 16 NM, one to NM tiles of 16): the weights' bytes are all that counts, so no tile of them goes through LDS.  A workgroup owns 16
// hidden units; its four waves take a quarter of k each and load the 16 gate rows and 16 up rows straight into fragments, four chunks of 128
// bytes in flight (16 loads of 16 bytes a lane), x being the other operand; their sums meet in LDS, in order.
// v_mfma 16 x 16: rows are hidden units, columns rows of x.
template <typename T, int NM>
__global__ __launch_bounds__(256) void gl_rows_kernel(GlArgs p)
{
    constexpr int BK = GlNum<T>::BK, E = GlNum<T>::E, IN = 4;
    __shared__ float red[4][2][NM][16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, kg = lane >> 4;
    const long f0 = 16L * blockIdx.x;
    const int chunks = (int)((p.K + BK - 1) / BK), per = (chunks + 3) / 4, c0 = wave * per, c1 = c0 + per < chunks ? c0 + per : chunks;
    const char* bases[3] = {(const char*)p.w.p[0] + f0 * p.w.ld[0] * (long)sizeof(T), (const char*)p.w.p[1] + f0 * p.w.ld[1] * (long)sizeof(T), (const char*)p.x.p[0]};
    __amdgpu_buffer_rsrc_t rs[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) rs[q] = __builtin_amdgcn_make_buffer_rsrc((void*)bases[q], 0, 0x7fffffff, 0x00020000);
    unsigned off[2 + NM];
#pragma unroll
    for (int q = 0; q < 2; ++q) off[q] = f0 + l16 < p.F ? (unsigned)l16 * (unsigned)(p.w.ld[q] * (long)sizeof(T)) + 16u * kg : GL_NONE;
#pragma unroll
    for (int n = 0; n < NM; ++n) off[2 + n] = 16 * n + l16 < p.M ? (unsigned)(16 * n + l16) * (unsigned)(p.x.ld[0] * (long)sizeof(T)) + 16u * kg : GL_NONE;
    f32x4 acc[2][NM];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int n = 0; n < NM; ++n) acc[w][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c = c0; c < c1; c += IN) {
        gl_u32x4 r[IN][2][2 + NM];
#pragma unroll
        for (int d = 0; d < IN; ++d)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bool on = c + d < c1 && (c + d) * BK + (4 * j + kg) * E < p.K;
#pragma unroll
                for (int q = 0; q < 2 + NM; ++q)
                    r[d][j][q] = __builtin_amdgcn_raw_buffer_load_b128(rs[q < 2 ? q : 2], on ? off[q] : GL_NONE, (unsigned)(c + d) * 128u + 64u * j, 0);
            }
#pragma unroll
        for (int d = 0; d < IN; ++d)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int n = 0; n < NM; ++n)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const gl_u32x4 a[1] = {r[d][j][w]}, b[1] = {r[d][j][2 + n]};
                        f32x4 one[1][1] = {{acc[w][n]}};
#pragma unroll
                        for (int m = 0; m < gl_products_of<T, 1, 1>(); ++m) gl_mma<T, 1, 1>(a, b, one, m);
                        acc[w][n] = one[0][0];
                    }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int n = 0; n < NM; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) red[wave][w][n][l16][4 * kg + q] = acc[w][n][q];
    __syncthreads();
    const int f = threadIdx.x & 15;
#pragma unroll
    for (int n = 0; n < NM; ++n) {
        const int row = threadIdx.x >> 4;
        const long m = 16 * n + row;
        if (m >= p.M || f0 + f >= p.F) continue;
        float g = p.bg ? gl_ld((const T*)p.bg + f0 + f) : 0.f, u = p.bu ? gl_ld((const T*)p.bu + f0 + f) : 0.f, a, slope;
#pragma unroll
        for (int w = 0; w < 4; ++w) { g += red[w][0][n][row][f]; u += red[w][1][n][row][f]; }
        if (sizeof(T) == 4 && p.kept) {
            p.kept[m * 2 * p.Fp + f0 + f] = g;
            p.kept[m * 2 * p.Fp + p.Fp + f0 + f] = u;
        }
        gl_act<sizeof(T) == 4>(g, p.act, a, slope);
        const float y[1] = {a * u};
        seq_store<1>((T*)p.y + m * p.F + f0 + f, y);
    }
}

template <typename T, int TI, int TJ>
__global__ __launch_bounds__(256, 2) void gl_product_kernel(GlJobs all)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int G = TJ / 8, RP = 256 / G;
    int q = 0;
    if (all.n > 1 && (int)blockIdx.x >= all.j[1].first) q = 1;
    if (all.n > 2 && (int)blockIdx.x >= all.j[2].first) q = 2;
    const GlJob& p = all.j[q];
    const long idx = gl_tile_of((long)blockIdx.x - p.first, p.tiles * p.splits);
    const long split = idx / p.tiles, tile = idx % p.tiles;
    const long i0 = tile / p.tj * TI, j0 = tile % p.tj * TJ;
    const int c0 = (int)split * p.run, c1 = c0 + p.run < p.chunks ? c0 + p.run : p.chunks;
    f32x4 acc[TI / 32][TJ / 32];
    if (p.a_kr) gl_loop<T, TI, TJ, GL_KR, GL_KR>(lds, acc, p.a, i0, p.b, j0, p.K, p.per, c0, c1);
    else gl_loop<T, TI, TJ, GL_KC, GL_KR>(lds, acc, p.a, i0, p.b, j0, p.K, p.per, c0, c1);
    float* t = reinterpret_cast<float*>(lds);
    gl_dump<TI, TJ>(t, acc);
    const int cg = threadIdx.x % G;
    const long j = j0 + cg * 8, left = p.J - j;
    if (left <= 0) return;
    const bool vec = p.J % 8 == 0;                                    // (outputs start on 16 bytes: checked by the host)
    for (int row = threadIdx.x / G; row < TI; row += RP) {
        const long i = i0 + row;
        if (i >= p.I) break;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = t[row * (TJ + 4) + cg * 8 + e];
        if (p.splits > 1) gl_store8(p.part + (split * p.I + i) * p.J + j, x, vec, left);
        else gl_store8((T*)p.out + i * p.J + j, x, vec, left);
    }
}

// What is left of the backward pass, one launch: the runs of the split products added up, and the row tiles' column sums of dg | du (the last
// plane of the grid).  64 results a workgroup; its four waves take every fourth summand each (in order, eight loads in flight), and their four
// sums are added in order.
struct GlFinish {
    const float* part[4];     // [n][count]
    long n[4], count[4];      // summands, results
    void* out[4];
    void* up;                 // the column sums' second half
};
template <typename T>
__global__ __launch_bounds__(256) void gl_finish_kernel(GlFinish p, int bias)
{
    __shared__ float part[4][64];
    const int q = blockIdx.y, w = threadIdx.x >> 6;
    const long count = p.count[q], e = (long)blockIdx.x * 64 + (threadIdx.x & 63);
    if ((long)blockIdx.x * 64 >= count) return;
    float s = 0.f;
    if (e < count)
#pragma unroll 8
        for (long k = w; k < p.n[q]; k += 4) s += p.part[q][k * count + e];
    part[w][threadIdx.x & 63] = s;
    __syncthreads();
    if (w == 0 && e < count) {
        const float x[1] = {part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x]};
        T* out = (T*)p.out[q];
        long at = e;
        if (q == bias && e >= count / 2) { out = (T*)p.up; at = e - count / 2; }
        if (out) seq_store<1>(out + at, x);
    }
}

// rows copied to rows of whole 16-byte units, 0 behind K: operands whose rows do not start on 16 bytes
struct GlPack {
    const void* src[3];
    long ld[3], rows[3];
    void* dst[3];
    long K, Kp;
    int n;
};
template <typename T>
__global__ __launch_bounds__(256) void gl_pack_kernel(GlPack p)
{
    for (int q = 0; q < p.n; ++q) {
        const long units = p.Kp / 8, all = p.rows[q] * units;
        for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < all; e += (long)gridDim.x * 256) {
            const long row = e / units, k = (e - row * units) * 8;
            float x[8];
            gl_load8((const T*)p.src[q] + row * p.ld[q] + k, x, false, p.K - k);
            gl_store8((T*)p.dst[q] + row * p.Kp + k, x, true, 8);
        }
    }
}

constexpr long GL_WIDE = 1L << 20;     // widest K and F: 256 rows of dg | du lie within 32-bit offsets
int gl_check(int64_t M, int64_t K, int64_t F, int dtype, int act)
{
    HN_REQUIRE(M >= 0 && K >= 0 && F >= 0 && M < (1L << 31) && K < GL_WIDE && F < GL_WIDE, "hn_gated_linear: bad sizes M=%ld K=%ld F=%ld", (long)M, (long)K,
               (long)F);
    HN_REQUIRE(dtype == SEQ_F32 || dtype == SEQ_BF16, "hn_gated_linear: dtype is 0 (float32) or 1 (bf16)");
    HN_REQUIRE(act >= GL_SILU && act <= GL_RELU, "hn_gated_linear: activation is 0 (silu), 1 (gelu), 2 (sigmoid) or 3 (relu)");
    return 0;
}

size_t gl_round(size_t n) { return (n + 255) & ~(size_t)255; }
long gl_up8(long n) { return (n + 7) & ~7L; }

struct GlIn {
    const void *x, *wg, *wu;
    long ldx, ldg, ldu, M, K, F;
    int size;             // bytes of an element
};
// whether the tiles may read a matrix where it lies: rows of whole 16-byte units, 256 of them within 32-bit offsets
bool gl_aligned(const GlIn& in, const void* p, long ld)
{
    return (size_t)p % 16 == 0 && ld * in.size % 16 == 0 && in.K * in.size % 16 == 0 && ld * in.size < (1L << 23);
}

// workspace in order: x and w in whole units where they are not, dgu, column sums, partial products
struct GlPlan {
    int gate, prod;                                   // shapes
    size_t x, wg, wu, dgu, slab, part[3], bytes;      // offsets; 0-size parts share one
    bool pack_x, pack_g, pack_u, pp_gate, pp_prod;
    int splits[3], run[3];
};
long gl_tiles(long I, long J, int ti, int tj) { return ((I + ti - 1) / ti) * ((J + tj - 1) / tj); }

// 0 64 x 64, 1 128 x 64, 2 128 x 128 (bf16 alone), 3 64 x 32, 4 32 x 32 (float32 alone)
int gl_shape_i(int shape) { return shape == 4 ? 32 : shape == 0 || shape == 3 ? 64 : 128; }
int gl_shape_j(int shape) { return shape == 2 ? 128 : shape >= 3 ? 32 : 64; }
// The gate's tile shape: the one that leaves the fullest of 256 compute units the least to do -- its tiles, times a tile's size, times what a
// shape costs beyond its size.
//   bf16     feels the small tile's operand reads (M 2048, K 1024, F 4096: 77 / 50 / 49 us in the order of the shapes; M 512, K 1024, F 2048: 13.8 /
//            12.2 / 16.5; M 256, K 512, F 1024: 6.0 / 8.2 / 11.4, and 5.8 by 64 x 32)
//   float32  is bound by its products, whose time goes with a unit's tiles alone: the small ones where the larger leave units empty, in the first
//            round or the last (32 x 32 / 64 x 32 / 64 x 64: M 256, K 512, F 512: 7.7 / 9.7 / 13.6; M 512, K 1024, F 1365: 31.9 / 30.8 / 38.2; M 2048,
//            K 1024, F 4096: 300 / 273 / 266, and 255 by 128 x 64), 128 x 64 where it gives two tiles a unit, which hide each other's waits
int gl_gate_shape(int size, long M, long F)
{
    static const struct { int shape; double cost; } bf16[3] = {{0, 1.6}, {1, 2.5}, {2, 4.0}}, f32[4] = {{4, 0.28}, {3, 0.525}, {0, 1.0}, {1, 2.0}};
    int best = 0;
    double least = 0;
    for (int q = 0; q < (size == 2 ? 3 : 4); ++q) {
        const int shape = size == 2 ? bf16[q].shape : f32[q].shape;
        const long tiles = gl_tiles(M, F, gl_shape_i(shape), gl_shape_j(shape) / 2);
        if (size == 4 && shape == 1 && tiles < 512) break;                    // (M 1000, K 512, F 1000: 21.6 by 64 x 64 against 23.7)
        const double cost = (double)((tiles + 255) / 256) * (size == 2 ? bf16[q].cost : f32[q].cost);
        if (q == 0 || cost <= least) { best = shape; least = cost; }
    }
    return best;
}
// The products' shape: 128 x 128 in bf16 where that gives at least 320 tiles (M 16384, K 256, F 2048: products 134 us against 155; below, 64 x 64
// fills the device better: M 2000, K 1024, F 1365: 49 against 54), else 64 x 64 (float32, M 1999, K 1000, F 1365: 205 against 222)
int gl_product_shape(int size, long M, long K, long F) { return size == 2 && gl_tiles(M, K, 128, 128) + 2 * gl_tiles(F, K, 128, 128) >= 320 ? 2 : 0; }

GlPlan gl_plan(const GlIn& in, bool backward)
{
    GlPlan p = {};
    const long bk = 128 / in.size, M = in.M, K = in.K, F = in.F;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += gl_round(n); return o; };
    p.pack_x = K > 0 && !gl_aligned(in, in.x, in.ldx);
    p.pack_g = K > 0 && !gl_aligned(in, in.wg, in.ldg);
    p.pack_u = K > 0 && !gl_aligned(in, in.wu, in.ldu);
    p.x = take(p.pack_x ? (size_t)M * gl_up8(K) * in.size : 0);
    p.wg = take(p.pack_g ? (size_t)F * gl_up8(K) * in.size : 0);
    p.wu = take(p.pack_u ? (size_t)F * gl_up8(K) * in.size : 0);
    // the ping-pong tiles where they fill three quarters of the device (M 8192, K 256, F 1024, 256 tiles: 15.8 us against 21.5; M 2000, K 1024,
    // F 1365, 88 tiles: 38 against 25)
    const long ldg = p.pack_g ? gl_up8(K) : in.ldg, ldu = p.pack_u ? gl_up8(K) : in.ldu;
    const bool pp = in.size == 2;
    p.pp_gate = pp && K >= 128 && gl_tiles(M, F, 256, 128) >= 192;
    p.gate = gl_gate_shape(in.size, M, F);
    if (backward) {
        p.dgu = take((size_t)M * 2 * gl_up8(F) * in.size);
        p.slab = take((size_t)((M + 31) / 32) * 2 * F * 4);
        const long I[3] = {M, F, F}, chunks[3] = {2 * ((F + bk - 1) / bk), (M + bk - 1) / bk, (M + bk - 1) / bk};
        // the products' ping-pong tiles go out one a compute unit, 2.0 us a chunk: worth it where the longest tile, or all of them over 256
        // units, end before the smaller tiles would at 600 TFLOP/s (M 8192, K 1024, F 4096: 264 us against 412; M 4096, K 1024, F 2048: 115 against 103)
        const long cx = 2 * ((F + 63) / 64), cw = (M + 63) / 64, work = gl_tiles(M, K, 256, 256) * cx + 2 * gl_tiles(F, K, 256, 256) * cw;
        const double longest = (double)(cx > cw ? cx : cw), mean = (double)work / 256;
        p.pp_prod = pp && ldg == ldu && M >= 128 && F >= 64 && 2.0 * (longest > mean ? longest : mean) < 8.0 * M * K * F / 600e6;
        p.prod = gl_product_shape(in.size, M, K, F);
        long all = 0, tiles[3];
        for (int q = 0; q < 3; ++q) {
            tiles[q] = gl_tiles(I[q], K, gl_shape_i(p.prod), gl_shape_j(p.prod));
            all += tiles[q] * chunks[q];
        }
        // a product whose k axis is longer than its share is cut into runs of about the same number of chunks for all: a 256th of the chunks, in
        // float32, where two workgroups on a unit hide each other's waits, a 512th, and 4 at least (products of M 512, K 512, F 1024 with the rest of the
        // backward pass: float32 34.3 us by 512, 40.8 by 256; bf16 22.0 by 256, 31.3 by 256 workgroups for each product by itself)
        const long units = in.size == 2 ? 256 : 512, even = all / units > 4 ? all / units : 4;
        for (int q = 0; q < 3; ++q) {
            long s = (2 * chunks[q] + even) / (2 * even);
            if (s < 1 || p.pp_prod) s = 1;
            p.run[q] = (int)((chunks[q] + s - 1) / s);
            if (p.run[q] < 1) p.run[q] = 1;
            p.splits[q] = (int)((chunks[q] + p.run[q] - 1) / p.run[q]);
            if (p.splits[q] < 1) p.splits[q] = 1;
            p.part[q] = take(p.splits[q] > 1 ? (size_t)p.splits[q] * I[q] * K * 4 : 0);
        }
    }
    p.bytes = at;
    return p;
}

template <typename T>
int gl_prepare(const GlIn& in, const GlPlan& pl, char* ws, GlOpd& x, GlOpd& w, hipStream_t s)
{
    const long Kp = gl_up8(in.K);
    GlPack pk = {};
    pk.K = in.K; pk.Kp = Kp;
    x = GlOpd{{in.x, in.x}, {in.ldx, in.ldx}, in.M};
    w = GlOpd{{in.wg, in.wu}, {in.ldg, in.ldu}, in.F};
    auto add = [&](const void*& p, long& ld, long rows, size_t at) {
        pk.src[pk.n] = p; pk.ld[pk.n] = ld; pk.rows[pk.n] = rows; pk.dst[pk.n] = ws + at;
        p = ws + at;
        ld = Kp;
        ++pk.n;
    };
    if (pl.pack_x) { add(x.p[0], x.ld[0], in.M, pl.x); x.p[1] = x.p[0]; x.ld[1] = x.ld[0]; }
    if (pl.pack_g) add(w.p[0], w.ld[0], in.F, pl.wg);
    if (pl.pack_u) add(w.p[1], w.ld[1], in.F, pl.wu);
    if (pk.n) {
        long most = 0;
        for (int q = 0; q < pk.n; ++q) most = pk.rows[q] * (Kp / 8) > most ? pk.rows[q] * (Kp / 8) : most;
        long g = (most + 255) / 256;
        if (g > 2048) g = 2048;
        hipLaunchKernelGGL((gl_pack_kernel<T>), dim3((unsigned)(g < 1 ? 1 : g)), dim3(256), 0, s, pk);
        HN_LAUNCH_CHECK();
    }
    return 0;
}

// a kernel that takes more than 64 KiB of LDS has to say so, once per device
int gl_big_lds(const void* kern, int bytes, bool (&told)[64])
{
    if (bytes <= 65536) return 0;
    int dev = 0;
    HN_HIP(hipGetDevice(&dev));
    if (dev >= 0 && dev < 64 && told[dev]) return 0;
    HN_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev >= 0 && dev < 64) told[dev] = true;
    return 0;
}

template <typename T, int TI, int TJ, bool BWD>
int gl_gate_run(const GlArgs& p, hipStream_t s)
{
    const long n = gl_tiles(p.M, p.F, TI, TJ / 2);
    SEQ_REQUIRE_GRID(n, 256, "hn_gated_linear");
    static bool told[64] = {};
    if (const int rc = gl_big_lds(reinterpret_cast<const void*>(gl_gate_kernel<T, TI, TJ, BWD>), gl_lds_bytes<TI, TJ>(), told)) return rc;
    hipLaunchKernelGGL((gl_gate_kernel<T, TI, TJ, BWD>), dim3((unsigned)n), dim3(256), (gl_lds_bytes<TI, TJ>()), s, p);
    HN_LAUNCH_CHECK();
    return 0;
}

template <typename T, bool BWD>
int gl_gate(int shape, const GlArgs& p, hipStream_t s)
{
    if constexpr (sizeof(T) == 2)
        if (shape == 2) return gl_gate_run<T, 128, 128, BWD>(p, s);
    if constexpr (sizeof(T) == 4) {
        if (shape == 3) return gl_gate_run<T, 64, 32, BWD>(p, s);
        if (shape == 4) return gl_gate_run<T, 32, 32, BWD>(p, s);
    }
    return shape == 0 ? gl_gate_run<T, 64, 64, BWD>(p, s) : gl_gate_run<T, 128, 64, BWD>(p, s);
}

template <typename T, int TI, int TJ>
int gl_products_run(GlJobs& jobs, hipStream_t s)
{
    long n = 0;
    for (int q = 0; q < jobs.n; ++q) {
        GlJob& j = jobs.j[q];
        j.tj = (j.J + TJ - 1) / TJ;
        j.tiles = gl_tiles(j.I, j.J, TI, TJ);
        j.first = (int)n;
        n += j.tiles * j.splits;
        SEQ_REQUIRE_GRID(n, 256, "hn_gated_linear_bwd");
    }
    if (n == 0) return 0;
    static bool told[64] = {};
    if (const int rc = gl_big_lds(reinterpret_cast<const void*>(gl_product_kernel<T, TI, TJ>), gl_lds_bytes<TI, TJ>(), told)) return rc;
    hipLaunchKernelGGL((gl_product_kernel<T, TI, TJ>), dim3((unsigned)n), dim3(256), (gl_lds_bytes<TI, TJ>()), s, jobs);
    HN_LAUNCH_CHECK();
    return 0;
}

template <typename T>
int gl_products(int shape, GlJobs& jobs, hipStream_t s)
{
    if constexpr (sizeof(T) == 2)
        if (shape == 2) return gl_products_run<T, 128, 128>(jobs, s);
    return gl_products_run<T, 64, 64>(jobs, s);
}

template <typename T>
int gl_forward(const GlIn& in, GlArgs p, char* ws, hipStream_t s)
{
    const GlPlan pl = gl_plan(in, false);
    if (const int rc = gl_prepare<T>(in, pl, ws, p.x, p.w, s)) return rc;
    if (in.M <= 32) {                 // (K 1024, F 4096, bf16 / float32: M 1 5.7 us against 10.6 / 10.5 against 23.0, M 32 7.9 / 10.7 and 15.6 / 23.2)
        const dim3 grid((unsigned)((in.F + 15) / 16));
        if (in.M <= 16) hipLaunchKernelGGL((gl_rows_kernel<T, 1>), grid, dim3(256), 0, s, p);
        else hipLaunchKernelGGL((gl_rows_kernel<T, 2>), grid, dim3(256), 0, s, p);
        HN_LAUNCH_CHECK();
        return 0;
    }
    if (pl.pp_gate) return hn_launch_gated_linear_pp_gate(p, false, s);
    return gl_gate<T, false>(pl.gate, p, s);
}

template <typename T>
int gl_backward(const GlIn& in, GlArgs p, char* ws, void* dx, void* dwg, void* dwu, void* dbg, void* dbu, hipStream_t s)
{
    const GlPlan pl = gl_plan(in, true);
    const long bk = GlNum<T>::BK, Fp = p.Fp;
    const int rows = p.kept ? 64 : pl.pp_gate ? 128 : gl_shape_i(pl.gate);                 // of a column-sum tile
    if (const int rc = gl_prepare<T>(in, pl, ws, p.x, p.w, s)) return rc;
    p.dgu = ws + pl.dgu;
    p.slab = dbg || dbu ? (float*)(ws + pl.slab) : nullptr;
    if (in.M > 0 && in.F > 0 && p.kept) {
        const long n = gl_tiles(in.M, in.F, 64, 64);
        SEQ_REQUIRE_GRID(n, 256, "hn_gated_linear_bwd");
        hipLaunchKernelGGL(gl_slope_kernel, dim3((unsigned)n), dim3(256), 0, s, p);
        HN_LAUNCH_CHECK();
    } else if (in.M > 0 && in.F > 0)
        if (const int rc = pl.pp_gate ? hn_launch_gated_linear_pp_gate(p, true, s) : gl_gate<T, true>(pl.gate, p, s)) return rc;
    GlJobs jobs = {};
    void* outs[3] = {dx, dwg, dwu};
    for (int q = 0; q < 3; ++q) {
        if (!outs[q] || in.K == 0 || (q == 0 ? in.M : in.F) == 0) continue;
        GlJob& j = jobs.j[jobs.n++];
        const T* dgu = (const T*)p.dgu;
        if (q == 0) {
            j.a = GlOpd{{dgu, dgu + Fp}, {2 * Fp, 2 * Fp}, in.M};
            j.b = GlOpd{{p.w.p[0], p.w.p[1]}, {p.w.ld[0], p.w.ld[1]}, in.K};
            j.I = in.M; j.K = in.F;
            j.per = (int)((in.F + bk - 1) / bk);
            j.chunks = 2 * j.per;
        } else {
            j.a = GlOpd{{q == 1 ? dgu : dgu + Fp, nullptr}, {2 * Fp, 0}, in.F};
            j.b = GlOpd{{p.x.p[0], nullptr}, {p.x.ld[0], 0}, in.K};
            j.I = in.F; j.K = in.M;
            j.per = j.chunks = (int)((in.M + bk - 1) / bk);
            j.a_kr = 1;
        }
        j.J = in.K;
        j.out = outs[q];
        j.splits = pl.splits[q]; j.run = pl.run[q];
        j.part = (float*)(ws + pl.part[q]);
    }
    if (const int rc = pl.pp_prod ? hn_launch_gated_linear_pp_products(jobs, s) : gl_products<T>(pl.prod, jobs, s)) return rc;
    GlFinish fin = {};
    int planes = 0, bias = -1;
    long most = 0;
    auto add = [&](const float* part, long n, long count, void* out) {
        fin.part[planes] = part; fin.n[planes] = n; fin.count[planes] = count; fin.out[planes] = out;
        most = count > most ? count : most;
        return planes++;
    };
    for (int q = 0; q < jobs.n; ++q)
        if (jobs.j[q].splits > 1) add(jobs.j[q].part, jobs.j[q].splits, jobs.j[q].I * jobs.j[q].J, jobs.j[q].out);
    if ((dbg || dbu) && in.F > 0) {
        bias = add(p.slab, (in.M + rows - 1) / rows, 2 * in.F, dbg);
        fin.up = dbu;
    }
    if (planes) {
        SEQ_REQUIRE_GRID((most + 63) / 64, 256, "hn_gated_linear_bwd");
        hipLaunchKernelGGL((gl_finish_kernel<T>), dim3((unsigned)((most + 63) / 64), planes), dim3(256), 0, s, fin, bias);
    }
    HN_LAUNCH_CHECK();
    return 0;
}

GlIn gl_in(const void* x, int64_t ldx, const void* wg, int64_t ldg, const void* wu, int64_t ldu, int64_t M, int64_t K, int64_t F, int dtype)
{
    return GlIn{x, wg, wu, ldx, ldg, ldu, M, K, F, dtype == SEQ_F32 ? 4 : 2};
}

}  // namespace

extern "C" size_t hn_gated_linear_workspace(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up, int64_t M,
                                            int64_t K, int64_t F, int dtype, int backward)
{
    if (M < 0 || K < 0 || F < 0 || M >= (1L << 31) || K >= GL_WIDE || F >= GL_WIDE || (dtype != SEQ_F32 && dtype != SEQ_BF16)) return 0;
    return gl_plan(gl_in(x, ldx, w_gate, ld_gate, w_up, ld_up, M, K, F, dtype), backward != 0).bytes;
}

extern "C" size_t hn_gated_linear_kept(int64_t M, int64_t K, int64_t F, int dtype)
{
    return dtype == SEQ_F32 && K >= 128 && K < GL_WIDE && M > 0 && F > 0 && M < (1L << 31) && F < GL_WIDE ? (size_t)M * 2 * gl_up8(F) : 0;
}

extern "C" int hn_gated_linear(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up, const void* b_gate,
                               const void* b_up, void* y, float* kept, void* workspace, size_t workspace_bytes, int64_t M, int64_t K, int64_t F,
                               int dtype, int act, void* stream)
{
    if (const int rc = gl_check(M, K, F, dtype, act)) return rc;
    if (M == 0 || F == 0) return 0;
    HN_REQUIRE(y && (K == 0 || (x && w_gate && w_up)), "hn_gated_linear: null pointer");
    HN_REQUIRE(ldx >= 0 && ld_gate >= 0 && ld_up >= 0, "hn_gated_linear: negative row stride");
    const GlIn in = gl_in(x, ldx, w_gate, ld_gate, w_up, ld_up, M, K, F, dtype);
    HN_REQUIRE(workspace_bytes >= gl_plan(in, false).bytes && (workspace || workspace_bytes == 0) && (size_t)workspace % 16 == 0,
               "hn_gated_linear: workspace too small or not aligned to 16 bytes");
    GlArgs p = {};
    HN_REQUIRE(!kept || (hn_gated_linear_kept(M, K, F, dtype) && (size_t)kept % 16 == 0), "hn_gated_linear: kept is null where hn_gated_linear_kept is 0, else on 16 bytes");
    p.bg = b_gate; p.bu = b_up; p.y = y; p.kept = kept;
    p.M = M; p.K = K; p.F = F; p.Fp = gl_up8(F); p.act = act;
    p.y_vec = (size_t)y % 16 == 0 && F * in.size % 16 == 0;
    return dtype == SEQ_BF16 ? gl_forward<seq_bf16>(in, p, (char*)workspace, (hipStream_t)stream) : gl_forward<float>(in, p, (char*)workspace, (hipStream_t)stream);
}

extern "C" int hn_gated_linear_bwd(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up, const void* b_gate,
                                   const void* b_up, const void* dy, int64_t ld_dy, const float* kept, void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up,
                                   void* workspace, size_t workspace_bytes, int64_t M, int64_t K, int64_t F, int dtype, int act, void* stream)
{
    if (const int rc = gl_check(M, K, F, dtype, act)) return rc;
    HN_REQUIRE(M == 0 || F == 0 || (dy && (K == 0 || (x && w_gate && w_up))), "hn_gated_linear_bwd: null pointer");
    HN_REQUIRE(ldx >= 0 && ld_gate >= 0 && ld_up >= 0 && ld_dy >= 0, "hn_gated_linear_bwd: negative row stride");
    const GlIn in = gl_in(x, ldx, w_gate, ld_gate, w_up, ld_up, M, K, F, dtype);
    HN_REQUIRE(workspace_bytes >= gl_plan(in, true).bytes && (workspace || workspace_bytes == 0) && (size_t)workspace % 16 == 0,
               "hn_gated_linear_bwd: workspace too small or not aligned to 16 bytes");
    HN_REQUIRE((size_t)dx % 16 == 0 && (size_t)dw_gate % 16 == 0 && (size_t)dw_up % 16 == 0, "hn_gated_linear_bwd: dx, dw_gate and dw_up start on 16 bytes");
    GlArgs p = {};
    HN_REQUIRE(!kept || (hn_gated_linear_kept(M, K, F, dtype) && (size_t)kept % 16 == 0), "hn_gated_linear_bwd: kept is null where hn_gated_linear_kept is 0, else on 16 bytes");
    p.bg = b_gate; p.bu = b_up; p.dy = dy; p.ldd = ld_dy; p.kept = const_cast<float*>(kept);
    p.M = M; p.K = K; p.F = F; p.Fp = gl_up8(F); p.act = act;
    p.dy_vec = (size_t)dy % 16 == 0 && ld_dy * in.size % 16 == 0;
    return dtype == SEQ_BF16 ? gl_backward<seq_bf16>(in, p, (char*)workspace, dx, dw_gate, dw_up, db_gate, db_up, (hipStream_t)stream)
                             : gl_backward<float>(in, p, (char*)workspace, dx, dw_gate, dw_up, db_gate, db_up, (hipStream_t)stream);
}
