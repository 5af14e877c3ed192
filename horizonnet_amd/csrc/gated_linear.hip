// Gated linear block, both projections, the activation and the product in one kernel, with its backward pass:
//
//     g = x Wg^T + bg     u = x Wu^T + bu     y = act(g) * u            x [M][K], W [F][K] (the layout of a Linear's weight), y [M][F]
//
// g and u are never stored.  The backward pass forms them again tile by tile and writes what the products need,
//     dg = dy u act'(g)      du = dy act(g)        (one [M][2F] buffer, dg | du, in the inputs' type)
// then  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x;  the bias gradients are column sums of the unrounded dg, du, per row tile into a
// slab that a last pass adds in order (no atomics: the same bits every time).
#include "gated_linear_tile.h"

namespace {

// both projections of TS rows x TS/2 hidden units, and y, or dg and du
template <typename T, int TS, bool BWD>
__global__ __launch_bounds__(256) void gl_gate_kernel(GlArgs p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int N = TS / 32, G = TS / 16, RP = 256 / G;             // 8-column groups of a row, rows of a pass
    const long nt = (p.F + TS / 2 - 1) / (TS / 2), mt = (p.M + TS - 1) / TS;
    const long tile = gl_tile_of(blockIdx.x, nt * mt);
    const long m0 = tile / nt * TS, f0 = tile % nt * (TS / 2);
    f32x4 acc[N][N];
    const int chunks = (int)((p.K + GlNum<T>::BK - 1) / GlNum<T>::BK);
    gl_loop<T, TS, GL_KC, GL_DUAL>(lds, acc, p.x, m0, p.w, f0, p.K, chunks, 0, chunks);
    float* t = reinterpret_cast<float*>(lds);
    gl_dump<TS>(t, acc);
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
    for (int ps = 0; ps < TS / RP; ++ps) {
        const int row = row0 + ps * RP;
        const long m = m0 + row;
        if (m < p.M && left > 0) {
            float g[8], u[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 tg = *reinterpret_cast<const f32x4*>(t + row * (TS + 4) + col + 4 * h);
                const f32x4 tu = *reinterpret_cast<const f32x4*>(t + row * (TS + 4) + col + 16 + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) { g[4 * h + e] = tg[e] + bg[4 * h + e]; u[4 * h + e] = tu[e] + bu[4 * h + e]; }
            }
            if constexpr (!BWD) {
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
                    g[e] = d[e] * u[e] * slope;                       // (0 in the columns up to Fp, which the products read: d is)
                    u[e] = d[e] * a;
                    sg[e] += g[e];
                    su[e] += u[e];
                }
                gl_store8((T*)p.dgu + m * 2 * p.Fp + f, g, true, 8);
                gl_store8((T*)p.dgu + m * 2 * p.Fp + p.Fp + f, u, true, 8);
            }
        }
    }
    if (BWD && p.slab) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            t[row0 * (TS + 1) + cg * 8 + e] = sg[e];
            t[row0 * (TS + 1) + TS / 2 + cg * 8 + e] = su[e];
        }
        __syncthreads();
        if (threadIdx.x < TS) {
            const int c = threadIdx.x % (TS / 2), up = threadIdx.x / (TS / 2);
            float sum = 0.f;
            for (int r = 0; r < RP; ++r) sum += t[r * (TS + 1) + up * (TS / 2) + c];
            if (f0 + c < p.F) p.slab[(m0 / TS) * 2 * p.F + up * p.F + f0 + c] = sum;
        }
    }
}

template <typename T, int TS>
__global__ __launch_bounds__(256) void gl_product_kernel(GlJobs all)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int N = TS / 32, G = TS / 8, RP = 256 / G;
    int q = 0;
    if (all.n > 1 && (int)blockIdx.x >= all.j[1].first) q = 1;
    if (all.n > 2 && (int)blockIdx.x >= all.j[2].first) q = 2;
    const GlJob& p = all.j[q];
    const long idx = gl_tile_of((long)blockIdx.x - p.first, p.tiles * p.splits);
    const long split = idx / p.tiles, tile = idx % p.tiles;
    const long i0 = tile / p.tj * TS, j0 = tile % p.tj * TS;
    const int c0 = (int)split * p.run, c1 = c0 + p.run < p.chunks ? c0 + p.run : p.chunks;
    f32x4 acc[N][N];
    if (p.a_kr) gl_loop<T, TS, GL_KR, GL_KR>(lds, acc, p.a, i0, p.b, j0, p.K, p.per, c0, c1);
    else gl_loop<T, TS, GL_KC, GL_KR>(lds, acc, p.a, i0, p.b, j0, p.K, p.per, c0, c1);
    float* t = reinterpret_cast<float*>(lds);
    gl_dump<TS>(t, acc);
    const int cg = threadIdx.x % G;
    const long j = j0 + cg * 8, left = p.J - j;
    if (left <= 0) return;
    const bool vec = p.J % 8 == 0;                                    // (outputs start on 16 bytes: checked by the host)
    for (int row = threadIdx.x / G; row < TS; row += RP) {
        const long i = i0 + row;
        if (i >= p.I) break;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = t[row * (TS + 4) + cg * 8 + e];
        if (p.splits > 1) gl_store8(p.part + (split * p.I + i) * p.J + j, x, vec, left);
        else gl_store8((T*)p.out + i * p.J + j, x, vec, left);
    }
}

// the runs of the split products added in order
template <typename T>
__global__ __launch_bounds__(256) void gl_join_kernel(GlJobs all)
{
    for (int q = 0; q < all.n; ++q) {
        const GlJob& p = all.j[q];
        if (p.splits <= 1) continue;
        const long n = p.I * p.J;
        for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long)gridDim.x * 256) {
            float s[1] = {0.f};
            for (int k = 0; k < p.splits; ++k) s[0] += p.part[k * n + e];
            seq_store<1>((T*)p.out + e, s);
        }
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

template <typename T>
__global__ __launch_bounds__(256) void gl_bias_kernel(const float* slab, long tiles, long F, T* dbg, T* dbu)
{
    const long c = (long)blockIdx.x * 256 + threadIdx.x;
    if (c >= 2 * F) return;
    float s[1] = {0.f};
    for (long t = 0; t < tiles; ++t) s[0] += slab[t * 2 * F + c];
    if (c < F) { if (dbg) seq_store<1>(dbg + c, s); }
    else if (dbu) seq_store<1>(dbu + c - F, s);
}

int gl_check(int64_t M, int64_t K, int64_t F, int dtype, int act)
{
    HN_REQUIRE(M >= 0 && K >= 0 && F >= 0 && M < (1L << 31) && K < (1L << 24) && F < (1L << 24), "hn_gated_linear: bad sizes M=%ld K=%ld F=%ld", (long)M, (long)K,
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
// whether the tiles may read a matrix where it lies: rows of whole 16-byte units
bool gl_aligned(const GlIn& in, const void* p, long ld) { return (size_t)p % 16 == 0 && ld * in.size % 16 == 0 && in.K * in.size % 16 == 0; }

// workspace in order: x and w in whole units where they are not, dgu, column sums, partial products
struct GlPlan {
    int ts_gate, ts_prod;
    size_t x, wg, wu, dgu, slab, part[3], bytes;      // offsets; 0-size parts share one
    bool pack_x, pack_g, pack_u, pp_gate, pp_prod;
    int splits[3], run[3];
};
constexpr long GL_PP_TILES = 192;
long gl_tiles(long I, long J, int ti, int tj) { return ((I + ti - 1) / ti) * ((J + tj - 1) / tj); }

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
    // the ping-pong tiles where they nearly fill the device; their loader's offsets are 32 bits over 256 rows
    const long most = 1L << 22, ldx = p.pack_x ? gl_up8(K) : in.ldx, ldg = p.pack_g ? gl_up8(K) : in.ldg, ldu = p.pack_u ? gl_up8(K) : in.ldu;
    const bool pp = in.size == 2 && ldx < most && ldg < most && ldu < most && F < most / 2;
    p.pp_gate = pp && K >= 128 && gl_tiles(M, F, 256, 128) >= GL_PP_TILES;
    // the large tile where it still gives every compute unit a workgroup
    p.ts_gate = gl_tiles(M, F, 128, 64) >= 256 ? 128 : 64;
    if (backward) {
        p.dgu = take((size_t)M * 2 * gl_up8(F) * in.size);
        p.slab = take((size_t)((M + 63) / 64) * 2 * F * 4);
        const long I[3] = {M, F, F}, chunks[3] = {2 * ((F + bk - 1) / bk), (M + bk - 1) / bk, (M + bk - 1) / bk};
        p.pp_prod = pp && ldg == ldu && M >= 128 && F >= 64 && gl_tiles(M, K, 256, 256) + 2 * gl_tiles(F, K, 256, 256) >= GL_PP_TILES;
        p.ts_prod = gl_tiles(M, K, 128, 128) + 2 * gl_tiles(F, K, 128, 128) >= 512 ? 128 : 64;
        for (int q = 0; q < 3; ++q) {
            // few tiles with a long k axis: runs of at least 4 chunks, as many as bring the product to 256 workgroups
            const long tiles = gl_tiles(I[q], K, p.ts_prod, p.ts_prod);
            long s = tiles > 0 ? 256 / tiles : 1;
            if (s > chunks[q] / 4) s = chunks[q] / 4;
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

template <typename T, int TS, bool BWD>
int gl_gate(const GlArgs& p, hipStream_t s)
{
    const long n = gl_tiles(p.M, p.F, TS, TS / 2);
    HN_REQUIRE(n <= 0x7fffffffL, "hn_gated_linear: too many tiles");
    static bool told[64] = {};
    if (const int rc = gl_big_lds(reinterpret_cast<const void*>(gl_gate_kernel<T, TS, BWD>), gl_lds_bytes<TS>(), told)) return rc;
    hipLaunchKernelGGL((gl_gate_kernel<T, TS, BWD>), dim3((unsigned)n), dim3(256), gl_lds_bytes<TS>(), s, p);
    HN_LAUNCH_CHECK();
    return 0;
}

template <typename T, int TS>
int gl_products(GlJobs& jobs, hipStream_t s)
{
    long n = 0, most = 0;
    for (int q = 0; q < jobs.n; ++q) {
        GlJob& j = jobs.j[q];
        j.tj = (j.J + TS - 1) / TS;
        j.tiles = gl_tiles(j.I, j.J, TS, TS);
        j.first = (int)n;
        n += j.tiles * j.splits;
        HN_REQUIRE(n <= 0x7fffffffL, "hn_gated_linear_bwd: too many tiles");
        if (j.splits > 1 && j.I * j.J > most) most = j.I * j.J;
    }
    if (n == 0) return 0;
    static bool told[64] = {};
    if (const int rc = gl_big_lds(reinterpret_cast<const void*>(gl_product_kernel<T, TS>), gl_lds_bytes<TS>(), told)) return rc;
    hipLaunchKernelGGL((gl_product_kernel<T, TS>), dim3((unsigned)n), dim3(256), gl_lds_bytes<TS>(), s, jobs);
    HN_LAUNCH_CHECK();
    if (most) {
        long g = (most + 255) / 256;
        if (g > 2048) g = 2048;
        hipLaunchKernelGGL((gl_join_kernel<T>), dim3((unsigned)g), dim3(256), 0, s, jobs);
        HN_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T>
int gl_forward(const GlIn& in, GlArgs p, char* ws, hipStream_t s)
{
    const GlPlan pl = gl_plan(in, false);
    if (const int rc = gl_prepare<T>(in, pl, ws, p.x, p.w, s)) return rc;
    if (pl.pp_gate) return hn_launch_gated_linear_pp_gate(p, false, s);
    return pl.ts_gate == 128 ? gl_gate<T, 128, false>(p, s) : gl_gate<T, 64, false>(p, s);
}

template <typename T>
int gl_backward(const GlIn& in, GlArgs p, char* ws, void* dx, void* dwg, void* dwu, void* dbg, void* dbu, hipStream_t s)
{
    const GlPlan pl = gl_plan(in, true);
    const long bk = GlNum<T>::BK, Fp = p.Fp;
    const int rows = pl.pp_gate ? 128 : pl.ts_gate;                   // of a column-sum tile
    if (const int rc = gl_prepare<T>(in, pl, ws, p.x, p.w, s)) return rc;
    p.dgu = ws + pl.dgu;
    p.slab = dbg || dbu ? (float*)(ws + pl.slab) : nullptr;
    if (in.M > 0 && in.F > 0)
        if (const int rc = pl.pp_gate ? hn_launch_gated_linear_pp_gate(p, true, s) : pl.ts_gate == 128 ? gl_gate<T, 128, true>(p, s) : gl_gate<T, 64, true>(p, s))
            return rc;
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
    if (const int rc = pl.pp_prod ? hn_launch_gated_linear_pp_products(jobs, s) : pl.ts_prod == 128 ? gl_products<T, 128>(jobs, s) : gl_products<T, 64>(jobs, s)) return rc;
    if ((dbg || dbu) && in.F > 0)
        hipLaunchKernelGGL((gl_bias_kernel<T>), dim3((unsigned)((2 * in.F + 255) / 256)), dim3(256), 0, s, p.slab, (in.M + rows - 1) / rows, in.F, (T*)dbg, (T*)dbu);
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
    if (M < 0 || K < 0 || F < 0 || M >= (1L << 31) || K >= (1L << 24) || F >= (1L << 24) || (dtype != SEQ_F32 && dtype != SEQ_BF16)) return 0;
    return gl_plan(gl_in(x, ldx, w_gate, ld_gate, w_up, ld_up, M, K, F, dtype), backward != 0).bytes;
}

extern "C" int hn_gated_linear(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up, const void* b_gate,
                               const void* b_up, void* y, void* workspace, size_t workspace_bytes, int64_t M, int64_t K, int64_t F, int dtype, int act,
                               void* stream)
{
    if (const int rc = gl_check(M, K, F, dtype, act)) return rc;
    if (M == 0 || F == 0) return 0;
    HN_REQUIRE(y && (K == 0 || (x && w_gate && w_up)), "hn_gated_linear: null pointer");
    const GlIn in = gl_in(x, ldx, w_gate, ld_gate, w_up, ld_up, M, K, F, dtype);
    HN_REQUIRE(workspace_bytes >= gl_plan(in, false).bytes && (workspace || workspace_bytes == 0) && (size_t)workspace % 16 == 0,
               "hn_gated_linear: workspace too small or not aligned to 16 bytes");
    GlArgs p = {};
    p.bg = b_gate; p.bu = b_up; p.y = y;
    p.M = M; p.K = K; p.F = F; p.Fp = gl_up8(F); p.act = act;
    p.y_vec = (size_t)y % 16 == 0 && F * in.size % 16 == 0;
    return dtype == SEQ_BF16 ? gl_forward<seq_bf16>(in, p, (char*)workspace, (hipStream_t)stream) : gl_forward<float>(in, p, (char*)workspace, (hipStream_t)stream);
}

extern "C" int hn_gated_linear_bwd(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up, const void* b_gate,
                                   const void* b_up, const void* dy, int64_t ld_dy, void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up,
                                   void* workspace, size_t workspace_bytes, int64_t M, int64_t K, int64_t F, int dtype, int act, void* stream)
{
    if (const int rc = gl_check(M, K, F, dtype, act)) return rc;
    HN_REQUIRE(M == 0 || F == 0 || (dy && (K == 0 || (x && w_gate && w_up))), "hn_gated_linear_bwd: null pointer");
    const GlIn in = gl_in(x, ldx, w_gate, ld_gate, w_up, ld_up, M, K, F, dtype);
    HN_REQUIRE(workspace_bytes >= gl_plan(in, true).bytes && (workspace || workspace_bytes == 0) && (size_t)workspace % 16 == 0,
               "hn_gated_linear_bwd: workspace too small or not aligned to 16 bytes");
    HN_REQUIRE((size_t)dx % 16 == 0 && (size_t)dw_gate % 16 == 0 && (size_t)dw_up % 16 == 0, "hn_gated_linear_bwd: dx, dw_gate and dw_up start on 16 bytes");
    GlArgs p = {};
    p.bg = b_gate; p.bu = b_up; p.dy = dy; p.ldd = ld_dy;
    p.M = M; p.K = K; p.F = F; p.Fp = gl_up8(F); p.act = act;
    p.dy_vec = (size_t)dy % 16 == 0 && ld_dy * in.size % 16 == 0;
    return dtype == SEQ_BF16 ? gl_backward<seq_bf16>(in, p, (char*)workspace, dx, dw_gate, dw_up, db_gate, db_up, (hipStream_t)stream)
                             : gl_backward<float>(in, p, (char*)workspace, dx, dw_gate, dw_up, db_gate, db_up, (hipStream_t)stream);
}
