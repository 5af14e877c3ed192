// Gated linear block, both projections, the activation and the product in one kernel, with its backward pass:
//
//     g = x Wg^T + bg     u = x Wu^T + bu     y = act(g) * u            x [M][K], W [F][K] (the layout of a Linear's weight), y [M][F]
//
// g and u are never stored.  The backward pass forms them again tile by tile and writes what the products need,
//     dg = dy u act'(g)      du = dy act(g)        (one [M][2F] buffer, dg | du, in the inputs' type)
// then  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x;  the bias gradients are column sums of the unrounded dg, du, per row tile into a
// slab that a last pass adds in order (no atomics: the same bits every time).
#include "seq_common.h"

namespace {

constexpr int ACT_SILU = 0, ACT_GELU = 1, ACT_SIGMOID = 2, ACT_RELU = 3;

// value and slope of the activation
template <bool EXACT>
__device__ __forceinline__ void gl_act(float z, int act, float& a, float& slope)
{
    if (act == ACT_RELU) {
        a = z > 0.f ? z : (z != z ? z : 0.f);
        slope = z > 0.f ? 1.f : 0.f;
    } else if (act == ACT_GELU) {
        const float cdf = 0.5f * erfcf(-0.70710678118654752f * z);
        a = z * cdf;
        slope = fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), cdf);
    } else {
        float s, rest;
        seq_logistic<EXACT>(z, s, rest);
        if (act == ACT_SIGMOID) { a = s; slope = s * rest; }
        else { a = z * s; slope = fmaf(z * s, rest, s); }
    }
}

struct GlArgs {
    const void *x, *wg, *wu, *bg, *bu, *dy;
    long ldx, ldg, ldu, ldd;
    void *y, *dgu, *dx, *dwg, *dwu;
    float* slab;          // [row tiles][2F]
    long M, K, F;
    int act;
};

__device__ __forceinline__ float gl_ld(const float* p) { return *p; }
__device__ __forceinline__ float gl_ld(const seq_bf16* p) { return seq_from_bf16(*p); }

constexpr int BT = 64, BK = 16;

// one operand tile [64][16] of a matrix with element strides (si, sk), zero outside (n, kn)
template <typename T>
__device__ __forceinline__ void gl_tile(float (&s)[BK][BT + 1], const T* p, long i0, long n, long si, long k0, long kn, long sk)
{
    for (int e = threadIdx.x; e < BT * BK; e += 256) {
        const bool kfast = sk == 1;
        const int i = kfast ? e / BK : e % BT, k = kfast ? e % BK : e / BT;
        s[k][i] = i0 + i < n && k0 + k < kn ? gl_ld(p + (i0 + i) * si + (k0 + k) * sk) : 0.f;
    }
}
__device__ __forceinline__ void gl_mac(float (&acc)[4][4], const float (&a)[BK][BT + 1], const float (&b)[BK][BT + 1], int ti, int tj)
{
#pragma unroll
    for (int k = 0; k < BK; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[k][ti + 16 * i], b[k][tj + 16 * j], acc[i][j]);
}

template <typename T, bool BWD>
__global__ __launch_bounds__(256) void gl_gate_kernel(GlArgs p)
{
    __shared__ float xs[BK][BT + 1], gs[BK][BT + 1], us[BK][BT + 1];
    __shared__ float red[2][16][BT];
    const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
    const long nt = (p.F + BT - 1) / BT;
    const long m0 = blockIdx.x / nt * BT, f0 = blockIdx.x % nt * BT;
    float ag[4][4] = {}, au[4][4] = {};
    for (long k0 = 0; k0 < p.K; k0 += BK) {
        gl_tile(xs, (const T*)p.x, m0, p.M, p.ldx, k0, p.K, 1L);
        gl_tile(gs, (const T*)p.wg, f0, p.F, p.ldg, k0, p.K, 1L);
        gl_tile(us, (const T*)p.wu, f0, p.F, p.ldu, k0, p.K, 1L);
        __syncthreads();
        gl_mac(ag, xs, gs, ti, tj);
        gl_mac(au, xs, us, ti, tj);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const long f = f0 + tj + 16 * j;
        const float bg = p.bg && f < p.F ? gl_ld((const T*)p.bg + f) : 0.f, bu = p.bu && f < p.F ? gl_ld((const T*)p.bu + f) : 0.f;
        float sg = 0.f, su = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long m = m0 + ti + 16 * i;
            if (m < p.M && f < p.F) {
                float a, slope;
                const float u = au[i][j] + bu;
                gl_act<sizeof(T) == 4>(ag[i][j] + bg, p.act, a, slope);
                if (!BWD) {
                    float o[1] = {a * u};
                    seq_store<1>((T*)p.y + m * p.F + f, o);
                } else {
                    const float dy = gl_ld((const T*)p.dy + m * p.ldd + f);
                    float dg[1] = {dy * u * slope}, du[1] = {dy * a};
                    sg += dg[0];
                    su += du[0];
                    seq_store<1>((T*)p.dgu + m * 2 * p.F + f, dg);
                    seq_store<1>((T*)p.dgu + m * 2 * p.F + p.F + f, du);
                }
            }
        }
        if (BWD) { red[0][ti][tj + 16 * j] = sg; red[1][ti][tj + 16 * j] = su; }
    }
    if (BWD && p.slab) {
        __syncthreads();
        if (threadIdx.x < 2 * BT) {
            const int w = threadIdx.x / BT, c = threadIdx.x % BT;
            float s = 0.f;
            for (int i = 0; i < 16; ++i) s += red[w][i][c];
            if (f0 + c < p.F) p.slab[(m0 / BT) * 2 * p.F + w * p.F + f0 + c] = s;
        }
    }
}

// out[i][j] = sum_k A(i, k) B(j, k), over one or two operand pairs; element strides everywhere
template <typename T>
__global__ __launch_bounds__(256) void gl_product_kernel(const T* a0, const T* b0, const T* a1, const T* b1, long ai, long ak, long bj, long bk, long bj1, long bk1,
                                                         T* out, long I, long J, long Kn)
{
    __shared__ float as[BK][BT + 1], bs[BK][BT + 1];
    const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
    const long nt = (J + BT - 1) / BT;
    const long i0 = blockIdx.x / nt * BT, j0 = blockIdx.x % nt * BT;
    float acc[4][4] = {};
    for (int q = 0; q < (a1 ? 2 : 1); ++q)
        for (long k0 = 0; k0 < Kn; k0 += BK) {
            gl_tile(as, q ? a1 : a0, i0, I, ai, k0, Kn, ak);
            gl_tile(bs, q ? b1 : b0, j0, J, q ? bj1 : bj, k0, Kn, q ? bk1 : bk);
            __syncthreads();
            gl_mac(acc, as, bs, ti, tj);
            __syncthreads();
        }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long r = i0 + ti + 16 * i, c = j0 + tj + 16 * j;
            float o[1] = {acc[i][j]};
            if (r < I && c < J) seq_store<1>(out + r * J + c, o);
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
    HN_REQUIRE(act >= ACT_SILU && act <= ACT_RELU, "hn_gated_linear: activation is 0 (silu), 1 (gelu), 2 (sigmoid) or 3 (relu)");
    return 0;
}
int gl_grid(long I, long J, dim3& g)
{
    const long n = ((I + BT - 1) / BT) * ((J + BT - 1) / BT);
    HN_REQUIRE(n <= 0x7fffffffL, "hn_gated_linear: too many tiles");
    g = dim3((unsigned)n);
    return 0;
}

template <typename T>
int gl_backward(GlArgs& p, void* dbg, void* dbu, hipStream_t s)
{
    dim3 g;
    if (p.F > 0 && p.M > 0) {
        if (int rc = gl_grid(p.M, p.F, g)) return rc;
        hipLaunchKernelGGL((gl_gate_kernel<T, true>), g, dim3(256), 0, s, p);
    }
    const T* dg = (const T*)p.dgu;
    if (p.dx && p.M > 0 && p.K > 0) {
        if (int rc = gl_grid(p.M, p.K, g)) return rc;
        hipLaunchKernelGGL((gl_product_kernel<T>), g, dim3(256), 0, s, dg, (const T*)p.wg, dg + p.F, (const T*)p.wu, 2 * p.F, 1L, 1L, p.ldg, 1L, p.ldu, (T*)p.dx,
                           p.M, p.K, p.F);
    }
    if (p.F > 0 && p.K > 0) {
        if (int rc = gl_grid(p.F, p.K, g)) return rc;
        if (p.dwg)
            hipLaunchKernelGGL((gl_product_kernel<T>), g, dim3(256), 0, s, dg, (const T*)p.x, (const T*)nullptr, (const T*)nullptr, 1L, 2 * p.F, 1L, p.ldx, 0L, 0L,
                               (T*)p.dwg, p.F, p.K, p.M);
        if (p.dwu)
            hipLaunchKernelGGL((gl_product_kernel<T>), g, dim3(256), 0, s, dg + p.F, (const T*)p.x, (const T*)nullptr, (const T*)nullptr, 1L, 2 * p.F, 1L, p.ldx,
                               0L, 0L, (T*)p.dwu, p.F, p.K, p.M);
    }
    if ((dbg || dbu) && p.F > 0)
        hipLaunchKernelGGL((gl_bias_kernel<T>), dim3((unsigned)((2 * p.F + 255) / 256)), dim3(256), 0, s, p.slab, (p.M + BT - 1) / BT, p.F, (T*)dbg, (T*)dbu);
    HN_LAUNCH_CHECK();
    return 0;
}

size_t gl_round(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

extern "C" size_t hn_gated_linear_workspace(int64_t M, int64_t K, int64_t F, int dtype, int backward)
{
    (void)K;
    if (!backward || M <= 0 || F <= 0) return 0;
    return gl_round((size_t)M * 2 * F * (dtype == SEQ_F32 ? 4 : 2)) + gl_round((size_t)((M + BT - 1) / BT) * 2 * F * 4);
}

extern "C" int hn_gated_linear(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up, const void* b_gate,
                               const void* b_up, void* y, void* workspace, size_t workspace_bytes, int64_t M, int64_t K, int64_t F, int dtype, int act,
                               void* stream)
{
    if (const int rc = gl_check(M, K, F, dtype, act)) return rc;
    if (M == 0 || F == 0) return 0;
    HN_REQUIRE(y && (K == 0 || (x && w_gate && w_up)), "hn_gated_linear: null pointer");
    HN_REQUIRE(workspace_bytes >= hn_gated_linear_workspace(M, K, F, dtype, 0), "hn_gated_linear: workspace too small");
    (void)workspace;
    GlArgs p = {};
    p.x = x; p.wg = w_gate; p.wu = w_up; p.bg = b_gate; p.bu = b_up; p.y = y;
    p.ldx = ldx; p.ldg = ld_gate; p.ldu = ld_up;
    p.M = M; p.K = K; p.F = F; p.act = act;
    dim3 g;
    if (const int rc = gl_grid(M, F, g)) return rc;
    if (dtype == SEQ_BF16) hipLaunchKernelGGL((gl_gate_kernel<seq_bf16, false>), g, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((gl_gate_kernel<float, false>), g, dim3(256), 0, (hipStream_t)stream, p);
    HN_LAUNCH_CHECK();
    return 0;
}

extern "C" int hn_gated_linear_bwd(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up, const void* b_gate,
                                   const void* b_up, const void* dy, int64_t ld_dy, void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up,
                                   void* workspace, size_t workspace_bytes, int64_t M, int64_t K, int64_t F, int dtype, int act, void* stream)
{
    if (const int rc = gl_check(M, K, F, dtype, act)) return rc;
    HN_REQUIRE(M == 0 || F == 0 || (dy && (K == 0 || (x && w_gate && w_up))), "hn_gated_linear_bwd: null pointer");
    HN_REQUIRE(workspace_bytes >= hn_gated_linear_workspace(M, K, F, dtype, 1) && (workspace || workspace_bytes == 0), "hn_gated_linear_bwd: workspace too small");
    GlArgs p = {};
    p.x = x; p.wg = w_gate; p.wu = w_up; p.bg = b_gate; p.bu = b_up; p.dy = dy;
    p.ldx = ldx; p.ldg = ld_gate; p.ldu = ld_up; p.ldd = ld_dy;
    p.dx = dx; p.dwg = dw_gate; p.dwu = dw_up;
    p.M = M; p.K = K; p.F = F; p.act = act;
    p.dgu = workspace;
    p.slab = (db_gate || db_up) ? (float*)((char*)workspace + gl_round((size_t)M * 2 * F * (dtype == SEQ_F32 ? 4 : 2))) : nullptr;
    return dtype == SEQ_BF16 ? gl_backward<seq_bf16>(p, db_gate, db_up, (hipStream_t)stream) : gl_backward<float>(p, db_gate, db_up, (hipStream_t)stream);
}
