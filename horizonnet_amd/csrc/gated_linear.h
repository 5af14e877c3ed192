// What the two families of kernels of the gated linear block share: operands, jobs, the activation (gated_linear.hip: 32 to 128 wide tiles for every
// size and type; gated_linear_pp.hip: 256 x 256 ping-pong tiles for large bf16 sizes).
#pragma once
#include "seq_common.h"

constexpr int GL_SILU = 0, GL_GELU = 1, GL_SIGMOID = 2, GL_RELU = 3;

// One operand.  Two sources: the two halves of a longer k axis, or the gate and the up matrix.
struct GlOpd {
    const void* p[2];
    long ld[2];
    long n;               // extent of the operand's own index
};

// both projections, and y (forward) or dg | du (backward)
struct GlArgs {
    GlOpd x, w;           // w: gate and up matrices
    const void *bg, *bu, *dy;
    long ldd;
    void *y, *dgu;        // dgu: dg | du, rows of 2 Fp
    float* kept;          // g | u as the forward pass formed them, rows of 2 Fp, or null
    float* slab;          // [row tiles][2F] column sums of dg | du, or null
    long M, K, F, Fp;
    int act, dy_vec, y_vec;
};

// a product of the backward pass: out[I][J] over `chunks` chunks of k (`per` of each source, K k's of each), cut into `splits` runs of `run`
struct GlJob {
    GlOpd a, b;
    long I, J, K;
    int per, chunks, splits, run;
    int a_kr;
    int first;            // first workgroup
    long tj, tiles;
    void* out;
    float* part;          // [splits][I][J] float32 where splits > 1
};
struct GlJobs {
    GlJob j[3];
    int n;
};

int hn_launch_gated_linear_pp_gate(const GlArgs& p, bool backward, hipStream_t s);
int hn_launch_gated_linear_pp_products(GlJobs& jobs, hipStream_t s);

namespace {

// Value and slope of the activation.  bf16 (not EXACT): the sigmoid from one exponential and one reciprocal.  silu takes 1 - s by subtraction, whose
// loss is far below the step of a bf16 result: s and 1 - s enter its slope beside terms of their own size.  sigmoid's slope s (1 - s) has 1 - s as a bare
// factor (the subtraction is 17 % off at z 15 and 0 from 17 on), so it is e^-z s there.
template <bool EXACT>
__device__ __forceinline__ void gl_act(float z, int act, float& a, float& slope)
{
    if (act == GL_RELU) {
        a = z > 0.f ? z : (z != z ? z : 0.f);
        slope = z <= 0.f ? 0.f : 1.f;
    } else if (act == GL_GELU) {
        const float cdf = 0.5f * erfcf(-0.70710678118654752f * z);
        a = z * cdf;
        slope = fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), cdf);
    } else {
        float s, rest;
        if constexpr (EXACT) {
            seq_logistic<true>(z, s, rest);
        } else {
            const float e = __expf(-z);
            s = __builtin_amdgcn_rcpf(1.f + e);
            rest = act == GL_SIGMOID ? fminf(e, 3.0e38f) * s : 1.f - s;     // (s is 0 where e is infinite)
        }
        if (act == GL_SIGMOID) { a = s; slope = s * rest; }
        else { a = z * s; slope = fmaf(a, rest, s); }
    }
}

typedef unsigned int gl_u32x4 __attribute__((ext_vector_type(4)));
typedef short gl_s16x4 __attribute__((ext_vector_type(4)));

// 8 neighbouring values of a row: one or two 16-byte accesses where `vec` says that the row allows it, else one by one up to `n`
__device__ __forceinline__ void gl_store8(float* p, const float (&x)[8], bool vec, long n)
{
    if (vec && n >= 8) {
        *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = x[e];
    }
}
__device__ __forceinline__ void gl_store8(seq_bf16* p, const float (&x)[8], bool vec, long n)
{
    if (vec && n >= 8) {
        *reinterpret_cast<gl_u32x4*>(p) = gl_u32x4{seq_pack2(x[0], x[1]), seq_pack2(x[2], x[3]), seq_pack2(x[4], x[5]), seq_pack2(x[6], x[7])};
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = (seq_bf16)(seq_pack2(x[e], 0.f) & 0xffffu);
    }
}
__device__ __forceinline__ void gl_load8(const float* p, float (&x)[8], bool vec, long n)
{
    if (vec && n >= 8) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e < n ? p[e] : 0.f;
    }
}
__device__ __forceinline__ void gl_open8(gl_u32x4 t, float (&x)[8])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned w = t[e];
        x[2 * e] = __builtin_bit_cast(float, w << 16);
        x[2 * e + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
    }
}
__device__ __forceinline__ void gl_load8(const seq_bf16* p, float (&x)[8], bool vec, long n)
{
    if (vec && n >= 8) {
        gl_open8(*reinterpret_cast<const gl_u32x4*>(p), x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e < n ? seq_from_bf16(p[e]) : 0.f;
    }
}
__device__ __forceinline__ float gl_ld(const float* p) { return *p; }
__device__ __forceinline__ float gl_ld(const seq_bf16* p) { return seq_from_bf16(*p); }

// neighbouring tiles (they share operands) on one XCD, which has an L2 of its own: workgroups go round the 8 XCDs
__device__ __forceinline__ long gl_tile_of(long bid, long n)
{
    const long q = n >> 3, r = n & 7, xcd = bid & 7;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
}

// the same for a grid of mt x nt tiles, in bands of GL_BAND rows of tiles walked column by column: the tiles that an XCD works on at a time then
// need GL_BAND row operands and a few column operands, not one row's and all columns'
// (bands of 4 against 1, bf16 forward at M 16384, K 1024, F 4096: 249.5 us against 266.6; 8: 248.9)
constexpr long GL_BAND = 4;
__device__ __forceinline__ void gl_tile_at(long bid, long mt, long nt, long& row, long& col)
{
    const long t = gl_tile_of(bid, mt * nt), band = t / (GL_BAND * nt), first = band * GL_BAND, rest = t - first * nt;
    const long rows = mt - first < GL_BAND ? mt - first : GL_BAND;
    col = rest / rows;
    row = first + rest - col * rows;
}

}  // namespace
