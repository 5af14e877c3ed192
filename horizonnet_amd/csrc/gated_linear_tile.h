// Matrix-core tiles of the gated linear block (gated_linear.hip): C[i][j] = sum_k A(i, k) B(j, k), bf16 or float32 operands, float32 sums.
//
// A workgroup of 4 waves (2 x 2) owns a TS x TS tile and walks k in chunks of 128 bytes, two LDS buffers, the next chunk's global loads in
// registers while the matrix cores work on this one.  An operand lies either with k contiguous (KC: rows of 128 bytes in LDS) or with its
// own index contiguous (KR: one LDS row per k), so no product needs a transposed copy of its inputs:
//   KC  16-byte unit u of row r sits at u ^ (r & 7); a lane reads 16 bytes of its row: 8 bf16 k's, or 4 float32 k's for four MFMAs
//   KR  bf16: the transposing LDS read gives each lane 4 k's of its column; float32: one 4-byte read per k.  32-byte (64-byte) blocks of a
//       row are exchanged so that the rows read together lie in different banks
// v_mfma_f32_16x16x32_bf16 / v_mfma_f32_16x16x4_f32: lane l holds A row (B column) l % 16 at k group l / 16, and C column l % 16, rows
// 4 (l / 16) .. + 3.  The order of k inside a chunk differs from memory order but is the same for both operands.
#pragma once
#include "gated_linear.h"

namespace {

typedef __bf16 gl_bf16x8 __attribute__((ext_vector_type(8)));

enum { GL_KC = 0, GL_KR = 1, GL_DUAL = 2 };      // GL_DUAL: KC rows, 16 of the first matrix and 16 of the second in turn

template <typename T>
struct GlNum {
    static constexpr int E = 16 / (int)sizeof(T);          // elements of a 16-byte unit
    static constexpr int BK = 128 / (int)sizeof(T);        // k's of a chunk
};

// byte address of unit (16 bytes) cu of LDS row k of a KR tile
template <typename T, int TS>
__device__ __forceinline__ int gl_kr_at(int k, int cu)
{
    if constexpr (sizeof(T) == 2) {
        const int swz = TS == 64 ? ((k >> 1) & 1) ^ (2 * ((k >> 3) & 1)) : (2 * (k & 3)) ^ ((k >> 3) & 1);
        return k * (TS * 2) + (((cu >> 1) ^ swz) * 32) + (cu & 1) * 16;
    } else {
        return k * (TS * 4) + (((cu >> 2) ^ ((k >> 2) & 3)) * 64) + (cu & 3) * 16;
    }
}

// this thread's units of one operand's chunk: global memory -> registers (0 outside), registers -> LDS
template <typename T, int TS, int KIND>
__device__ __forceinline__ void gl_fetch(gl_u32x4 (&r)[TS / 32], const GlOpd& o, int src, long i0, long k0, long K)
{
    constexpr int E = GlNum<T>::E;
#pragma unroll
    for (int q = 0; q < TS / 32; ++q) {
        const int u = (int)threadIdx.x + 256 * q;
        const T* at;
        bool on;
        if constexpr (KIND == GL_KR) {
            const int k = u / (TS / E), cu = u % (TS / E);
            on = k0 + k < K && i0 + cu * E < o.n;
            at = (const T*)o.p[src] + (k0 + k) * o.ld[src] + i0 + cu * E;
        } else {
            const int row = u >> 3, unit = u & 7;
            long i = i0 + row;
            int s = src;
            if constexpr (KIND == GL_DUAL) { i = i0 + (row >> 5) * 16 + (row & 15); s = (row >> 4) & 1; }
            on = i < o.n && k0 + unit * E < K;
            at = (const T*)(s ? o.p[1] : o.p[0]) + i * (s ? o.ld[1] : o.ld[0]) + k0 + unit * E;
        }
        r[q] = gl_u32x4{0, 0, 0, 0};
        if (on) r[q] = *reinterpret_cast<const gl_u32x4*>(at);
    }
}
template <typename T, int TS, int KIND>
__device__ __forceinline__ void gl_put(char* lds, const gl_u32x4 (&r)[TS / 32])
{
    constexpr int E = GlNum<T>::E;
#pragma unroll
    for (int q = 0; q < TS / 32; ++q) {
        const int u = (int)threadIdx.x + 256 * q;
        int at;
        if constexpr (KIND == GL_KR) {
            at = gl_kr_at<T, TS>(u / (TS / E), u % (TS / E));
        } else {
            const int row = u >> 3, unit = u & 7;
            at = row * 128 + ((unit ^ (row & 7)) * 16);
        }
        *reinterpret_cast<gl_u32x4*>(lds + at) = r[q];
    }
}
// fragment of the 16 operand indices 16 ib .. + 15 at k step st (half a chunk)
template <typename T, int TS, int KIND>
__device__ __forceinline__ gl_u32x4 gl_frag(const char* lds, int ib, int st)
{
    const int lane = threadIdx.x & 63, l16 = lane & 15, kg = lane >> 4;
    if constexpr (KIND != GL_KR) {
        const int row = ib * 16 + l16;
        return *reinterpret_cast<const gl_u32x4*>(lds + row * 128 + (((4 * st + kg) ^ (row & 7)) * 16));
    } else if constexpr (sizeof(T) == 2) {
        gl_u32x4 v;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int k = 32 * st + 8 * kg + 4 * q + (l16 >> 2);
            const int at = gl_kr_at<T, TS>(k, 2 * ib) + (lane & 3) * 8;
            const gl_s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) gl_s16x4*)(lds + at));
            const uint2 w = __builtin_bit_cast(uint2, t);
            v[2 * q] = w.x;
            v[2 * q + 1] = w.y;
        }
        return v;
    } else {
        gl_u32x4 v;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int k = 16 * st + 4 * kg + t;
            v[t] = *reinterpret_cast<const unsigned*>(lds + gl_kr_at<T, TS>(k, 4 * ib) + l16 * 4);
        }
        return v;
    }
}
template <typename T>
__device__ __forceinline__ f32x4 gl_mma(gl_u32x4 a, gl_u32x4 b, f32x4 c)
{
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gl_bf16x8, a), __builtin_bit_cast(gl_bf16x8, b), c, 0, 0, 0);
    } else {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t], y[t], c, 0, 0, 0);
        return c;
    }
}

template <int TS>
constexpr int gl_lds_bytes() { return TS * (TS + 4) * 4 > 4 * TS * 128 ? TS * (TS + 4) * 4 : 4 * TS * 128; }

// chunks c0 .. c1 - 1 of the k axis (`per` chunks per source, K elements per source) into the wave's TS/2 x TS/2 accumulators
template <typename T, int TS, int KA, int KB>
__device__ __forceinline__ void gl_loop(char* lds, f32x4 (&acc)[TS / 32][TS / 32], const GlOpd& a, long i0, const GlOpd& b, long j0, long K, int per, int c0, int c1)
{
    constexpr int N = TS / 32, BUF = TS * 128;
    constexpr long BK = GlNum<T>::BK;
    const int wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
    gl_u32x4 ra[N], rb[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto fetch = [&](int c) {
        const int src = c >= per ? 1 : 0;
        const long k0 = (long)(c - src * per) * BK;
        gl_fetch<T, TS, KA>(ra, a, src, i0, k0, K);
        gl_fetch<T, TS, KB>(rb, b, src, j0, k0, K);
    };
    if (c0 < c1) fetch(c0);
    for (int c = c0; c < c1; ++c) {
        char* buf = lds + ((c - c0) & 1) * 2 * BUF;
        gl_put<T, TS, KA>(buf, ra);
        gl_put<T, TS, KB>(buf + BUF, rb);
        __syncthreads();                             // (a buffer is filled again two chunks later: behind every reader's next barrier)
        if (c + 1 < c1) fetch(c + 1);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            gl_u32x4 fa[N], fb[N];
#pragma unroll
            for (int i = 0; i < N; ++i) fa[i] = gl_frag<T, TS, KA>(buf, wi * N + i, st);
#pragma unroll
            for (int j = 0; j < N; ++j) fb[j] = gl_frag<T, TS, KB>(buf + BUF, wj * N + j, st);
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) acc[i][j] = gl_mma<T>(fa[i], fb[j], acc[i][j]);
        }
    }
    __syncthreads();
}
// accumulators -> float32 tile in LDS, rows of TS + 4
template <int TS>
__device__ __forceinline__ void gl_dump(float* t, const f32x4 (&acc)[TS / 32][TS / 32])
{
    constexpr int N = TS / 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) t[((wi * N + i) * 16 + 4 * (lane >> 4) + r) * (TS + 4) + (wj * N + j) * 16 + (lane & 15)] = acc[i][j][r];
    __syncthreads();
}

}  // namespace
