// Matrix-core tiles of the gated linear block (gated_linear.hip): C[i][j] = sum_k A(i, k) B(j, k), bf16 or float32 operands, float32 sums.
//
// A workgroup of 4 waves (2 x 2) owns a TI x TJ tile and walks k in chunks of 128 bytes, two LDS buffers, the next two chunks' global loads
// in registers while the matrix cores work on this one.  An operand lies either with k contiguous (KC: rows of 128 bytes in LDS) or with its
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

// This thread's units of one operand: byte offsets from a uniform base that moves from chunk to chunk.  The loads go through the bounds check
// of a buffer descriptor: an offset past its end reads 0 and no lane branches, so the loads of two chunks stay in flight by their count.
// (A tile's rows span less than 2^31 bytes: the host copies operands with longer strides.)
constexpr unsigned GL_NONE = 0x80000000u;
template <typename T, int TS, int KIND>
struct GlLoader {
    static constexpr int Q = TS / 32, E = GlNum<T>::E;
    const char* base;
    long step;
    unsigned off[Q];
    int k[Q];                 // k of the unit within a chunk

    // the first chunk at k0 of source src
    __device__ __forceinline__ void aim(const GlOpd& o, int src, long i0, long k0)
    {
        // (GL_DUAL: rows 16 .. 31 of every 32 come from the up matrix: those of waves 2 and 3)
        const int m = KIND == GL_DUAL ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 7) : src;
        const long ld = m ? o.ld[1] : o.ld[0], rest = o.n - i0;
        const T* p = (const T*)(m ? o.p[1] : o.p[0]);
        base = (const char*)(KIND == GL_KR ? p + k0 * ld + i0 : p + i0 * ld + k0);
        step = (KIND == GL_KR ? GlNum<T>::BK * ld : GlNum<T>::BK) * (long)sizeof(T);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int u = (int)threadIdx.x + 256 * q;
            if constexpr (KIND == GL_KR) {
                const int x = u % (TS / E) * E;
                k[q] = u / (TS / E);
                off[q] = x < rest ? ((unsigned)k[q] * (unsigned)ld + (unsigned)x) * (unsigned)sizeof(T) : GL_NONE;
            } else {
                const int row = u >> 3, x = KIND == GL_DUAL ? (row >> 5) * 16 + (row & 15) : row;
                k[q] = (u & 7) * E;
                off[q] = x < rest ? ((unsigned)x * (unsigned)ld + (unsigned)k[q]) * (unsigned)sizeof(T) : GL_NONE;
            }
        }
    }
    // the current chunk, of which `left` k's exist; then on to the next
    __device__ __forceinline__ void fetch(gl_u32x4 (&r)[Q], int left)
    {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int q = 0; q < Q; ++q) r[q] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, k[q] < left ? off[q] : GL_NONE, 0, 0);
        base += step;
    }
};
// unit q: registers -> LDS
template <typename T, int TS, int KIND>
__device__ __forceinline__ void gl_put(char* lds, gl_u32x4 r, int q)
{
    constexpr int E = GlNum<T>::E;
    const int u = (int)threadIdx.x + 256 * q;
    int at;
    if constexpr (KIND == GL_KR) {
        at = gl_kr_at<T, TS>(u / (TS / E), u % (TS / E));
    } else {
        const int row = u >> 3, unit = u & 7;
        at = row * 128 + ((unit ^ (row & 7)) * 16);
    }
    *reinterpret_cast<gl_u32x4*>(lds + at) = r;
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
// product m of a k step over NI x NJ tiles of 16 x 16: NI * NJ of them in bf16; in float32 four times as many, one k group after the other over
// all tiles, so that none waits for the one before it
template <typename T, int NI, int NJ>
constexpr int gl_products_of() { return NI * NJ * (sizeof(T) == 2 ? 1 : 4); }
template <typename T, int NI, int NJ>
__device__ __forceinline__ void gl_mma(const gl_u32x4 (&a)[NI], const gl_u32x4 (&b)[NJ], f32x4 (&c)[NI][NJ], int m)
{
    const int t = m / (NI * NJ), i = m / NJ % NI, j = m % NJ;
    if constexpr (sizeof(T) == 2) {
        c[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gl_bf16x8, a[i]), __builtin_bit_cast(gl_bf16x8, b[j]), c[i][j], 0, 0, 0);
    } else {
        const f32x4 x = __builtin_bit_cast(f32x4, a[i]), y = __builtin_bit_cast(f32x4, b[j]);
        c[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t], y[t], c[i][j], 0, 0, 0);
    }
}
// products M0 .. M1 - 1 with the other operations 0 .. OPS - 1 spread between the first half of them: the matrix pipe works on while they issue,
// and they have the other half to return
template <int M0, int M1, int OPS, class Product, class Other>
__device__ __forceinline__ void gl_weave(Product product, Other other)
{
    constexpr int H = (M1 - M0 + 1) / 2;
#pragma unroll
    for (int m = M0; m < M1; ++m) {
        product(m);
        if (m - M0 < H)
#pragma unroll
            for (int s = (m - M0) * OPS / H; s < (m - M0 + 1) * OPS / H; ++s) other(s);
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <int TI, int TJ>
constexpr int gl_lds_bytes() { return TI * (TJ + 4) * 4 > 2 * (TI + TJ) * 128 ? TI * (TJ + 4) * 4 : 2 * (TI + TJ) * 128; }

// chunks c0 .. c1 - 1 of the k axis (`per` chunks per source, K elements per source) into the wave's TI/2 x TJ/2 accumulators
template <typename T, int TI, int TJ, int KA, int KB>
__device__ __forceinline__ void gl_loop(char* lds, f32x4 (&acc)[TI / 32][TJ / 32], const GlOpd& a, long i0, const GlOpd& b, long j0, long K, int per, int c0,
                                        int c1)
{
    constexpr int NI = TI / 32, NJ = TJ / 32, BUF = (TI + TJ) * 128;
    constexpr int BK = GlNum<T>::BK;
    const int wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
    constexpr int D = 2;                             // chunks whose loads are in flight (4 measured the same: this is not what it waits for)
    gl_u32x4 ra[D][NI], rb[D][NJ];
    GlLoader<T, TI, KA> la;
    GlLoader<T, TJ, KB> lb;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto aim = [&](int src, int c) {
        la.aim(a, src, i0, (long)c * BK);
        lb.aim(b, src, j0, (long)c * BK);
    };
    auto fetch = [&](int c, int set) {               // chunk c, the next in turn; zeros behind the last
        if (c == per && c < c1) aim(1, 0);
        const long rest = c < c1 ? K - (long)(c >= per ? c - per : c) * BK : 0;
        const int left = rest < BK ? (int)rest : BK;
        la.fetch(ra[set], left);
        lb.fetch(rb[set], left);
    };
    gl_u32x4 fa[2][NI], fb[2][NJ];                   // fragments of the two k steps
    auto put = [&](int set, int q) {                 // unit q of the chunk in registers `set` into its buffer
        char* buf = lds + (set & 1) * BUF;
        if (q < NI) gl_put<T, TI, KA>(buf, ra[set][q], q);
        else gl_put<T, TJ, KB>(buf + TI * 128, rb[set][q - NI], q - NI);
    };
    auto read = [&](int set, int st, int q) {
        const char* buf = lds + (set & 1) * BUF;
        if (q < NI) fa[st][q] = gl_frag<T, TI, KA>(buf, wi * NI + q, st);
        else fb[st][q - NI] = gl_frag<T, TJ, KB>(buf + TI * 128, wj * NJ + q - NI, st);
    };
    // Chunk c, which came through registers `set`: the first step's products beside the reads of the second step's fragments; half of the second step's beside
    // the next chunk's way into the other buffer (read last before the barrier of chunk c - 1); the other half, behind the barrier, beside the
    // reads of its first fragments.  Behind the last chunk all of this moves zeros.
    constexpr int NP = gl_products_of<T, NI, NJ>(), OPS = NI + NJ;
    auto work = [&](int c, int set) {
        const int next = (set + 1) % D;
        fetch(c + D, set);
        __builtin_amdgcn_sched_barrier(0);
        gl_weave<0, NP, OPS>([&](int m) { gl_mma<T, NI, NJ>(fa[0], fb[0], acc, m); }, [&](int q) { read(set, 1, q); });
        gl_weave<0, NP / 2, OPS>([&](int m) { gl_mma<T, NI, NJ>(fa[1], fb[1], acc, m); }, [&](int q) { put(next, q); });
        __syncthreads();
        gl_weave<NP / 2, NP, OPS>([&](int m) { gl_mma<T, NI, NJ>(fa[1], fb[1], acc, m); }, [&](int q) { read(next, 0, q); });
    };
    if (c0 < c1) {
        if (c0 < per) aim(0, c0); else if (c0 > per) aim(1, c0 - per);
#pragma unroll
        for (int d = 0; d < D; ++d) fetch(c0 + d, d);
#pragma unroll
        for (int q = 0; q < OPS; ++q) put(0, q);
        __syncthreads();
#pragma unroll
        for (int q = 0; q < OPS; ++q) read(0, 0, q);
        int c = c0;
        for (; c + D <= c1; c += D)
#pragma unroll
            for (int d = 0; d < D; ++d) work(c + d, d);
#pragma unroll
        for (int d = 0; d < D - 1; ++d)
            if (c + d < c1) work(c + d, d);
    }
    __syncthreads();
}
// accumulators -> float32 tile in LDS, rows of TJ + 4
template <int TI, int TJ>
__device__ __forceinline__ void gl_dump(float* t, const f32x4 (&acc)[TI / 32][TJ / 32])
{
    constexpr int NI = TI / 32, NJ = TJ / 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) t[((wi * NI + i) * 16 + 4 * (lane >> 4) + r) * (TJ + 4) + (wj * NJ + j) * 16 + (lane & 15)] = acc[i][j][r];
    __syncthreads();
}

}  // namespace
