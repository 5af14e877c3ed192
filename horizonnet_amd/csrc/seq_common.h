// Shared by the sequence operators (gated_recurrence.hip, gated_linear*.hip, dropout.hip): element types, vector access, logistic pair.
#pragma once
#include "hn_common.h"

// A launch holds fewer than 2^32 threads, whatever its number of workgroups
#define SEQ_REQUIRE_GRID(blocks, threads, what)                                                                             \
    HN_REQUIRE((long)(blocks) * (threads) < (1L << 32), what ": too large: %ld workgroups of %d threads, and a launch holds fewer than 2^32 threads", \
               (long)(blocks), (int)(threads))

namespace {

typedef unsigned short seq_bf16;      // storage of one bf16 value

constexpr int SEQ_F32 = 0, SEQ_BF16 = 1;

__device__ __forceinline__ float seq_from_bf16(unsigned short u) { return __builtin_bit_cast(float, (unsigned)u << 16); }

// two floats -> two bf16, round to nearest even: the one rounding of a stored result
__device__ __forceinline__ unsigned seq_pack2(float lo, float hi)
{
    unsigned r;
    asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(lo), "v"(hi));
    return r;
}

// VEC (1 or 4) neighbouring values as they lie in memory.  The vector types ask for no more than the element's own alignment: global memory is
// read and written at any of them, so rows of an odd number of channels take the same wide accesses.
typedef float seq_f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short seq_u16x4u __attribute__((ext_vector_type(4), aligned(2)));
template <typename T, int VEC>
struct SeqRaw;
template <>
struct SeqRaw<float, 4> { typedef seq_f32x4u type; };
template <>
struct SeqRaw<float, 1> { typedef float type; };
template <>
struct SeqRaw<seq_bf16, 4> { typedef seq_u16x4u type; };
template <>
struct SeqRaw<seq_bf16, 1> { typedef seq_bf16 type; };

__device__ __forceinline__ void seq_open(seq_f32x4u r, float (&x)[4]) { x[0] = r[0]; x[1] = r[1]; x[2] = r[2]; x[3] = r[3]; }
__device__ __forceinline__ void seq_open(float r, float (&x)[1]) { x[0] = r; }
__device__ __forceinline__ void seq_open(seq_u16x4u r, float (&x)[4])
{
    const uint2 t = __builtin_bit_cast(uint2, r);
    x[0] = __builtin_bit_cast(float, t.x << 16); x[1] = __builtin_bit_cast(float, t.x & 0xffff0000u);
    x[2] = __builtin_bit_cast(float, t.y << 16); x[3] = __builtin_bit_cast(float, t.y & 0xffff0000u);
}
__device__ __forceinline__ void seq_open(seq_bf16 r, float (&x)[1]) { x[0] = seq_from_bf16(r); }

template <int VEC, typename T>
__device__ __forceinline__ void seq_load(const T* p, float (&x)[VEC])
{
    seq_open(*reinterpret_cast<const typename SeqRaw<T, VEC>::type*>(p), x);
}
__device__ __forceinline__ void seq_put(float* p, const float (&x)[4]) { *reinterpret_cast<seq_f32x4u*>(p) = seq_f32x4u{x[0], x[1], x[2], x[3]}; }
__device__ __forceinline__ void seq_put(float* p, const float (&x)[1]) { *p = x[0]; }
__device__ __forceinline__ void seq_put(seq_bf16* p, const float (&x)[4])
{
    const uint2 t = make_uint2(seq_pack2(x[0], x[1]), seq_pack2(x[2], x[3]));
    *reinterpret_cast<seq_u16x4u*>(p) = __builtin_bit_cast(seq_u16x4u, t);
}
__device__ __forceinline__ void seq_put(seq_bf16* p, const float (&x)[1]) { *p = (seq_bf16)(seq_pack2(x[0], 0.f) & 0xffffu); }
template <int VEC, typename T>
__device__ __forceinline__ void seq_store(T* p, const float (&x)[VEC])
{
    seq_put(p, x);
}

// e^x for a factor of a float32 result.  EXACT: x is any float32, the library's exponential.  Else x is a bf16 value: its 8 bits times the 16 of
// SEQ_LOG2E are exact in float32, so 2^t takes no error from its argument, and what the constant leaves out, x SEQ_LOG2E_REST natural units
// (at most 5e-4 where the result is a normal number), is a factor 1 + c.  The constant of c is turned by 0.9e-4 to the side of e^c - 1 = c + c^2 / 2 for results
// below 1 (DOWN) or above.  Off by 4 u (u = 2^-24): 2 of v_exp_f32, 1 of the last sum, 0.9 of e^c.  The short exponential (2 instructions, |x| u) takes 3 fewer.
constexpr float SEQ_LOG2E = 0x1.7154p0f, SEQ_LOG2E_REST = 4.88849518e-6f;
template <bool EXACT, bool DOWN>
__device__ __forceinline__ float seq_exp(float x)
{
    if constexpr (EXACT) return expf(x);
    const float c = __builtin_amdgcn_fmed3f(x * (SEQ_LOG2E_REST * (DOWN ? 0.99991f : 1.00009f)), -0x1p-10f, 0x1p-10f);   // (x may be infinite)
    const float e = __builtin_amdgcn_exp2f(x * SEQ_LOG2E);
    return fmaf(e, c, e);
}

// s(x) and 1 - s(x) = s(-x) from ONE exponential of -|x|: neither is formed by a subtraction from 1, so the small one keeps its relative
// precision (a long memory is a small 1 - a).  Both are right to float32's last bits in both modes: the states that they make are float32, whatever the
// type of the inputs (exponential 4 u, sum and reciprocal 2 u, product u).
template <bool EXACT>
__device__ __forceinline__ void seq_logistic(float x, float& s, float& rest)
{
    const float e = seq_exp<EXACT, true>(-fabsf(x));
    const float big = __builtin_amdgcn_rcpf(1.0f + e);
    const float small = e * big;
    s = x >= 0.f ? big : small;
    rest = x >= 0.f ? small : big;
}

// s(x) alone, for a factor of a result that is stored in T.  EXACT: T is float32.  Otherwise the 2-instruction exponential, whose relative error
// |x| 2^-23 is far below a bf16 step.  Its overflow gives the right 0
template <bool EXACT>
__device__ __forceinline__ float seq_sigmoid(float x)
{
    return __builtin_amdgcn_rcpf(1.0f + (EXACT ? expf(-x) : __expf(-x)));
}

// s(x) for a factor of a float32 result, in both modes
template <bool EXACT>
__device__ __forceinline__ float seq_sigmoid_full(float x)
{
    return __builtin_amdgcn_rcpf(1.0f + seq_exp<EXACT, false>(-x));
}

// The counter-based generator of every dropout here: 32 bits for element `index` of the stream base = seed * SEQ_DROPOUT_STRIDE (a 64-bit
// finaliser of two odd multiplications; the stride is 2^64 over the golden ratio).
constexpr unsigned long long SEQ_DROPOUT_STRIDE = 0x9e3779b97f4a7c15ULL;
__device__ __forceinline__ unsigned seq_dropout_bits(unsigned long long base, unsigned long long index)
{
    unsigned long long x = base + index;
    x ^= x >> 33; x *= 0xff51afd7ed558ccdULL; x ^= x >> 33; x *= 0xc4ceb9fe1a85ec53ULL; x ^= x >> 33;
    return (unsigned)x;
}

}  // namespace
