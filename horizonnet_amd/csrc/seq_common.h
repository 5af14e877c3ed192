// Shared by the sequence operators (gated_recurrence.hip, gated_linear*.hip, dropout.hip): element types, vector access, logistic pair.
#pragma once
#include "hn_common.h"

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

template <int VEC>
__device__ __forceinline__ void seq_load(const float* p, float (&x)[VEC])
{
    if constexpr (VEC == 4) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(p);
        x[0] = t[0]; x[1] = t[1]; x[2] = t[2]; x[3] = t[3];
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = p[k];
    }
}
template <int VEC>
__device__ __forceinline__ void seq_load(const seq_bf16* p, float (&x)[VEC])
{
    if constexpr (VEC == 4) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        x[0] = __builtin_bit_cast(float, t.x << 16); x[1] = __builtin_bit_cast(float, t.x & 0xffff0000u);
        x[2] = __builtin_bit_cast(float, t.y << 16); x[3] = __builtin_bit_cast(float, t.y & 0xffff0000u);
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = seq_from_bf16(p[k]);
    }
}
template <int VEC>
__device__ __forceinline__ void seq_store(float* p, const float (&x)[VEC])
{
    if constexpr (VEC == 4) {
        *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) p[k] = x[k];
    }
}
template <int VEC>
__device__ __forceinline__ void seq_store(seq_bf16* p, const float (&x)[VEC])
{
    if constexpr (VEC == 4) {
        *reinterpret_cast<uint2*>(p) = make_uint2(seq_pack2(x[0], x[1]), seq_pack2(x[2], x[3]));
    } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) p[k] = (seq_bf16)(seq_pack2(x[k], 0.f) & 0xffffu);
    }
}

// s(x) and 1 - s(x) = s(-x) from ONE exponential of -|x|: neither is formed by a subtraction from 1, so the small one keeps its relative
// precision (a long memory is a small 1 - a).  EXACT: float32 outputs; otherwise the 2-instruction exponential, whose relative error
// |x| 2^-23 is far below a bf16 step.
template <bool EXACT>
__device__ __forceinline__ void seq_logistic(float x, float& s, float& rest)
{
    const float e = EXACT ? expf(-fabsf(x)) : __expf(-fabsf(x));
    const float big = __builtin_amdgcn_rcpf(1.0f + e);
    const float small = e * big;
    s = x >= 0.f ? big : small;
    rest = x >= 0.f ? small : big;
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
