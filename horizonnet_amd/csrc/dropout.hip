// Dropout with an optional residual sum, y = r + x keep / (1 - p), its mask never stored: element i is kept iff the generator's 32 bits at
// (seed, i) reach p 2^32.  The generator is the training step's own (seq_dropout_bits in seq_common.h), so dropout(x, p, 2 seed + 1 + l) draws
// the mask the engine draws behind LSTM layer l.  The gradient of x is the same pass over dy, that of r is dy itself.
//
// 2 tensors (3 with a residual) against 22 vector instructions an element, six of them the 32-bit products of the generator's two 64-bit ones, which
// take four times as long as others.  16.8 M elements in bf16: 17.4 us with a residual (101 MB, 5.8 TB/s: HBM), 15.0 us without (67 MB, 4.5 TB/s:
// the generator, about as long as the traffic); a large copy reaches 5.0.  The seed may lie on the device, where a captured
// step that adds to it draws a new mask on every replay.
#include "seq_common.h"

namespace {

constexpr int VEC = 4;      // elements a thread takes at once

template <typename T, bool RES>
__global__ __launch_bounds__(256) void seq_dropout_kernel(const T* __restrict__ x, const T* __restrict__ r, T* __restrict__ y, long n, unsigned thr,
                                                          float scale, unsigned long long seed, const unsigned long long* seed_dev)
{
    const unsigned long long base = (seed_dev ? *seed_dev : seed) * SEQ_DROPOUT_STRIDE;
    const long step = (long)gridDim.x * 256 * VEC;
    for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * VEC; i < n; i += step) {
        float a[VEC], b[VEC];
        if (i + VEC <= n) {
            seq_load<VEC>(x + i, a);
            if (RES) seq_load<VEC>(r + i, b);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float t = seq_dropout_bits(base, (unsigned long long)(i + k)) >= thr ? a[k] * scale : 0.f;
                a[k] = RES ? t + b[k] : t;
            }
            seq_store<VEC>(y + i, a);
        } else {
            for (long j = i; j < n; ++j) {
                float c[1], d[1];
                seq_load<1>(x + j, c);
                if (RES) seq_load<1>(r + j, d);
                const float t = seq_dropout_bits(base, (unsigned long long)j) >= thr ? c[0] * scale : 0.f;
                c[0] = RES ? t + d[0] : t;
                seq_store<1>(y + j, c);
            }
        }
    }
}

template <typename T>
void dropout_launch(const void* x, const void* r, void* y, long n, unsigned thr, float scale, unsigned long long seed, const void* seed_dev, hipStream_t s)
{
    long g = (n + 256L * VEC - 1) / (256L * VEC);
    if (g > 4096) g = 4096;
    const dim3 grid((unsigned)g);
    if (r)
        hipLaunchKernelGGL((seq_dropout_kernel<T, true>), grid, dim3(256), 0, s, (const T*)x, (const T*)r, (T*)y, n, thr, scale, seed,
                           (const unsigned long long*)seed_dev);
    else
        hipLaunchKernelGGL((seq_dropout_kernel<T, false>), grid, dim3(256), 0, s, (const T*)x, (const T*)nullptr, (T*)y, n, thr, scale, seed,
                           (const unsigned long long*)seed_dev);
}

}  // namespace

extern "C" int hn_dropout(const void* x, const void* residual, void* y, int64_t n, int dtype, float p, uint64_t seed, const void* seed_dev, void* stream)
{
    HN_REQUIRE(n >= 0 && p >= 0.f && p < 1.f, "hn_dropout: n=%ld, p=%g (0 <= p < 1)", (long)n, (double)p);
    HN_REQUIRE(dtype == SEQ_F32 || dtype == SEQ_BF16, "hn_dropout: dtype is 0 (float32) or 1 (bf16)");
    if (n == 0) return 0;
    HN_REQUIRE(x && y, "hn_dropout: null pointer");
    const unsigned thr = (unsigned)((double)p * 4294967296.0);
    const float scale = 1.0f / (1.0f - p);
    if (dtype == SEQ_BF16) dropout_launch<seq_bf16>(x, residual, y, n, thr, scale, seed, seed_dev, (hipStream_t)stream);
    else dropout_launch<float>(x, residual, y, n, thr, scale, seed, seed_dev, (hipStream_t)stream);
    HN_LAUNCH_CHECK();
    return 0;
}
