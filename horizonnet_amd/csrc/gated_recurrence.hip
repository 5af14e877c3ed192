// Gated linear recurrence over the sequence axis, forward, backward and single step:
//
//     a_t = s(f_t)     h_t = a_t h_{t-1} + (1 - a_t) v_t     y_t = s(o_t) h_t          (s: logistic function; every channel by itself)
//
// Unlike the LSTM layers (lstm*.hip), whose recurrent product forces one step after the other, the map of a run of steps on the state is
// affine, h -> A h + H, and two runs join as (A1, H1) then (A2, H2) = (A1 A2, A2 H1 + H2): time is parallel.
//
// A workgroup owns CL * VEC channels of one sequence (128 bytes of a row where the device is full, 16 to 64 in the forms for small sizes) and walks its
// time in tiles of 128 steps (256 where few workgroups have a short sequence, 32 or 64 where it is shorter): TL time lanes of L consecutive steps each,
// all of a tile's loads in flight at once and the next tile's behind them.  Each lane folds its steps to (A, H) in registers, a wave joins its lanes by
// shuffles, the waves meet in LDS once per tile, and every lane runs its steps again from registers with its true incoming state: each input is read from
// memory once.  What bounds it is HBM (4 tensors forward, 7 backward), with the two gates' exponentials and reciprocals close behind.  bf16, T 256, B 32,
// C 1024: 16.3 us forward (67 MB, 4.1 TB/s), 26.9 us backward (117 MB, 4.4 TB/s), where a large copy reaches 5.0.
//
// With few channels in flight (B * C small) and a long sequence the tiles of one sequence are spread over S workgroups ("spans"): a first
// launch folds every span to (A, H), and the second joins the spans before its own, in order, in front of its first tile.
//
// Backward, with dh_t the gradient of h_t and e_t = a_t dh_t what reaches h_{t-1}:
//     dh_t = dy_t s(o_t) + e_{t+1},   dv = (1 - a) dh,   df = dh (h_{t-1} - v) a (1 - a),   do = dy h s(o) (1 - s(o)),   dh_0 = e_1
// e is the same kind of affine scan, run from the end with the same a.  The states are not kept but for one per tile, 4 bytes a channel (of a bf16 tensor
// 1/64 at tiles of 128, 2 / T where T is one tile, written by the forward pass): the backward tile runs its steps again.
//
// All states, products and sums are float32; results are rounded once, at their store.  Time runs in processing order tau = 0 .. T-1,
// t = tau or T-1-tau (reverse); a step at or past its sequence's length is the identity (A = 1, H = 0), is not loaded, and stores 0.
#include "seq_common.h"

#include <type_traits>

namespace {

constexpr int TINY = 32, SMALL = 64, SHORT = 128, LONG = 256;    // steps of a tile = steps between two kept states

struct RecArgs {
    const void *f, *v, *o, *dy;           // o may be null: y = h
    long ft, fb, vt, vb, ot, ob, dt, db;  // element strides of the time and sequence axes (channels: 1)
    const float* h0;                      // [B][C] or null
    const float* dlast;                   // [B][C] or null
    const int* lengths;                   // [B] or null
    void *y, *df, *dv, *dout;             // contiguous [T][B][C]
    float* last;                          // [B][C] (backward: dh0)
    float* states;                        // [tiles][B][C] or null
    float* agg;                           // [S][2][B][C]: A, then H
    long T, B, C;                         // C: all channels
    int Cd;                               // channels of one direction
    int reverse;                          // of the first direction (a second one runs the other way)
    int groups;                           // channel groups of one direction
    int dirs;
    int S, span;                          // spans and tiles per span
};

template <int CW, int NW>
struct RecShared {
    float A[2][NW][CW], H[2][NW][CW], E[2][NW][CW];
};
__device__ __forceinline__ void rec_lds(const float* p, float (&x)[4])
{
    const f32x4 t = *reinterpret_cast<const f32x4*>(p);
    x[0] = t[0]; x[1] = t[1]; x[2] = t[2]; x[3] = t[3];
}
__device__ __forceinline__ void rec_lds(const float* p, float (&x)[1]) { x[0] = *p; }
__device__ __forceinline__ void rec_lds_put(float* p, const float (&x)[4]) { *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]}; }
__device__ __forceinline__ void rec_lds_put(float* p, const float (&x)[1]) { *p = x[0]; }

// Products of gates over a run of steps.  Such a product underflows, but it is 0 only where one of its gates is: an infinite state meets it, and has to
// stay infinite as it does step by step.  So a product has the smallest float32 above 0 for its floor wherever both factors are above 0 (bits of numbers
// >= 0 are ordered as integers, NaN last).  A finite state gets at most 2^-149 of itself in place of less.
__device__ __forceinline__ unsigned rec_bits(float x) { return __builtin_bit_cast(unsigned, x); }
__device__ __forceinline__ float rec_floor(float product, unsigned least)      // least: bits of the smallest factor
{
    return __builtin_bit_cast(float, max(rec_bits(product), min(least, 1u)));
}
__device__ __forceinline__ float rec_join(float a, float b) { return rec_floor(a * b, min(rec_bits(a), rec_bits(b))); }
// Whether a wave's joins need the floor: not while every lane's own product leaves the product of all the wave's time lanes above 2^-126 (T 256, B 32, C 1024
// forward: bf16 17.4 us without floors, 17.6 so, 18.1 with them everywhere; float32 27.1, 27.2, 28.3)
template <int CL, int VEC>
__device__ __forceinline__ bool rec_deep(const float (&A)[VEC])
{
    constexpr float LIMIT = CL == 8 ? 0x1p-15f : 0x1p-31f;
    static_assert(CL == 8 || CL == 16, "");
    float least = A[0];
#pragma unroll
    for (int k = 1; k < VEC; ++k) least = fminf(least, A[k]);
    return __any(least < LIMIT);
}
// the floor of a lane's own product, from its gates
template <int L, int VEC>
__device__ __forceinline__ void rec_lift(const float (&as)[L][VEC], float (&A)[VEC])
{
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        unsigned least = 1u;
#pragma unroll
        for (int i = 0; i < L; ++i) least = min(least, rec_bits(as[i][k]));
        A[k] = rec_floor(A[k], least);
    }
}

// x of the lane `by` lanes below / above; `none` past the wave's end
__device__ __forceinline__ float rec_up(float x, int by, int lane, float none)
{
    const float t = __shfl(x, lane - by, 64);
    return lane >= by ? t : none;
}
__device__ __forceinline__ float rec_down(float x, int by, int lane, float none)
{
    const float t = __shfl(x, lane + by, 64);
    return lane + by < 64 ? t : none;
}

// where a thread works: sequence b, channel c of all (bc = b C + c), span s; valid steps by processing time: first <= tau < end
struct RecPlace {
    long b, c, bc, first, end;
    int s;
    bool back, live, whole;               // whole: every channel of the workgroup exists
    int cl, tl;
};
template <int CL, int VEC>
__device__ __forceinline__ RecPlace rec_place(const RecArgs& p)
{
    RecPlace r;
    unsigned i = blockIdx.x;              // (the grid has fewer than 2^31 workgroups: 32-bit divisions)
    const unsigned per = (unsigned)p.groups, q = i / per, g = i - q * per, q2 = p.dirs == 2 ? q >> 1 : q;
    const int d = (int)(q - q2 * (unsigned)p.dirs);
    r.s = (int)(q2 / (unsigned)p.B);
    r.b = q2 - (unsigned)r.s * (unsigned)p.B;
    r.cl = threadIdx.x & (CL - 1);
    r.tl = threadIdx.x / CL;
    long cd = (long)g * CL * VEC + r.cl * VEC;
    r.back = (p.reverse != 0) != (d != 0);
    r.live = cd < p.Cd;
    if (r.live && cd > p.Cd - VEC) cd = p.Cd - VEC;   // the last lane's channels end with the row: those that it shares get the same bits twice
    r.whole = (long)(g + 1) * CL * VEC <= p.Cd;
    r.c = (long)d * p.Cd + cd;
    r.bc = r.b * p.C + r.c;
    long len = p.T;
    if (p.lengths) { len = p.lengths[r.b]; len = len < 0 ? 0 : len > p.T ? p.T : len; }
    r.first = r.back ? p.T - len : 0;
    r.end = r.back ? p.T : len;
    return r;
}

// the maps of spans s0 .. s1 - 1 (counted from agg by `dir`), joined in this order; the loads of four spans in flight at once
template <int VEC>
__device__ __forceinline__ void rec_spans_fold(const float* agg, long BC, long bc, bool live, int s0, int s1, int dir, float (&A)[VEC], float (&H)[VEC])
{
#pragma unroll
    for (int k = 0; k < VEC; ++k) { A[k] = 1.f; H[k] = 0.f; }
    if (!live) return;
    for (int s = s0; s < s1; s += 4) {
        float a[4][VEC], h[4][VEC];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const long at = 2L * dir * (s + q < s1 ? s + q : s1 - 1) * BC + bc;
            seq_load<VEC>(agg + at, a[q]);
            seq_load<VEC>(agg + at + BC, h[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (s + q < s1) {
                    H[k] = fmaf(a[q][k], H[k], h[q][k]);
                    A[k] = rec_join(A[k], a[q][k]);
                }
    }
}

// PASS 0: outputs; 1: fold every span to (A, H) only
template <typename T, int TILE, int CL, int VEC, int L, int PASS>
__global__ __launch_bounds__(TILE / L * CL, 2) void gated_recurrence_kernel(RecArgs p)
{
    constexpr int TL = TILE / L, NW = TL * CL / 64;
    constexpr bool EXACT = sizeof(T) == 4;
    typedef typename SeqRaw<T, VEC>::type Raw;
    __shared__ RecShared<CL * VEC, NW> sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const RecPlace w = rec_place<CL, VEC>(p);
    const long BC = p.B * p.C;
    const int tiles = (int)((p.T + TILE - 1) / TILE);

    float carry[VEC], all[VEC];                               // state in front of the tile; PASS 1: product of a so far
#pragma unroll
    for (int k = 0; k < VEC; ++k) { carry[k] = 0.f; all[k] = 1.f; }
    if (PASS == 0 && w.live) {
        if (p.h0) seq_load<VEC>(p.h0 + w.bc, carry);
    }
    if (PASS == 0 && w.s > 0) {                               // the spans in front of this one, in order: a run of them per time lane
        float A[VEC], H[VEC];
        const int run = (w.s + TL - 1) / TL, s0 = w.tl * run, s1 = s0 + run < w.s ? s0 + run : w.s;
        rec_spans_fold<VEC>(p.agg, BC, w.bc, w.live, s0, s1, 1, A, H);
#pragma unroll
        for (int st = CL; st < 64; st *= 2)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a1 = rec_up(A[k], st, lane, 1.f), h1 = rec_up(H[k], st, lane, 0.f);
                H[k] = fmaf(A[k], h1, H[k]);
                A[k] = rec_join(A[k], a1);
            }
        const int par = (w.s * p.span + 1) & 1;               // (the first tile takes the other buffer)
        if (lane >= 64 - CL) {
            rec_lds_put(&sh.A[par][wave][w.cl * VEC], A);
            rec_lds_put(&sh.H[par][wave][w.cl * VEC], H);
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NW; ++q) {
            rec_lds(&sh.A[par][q][w.cl * VEC], A);
            rec_lds(&sh.H[par][q][w.cl * VEC], H);
#pragma unroll
            for (int k = 0; k < VEC; ++k) carry[k] = fmaf(A[k], carry[k], H[k]);
        }
    }
    const bool gate = PASS == 0 && p.o != nullptr;
    const long sf = w.back ? -p.ft : p.ft, sv = w.back ? -p.vt : p.vt, so = w.back ? -p.ot : p.ot, sy = w.back ? -BC : BC;
    const long t0 = w.back ? p.T - 1 : 0;
    const T* f = (const T*)p.f + w.b * p.fb + w.c + t0 * p.ft;
    const T* v = (const T*)p.v + w.b * p.vb + w.c + t0 * p.vt;
    const T* o = gate ? (const T*)p.o + w.b * p.ob + w.c + t0 * p.ot : nullptr;
    T* y = (T*)p.y + w.bc + t0 * BC;

    const int k0 = w.s * p.span, k1 = k0 + p.span < tiles ? k0 + p.span : tiles;
    Raw fr[L], vr[L], nr[L];
    auto full = [&](int kt) { return w.whole && (long)kt * TILE >= w.first && (kt + 1L) * TILE <= w.end; };      // (the same for the whole workgroup)
    auto fetch = [&](int kt) {
        const long tau0 = (long)kt * TILE + w.tl * L;
        const T *pf = f + tau0 * sf, *pv = v + tau0 * sv, *po = o + tau0 * so;
        if (full(kt)) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                fr[i] = *reinterpret_cast<const Raw*>(pf + i * sf);
                vr[i] = *reinterpret_cast<const Raw*>(pv + i * sv);
            }
            if (gate)
#pragma unroll
                for (int i = 0; i < L; ++i) nr[i] = *reinterpret_cast<const Raw*>(po + i * so);
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i)
                if (w.live && tau0 + i >= w.first && tau0 + i < w.end) {
                    fr[i] = *reinterpret_cast<const Raw*>(pf + i * sf);
                    vr[i] = *reinterpret_cast<const Raw*>(pv + i * sv);
                    if (gate) nr[i] = *reinterpret_cast<const Raw*>(po + i * so);
                } else {
                    fr[i] = Raw{}; vr[i] = Raw{};
                    if (PASS == 0) nr[i] = Raw{};
                }
        }
    };
    if (k0 < k1) fetch(k0);
    for (int kt = k0; kt < k1; ++kt) {
        const int par = kt & 1;
        const long tau0 = (long)kt * TILE + w.tl * L;
        const bool inside = full(kt);
        if (PASS == 0 && p.states && w.live && w.tl == 0) seq_store<VEC>(p.states + (long)kt * BC + w.bc, carry);
        float as[L][VEC], bs[L][VEC], A[VEC], H[VEC];
        unsigned low[VEC];                                    // PASS 1: bits of the lane's smallest gate, at most 1 (PASS 0 has the gates at hand)
        Raw og[L];
#pragma unroll
        for (int k = 0; k < VEC; ++k) { A[k] = 1.f; H[k] = 0.f; low[k] = 1u; }
        auto fold = [&](auto masked) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                float x[VEC], z[VEC];
                seq_open(fr[i], x);
                seq_open(vr[i], z);
                if (PASS == 0) og[i] = nr[i];
                const bool on = !decltype(masked)::value || (w.live && tau0 + i >= w.first && tau0 + i < w.end);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    float a, rest;
                    seq_logistic<EXACT>(x[k], a, rest);
                    as[i][k] = on ? a : 1.f;
                    bs[i][k] = on ? rest * z[k] : 0.f;
                    A[k] *= as[i][k];
                    if (PASS == 1) low[k] = min(low[k], rec_bits(as[i][k]));
                    H[k] = fmaf(as[i][k], H[k], bs[i][k]);
                }
            }
        };
        if (inside) fold(std::false_type{}); else fold(std::true_type{});
        if (kt + 1 < k1) fetch(kt + 1);
        // inclusive join over the wave's time lanes, then the exclusive values of this lane
        float Ax[VEC], Hx[VEC];
        auto join = [&](auto deep) {
#pragma unroll
            for (int st = CL; st < 64; st *= 2)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float a1 = rec_up(A[k], st, lane, 1.f), h1 = rec_up(H[k], st, lane, 0.f);
                    H[k] = fmaf(A[k], h1, H[k]);
                    A[k] = decltype(deep)::value ? rec_join(A[k], a1) : A[k] * a1;
                }
        };
        if (rec_deep<CL>(A)) {
            if (PASS == 0) rec_lift(as, A);
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k) A[k] = rec_floor(A[k], low[k]);
            join(std::true_type{});
        } else {
            join(std::false_type{});
        }
        if (lane >= 64 - CL) {
            rec_lds_put(&sh.A[par][wave][w.cl * VEC], A);
            rec_lds_put(&sh.H[par][wave][w.cl * VEC], H);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) { Ax[k] = rec_up(A[k], CL, lane, 1.f); Hx[k] = rec_up(H[k], CL, lane, 0.f); }
        __syncthreads();                                      // (two buffers: a wave is at most one tile ahead of the slowest reader)
        float h[VEC];
#pragma unroll
        for (int q = 0; q < NW; ++q) {
            float a[VEC], b[VEC];
            rec_lds(&sh.A[par][q][w.cl * VEC], a);
            rec_lds(&sh.H[par][q][w.cl * VEC], b);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                h[k] = q == 0 || q == wave ? carry[k] : h[k];
                carry[k] = fmaf(a[k], carry[k], b[k]);
                if (PASS == 1) all[k] = rec_join(all[k], a[k]);
            }
        }
        if (PASS == 0) {
            T* py = y + tau0 * sy;
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[k] = fmaf(Ax[k], h[k], Hx[k]);
            auto emit = [&](auto masked) {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    float g[VEC], out[VEC];
                    if (gate) seq_open(og[i], g);
                    const bool on = !decltype(masked)::value || (tau0 + i >= w.first && tau0 + i < w.end);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        h[k] = fmaf(as[i][k], h[k], bs[i][k]);
                        out[k] = gate ? seq_sigmoid<EXACT>(g[k]) * h[k] : h[k];
                        out[k] = on ? out[k] : 0.f;
                    }
                    if (!decltype(masked)::value || (w.live && tau0 + i < p.T)) seq_store<VEC>(py + i * sy, out);
                }
            };
            if (inside) emit(std::false_type{}); else emit(std::true_type{});
        }
    }
    if (w.live && w.tl == 0) {
        if (PASS == 1) {
            seq_store<VEC>(p.agg + 2L * w.s * BC + w.bc, all);
            seq_store<VEC>(p.agg + (2L * w.s + 1) * BC + w.bc, carry);
        } else if (k1 == tiles) {
            seq_store<VEC>(p.last + w.bc, carry);
        }
    }
}

// PASS 0: gradients; 1: fold every span to the map of e over it
template <typename T, int TILE, int CL, int VEC, int L, int PASS>
__global__ __launch_bounds__(TILE / L * CL, 2) void gated_recurrence_bwd_kernel(RecArgs p)
{
    constexpr int TL = TILE / L, NW = TL * CL / 64;
    constexpr bool EXACT = sizeof(T) == 4;
    typedef typename SeqRaw<T, VEC>::type Raw;
    __shared__ RecShared<CL * VEC, NW> sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const RecPlace w = rec_place<CL, VEC>(p);
    const long BC = p.B * p.C;
    const int tiles = (int)((p.T + TILE - 1) / TILE);

    float carry[VEC], all[VEC];                               // e behind the tile
#pragma unroll
    for (int k = 0; k < VEC; ++k) { carry[k] = 0.f; all[k] = 1.f; }
    if (PASS == 0 && w.live) {
        if (p.dlast) seq_load<VEC>(p.dlast + w.bc, carry);
    }
    if (PASS == 0 && w.s + 1 < p.S) {                         // the spans behind this one, from the last: a run of them per time lane
        float A[VEC], E[VEC];
        const int n = p.S - 1 - w.s, run = (n + TL - 1) / TL, s0 = w.tl * run, s1 = s0 + run < n ? s0 + run : n;
        rec_spans_fold<VEC>(p.agg + 2 * (p.S - 1L) * BC, BC, w.bc, w.live, s0, s1, -1, A, E);
#pragma unroll
        for (int st = CL; st < 64; st *= 2)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a1 = rec_up(A[k], st, lane, 1.f), e1 = rec_up(E[k], st, lane, 0.f);
                E[k] = fmaf(A[k], e1, E[k]);
                A[k] = rec_join(A[k], a1);
            }
        const int last = w.s * p.span + p.span < tiles ? w.s * p.span + p.span - 1 : tiles - 1, par = (last + 1) & 1;
        if (lane >= 64 - CL) {
            rec_lds_put(&sh.A[par][wave][w.cl * VEC], A);
            rec_lds_put(&sh.E[par][wave][w.cl * VEC], E);
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NW; ++q) {
            rec_lds(&sh.A[par][q][w.cl * VEC], A);
            rec_lds(&sh.E[par][q][w.cl * VEC], E);
#pragma unroll
            for (int k = 0; k < VEC; ++k) carry[k] = fmaf(A[k], carry[k], E[k]);
        }
    }
    const bool gate = p.o != nullptr;
    const long sf = w.back ? -p.ft : p.ft, sv = w.back ? -p.vt : p.vt, so = w.back ? -p.ot : p.ot, sd = w.back ? -p.dt : p.dt, sy = w.back ? -BC : BC;
    const long t0 = w.back ? p.T - 1 : 0;
    const T* f = (const T*)p.f + w.b * p.fb + w.c + t0 * p.ft;
    const T* v = (const T*)p.v + w.b * p.vb + w.c + t0 * p.vt;
    const T* o = gate ? (const T*)p.o + w.b * p.ob + w.c + t0 * p.ot : nullptr;
    const T* dy = (const T*)p.dy + w.b * p.db + w.c + t0 * p.dt;

    const int k0 = w.s * p.span, k1 = k0 + p.span < tiles ? k0 + p.span : tiles;
    Raw fr[L], vr[L], og[L], gr[L];
    float hin[VEC];
    auto full = [&](int kt) { return w.whole && (long)kt * TILE >= w.first && (kt + 1L) * TILE <= w.end; };
    for (int kt = k1 - 1; kt >= k0; --kt) {
        const int par = kt & 1;
        const long tau0 = (long)kt * TILE + w.tl * L;
        const bool inside = full(kt);
        {
            const T *pf = f + tau0 * sf, *pv = v + tau0 * sv, *po = o + tau0 * so, *pd = dy + tau0 * sd;
            if (inside) {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    fr[i] = *reinterpret_cast<const Raw*>(pf + i * sf);
                    if (PASS == 0) vr[i] = *reinterpret_cast<const Raw*>(pv + i * sv);
                    gr[i] = *reinterpret_cast<const Raw*>(pd + i * sd);
                }
                if (gate)
#pragma unroll
                    for (int i = 0; i < L; ++i) og[i] = *reinterpret_cast<const Raw*>(po + i * so);
            } else {
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    fr[i] = Raw{}; og[i] = Raw{}; gr[i] = Raw{};
                    if (PASS == 0) vr[i] = Raw{};
                    if (w.live && tau0 + i >= w.first && tau0 + i < w.end) {
                        fr[i] = *reinterpret_cast<const Raw*>(pf + i * sf);
                        if (PASS == 0) vr[i] = *reinterpret_cast<const Raw*>(pv + i * sv);
                        if (gate) og[i] = *reinterpret_cast<const Raw*>(po + i * so);
                        gr[i] = *reinterpret_cast<const Raw*>(pd + i * sd);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) hin[k] = 0.f;
            if (PASS == 0 && w.live) seq_load<VEC>(p.states + (long)kt * BC + w.bc, hin);
        }
        // both scans at once: (A, H) from the front, (A, E) from the end.  gs = dy s(o), what h_t gets from y
        float A[VEC], H[VEC], E[VEC];
        float as[L][VEC], rs[L][VEC], gs[L][VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) { A[k] = 1.f; H[k] = 0.f; E[k] = 0.f; }
        auto fold = [&](auto masked) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                float x[VEC], z[VEC], g[VEC], q[VEC];
                seq_open(fr[i], x);
                if (PASS == 0) seq_open(vr[i], z);
                if (gate) seq_open(og[i], q);
                seq_open(gr[i], g);
                const bool on = !decltype(masked)::value || (w.live && tau0 + i >= w.first && tau0 + i < w.end);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    float a, rest;
                    seq_logistic<EXACT>(x[k], a, rest);
                    as[i][k] = on ? a : 1.f;
                    rs[i][k] = on ? rest : 0.f;
                    gs[i][k] = gate ? g[k] * seq_sigmoid_full<EXACT>(q[k]) : g[k];    // (0 where the step is not taken: g is)
                    A[k] *= as[i][k];
                    if (PASS == 0) H[k] = fmaf(as[i][k], H[k], rs[i][k] * z[k]);
                }
            }
        };
        if (inside) fold(std::false_type{}); else fold(std::true_type{});
#pragma unroll
        for (int i = L - 1; i >= 0; --i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) E[k] = as[i][k] * (gs[i][k] + E[k]);
        float Af[VEC], Ar[VEC], Hx[VEC], Ex[VEC];
        auto join = [&](auto deep) {
            constexpr bool DEEP = decltype(deep)::value;
#pragma unroll
            for (int k = 0; k < VEC; ++k) { Af[k] = A[k]; Ar[k] = A[k]; }
#pragma unroll
            for (int st = CL; st < 64; st *= 2)
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float a2 = rec_down(Ar[k], st, lane, 1.f), e2 = rec_down(E[k], st, lane, 0.f);
                    E[k] = fmaf(Ar[k], e2, E[k]);
                    Ar[k] = DEEP ? rec_join(Ar[k], a2) : Ar[k] * a2;
                    if (PASS == 0) {
                        const float a1 = rec_up(Af[k], st, lane, 1.f), h1 = rec_up(H[k], st, lane, 0.f);
                        H[k] = fmaf(Af[k], h1, H[k]);
                        Af[k] = DEEP ? rec_join(Af[k], a1) : Af[k] * a1;
                    }
                }
        };
        if (rec_deep<CL>(A)) {
            rec_lift(as, A);
            join(std::true_type{});
        } else {
            join(std::false_type{});
        }
        if (lane < CL) {                                      // the wave's first time lane: the whole wave from the end
            rec_lds_put(&sh.A[par][wave][w.cl * VEC], Ar);
            rec_lds_put(&sh.E[par][wave][w.cl * VEC], E);
        }
        if (PASS == 0 && lane >= 64 - CL) rec_lds_put(&sh.H[par][wave][w.cl * VEC], H);
        if (PASS == 0) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                Af[k] = rec_up(Af[k], CL, lane, 1.f); Hx[k] = rec_up(H[k], CL, lane, 0.f);
                Ar[k] = rec_down(Ar[k], CL, lane, 1.f); Ex[k] = rec_down(E[k], CL, lane, 0.f);
            }
        }
        __syncthreads();
        float h[VEC], e[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[k] = hin[k];
        if (PASS == 0)
            for (int q = 0; q < wave; ++q) {
                float a[VEC], b[VEC];
                rec_lds(&sh.A[par][q][w.cl * VEC], a);
                rec_lds(&sh.H[par][q][w.cl * VEC], b);
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[k] = fmaf(a[k], h[k], b[k]);
            }
#pragma unroll
        for (int q = NW - 1; q >= 0; --q) {
            float a[VEC], b[VEC];
            rec_lds(&sh.A[par][q][w.cl * VEC], a);
            rec_lds(&sh.E[par][q][w.cl * VEC], b);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                e[k] = q == NW - 1 || q == wave ? carry[k] : e[k];
                carry[k] = fmaf(a[k], carry[k], b[k]);
                if (PASS == 1) all[k] = rec_join(all[k], a[k]);
            }
        }
        if (PASS == 0) {
            float hs[L][VEC];                                 // the state in front of each step
#pragma unroll
            for (int k = 0; k < VEC; ++k) { h[k] = fmaf(Af[k], h[k], Hx[k]); e[k] = fmaf(Ar[k], e[k], Ex[k]); }
#pragma unroll
            for (int i = 0; i < L; ++i) {
                float z[VEC];
                seq_open(vr[i], z);
#pragma unroll
                for (int k = 0; k < VEC; ++k) { hs[i][k] = h[k]; h[k] = fmaf(as[i][k], h[k], rs[i][k] * z[k]); }
            }
            const long at = w.bc + t0 * BC + tau0 * sy;
            T *xf = (T*)p.df + at, *xv = (T*)p.dv + at, *xo = gate ? (T*)p.dout + at : nullptr;
            auto emit = [&](auto masked) {
#pragma unroll
                for (int i = L - 1; i >= 0; --i) {
                    float z[VEC], q[VEC], gf[VEC], gv[VEC], go[VEC];
                    seq_open(vr[i], z);
                    if (gate) seq_open(og[i], q);
                    const bool on = !decltype(masked)::value || (tau0 + i >= w.first && tau0 + i < w.end);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        const float dh = gs[i][k] + e[k];
                        e[k] = as[i][k] * dh;
                        gf[k] = on ? e[k] * rs[i][k] * (hs[i][k] - z[k]) : 0.f;
                        gv[k] = on ? dh * rs[i][k] : 0.f;
                        if (gate) go[k] = on ? gs[i][k] * h[k] * seq_sigmoid<EXACT>(-q[k]) : 0.f;
                        h[k] = hs[i][k];
                    }
                    if (!decltype(masked)::value || (w.live && tau0 + i < p.T)) {
                        seq_store<VEC>(xf + i * sy, gf);
                        seq_store<VEC>(xv + i * sy, gv);
                        if (gate) seq_store<VEC>(xo + i * sy, go);
                    }
                }
            };
            if (inside) emit(std::false_type{}); else emit(std::true_type{});
        }
    }
    if (w.live && w.tl == 0) {
        if (PASS == 1) {
            seq_store<VEC>(p.agg + 2L * w.s * BC + w.bc, all);
            seq_store<VEC>(p.agg + (2L * w.s + 1) * BC + w.bc, carry);
        } else if (k0 == 0 && p.last) {
            seq_store<VEC>(p.last + w.bc, carry);
        }
    }
}

// one step per sequence, state in place: serving
template <typename T, int VEC>
__global__ __launch_bounds__(256) void gated_recurrence_step_kernel(const T* f, const T* v, const T* o, long fb, long vb, long ob, float* state, T* y,
                                                                    long B, int C)
{
    constexpr bool EXACT = sizeof(T) == 4;
    const int per = C / VEC;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= B * per) return;
    const long b = i / per, c = (i - b * per) * VEC;
    float fx[VEC], vx[VEC], ox[VEC], h[VEC], out[VEC];
    seq_load<VEC>(f + b * fb + c, fx);
    seq_load<VEC>(v + b * vb + c, vx);
    if (o) seq_load<VEC>(o + b * ob + c, ox);
    seq_load<VEC>(state + b * C + c, h);
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        float a, rest;
        seq_logistic<EXACT>(fx[k], a, rest);
        h[k] = fmaf(a, h[k], rest * vx[k]);
        out[k] = o ? seq_sigmoid<EXACT>(ox[k]) * h[k] : h[k];
    }
    seq_store<VEC>(state + b * C + c, h);
    seq_store<VEC>(y + b * C + c, out);
}

// How a size is cut, by the sizes alone (the states and the workspace go by it).  rows: groups of 64 channels of all sequences.
//   tiles   128 steps, the last tile's loads beside this one's work; 256 by twice the threads for T 129 .. 512 while they leave the device half
//           empty (T 256, B 4, C 1024 bf16: 5.9 us against 14.6; B 1: 4.6 against 5.0); 32 or 64 for sequences no longer than that, whose other time
//           lanes would idle (float32 T 8, B 300, C 512: 15.1 us against 46.3; T 64, B 64, C 1024: 16.9 against 24.7)
//   spans   a lone workgroup walks its tiles one after the other (T 32768, B 1, C 512 float32 forward: 339 us whole, 76 cut); a second launch costs 5 us
//           and half as many reads again.  So longer sequences are cut while rows < 128, into as many spans as make 1024 workgroups (T 1201, B 1, C 512
//           float32: 11.0 us against 16.8; T 4096, B 8, C 512: 73 against 146, bf16 45 against 156), and not beyond (T 1024, B 32, C 512 float32,
//           rows 256: 47 us whole against 74 cut)
struct RecPlan {
    int tile, S, span;
};
RecPlan rec_plan(long T, long B, long C, int dirs)
{
    RecPlan p;
    const long rows = (C / dirs + 63) / 64 * dirs * B;
    p.tile = T <= TINY ? TINY : T <= SMALL ? SMALL : T > SHORT && T <= 2 * LONG && rows < 256 ? LONG : SHORT;
    const long tiles = (T + p.tile - 1) / p.tile;
    long s = T > 2 * LONG && rows < 128 ? 1024 / rows : 1;
    s = s > 128 ? 128 : s;
    if (s > tiles) s = tiles;
    p.span = s < 1 ? 1 : (int)((tiles + s - 1) / s);
    p.S = tiles < 1 ? 1 : (int)((tiles + p.span - 1) / p.span);
    return p;
}

template <typename T, int TILE, int CL, int VEC, int L, bool BWD>
int rec_launch(RecArgs p, const RecPlan& plan, hipStream_t s)
{
    p.groups = hn_cdiv(p.Cd, CL * VEC);
    p.S = plan.S;
    p.span = plan.span;
    const long n = (long)p.groups * p.dirs * p.B * p.S;
    SEQ_REQUIRE_GRID(n, TILE / L * CL, "hn_gated_recurrence");
    const dim3 grid((unsigned)n), block(TILE / L * CL);
    if constexpr (BWD) {
        if constexpr (TILE == SHORT)              // (the other tiles are never cut into spans)
            if (p.S > 1) hipLaunchKernelGGL((gated_recurrence_bwd_kernel<T, TILE, CL, VEC, L, 1>), grid, block, 0, s, p);
        hipLaunchKernelGGL((gated_recurrence_bwd_kernel<T, TILE, CL, VEC, L, 0>), grid, block, 0, s, p);
    } else {
        if constexpr (TILE == SHORT)
            if (p.S > 1) hipLaunchKernelGGL((gated_recurrence_kernel<T, TILE, CL, VEC, L, 1>), grid, block, 0, s, p);
        hipLaunchKernelGGL((gated_recurrence_kernel<T, TILE, CL, VEC, L, 0>), grid, block, 0, s, p);
    }
    HN_LAUNCH_CHECK();
    return 0;
}

// Four channels a lane and 128 bytes of a row per workgroup where the device is full: 8 steps a lane in bf16 (fewer joins an element: 17.4 us against
// 23.8 forward, 27.8 against 34.3 backward at T 256, B 32, C 1024), 4 in float32 (16 bytes a load: 29.5 against 36.1 forward, 45.3 against 51.9 backward
// at T 1201, B 7, C 333).  While all workgroups are resident at once, 8 waves a compute unit, the time is a lane's own chain, and less work a lane is
// faster: one channel a lane (T 256, B 1, C 1024, forward / backward: float32 4.6 / 6.0 us against 6.4 / 9.9, bf16 4.6 / 6.0 against 7.6 / 11.3; past
// that bound it loses: T 256, B 4 15.0 against 5.9), then, in bf16, half the steps (T 256, B 4: 5.9 / 8.6 against 7.9 / 12.0; past the bound, T 256, B 15:
// 15.1 against 8.9).  Rows of fewer than four channels take one a lane always.  (Times of a call in a captured graph, both launches where it has two.)
template <bool BWD, int TILE>
int rec_dispatch_tile(const RecArgs& p, const RecPlan& plan, int dtype, hipStream_t s)
{
    auto resident = [&](int channels) { return (double)hn_cdiv(p.Cd, channels) * p.dirs * p.B * plan.S * (TILE / 4 * 8) <= 256 * 512; };
    const bool bf16 = dtype == SEQ_BF16;
    if (p.Cd < 4 || resident(8)) return bf16 ? rec_launch<seq_bf16, TILE, 8, 1, 4, BWD>(p, plan, s) : rec_launch<float, TILE, 8, 1, 4, BWD>(p, plan, s);
    if (!bf16) return rec_launch<float, TILE, 8, 4, 4, BWD>(p, plan, s);
    return resident(32) ? rec_launch<seq_bf16, TILE, 8, 4, 4, BWD>(p, plan, s) : rec_launch<seq_bf16, TILE, 16, 4, 8, BWD>(p, plan, s);
}
template <bool BWD>
int rec_dispatch(const RecArgs& p, int dtype, hipStream_t s)
{
    const RecPlan plan = rec_plan(p.T, p.B, p.C, p.dirs);
    if (plan.tile == TINY) return rec_dispatch_tile<BWD, TINY>(p, plan, dtype, s);
    if (plan.tile == SMALL) return rec_dispatch_tile<BWD, SMALL>(p, plan, dtype, s);
    return plan.tile == LONG ? rec_dispatch_tile<BWD, LONG>(p, plan, dtype, s) : rec_dispatch_tile<BWD, SHORT>(p, plan, dtype, s);
}

int rec_check(long T, long B, long C, int dtype, int direction)
{
    HN_REQUIRE(T >= 0 && B >= 0 && C >= 0 && T < (1L << 31) && B < (1L << 31) && C < (1L << 30), "hn_gated_recurrence: bad sizes T=%ld B=%ld C=%ld", T, B, C);
    HN_REQUIRE(dtype == SEQ_F32 || dtype == SEQ_BF16, "hn_gated_recurrence: dtype is 0 (float32) or 1 (bf16)");
    HN_REQUIRE(direction >= 0 && direction <= 2, "hn_gated_recurrence: direction is 0 (forward), 1 (reverse) or 2 (both halves)");
    HN_REQUIRE(direction != 2 || C % 2 == 0, "hn_gated_recurrence: both directions need an even number of channels, got %ld", C);
    return 0;
}

}  // namespace

extern "C" size_t hn_gated_recurrence_states(int64_t T, int64_t B, int64_t C)
{
    return T <= 0 || B <= 0 || C <= 0 ? 0 : (size_t)((T + SHORT - 1) / SHORT) * B * C;
}

extern "C" size_t hn_gated_recurrence_workspace(int64_t T, int64_t B, int64_t C, int direction)
{
    if (T <= 0 || B <= 0 || C <= 0 || T >= (1L << 31) || B >= (1L << 31) || C >= (1L << 30) || (direction == 2 && C % 2)) return 0;      // (sizes that the calls refuse)
    const RecPlan p = rec_plan(T, B, C, direction == 2 ? 2 : 1);
    return p.S > 1 ? (size_t)p.S * 2 * B * C : 0;
}

extern "C" int hn_gated_recurrence(const void* f, int64_t f_t, int64_t f_b, const void* v, int64_t v_t, int64_t v_b, const void* o, int64_t o_t, int64_t o_b,
                                   const float* h0, const int* lengths, void* y, float* h_last, float* states, float* workspace, size_t workspace_floats,
                                   int64_t T, int64_t B, int64_t C, int dtype, int direction, void* stream)
{
    if (const int rc = rec_check(T, B, C, dtype, direction)) return rc;
    if (B == 0 || C == 0) return 0;
    HN_REQUIRE(h_last && (T == 0 || (f && v && y)), "hn_gated_recurrence: null pointer");
    HN_REQUIRE(workspace_floats >= hn_gated_recurrence_workspace(T, B, C, direction) && (workspace || workspace_floats == 0), "hn_gated_recurrence: workspace too small");
    RecArgs p = {};
    p.f = f; p.v = v; p.o = o;
    p.ft = f_t; p.fb = f_b; p.vt = v_t; p.vb = v_b; p.ot = o_t; p.ob = o_b;
    p.h0 = h0; p.lengths = lengths; p.y = y; p.last = h_last; p.states = states; p.agg = workspace;
    p.T = T; p.B = B; p.C = C;
    p.dirs = direction == 2 ? 2 : 1;
    p.Cd = (int)(C / p.dirs);
    p.reverse = direction == 1;
    return rec_dispatch<false>(p, dtype, (hipStream_t)stream);
}

extern "C" int hn_gated_recurrence_bwd(const void* f, int64_t f_t, int64_t f_b, const void* v, int64_t v_t, int64_t v_b, const void* o, int64_t o_t,
                                       int64_t o_b, const void* dy, int64_t dy_t, int64_t dy_b, const float* dh_last, const int* lengths, const float* states,
                                       void* df, void* dv, void* d_o, float* dh0, float* workspace, size_t workspace_floats, int64_t T, int64_t B, int64_t C,
                                       int dtype, int direction, void* stream)
{
    if (const int rc = rec_check(T, B, C, dtype, direction)) return rc;
    if (B == 0 || C == 0) return 0;
    HN_REQUIRE(T == 0 || (f && v && dy && states && df && dv && (!o || d_o)), "hn_gated_recurrence_bwd: null pointer");
    HN_REQUIRE(workspace_floats >= hn_gated_recurrence_workspace(T, B, C, direction) && (workspace || workspace_floats == 0),
               "hn_gated_recurrence_bwd: workspace too small");
    RecArgs p = {};
    p.f = f; p.v = v; p.o = o; p.dy = dy;
    p.ft = f_t; p.fb = f_b; p.vt = v_t; p.vb = v_b; p.ot = o_t; p.ob = o_b; p.dt = dy_t; p.db = dy_b;
    p.dlast = dh_last; p.lengths = lengths; p.df = df; p.dv = dv; p.dout = d_o; p.last = dh0; p.states = const_cast<float*>(states); p.agg = workspace;
    p.T = T; p.B = B; p.C = C;
    p.dirs = direction == 2 ? 2 : 1;
    p.Cd = (int)(C / p.dirs);
    p.reverse = direction == 1;
    return rec_dispatch<true>(p, dtype, (hipStream_t)stream);
}

extern "C" int hn_gated_recurrence_step(const void* f, int64_t f_b, const void* v, int64_t v_b, const void* o, int64_t o_b, float* state, void* y, int64_t B,
                                        int64_t C, int dtype, void* stream)
{
    if (const int rc = rec_check(1, B, C, dtype, 0)) return rc;
    if (B == 0 || C == 0) return 0;
    HN_REQUIRE(f && v && state && y, "hn_gated_recurrence_step: null pointer");
    const bool v4 = C % 4 == 0;           // (lanes that shared channels would update the state twice)
    const long n = B * (v4 ? C / 4 : C);
    SEQ_REQUIRE_GRID((n + 255) / 256, 256, "hn_gated_recurrence_step");
    const dim3 grid((unsigned)((n + 255) / 256));
    hipStream_t s = (hipStream_t)stream;
#define HN_STEP(T, VEC) \
    hipLaunchKernelGGL((gated_recurrence_step_kernel<T, VEC>), grid, dim3(256), 0, s, (const T*)f, (const T*)v, (const T*)o, f_b, v_b, o_b, state, (T*)y, B, (int)C)
    if (dtype == SEQ_BF16) { if (v4) HN_STEP(seq_bf16, 4); else HN_STEP(seq_bf16, 1); }
    else { if (v4) HN_STEP(float, 4); else HN_STEP(float, 1); }
#undef HN_STEP
    HN_LAUNCH_CHECK();
    return 0;
}
