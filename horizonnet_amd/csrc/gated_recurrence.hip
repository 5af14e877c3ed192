// Gated linear recurrence over the sequence axis, forward, backward and single step:
//
//     a_t = s(f_t)     h_t = a_t h_{t-1} + (1 - a_t) v_t     y_t = s(o_t) h_t          (s: logistic function; every channel by itself)
//
// Unlike the LSTM layers (lstm*.hip), whose recurrent product forces one step after the other, the map of a run of steps on the state is
// affine, h -> A h + H, and two runs join as (A1, H1) then (A2, H2) = (A1 A2, A2 H1 + H2): time is parallel.
//
// A workgroup owns CW = CL * VEC channels of one sequence and walks its time in tiles of 256 steps: TL time lanes of L consecutive steps
// each (TL * L = 256), all of a tile's loads in flight at once.  Each lane folds its steps to (A, H) in registers, a wave joins its lanes by
// shuffles, the waves meet in LDS once per tile, and every lane runs its steps again from registers with its true incoming state: each
// input is read from memory once.  What bounds it is HBM: 4 tensors forward, 7 backward, at ~30 flops per element.
//
// With few channels in flight (B * C small) and a long sequence the tiles of one sequence are spread over S workgroups ("spans"): a first
// launch folds every span to (A, H), and the second joins the spans before its own, in order, in front of its first tile.
//
// Backward, with dh_t the gradient of h_t and e_t = a_t dh_t what reaches h_{t-1}:
//     dh_t = dy_t s(o_t) + e_{t+1},   dv = (1 - a) dh,   df = dh (h_{t-1} - v) a (1 - a),   do = dy h s(o) (1 - s(o)),   dh_0 = e_1
// e is the same kind of affine scan, run from the end with the same a.  The states are not kept but for one per 256 steps (written by the
// forward pass, 1/64 of a bf16 tensor): the backward tile runs its 256 steps again.
//
// All states, products and sums are float32; results are rounded once, at their store.  Time runs in processing order tau = 0 .. T-1,
// t = tau or T-1-tau (reverse); a step at or past its sequence's length is the identity (A = 1, H = 0), is not loaded, and stores 0.
#include "seq_common.h"

namespace {

constexpr int TILE = 256;                 // steps of a tile = steps between two kept states

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

template <int CL, int VEC, int NW>
struct RecShared {
    float A[2][NW][CL * VEC], H[2][NW][CL * VEC], E[2][NW][CL * VEC];
};

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

struct RecPlace {
    long b, c0, s;
    int d;
};
template <int CW>
__device__ __forceinline__ RecPlace rec_place(const RecArgs& p)
{
    long i = blockIdx.x;
    RecPlace r;
    const long g = i % p.groups; i /= p.groups;
    r.d = (int)(i % p.dirs); i /= p.dirs;
    r.b = i % p.B;
    r.s = i / p.B;
    r.c0 = g * CW;
    return r;
}

// PASS 0: outputs; 1: fold every span to (A, H) only
template <typename T, int CL, int VEC, int L, int PASS>
__global__ __launch_bounds__(TILE / L * CL) void gated_recurrence_kernel(RecArgs p)
{
    constexpr int NT = TILE / L * CL, NW = NT / 64;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ RecShared<CL, VEC, NW> sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cl = lane & (CL - 1), tl = threadIdx.x / CL;
    const RecPlace w = rec_place<CL * VEC>(p);
    const bool back = (p.reverse != 0) != (w.d != 0);
    const long cd = w.c0 + cl * VEC;                          // channel within the direction
    const bool live = cd < p.Cd;                              // (VEC divides Cd)
    const long c = (long)w.d * p.Cd + cd;
    const long bc = w.b * p.C + c;
    long len = p.T;
    if (p.lengths) { len = p.lengths[w.b]; len = len < 0 ? 0 : len > p.T ? p.T : len; }

    float carry[VEC], all[VEC];                               // state in front of the tile; PASS 1: product of a so far
#pragma unroll
    for (int k = 0; k < VEC; ++k) { carry[k] = 0.f; all[k] = 1.f; }
    if (PASS == 0 && live) {
        if (p.h0) seq_load<VEC>(p.h0 + bc, carry);
        for (long s = 0; s < w.s; ++s) {                      // the spans in front of this one, in order
            float A[VEC], H[VEC];
            seq_load<VEC>(p.agg + (2 * s) * p.B * p.C + bc, A);
            seq_load<VEC>(p.agg + (2 * s + 1) * p.B * p.C + bc, H);
#pragma unroll
            for (int k = 0; k < VEC; ++k) carry[k] = fmaf(A[k], carry[k], H[k]);
        }
    }
    const T* f = (const T*)p.f + w.b * p.fb + c;
    const T* v = (const T*)p.v + w.b * p.vb + c;
    const T* o = p.o ? (const T*)p.o + w.b * p.ob + c : nullptr;
    T* y = (T*)p.y + bc;

    const long tiles = (p.T + TILE - 1) / TILE;
    const long k0 = w.s * p.span, k1 = k0 + p.span < tiles ? k0 + p.span : tiles;
    for (long kt = k0; kt < k1; ++kt) {
        const int par = (int)(kt & 1);
        const long tau0 = kt * TILE + tl * L;
        if (PASS == 0 && p.states && live && tl == 0) seq_store<VEC>(p.states + kt * p.B * p.C + bc, carry);
        float fr[L][VEC], vr[L][VEC], og[L][VEC];
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const long tau = tau0 + i, t = back ? p.T - 1 - tau : tau;
            if (live && tau < p.T && t < len) {
                seq_load<VEC>(f + t * p.ft, fr[i]);
                seq_load<VEC>(v + t * p.vt, vr[i]);
                if (PASS == 0 && o) seq_load<VEC>(o + t * p.ot, og[i]);
            }
        }
        float A[VEC], H[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) { A[k] = 1.f; H[k] = 0.f; }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const long tau = tau0 + i, t = back ? p.T - 1 - tau : tau;
            const bool on = live && tau < p.T && t < len;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                float a, rest;
                seq_logistic<EXACT>(fr[i][k], a, rest);
                a = on ? a : 1.f;
                const float b = on ? rest * vr[i][k] : 0.f;
                A[k] *= a;
                H[k] = fmaf(a, H[k], b);
                fr[i][k] = a;
                vr[i][k] = b;
            }
        }
        // inclusive join over the wave's time lanes, then the exclusive values of this lane
        float Ax[VEC], Hx[VEC];
#pragma unroll
        for (int st = CL; st < 64; st *= 2)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a1 = rec_up(A[k], st, lane, 1.f), h1 = rec_up(H[k], st, lane, 0.f);
                H[k] = fmaf(A[k], h1, H[k]);
                A[k] *= a1;
            }
#pragma unroll
        for (int k = 0; k < VEC; ++k) { Ax[k] = rec_up(A[k], CL, lane, 1.f); Hx[k] = rec_up(H[k], CL, lane, 0.f); }
        if (lane >= 64 - CL) {
            seq_store<VEC>(&sh.A[par][wave][cl * VEC], A);
            seq_store<VEC>(&sh.H[par][wave][cl * VEC], H);
        }
        __syncthreads();                                      // (two buffers: a wave is at most one tile ahead of the slowest reader)
        float h[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[k] = carry[k];
#pragma unroll
        for (int q = 0; q < NW; ++q) {
            float a[VEC], b[VEC];
            seq_load<VEC>(&sh.A[par][q][cl * VEC], a);
            seq_load<VEC>(&sh.H[par][q][cl * VEC], b);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                if (q == wave) h[k] = carry[k];
                carry[k] = fmaf(a[k], carry[k], b[k]);
                if (PASS == 1) all[k] *= a[k];
            }
        }
        if (PASS == 0) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[k] = fmaf(Ax[k], h[k], Hx[k]);
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const long tau = tau0 + i, t = back ? p.T - 1 - tau : tau;
                const bool on = t < len;
                float out[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    h[k] = fmaf(fr[i][k], h[k], vr[i][k]);
                    float g = 1.f, rest;
                    if (o) seq_logistic<EXACT>(og[i][k], g, rest);
                    out[k] = on ? g * h[k] : 0.f;
                }
                if (live && tau < p.T) seq_store<VEC>(y + t * p.B * p.C, out);
            }
        }
    }
    if (live && tl == 0) {
        if (PASS == 1) {
            seq_store<VEC>(p.agg + (2 * w.s) * p.B * p.C + bc, all);
            seq_store<VEC>(p.agg + (2 * w.s + 1) * p.B * p.C + bc, carry);
        } else if (k1 == tiles) {
            seq_store<VEC>(p.last + bc, carry);
        }
    }
}

// PASS 0: gradients; 1: fold every span to the map of e over it
template <typename T, int CL, int VEC, int L, int PASS>
__global__ __launch_bounds__(TILE / L * CL) void gated_recurrence_bwd_kernel(RecArgs p)
{
    constexpr int NT = TILE / L * CL, NW = NT / 64;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ RecShared<CL, VEC, NW> sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cl = lane & (CL - 1), tl = threadIdx.x / CL;
    const RecPlace w = rec_place<CL * VEC>(p);
    const bool back = (p.reverse != 0) != (w.d != 0);
    const long cd = w.c0 + cl * VEC;
    const bool live = cd < p.Cd;
    const long c = (long)w.d * p.Cd + cd;
    const long bc = w.b * p.C + c, BC = p.B * p.C;
    long len = p.T;
    if (p.lengths) { len = p.lengths[w.b]; len = len < 0 ? 0 : len > p.T ? p.T : len; }

    float carry[VEC], all[VEC];                               // e behind the tile
#pragma unroll
    for (int k = 0; k < VEC; ++k) { carry[k] = 0.f; all[k] = 1.f; }
    if (PASS == 0 && live) {
        if (p.dlast) seq_load<VEC>(p.dlast + bc, carry);
        for (long s = p.S - 1; s > w.s; --s) {
            float A[VEC], E[VEC];
            seq_load<VEC>(p.agg + (2 * s) * BC + bc, A);
            seq_load<VEC>(p.agg + (2 * s + 1) * BC + bc, E);
#pragma unroll
            for (int k = 0; k < VEC; ++k) carry[k] = fmaf(A[k], carry[k], E[k]);
        }
    }
    const T* f = (const T*)p.f + w.b * p.fb + c;
    const T* v = (const T*)p.v + w.b * p.vb + c;
    const T* o = p.o ? (const T*)p.o + w.b * p.ob + c : nullptr;
    const T* dy = (const T*)p.dy + w.b * p.db + c;

    const long tiles = (p.T + TILE - 1) / TILE;
    const long k0 = w.s * p.span, k1 = k0 + p.span < tiles ? k0 + p.span : tiles;
    for (long kt = k1 - 1; kt >= k0; --kt) {
        const int par = (int)(kt & 1);
        const long tau0 = kt * TILE + tl * L;
        float fr[L][VEC], vr[L][VEC], og[L][VEC], gr[L][VEC];
        float hin[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) hin[k] = 0.f;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const long tau = tau0 + i, t = back ? p.T - 1 - tau : tau;
            if (live && tau < p.T && t < len) {
                seq_load<VEC>(f + t * p.ft, fr[i]);
                if (PASS == 0) seq_load<VEC>(v + t * p.vt, vr[i]);
                if (o) seq_load<VEC>(o + t * p.ot, og[i]);
                seq_load<VEC>(dy + t * p.dt, gr[i]);
            }
        }
        if (PASS == 0 && live) seq_load<VEC>(p.states + kt * BC + bc, hin);
        // both scans at once: (A, H) from the front, (A, E) from the end
        float A[VEC], H[VEC], E[VEC];
        float rr[L][VEC];                                     // 1 - a
#pragma unroll
        for (int k = 0; k < VEC; ++k) { A[k] = 1.f; H[k] = 0.f; E[k] = 0.f; }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const long tau = tau0 + i, t = back ? p.T - 1 - tau : tau;
            const bool on = live && tau < p.T && t < len;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                float a, rest;
                seq_logistic<EXACT>(fr[i][k], a, rest);
                fr[i][k] = a = on ? a : 1.f;
                rr[i][k] = rest = on ? rest : 0.f;
                vr[i][k] = on && PASS == 0 ? vr[i][k] : 0.f;
                gr[i][k] = on ? gr[i][k] : 0.f;
                og[i][k] = on ? og[i][k] : 0.f;
                A[k] *= a;
                if (PASS == 0) H[k] = fmaf(a, H[k], rest * vr[i][k]);
            }
        }
#pragma unroll
        for (int i = L - 1; i >= 0; --i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                float s = 1.f, rest = 0.f;
                if (o) seq_logistic<EXACT>(og[i][k], s, rest);
                E[k] = fr[i][k] * fmaf(gr[i][k], s, E[k]);
            }
        float Af[VEC], Ar[VEC], Hx[VEC], Ex[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) { Af[k] = A[k]; Ar[k] = A[k]; }
#pragma unroll
        for (int st = CL; st < 64; st *= 2)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a2 = rec_down(Ar[k], st, lane, 1.f), e2 = rec_down(E[k], st, lane, 0.f);
                E[k] = fmaf(Ar[k], e2, E[k]);
                Ar[k] *= a2;
                if (PASS == 0) {
                    const float a1 = rec_up(Af[k], st, lane, 1.f), h1 = rec_up(H[k], st, lane, 0.f);
                    H[k] = fmaf(Af[k], h1, H[k]);
                    Af[k] *= a1;
                }
            }
        if (lane < CL) {                                      // the wave's first time lane: the whole wave from the end
            seq_store<VEC>(&sh.A[par][wave][cl * VEC], Ar);
            seq_store<VEC>(&sh.E[par][wave][cl * VEC], E);
        }
        if (PASS == 0 && lane >= 64 - CL) seq_store<VEC>(&sh.H[par][wave][cl * VEC], H);
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
#pragma unroll
        for (int q = 0; q < NW; ++q)
            if (PASS == 0 && q < wave) {
                float a[VEC], b[VEC];
                seq_load<VEC>(&sh.A[par][q][cl * VEC], a);
                seq_load<VEC>(&sh.H[par][q][cl * VEC], b);
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[k] = fmaf(a[k], h[k], b[k]);
            }
#pragma unroll
        for (int q = NW - 1; q >= 0; --q) {
            float a[VEC], b[VEC];
            seq_load<VEC>(&sh.A[par][q][cl * VEC], a);
            seq_load<VEC>(&sh.E[par][q][cl * VEC], b);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                if (q == wave) e[k] = carry[k];
                carry[k] = fmaf(a[k], carry[k], b[k]);
                if (PASS == 1) all[k] *= a[k];
            }
        }
        if (PASS == 0) {
            float hs[L][VEC];                                 // the state in front of each step
#pragma unroll
            for (int k = 0; k < VEC; ++k) { h[k] = fmaf(Af[k], h[k], Hx[k]); e[k] = fmaf(Ar[k], e[k], Ex[k]); }
#pragma unroll
            for (int i = 0; i < L; ++i)
#pragma unroll
                for (int k = 0; k < VEC; ++k) { hs[i][k] = h[k]; h[k] = fmaf(fr[i][k], h[k], rr[i][k] * vr[i][k]); }
#pragma unroll
            for (int i = L - 1; i >= 0; --i) {
                const long tau = tau0 + i, t = back ? p.T - 1 - tau : tau;
                const bool on = t < len;
                float xf[VEC], xv[VEC], xo[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    float s = 1.f, rest = 0.f;
                    if (o) seq_logistic<EXACT>(og[i][k], s, rest);
                    const float dh = fmaf(gr[i][k], s, e[k]);
                    e[k] = fr[i][k] * dh;
                    xf[k] = on ? e[k] * rr[i][k] * (hs[i][k] - vr[i][k]) : 0.f;
                    xv[k] = on ? dh * rr[i][k] : 0.f;
                    xo[k] = on ? gr[i][k] * h[k] * s * rest : 0.f;
                    h[k] = hs[i][k];
                }
                if (live && tau < p.T) {
                    const long at = t * BC + bc;
                    seq_store<VEC>((T*)p.df + at, xf);
                    seq_store<VEC>((T*)p.dv + at, xv);
                    if (o) seq_store<VEC>((T*)p.dout + at, xo);
                }
            }
        }
    }
    if (live && tl == 0) {
        if (PASS == 1) {
            seq_store<VEC>(p.agg + (2 * w.s) * BC + bc, all);
            seq_store<VEC>(p.agg + (2 * w.s + 1) * BC + bc, carry);
        } else if (k0 == 0 && p.last) {
            seq_store<VEC>(p.last + bc, carry);
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
        float a, rest, g = 1.f, unused;
        seq_logistic<EXACT>(fx[k], a, rest);
        if (o) seq_logistic<EXACT>(ox[k], g, unused);
        h[k] = fmaf(a, h[k], rest * vx[k]);
        out[k] = g * h[k];
    }
    seq_store<VEC>(state + b * C + c, h);
    seq_store<VEC>(y + b * C + c, out);
}

// spans: as many as bring the launch to 1024 workgroups, whole tiles each
void rec_spans(long T, long rows_groups, int& S, int& span)
{
    const long tiles = (T + TILE - 1) / TILE;
    long s = rows_groups > 0 ? 1024 / rows_groups : 1;
    s = s < 1 ? 1 : s > 64 ? 64 : s;
    if (s > tiles) s = tiles < 1 ? 1 : tiles;
    span = (int)((tiles + s - 1) / s);
    if (span < 1) span = 1;
    S = (int)((tiles + span - 1) / span);
    if (S < 1) S = 1;
}

bool rec_vec4(const RecArgs& p, int dtype, bool bwd)
{
    const size_t al = dtype == SEQ_F32 ? 16 : 8;
    auto ok = [&](const void* q, long st, long sb) { return q == nullptr || ((size_t)q % al == 0 && st % 4 == 0 && sb % 4 == 0); };
    auto okf = [&](const void* q) { return (size_t)q % 16 == 0; };
    return p.Cd % 4 == 0 && ok(p.f, p.ft, p.fb) && ok(p.v, p.vt, p.vb) && ok(p.o, p.ot, p.ob) && ok(p.y, 0, 0) && okf(p.h0) && okf(p.last) && okf(p.states) &&
           okf(p.agg) && okf(p.dlast) && (!bwd || (ok(p.dy, p.dt, p.db) && ok(p.df, 0, 0) && ok(p.dv, 0, 0) && ok(p.dout, 0, 0)));
}

template <typename T, int CL, int VEC, int L>
int rec_launch(RecArgs p, bool bwd, hipStream_t s)
{
    p.groups = hn_cdiv(p.Cd, CL * VEC);
    const long rows = (long)p.groups * p.dirs * p.B;
    rec_spans(p.T, rows, p.S, p.span);
    HN_REQUIRE(rows * p.S <= 0x7fffffffL, "hn_gated_recurrence: too many sequences x channels");
    const dim3 grid((unsigned)(rows * p.S)), block(TILE / L * CL);
    if (p.S > 1) {
        if (bwd) hipLaunchKernelGGL((gated_recurrence_bwd_kernel<T, CL, VEC, L, 1>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((gated_recurrence_kernel<T, CL, VEC, L, 1>), grid, block, 0, s, p);
        HN_LAUNCH_CHECK();
    }
    if (bwd) hipLaunchKernelGGL((gated_recurrence_bwd_kernel<T, CL, VEC, L, 0>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((gated_recurrence_kernel<T, CL, VEC, L, 0>), grid, block, 0, s, p);
    HN_LAUNCH_CHECK();
    return 0;
}

int rec_dispatch(const RecArgs& p, int dtype, bool bwd, hipStream_t s)
{
    const bool v4 = rec_vec4(p, dtype, bwd);
    if (dtype == SEQ_BF16) return v4 ? rec_launch<seq_bf16, 8, 4, 4>(p, bwd, s) : rec_launch<seq_bf16, 32, 1, 16>(p, bwd, s);
    return v4 ? rec_launch<float, 8, 4, 4>(p, bwd, s) : rec_launch<float, 32, 1, 16>(p, bwd, s);
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
    return T <= 0 || B <= 0 || C <= 0 ? 0 : (size_t)((T + TILE - 1) / TILE) * B * C;
}

// (the largest number of spans any variant of this size takes)
extern "C" size_t hn_gated_recurrence_workspace(int64_t T, int64_t B, int64_t C)
{
    if (T <= TILE || B <= 0 || C <= 0) return 0;
    const long tiles = (T + TILE - 1) / TILE;
    return (size_t)(tiles < 64 ? tiles : 64) * 2 * B * C;
}

extern "C" int hn_gated_recurrence(const void* f, int64_t f_t, int64_t f_b, const void* v, int64_t v_t, int64_t v_b, const void* o, int64_t o_t, int64_t o_b,
                                   const float* h0, const int* lengths, void* y, float* h_last, float* states, float* workspace, size_t workspace_floats,
                                   int64_t T, int64_t B, int64_t C, int dtype, int direction, void* stream)
{
    if (const int rc = rec_check(T, B, C, dtype, direction)) return rc;
    if (B == 0 || C == 0) return 0;
    HN_REQUIRE(h_last && (T == 0 || (f && v && y)), "hn_gated_recurrence: null pointer");
    HN_REQUIRE(workspace_floats >= hn_gated_recurrence_workspace(T, B, C) && (workspace || workspace_floats == 0), "hn_gated_recurrence: workspace too small");
    RecArgs p = {};
    p.f = f; p.v = v; p.o = o;
    p.ft = f_t; p.fb = f_b; p.vt = v_t; p.vb = v_b; p.ot = o_t; p.ob = o_b;
    p.h0 = h0; p.lengths = lengths; p.y = y; p.last = h_last; p.states = states; p.agg = workspace;
    p.T = T; p.B = B; p.C = C;
    p.dirs = direction == 2 ? 2 : 1;
    p.Cd = (int)(C / p.dirs);
    p.reverse = direction == 1;
    return rec_dispatch(p, dtype, false, (hipStream_t)stream);
}

extern "C" int hn_gated_recurrence_bwd(const void* f, int64_t f_t, int64_t f_b, const void* v, int64_t v_t, int64_t v_b, const void* o, int64_t o_t,
                                       int64_t o_b, const void* dy, int64_t dy_t, int64_t dy_b, const float* dh_last, const int* lengths, const float* states,
                                       void* df, void* dv, void* d_o, float* dh0, float* workspace, size_t workspace_floats, int64_t T, int64_t B, int64_t C,
                                       int dtype, int direction, void* stream)
{
    if (const int rc = rec_check(T, B, C, dtype, direction)) return rc;
    if (B == 0 || C == 0) return 0;
    HN_REQUIRE(T == 0 || (f && v && dy && states && df && dv && (!o || d_o)), "hn_gated_recurrence_bwd: null pointer");
    HN_REQUIRE(workspace_floats >= hn_gated_recurrence_workspace(T, B, C) && (workspace || workspace_floats == 0),
               "hn_gated_recurrence_bwd: workspace too small");
    RecArgs p = {};
    p.f = f; p.v = v; p.o = o; p.dy = dy;
    p.ft = f_t; p.fb = f_b; p.vt = v_t; p.vb = v_b; p.ot = o_t; p.ob = o_b; p.dt = dy_t; p.db = dy_b;
    p.dlast = dh_last; p.lengths = lengths; p.df = df; p.dv = dv; p.dout = d_o; p.last = dh0; p.states = const_cast<float*>(states); p.agg = workspace;
    p.T = T; p.B = B; p.C = C;
    p.dirs = direction == 2 ? 2 : 1;
    p.Cd = (int)(C / p.dirs);
    p.reverse = direction == 1;
    return rec_dispatch(p, dtype, true, (hipStream_t)stream);
}

extern "C" int hn_gated_recurrence_step(const void* f, int64_t f_b, const void* v, int64_t v_b, const void* o, int64_t o_b, float* state, void* y, int64_t B,
                                        int64_t C, int dtype, void* stream)
{
    if (const int rc = rec_check(1, B, C, dtype, 0)) return rc;
    if (B == 0 || C == 0) return 0;
    HN_REQUIRE(f && v && state && y, "hn_gated_recurrence_step: null pointer");
    const size_t al = dtype == SEQ_F32 ? 16 : 8;
    auto ok = [&](const void* q, int64_t sb) { return q == nullptr || ((size_t)q % al == 0 && sb % 4 == 0); };
    const bool v4 = C % 4 == 0 && ok(f, f_b) && ok(v, v_b) && ok(o, o_b) && ok(y, 0) && (size_t)state % 16 == 0;
    const long n = B * (v4 ? C / 4 : C);
    HN_REQUIRE((n + 255) / 256 <= 0x7fffffffL, "hn_gated_recurrence_step: too many sequences x channels");
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
