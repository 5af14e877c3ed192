// Large bf16 sizes of the gated linear block: 256 x 256 tiles, 8 waves, the ping-pong schedule of conv_igemm_bf16_pp.hip (its header explains
// the phases and waits in full; tools/pp_schedule_model.py checks them) with plain matrix operands instead of convolution taps.
//
// Two wave groups run the same four phases of a 64-deep chunk one barrier apart: while one issues the 8 MFMAs of a phase (4 row tiles x 2 k
// steps of v_mfma_f32_32x32x16_bf16), its SIMD partner reads the next phase's fragments and issues LDS-DMA.  A chunk lies in four 16 KiB
// regions A0 | A1 (rows of group 0 / 1) and B0 | B1 (left / right 32 columns of every wave's 64).  The DMA queue stays in flight across the
// raw barriers and is counted by hand (two pieces per wave and region, s_waitcnt vmcnt(6) twice a chunk).
//
//   gate      A = x, B0 = gate rows, B1 = up rows of the same 128 hidden units: a lane's two accumulators hold g and u of the same element, so
//             the activation and the product (or dg and du) follow in registers.  A persistent workgroup's loader runs into its next tile.
//   products  dx: A = dg | du with k contiguous; dw: A = the same buffer with k along its rows; B = the weights / x with k along the rows.  An
//             operand with k along its rows (KR) lies in LDS as [64 k][128] and is read by the transposing LDS read.  All of them are ONE
//             launch, a workgroup per tile, longest k first, so that unequal jobs still fill the device.
//
// Bound by the matrix pipe and, between a tile's last product and the next one's first, by the epilogue that all compute units reach at about the
// same time.  M 8192, K 1024, F 4096: gate 140 us forward (0.98 PFLOP/s), 177 us backward (dy read, dg | du written), the products 257 - 280 us (1.07 -
// 0.98 PFLOP/s, by card); M 16384 forward 248 us (1.11).  A large library product reaches 1.26.
//
// KR regions: 32-byte block u of row k sits at u ^ (2 (k & 3)): the 4 rows x 2 blocks that 32 lanes read together lie in all 64 banks once.
#include "gated_linear.h"
#include "conv_bf16_args.h"
#include "conv_bf16_pp.h"

namespace {

constexpr int GP_BUF = 65536, GP_REGION = 16384, GP_BOFF = 32768, GP_SLAB = 131072, GP_LDS = 163840;

struct GpTile {                           // a tile: where it starts, its k axis
    long i0, j0;
    int chunks;
};

// One operand's loader: two regions of 128 rows (or columns), this thread's two pieces of each.  Both sources of a longer k axis have the
// same stride; the two regions may lie in two matrices.
struct GpCursor {
    const char* at[2];                    // the current chunk of region 0 / 1
    const char* second;                   // the second source's first chunk
    long step;                            // bytes from chunk to chunk
    unsigned off[4], cur[4];              // [2 region + pass]: byte offset or OOB; cur: with what lies behind the k axis's end taken off
    bool mine[2];                         // [pass]: whether this thread's k's lie before the end in a last chunk
    int chunk, per, left;                 // chunk within the source, chunks of a source, chunks left of the tile

    __device__ __forceinline__ void mask()
    {
        const bool last = chunk == per - 1;
#pragma unroll
        for (int k = 0; k < 4; ++k) cur[k] = !last || mine[k & 1] ? off[k] : OOB;
    }
    __device__ __forceinline__ void dead()
    {
#pragma unroll
        for (int k = 0; k < 4; ++k) off[k] = cur[k] = OOB;
        left = 0x7fffffff;
        per = 0x7fffffff;
        step = 0;
    }
    // to the tile's next chunk; false: there is none
    __device__ __forceinline__ bool next()
    {
        if (--left == 0) return false;
        if (++chunk == per) {
            chunk = 0;
            at[0] = at[1] = second;
        } else {
            at[0] += step;
            at[1] += step;
        }
        mask();
        return true;
    }
};

__device__ __forceinline__ void gp_issue(const GpCursor& c, unsigned dst, int reg)
{
    const u32x4 r = pp_rsrc(c.at[reg]);
#pragma unroll
    for (int ps = 0; ps < 2; ++ps) pp_dma16<0>(r, dst + ps * 8192, reg ? c.cur[2 + ps] : c.cur[ps], 0u);
}

// The chunk stream of one workgroup.  W: what differs -- tile(vb, t) decodes tile number vb (false: none), setup_a / setup_b aim a cursor at
// it, finish(t, acc) takes the accumulators.
template <bool AKR, bool BKR, class W>
__device__ __forceinline__ void gp_run(W& w, char* smem)
{
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = wave >> 2, wn = wave & 3;
    const int fr = lane & 31, half = lane >> 5, fswz = (fr >> 1) & 7;
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;

    GpCursor ca, cb;
    GpTile t;
    int avb = (int)blockIdx.x, bvb = avb, vb = avb;
    if (!w.tile(vb, t)) return;
    w.setup_a(avb, ca);
    w.setup_b(bvb, cb);
    auto advance_a = [&]() {
        if (!ca.next()) {
            avb += (int)gridDim.x;
            if (!w.setup_a(avb, ca)) ca.dead();
        }
    };
    auto advance_b = [&]() {
        if (!cb.next()) {
            bvb += (int)gridDim.x;
            if (!w.setup_b(bvb, cb)) cb.dead();
        }
    };
    auto issue_a = [&](int buf, int reg) { gp_issue(ca, lds0 + (unsigned)(buf * GP_BUF + reg * GP_REGION + wave * 1024), reg); };
    auto issue_b = [&](int buf, int reg) { gp_issue(cb, lds0 + (unsigned)(buf * GP_BUF + GP_BOFF + reg * GP_REGION + wave * 1024), reg); };

    // fragment addresses inside the current buffer
    unsigned rd_a[4], rd_b[4];
    const int r4 = (lane >> 2) & 3, b16 = (lane >> 4) & 1;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const unsigned ks = (unsigned)(((2 * s + half) ^ fswz) * 16);
        const unsigned kr = (unsigned)((8 * half + r4) * 256 + b16 * 32 + (lane & 3) * 8);
        rd_a[s] = (unsigned)(g * GP_REGION) + (AKR ? kr + (unsigned)((s ^ r4) * 64) : (unsigned)(fr * ROWB) + ks);      // KR: s is the row tile
        rd_b[s] = (unsigned)GP_BOFF + (BKR ? kr + (unsigned)((wn ^ r4) * 64) : (unsigned)((32 * wn + fr) * ROWB) + ks);
    }
    u32x4 fa[4][2], fb[2];
    auto tr = [&](unsigned at) {          // 8 k's of this lane's column
        u32x4 v;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) gl_s16x4*)(smem + at + q * 1024)));
            v[2 * q] = x.x;
            v[2 * q + 1] = x.y;
        }
        return v;
    };
    auto read_a = [&](int h) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int sh = 0; sh < 2; ++sh) {
                if constexpr (AKR) fa[i][sh] = tr(rd_a[i] + (2 * h + sh) * 4096);
                else fa[i][sh] = *reinterpret_cast<const u32x4*>(smem + rd_a[2 * h + sh] + i * 32 * ROWB);
            }
    };
    auto read_b = [&](int j, int h) {
#pragma unroll
        for (int sh = 0; sh < 2; ++sh) {
            if constexpr (BKR) fb[sh] = tr(rd_b[0] + (2 * h + sh) * 4096 + j * GP_REGION);
            else fb[sh] = *reinterpret_cast<const u32x4*>(smem + rd_b[2 * h + sh] + j * GP_REGION);
        }
    };
    f32x16 acc[4][2];
    auto clear = [&](float c0, float c1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) { acc[i][0][r] = c0; acc[i][1][r] = c1; }
    };
    auto mm = [&](int j) {
#pragma unroll
        for (int sh = 0; sh < 2; ++sh)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fa[i][sh]), __builtin_bit_cast(bf16x8, fb[sh]), acc[i][j], 0, 0, 0);
    };
    float c0 = 0.f, c1 = 0.f;             // what the sums of the lane's two columns start from: the biases
    w.start(t, c0, c1);
    clear(c0, c1);

    // chunk 0 whole, the A regions of chunk 1 (its B regions follow in phases 1 and 2 of chunk 0)
    issue_a(0, 0); issue_a(0, 1); issue_b(0, 0); issue_b(0, 1);
    advance_a();
    advance_b();
    issue_a(1, 0); issue_a(1, 1);
    asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    pp_bar_raw();
    if (g == 1) pp_bar_raw();

    int buf = 0, ckc = 0;
    while (true) {
        read_a(0);                        // phase 1: columns j 0, k half 0
        read_b(0, 0);
        issue_b(buf ^ 1, 0);
        asm volatile("s_waitcnt vmcnt(6)" ::: "memory");      // B1 of this chunk has landed
        pp_bar_raw();
        mm(0);
        pp_bar_raw();
        read_b(1, 0);                     // phase 2: j 1, k half 0
        issue_b(buf ^ 1, 1);
        advance_a();
        pp_bar_raw();
        mm(1);
        pp_bar_raw();
        read_a(1);                        // phase 3: j 0, k half 1: last reads of A0, A1, B0
        read_b(0, 1);
        advance_b();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        pp_bar_raw();
        mm(0);
        pp_bar_raw();
        read_b(1, 1);                     // phase 4: j 1, k half 1
        issue_a(buf, 0);                  // the chunk after next, into the regions read last in phase 3
        issue_a(buf, 1);
        asm volatile("s_waitcnt vmcnt(6)" ::: "memory");      // A0, A1, B0 of the next chunk have landed
        pp_bar_raw();
        mm(1);
        pp_bar_raw();
        buf ^= 1;
#pragma unroll
        for (int s = 0; s < 4; ++s) { rd_a[s] ^= (unsigned)GP_BUF; rd_b[s] ^= (unsigned)GP_BUF; }
        if (++ckc == t.chunks) {
            ckc = 0;
            if (g == 0) pp_bar_raw();         // the groups meet for the epilogue ...
            w.finish(t, acc, reinterpret_cast<float*>(smem + GP_SLAB + wave * 4096));
            vb += (int)gridDim.x;
            if (!w.tile(vb, t)) break;
            w.start(t, c0, c1);
            clear(c0, c1);
            if (g == 1) pp_bar_raw();         // ... and part again behind it
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // surplus pieces (out of range: zeros)
}

// aims a cursor at rows with k contiguous: region reg holds rows row(reg, c), c < 128, of matrix reg with row stride ld[reg]
template <class Row>
__device__ __forceinline__ void gp_aim_kc(GpCursor& c, long left_rows, const long (&ld)[2], long K, int chunks, Row row)
{
    const int lrow = threadIdx.x >> 3, lcol = (threadIdx.x & 7) ^ ((lrow >> 1) & 7);
    c.step = 128;
    c.per = (int)((K + 63) >> 6);
    c.chunk = 0;
    c.left = chunks;
    c.mine[0] = c.mine[1] = lcol * 8 < (int)(K - 64L * (c.per - 1));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = row(k >> 1, lrow + 64 * (k & 1));
        c.off[k] = r < left_rows ? (unsigned)r * (unsigned)ld[k >> 1] * 2u + (unsigned)lcol * 16u : OOB;
    }
    c.mask();
}
// aims a cursor at [K][n], k along the rows: region reg holds columns col(reg, c), c < 128 (16-byte units stay whole)
template <class Col>
__device__ __forceinline__ void gp_aim_kr(GpCursor& c, long left_cols, long ld, long K, int chunks, Col col)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, unit = (lane & 15) ^ (4 * (lane >> 4));
    c.step = 128L * ld;
    c.per = (int)((K + 63) >> 6);
    c.chunk = 0;
    c.left = chunks;
    const int tail = (int)(K - 64L * (c.per - 1));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int kr = 4 * ((k & 1) * 8 + wave) + (lane >> 4), x = col(k >> 1, unit * 8);
        if (k < 2) c.mine[k] = kr < tail;
        c.off[k] = x < left_cols ? (unsigned)kr * (unsigned)ld * 2u + (unsigned)x * 2u : OOB;
    }
    c.mask();
}

// 16 rows of the wave's accumulators (row tile i, upper or lower half) through its LDS slab: float32 rows of 64, 4-float blocks exchanged by row
__device__ __forceinline__ void gp_slab_put(float* slab, const f32x16 (&acc)[4][2], int i, int hb)
{
    const int lane = threadIdx.x & 63, fr = lane & 31, half = lane >> 5;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int rr = 0; rr < 8; ++rr) {
            const int row = (rr & 3) + 8 * (rr >> 2) + 4 * half, blk = (8 * j + (fr >> 2)) ^ (rr & 3);
            slab[row * 64 + blk * 4 + (fr & 3)] = acc[i][j][8 * hb + rr];
        }
}
__device__ __forceinline__ void gp_slab_get(const float* slab, int row, int blk, float (&x)[8])
{
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(slab + row * 64 + ((blk + h) ^ (row & 3)) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * h + e] = t[e];
    }
}

// ---- both projections ----
template <bool BWD, int ACT>
struct GpGate {
    const GlArgs& p;
    int nt, total, chunks;
    __device__ __forceinline__ bool tile(int vb, GpTile& t) const
    {
        if (vb >= total) return false;
        long row, col;
        gl_tile_at(vb, total / nt, nt, row, col);
        t.i0 = 256L * __builtin_amdgcn_readfirstlane((int)row);
        t.j0 = 128L * __builtin_amdgcn_readfirstlane((int)col);
        t.chunks = chunks;
        return true;
    }
    __device__ __forceinline__ bool setup_a(int vb, GpCursor& c) const
    {
        GpTile t;
        if (!tile(vb, t)) return false;
        c.at[0] = c.at[1] = c.second = (const char*)p.x.p[0] + t.i0 * p.x.ld[0] * 2;
        gp_aim_kc(c, p.M - t.i0, p.x.ld, p.K, chunks, [](int reg, int r) { return 128 * reg + r; });
        return true;
    }
    __device__ __forceinline__ bool setup_b(int vb, GpCursor& c) const
    {
        GpTile t;
        if (!tile(vb, t)) return false;
        c.at[0] = c.second = (const char*)p.w.p[0] + t.j0 * p.w.ld[0] * 2;
        c.at[1] = (const char*)p.w.p[1] + t.j0 * p.w.ld[1] * 2;
        gp_aim_kc(c, p.F - t.j0, p.w.ld, p.K, chunks, [](int, int r) { return r; });
        return true;
    }
    __device__ __forceinline__ void start(const GpTile& t, float& c0, float& c1) const
    {
        const long f = t.j0 + 32 * (threadIdx.x >> 6 & 3) + (threadIdx.x & 31);
        if (p.bg) c0 = f < p.F ? gl_ld((const seq_bf16*)p.bg + f) : 0.f;
        if (p.bu) c1 = f < p.F ? gl_ld((const seq_bf16*)p.bu + f) : 0.f;
    }
    __device__ __forceinline__ void finish(const GpTile& t, f32x16 (&acc)[4][2], float* slab) const
    {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), gg = wave >> 2, wn = wave & 3;
        const long m0 = t.i0 + 128 * gg;
        const int row = lane >> 2, cq = lane & 3;             // of a store: 16 rows, 8 hidden units a lane
        const long f = t.j0 + 32 * wn + 8 * cq, left = p.F - f;
        if constexpr (!BWD) {
            // the activation where the accumulators lie (a lane: one hidden unit, 64 rows), rounded, then turned in LDS 64 rows at a time: 64-byte
            // rows, 16-byte units exchanged by row
            seq_bf16* sh = reinterpret_cast<seq_bf16*>(slab);
            const int fr = lane & 31, half = lane >> 5;
#pragma unroll
            for (int ih = 0; ih < 2; ++ih) {
#pragma unroll
                for (int i2 = 0; i2 < 2; ++i2)
#pragma unroll
                    for (int r = 0; r < 16; r += 2) {
                        const int i = 2 * ih + i2, lr = 32 * i2 + (r & 3) + 8 * (r >> 2) + 4 * half;      // rows lr, lr + 1
                        float a0, a1, slope;
                        gl_act<false>(acc[i][0][r], ACT, a0, slope);
                        gl_act<false>(acc[i][0][r + 1], ACT, a1, slope);
                        const unsigned v = seq_pack2(a0 * acc[i][1][r], a1 * acc[i][1][r + 1]);
                        const int unit = ((fr >> 3) ^ (lr >> 2 & 3)) * 8 + (fr & 7);
                        sh[lr * 32 + unit] = (seq_bf16)v;
                        sh[(lr + 1) * 32 + unit] = (seq_bf16)(v >> 16);
                    }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int lr = 16 * q + row;
                    const long m = m0 + 64 * ih + lr;
                    const gl_u32x4 v = *reinterpret_cast<const gl_u32x4*>(sh + lr * 32 + (cq ^ (lr >> 2 & 3)) * 8);
                    if (m < p.M && left > 0) {
                        if (p.y_vec && left >= 8) {
                            *reinterpret_cast<gl_u32x4*>((seq_bf16*)p.y + m * p.F + f) = v;
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const unsigned x = v[e >> 1];
                                if (e < left) ((seq_bf16*)p.y)[m * p.F + f + e] = (seq_bf16)(e & 1 ? x >> 16 : x);
                            }
                        }
                    }
                }
            }
        } else {
            // 16 rows at a time through the slab: g in the left half of its rows, u in the right; the rows' dy four rounds ahead
            // (a load waits for the stores before it)
            float sg[8], su[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) sg[e] = su[e] = 0.f;
            const bool fast = p.dy_vec && t.i0 + 256 <= p.M && t.j0 + 128 <= p.F;      // (the whole tile exists)
            constexpr int RING = 4;                           // (more would spill; 2 measured 176.6 us against 172.2)
            gl_u32x4 ring[RING];
            const seq_bf16* pd = (const seq_bf16*)p.dy + (m0 + row) * p.ldd + f;
            if (fast)
#pragma unroll
                for (int q = 0; q < RING; ++q) ring[q] = *reinterpret_cast<const gl_u32x4*>(pd + 16L * q * p.ldd);
#pragma unroll
            for (int rd = 0; rd < 8; ++rd) {
                const long m = m0 + 16 * rd + row;
                const bool on = m < p.M && left > 0;
                float d[8], gv[8], uv[8];
                gp_slab_put(slab, acc, rd >> 1, rd & 1);
                gp_slab_get(slab, row, 2 * cq, gv);
                gp_slab_get(slab, row, 8 + 2 * cq, uv);
                if (fast) {
                    gl_open8(ring[rd & (RING - 1)], d);
                    if (rd + RING < 8) ring[rd & (RING - 1)] = *reinterpret_cast<const gl_u32x4*>(pd + 16L * (rd + RING) * p.ldd);
                } else if (on) {
                    gl_load8((const seq_bf16*)p.dy + m * p.ldd + f, d, p.dy_vec, left);
#pragma unroll
                    for (int e = 0; e < 8; ++e)               // the products read the columns up to Fp: 0, also where a row of x is infinite
                        if (e >= left) gv[e] = uv[e] = 0.f;
                }
                if (on) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float a, slope;
                        gl_act<false>(gv[e], ACT, a, slope);
                        gv[e] = d[e] * uv[e] * slope;
                        uv[e] = d[e] * a;
                    }
                    if (p.slab) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) { sg[e] += gv[e]; su[e] += uv[e]; }
                    }
                    gl_store8((seq_bf16*)p.dgu + m * 2 * p.Fp + f, gv, true, 8);
                    gl_store8((seq_bf16*)p.dgu + m * 2 * p.Fp + p.Fp + f, uv, true, 8);
                }
            }
            if (p.slab && m0 < p.M) {                         // the 16 row lanes joined, one slab row per 128 rows
#pragma unroll
                for (int st = 4; st < 64; st *= 2)
#pragma unroll
                    for (int e = 0; e < 8; ++e) { sg[e] += __shfl_xor(sg[e], st, 64); su[e] += __shfl_xor(su[e], st, 64); }
                if (row == 0 && left > 0) {
                    float* to = p.slab + m0 / 128 * 2 * p.F + f;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < left) { to[e] = sg[e]; to[p.F + e] = su[e]; }
                }
            }
        }
    }
};

template <bool BWD, int ACT>
__global__ __launch_bounds__(512) void gl_gate_pp_kernel(GlArgs p, int nt, int total)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    GpGate<BWD, ACT> w{p, nt, total, (int)((p.K + 63) >> 6)};
    gp_run<false, false>(w, smem);
}

// ---- the backward pass's products: one tile a workgroup ----
struct GpProduct {
    const GlJob& p;
    long tile_no;
    __device__ __forceinline__ bool tile(int vb, GpTile& t) const
    {
        if (vb != (int)blockIdx.x) return false;
        const int tj = (int)p.tj, it = (int)tile_no / tj;
        t.i0 = 256L * __builtin_amdgcn_readfirstlane(it);
        t.j0 = 256L * __builtin_amdgcn_readfirstlane((int)tile_no - it * tj);
        t.chunks = p.chunks;
        return true;
    }
    __device__ __forceinline__ bool setup_a(int vb, GpCursor& c) const
    {
        GpTile t;
        if (!tile(vb, t)) return false;
        const long at = p.a_kr ? t.i0 * 2 : t.i0 * p.a.ld[0] * 2;
        c.at[0] = c.at[1] = (const char*)p.a.p[0] + at;
        c.second = (const char*)p.a.p[1] + at;
        auto rows = [](int reg, int r) { return 128 * reg + r; };
        if (p.a_kr) gp_aim_kr(c, p.a.n - t.i0, p.a.ld[0], p.K, p.chunks, rows);
        else gp_aim_kc(c, p.a.n - t.i0, p.a.ld, p.K, p.chunks, rows);
        return true;
    }
    __device__ __forceinline__ bool setup_b(int vb, GpCursor& c) const
    {
        GpTile t;
        if (!tile(vb, t)) return false;
        c.at[0] = c.at[1] = (const char*)p.b.p[0] + t.j0 * 2;
        c.second = (const char*)p.b.p[1] + t.j0 * 2;
        gp_aim_kr(c, p.b.n - t.j0, p.b.ld[0], p.K, p.chunks, [](int reg, int x) { return 64 * (x >> 5) + 32 * reg + (x & 31); });
        return true;
    }
    __device__ __forceinline__ void start(const GpTile&, float&, float&) const {}
    __device__ __forceinline__ void finish(const GpTile& t, f32x16 (&acc)[4][2], float* slab) const
    {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), gg = wave >> 2, wn = wave & 3;
        const int er = lane >> 3, c8 = lane & 7;
        const long j = t.j0 + 64 * wn + 8 * c8, left = p.J - j;
        const bool vec = p.J % 8 == 0;
#pragma unroll
        for (int rd = 0; rd < 8; ++rd) {
            gp_slab_put(slab, acc, rd >> 1, rd & 1);
#pragma unroll
            for (int sr = 0; sr < 2; ++sr) {
                const long i = t.i0 + 128 * gg + 16 * rd + 8 * sr + er;
                float x[8];
                gp_slab_get(slab, 8 * sr + er, 2 * c8, x);
                if (i < p.I && left > 0) gl_store8((seq_bf16*)p.out + i * p.J + j, x, vec, left);
            }
        }
    }
};

__global__ __launch_bounds__(512) void gl_product_pp_kernel(GlJobs all)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int q = 0;
    if (all.n > 1 && (int)blockIdx.x >= all.j[1].first) q = 1;
    if (all.n > 2 && (int)blockIdx.x >= all.j[2].first) q = 2;
    const GlJob& p = all.j[q];
    GpProduct w{p, gl_tile_of((long)blockIdx.x - p.first, p.tiles)};
    if (p.a_kr) gp_run<true, true>(w, smem);
    else gp_run<false, true>(w, smem);
}

template <class Kernel>
int gp_ready(Kernel kern, bool (&told)[64], int& cus)
{
    static int n_cu[64] = {};
    int dev = 0;
    HN_HIP(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !told[dev] || !n_cu[dev]) {
        HN_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, GP_LDS));
        int n = 0;
        HN_HIP(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev));
        cus = n;
        if (dev >= 0 && dev < 64) { n_cu[dev] = n; told[dev] = true; }
        return 0;
    }
    cus = n_cu[dev];
    return 0;
}

template <bool BWD, int ACT>
int gp_gate(const GlArgs& p, hipStream_t s)
{
    static bool told[64] = {};
    int cus = 256;
    if (const int rc = gp_ready(gl_gate_pp_kernel<BWD, ACT>, told, cus)) return rc;
    const int nt = hn_cdiv(p.F, 128);
    const long total = (long)hn_cdiv(p.M, 256) * nt;
    HN_REQUIRE(total > 0 && total <= 0x3fffffffL, "hn_gated_linear: too many tiles");
    hipLaunchKernelGGL((gl_gate_pp_kernel<BWD, ACT>), dim3((unsigned)(total < cus ? total : cus)), dim3(512), GP_LDS, s, p, nt, (int)total);
    HN_LAUNCH_CHECK();
    return 0;
}

}  // namespace

int hn_launch_gated_linear_pp_gate(const GlArgs& p, bool backward, hipStream_t s)
{
    switch (p.act) {
    case GL_SILU: return backward ? gp_gate<true, GL_SILU>(p, s) : gp_gate<false, GL_SILU>(p, s);
    case GL_GELU: return backward ? gp_gate<true, GL_GELU>(p, s) : gp_gate<false, GL_GELU>(p, s);
    case GL_SIGMOID: return backward ? gp_gate<true, GL_SIGMOID>(p, s) : gp_gate<false, GL_SIGMOID>(p, s);
    default: return backward ? gp_gate<true, GL_RELU>(p, s) : gp_gate<false, GL_RELU>(p, s);
    }
}

int hn_launch_gated_linear_pp_products(GlJobs& jobs, hipStream_t s)
{
    static bool told[64] = {};
    int cus = 256;
    if (const int rc = gp_ready(gl_product_pp_kernel, told, cus)) return rc;
    for (int q = 1; q < jobs.n; ++q)              // longest k first: the short tiles fill the rest of the device
        for (int r = q; r > 0 && jobs.j[r].chunks > jobs.j[r - 1].chunks; --r) {
            const GlJob t = jobs.j[r];
            jobs.j[r] = jobs.j[r - 1];
            jobs.j[r - 1] = t;
        }
    long n = 0;
    for (int q = 0; q < jobs.n; ++q) {
        GlJob& j = jobs.j[q];
        j.tj = hn_cdiv(j.J, 256);
        j.tiles = (long)hn_cdiv(j.I, 256) * j.tj;
        j.first = (int)n;
        n += j.tiles;
        HN_REQUIRE(j.splits == 1 && j.chunks >= 1, "hn_gated_linear_bwd: a product of whole k axes");
        SEQ_REQUIRE_GRID(n, 512, "hn_gated_linear_bwd");
    }
    if (n == 0) return 0;
    hipLaunchKernelGGL(gl_product_pp_kernel, dim3((unsigned)n), dim3(512), GP_LDS, s, jobs);
    HN_LAUNCH_CHECK();
    return 0;
}
