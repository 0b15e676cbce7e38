// k_mxg.hip - grouped GEMM of MXFP4 expert tables on the scaled MFMA: gate/up
// with the GLU (or relu^2) and the next product's operand in the epilogue, and
// the plain product.  Format and operand: mx.hpp.
//
// A work-group of WM x WN waves owns a balanced tile of at most BM = 32 R WM
// dispatched rows of one expert and 32 C WN weight rows (GLU: half of them gate
// rows, the others the matching up rows); a wave R row tiles and C column
// tiles of 32 on v_mfma_scale_f32_32x32x64_f8f6f4: four MFMAs per (row tile,
// column tile, two blocks), one per digit.  Lane half h of the MFMA takes block
// 2 step + h.
//
// The K loop runs over granules of four blocks (two steps).  Weights: each
// lane loads the blocks of its own weight rows into registers, a granule ahead
// (34 bytes of a row per step and 68 per granule lie together).  Activations:
// through two LDS buffers, a granule ahead, 400 bytes per row (four blocks of
// 96 and their scale words; 100 dwords apart, the rows of 8 lanes start on
// different banks), 8 threads to a row's 128 bytes.
#include "act.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "mx.hpp"

namespace mimoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int MXG_ROW = 4 * MX_XB + 16;   // LDS bytes of a row's granule

template <int DIG>
__device__ __forceinline__ f32x16 mxg_mfma(const i32x8 &a, const i32x8 &b, const f32x16 &c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 2, 4, DIG, sa, 0, sb);
}

template <int EPI, int R, int C, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, R == 1 ? 2 : 1) k_mxg(MxArgs g) {
    constexpr int BM = 32 * R * WM, NT = 64 * WM * WN;
    constexpr bool GLU = EPI == MX_GLU;
    constexpr int RG = BM / (NT / 8);   // row groups of a granule's loads (NT / 8 rows each)
    static_assert(BM % (NT / 8) == 0 && BM <= NT, "whole row groups, a row per thread");
    __shared__ __attribute__((aligned(16))) uint8_t sx[2][BM * MXG_ROW];
    __shared__ int s_p[BM];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l32 = lane & 31, h = lane >> 5;
    const MxSide s = g;
    // work-group 8 q + x on XCD x: the x-th eighth of the tiles in expert
    // order, one after another, column tile q % ncb (the column tiles of a row
    // tile share that XCD's L2 for the activations, the row tiles of an expert
    // for the weights)
    const int q8 = blockIdx.x >> 3, nt = *g.n_tiles, per = (nt + 7) >> 3, kk = q8 / g.ncb;
    const int tile = (int)(blockIdx.x & 7) * per + kk, cb = q8 - kk * g.ncb;
    if (kk >= per || tile >= nt) return;
    const int e = g.tile_e[tile], start = g.tile_start[tile], mrows = g.tile_rows[tile];
    const int nb = (int)(s.a.K / 32), ng = (nb + 3) / 4;
    const int wr = wave / WN, wc = wave - wr * WN;
    // the lane's weight rows (past the matrix: row 0, not stored); GLU: even
    // column tiles gate rows, odd ones the matching up rows
    constexpr int CW = GLU ? 16 * C : 32 * C;   // columns of y (of the activation rows) per wave
    const int64_t n0 = ((int64_t)cb * WN + wc) * CW;
    const uint8_t *rowp[C];
#pragma unroll
    for (int ct = 0; ct < C; ++ct) {
        const int64_t col = n0 + 32 * (GLU ? ct / 2 : ct) + l32;
        int64_t row = col < s.ncols ? col : 0;
        if (GLU && (ct & 1) && !s.fused) {
            rowp[ct] = s.b.data + (int64_t)e * s.b.mat_bytes + row * s.b.row_bytes;
        } else {
            if (GLU && (ct & 1)) row += s.I;
            rowp[ct] = s.a.data + (int64_t)e * s.a.mat_bytes + row * s.a.row_bytes;
        }
    }
    // the rows of this thread's activation loads (past the tile: its first row, not stored)
    const int kdiv = g.ne11 == 1 ? g.K : 1, l8 = tid & 7;
    const uint8_t *xrow[RG];
    const uint32_t *xsc;
#pragma unroll
    for (int j = 0; j < RG; ++j) {
        const int r = j * (NT / 8) + (tid >> 3), p = g.perm[start + (r < mrows ? r : 0)];
        xrow[j] = s.x.xb + (int64_t)(kdiv > 1 ? p / kdiv : p) * nb * MX_XB;
    }
    const int srow = tid % BM;   // scale words: thread (row, part of the granule's four)
    constexpr int SW = 4 * BM / NT > 0 ? 4 * BM / NT : 1;   // words per thread
    {
        const int p = g.perm[start + (srow < mrows ? srow : 0)];
        if (tid < BM) s_p[tid] = p;
        xsc = s.x.xs + (int64_t)(kdiv > 1 ? p / kdiv : p) * nb;
    }
    MxRaw raw[2][C];
    auto load_w = [&](int gr) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int b = 4 * gr + 2 * t + h;
#pragma unroll
            for (int ct = 0; ct < C; ++ct) mx_load(rowp[ct] + MX_BYTES * (b < nb ? b : nb - 1), raw[t][ct]);
        }
    };
    uint4 areg[RG][3];
    uint32_t asc[SW];
    auto load_a = [&](int gr) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < RG; ++j)
#pragma unroll
            for (int c = 0; c < 3; ++c) {
                const int q = 8 * c + l8;   // 16-byte piece of the row's granule
                areg[j][c] = make_uint4(0, 0, 0, 0);
                if (4 * gr + q / 6 < nb) areg[j][c] = *(const uint4 *)(xrow[j] + (4 * (int64_t)gr * MX_XB + 16 * q));
            }
#pragma unroll
        for (int i = 0; i < SW; ++i) {
            const int b = 4 * gr + (tid / BM) * SW + i;
            asc[i] = b < nb ? xsc[b] : MX_ONE * 0x01010101u;
        }
    };
    auto store_a = [&](uint8_t *x) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < RG; ++j)
#pragma unroll
            for (int c = 0; c < 3; ++c) *(uint4 *)(x + (j * (NT / 8) + (tid >> 3)) * MXG_ROW + 16 * (8 * c + l8)) = areg[j][c];
        if (NT <= 4 * BM || tid < 4 * BM)
#pragma unroll
            for (int i = 0; i < SW; ++i) *(uint32_t *)(x + srow * MXG_ROW + 4 * MX_XB + 4 * ((tid / BM) * SW + i)) = asc[i];
    };
    f32x16 acc[R][C];
#pragma unroll
    for (int rt = 0; rt < R; ++rt)
#pragma unroll
        for (int ct = 0; ct < C; ++ct)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[rt][ct][i] = 0.f;
    load_w(0);
    load_a(0);
    store_a(sx[0]);
    lds_barrier();
    const int nrt = (mrows - 32 * R * wr + 31) >> 5;   // row tiles of this wave that hold rows
    for (int gr = 0; gr < ng; ++gr) {
        const bool more = gr + 1 < ng;
        // the granule's weight operands out of the loaded dwords, whose registers take the next granule's
        i32x8 B[2][C];
        int sb[2][C];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int b = 4 * gr + 2 * t + h;
            const bool in = b < nb;
#pragma unroll
            for (int ct = 0; ct < C; ++ct) {
                const uint32_t mis = (uint32_t)((uintptr_t)rowp[ct] + (uint32_t)(MX_BYTES * (in ? b : nb - 1))) & 3u;
                uint32_t c[4];
                mx_codes(raw[t][ct], mis, c);
                // (a block past the row: the operand's digits are zero, the scale any number)
                sb[t][ct] = in ? (int)mx_scale(raw[t][ct], mis) : (int)MX_ONE;
                B[t][ct] = i32x8{(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
            }
        }
        if (more) {
            load_w(gr + 1);
            load_a(gr + 1);
        }
        const uint8_t *X = sx[gr & 1];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int rt = 0; rt < R; ++rt) {
                if (rt >= nrt) break;
                const uint8_t *xr = X + (32 * (R * wr + rt) + l32) * MXG_ROW;
                const uint8_t *x = xr + (2 * t + h) * MX_XB;
                const int sa = *(const int *)(xr + 4 * MX_XB + 4 * (2 * t + h));
                i32x8 A[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 lo = *(const uint4 *)(x + 16 * i);
                    const uint2 hi = *(const uint2 *)(x + 64 + 8 * i);
                    A[i] = i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, 0, 0};
                }
#pragma unroll
                for (int ct = 0; ct < C; ++ct) acc[rt][ct] = mxg_mfma<0>(A[0], B[t][ct], acc[rt][ct], sa, sb[t][ct]);
#pragma unroll
                for (int ct = 0; ct < C; ++ct) acc[rt][ct] = mxg_mfma<1>(A[1], B[t][ct], acc[rt][ct], sa, sb[t][ct]);
#pragma unroll
                for (int ct = 0; ct < C; ++ct) acc[rt][ct] = mxg_mfma<2>(A[2], B[t][ct], acc[rt][ct], sa, sb[t][ct]);
#pragma unroll
                for (int ct = 0; ct < C; ++ct) acc[rt][ct] = mxg_mfma<3>(A[3], B[t][ct], acc[rt][ct], sa, sb[t][ct]);
            }
        if (more) store_a(sx[(gr + 1) & 1]);
        lds_barrier();
    }
    // accumulator i of the lane: row 8 (i / 4) + 4 h + i % 4 of the row tile, column l32
    if constexpr (EPI == MX_STORE) {
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int m = 32 * (R * wr + rt) + 8 * (i >> 2) + 4 * h + (i & 3);
                if (m >= mrows) continue;
                float *y = s.y + (int64_t)s_p[m] * s.ldy;
#pragma unroll
                for (int ct = 0; ct < C; ++ct) {
                    const int64_t n = n0 + 32 * ct + l32;
                    if (n < s.ncols) y[n] = acc[rt][ct][i];
                }
            }
    } else {
        // (4 KB of the wave's own: no wave reads the activations any more)
        float *v = (float *)(sx[0] + 4096 * wave);
        static_assert(4096 * WM * WN <= 2 * BM * MXG_ROW, "LDS of the epilogue");
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
#pragma unroll
            for (int ct = 0; ct < (GLU ? C / 2 : C); ++ct) {
                const int64_t n = n0 + 32 * ct;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    v[(8 * (i >> 2) + 4 * h + (i & 3)) * 32 + l32] =
                        GLU ? act_pair(g.act, acc[rt][2 * ct][i], acc[rt][2 * ct + 1][i]) : relu_sqr(acc[rt][ct][i]);
                wave_lds_sync();
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int r = 16 * q + (lane >> 2), m = 32 * (R * wr + rt) + r;
                    float t[8];
                    mx_load8<true>(v + 32 * r, lane & 3, t);
                    const bool live = m < mrows && n < s.ncols;
                    const int64_t ob = (int64_t)s_p[live ? m : 0] * (s.ncols / 32) + n / 32;
                    mx_store_block(t, s.o.xb + ob * MX_XB, s.o.xs + ob, lane & 3, live);
                }
                wave_lds_sync();   // (rewritten next)
            }
    }
}

template <int EPI>
static int mxg_launch(const MxArgs &a, hipStream_t st) {
    MxArgs g = a;
    constexpr int COLS = EPI == MX_GLU ? 128 : 256;   // per work-group
    g.ncb = (int)((g.ncols + COLS - 1) / COLS);
    const int64_t wgs = 8 * (int64_t)g.ncb * ((g.max_tiles + 7) / 8);
    if (wgs > 0x7fffffff) return -6;
    if (g.bm == MXG_BM) hipLaunchKernelGGL((k_mxg<EPI, 2, 4, 2, 2>), dim3((unsigned)wgs), dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_mxg<EPI, 1, 2, 1, 4>), dim3((unsigned)wgs), dim3(256), 0, st, g);
    return hip_check_launch();
}

int launch_mxg(const MxArgs &g, hipStream_t st) {
    if (g.max_tiles <= 0) return 0;
    if (g.bm != MXG_BM && g.bm != MXG_BM_SMALL) return -6;
    if (g.a.type != 39 || g.a.K % 32 || g.a.K > 0x7fffffff || (g.epi != MX_STORE && g.ncols % 32)) return -6;
    switch (g.epi) {
    case MX_STORE: return mxg_launch<MX_STORE>(g, st);
    case MX_GLU: return mxg_launch<MX_GLU>(g, st);
    case MX_RELU_SQR: return mxg_launch<MX_RELU_SQR>(g, st);
    default: return -6;
    }
}

}  // namespace mimoe
