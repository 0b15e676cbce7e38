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
// The K loop runs over granules of four blocks (two steps).
//  * weights: the 256 weight rows' runs of a granule (68 bytes) reach one of
//    two LDS buffers by buffer loads that write LDS directly, a granule ahead,
//    each row as five 16-byte pieces from the dword at or below its first byte
//    (blocks start at any byte, and rows may be misaligned; rows 20 dwords
//    apart start on 16 different banks).
//  * activations: a granule ahead in registers, one LDS buffer, 400 bytes per
//    row (four blocks of 96 and their scale words; 100 dwords apart, the rows
//    of 8 lanes start on different banks), 8 threads to a row's 128 bytes.
// Two work-groups to a CU (three with 32-row tiles), one's waits and stores
// beside the other's MFMAs.
#include "act.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "mx.hpp"

namespace mimoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int MXG_ROW = 4 * MX_XB + 16;   // LDS bytes of an activation row's granule
constexpr int MXG_WROWS = 256, MXG_WROW = 80, MXG_WRUN = 4 * MX_BYTES;   // weight rows of a work-group, LDS bytes of one's granule, bytes of its run
constexpr int MXG_WLD = 64 * MXG_WROW / 1024;   // a wave's loads of 64 rows

typedef __attribute__((address_space(3))) void lds_void_t;

// this wave's vector-memory loads and LDS accesses complete, then the barrier
__device__ __forceinline__ void mxg_sync() {
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0), lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
}

template <int DIG>
__device__ __forceinline__ f32x16 mxg_mfma(const i32x8 &a, const i32x8 &b, const f32x16 &c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 2, 4, DIG, sa, 0, sb);
}

template <int EPI, int R, int C, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(WM == 1 ? 3 : 2))) k_mxg(MxArgs g) {
    constexpr int BM = 32 * R * WM, NT = 64 * WM * WN;
    constexpr bool GLU = EPI == MX_GLU;
    constexpr int RG = BM / (NT / 8);   // row groups of a granule's loads (NT / 8 rows each)
    static_assert(BM % (NT / 8) == 0 && BM <= NT, "whole row groups, a row per thread");
    __shared__ __attribute__((aligned(16))) uint8_t sx[BM * MXG_ROW];
    __shared__ __attribute__((aligned(16))) uint8_t sw0[MXG_WROWS * MXG_WROW];
    __shared__ __attribute__((aligned(16))) uint8_t sw1[MXG_WROWS * MXG_WROW];
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
    // Columns of y (of the activation rows) of a work-group and a wave.  The
    // 256 weight rows in LDS: those of the columns in order (GLU: 128 gate
    // rows, then the 128 matching up rows); wave w loads rows 64 w .. 64 w + 63.
    constexpr int CB = GLU ? MXG_WROWS / 2 : MXG_WROWS, CW = CB / WN;
    static_assert(WM * WN == 4 && 32 * C * WN == MXG_WROWS, "four waves, 256 weight rows");
    const int64_t c0 = (int64_t)cb * CB, n0 = c0 + CW * wc;
    __amdgpu_buffer_rsrc_t wr_rsrc;
    uint32_t woff[MXG_WLD];
    {
        const bool up = GLU && wave >= 2;
        const ExpertMat &m = up && !s.fused ? s.b : s.a;
        const int64_t r0 = c0 + 64 * (GLU ? wave & 1 : wave), left = s.ncols - r0, row0 = (left > 0 ? r0 : 0) + (up && s.fused ? s.I : 0);
        const uint8_t *p = m.data + (int64_t)e * m.mat_bytes + row0 * m.row_bytes;
        const uint32_t mis = (uint32_t)(uintptr_t)p & 3u, rb = (uint32_t)m.row_bytes;
        // (a dword past the last row's bytes reads as zero, as do the rows past the matrix)
        const uint32_t bytes = left > 0 ? (mis + ((left < 64 ? (uint32_t)left : 64u) - 1) * rb + (uint32_t)nb * MX_BYTES + 3) & ~3u : 0u;
        wr_rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p - mis), (short)0, (int)bytes, 0x00020000);
#pragma unroll
        for (int j = 0; j < MXG_WLD; ++j) {
            const uint32_t q = 64u * (uint32_t)j + (uint32_t)lane, r = q / 5u, k = q - 5u * r;
            woff[j] = ((mis + r * rb) & ~3u) + 16u * k;
        }
    }
    auto load_w = [&](int gr, uint8_t *sw) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < MXG_WLD; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr_rsrc, (lds_void_t *)(sw + 64 * MXG_WROW * wave + 1024 * j), 16, (int)woff[j],
                                                     MXG_WRUN * gr, 0, 0);
    };
    // where the lane's weight rows start in the buffer: their first byte's place
    uint32_t wat[C];
#pragma unroll
    for (int ct = 0; ct < C; ++ct) {
        const int lr = GLU ? 128 * (ct & 1) + CW * wc + 32 * (ct / 2) + l32 : CW * wc + 32 * ct + l32;   // its row in LDS
        const bool up = GLU && (ct & 1);
        const ExpertMat &m = up && !s.fused ? s.b : s.a;
        const int64_t row = c0 + (GLU ? lr & 127 : lr) + (up && s.fused ? s.I : 0);
        wat[ct] = (uint32_t)(MXG_WROW * lr) + ((uint32_t)((uintptr_t)m.data + (uintptr_t)((int64_t)e * m.mat_bytes + row * m.row_bytes)) & 3u);
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
    const int nrt = (mrows - 32 * R * wr + 31) >> 5;   // row tiles of this wave that hold rows
    // the products of granule gr, its weights at sw
    auto granule = [&](int gr, const uint8_t *sw) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const bool in = 4 * gr + 2 * t + h < nb;
            i32x8 B[C];
            int sb[C];
#pragma unroll
            for (int ct = 0; ct < C; ++ct) {
                const uint32_t at = wat[ct] + (uint32_t)(MX_BYTES * (2 * t + h));
                MxRaw raw;
#pragma unroll
                for (int i = 0; i < 5; ++i) raw.w[i] = *(const uint32_t *)(sw + (at & ~3u) + 4 * i);
                uint32_t c[4];
                mx_codes(raw, at & 3u, c);
                // (a block past the row: the operand's digits are zero, the scale any number)
                sb[ct] = in ? (int)mx_scale(raw, at & 3u) : (int)MX_ONE;
                B[ct] = i32x8{(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
            }
#pragma unroll
            for (int rt = 0; rt < R; ++rt) {
                if (rt >= nrt) break;
                const uint8_t *xr = sx + (32 * (R * wr + rt) + l32) * MXG_ROW;
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
                for (int ct = 0; ct < C; ++ct) acc[rt][ct] = mxg_mfma<0>(A[0], B[ct], acc[rt][ct], sa, sb[ct]);
#pragma unroll
                for (int ct = 0; ct < C; ++ct) acc[rt][ct] = mxg_mfma<1>(A[1], B[ct], acc[rt][ct], sa, sb[ct]);
#pragma unroll
                for (int ct = 0; ct < C; ++ct) acc[rt][ct] = mxg_mfma<2>(A[2], B[ct], acc[rt][ct], sa, sb[ct]);
#pragma unroll
                for (int ct = 0; ct < C; ++ct) acc[rt][ct] = mxg_mfma<3>(A[3], B[ct], acc[rt][ct], sa, sb[ct]);
            }
        }
    };
    auto turn = [&](int gr, const uint8_t *cur, uint8_t *nxt) __attribute__((always_inline)) {
        const bool more = gr + 1 < ng;
        if (more) {
            load_a(gr + 1);
            load_w(gr + 1, nxt);
        }
        granule(gr, cur);
        mxg_sync();   // the next granule has come, and no wave reads this one's activations
        if (more) {
            store_a(sx);
            lds_barrier();
        }
    };
    load_w(0, sw0);
    load_a(0);
    store_a(sx);
    mxg_sync();
    for (int gr = 0; gr < ng; gr += 2) {
        turn(gr, sw0, sw1);
        if (gr + 1 < ng) turn(gr + 1, sw1, sw0);
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
        // (4 KB of the wave's own in a weights' buffer, which no wave reads or loads any more)
        float *v = (float *)(sw0 + 4096 * wave);
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
    constexpr int COLS = EPI == MX_GLU ? MXG_WROWS / 2 : MXG_WROWS;   // per work-group
    g.ncb = (int)((g.ncols + COLS - 1) / COLS);
    const int64_t wgs = 8 * (int64_t)g.ncb * ((g.max_tiles + 7) / 8);
    if (wgs > 0x7fffffff) return -6;
    if (g.bm == MXG_BM) hipLaunchKernelGGL((k_mxg<EPI, 1, 4, 2, 2>), dim3((unsigned)wgs), dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_mxg<EPI, 1, 2, 1, 4>), dim3((unsigned)wgs), dim3(256), 0, st, g);
    return hip_check_launch();
}

int launch_mxg(const MxArgs &g, hipStream_t st) {
    if (g.max_tiles <= 0) return 0;
    if (g.bm != MXG_BM && g.bm != MXG_BM_SMALL) return -6;
    if (g.a.row_bytes > MXG_MAX_ROW_BYTES || (g.epi == MX_GLU && !g.fused && g.b.row_bytes > MXG_MAX_ROW_BYTES)) return -6;
    if (g.a.type != 39 || g.a.K % 32 || g.a.K > 0x7fffffff || (g.epi != MX_STORE && g.ncols % 32)) return -6;
    switch (g.epi) {
    case MX_STORE: return mxg_launch<MX_STORE>(g, st);
    case MX_GLU: return mxg_launch<MX_GLU>(g, st);
    case MX_RELU_SQR: return mxg_launch<MX_RELU_SQR>(g, st);
    default: return -6;
    }
}

}  // namespace mimoe
