// k_mxg.hip - grouped GEMM of MXFP4 expert tables on the scaled MFMA: gate/up
// with the GLU (or relu^2) and the next product's operand in the epilogue, and
// the plain product.  Format and operand: mx.hpp.
//
// A work-group of 4 waves owns a balanced tile of at most MXG_BM dispatched
// rows of one expert and 128 weight rows (GLU: 64 gate rows and the matching
// up rows): wave (wr, wc) two row tiles and two column tiles of 32 on
// v_mfma_scale_f32_32x32x64_f8f6f4, four MFMAs per (row tile, column tile,
// two blocks), one per digit.  Lane half h of the MFMA takes block 2 step + h.
#include "act.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "mx.hpp"

namespace mimoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int EPI>
__global__ void __launch_bounds__(256) k_mxg(MxArgs g) {
    __shared__ __attribute__((aligned(16))) uint8_t sx[2][MXG_BM * MX_XB];
    __shared__ uint32_t ss[2][MXG_BM];
    __shared__ int s_p[MXG_BM];
    __shared__ __attribute__((aligned(16))) float s_v[4][32 * 32];
    constexpr bool GLU = EPI == MX_GLU;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l32 = lane & 31, h = lane >> 5;
    const MxSide s = g;
    const int tile = blockIdx.x / g.ncb, cb = blockIdx.x - tile * g.ncb;
    if (tile >= *g.n_tiles) return;
    const int e = g.tile_e[tile], start = g.tile_start[tile], mrows = g.tile_rows[tile];
    const int nb = (int)(s.a.K / 32);
    if (tid < MXG_BM) s_p[tid] = g.perm[start + (tid < mrows ? tid : 0)];
    __syncthreads();
    const int wr = wave >> 1, wc = wave & 1;
    // the lane's weight rows (past the matrix: row 0, not stored)
    const int64_t n0 = (int64_t)cb * (GLU ? 64 : 128) + (GLU ? 32 : 64) * wc;
    const uint8_t *rowp[2];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        const int64_t col = n0 + (GLU ? 0 : 32 * ct) + l32;
        int64_t row = col < s.ncols ? col : 0;
        if (GLU && ct == 1 && !s.fused) {
            rowp[ct] = s.b.data + (int64_t)e * s.b.mat_bytes + row * s.b.row_bytes;
        } else {
            if (GLU && ct == 1) row += s.I;
            rowp[ct] = s.a.data + (int64_t)e * s.a.mat_bytes + row * s.a.row_bytes;
        }
    }
    f32x16 acc[2][2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[rt][ct][i] = 0.f;
    const int kdiv = g.ne11 == 1 ? g.K : 1;
    for (int b0 = 0; b0 < nb; b0 += 2) {
        const bool in = b0 + h < nb;
        MxRaw w[2];
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) mx_load(rowp[ct] + MX_BYTES * (int64_t)(in ? b0 + h : 0), w[ct]);
        __syncthreads();
        for (int i = tid; i < 2 * MXG_BM * 6; i += 256) {
            const int hb = i >= MXG_BM * 6, q = i - hb * MXG_BM * 6, r = q / 6;
            const int64_t xr = kdiv > 1 ? s_p[r] / kdiv : s_p[r];
            uint4 v = make_uint4(0, 0, 0, 0);
            if (b0 + hb < nb) v = *(const uint4 *)(s.x.xb + (xr * nb + b0 + hb) * MX_XB + 16 * (q - 6 * r));
            *(uint4 *)(sx[hb] + 16 * q) = v;
        }
        {
            const int hb = tid >> 7, r = tid & 127;
            const int64_t xr = kdiv > 1 ? s_p[r] / kdiv : s_p[r];
            ss[hb][r] = b0 + hb < nb ? s.x.xs[xr * nb + b0 + hb] : MX_ONE * 0x01010101u;
        }
        __syncthreads();
        i32x8 B[2];
        int sb[2];
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
            const uint32_t mis = (uint32_t)(uintptr_t)(rowp[ct] + MX_BYTES * (int64_t)(in ? b0 + h : 0)) & 3u;
            uint32_t c[4];
            mx_codes(w[ct], mis, c);
            B[ct] = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) B[ct][i] = in ? (int)c[i] : 0;
            sb[ct] = in ? (int)mx_scale(w[ct], mis) : (int)MX_ONE;
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            const int r = 64 * wr + 32 * rt + l32;
            const uint8_t *x = sx[h] + MX_XB * r;
            const int sa = (int)ss[h][r];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 lo = *(const uint4 *)(x + 16 * i);
                const uint2 hi = *(const uint2 *)(x + 64 + 8 * i);
                const i32x8 A = {(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, 0, 0};
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) {
                    f32x16 &c = acc[rt][ct];
                    if (i == 0) c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B[ct], c, 2, 4, 0, sa, 0, sb[ct]);
                    else if (i == 1) c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B[ct], c, 2, 4, 1, sa, 0, sb[ct]);
                    else if (i == 2) c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B[ct], c, 2, 4, 2, sa, 0, sb[ct]);
                    else c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B[ct], c, 2, 4, 3, sa, 0, sb[ct]);
                }
            }
        }
    }
    // accumulator i of the lane: row 8 (i / 4) + 4 h + i % 4 of the row tile, column l32
    if constexpr (EPI == MX_STORE) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int m = 64 * wr + 32 * rt + 8 * (i >> 2) + 4 * h + (i & 3);
                    const int64_t n = n0 + 32 * ct + l32;
                    if (m < mrows && n < s.ncols) s.y[(int64_t)s_p[m] * s.ldy + n] = acc[rt][ct][i];
                }
    } else {
        float *v = s_v[wave];
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int ct = 0; ct < (GLU ? 1 : 2); ++ct) {
                const int64_t n = n0 + 32 * ct;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    v[(8 * (i >> 2) + 4 * h + (i & 3)) * 32 + l32] = GLU ? act_pair(g.act, acc[rt][0][i], acc[rt][1][i]) : relu_sqr(acc[rt][ct][i]);
                wave_lds_sync();
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int r = 16 * q + (lane >> 2), m = 64 * wr + 32 * rt + r;
                    float t[8];
                    mx_load8<true>(v + 32 * r, lane & 3, t);
                    const int64_t ob = (int64_t)s_p[m] * (s.ncols / 32) + n / 32;
                    mx_store_block(t, s.o.xb + ob * MX_XB, s.o.xs + ob, lane & 3, m < mrows && n < s.ncols);
                }
                wave_lds_sync();   // (rewritten next)
            }
    }
}

template <int EPI>
static int mxg_launch(const MxArgs &a, hipStream_t st) {
    MxArgs g = a;
    constexpr int COLS = EPI == MX_GLU ? 64 : 128;
    g.ncb = (int)((g.ncols + COLS - 1) / COLS);
    const int64_t wgs = (int64_t)g.ncb * g.max_tiles;
    if (wgs > 0x7fffffff) return -6;
    hipLaunchKernelGGL(k_mxg<EPI>, dim3((unsigned)wgs), dim3(256), 0, st, g);
    return hip_check_launch();
}

int launch_mxg(const MxArgs &g, hipStream_t st) {
    if (g.max_tiles <= 0) return 0;
    if (g.a.type != 39 || g.a.K % 32 || g.a.K > 0x7fffffff || (g.epi != MX_STORE && g.ncols % 32)) return -6;
    switch (g.epi) {
    case MX_STORE: return mxg_launch<MX_STORE>(g, st);
    case MX_GLU: return mxg_launch<MX_GLU>(g, st);
    case MX_RELU_SQR: return mxg_launch<MX_RELU_SQR>(g, st);
    default: return -6;
    }
}

}  // namespace mimoe
