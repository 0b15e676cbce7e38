// k_mxg.hip - grouped GEMM of MXFP4 expert tables on the scaled MFMA: gate/up
// with the GLU (or relu^2) and the next product's operand in the epilogue, and
// the plain product.  Format and operand: mx.hpp.
//
// A work-group of WM x WN = 4 waves owns a balanced tile of at most BM = 32 WM
// dispatched rows of one expert and 256 weight rows (GLU: 128 gate rows and the
// matching 128 up rows); a wave 32 rows and C column tiles of 32 on
// v_mfma_scale_f32_32x32x64_f8f6f4: four MFMAs per (column tile, two blocks),
// one per digit.  Lane half h of the MFMA takes block 2 step + h.
//
// The K loop runs over steps of two blocks.  While step s's MFMAs run, step s +
// 1's operands are read from LDS into registers and step s + 3's loads go out,
// straight into LDS (buffer_load ... lds, 16-byte pieces):
//  * activations: rings of three buffers, 208 bytes per row and step (two
//    blocks' digits and the scale words; 52 dwords apart, the rows of 8 lanes
//    start on different banks); rows past the tile read out of range (no
//    memory traffic);
//  * weights: granules of two steps in two buffers, each of the 256 rows' runs
//    of 68 bytes as five pieces from the dword at or below its first byte
//    (blocks start at any byte, and rows may be misaligned).
// One barrier per step; the loads of the step stay in flight across it, the
// older ones have come (all loads are made, past the last step its own again:
// the counted waits rely on it).
#include "act.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "mx.hpp"

namespace mimoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr int MXG_ROW = 2 * MX_XB + 16;   // LDS bytes of an activation row's step
constexpr int MXG_WROWS = 256, MXG_WROW = 80, MXG_WRUN = 4 * MX_BYTES;   // weight rows of a work-group, LDS bytes of one's granule, bytes of its run
constexpr int MXG_WLD = 64 * MXG_WROW / 1024;   // a wave's loads of 64 rows
constexpr uint32_t MXG_FAR = 0xF8000000u;       // an offset past the rows (at most MXG_MAX_X bytes), far from wrapping

// at most N vector-memory loads of this wave outstanding and no LDS access, then the barrier
template <int N>
__device__ __forceinline__ void mxg_sync() {
    static_assert(N >= 0 && N < 64, "vmcnt");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
    asm volatile("s_barrier" ::: "memory");
}

template <int DIG>
__device__ __forceinline__ f32x16 mxg_mfma(const i32x8 &a, const i32x8 &b, const f32x16 &c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 2, 4, DIG, sa, 0, sb);
}

// The lane's block i (0 .. 3) of a granule out of its row's LDS pieces: the
// block's first byte is byte o = 0 .. 6 past a multiple of 16, so 24 bytes hold
// it (a 16- and an 8-byte read: dword by dword the reads of 32 rows 20 dwords
// apart take 8 cycles each, these 5 and 4.6).
struct MxgRaw {
    u32x4 a;
    uint32_t b[2];
};
__device__ __forceinline__ void mxg_read(const uint8_t *sw, uint32_t at, MxgRaw &r) {
    const uint8_t *p = sw + (at & ~15u);
    r.a = *(const u32x4 *)p;
    const uint2 b = *(const uint2 *)(p + 16);
    r.b[0] = b.x;
    r.b[1] = b.y;
}
__device__ __forceinline__ void mxg_unpack(const MxgRaw &r, uint32_t at, i32x8 &c, int &scale) {
    const uint32_t o = at & 15u, w[6] = {r.a[0], r.a[1], r.a[2], r.a[3], r.b[0], r.b[1]};
    const bool up = o >= 3u;   // the codes, from byte o + 1, start in dword 1
    uint32_t x[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) x[i] = up ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = (int)__builtin_amdgcn_alignbyte(x[i + 1], x[i], (o + 1u) & 3u);
    scale = (int)(((o >= 4u ? w[1] : w[0]) >> (8u * (o & 3u))) & 0xffu);
}

// a step's operands in registers
template <int C>
struct MxgOps {
    MxgRaw w[C];
    u32x4 lo[4];
    uint2 hi[4];
    int sa;
};

template <int EPI, int C, int WM, int WN>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) k_mxg(MxArgs g) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int BM = 32 * WM;
    constexpr bool GLU = EPI == MX_GLU;
    static_assert(WM * WN == 4 && 32 * C * WN == MXG_WROWS, "four waves, 256 weight rows");
    // loads of a step's activations: 64 pieces each, dealt to the waves (the last ones to several)
    constexpr int ALD = (BM * 13 + 63) / 64, NAL = (ALD + 3) / 4;
    __shared__ __attribute__((aligned(16))) uint8_t sa0[1024 * ALD];
    __shared__ __attribute__((aligned(16))) uint8_t sa1[1024 * ALD];
    __shared__ __attribute__((aligned(16))) uint8_t sa2[1024 * ALD];
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
    const int nb = (int)(s.a.K / 32), ns = (nb + 1) / 2;
    const int wr = wave / WN, wc = wave - wr * WN;
    // Columns of y (of the activation rows) of a work-group and a wave.  The
    // 256 weight rows in LDS: those of the columns in order (GLU: 128 gate
    // rows, then the 128 matching up rows); wave w loads rows 64 w .. 64 w + 63.
    constexpr int CB = GLU ? MXG_WROWS / 2 : MXG_WROWS, CW = CB / WN;
    const int64_t c0 = (int64_t)cb * CB, n0 = c0 + CW * wc;
    __amdgpu_buffer_rsrc_t wrsrc;
    uint32_t woff[MXG_WLD];
    {
        const bool up = GLU && wave >= 2;
        const ExpertMat &m = up && !s.fused ? s.b : s.a;
        // (rows past the matrix: its last row again, not stored)
        const int64_t r0 = c0 + 64 * (GLU ? wave & 1 : wave), first = r0 < s.ncols ? r0 : s.ncols - 1, left = s.ncols - first;
        const uint8_t *p = m.data + (int64_t)e * m.mat_bytes + (first + (up && s.fused ? s.I : 0)) * m.row_bytes;
        const uint32_t mis = (uint32_t)(uintptr_t)p & 3u, rb = (uint32_t)m.row_bytes, last = (left < 64 ? (uint32_t)left : 64u) - 1;
        // (a dword past the last row's bytes reads as zero)
        const uint32_t bytes = (mis + last * rb + (uint32_t)nb * MX_BYTES + 3) & ~3u;
        wrsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p - mis), (short)0, (int)bytes, 0x00020000);
#pragma unroll
        for (int j = 0; j < MXG_WLD; ++j) {
            const uint32_t q = 64u * (uint32_t)j + (uint32_t)lane, r = q / 5u, k = q - 5u * r;
            woff[j] = ((mis + (r < last ? r : last) * rb) & ~3u) + 16u * k;
        }
    }
    // granule gr's weights
    auto load_w = [&](int gr, uint8_t *sw) __attribute__((always_inline)) {
        gr = imin(gr, (nb - 1) / 4);
#pragma unroll
        for (int j = 0; j < MXG_WLD; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wrsrc, (lds_void_t *)(sw + 64 * MXG_WROW * wave + 1024 * j), 16, (int)woff[j],
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
    // this lane's pieces of the activations (past the tile: out of range)
    const int kdiv = g.ne11 == 1 ? g.K : 1;
    const __amdgpu_buffer_rsrc_t arsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(s.x), (short)0, (int)(uint32_t)(s.xrows * mx_row(nb)), 0x00020000);
    uint32_t aoff[NAL];
#pragma unroll
    for (int i = 0; i < NAL; ++i) {
        const int j = wave + 4 * i < ALD ? wave + 4 * i : ALD - 1, q = 64 * j + lane, r = q / 13, k = q - 13 * r;
        const int p = r < mrows ? g.perm[start + r] : -1;
        aoff[i] = p < 0 ? MXG_FAR : (uint32_t)(kdiv > 1 ? p / kdiv : p) * (uint32_t)mx_row(nb) + 16u * (uint32_t)k;
    }
    if (tid < BM) s_p[tid] = tid < mrows ? g.perm[start + tid] : 0;
    // step st's activations
    auto load_a = [&](int st, uint8_t *sa) __attribute__((always_inline)) {
        __amdgpu_buffer_rsrc_t r = arsrc;   // the builtin takes no const-qualified resource
        st = imin(st, ns - 1);
#pragma unroll
        for (int i = 0; i < NAL; ++i) {
            const int j = wave + 4 * i < ALD ? wave + 4 * i : ALD - 1;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t *)(sa + 1024 * j), 16, (int)aoff[i], MX_XG * (st >> 1) + 2 * MX_XB * (st & 1), 0, 0);
        }
    };
    // the operands of a step of parity T out of LDS
    auto take = [&](MxgOps<C> &o, int T, const uint8_t *sa, const uint8_t *sw) __attribute__((always_inline)) {
#pragma unroll
        for (int ct = 0; ct < C; ++ct) mxg_read(sw, wat[ct] + (uint32_t)(MX_BYTES * (2 * T + h)), o.w[ct]);
        const uint8_t *xr = sa + (32 * wr + l32) * MXG_ROW, *x = xr + 16 * T + MX_XB * h;
        o.sa = *(const int *)(xr + (T ? 0 : 2 * MX_XB) + 4 * (2 * T + h));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o.lo[i] = *(const u32x4 *)(x + 16 * i);
            o.hi[i] = *(const uint2 *)(x + 64 + 8 * i);
        }
    };
    f32x16 acc[C];
#pragma unroll
    for (int ct = 0; ct < C; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[ct][i] = 0.f;
    const bool rows = mrows > 32 * wr;   // the wave has rows
    auto products = [&](const MxgOps<C> &o, int T, int st) __attribute__((always_inline)) {
        if (!rows) return;
        i32x8 B[C];
        int sb[C];
#pragma unroll
        for (int ct = 0; ct < C; ++ct) {
            B[ct] = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
            mxg_unpack(o.w[ct], wat[ct] + (uint32_t)(MX_BYTES * (2 * T + h)), B[ct], sb[ct]);
        }
        // (the block past a row of an odd number: the operand's digits are zero, the scale any number)
        if (2 * st + 1 >= nb) {
#pragma unroll
            for (int ct = 0; ct < C; ++ct) sb[ct] = h ? (int)MX_ONE : sb[ct];
        }
        i32x8 A[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            A[i] = i32x8{(int)o.lo[i][0], (int)o.lo[i][1], (int)o.lo[i][2], (int)o.lo[i][3], (int)o.hi[i].x, (int)o.hi[i].y, 0, 0};
#pragma unroll
        for (int ct = 0; ct < C; ++ct) acc[ct] = mxg_mfma<0>(A[0], B[ct], acc[ct], o.sa, sb[ct]);
#pragma unroll
        for (int ct = 0; ct < C; ++ct) acc[ct] = mxg_mfma<1>(A[1], B[ct], acc[ct], o.sa, sb[ct]);
#pragma unroll
        for (int ct = 0; ct < C; ++ct) acc[ct] = mxg_mfma<2>(A[2], B[ct], acc[ct], o.sa, sb[ct]);
#pragma unroll
        for (int ct = 0; ct < C; ++ct) acc[ct] = mxg_mfma<3>(A[3], B[ct], acc[ct], o.sa, sb[ct]);
    };
    load_w(0, sw0);
    load_a(0, sa0);
    load_w(1, sw1);
    load_a(1, sa1);
    load_a(2, sa2);
    mxg_sync<0>();
    MxgOps<C> ops[2];
    take(ops[0], 0, sa0, sw0);
    mxg_sync<0>();
    // Step st: buffers by st % 3, granules by st / 2 % 2, registers by st % 2:
    // twelve steps to a turn.  sa_free held step st's activations, sa_next
    // holds step st + 1's; sw_next holds step st + 1's weights, at odd steps
    // sw_free held step st's.
#define MXG_STEP(I, sa_free, sa_next, sw_next, sw_free)                  \
    if (st0 + I >= ns) break;                                            \
    load_a(st0 + I + 3, sa_free);                                        \
    if (I & 1) load_w((st0 + I) / 2 + 2, sw_free);                       \
    take(ops[(I + 1) & 1], (I + 1) & 1, sa_next, sw_next);               \
    products(ops[I & 1], I & 1, st0 + I);                                \
    mxg_sync<NAL + (I & 1) * MXG_WLD>();
    for (int st0 = 0;; st0 += 12) {
        MXG_STEP(0, sa0, sa1, sw0, sw0)
        MXG_STEP(1, sa1, sa2, sw1, sw0)
        MXG_STEP(2, sa2, sa0, sw1, sw1)
        MXG_STEP(3, sa0, sa1, sw0, sw1)
        MXG_STEP(4, sa1, sa2, sw0, sw0)
        MXG_STEP(5, sa2, sa0, sw1, sw0)
        MXG_STEP(6, sa0, sa1, sw1, sw1)
        MXG_STEP(7, sa1, sa2, sw0, sw1)
        MXG_STEP(8, sa2, sa0, sw0, sw0)
        MXG_STEP(9, sa0, sa1, sw1, sw0)
        MXG_STEP(10, sa1, sa2, sw1, sw1)
        MXG_STEP(11, sa2, sa0, sw0, sw1)
    }
#undef MXG_STEP
    mxg_sync<0>();   // (the loads past the last step)
    if (!rows) return;
    // accumulator i of the lane: row 8 (i / 4) + 4 h + i % 4 of the row tile, column l32
    if constexpr (EPI == MX_STORE) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int m = 32 * wr + 8 * (i >> 2) + 4 * h + (i & 3);
            if (m >= mrows) continue;
            float *y = s.y + (int64_t)s_p[m] * s.ldy;
#pragma unroll
            for (int ct = 0; ct < C; ++ct) {
                const int64_t n = n0 + 32 * ct + l32;
                if (n < s.ncols) y[n] = acc[ct][i];
            }
        }
    } else {
        // (4 KB of the wave's own in a weights' buffer, which no wave reads or loads any more)
        float *v = (float *)(sw0 + 4096 * wave);
#pragma unroll
        for (int ct = 0; ct < (GLU ? C / 2 : C); ++ct) {
            const int64_t n = n0 + 32 * ct;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                v[(8 * (i >> 2) + 4 * h + (i & 3)) * 32 + l32] = GLU ? act_pair(g.act, acc[2 * ct][i], acc[2 * ct + 1][i]) : relu_sqr(acc[ct][i]);
            wave_lds_sync();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int r = 16 * q + (lane >> 2), m = 32 * wr + r;
                float t[8];
                mx_load8<true>(v + 32 * r, lane & 3, t);
                const bool live = m < mrows && n < s.ncols;
                uint8_t *row = s.o + (int64_t)s_p[live ? m : 0] * mx_row(s.ncols / 32);
                mx_store_block(t, row, n / 32, lane & 3, live);
                if (live && n + 32 == s.ncols) mx_store_pad(row, s.ncols / 32, lane & 3);
            }
            wave_lds_sync();   // (rewritten next)
        }
    }
#endif
}

template <int EPI>
static int mxg_launch(const MxArgs &a, hipStream_t st) {
    MxArgs g = a;
    constexpr int COLS = EPI == MX_GLU ? MXG_WROWS / 2 : MXG_WROWS;   // per work-group
    g.ncb = (int)((g.ncols + COLS - 1) / COLS);
    const int64_t wgs = 8 * (int64_t)g.ncb * ((g.max_tiles + 7) / 8);
    if (wgs > 0x7fffffff) return -6;
    if (g.bm == MXG_BM) hipLaunchKernelGGL((k_mxg<EPI, 4, 2, 2>), dim3((unsigned)wgs), dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_mxg<EPI, 2, 1, 4>), dim3((unsigned)wgs), dim3(256), 0, st, g);
    return hip_check_launch();
}

int launch_mxg(const MxArgs &g, hipStream_t st) {
    if (g.max_tiles <= 0) return 0;
    if (g.bm != MXG_BM && g.bm != MXG_BM_SMALL) return -6;
    if (g.a.row_bytes > MXG_MAX_ROW_BYTES || (g.epi == MX_GLU && !g.fused && g.b.row_bytes > MXG_MAX_ROW_BYTES)) return -6;
    if (g.a.type != 39 || g.a.K % 32 || g.a.K > 0x7fffffff || (g.epi != MX_STORE && g.ncols % 32)) return -6;
    if (g.xrows <= 0 || g.xrows * mx_row(g.a.K / 32) > MXG_MAX_X || (uintptr_t)g.x % 16) return -6;
    switch (g.epi) {
    case MX_STORE: return mxg_launch<MX_STORE>(g, st);
    case MX_GLU: return mxg_launch<MX_GLU>(g, st);
    case MX_RELU_SQR: return mxg_launch<MX_RELU_SQR>(g, st);
    default: return -6;
    }
}

}  // namespace mimoe
