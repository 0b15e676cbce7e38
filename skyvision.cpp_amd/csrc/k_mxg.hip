// k_mxg.hip - grouped GEMM of MXFP4 expert tables on the scaled MFMA: gate/up
// with the GLU (or relu^2) and the next product's operand in the epilogue, and
// the plain product.  Format and operand: mx.hpp.
//
// A work-group of WM x WN waves owns a balanced tile of at most BM = 32 WM
// dispatched rows of one expert and WROWS = 32 C WN weight rows (GLU: half of
// them gate rows, half the matching up rows); a wave 32 rows and C column tiles
// of 32 on v_mfma_scale_f32_32x32x64_f8f6f4: four MFMAs per (column tile, two
// blocks), one per digit.  Lane half h of the MFMA takes block 2 step + h.
//
// The K loop runs over steps of two blocks.  While step s's MFMAs run, step s +
// 1's operands are read from LDS into registers and step s + 3's loads go out,
// straight into LDS (buffer_load ... lds, 16-byte pieces):
//  * activations: a ring of three buffers, 192 bytes of digits per row and step
//    (12 pieces at a multiple of 64 bytes; in LDS piece k of row r at k ^ (r /
//    4 % 4): the rows of 16 lanes on different banks); rows past the tile read
//    out of range (no memory traffic).  Each lane's own scale words go to
//    registers, four steps ahead.
//  * weights: stages of four blocks in two buffers, each row's run of 68 bytes
//    as 5 pieces from the dword at or below its first byte (blocks start at any
//    byte, and rows may be misaligned).
// One barrier per step; the loads of the step stay in flight across it, those
// that the next steps need have come (all loads are made, past the last step its
// own again: the counted waits rely on it).
//
// Two tiles.  64 rows x 256 weight rows, four waves, 78 KB of LDS, two
// work-groups to a CU: many rows per expert.  32 x 128, two waves, 39 KB, four
// to a CU: few, where the tables' stream counts and more work-groups that wait
// apart carry it (128 rows of 128 experts, K 2048: 32 x 256 in four waves 37 us,
// 32 x 128 29; 301 tokens of 8 slots, K 704, N 2816: both 65).  A step's loads go
// out in front of its LDS reads, in the small tile between its MFMAs (64 rows of
// 64 experts 50 -> 47 us; the large tile 240 -> 246).
//
// What bounds the large tile (16384 rows of 64 experts, K 2048, N 2048: 223 us
// of a call of 239, 241 - 248 under a profiler; 610 TFLOP/s of the contract's
// products, four times that on the MFMA): a wave's
// step is 57 vector instructions (most of them unpack weights), 12 LDS reads and
// 16 MFMAs, and two waves to a SIMD overlap them in part: without the loop's
// loads it takes 175 us, without the MFMAs 185, the stores are 22 of it.  Of the
// load path it takes 59%: that takes 60 B per cycle and CU of contiguous runs and
// 22 of runs of 5 pieces.  128-row tiles with runs of 9 pieces (8 waves, or 4 of
// 64 x 128 in 512 registers) were slower: 250 and 270 against 246.
#include "act.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "mx.hpp"

namespace mimoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr int MXG_ROW = 2 * MX_XB;              // LDS bytes of an activation row's step
constexpr uint32_t MXG_FAR = 0xF8000000u;       // an offset past the rows (at most MXG_MAX_X bytes), far from wrapping

template <int N> struct Const { static constexpr int value = N; };

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

// The lane's block 2 T + h (T = 0, 1) of a stage out of its row's LDS pieces:
// with m = 0 .. 3 the row's misalignment, its first byte is byte o = m + 2 T + h
// past 32 T + 16 h, so 24 bytes from there hold it.  (Wide reads: dword by dword
// the reads of 32 rows 20 dwords apart take 8 cycles each, these 5.)
struct MxgRaw {
    u32x4 a;
    uint2 b;
};
template <int T>
__device__ __forceinline__ void mxg_read(const uint8_t *p, MxgRaw &r) {   // p: the row's pieces + 16 h
    r.a = *(const u32x4 *)(p + 32 * T);
    r.b = *(const uint2 *)(p + 32 * T + 16);
}
template <int T>
__device__ __forceinline__ void mxg_unpack(const MxgRaw &r, uint32_t mh, i32x8 &c, int &scale) {   // mh: m + h
    const uint32_t o = mh + 2 * T, w[6] = {r.a[0], r.a[1], r.a[2], r.a[3], r.b.x, r.b.y};
    const bool up = o >= 3u;   // the codes, from byte o + 1 <= 7, start in dword 1
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
};

template <int EPI, int C, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2))) k_mxg(MxArgs g) {
#ifdef __HIP_DEVICE_COMPILE__   // (the host pass needs the stub alone)
    constexpr int BM = 32 * WM, NW = WM * WN;
    constexpr bool GLU = EPI == MX_GLU;
    constexpr int WROWS = 32 * C * WN;   // weight rows of a work-group
    static_assert(WROWS % 128 == 0 && BM <= 64 * NW, "groups of 64 weight rows, a row per thread");
    constexpr bool SPREAD = C == 2;   // a step's loads between its MFMAs
    // loads of 64 pieces, dealt to the waves (where they do not go up evenly, the last one to several)
    constexpr int AI = BM * 12 / 64, NAL = (AI + NW - 1) / NW;
    constexpr int KG = 4, WPC = 5, WROW = 16 * WPC, WI = WROWS / 64 * WPC, NWL = (WI + NW - 1) / NW, KS = KG / 2;
    __shared__ __attribute__((aligned(16))) uint8_t sa0[BM * MXG_ROW];
    __shared__ __attribute__((aligned(16))) uint8_t sa1[BM * MXG_ROW];
    __shared__ __attribute__((aligned(16))) uint8_t sa2[BM * MXG_ROW];
    __shared__ __attribute__((aligned(16))) uint8_t sw0[WROWS * WROW];
    __shared__ __attribute__((aligned(16))) uint8_t sw1[WROWS * WROW];
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
    // WROWS weight rows in LDS: those of the columns in order (GLU: half of them
    // gate rows, then the matching up rows), loaded by groups of 64.
    constexpr int CB = GLU ? WROWS / 2 : WROWS, CW = CB / WN;
    const int64_t c0 = (int64_t)cb * CB, n0 = c0 + CW * wc;
    __amdgpu_buffer_rsrc_t wrsrc[NWL];
    uint32_t woff[NWL];
#pragma unroll
    for (int i = 0; i < NWL; ++i) {
        const int j = imin(wave + NW * i, WI - 1), grp = j / WPC;
        const bool up = GLU && grp >= WROWS / 128;
        const ExpertMat &m = up && !s.fused ? s.b : s.a;
        // (rows past the matrix: its last row again, not stored)
        const int64_t r0 = c0 + 64 * (GLU ? grp % (WROWS / 128) : grp), first = r0 < s.ncols ? r0 : s.ncols - 1, left = s.ncols - first;
        const uint8_t *p = m.data + (int64_t)e * m.mat_bytes + (first + (up && s.fused ? s.I : 0)) * m.row_bytes;
        const uint32_t mis = (uint32_t)(uintptr_t)p & 3u, rb = (uint32_t)m.row_bytes, last = (left < 64 ? (uint32_t)left : 64u) - 1;
        // (a dword past the last row's bytes reads as zero)
        const uint32_t bytes = (mis + last * rb + (uint32_t)nb * MX_BYTES + 3) & ~3u;
        wrsrc[i] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p - mis), (short)0, (int)bytes, 0x00020000);
        const uint32_t q = 64u * (uint32_t)(j - grp * WPC) + (uint32_t)lane, r = q / (uint32_t)WPC, k = q - (uint32_t)WPC * r;
        woff[i] = ((mis + (r < last ? r : last) * rb) & ~3u) + 16u * k;
    }
    // stage sg's weights (the wave's loads i0 .. i1)
    auto load_w = [&](int sg, uint8_t *sw, int i0, int i1) __attribute__((always_inline)) {
        sg = imin(sg, (nb - 1) / KG);
#pragma unroll
        for (int i = i0; i < i1; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wrsrc[i], (lds_void_t *)(sw + 1024 * imin(wave + NW * i, WI - 1)), 16, (int)woff[i],
                                                     KG * MX_BYTES * sg, 0, 0);
    };
    // the lane's first weight row in LDS (column tile ct: 32 rows on per tile;
    // GLU: even tiles gate rows, odd ones up rows), and its rows' misalignment
    // (rows 32 apart have the same) + h
    const uint32_t wat = (uint32_t)(WROW * (CW * wc + l32) + 16 * h);
    uint32_t mh[2];
#pragma unroll
    for (int up = 0; up < (GLU ? 2 : 1); ++up) {
        const ExpertMat &m = up && !s.fused ? s.b : s.a;
        const int64_t row = c0 + CW * wc + l32 + (up && s.fused ? s.I : 0);
        mh[up] = ((uint32_t)((uintptr_t)m.data + (uintptr_t)((int64_t)e * m.mat_bytes + row * m.row_bytes)) & 3u) + (uint32_t)h;
    }
    // this lane's pieces of the activations (past the tile: out of range)
    const int kdiv = g.ne11 == 1 ? g.K : 1;
    const uint32_t drow = (uint32_t)mx_drow(nb);
    const __amdgpu_buffer_rsrc_t arsrc = __builtin_amdgcn_make_buffer_rsrc(s.x.d, (short)0, (int)(uint32_t)(s.xrows * (int64_t)drow), 0x00020000);
    uint32_t aoff[NAL];
#pragma unroll
    for (int i = 0; i < NAL; ++i) {
        const int q = 64 * imin(wave + NW * i, AI - 1) + lane, r = q / 12, k = (q - 12 * r) ^ ((r >> 2) & 3);
        const int p = r < mrows ? g.perm[start + r] : -1;
        aoff[i] = p < 0 ? MXG_FAR : (uint32_t)(kdiv > 1 ? p / kdiv : p) * drow + 16u * (uint32_t)k;
    }
    if (tid < BM) s_p[tid] = tid < mrows ? g.perm[start + tid] : 0;
    // step st's activations
    auto load_a = [&](int st, uint8_t *sa, int i0, int i1) __attribute__((always_inline)) {
        __amdgpu_buffer_rsrc_t r = arsrc;   // the builtin takes no const-qualified resource
        st = imin(st, ns - 1);
#pragma unroll
        for (int i = i0; i < i1; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t *)(sa + 1024 * imin(wave + NW * i, AI - 1)), 16, (int)aoff[i], MXG_ROW * st, 0, 0);
    };
    // the lane's row of scale words (past the tile: the tile's first row's), four blocks at a time
    const uint32_t *srow;
    {
        const int r = 32 * wr + l32, p = g.perm[start + (r < mrows ? r : 0)];
        srow = s.x.s + (int64_t)(kdiv > 1 ? p / kdiv : p) * mx_srow(nb);
    }
    auto load_s = [&](int gr) __attribute__((always_inline)) { return *(const u32x4 *)(srow + 4 * imin(gr, (nb - 1) / 4)); };
    // the lane's pieces of its activation row in LDS
    uint32_t xo[6];
#pragma unroll
    for (int k = 0; k < 6; ++k) xo[k] = (uint32_t)(MXG_ROW * (32 * wr + l32) + 16 * ((6 * h + k) ^ ((l32 >> 2) & 3)));
    f32x16 acc[C];
#pragma unroll
    for (int ct = 0; ct < C; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[ct][i] = 0.f;
    const bool rows = mrows > 32 * wr;   // the wave has rows
    load_w(0, sw0, 0, NWL);
    load_a(0, sa0, 0, NAL);
    load_w(1, sw1, 0, NWL);
    load_a(1, sa1, 0, NAL);
    load_a(2, sa2, 0, NAL);
    u32x4 sc[3] = {load_s(0), load_s(1), load_s(1)};
    MxgOps<C> ops[2];
    // the operands of step T of a stage out of LDS
#define MXG_TAKE(o, T, sa, sw)                                                                                     \
    {                                                                                                              \
        _Pragma("unroll") for (int ct = 0; ct < C; ++ct) mxg_read<T>((sw) + wat + WROW * (GLU ? WROWS / 2 * (ct & 1) + 32 * (ct / 2) : 32 * ct), (o).w[ct]); \
        _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                                            \
            (o).lo[i] = *(const u32x4 *)((sa) + xo[i]);                                                            \
            (o).hi[i] = *(const uint2 *)((sa) + xo[4 + (i >> 1)] + 8 * (i & 1));                                   \
        }                                                                                                          \
    }
    auto products = [&](const MxgOps<C> &o, auto T, int st, int sa, auto &&between) __attribute__((always_inline)) {
        i32x8 B[C];
        int sb[C];
#pragma unroll
        for (int ct = 0; ct < C; ++ct) {
            B[ct] = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
            mxg_unpack<T.value>(o.w[ct], mh[GLU ? ct & 1 : 0], B[ct], sb[ct]);
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
        if (rows) {
#pragma unroll
            for (int ct = 0; ct < C; ++ct) acc[ct] = mxg_mfma<0>(A[0], B[ct], acc[ct], sa, sb[ct]);
        }
        between(0);
        if (rows) {
#pragma unroll
            for (int ct = 0; ct < C; ++ct) acc[ct] = mxg_mfma<1>(A[1], B[ct], acc[ct], sa, sb[ct]);
        }
        between(1);
        if (rows) {
#pragma unroll
            for (int ct = 0; ct < C; ++ct) acc[ct] = mxg_mfma<2>(A[2], B[ct], acc[ct], sa, sb[ct]);
        }
        between(2);
        if (rows) {
#pragma unroll
            for (int ct = 0; ct < C; ++ct) acc[ct] = mxg_mfma<3>(A[3], B[ct], acc[ct], sa, sb[ct]);
        }
        between(3);
    };
    mxg_sync<0>();
    MXG_TAKE(ops[0], 0, sa0, sw0)
    mxg_sync<0>();
    // Step st = st0 + I: buffers by st % 3, stages by st / KS % 2, scale words by
    // st / 2 % 3, registers by st % 2: 6 KS steps to a turn.  The loads of step
    // st: scale words of step st + 4 (even steps), activations of step st + 3
    // over step st's, and after a stage's last step the stage after next over
    // it.  At its end at most its own loads are out.
#define MXG_A(k) ((k) % 3 == 0 ? sa0 : (k) % 3 == 1 ? sa1 : sa2)
#define MXG_W(k) ((k) / KS % 2 == 0 ? sw0 : sw1)
    // step st's loads, part k of n
    auto loads = [&](int st, auto I, int k, int n) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        load_a(st + 3, MXG_A(I.value), NAL * k / n, NAL * (k + 1) / n);
        if constexpr (I.value % KS == KS - 1) load_w(st / KS + 2, MXG_W(I.value), NWL * k / n, NWL * (k + 1) / n);
        __builtin_amdgcn_sched_barrier(0);
    };
    static_assert(6 * KS == 12, "steps of a turn");
#define MXG_STEP(I)                                                                       \
    {                                                                                     \
        if (st0 + (I) >= ns) break;                                                       \
        const u32x4 w4 = sc[(I) / 2 % 3];                                                 \
        const int sa = (int)((I) % 2 == 0 ? (h ? w4[1] : w4[0]) : (h ? w4[3] : w4[2]));   \
        if constexpr ((I) % 2 == 0) sc[((I) / 2 + 2) % 3] = load_s((st0 + (I)) / 2 + 2);  \
        asm volatile("" ::: "memory");                                                    \
        if constexpr (!SPREAD) loads(st0 + (I), Const<(I)>{}, 0, 1);                      \
        MXG_TAKE(ops[((I) + 1) & 1], ((I) + 1) % KS, MXG_A((I) + 1), MXG_W((I) + 1))      \
        products(ops[(I) & 1], Const<(I) % KS>{}, st0 + (I), sa, [&](int k) __attribute__((always_inline)) { \
            if constexpr (SPREAD) loads(st0 + (I), Const<(I)>{}, k, 4);                   \
        });                                                                               \
        mxg_sync<((I) % 2 == 0) + NAL + ((I) % KS == KS - 1) * NWL>();                    \
    }
    for (int st0 = 0;; st0 += 6 * KS) {
        MXG_STEP(0) MXG_STEP(1) MXG_STEP(2) MXG_STEP(3) MXG_STEP(4) MXG_STEP(5) MXG_STEP(6) MXG_STEP(7)
        MXG_STEP(8) MXG_STEP(9) MXG_STEP(10) MXG_STEP(11)
    }
#undef MXG_STEP
#undef MXG_TAKE
#undef MXG_A
#undef MXG_W
    mxg_sync<0>();   // (the loads past the last step)
    if (!rows) return;
    // accumulator i of the lane: row 8 (i / 4) + 4 h + i % 4 of the row tile, column l32
    if constexpr (EPI == MX_STORE) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int m = 32 * wr + 8 * (i >> 2) + 4 * h + (i & 3);
            if (m >= mrows) continue;
            // (nontemporal: 16384 rows of 2048 columns 245 -> 241 us)
            float *y = s.y + (int64_t)s_p[m] * s.ldy;
#pragma unroll
            for (int ct = 0; ct < C; ++ct) {
                const int64_t n = n0 + 32 * ct + l32;
                if (n < s.ncols) __builtin_nontemporal_store(acc[ct][i], y + n);
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
                v[(8 * (i >> 2) + 4 * h + (i & 3)) * 32 + l32] = GLU ? act_pair(g.act, acc[2 * ct][i], acc[2 * ct + 1][i]) : mx_relu_sqr(acc[ct][i]);
            wave_lds_sync();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int r = 16 * q + (lane >> 2), m = 32 * wr + r;
                float t[8];
                mx_load8<true>(v + 32 * r, lane & 3, t);
                const bool live = m < mrows && n < s.ncols;
                const int onb = (int)(s.ncols / 32), p = s_p[live ? m : 0];
                mx_store_block(t, s.o, p, n / 32, onb, lane & 3, live);
                if (live && n + 32 == s.ncols) mx_store_pad(s.o, p, onb, lane & 3);
            }
            wave_lds_sync();   // (rewritten next)
        }
    }
#endif
}

template <int EPI, int C, int WM, int WN>
static int mxg_launch(const MxArgs &a, hipStream_t st) {
    MxArgs g = a;
    constexpr int COLS = 32 * C * WN / (EPI == MX_GLU ? 2 : 1);   // per work-group
    g.ncb = (int)((g.ncols + COLS - 1) / COLS);
    const int64_t wgs = 8 * (int64_t)g.ncb * ((g.max_tiles + 7) / 8);
    if (wgs > 0x7fffffff) return -6;
    hipLaunchKernelGGL((k_mxg<EPI, C, WM, WN>), dim3((unsigned)wgs), dim3(64 * WM * WN), 0, st, g);
    return hip_check_launch();
}

template <int EPI>
static int mxg_tiles(const MxArgs &g, hipStream_t st) {
    return g.bm == MXG_BM ? mxg_launch<EPI, 4, 2, 2>(g, st) : mxg_launch<EPI, 2, 1, 2>(g, st);
}

int launch_mxg(const MxArgs &g, hipStream_t st) {
    if (g.max_tiles <= 0) return 0;
    if (g.bm != MXG_BM && g.bm != MXG_BM_SMALL) return -6;
    if (g.a.row_bytes > MXG_MAX_ROW_BYTES || (g.epi == MX_GLU && !g.fused && g.b.row_bytes > MXG_MAX_ROW_BYTES)) return -6;
    if (g.a.type != 39 || g.a.K % 32 || g.a.K > 0x7fffffff || (g.epi != MX_STORE && g.ncols % 32)) return -6;
    if (g.xrows <= 0 || g.xrows * mx_drow(g.a.K / 32) > MXG_MAX_X || (uintptr_t)g.x.d % 16 || (uintptr_t)g.x.s % 16) return -6;
    switch (g.epi) {
    case MX_STORE: return mxg_tiles<MX_STORE>(g, st);
    case MX_GLU: return mxg_tiles<MX_GLU>(g, st);
    case MX_RELU_SQR: return mxg_tiles<MX_RELU_SQR>(g, st);
    default: return -6;
    }
}

}  // namespace mimoe
