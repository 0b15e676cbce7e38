// k_mx.hip - MXFP4 expert tables (ggml type 39; format and operand: mx.hpp):
// the quantizer of weight rows, mi_dequantize, the operand rows of the
// products, and the grouped product of few rows per expert.  The grouped GEMM
// is k_mxg.hip.
#include "act.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "mx.hpp"

namespace mimoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------ quantizer
// e = floor(log2 amax) - 2 + 127, at least 0 (from the exponent bits: exact);
// a value's step is the number of midpoints of the E2M1 steps that |x| 2^(127
// - e) exceeds (ties to the smaller step, as ggml's search for the first
// nearest code gives them; above 6: 6), the scaling by a power of two exact.
// A block with an infinity or a NaN: e = 255, codes 0.
//
// Bound by the stream (4 B in, 17/32 B out a value).  A work-group takes 256
// blocks, four lanes a block (16-byte loads, a dword of codes per lane), and
// the 17-byte blocks leave through LDS in 16-byte stores: 2.7e8 values in 273
// us, 4.5 TB/s read and written (a large copy: 5.1).
constexpr int MXQ_BLOCKS = 256;

template <bool VEC>
__global__ void __launch_bounds__(256) k_quantize_mx(const float *__restrict__ src, uint8_t *__restrict__ dst, int64_t nblocks) {
    __shared__ __attribute__((aligned(16))) uint8_t so[MXQ_BLOCKS * MX_BYTES];
    const int64_t b0 = (int64_t)blockIdx.x * MXQ_BLOCKS;
    const int nb = nblocks - b0 < MXQ_BLOCKS ? (int)(nblocks - b0) : MXQ_BLOCKS;
    const int s = threadIdx.x & 3;
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = 64 * i + ((int)threadIdx.x >> 2);
        mx_load8<VEC>(src + 32 * (b0 + (b < nb ? b : nb - 1)), s, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = 64 * i + ((int)threadIdx.x >> 2);
        uint32_t a[8], m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            a[j] = __builtin_bit_cast(uint32_t, v[i][j]) & 0x7fffffffu;
            m = a[j] > m ? a[j] : m;
        }
        const uint32_t m1 = (uint32_t)dpp_i<0xB1>((int)m);
        m = m1 > m ? m1 : m;
        const uint32_t m2 = (uint32_t)dpp_i<0x4E>((int)m);
        m = m2 > m ? m2 : m;
        const int ex = (int)(m >> 23), e = ex == 255 ? 255 : ex > 2 ? ex - 2 : 0;
        uint32_t w = 0;
        if (e != 255) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float r = __builtin_ldexpf(__builtin_bit_cast(float, a[j]), 127 - e);
                const uint32_t c = (r > 0.25f) + (r > 0.75f) + (r > 1.25f) + (r > 1.75f) + (r > 2.5f) + (r > 3.5f) + (r > 5.0f);
                const uint32_t sign = c ? (__builtin_bit_cast(uint32_t, v[i][j]) >> 31) << 3 : 0u;   // (0 has no sign)
                w |= (c | sign) << (8 * (j & 3) + (j >= 4 ? 4 : 0));
            }
        }
        uint8_t *o = so + MX_BYTES * b;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[1 + 4 * s + j] = (uint8_t)(w >> (8 * j));
        if (s == 0) o[0] = (uint8_t)e;
    }
    __syncthreads();
    uint8_t *d = dst + MX_BYTES * b0;
    const int n = MX_BYTES * nb, n16 = (uintptr_t)d % 16 == 0 ? n / 16 : 0;
    for (int i = threadIdx.x; i < n16; i += 256) *(uint4 *)(d + 16 * i) = *(const uint4 *)(so + 16 * i);
    for (int i = 16 * n16 + (int)threadIdx.x; i < n; i += 256) d[i] = so[i];
}

int launch_quantize_mx(const float *src, void *dst, int64_t nblocks, hipStream_t st) {
    if (nblocks <= 0) return 0;
    const int64_t wgs = (nblocks + MXQ_BLOCKS - 1) / MXQ_BLOCKS;
    if (wgs > 0x7fffffff) return -6;
    if ((uintptr_t)src % 16 == 0) hipLaunchKernelGGL(k_quantize_mx<true>, dim3((unsigned)wgs), dim3(256), 0, st, src, (uint8_t *)dst, nblocks);
    else hipLaunchKernelGGL(k_quantize_mx<false>, dim3((unsigned)wgs), dim3(256), 0, st, src, (uint8_t *)dst, nblocks);
    return hip_check_launch();
}

// ------------------------------------------------------------------ rows to fp32
// Values of 32-value blocks (Q4_0, Q5_0, Q8_0, MXFP4) and F16 as fp32, each
// product exact or rounded once.  Bound by the stores.  A work-group takes 128
// blocks: their bytes reach LDS in dwords from the one at or below the first,
// each thread writes four consecutive values at a time.
constexpr int DQ_BLOCKS = 128;
template <int WT> constexpr int dq_bytes() { return WT == 1 ? 64 : WT == 2 ? 18 : WT == 6 ? 22 : WT == 8 ? 34 : MX_BYTES; }

template <int WT>
__device__ __forceinline__ void dq_values4(const uint8_t *b, int q, float (&o)[4]) {   // values 4 q .. 4 q + 3 of the block at b
    if constexpr (WT == 39) {
        const uint32_t e = b[0];
        // 2^(e - 127) as fp32 bits (e = 0: a denormal; 255: NaN)
        const float d = __builtin_bit_cast(float, e == 255u ? 0x7fc00000u : e ? e << 23 : 0x00400000u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c = (uint32_t)b[1 + 4 * (q & 3) + j] >> (q >= 4 ? 4 : 0);
            // twice the step, 0 1 2 3 4 6 8 12 as nibbles
            const float t = 0.5f * (float)((0xC8643210u >> (4 * (c & 7u))) & 15u);
            o[j] = (c & 8u ? -t : t) * d;
        }
    } else {
        auto half_at = [&](int i) __attribute__((always_inline)) { return fp16_bits_to_f32((uint32_t)b[i] | (uint32_t)b[i + 1] << 8); };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = 4 * q + j;
            if constexpr (WT == 1) o[j] = half_at(2 * i);
            else if constexpr (WT == 8) o[j] = half_at(0) * (float)(int8_t)b[2 + i];
            else {
                int c = (b[(WT == 6 ? 6 : 2) + (i & 15)] >> (i >= 16 ? 4 : 0)) & 15;
                if constexpr (WT == 6) c |= ((b[2 + (i >> 3)] >> (i & 7)) & 1) << 4;
                o[j] = half_at(0) * (float)(c - (WT == 6 ? 16 : 8));
            }
        }
    }
}

template <int WT>
__global__ void __launch_bounds__(256) k_dequantize(const uint8_t *__restrict__ src, float *__restrict__ dst, int64_t nblocks) {
    constexpr int BB = dq_bytes<WT>();
    __shared__ uint32_t sw[(DQ_BLOCKS * BB + 8) / 4];
    const int64_t b0 = (int64_t)blockIdx.x * DQ_BLOCKS;
    const int nb = nblocks - b0 < DQ_BLOCKS ? (int)(nblocks - b0) : DQ_BLOCKS;
    const uint8_t *p = src + BB * b0;
    const int mis = (int)((uintptr_t)p & 3u), nw = (mis + BB * nb + 3) / 4;   // (every dword holds a byte of the blocks)
    for (int i = threadIdx.x; i < nw; i += 256) sw[i] = ((const uint32_t *)(p - mis))[i];
    __syncthreads();
    const uint8_t *b = (const uint8_t *)sw + mis;
    float *o = dst + 32 * b0;
    const bool vec = (uintptr_t)dst % 16 == 0;
    for (int i = threadIdx.x; i < 8 * nb; i += 256) {
        float v[4];
        dq_values4<WT>(b + BB * (i >> 3), i & 7, v);
        if (vec) *(float4 *)(o + 4 * i) = make_float4(v[0], v[1], v[2], v[3]);
        else {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[4 * i + j] = v[j];
        }
    }
}

int launch_dequantize(int type, const void *src, float *dst, int64_t nblocks, hipStream_t st) {
    if (nblocks <= 0) return 0;
    const int64_t wgs = (nblocks + DQ_BLOCKS - 1) / DQ_BLOCKS;
    if (wgs > 0x7fffffff) return -6;
    const dim3 grid((unsigned)wgs), block(256);
    const uint8_t *s = (const uint8_t *)src;
    switch (type) {
    case 1: hipLaunchKernelGGL(k_dequantize<1>, grid, block, 0, st, s, dst, nblocks); break;
    case 2: hipLaunchKernelGGL(k_dequantize<2>, grid, block, 0, st, s, dst, nblocks); break;
    case 6: hipLaunchKernelGGL(k_dequantize<6>, grid, block, 0, st, s, dst, nblocks); break;
    case 8: hipLaunchKernelGGL(k_dequantize<8>, grid, block, 0, st, s, dst, nblocks); break;
    case 39: hipLaunchKernelGGL(k_dequantize<39>, grid, block, 0, st, s, dst, nblocks); break;
    default: return -3;
    }
    return hip_check_launch();
}

// ------------------------------------------------------------------ operand rows
// Rows of K values (K % 32 == 0, row r at src + r * ld) into the operand
// (mx.hpp): four threads per block.  Memory-bound.
template <bool VEC>
__global__ void __launch_bounds__(256) k_prep_mx(const float *__restrict__ src, int64_t ld, int64_t nrows, int nb, MxRows o, bool few) {
    mx_prep_thread<VEC>(src, ld, nrows, nb, o, few, (int64_t)blockIdx.x * 256 + threadIdx.x);
}

int launch_prep_mx(const float *src, int64_t ld, int64_t nrows, int64_t K, const MxRows &o, bool few, hipStream_t st) {
    if (nrows <= 0) return 0;
    if (K % 32 || K > 0x7fffffff) return -6;
    const int64_t wgs = (nrows * (K / 8) + 255) / 256;
    if (wgs > 0x7fffffff) return -6;
    if (mx_prep_vec(src, ld))
        hipLaunchKernelGGL(k_prep_mx<true>, dim3((unsigned)wgs), dim3(256), 0, st, src, ld, nrows, (int)(K / 32), o, few);
    else hipLaunchKernelGGL(k_prep_mx<false>, dim3((unsigned)wgs), dim3(256), 0, st, src, ld, nrows, (int)(K / 32), o, few);
    return hip_check_launch();
}

// ------------------------------------------------------------------ few rows
// act_pair (act.hpp) in fp64, rounded once: a value that differs in its last
// bits would move an 8-bit code of the operand that it becomes.  (A call: inlined,
// the constants of exp and erf are kept in registers through the products'
// loops and do not fit.)
template <int ACT>
__device__ __attribute__((noinline)) float mx_act(double a, double b) {
    const double SQRT_2_INV = 0.70710678118654752440, SQRT_2_OVER_PI = 0.79788456080286535588;
    if constexpr (ACT == 0) return (float)(a / (1.0 + exp(-a)) * b);
    else if constexpr (ACT == 1) return (float)(0.5 * a * (1.0 + erf(a * SQRT_2_INV)) * (b + 1.0));
    // (1 + tanh(u)) / 2 = 1 / (1 + exp(-2 u))
    else if constexpr (ACT == 2) return (float)(a / (1.0 + exp(-2.0 * SQRT_2_OVER_PI * a * (1.0 + 0.044715 * a * a))) * b);
    else if constexpr (ACT == 3) return (float)(0.5 * a * (1.0 + erf(a * SQRT_2_INV)) * b);
    else return (float)mx_relu_sqr(a);
}

// A 16-row weight tile times rows of activations, by one wave: the lane's
// blocks of its weight row (row lane % 16; step u's block 4 (s0 + u) + lane /
// 16) in registers, the activations in LDS.
//
// A step is v_mfma_scale_f32_16x16x128_f8f6f4 on four blocks of the 16 rows
// (the 16 bytes of codes as they are) against two rows of activations: column
// c = 8 j + 2 b + i holds digit i of row j's block b of the step and zeros in
// the other three blocks, so each of the 16 x 16 results is one digit's sum
// over one block, an integer of at most 13 bits times a power of two: exact in
// fp32 as long as that lies in its normal range (both scales are in it: a sum
// past 2^128 is infinite, one below 2^-126 may be zero).  Times the block's
// significand they are added in fp64, so the result is the exact sum but for
// roundings at 2^-53, and what follows (the GLU's values, in fp64 and rounded
// once, and their codes) does not depend on an order of sums unless a value
// lies that near to a border.  What bounds it beside the weights' bytes is the vector
// work of a step (unpacking 17-byte blocks, four conversions and fp64
// multiply-adds): two rows share it all; with the significand in the digits
// (four, a column of each) a row had it alone, and 120 rows of 64 experts
// (K 2048, 2048 rows) took 60 us instead of 52.
//
// Loads: two per step and lane (the five dwords of its block, at dword
// aligned addresses), 68 bytes of a row together; the load path takes such a
// step in about 50 cycles (22 B per cycle and CU, twice the HBM's share).
template <int U>
struct MxTile {
    MxRaw w[U];
    const uint8_t *row;   // the lane's weight row
    // steps s0 .. s0 + sn - 1 of the row's blocks, of which there are nb
    __device__ __forceinline__ void load(int s0, int sn, int nb, int lane) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = 4 * (s0 + u) + (lane >> 4);
            if (u < sn) mx_load(row + MX_BYTES * (int64_t)(b < nb ? b : 0), w[u]);   // (past the row: block 0; the operand is zero there)
        }
    }
    // acc += steps s0 .. times the n (1 or 2) rows whose digits (blocks filled
    // up to whole steps with zeros) from step sx on are at x + xo[j] and words
    // at xs[j]; 16 zeros at x + zo.  All in LDS.
    __device__ __forceinline__ void products(int s0, int sn, int nb, int lane, const uint8_t *x, const int (&xo)[2], int zo, const uint32_t *const (&xs)[2],
                                             int sx, int n, double (&acc)[4]) const {
        const int r16 = lane & 15, grp = lane >> 4, j = r16 >> 3, b = (r16 >> 1) & 3, dig = r16 & 1;
        const bool on = b == grp && j < n;   // the lane's column holds a digit of the lane's block
        const int at = (j ? xo[1] : xo[0]) + MX_FB * (4 * (s0 - sx) + grp), stride = on ? 4 * MX_FB : 0;
        const uint8_t *lo = x + (on ? at + 16 * dig : zo), *hi = x + (on ? at + 32 + 8 * dig : zo);
        const uint32_t *word = (j && n > 1 ? xs[1] : xs[0]) + 4 * (s0 - sx) + b;
        // (four blocks are 68 bytes: the lane's blocks are all misaligned alike)
        const uint32_t mis = (uint32_t)((uintptr_t)row + (uint32_t)(MX_BYTES * grp)) & 3u;
        const auto step = [&](int u) __attribute__((always_inline)) {
            uint32_t c[4];
            mx_codes(w[u], mis, c);
            int sa = (int)mx_scale(w[u], mis);
            // (past the row's last block: any codes, times zeros)
            if (4 * (s0 + u) + 4 > nb) sa = 4 * (s0 + u) + grp < nb ? sa : (int)MX_ONE;
            const i32x8 A = {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
            const uint4 xl = *(const uint4 *)(lo + stride * u);
            const uint2 xh = *(const uint2 *)(hi + stride * u);
            const uint32_t wd = word[4 * u];
            const i32x8 B = {(int)xl.x, (int)xl.y, (int)xl.z, (int)xl.w, (int)xh.x, (int)xh.y, 0, 0};
            float4_t z = {0.f, 0.f, 0.f, 0.f};
            z = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, z, 4, 2, 0, sa, 0, (int)(wd + 5u * (uint32_t)dig));
            const double f = (double)__builtin_bit_cast(float, wd & 0xffffff00u);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fma((double)z[i], f, acc[i]);
        };
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u < sn) step(u);
    }
};

// rows 4 (lane / 16) + i, a partial per column: the sum over a row of
// activations' 8 columns
__device__ __forceinline__ double mx_columns(double a) {
    a = dpp_add<0xB1>(a);
    a = dpp_add<0x4E>(a);
    return dpp_add<0x141>(a);
}

// Grouped product of few rows per expert.  A work-group (8 waves) owns 64
// weight rows of one active expert (GLU: 32 gate rows and the matching up
// rows) as four 16-row tiles, two waves to a tile, each half of the blocks.
// The expert's rows run MXV_NT at a time through LDS, the lanes' weight blocks
// staying in registers for all of them (rows of at most MXV_KB blocks; longer
// ones are loaded again).  Its time is its chain: one row through 8 experts (K
// 2048, 1536 rows each) 8.9 us, 13.4 MB; with ranking and GLU 12, of which the
// ranking is 2.0, the weights' latency 2.7, the products 1.3, the GLU 0.5.
//
// With g.logits the work-group ranks the tokens' experts itself (a wave per
// token) and finds its rows among them, with g.ids it finds them among the
// ids: work-group row j belongs to slot j, and leaves unless the slot is its
// expert's first.
constexpr int MXV_NT = 2, MXV_WAVES = 8, MXV_U = 8;   // U: steps of a wave in registers at a time
constexpr int MXV_KB = 4 * 2 * MXV_U;                  // blocks of a pass over K (both wave halves)

// ACT: the activation, or -1 for the plain product
template <int ACT, bool SH>
__global__ void __launch_bounds__(64 * MXV_WAVES) __attribute__((amdgpu_waves_per_eu(4))) k_mxv(MxArgs g) {
    constexpr int XROW = MXV_KB * MX_FB, ZERO = MXV_NT * XROW;
    __shared__ __attribute__((aligned(16))) uint8_t sx[ZERO + 16];   // (16 zeros last)
    __shared__ uint32_t ss[MXV_NT][MXV_KB];
    __shared__ double s_sum[MXV_NT][128];
    __shared__ __attribute__((aligned(16))) float s_v[MXV_NT][64];
    __shared__ int s_p[MXV_IDS];
    __shared__ int s_cnt[MXV_WAVES];
    constexpr bool STORE = ACT < 0, GLU = !STORE && ACT != ACT_RELU_SQR;
    constexpr int COLS = GLU ? 32 : 64;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const bool shared = SH && (int)blockIdx.x < g.sh_wgs;
    const MxSide s = shared ? g.sh : (const MxSide &)g;
    int e = 0, cnt, cb;
    const int32_t *perm = nullptr;   // the rows (null: in s_p)
    if (shared) {
        cb = blockIdx.x;
        cnt = (int)g.sh_rows;
    } else {
        const unsigned lin = blockIdx.x - (SH ? g.sh_wgs : 0), j = lin / (unsigned)g.ncb;
        cb = (int)(lin - j * (unsigned)g.ncb);
        if (g.ids || (!STORE && g.logits)) {
            int id;
            if (!STORE && g.logits) {
                // (s_p holds the ids until the rows are found: at most MXV_FRONT_T tokens)
                const int T = (int)(g.rows / g.K);
                if (wave < T) {
                    int mysel;
                    float myw;
                    topk_softmax_wave(g.logits + wave * g.n_expert, g.n_expert, g.K, lane, mysel, myw, lin == 0, g.gating);
                    if (lane < g.K) {
                        s_p[wave * g.K + lane] = mysel;
                        if (lin == 0) {
                            g.sel[wave * g.K + lane] = mysel;
                            g.w[wave * g.K + lane] = myw;
                        }
                    }
                }
                __syncthreads();
                id = tid < g.rows ? s_p[tid] : -1;
                e = s_p[j];
                __syncthreads();
            } else {
                id = tid < g.rows ? g.ids[tid] : -1;
                e = g.ids[j];
            }
            if ((unsigned)e >= (unsigned)g.n_expert) {
                if (g.bad_total && cb == 0 && tid == 0) atomicAdd(g.bad_total, 1);
                if (STORE && g.zero_rows && tid < COLS && (int64_t)cb * COLS + tid < s.ncols) s.y[j * s.ldy + (int64_t)cb * COLS + tid] = 0.f;
                return;
            }
            const uint64_t m = __ballot(id == e);
            if (lane == 0) s_cnt[wave] = __popcll(m);
            __syncthreads();
            int before = 0, total = 0;
#pragma unroll
            for (int i = 0; i < MXV_WAVES; ++i) {
                if (i < wave) before += s_cnt[i];
                total += s_cnt[i];
            }
            if (id == e) s_p[before + __popcll(m & ((1ull << lane) - 1))] = tid;
            __syncthreads();
            if (s_p[0] != (int)j) return;
            cnt = total;
        } else {
            if ((int)j >= *g.n_active) return;
            e = g.active_e[j];
            cnt = g.counts[e];
            perm = g.perm + g.offsets[e];
        }
    }
    if (tid < 4) ((uint32_t *)(sx + ZERO))[tid] = 0;
    const int tile = wave >> 1, half = wave & 1, r16 = lane & 15, grp = lane >> 4;
    // the lane's weight row (past the matrix: row 0, not stored)
    const int64_t col = (int64_t)cb * COLS + 16 * (GLU ? tile & 1 : tile) + r16;
    const int64_t wrow = (col < s.ncols ? col : 0) + (GLU && tile >= 2 && s.fused ? s.I : 0);
    const ExpertMat &wm = GLU && tile >= 2 && !s.fused ? s.b : s.a;
    MxTile<MXV_U> w;
    w.row = wm.data + (int64_t)e * wm.mat_bytes + wrow * wm.row_bytes;
    const int nb = (int)(s.a.K / 32);
    const int kdiv = g.ne11 == 1 && !shared ? g.K : 1;
    for (int q0 = 0; q0 < cnt; q0 += MXV_IDS) {   // (rows that fit s_p)
        const int qn = cnt - q0 < MXV_IDS ? cnt - q0 : MXV_IDS;
        if (shared || perm) {
            if (q0) __syncthreads();
            for (int i = tid; i < qn; i += 64 * MXV_WAVES) s_p[i] = shared ? q0 + i : perm[q0 + i];
            __syncthreads();
        }
        for (int n0 = 0; n0 < qn; n0 += MXV_NT) {
            const int nt = qn - n0 < MXV_NT ? qn - n0 : MXV_NT;
            double acc[MXV_NT / 2][4];
#pragma unroll
            for (int n = 0; n < MXV_NT / 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][i] = 0.0;
            for (int k0 = 0; k0 < nb; k0 += MXV_KB) {
                const int kn = nb - k0 < MXV_KB ? nb - k0 : MXV_KB, nst = (kn + 3) / 4, h0 = (nst + 1) / 2;
                const int s0 = k0 / 4 + (half ? h0 : 0), sn = half ? nst - h0 : h0;   // the wave's steps
                // the rows' operands (in front of the weights' loads: they are
                // stored to LDS while those are on their way)
                const bool fx = STORE && !shared && g.xf;
                static_assert(2 * MXV_KB * MX_FB / 16 <= 64 * MXV_WAVES && 8 * MXV_KB <= 64 * MXV_WAVES && MXV_NT % 2 == 0, "a piece, or a quarter block, of two rows per thread");
                // this thread's piece xi (fx: quarter of block xi / 4) of rows xn, xn + 2, ..; rows are filled up to whole steps
                const int per = fx ? 4 * kn : 3 * 4 * nst, xn = tid >= per ? 1 : 0, xi = tid - (xn ? per : 0);
                u32x4 xv[MXV_NT / 2][2];
                uint32_t xs1[MXV_NT / 2];
#pragma unroll
                for (int n = 0; n < MXV_NT / 2; ++n) {
                    xv[n][0] = xv[n][1] = u32x4{0, 0, 0, 0};
                    xs1[n] = MX_ONE;
                    if (2 * n + xn >= nt || xi >= per) continue;
                    const int p = s_p[n0 + 2 * n + xn];
                    const int64_t r = kdiv > 1 ? p / kdiv : p;
                    if (fx) {
                        const u32x4 *src = (const u32x4 *)(g.xf + r * s.a.K + 32 * (k0 + (xi >> 2))) + (xi & 3);
                        xv[n][0] = src[0];
                        xv[n][1] = src[4];
                    } else {
                        if (xi < 3 * kn) xv[n][0] = ((const u32x4 *)(s.x.d + r * (int64_t)(nb * MX_FB) + (int64_t)MX_FB * k0))[xi];
                        if (xi < kn) xs1[n] = s.x.s[r * nb + k0 + xi];
                    }
                }
                asm volatile("" ::: "memory");
                if (nb > MXV_KB || (n0 == 0 && q0 == 0)) w.load(s0, sn, nb, lane);
                if (k0 || n0 || q0) __syncthreads();   // (the activations before are read)
#pragma unroll
                for (int n = 0; n < MXV_NT / 2; ++n) {
                    if (2 * n >= nt) continue;
                    const int m = 2 * n + xn;
                    if (fx) {
                        const MxRows o = {sx + XROW * m, ss[m]};
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, (uint32_t)xv[n][i >> 2][i & 3]);
                        mx_store_few(v, o, 0, xi >> 2, 0, xi & 3, xi < per);
                        // (the blocks that fill up the last step)
                        if (tid < 3 * (4 * nst - kn)) {
                            *(u32x4 *)(sx + XROW * 2 * n + MX_FB * kn + 16 * tid) = u32x4{0, 0, 0, 0};
                            *(u32x4 *)(sx + XROW * (2 * n + 1) + MX_FB * kn + 16 * tid) = u32x4{0, 0, 0, 0};
                        }
                        if (tid < 4 * nst - kn) ss[2 * n][kn + tid] = ss[2 * n + 1][kn + tid] = MX_ONE;
                    } else if (xi < per) {
                        *(u32x4 *)(sx + XROW * m + 16 * xi) = xv[n][0];
                        if (xi < 4 * nst) ss[m][xi] = xs1[n];
                    }
                }
                __syncthreads();
#pragma unroll
                for (int n = 0; n < MXV_NT / 2; ++n) {
                    if (2 * n >= nt) continue;
                    const int xo[2] = {XROW * 2 * n, XROW * (2 * n + 1)};
                    const uint32_t *const xs[2] = {ss[2 * n], ss[2 * n + 1]};
                    w.products(s0, sn, nb, lane, sx, xo, ZERO, xs, k0 / 4, nt - 2 * n, acc[n]);
                }
            }
#pragma unroll
            for (int n = 0; n < MXV_NT / 2; ++n) {
                if (2 * n >= nt) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const double a = mx_columns(acc[n][i]);
                    if ((r16 & 7) == 0) s_sum[2 * n + (r16 >> 3)][64 * half + 16 * tile + 4 * grp + i] = a;
                }
            }
            __syncthreads();
            if constexpr (STORE) {
                const int c = tid & 63, n = tid >> 6;
                const int64_t cc = (int64_t)cb * COLS + c;
                if (n < nt && cc < s.ncols) {
                    const int p = s_p[n0 + n];
                    const float v = (float)(s_sum[n][c] + s_sum[n][64 + c]);
                    s.y[(int64_t)p * s.ldy + cc] = shared && g.sh_w ? v * g.sh_w[p] : v;
                }
            } else {
                // the next product's operand: each 32 columns are a block
                const int c = tid % COLS, n = tid / COLS;
                if (n < nt) {
                    const double a = s_sum[n][c] + s_sum[n][64 + c];
                    const double b = GLU ? s_sum[n][32 + c] + s_sum[n][96 + c] : 0.0;
                    s_v[n][c] = mx_act<ACT>(a, b);
                }
                __syncthreads();
                if (tid < MXV_NT * COLS / 8) {
                    const int m = tid / (COLS / 8), blk = (tid >> 2) % (COLS / 32), onb = (int)(s.ncols / 32);
                    float v[8];
                    mx_load8<true>(s_v[m] + 32 * blk, tid & 3, v);
                    const int64_t r = m < nt ? s_p[n0 + m] : 0, b = (int64_t)cb * (COLS / 32) + blk;
                    mx_store_few(v, s.o, r, b, onb, tid & 3, m < nt && b < onb);
                }
            }
            // (s_sum and s_v are written again after the barriers in front of the next rows' products)
        }
    }
}

template <int ACT>
static int mxv_launch(const MxArgs &a, hipStream_t st) {
    MxArgs g = a;
    constexpr int COLS = ACT >= 0 && ACT != ACT_RELU_SQR ? 32 : 64;
    g.ncb = (int)((g.ncols + COLS - 1) / COLS);
    g.sh_wgs = g.sh_rows > 0 ? (int)((g.sh.ncols + COLS - 1) / COLS) : 0;
    const int64_t wgs = g.sh_wgs + (int64_t)g.ncb * (g.ids || g.logits ? g.rows : g.max_active);
    if (wgs > 0x7fffffff) return -6;
    const dim3 grid((unsigned)wgs), block(64 * MXV_WAVES);
    if (g.sh_wgs) hipLaunchKernelGGL((k_mxv<ACT, true>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((k_mxv<ACT, false>), grid, block, 0, st, g);
    return hip_check_launch();
}

static bool mx_side_ok(const MxArgs &g, const MxSide &s) {
    return s.a.type == 39 && s.a.K % 32 == 0 && s.a.K <= 0x7fffffff && !(g.epi != MX_STORE && s.ncols % 32);
}

int launch_mxv(const MxArgs &g, hipStream_t st) {
    if (g.max_active <= 0) return 0;
    if (!mx_side_ok(g, g) || (g.sh_rows > 0 && !mx_side_ok(g, g.sh))) return -6;
    if ((g.ids || g.logits) && (g.rows > MXV_IDS || g.n_expert <= 0)) return -6;
    if (g.logits && (g.epi == MX_STORE || g.rows > (int64_t)MXV_FRONT_T * g.K || g.rows % g.K || g.K > 64 || g.n_expert > 64 * TOPK_MAX_PER_LANE)) return -6;
    if (g.xf && (g.epi != MX_STORE || (uintptr_t)g.xf % 16)) return -6;
    if (g.epi == MX_STORE) return mxv_launch<-1>(g, st);
    if (g.epi == MX_RELU_SQR) return mxv_launch<ACT_RELU_SQR>(g, st);
    switch (g.act) {
    case 0: return mxv_launch<0>(g, st);
    case 1: return mxv_launch<1>(g, st);
    case 2: return mxv_launch<2>(g, st);
    case 3: return mxv_launch<3>(g, st);
    default: return -6;
    }
}

// ------------------------------------------------------------------ a few tokens' layer: front
// The norm, the router's logits and the operand rows of up to MXV_FRONT_T
// tokens in one launch: a wave per expert, lane c the row's 64-value chunk c
// in the router's fixed fp64 order (k_route.hip: s outer, g inner; chunk
// partials in chunk order, those of token t by lane t).  The router's rows are
// read in address order and go through LDS like the tokens' rows (chunk c's
// float4 q at slot 16 c + (q + c) % 16: 16 lanes that read chunks c .. c + 15
// hit 16 different slots); reading its chunk by itself each lane of a load is
// on a line of its own, and a launch of 64 experts (D 2048) takes 7.6 us
// instead of 5.8.  Every work-group normalizes the tokens' rows itself, a wave per
// token in k_norm_rows' order (the bits of mi_norm), while its router rows are
// on their way; the operand blocks are dealt to the work-groups.
constexpr int MXF_WAVES = 4;
static_assert(MXV_FRONT_T <= MXF_WAVES, "a wave per token");

__device__ __forceinline__ int mxf_slot(int c, int q) { return 16 * c + ((q + c) & 15); }

// k_norm_rows' sum of the NORM_T threads' partials, thread t = lane + 64 m at p[m]
__device__ __forceinline__ double mxf_norm_sum(double (&p)[4]) {
    double r = (p[0] + p[2]) + (p[1] + p[3]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t b = __builtin_bit_cast(uint64_t, r);
        const uint64_t n = ((uint64_t)(uint32_t)__shfl_down((int)(b >> 32), o, 64) << 32) | (uint32_t)__shfl_down((int)(uint32_t)b, o, 64);
        r = r + __builtin_bit_cast(double, n);
    }
    const uint64_t b = __builtin_bit_cast(uint64_t, r);
    return __builtin_bit_cast(double, ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) |
                                          (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b));
}

// four floats at p, aligned to one
__device__ __forceinline__ float4_t mxf_load4(const float *p) {
    float4_t v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, 4), 16);
    return v;
}

template <int DM>   // D <= 1024 DM
__global__ void __launch_bounds__(64 * MXF_WAVES) k_mx_front(MxFrontArgs g) {
    __shared__ __attribute__((aligned(16))) float4 sx[MXV_FRONT_T][256 * DM];
    __shared__ __attribute__((aligned(16))) float4 sw[MXF_WAVES][256 * DM];
    __shared__ double sp[MXF_WAVES][MXV_FRONT_T][65];
    static_assert(16 * DM <= 64, "a chunk per lane");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int D = g.D, nch = D >> 6, e = blockIdx.x * MXF_WAVES + wave;
    // (a row past the experts: row 0, not stored)
    float4_t w[4 * DM];
    const float *wr = g.W + (int64_t)(e < g.E ? e : 0) * D;
#pragma unroll
    for (int m = 0; m < 4 * DM; ++m) w[m] = 256 * m + 4 * lane < D ? *(const float4_t *)(wr + 256 * m + 4 * lane) : float4_t{0.f, 0.f, 0.f, 0.f};
    if (wave < g.T) {
        const float *x = g.xr + (int64_t)wave * D;
        float v[DM][4][4];   // piece k, m: elements 1024 k + 4 (lane + 64 m) + j
#pragma unroll
        for (int k = 0; k < DM; ++k)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int i = 1024 * k + 4 * (lane + 64 * m);
                const float4_t a = i < D ? *(const float4_t *)(x + i) : float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 4; ++j) v[k][m][j] = a[j];
            }
        float mean = 0.f, sc = 1.f;
        float4_t nw[DM][4], nbias[DM][4];   // (norm_apply's, read beside the rows)
        if (g.norm.kind != NORM_NONE) {
#pragma unroll
            for (int k = 0; k < DM; ++k)
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int i = 1024 * k + 4 * (lane + 64 * m);
                    nw[k][m] = g.norm.w && i < D ? mxf_load4(g.norm.w + i) : float4_t{0.f, 0.f, 0.f, 0.f};
                    nbias[k][m] = g.norm.kind == NORM_LAYER && g.norm.b && i < D ? mxf_load4(g.norm.b + i) : float4_t{0.f, 0.f, 0.f, 0.f};
                }
            double p[4];
            if (g.norm.kind == NORM_LAYER) {
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    p[m] = 0.0;
#pragma unroll
                    for (int k = 0; k < DM; ++k)
#pragma unroll
                        for (int j = 0; j < 4; ++j) p[m] = p[m] + (double)v[k][m][j];
                }
                mean = (float)(mxf_norm_sum(p) / (double)D);
            }
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                p[m] = 0.0;
#pragma unroll
                for (int k = 0; k < DM; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (1024 * k + 4 * (lane + 64 * m) + j < D) {
                            const float d = g.norm.kind == NORM_LAYER ? v[k][m][j] - mean : v[k][m][j];
                            p[m] = p[m] + (double)(d * d);
                        }
            }
            sc = 1.0f / sqrtf((float)(mxf_norm_sum(p) / (double)D) + g.norm.eps);
        }
#pragma unroll
        for (int k = 0; k < DM; ++k)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int i = 1024 * k + 4 * (lane + 64 * m);
                if (i >= D) continue;
                float o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // norm_apply
                    o[j] = v[k][m][j];
                    if (g.norm.kind != NORM_NONE) o[j] = (g.norm.kind == NORM_RMS ? o[j] : o[j] - mean) * sc;
                    if (g.norm.kind != NORM_NONE && g.norm.w) o[j] = o[j] * nw[k][m][j];
                    if (g.norm.kind == NORM_LAYER && g.norm.b) o[j] = o[j] + nbias[k][m][j];
                }
                sx[wave][mxf_slot(i >> 6, (i & 63) >> 2)] = make_float4(o[0], o[1], o[2], o[3]);
            }
    }
#pragma unroll
    for (int m = 0; m < 4 * DM; ++m) {
        const int i = 256 * m + 4 * lane;
        if (i < D) sw[wave][mxf_slot(i >> 6, (i & 63) >> 2)] = make_float4(w[m][0], w[m][1], w[m][2], w[m][3]);
    }
    __syncthreads();
    // operand blocks: four threads each, from the rows in LDS or (another router input) from x
    const int nb = D >> 5;
    for (int i = blockIdx.x * (64 * MXF_WAVES) + tid; i < 4 * nb * g.T; i += gridDim.x * (64 * MXF_WAVES)) {
        const int t = (i >> 2) / nb, b = (i >> 2) - t * nb, s = i & 3;
        float v[8];
        if (g.x == g.xr) {
            const float4 lo = sx[t][mxf_slot(b >> 1, 8 * (b & 1) + s)], hi = sx[t][mxf_slot(b >> 1, 8 * (b & 1) + 4 + s)];
            v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
        } else {
            mx_load8<true>(g.x + (int64_t)t * D + 32 * b, s, v);
        }
        mx_store_few(v, g.o, t, b, nb, s, true);
    }
    // (a lane past the chunks: chunk 0, not added; tokens past g.T: the last one's row again)
    const int c = lane < nch ? lane : 0;
    double part[MXV_FRONT_T];
    const float4 *xt[MXV_FRONT_T];
#pragma unroll
    for (int t = 0; t < MXV_FRONT_T; ++t) {
        part[t] = 0.0;
        xt[t] = sx[imin(t, g.T - 1)];
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        float wv[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) *(float4 *)wv[q] = sw[wave][mxf_slot(c, 4 * q + s)];
#pragma unroll
        for (int t = 0; t < MXV_FRONT_T; ++t) {
            if (t >= g.T) continue;
            float xv[4][4];
#pragma unroll
            for (int q = 0; q < 4; ++q) *(float4 *)xv[q] = xt[t][mxf_slot(c, 4 * q + s)];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) part[t] = fma((double)wv[q][j], (double)xv[q][j], part[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < MXV_FRONT_T; ++t) sp[wave][t][lane] = lane < nch ? part[t] : 0.0;
    wave_lds_sync();
    if (lane < g.T && e < g.E) {
        // (zeros past the chunks: a sum from 0.0 on keeps its bits)
        double acc = 0.0;
#pragma unroll
        for (int k = 0; k < 16 * DM; ++k) acc = acc + sp[wave][lane][k];
        float v = (float)acc;
        if (g.b) v = v + g.b[e];
        g.logits[(int64_t)lane * g.E + e] = v;
    }
}

bool mx_front_ok(const MxFrontArgs &g) {
    return g.T >= 1 && g.T <= MXV_FRONT_T && g.D % 64 == 0 && g.D <= 4096 && (uintptr_t)g.W % 16 == 0 && (uintptr_t)g.x % 16 == 0 &&
           (uintptr_t)g.xr % 16 == 0;
}

int launch_mx_front(const MxFrontArgs &g, hipStream_t st) {
    if (!mx_front_ok(g) || (g.norm.kind != NORM_NONE && g.x != g.xr)) return -6;
    const dim3 grid((unsigned)((g.E + MXF_WAVES - 1) / MXF_WAVES)), block(64 * MXF_WAVES);
    if (g.D <= 2048) hipLaunchKernelGGL(k_mx_front<2>, grid, block, 0, st, g);
    else hipLaunchKernelGGL(k_mx_front<4>, grid, block, 0, st, g);
    return hip_check_launch();
}

// ------------------------------------------------------------------ a few tokens' layer: down
// The down product of all slots of a token, the shared expert's with them, the
// weighted sum and the residual in one launch: a work-group owns COLS columns
// of one token, wave k (k + 8, ..) a 16-row tile of slot k's expert.  With
// COLS = 8 the tile's upper eight rows are the lower ones again (no traffic):
// twice the work-groups for a call of one token.  The sums have the bits of
// launch_combine on the slots' rounded rows.  Work-group 8 q + x on XCD x: the
// tokens of a column group one after another on one XCD, whose L2 then holds
// the experts' rows that they share.  One token through 8 experts (K 1024, 2048
// columns) 5.8 us, 15 tokens 32.5 (the product, then the sum, as launches of
// their own: 50 and 4).
constexpr int MXD_WAVES = 8, MXD_U = 8, MXD_KMAX = 64;

template <int COLS>
__global__ void __launch_bounds__(64 * MXD_WAVES) __attribute__((amdgpu_waves_per_eu(4))) k_mxd(MxDownArgs g) {
    constexpr int XROW = 4 * MXD_U * MX_FB;
    __shared__ __attribute__((aligned(16))) uint8_t sx[MXD_WAVES * XROW + 16];   // (16 zeros last)
    __shared__ __attribute__((aligned(16))) uint32_t ss[MXD_WAVES][4 * MXD_U];
    __shared__ float s_z[MXD_KMAX + 1][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int q = blockIdx.x >> 3, grp = q / g.T, t = q - grp * g.T;
    const int64_t n0 = (int64_t)COLS * (8 * grp + ((int)blockIdx.x & 7));
    if (n0 >= g.D) return;
    if (tid < 4) ((uint32_t *)(sx + MXD_WAVES * XROW))[tid] = 0;
    __syncthreads();
    const int slots = g.K + (g.sh_a.data ? 1 : 0);
    for (int k = wave; k < slots; k += MXD_WAVES) {
        const bool shared = k == g.K;
        const ExpertMat &m = shared ? g.sh_a : g.a;
        const MxRows &x = shared ? g.sh_x : g.x;
        const int p = t * g.K + k, e = shared ? 0 : g.sel[p];
        const int64_t r = shared ? t : p;
        const int nb = (int)(m.K / 32);
        if ((unsigned)e >= (unsigned)(shared ? 1 : g.E)) continue;   // (the router's ids: not expected)
        MxTile<MXD_U> w;
        w.row = m.data + (int64_t)e * m.mat_bytes + (n0 + (lane & (COLS - 1))) * m.row_bytes;
        double acc[4] = {0.0, 0.0, 0.0, 0.0};
        for (int k0 = 0; k0 < nb; k0 += 4 * MXD_U) {
            const int kn = imin(nb - k0, 4 * MXD_U), sn = (kn + 3) / 4;
            // (the operands in front of the weights: they are stored to LDS while those are on their way)
            const u32x4 *src = (const u32x4 *)(x.d + r * (int64_t)(nb * MX_FB) + (int64_t)MX_FB * k0);
            constexpr int NX = (4 * MXD_U * MX_FB + 1023) / 1024;
            u32x4 xv[NX];
            uint32_t xs1 = MX_ONE;
#pragma unroll
            for (int i = 0; i < NX; ++i) xv[i] = 64 * i + lane < kn * (MX_FB / 16) ? src[64 * i + lane] : u32x4{0, 0, 0, 0};
            if (lane < kn) xs1 = x.s[r * nb + k0 + lane];
            asm volatile("" ::: "memory");
            w.load(k0 / 4, sn, nb, lane);
            wave_lds_sync();   // (the activations before are read)
#pragma unroll
            for (int i = 0; i < NX; ++i)
                if (64 * i + lane < 4 * MXD_U * MX_FB / 16) *(u32x4 *)(sx + XROW * wave + 16 * (64 * i + lane)) = xv[i];
            if (lane < 4 * MXD_U) ss[wave][lane] = xs1;
            wave_lds_sync();
            const int xo[2] = {XROW * wave, XROW * wave};
            const uint32_t *const xs[2] = {ss[wave], ss[wave]};
            w.products(k0 / 4, sn, nb, lane, sx, xo, MXD_WAVES * XROW, xs, k0 / 4, 1, acc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double a = mx_columns(acc[i]);
            if ((lane & 15) == 0) s_z[k][4 * (lane >> 4) + i] = (float)a;
        }
    }
    __syncthreads();
    const int64_t n = n0 + tid;
    if (tid < COLS && n < g.D) {
        double s = 0.0;
        for (int k = 0; k < g.K; ++k) s = s + (double)(s_z[k][tid] * g.w[t * g.K + k]);
        float moe = (float)s;
        if (g.sh_a.data) moe = moe + (g.sh_w ? s_z[g.K][tid] * g.sh_w[t] : s_z[g.K][tid]);
        const int64_t o = (int64_t)t * g.D + n;
        g.out[o] = g.res ? g.res[o] + moe : moe;
    }
}

int launch_mxd(const MxDownArgs &g, hipStream_t st) {
    if (g.T < 1 || g.K < 1 || g.K > MXD_KMAX || g.D % 16 || g.a.type != 39 || g.a.K % 32 || (g.sh_a.data && (g.sh_a.type != 39 || g.sh_a.K % 32))) return -6;
    // eight columns a work-group where sixteen would leave half of the CUs idle
    // (layers of one token, D 2048: 26.7 us, in sixteen 27.9; with 168 of 256
    // CUs, D 2688, sixteen take 35.0 and eight 36.8)
    const bool narrow = 2 * (int64_t)g.T * (g.D / 16) <= g.n_cu;
    const int64_t groups = (g.D / (narrow ? 8 : 16) + 7) / 8;
    const dim3 grid((unsigned)(8 * groups * g.T)), block(64 * MXD_WAVES);
    if (narrow) hipLaunchKernelGGL(k_mxd<8>, grid, block, 0, st, g);
    else hipLaunchKernelGGL(k_mxd<16>, grid, block, 0, st, g);
    return hip_check_launch();
}

}  // namespace mimoe
