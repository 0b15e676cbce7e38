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
// the 17-byte blocks leave through LDS in 16-byte stores.
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
__global__ void __launch_bounds__(256) k_prep_mx(const float *__restrict__ src, int64_t ld, int64_t nrows, int nb,
                                                 uint8_t *__restrict__ rows) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, blk = i >> 2;
    const bool live = blk < nrows * nb;
    const int64_t r = live ? blk / nb : 0, b = live ? blk - r * nb : 0;
    float v[8];
    mx_load8<VEC>(src + r * ld + 32 * b, (int)(i & 3), v);
    uint8_t *row = rows + r * mx_row(nb);
    mx_store_block(v, row, b, (int)(i & 3), live);
    if (live && b == nb - 1) mx_store_pad(row, nb, (int)(i & 3));
}

int launch_prep_mx(const float *src, int64_t ld, int64_t nrows, int64_t K, uint8_t *rows, hipStream_t st) {
    if (nrows <= 0) return 0;
    if (K % 32 || K > 0x7fffffff) return -6;
    const int64_t wgs = (nrows * (K / 8) + 255) / 256;
    if (wgs > 0x7fffffff) return -6;
    if (ld % 4 == 0 && (uintptr_t)src % 16 == 0)
        hipLaunchKernelGGL(k_prep_mx<true>, dim3((unsigned)wgs), dim3(256), 0, st, src, ld, nrows, (int)(K / 32), rows);
    else hipLaunchKernelGGL(k_prep_mx<false>, dim3((unsigned)wgs), dim3(256), 0, st, src, ld, nrows, (int)(K / 32), rows);
    return hip_check_launch();
}

// ------------------------------------------------------------------ few rows
// act_pair (act.hpp) in fp64, rounded once: a value that differs in its last
// bits would move an 8-bit code of the operand that it becomes
__device__ inline float mx_act(int act, double a, double b) {
    const double SQRT_2_INV = 0.70710678118654752440, SQRT_2_OVER_PI = 0.79788456080286535588;
    switch (act) {
    case 0: return (float)(a / (1.0 + exp(-a)) * b);
    case 1: return (float)(0.5 * a * (1.0 + erf(a * SQRT_2_INV)) * (b + 1.0));
    case 2: return (float)(0.5 * a * (1.0 + tanh(SQRT_2_OVER_PI * a * (1.0 + 0.044715 * a * a))) * b);
    case 3: return (float)(0.5 * a * (1.0 + erf(a * SQRT_2_INV)) * b);
    default: {
        const double r = a > 0.0 ? a : a != a ? a : 0.0;
        return (float)(r * r);
    }
    }
}

// Grouped product of few rows per expert.  A work-group (8 waves) owns 64
// weight rows of one active expert (GLU: 32 gate rows and the matching up
// rows) as four 16-row tiles, two waves to a tile, each half of the blocks.
//
// A wave's step is v_mfma_scale_f32_16x16x128_f8f6f4 on four blocks of its 16
// rows (lane l: row l % 16, block l / 16 of the step, the 16 bytes of codes as
// they are) against one row of activations: column c = 4 b + i holds digit i
// of the step's block b and zeros in the other three, so each of the 16 x 16
// results is one digit's sum over one block, an integer of at most 13 bits
// times a power of two: exact in fp32 whatever the scales.  They are added in
// fp64, so the result is the exact sum rounded at 2^-53, and the GLU's values
// (in fp64, rounded once) and their codes do not depend on an order of sums.
//
// The expert's rows run MXV_NT at a time through LDS, the lanes' weight blocks
// staying in registers for them.
constexpr int MXV_NT = 4, MXV_WAVES = 8, MXV_U = 8;   // U: steps of a wave in registers at a time
constexpr int MXV_KB = 4 * 2 * MXV_U;                 // blocks of a pass over K (both wave halves)

template <int EPI, bool SH>
__global__ void __launch_bounds__(64 * MXV_WAVES) k_mxv(MxArgs g) {
    __shared__ __attribute__((aligned(16))) uint8_t sx[MXV_NT][MXV_KB / 4 * MX_XG];
    __shared__ double s_sum[MXV_NT][128];
    __shared__ float s_v[MXV_NT][64];
    __shared__ int s_p[MXV_IDS];
    __shared__ int s_cnt[MXV_WAVES];
    constexpr bool GLU = EPI == MX_GLU;
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
        if (g.ids) {
            // work-group row j belongs to slot j, and leaves unless the slot is its expert's first
            const int id = tid < g.rows ? g.ids[tid] : -1;
            e = g.ids[j];
            if ((unsigned)e >= (unsigned)g.n_expert) {
                if (g.bad_total && cb == 0 && tid == 0) atomicAdd(g.bad_total, 1);
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
    const int tile = wave >> 1, half = wave & 1, r16 = lane & 15, grp = lane >> 4;
    // the lane's weight row (past the matrix: row 0, not stored)
    const int64_t col = (int64_t)cb * COLS + 16 * (GLU ? tile & 1 : tile) + r16;
    const bool col_ok = col < s.ncols;
    int64_t wrow = col_ok ? col : 0;
    const uint8_t *rowp = s.a.data + (int64_t)e * s.a.mat_bytes;
    int64_t rb = s.a.row_bytes;
    if (GLU && tile >= 2) {
        if (s.fused) {
            wrow += s.I;
        } else {
            rowp = s.b.data + (int64_t)e * s.b.mat_bytes;
            rb = s.b.row_bytes;
        }
    }
    rowp += wrow * rb;
    const int nb = (int)(s.a.K / 32);
    const int kdiv = g.ne11 == 1 && !shared ? g.K : 1;
    const bool on = (r16 >> 2) == grp;   // the lane's column holds a digit of the lane's block
    const int dig = r16 & 3;
    for (int q0 = 0; q0 < cnt; q0 += MXV_IDS) {   // (rows that fit s_p)
        const int qn = cnt - q0 < MXV_IDS ? cnt - q0 : MXV_IDS;
        if (shared || perm) {
            if (q0) __syncthreads();
            for (int i = tid; i < qn; i += 64 * MXV_WAVES) s_p[i] = shared ? q0 + i : perm[q0 + i];
            __syncthreads();
        }
        for (int n0 = 0; n0 < qn; n0 += MXV_NT) {
            const int nt = qn - n0 < MXV_NT ? qn - n0 : MXV_NT;
            double acc[MXV_NT][4];
#pragma unroll
            for (int n = 0; n < MXV_NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][i] = 0.0;
            for (int k0 = 0; k0 < nb; k0 += MXV_KB) {
                const int kn = nb - k0 < MXV_KB ? nb - k0 : MXV_KB, nst = (kn + 3) / 4, h0 = (nst + 1) / 2;
                const int s0 = half ? h0 : 0, sn = half ? nst - h0 : h0;   // the wave's steps
                MxRaw w[MXV_U];
#pragma unroll
                for (int u = 0; u < MXV_U; ++u) {
                    const int b = 4 * (s0 + u) + grp;
                    if (u < sn) mx_load(rowp + MX_BYTES * (int64_t)(k0 + (b < kn ? b : 0)), w[u]);   // (past the row: block 0, not used)
                }
                if (k0 || n0 || q0) __syncthreads();   // (the activations before are read)
                for (int n = 0; n < nt; ++n) {
                    const int p = s_p[n0 + n];
                    const uint4 *src = (const uint4 *)(s.x + (int64_t)(kdiv > 1 ? p / kdiv : p) * mx_row(nb) + mx_row(k0));
                    for (int i = tid; i < nst * (MX_XG / 16); i += 64 * MXV_WAVES) *(uint4 *)(sx[n] + 16 * i) = src[i];
                }
                __syncthreads();
#pragma unroll
                for (int u = 0; u < MXV_U; ++u) {
                    if (u >= sn) break;
                    const int b = 4 * (s0 + u) + grp;
                    const bool in = b < kn;
                    const uint32_t mis = (uint32_t)(uintptr_t)(rowp + MX_BYTES * (int64_t)(k0 + (in ? b : 0))) & 3u;
                    uint32_t c[4];
                    mx_codes(w[u], mis, c);
                    const int sa = in ? (int)mx_scale(w[u], mis) : (int)MX_ONE;
                    i32x8 A = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < 4; ++i) A[i] = in ? (int)c[i] : 0;
#pragma unroll
                    for (int n = 0; n < MXV_NT; ++n) {
                        if (n >= nt) break;
                        i32x8 B = {0, 0, 0, 0, 0, 0, 0, 0};
                        int sb = (int)MX_ONE;
                        if (on && in) {
                            const uint8_t *x = sx[n] + MX_XG * (s0 + u) + MX_XB * grp + 8 * (grp & 2);   // (b = 4 (s0 + u) + grp)
                            const uint4 lo = *(const uint4 *)(x + 16 * dig);
                            const uint2 hi = *(const uint2 *)(x + 64 + 8 * dig);
                            B[0] = (int)lo.x; B[1] = (int)lo.y; B[2] = (int)lo.z; B[3] = (int)lo.w;
                            B[4] = (int)hi.x; B[5] = (int)hi.y;
                            sb = sx[n][MX_XG * (s0 + u) + 2 * MX_XB + 4 * grp + dig];
                        }
                        float4_t z = {0.f, 0.f, 0.f, 0.f};
                        z = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, z, 4, 2, 0, sa, 0, sb);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][i] += (double)z[i];
                    }
                }
            }
            // rows 4 (lane / 16) + i, a partial per column: the 16 columns, then the other half's
#pragma unroll
            for (int n = 0; n < MXV_NT; ++n) {
                if (n >= nt) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    double a = acc[n][i];
                    a = dpp_add<0xB1>(a);
                    a = dpp_add<0x4E>(a);
                    a = dpp_add<0x141>(a);
                    a = dpp_add<0x140>(a);
                    if (r16 == 0) s_sum[n][64 * half + 16 * tile + 4 * grp + i] = a;
                }
            }
            __syncthreads();
            if (EPI == MX_STORE) {
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
                    s_v[n][c] = mx_act(GLU ? g.act : ACT_RELU_SQR, a, b);
                }
                __syncthreads();
                if (tid < MXV_NT * COLS / 8) {
                    const int m = tid / (COLS / 8), blk = (tid >> 2) % (COLS / 32);
                    float v[8];
                    mx_load8<false>(s_v[m] + 32 * blk, tid & 3, v);
                    mx_store_block(v, s.o + (int64_t)(m < nt ? s_p[n0 + m] : 0) * mx_row(s.ncols / 32), (int64_t)cb * (COLS / 32) + blk, tid & 3,
                                   m < nt && (int64_t)cb * COLS + 32 * blk < s.ncols);
                }
            }
            // (s_sum and s_v are written again after the barriers in front of the next rows' products)
        }
    }
}

template <int EPI>
static int mxv_launch(const MxArgs &a, hipStream_t st) {
    MxArgs g = a;
    constexpr int COLS = EPI == MX_GLU ? 32 : 64;
    g.ncb = (int)((g.ncols + COLS - 1) / COLS);
    g.sh_wgs = g.sh_rows > 0 ? (int)((g.sh.ncols + COLS - 1) / COLS) : 0;
    const int64_t wgs = g.sh_wgs + (int64_t)g.ncb * (g.ids ? g.rows : g.max_active);
    if (wgs > 0x7fffffff) return -6;
    const dim3 grid((unsigned)wgs), block(64 * MXV_WAVES);
    if (g.sh_wgs) hipLaunchKernelGGL((k_mxv<EPI, true>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((k_mxv<EPI, false>), grid, block, 0, st, g);
    return hip_check_launch();
}

static bool mx_side_ok(const MxArgs &g, const MxSide &s) {
    return s.a.type == 39 && s.a.K % 32 == 0 && s.a.K <= 0x7fffffff && !(g.epi != MX_STORE && s.ncols % 32);
}

int launch_mxv(const MxArgs &g, hipStream_t st) {
    if (g.max_active <= 0) return 0;
    if (!mx_side_ok(g, g) || (g.sh_rows > 0 && !mx_side_ok(g, g.sh))) return -6;
    if (g.ids && (g.rows > MXV_IDS || g.n_expert <= 0)) return -6;
    switch (g.epi) {
    case MX_STORE: return mxv_launch<MX_STORE>(g, st);
    case MX_GLU: return mxv_launch<MX_GLU>(g, st);
    case MX_RELU_SQR: return mxv_launch<MX_RELU_SQR>(g, st);
    default: return -6;
    }
}

}  // namespace mimoe
