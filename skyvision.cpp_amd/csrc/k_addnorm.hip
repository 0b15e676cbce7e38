// k_addnorm.hip - the residual's addition, the row norm and its rows in 8 bits
// (mi_add_norm): h = x + add, y = norm(h) (norm.hpp: sums in fp64, every other
// step rounded to fp32), q = y in Q8_0 or Q8_K, ggml's quantize_row of y.
//
// One pass: a row's values stay in registers between the sums and the stores.
#include "common.hpp"
#include "lanes.hpp"
#include "launch.hpp"
#include "wave_ops.hpp"

namespace mimoe {

// codes of 4 values at 4 i of a row (8 lanes hold a 32-value block) to the
// row's Q8_0 blocks; live: the values are in the row
__device__ __forceinline__ void an_store_q8_0(const float (&v)[4], uint8_t *row, int i, bool live, bool words) {
    // the largest |v| as bits: a NaN or an infinity shows as 0x7f800000 or more
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
        m = u > m ? u : m;
    }
    uint32_t o = (uint32_t)dpp_i<0xB1>((int)m);
    m = o > m ? o : m;
    o = (uint32_t)dpp_i<0x4E>((int)m);
    m = o > m ? o : m;
    o = (uint32_t)dpp_i<0x141>((int)m);
    m = o > m ? o : m;
    const bool bad = m >= 0x7f800000u;
    const float d = __builtin_bit_cast(float, m) / 127.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    const uint32_t dh = bad ? 0x7e00u : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)d);
    // roundf(t): t + the number before 1/2 with t's sign, cut (|t| <= 127.5: the
    // sum of a fraction of 1/2 or more rounds to the next integer, of less stays below)
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float t = v[j] * id;
        q[j] = (uint32_t)(int)(t + __builtin_copysignf(0.49999997f, t));
    }
    uint32_t c = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[3], q[2], 0x0C0C0400u), __builtin_amdgcn_perm(q[1], q[0], 0x0C0C0400u), 0x05040100u);
    if (bad) c = 0u;
    // words (D % 64 == 0): a pair of blocks is 17 aligned words; words 0 .. 8 hold the even block's scale
    // and codes and the odd one's scale (the codes half a word off), the rest the
    // odd block's codes.  Lanes 0 .. 7 of 16 hold the even block.
    const uint32_t before = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0x111, 0xF, 0xF, false);   // the lane before (row_shr 1)
    const int k = i & 15;
    if (!live) return;
    uint8_t *blk = row + (i >> 3) * 34;
    if (words) {
        uint8_t *pair = row + (i >> 4) * 68;
        if (k < 8) {
            *(uint32_t *)(pair + 4 * k) = (k == 0 ? dh : before >> 16) | c << 16;
        } else {
            *(uint32_t *)(pair + 36 + 4 * (k - 8)) = c;
            if (k == 8) *(uint32_t *)(pair + 32) = before >> 16 | dh << 16;
        }
    } else {
        *(uint16_t *)(blk + 2 + 4 * (i & 7)) = (uint16_t)c;
        *(uint16_t *)(blk + 4 + 4 * (i & 7)) = (uint16_t)(c >> 16);
        if ((i & 7) == 0) *(uint16_t *)blk = (uint16_t)dh;
    }
}

// N blocks of 256 values held by a wave, lane l the values 4 l of each, to the
// row's Q8_K blocks ib0, ib0 + step, ..: d = 1 / iscale, iscale = -127 / the first
// value of the largest |.|, codes rint(iscale v) (|127 v / m| < 127.5: none leaves
// 8 bits) by the sum with 1.5 * 2^23, whose low bits hold the integer
template <int N>
__device__ __forceinline__ void an_store_q8_K(const float (&v)[N][4], uint8_t *row, int ib0, int step, int nblk, int lane) {
    uint32_t u[N][4], m[N];   // |v| and the largest as bits: a NaN or an infinity shows as 0x7f800000 or more
#pragma unroll
    for (int n = 0; n < N; ++n) {
        m[n] = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u[n][j] = __builtin_bit_cast(uint32_t, v[n][j]) & 0x7fffffffu;
            m[n] = u[n][j] > m[n] ? u[n][j] : m[n];
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) m[n] = wave_max_u(m[n]);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (ib0 + n * step >= nblk) continue;   // (uniform)
        // the first holder's sign, on the lanes' masks (a select among v's elements would
        // put v into memory): element 0's where it holds the largest, else element 1's, ..
        const uint32_t mu = (uint32_t)__builtin_amdgcn_readfirstlane((int)m[n]);
        const uint64_t h0 = __ballot(u[n][0] == mu), h1 = __ballot(u[n][1] == mu), h2 = __ballot(u[n][2] == mu),
                       h3 = __ballot(u[n][3] == mu);
        const uint64_t n0 = __ballot(v[n][0] < 0.f), n1 = __ballot(v[n][1] < 0.f), n2 = __ballot(v[n][2] < 0.f),
                       n3 = __ballot(v[n][3] < 0.f);
        const uint64_t neg = (h0 & n0) | (~h0 & ((h1 & n1) | (~h1 & ((h2 & n2) | (~h2 & n3)))));
        const int first = (int)__builtin_ctzll(h0 | h1 | h2 | h3);   // (some lane holds it)
        const float val = __builtin_bit_cast(float, mu | (uint32_t)((neg >> first) & 1) << 31);
        const bool bad = mu >= 0x7f800000u, zero = mu == 0u;
        const float iscale = bad || zero ? 0.f : -127.f / val;
        const float d = bad ? __builtin_nanf("") : zero ? 0.f : 1 / iscale;
        uint32_t q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = __builtin_bit_cast(uint32_t, (bad ? 0.f : iscale * v[n][j]) + 12582912.f);
        const uint32_t c = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[3], q[2], 0x0C0C0400u),
                                                 __builtin_amdgcn_perm(q[1], q[0], 0x0C0C0400u), 0x05040100u);
        int s = __builtin_amdgcn_sdot4(0x01010101, (int)c, 0, false);   // ggml's sums of 16 codes, over 4 lanes
        s += dpp_i<0xB1>(s);
        s += dpp_i<0x4E>(s);
        uint8_t *blk = row + (int64_t)(ib0 + n * step) * Q8K_BYTES;
        *(uint32_t *)(blk + 4 + 4 * lane) = c;
        if (lane == 0) *(float *)blk = d;
        if ((lane & 3) == 0) *(int16_t *)(blk + 260 + 2 * (lane >> 2)) = (int16_t)s;
    }
}

// 4 values at i of a row of D (zeros past it), at any float's address.  TAIL: D is
// no multiple of 4, the last piece goes value by value (without it a kernel has
// no such code: 4096 rows of 2048 to Q8_K 30.3 -> 28.7 us)
template <bool TAIL>
__device__ __forceinline__ void an_load4(const float *x, int i, int D, float (&v)[4]) {
    if constexpr (!TAIL) {
        float4_t a = {0.f, 0.f, 0.f, 0.f};
        if (i < D) a = *(const float4_a4 *)(x + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = a[j];
    } else if (i + 4 <= D) {
        const float4_t a = *(const float4_a4 *)(x + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = a[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i + j < D ? x[i + j] : 0.f;
    }
}
template <bool TAIL>
__device__ __forceinline__ void an_store4(float *x, int i, int D, const float (&v)[4]) {
    if (TAIL ? i + 4 <= D : i < D) {
        const float4_t a = {v[0], v[1], v[2], v[3]};
        *(float4_a4 *)(x + i) = a;
    } else if constexpr (TAIL) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < D) x[i + j] = v[j];
    }
}

// A work-group of W waves per row, thread i holding the values at 256 W k + 4 i,
// k < P.
// Bound by the memory: 4096 rows of 2048 with the sum and Q8_K codes, 110 MB in
// 21 us, the inputs in the last-level cache; 4096 rows of 8192 in fp32, 537 MB in
// 100 us (5.4 TB/s, a large copy 5.1).
template <int W, int P, bool TAIL>
__global__ void __launch_bounds__(64 * W) k_add_norm(AddNormArgs a, int D, double rD) {
    __shared__ double red[2][W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t t = blockIdx.x;
    const int id = (int)threadIdx.x;
    constexpr int ROUND = 256 * W;
    // the sum over the row, the same bits in every thread
    auto row_sum = [&](double v, double *r) __attribute__((always_inline)) {
        v = wave_sum_d(v);
        if (lane == 0) r[wave] = v;
        __syncthreads();
        double s = r[0];
#pragma unroll
        for (int i = 1; i < W; ++i) s += r[i];
        return s;
    };
    // sum / D, rounded to fp32: the quotient by the reciprocal and one correction (an
    // infinite sum stays one)
    auto mean = [&](double v) __attribute__((always_inline)) {
        const double e = v * rD, r = fma(fma(-e, (double)D, v), rD, e);
        return (float)(r == r ? r : e);
    };
    float v[P][4], ad[P][4];
    const float *x = a.x + t * a.ldx, *add = a.add + t * a.lda;
#pragma unroll
    for (int k = 0; k < P; ++k) an_load4<TAIL>(x, ROUND * k + 4 * id, D, v[k]);
    if (a.add) {
#pragma unroll
        for (int k = 0; k < P; ++k) an_load4<TAIL>(add, ROUND * k + 4 * id, D, ad[k]);
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k][j] = v[k][j] + ad[k][j];
    }
    float w[P][4], b[P][4];   // (on their way while the sums are formed)
#pragma unroll
    for (int k = 0; k < P; ++k) {
        if (a.norm.w) an_load4<TAIL>(a.norm.w, ROUND * k + 4 * id, D, w[k]);
        if (a.norm.b) an_load4<TAIL>(a.norm.b, ROUND * k + 4 * id, D, b[k]);
    }
    if (a.sum) {
#pragma unroll
        for (int k = 0; k < P; ++k) an_store4<TAIL>(a.sum + t * a.lds, ROUND * k + 4 * id, D, v[k]);
    }
    float m = 0.f;
    if (a.norm.kind == NORM_LAYER) {
        double s0 = 0.0, s1 = 0.0;   // (two chains)
#pragma unroll
        for (int k = 0; k < P; ++k) {
            s0 = s0 + (double)v[k][0];
            s1 = s1 + (double)v[k][1];
            s0 = s0 + (double)v[k][2];
            s1 = s1 + (double)v[k][3];
        }
        m = mean(row_sum(s0 + s1, red[0]));
    }
    double s0 = 0.0, s1 = 0.0;
#pragma unroll
    for (int k = 0; k < P; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float d = v[k][j] - m;   // (RMS: m = 0, exact)
            const float dd = ROUND * k + 4 * id + (TAIL ? j : 0) < D ? d * d : 0.f;
            if (j & 1) s1 = s1 + (double)dd;
            else s0 = s0 + (double)dd;
        }
    const float var = mean(row_sum(s0 + s1, red[1]));
    const float sc = 1.0f / sqrtf(var + a.norm.eps);
    const bool words = a.ldq % 4 == 0 && ((uintptr_t)a.q & 3) == 0 && D % 64 == 0;   // Q8_0 in whole words
#pragma unroll
    for (int k = 0; k < P; ++k) {
        const int i = ROUND * k + 4 * id;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float y = (v[k][j] - m) * sc;   // norm_apply, step for step
            if (a.norm.w) y = y * w[k][j];
            if (a.norm.b) y = y + b[k][j];
            v[k][j] = i + (TAIL ? j : 0) < D ? y : 0.f;
        }
        if (a.y) an_store4<TAIL>(a.y + t * a.ldy, i, D, v[k]);
        if (a.q && a.qtype == 8) an_store_q8_0(v[k], a.q + t * a.ldq, i >> 2, i < D, words);
    }
    if (a.q && a.qtype == 15) an_store_q8_K<P>(v, a.q + t * a.ldq, wave, W, D / QK, lane);
}

template <bool TAIL>
static int an_launch(const AddNormArgs &a, int64_t T, int D, hipStream_t st) {
#define AN(W, P) hipLaunchKernelGGL((k_add_norm<W, P, TAIL>), dim3((unsigned)T), dim3(64 * W), 0, st, a, D, 1.0 / (double)D)
    // few rows: more waves than hold the row (one row of 2048: 8 waves 2.65 us, 4
    // 2.9); many: fewer, whose sums and scalars cost less (2000 rows of 2048: 8 waves
    // 12.8 us, 2 11.3; 1024 rows of 4096 to Q8_K 18.9 and with 4 17.7)
    if (T >= 512 && D <= 1024) AN(2, 2);
    else if (T >= 512 && D <= 2048) AN(2, 4);
    else if (T >= 512 && D <= 4096) AN(4, 4);
    else if (D <= 2048) AN(8, 1);
    else if (D <= 4096) AN(16, 1);
    else if (D <= 8192) AN(16, 2);
    else AN(16, 4);
#undef AN
    return hip_check_launch();
}

int launch_add_norm(const AddNormArgs &a, int64_t T, int D, hipStream_t st) {
    if (T <= 0) return 0;
    if (D <= 0 || D > ADD_NORM_MAX_D || (a.norm.kind != NORM_RMS && a.norm.kind != NORM_LAYER)) return -6;
    if (a.q && a.qtype != 8 && a.qtype != 15) return -3;
    if (a.q && D % (a.qtype == 8 ? 32 : QK)) return -2;
    constexpr int64_t PASS = 1 << 21;   // rows of a launch (it covers fewer than 2^32 threads)
    for (int64_t t = 0; t < T; t += PASS) {
        AddNormArgs g = a;
        g.x += t * a.ldx;
        if (a.add) g.add += t * a.lda;
        if (a.sum) g.sum += t * a.lds;
        if (a.y) g.y += t * a.ldy;
        if (a.q) g.q += t * a.ldq;
        const int64_t n = T - t < PASS ? T - t : PASS;
        const int rc = D % 4 ? an_launch<true>(g, n, D, st) : an_launch<false>(g, n, D, st);
        if (rc) return rc;
    }
    return 0;
}

// values of Q8_K blocks, one wave per block
__global__ void __launch_bounds__(256) k_dequantize_q8k(const uint8_t *__restrict__ src, float *__restrict__ dst, int64_t nblocks) {
    const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= nblocks) return;
    const int lane = threadIdx.x & 63;
    const uint8_t *p = src + Q8K_BYTES * b;
    const float d = *(const float *)p;
    const uint32_t c = *(const uint32_t *)(p + 4 + 4 * lane);
    float *o = dst + 256 * b + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = d * (float)(int8_t)(c >> (8 * j));
}

int launch_dequantize_q8k(const void *src, float *dst, int64_t nblocks, hipStream_t st) {
    if (nblocks <= 0) return 0;
    constexpr int64_t PASS = 1 << 24;   // blocks of a launch (it covers fewer than 2^32 threads)
    for (int64_t b = 0; b < nblocks; b += PASS) {
        const int64_t n = nblocks - b < PASS ? nblocks - b : PASS;
        hipLaunchKernelGGL(k_dequantize_q8k, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, (const uint8_t *)src + Q8K_BYTES * b,
                           dst + QK * b, n);
        const int rc = hip_check_launch();
        if (rc) return rc;
    }
    return 0;
}

}  // namespace mimoe
