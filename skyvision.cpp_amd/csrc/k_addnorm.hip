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

constexpr float AN_MAX = 3.402823466e38f;

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

// N blocks of 256 values held by a wave, lane l the values 4 l of each: to the
// row's Q8_K blocks ib0, ib0 + step, ..
template <int N>
__device__ __forceinline__ void an_store_q8_K(const float (&v)[N][4], uint8_t *row, int ib0, int step, int nblk, int lane) {
    int q[N][4];
    float d[N];
    q8k_wave_n<N>(v, lane, q, d);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) bad |= !(fabsf(v[n][j]) <= AN_MAX);
        if (__ballot(bad)) {
            d[n] = __builtin_nanf("");
#pragma unroll
            for (int j = 0; j < 4; ++j) q[n][j] = 0;
        }
        const int s = q8k_bsum16(q[n]);
        if (ib0 + n * step >= nblk) continue;   // (uniform)
        uint8_t *blk = row + (int64_t)(ib0 + n * step) * Q8K_BYTES;
        *(uint32_t *)(blk + 4 + 4 * lane) = pack_i8x4(q[n]);
        if (lane == 0) *(float *)blk = d[n];
        if ((lane & 3) == 0) *(int16_t *)(blk + 260 + 2 * (lane >> 2)) = (int16_t)s;
    }
}

// 4 values at i of a row of D (zeros past it)
template <bool VEC>
__device__ __forceinline__ void an_load4(const float *x, int i, int D, float (&v)[4]) {
    if constexpr (VEC) {
        const float4 a = i < D ? *(const float4 *)(x + i) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i + j < D ? x[i + j] : 0.f;
    }
}
template <bool VEC>
__device__ __forceinline__ void an_store4(float *x, int i, int D, const float (&v)[4]) {
    if constexpr (VEC) {
        if (i < D) *(float4 *)(x + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < D) x[i + j] = v[j];
    }
}

// W waves per row (W = 1: four rows a work-group of four waves), thread i of
// them holding the values at 256 W k + 4 i, k < P.  VEC: rows of whole float4,
// 16-byte aligned (D % 4 == 0 where not: the row's tail is read value by value).
template <int W, int P, bool VEC>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) k_add_norm(AddNormArgs a, int64_t T, int D) {
    __shared__ double red[2][W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t t = W == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (W == 1 && t >= T) return;   // whole waves
    const int id = W == 1 ? lane : (int)threadIdx.x;
    constexpr int ROUND = 256 * W;
    // the sum over the row, the same bits in every thread
    auto row_sum = [&](double v, double *r) __attribute__((always_inline)) {
        v = wave_sum_d(v);
        if constexpr (W == 1) return v;
        if (lane == 0) r[wave] = v;
        __syncthreads();
        double s = r[0];
#pragma unroll
        for (int i = 1; i < W; ++i) s += r[i];
        return s;
    };
    float v[P][4], ad[P][4];
    const float *x = a.x + t * a.ldx, *add = a.add + t * a.lda;
#pragma unroll
    for (int k = 0; k < P; ++k) an_load4<VEC>(x, ROUND * k + 4 * id, D, v[k]);
    if (a.add) {
#pragma unroll
        for (int k = 0; k < P; ++k) an_load4<VEC>(add, ROUND * k + 4 * id, D, ad[k]);
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k][j] = v[k][j] + ad[k][j];
    }
    // a row of several waves waits for its sums: the weights come meanwhile (a
    // wave of its own has others to run, and the registers are the row's)
    constexpr bool EARLY = W > 1;
    float w[EARLY ? P : 1][4], b[EARLY ? P : 1][4];
    if constexpr (EARLY) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
            if (a.norm.w) an_load4<VEC>(a.norm.w, ROUND * k + 4 * id, D, w[k]);
            if (a.norm.b) an_load4<VEC>(a.norm.b, ROUND * k + 4 * id, D, b[k]);
        }
    }
    if (a.sum) {
#pragma unroll
        for (int k = 0; k < P; ++k) an_store4<VEC>(a.sum + t * a.lds, ROUND * k + 4 * id, D, v[k]);
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
        m = (float)(row_sum(s0 + s1, red[0]) / (double)D);
    }
    double s0 = 0.0, s1 = 0.0;
#pragma unroll
    for (int k = 0; k < P; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float d = ROUND * k + 4 * id + j < D ? v[k][j] - m : 0.f;   // (RMS: m = 0, exact)
            if (j & 1) s1 = s1 + (double)(d * d);
            else s0 = s0 + (double)(d * d);
        }
    const float var = (float)(row_sum(s0 + s1, red[1]) / (double)D);
    const float sc = 1.0f / sqrtf(var + a.norm.eps);
    const bool words = a.ldq % 4 == 0 && ((uintptr_t)a.q & 3) == 0 && D % 64 == 0;   // Q8_0 in whole words
#pragma unroll
    for (int k = 0; k < P; ++k) {
        const int i = ROUND * k + 4 * id;
        const int kw = EARLY ? k : 0;
        if constexpr (!EARLY) {
            if (a.norm.w) an_load4<VEC>(a.norm.w, i, D, w[0]);
            if (a.norm.b) an_load4<VEC>(a.norm.b, i, D, b[0]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float y = (v[k][j] - m) * sc;   // norm_apply, step for step
            if (a.norm.w) y = y * w[kw][j];
            if (a.norm.b) y = y + b[kw][j];
            v[k][j] = i + j < D ? y : 0.f;
        }
        if (a.y) an_store4<VEC>(a.y + t * a.ldy, i, D, v[k]);
        if (a.q && a.qtype == 8) an_store_q8_0(v[k], a.q + t * a.ldq, i >> 2, i < D, words);
    }
    if (a.q && a.qtype == 15) an_store_q8_K<P>(v, a.q + t * a.ldq, W == 1 ? 0 : wave, W, D / QK, lane);
}

template <bool VEC>
static int an_launch(const AddNormArgs &a, int64_t T, int D, hipStream_t st) {
#define AN(W, P) hipLaunchKernelGGL((k_add_norm<W, P, VEC>), dim3((unsigned)(W == 1 ? (T + 3) / 4 : T)), dim3(W == 1 ? 256 : 64 * W), 0, st, a, T, D)
    // the row over the waves of a work-group (more waves than it needs to hold the
    // row: one row of 2048, 8 waves 2.65 us, 4 2.9); a wave per row, without barriers,
    // for thousands of rows that leave as fp32 (4096 rows of 2048: 20.0 us against
    // 23.0; with codes, whose arithmetic then sits in one wave, 33.3 against 32.0, and
    // 1024 rows 8.3 against 6.6)
    if (T >= 2048 && D <= 2048 && !a.q) {
        if (D <= 1024) AN(1, 4);
        else AN(1, 8);
    } else if (D <= 2048) AN(8, 1);
    else if (D <= 4096) AN(16, 1);
    else if (D <= 8192) AN(16, 2);
    else AN(16, 4);
#undef AN
    return hip_check_launch();
}

int launch_add_norm(const AddNormArgs &a, int64_t T, int D, hipStream_t st) {
    if (T <= 0) return 0;
    if (D <= 0 || D > ADD_NORM_MAX_D || T > 0x7fffffff || (a.norm.kind != NORM_RMS && a.norm.kind != NORM_LAYER)) return -6;
    if (a.q && a.qtype != 8 && a.qtype != 15) return -3;
    if (a.q && D % (a.qtype == 8 ? 32 : QK)) return -2;
    auto vec = [](const void *p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 4 == 0; };   // null: fine
    const bool v = D % 4 == 0 && vec(a.x, a.ldx) && vec(a.add, a.lda) && vec(a.sum, a.lds) && vec(a.y, a.ldy) &&
                   vec(a.norm.w, 0) && vec(a.norm.b, 0);
    return v ? an_launch<true>(a, T, D, st) : an_launch<false>(a, T, D, st);
}

// values of Q8_K blocks, one wave per block
__global__ void __launch_bounds__(256) k_dequantize_q8k(const uint8_t *__restrict__ src, float *__restrict__ dst, int64_t nblocks) {
    const int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= nblocks) return;
    const int lane = threadIdx.x & 63;
    const uint8_t *p = src + 292 * b;
    const float d = *(const float *)p;
    const uint32_t c = *(const uint32_t *)(p + 4 + 4 * lane);
    float *o = dst + 256 * b + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = d * (float)(int8_t)(c >> (8 * j));
}

int launch_dequantize_q8k(const void *src, float *dst, int64_t nblocks, hipStream_t st) {
    if (nblocks <= 0) return 0;
    if ((nblocks + 3) / 4 > 0x7fffffff) return -6;
    hipLaunchKernelGGL(k_dequantize_q8k, dim3((unsigned)((nblocks + 3) / 4)), dim3(256), 0, st, (const uint8_t *)src, dst, nblocks);
    return hip_check_launch();
}

}  // namespace mimoe
