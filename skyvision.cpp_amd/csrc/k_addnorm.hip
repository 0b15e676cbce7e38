// k_addnorm.hip - the residual's addition, the row norm and its rows in 8 bits
// (mi_add_norm): h = x + add, y = norm(h) (norm.hpp: sums in fp64, every other
// step rounded to fp32), q = y in Q8_0 or Q8_K, ggml's quantize_row of y.
//
// One pass: a row's values stay in registers between the sums and the stores.
#include "common.hpp"
#include "launch.hpp"
#include "wave_ops.hpp"

namespace mimoe {

constexpr int AN_THREADS = 256;

__device__ __forceinline__ double wave_sum_d(double v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// sum over the work-group, in every thread
__device__ __forceinline__ double an_block_sum(double v, double *red) {
    v = wave_sum_d(v);
    __syncthreads();   // red may still be read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = red[0];
    for (int i = 1; i < AN_THREADS / 64; ++i) s += red[i];
    return s;
}

// codes of 4 values at 4 i (8 lanes hold a 32-value block): Q8_0 block at dst
__device__ __forceinline__ void an_store_q8_0(const float (&v)[4], uint8_t *row, int i, bool live) {
    float m = absmax4(v);
    // a NaN or an infinity anywhere in the block (amax alone misses NaN)
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) bad |= !(fabsf(v[j]) <= 3.402823466e38f);
    int b = bad;
    b |= dpp_i<0xB1>(b); b |= dpp_i<0x4E>(b); b |= dpp_i<0x141>(b);
    m = fmaxf(m, dpp_f<0xB1>(m));
    m = fmaxf(m, dpp_f<0x4E>(m));
    m = fmaxf(m, dpp_f<0x141>(m));
    const float d = m / 127.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    if (!live) return;
    uint8_t *blk = row + (i >> 3) * 34;
    uint16_t c[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int q0 = b ? 0 : (int)roundf(v[2 * j] * id), q1 = b ? 0 : (int)roundf(v[2 * j + 1] * id);
        c[j] = (uint16_t)((q0 & 0xff) | (q1 & 0xff) << 8);
    }
    *(uint16_t *)(blk + 2 + 4 * (i & 7)) = c[0];
    *(uint16_t *)(blk + 4 + 4 * (i & 7)) = c[1];
    if ((i & 7) == 0) *(uint16_t *)blk = b ? 0x7e00 : (uint16_t)f32_to_fp16_bits(d);
}

// codes of 4 values at 4 lane of block ib (one wave holds the block)
__device__ __forceinline__ void an_store_q8_K(const float (&v)[4], uint8_t *row, int ib, int lane) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) bad |= !(fabsf(v[j]) <= 3.402823466e38f);
    const bool b = __ballot(bad) != 0ull;
    int q[4];
    float d = q8k_wave(v, lane, q);
    if (b) {
        d = __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = 0;
    }
    const int s = q8k_bsum16(q);
    uint8_t *blk = row + (int64_t)ib * 292;
    *(uint32_t *)(blk + 4 + 4 * lane) = pack_i8x4(q);
    if (lane == 0) *(float *)blk = d;
    if ((lane & 3) == 0) *(int16_t *)(blk + 260 + 2 * (lane >> 2)) = (int16_t)s;
}

// One work-group per row, thread i holding the values at 1024 k + 4 i.
template <int P>
__global__ void __launch_bounds__(AN_THREADS) k_add_norm(AddNormArgs a, int D) {
    __shared__ double red[AN_THREADS / 64];
    const int64_t t = blockIdx.x;
    const int i4 = 4 * (int)threadIdx.x, lane = threadIdx.x & 63;
    float v[P][4];
#pragma unroll
    for (int k = 0; k < P; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = 1024 * k + i4 + j;
            float h = 0.f;
            if (i < D) {
                h = a.x[t * a.ldx + i];
                if (a.add) h = h + a.add[t * a.lda + i];
            }
            v[k][j] = h;
        }
    float m = 0.f;
    double acc = 0.0;
    if (a.norm.kind == NORM_LAYER) {
#pragma unroll
        for (int k = 0; k < P; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = acc + (double)v[k][j];
        m = (float)(an_block_sum(acc, red) / (double)D);
        acc = 0.0;
    }
#pragma unroll
    for (int k = 0; k < P; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (1024 * k + i4 + j < D) {
                const float d = v[k][j] - m;   // (RMS: m = 0, exact)
                acc = acc + (double)(d * d);
            }
    const float var = (float)(an_block_sum(acc, red) / (double)D);
    const float sc = 1.0f / sqrtf(var + a.norm.eps);
#pragma unroll
    for (int k = 0; k < P; ++k) {
        float o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = 1024 * k + i4 + j;
            o[j] = 0.f;
            if (i < D) {
                if (a.sum) a.sum[t * a.lds + i] = v[k][j];
                o[j] = norm_apply(a.norm, v[k][j], i, m, sc);
                if (a.y) a.y[t * a.ldy + i] = o[j];
            }
        }
        if (a.q && a.qtype == 8) an_store_q8_0(o, a.q + t * a.ldq, 256 * k + (int)threadIdx.x, 1024 * k + i4 < D);
        if (a.q && a.qtype == 15 && 1024 * k + 256 * (int)(threadIdx.x >> 6) < D)   // whole waves
            an_store_q8_K(o, a.q + t * a.ldq, 4 * k + (int)(threadIdx.x >> 6), lane);
    }
}

int launch_add_norm(const AddNormArgs &a, int64_t T, int D, hipStream_t st) {
    if (T <= 0) return 0;
    if (D <= 0 || D > ADD_NORM_MAX_D || T > 0x7fffffff || (a.norm.kind != NORM_RMS && a.norm.kind != NORM_LAYER)) return -6;
    if (a.q && a.qtype != 8 && a.qtype != 15) return -3;
    if (a.q && D % (a.qtype == 8 ? 32 : QK)) return -2;
    const dim3 grid((unsigned)T), block(AN_THREADS);
    if (D <= 2048) hipLaunchKernelGGL(k_add_norm<2>, grid, block, 0, st, a, D);
    else if (D <= 4096) hipLaunchKernelGGL(k_add_norm<4>, grid, block, 0, st, a, D);
    else if (D <= 8192) hipLaunchKernelGGL(k_add_norm<8>, grid, block, 0, st, a, D);
    else hipLaunchKernelGGL(k_add_norm<16>, grid, block, 0, st, a, D);
    return hip_check_launch();
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
