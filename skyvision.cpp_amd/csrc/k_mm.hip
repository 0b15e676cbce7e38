// k_mm.hip - dense products of 4-bit matrices and a few rows (mi_mul_mat):
//   y[t][n] = sum over blocks of (a's block . b's block), b in a's 8-bit form.
//   Q4_0 . Q8_0: d_a d_b sum (q - 8) c                          (32 values)
//   Q4_K . Q8_K: d_b (d sum_j sc_j sum_j q c - dmin sum_j m_j sum_j c)   (256)
// The sums over codes are exact integers, the blocks are added in fp32.
#include "b32.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "wave_ops.hpp"

namespace mimoe {

// b rows as the 8-bit type's blocks, one after another (34 / 292 bytes)
__global__ void __launch_bounds__(256) k_mm_rows_q8_0(const float *__restrict__ b, int64_t ldb, int64_t nb, int64_t T, uint8_t *__restrict__ o) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= nb * T) return;
    const float *x = b + (i / nb) * ldb + 32 * (i % nb);
    float m = 0.f;
    bool bad = false;
    for (int j = 0; j < 32; ++j) {
        m = fmaxf(m, fabsf(x[j]));
        bad |= !(fabsf(x[j]) <= 3.402823466e38f);
    }
    const float d = m / 127.0f, id = d != 0.f ? 1.0f / d : 0.f;
    const uint32_t dh = bad ? 0x7e00u : f32_to_fp16_bits(d);
    uint8_t *p = o + 34 * i;
    p[0] = (uint8_t)dh;
    p[1] = (uint8_t)(dh >> 8);
    for (int j = 0; j < 32; ++j) p[2 + j] = bad ? 0 : (uint8_t)(int8_t)roundf(x[j] * id);
}
__global__ void __launch_bounds__(256) k_mm_rows_q8_K(const float *__restrict__ b, int64_t ldb, int64_t nb, int64_t T, uint8_t *__restrict__ o) {
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= nb * T) return;   // whole waves
    const int lane = threadIdx.x & 63;
    const float *x = b + (i / nb) * ldb + 256 * (i % nb) + 4 * lane;
    float v[4];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = x[j];
        bad |= !(fabsf(v[j]) <= 3.402823466e38f);
    }
    int q[4];
    float d = q8k_wave(v, lane, q);
    if (__ballot(bad)) {
        d = __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = 0;
    }
    uint8_t *p = o + 292 * i;
    const int s = q8k_bsum16(q);
    *(uint32_t *)(p + 4 + 4 * lane) = pack_i8x4(q);
    if (lane == 0) *(float *)p = d;
    if ((lane & 3) == 0) *(int16_t *)(p + 260 + 2 * (lane >> 2)) = (int16_t)s;
}

template <int TYPE>
__global__ void __launch_bounds__(256) k_mm_simple(MmArgs g, const uint8_t *b, int64_t ldb) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= g.N * g.T) return;
    const int64_t n = i % g.N, t = i / g.N;
    const uint8_t *ar = g.a + n * g.row_bytes, *br = b + t * ldb;
    float acc = 0.f;
    if constexpr (TYPE == 2) {
        for (int64_t k = 0; k < g.K / 32; ++k) {
            const uint8_t *p = ar + 18 * k, *q = br + 34 * k;
            int s = 0;
            for (int j = 0; j < 16; ++j)
                s += ((p[2 + j] & 15) - 8) * (int8_t)q[2 + j] + ((p[2 + j] >> 4) - 8) * (int8_t)q[18 + j];
            float d = fp16_bits_to_f32(*(const uint16_t *)q);
            if (!(d <= 65504.f)) d = __builtin_nanf("");
            acc = fmaf((float)s, fp16_bits_to_f32(*(const uint16_t *)p) * d, acc);
        }
    } else {
        for (int64_t k = 0; k < g.K / 256; ++k) {
            const uint8_t *p = ar + 144 * k, *q = br + 292 * k;
            int s = 0, sm = 0;
            for (int j = 0; j < 8; ++j) {
                int sc, m, u = 0, v = 0;
                scale_min_k4(j, p + 4, sc, m);
                for (int l = 0; l < 32; ++l) {
                    const int c = (int8_t)q[4 + 32 * j + l];
                    u += ((p[16 + 32 * (j / 2) + l] >> (4 * (j & 1))) & 15) * c;
                    v += c;
                }
                s += sc * u;
                sm += m * v;
            }
            const float db = *(const float *)q;
            acc = fmaf((float)s, fp16_bits_to_f32(*(const uint16_t *)p) * db, acc);
            acc = fmaf((float)-sm, fp16_bits_to_f32(*(const uint16_t *)(p + 2)) * db, acc);
        }
    }
    g.y[t * g.ldy + n] = acc;
}

size_t mm_ws_bytes(int type, int btype, int64_t T, int64_t K) {
    if (btype != 0) return 0;
    return type == 2 ? (size_t)(T * (K / 32) * 34) : (size_t)(T * (K / 256) * 292);
}

int launch_mm(const MmArgs &g, hipStream_t st) {
    if (g.T <= 0) return 0;
    const int64_t nb = g.K / (g.type == 2 ? 32 : 256), bytes = g.type == 2 ? 34 : 292;
    const uint8_t *b = (const uint8_t *)g.b;
    int64_t ldb = g.ldb;
    if (g.btype == 0) {
        if (g.type == 2) hipLaunchKernelGGL(k_mm_rows_q8_0, dim3((unsigned)((nb * g.T + 255) / 256)), dim3(256), 0, st, (const float *)g.b, g.ldb / 4, nb, g.T, (uint8_t *)g.ws);
        else hipLaunchKernelGGL(k_mm_rows_q8_K, dim3((unsigned)((nb * g.T + 3) / 4)), dim3(256), 0, st, (const float *)g.b, g.ldb / 4, nb, g.T, (uint8_t *)g.ws);
        const int rc = hip_check_launch();
        if (rc) return rc;
        b = (const uint8_t *)g.ws;
        ldb = nb * bytes;
    }
    const dim3 grid((unsigned)((g.N * g.T + 255) / 256));
    if (g.type == 2) hipLaunchKernelGGL(k_mm_simple<2>, grid, dim3(256), 0, st, g, b, ldb);
    else hipLaunchKernelGGL(k_mm_simple<12>, grid, dim3(256), 0, st, g, b, ldb);
    return hip_check_launch();
}

}  // namespace mimoe
