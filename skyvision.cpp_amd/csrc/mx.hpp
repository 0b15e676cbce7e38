// mx.hpp - MXFP4 blocks (ggml type 39) and the operand of their products.
//
// A block is 17 bytes for 32 values: E8M0 scale byte e, then 16 bytes of E2M1
// codes (value j in the low nibble of byte j, value 16 + j in the high one); a
// value is 2^(e - 127) +-{0, .5, 1, 1.5, 2, 3, 4, 6}[code & 7]; e = 255 is NaN.
//
// The products' other operand is ggml's Q8_0 of the row (MXFP4's
// vec_dot_type): x^ = d q, d = amax / 127 as fp16, q = roundf(x / d) in
// [-127, 127].  With d = M 2^k (M its significand of at most 11 bits) x^ = n
// 2^k for the integer n = M q, |n| <= 127 * 2047 < 2^18, which is four
// balanced base-32 digits n = n0 + 32 n1 + 32^2 n2 + 32^3 n3, -16 <= n_i <= 15.
// E2M3 (6 bits) holds n_i / 8 exactly, its code being |n_i| and the sign, so
// x^ = sum_i E2M3(n_i) 2^(k + 5 i + 3) and a block's product with MXFP4
// weights is four scaled MFMAs (fp6 x fp4, scale bytes 2^(k + 5 i + 3) and e)
// without any unpacking of the weights and without a rounding before the
// sums: four times the work of one MFMA at four times the rate of fp16's.
//
// Operand layout (MxRows): the rows' digits, 96 bytes per block (digits 0..3's
// first 16 bytes, then digits 0..3's last 8 bytes; 32 codes of 6 bits in the
// weights' nibble order: code 2 j is value j, code 2 j + 1 value 16 + j), rows
// of an even number of blocks (a pair of blocks is 192 bytes at a multiple of
// 64); apart from them the rows' scale words, one per block (byte i: digit i's
// scale byte; 255 where the row's block holds a NaN or leaves the fp16 range
// of d), rows of a multiple of four words.  The blocks that fill up a row hold
// zeros.
//
// The products of few rows add the blocks' sums in fp64, where the significand
// costs nothing: their operand (the same MxRows, rows of nb blocks) holds the
// two digits of q alone, 48 bytes per block (digit 0's and 1's first 16 bytes,
// then their last 8), and a word per block: the float M / 1024 in its upper 24
// bits (NaN where x^ is none), digit 0's scale byte 2^(k + 10 + 3) in the low 8.
#pragma once

#include "common.hpp"
#include "launch.hpp"
#include "wave_ops.hpp"

namespace mimoe {

constexpr int MX_BYTES = 17;        // a block of weights
constexpr int MX_XB = 96;           // a block's digits in the operand
constexpr uint32_t MX_ONE = 127;    // scale byte of 1

constexpr int MX_FB = 48;           // a block's digits in the operand of few rows

// bytes of the digits and words of the scales of an operand row of nb blocks, and the bytes of both
__device__ __host__ constexpr int64_t mx_drow(int64_t nb) { return (nb + 1) / 2 * (2 * MX_XB); }
__device__ __host__ constexpr int64_t mx_srow(int64_t nb) { return (nb + 3) / 4 * 4; }
__device__ __host__ constexpr int64_t mx_row(int64_t nb) { return mx_drow(nb) + 4 * mx_srow(nb); }

// a + the value of the lane that CTRL pairs this one with (wave_ops.hpp)
template <int CTRL>
__device__ __forceinline__ double dpp_add(double a) {
    const uint64_t b = __builtin_bit_cast(uint64_t, a);
    const uint64_t o = ((uint64_t)(uint32_t)dpp_i<CTRL>((int)(b >> 32)) << 32) | (uint32_t)dpp_i<CTRL>((int)(uint32_t)b);
    return a + __builtin_bit_cast(double, o);
}

// a lane's 8 codes of digit i of its values' n (biased by 16 in every digit),
// 6 bits each, in the operand's order
__device__ __forceinline__ uint2 mx_digit(const uint32_t (&u)[8], int i) {
    uint32_t c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int t = (int)((u[(j >> 1) + 4 * (j & 1)] >> (5 * i)) & 31u) - 16;   // (value j / 2 of the low half, then of the high)
        c[j] = (uint32_t)(t < 0 ? 32 - t : t);
    }
    uint2 r;
    r.x = c[0] | c[1] << 6 | c[2] << 12 | c[3] << 18 | c[4] << 24 | c[5] << 30;
    r.y = c[5] >> 2 | c[6] << 4 | c[7] << 10;
    return r;
}

// A block by the four lanes 4 k .. 4 k + 3: lane s (= lane & 3) holds values 4
// s .. 4 s + 3 in v[0..3] and 16 + 4 s .. in v[4..7].  Its codes q, and d = M
// 2^(ex - 25) (ex at least 1); bad: d is no number.
struct MxBlock {
    int q[8], M;
    uint32_t ex;
    bool bad;
};
__device__ __forceinline__ MxBlock mx_block(const float (&v)[8]) {
    uint32_t m = 0;   // largest |x| by its bits: a NaN is above every number
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t a = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
        m = a > m ? a : m;
    }
    const uint32_t m1 = (uint32_t)dpp_i<0xB1>((int)m);
    m = m1 > m ? m1 : m;
    const uint32_t m2 = (uint32_t)dpp_i<0x4E>((int)m);
    m = m2 > m ? m2 : m;
    const float d = __builtin_bit_cast(float, m) / 127.0f;
    const float id = d != 0.0f ? 1.0f / d : 0.0f;
    const uint32_t dh = f32_to_fp16_bits(d), ex = dh >> 10, man = dh & 0x3ffu;   // (d >= 0 or NaN)
    MxBlock k;
    k.bad = (ex & 31u) == 31u;
    k.M = k.bad ? 0 : (int)(ex ? man + 1024u : man);
    k.ex = ex ? ex : 1u;
#pragma unroll
    for (int j = 0; j < 8; ++j) k.q[j] = (int)roundf(v[j] * id);
    return k;
}

// Block b of operand row r (of nb blocks): the lane writes digit s, lane 0 the
// scale word.  live: the lane writes (all four lanes of a block take part).
__device__ __forceinline__ void mx_store_block(const float (&v)[8], const MxRows &o, int64_t r, int64_t b, int nb, int s, bool live) {
    const MxBlock blk = mx_block(v);
    const uint32_t k = MX_ONE + 3 - 25 + blk.ex;
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = (uint32_t)(blk.M * blk.q[j] + 16 * (1 + 32 + 32 * 32 + 32 * 32 * 32));
    uint2 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = mx_digit(u, i);
    // 4 x 4 transpose among the four lanes: lane s gets digit s of the four
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        uint2 t = (s & 1) ? p[i] : p[i + 1];
        t.x = (uint32_t)dpp_i<0xB1>((int)t.x);
        t.y = (uint32_t)dpp_i<0xB1>((int)t.y);
        if (s & 1) p[i] = t;
        else p[i + 1] = t;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint2 t = (s & 2) ? p[i] : p[i + 2];
        t.x = (uint32_t)dpp_i<0x4E>((int)t.x);
        t.y = (uint32_t)dpp_i<0x4E>((int)t.y);
        if (s & 2) p[i] = t;
        else p[i + 2] = t;
    }
    if (!live) return;
    uint8_t *xb = o.d + r * mx_drow(nb) + MX_XB * b;
    *(uint4 *)(xb + 16 * s) = make_uint4(p[0].x, p[0].y | p[1].x << 16, p[1].x >> 16 | p[1].y << 16, p[2].x);
    *(uint2 *)(xb + 64 + 8 * s) = make_uint2(p[2].y | p[3].x << 16, p[3].x >> 16 | p[3].y << 16);
    if (s == 0) o.s[r * mx_srow(nb) + b] = blk.bad ? 0xffffffffu : k * 0x01010101u + 0x0f0a0500u;
}
// The same for few rows: lane s writes half s / 2 of digit s & 1
__device__ __forceinline__ void mx_store_few(const float (&v)[8], const MxRows &o, int64_t r, int64_t b, int nb, int s, bool live) {
    const MxBlock blk = mx_block(v);
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = (uint32_t)(blk.q[j] + 16 * (1 + 32));
    const uint2 p0 = mx_digit(u, 0), p1 = mx_digit(u, 1);
    uint2 t = (s & 1) ? p0 : p1;
    t.x = (uint32_t)dpp_i<0xB1>((int)t.x);
    t.y = (uint32_t)dpp_i<0xB1>((int)t.y);
    const uint2 lo = (s & 1) ? t : p0, hi = (s & 1) ? p1 : t;   // 6 bytes each
    if (!live) return;
    const uint32_t w0 = lo.x, w1 = lo.y | hi.x << 16, w2 = hi.x >> 16 | hi.y << 16;
    uint8_t *xb = o.d + r * (int64_t)(nb * MX_FB) + MX_FB * b;
    uint32_t *x16 = (uint32_t *)(xb + 16 * (s & 1)), *x8 = (uint32_t *)(xb + 32 + 8 * (s & 1));
    if (s < 2) {
        *(uint2 *)x16 = make_uint2(w0, w1);
        x16[2] = w2;
    } else {
        x16[3] = w0;
        *(uint2 *)x8 = make_uint2(w1, w2);
    }
    const uint32_t f = blk.bad ? 0x7fc00000u : __builtin_bit_cast(uint32_t, (float)blk.M * 0x1p-10f);
    if (s == 0) o.s[r * nb + b] = f | (blk.bad ? MX_ONE : MX_ONE + 3 + 10 - 25 + blk.ex);
}
// the blocks that fill up the row (mx_store_block), by the same lanes
__device__ __forceinline__ void mx_store_pad(const MxRows &o, int64_t r, int nb, int s) {
    if (nb & 1) {
        uint8_t *xb = o.d + r * mx_drow(nb) + MX_XB * (int64_t)nb;
        *(uint4 *)(xb + 16 * s) = make_uint4(0, 0, 0, 0);
        *(uint2 *)(xb + 64 + 8 * s) = make_uint2(0, 0);
    }
    for (int64_t b = nb; b & 3; ++b)
        if (s == 0) o.s[r * mx_srow(nb) + b] = MX_ONE * 0x01010101u;
}

// relu^2 between the two products, on either path: a NaN stays one (as in the
// gated forms), so an operand row that is no number shows in the layer's output
template <typename F>
__device__ __forceinline__ F mx_relu_sqr(F a) {
    const F r = a <= F(0) ? F(0) : a;
    return r * r;
}

// lane s's 8 values of the block at x
template <bool VEC>
__device__ __forceinline__ void mx_load8(const float *x, int s, float (&v)[8]) {
    if constexpr (VEC) {
        const float4 a = *(const float4 *)(x + 4 * s), b = *(const float4 *)(x + 16 + 4 * s);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = x[4 * s + j];
            v[4 + j] = x[16 + 4 * s + j];
        }
    }
}

// lane s's quarter of block b (of nb) of the row at src into operand row r;
// few: the operand of few rows
template <bool VEC>
__device__ __forceinline__ void mx_prep_quarter(const float *__restrict__ src, const MxRows &o, int64_t r, int64_t b, int nb, int s, bool few, bool live) {
    float v[8];
    mx_load8<VEC>(src + 32 * b, s, v);
    if (few) {
        mx_store_few(v, o, r, b, nb, s, live);
        return;
    }
    mx_store_block(v, o, r, b, nb, s, live);
    if (live && b == nb - 1) mx_store_pad(o, r, nb, s);
}
// Rows of 32 nb values (row r at src + r ld) into operand rows: four threads
// per block, thread i (of nrows nb 4, filled up to whole waves)
template <bool VEC>
__device__ __forceinline__ void mx_prep_thread(const float *__restrict__ src, int64_t ld, int64_t nrows, int nb, const MxRows &o, bool few, int64_t i) {
    const int64_t blk = i >> 2;
    const bool live = blk < nrows * nb;
    const int64_t r = live ? blk / nb : 0, b = live ? blk - r * nb : 0;
    mx_prep_quarter<VEC>(src + r * ld, o, r, b, nb, (int)(i & 3), few, live);
}
inline bool mx_prep_vec(const float *src, int64_t ld) { return ld % 4 == 0 && (uintptr_t)src % 16 == 0; }

// A weight block in registers: the five dwords from the one at or below its
// first byte (each holds a byte of the block: no read leaves the table's
// dwords), and its codes and scale byte; mis: its first byte's place there
struct MxRaw {
    uint32_t w[5];
};
__device__ __forceinline__ void mx_load(const uint8_t *p, MxRaw &r) {
    const uint8_t *q = p - ((uintptr_t)p & 3u);
    __builtin_memcpy(r.w, __builtin_assume_aligned(q, 4), 20);
}
__device__ __forceinline__ uint32_t mx_scale(const MxRaw &r, uint32_t mis) { return (r.w[0] >> (8 * mis)) & 0xffu; }
__device__ __forceinline__ void mx_codes(const MxRaw &r, uint32_t mis, uint32_t (&c)[4]) {
    // the codes start at byte mis + 1: in dword 0 (mis < 3) or 1
    const bool up = mis == 3u;
    const uint32_t sh = up ? 0u : mis + 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = up ? r.w[i + 1] : __builtin_amdgcn_alignbyte(r.w[i + 1], r.w[i], sh);
}

}  // namespace mimoe
