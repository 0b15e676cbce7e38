// k_mm.hip - dense products of 4-bit matrices and rows in 8 bits (mi_mul_mat):
//   y[t][n] = sum over blocks of (a's block . b's block), b in a's 8-bit form.
//   Q4_0 . Q8_0: d_a d_b sum (q - 8) c                                      (32 values)
//   Q4_K . Q8_K: d_b (d sum_j sc_j sum_j q c - dmin sum_j m_j sum_j c)     (256, j: 32 values)
// The sums over codes are exact integers (of a Q4_K block up to 63 * 15 * 127 * 256,
// 3.07e7: rounded once on the way to fp32), the blocks are added in fp32.
//
// Two kernels.  k_mv (up to 8 rows of b): a lane per 32 values of whole rows of
// the matrix on v_dot4_i32_i8, bound by the stream of the matrix: one row through
// 65536 x 2048 Q4_K (75 MB) 17.0 us = 4.5 TB/s out of the last-level cache, 18.6 us
// from memory (a large copy moves 5.1 TB/s); 2048 x 2048 3.6 us, of which the call's
// latency is most.
// k_mm (more): the codes' products on the int8 MFMA, whose 32 (16x16x32) or 64
// (16x16x64) products are one or two 32-value blocks of 16 tokens x 16 rows of
// the matrix, one group of 16 lanes per quarter of a block.  A lane holds a row's
// codes straight from the table's bytes; the tokens' operands lie in LDS in the
// lanes' order (MM records) for the whole K where they fit, written once per
// work-group, which then walks over row tiles: the matrix is read once per 16 to
// 64 tokens.  Bound by the vector instructions that unpack codes and apply the
// scales: 13 rows through 3712 x 2688 Q4_0 8.3 us (2.3 of them k_mm_rows), 200
// rows through 8192 x 2048 Q4_K 19.5 us (344 TFLOP/s; matrix units busy 28 % of
// k_mm's time, vector instructions besides issued in 47 %, the operands' way into
// LDS some 15 %).
#include <type_traits>

#include "b32.hpp"
#include "common.hpp"
#include "lanes.hpp"
#include "launch.hpp"
#include "wave_ops.hpp"

namespace mimoe {

typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(1))) void global_void_t;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));

constexpr int MM_LDS = 160 * 1024;
constexpr int MM_W = 8;   // waves of a k_mm work-group (16: 16 rows of 8192 x 2048 Q4_0 with the operands made in it 13.3 us, 8: 10.5)

// The operands of 16 tokens for one set of blocks (Q4_0: 4 blocks, 128 values;
// Q4_K: one of 256): the 8 code bytes of lane (token m, quarter g) per 32-value
// block j at 16 (64 (j / 2) + 16 g + m) + 8 (j & 1), then
//   Q4_0: the blocks' scales / 16, [4][16] f32
//   Q4_K: sums of 16 codes as fp16, 4 per lane (token m, sums 4 g .. 4 g + 3),
//         and the scales [16] f32
// A quarter g of a Q4_0 block is values 4 g .. 4 g + 3 and 16 + 4 g .. (what the
// nibbles of one dword of the table hold), of a Q4_K sub-block 8 g .. 8 g + 7.
template <int TYPE> struct MmRec;
template <> struct MmRec<2> { static constexpr int VALUES = 128, CODES = 2048, BYTES = 2048 + 256; };
template <> struct MmRec<12> { static constexpr int VALUES = 256, CODES = 4096, BYTES = 4096 + 512 + 64; };

// the largest |v| as bits (a NaN or an infinity: 0x7f800000 or more)
__device__ __forceinline__ uint32_t mm_amax8(const float (&v)[8]) {
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu;
        m = u > m ? u : m;
    }
    return m;
}
// the lowest bytes of eight words
__device__ __forceinline__ uint2 mm_bytes8(const uint32_t (&q)[8]) {
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __builtin_amdgcn_perm(q[2 * j + 1], q[2 * j], 0x0C0C0400u);
    return make_uint2(__builtin_amdgcn_perm(h[1], h[0], 0x05040100u), __builtin_amdgcn_perm(h[3], h[2], 0x05040100u));
}
// the lane's 8 of a block's values as codes, and the block's scale (NaN where a
// value is not finite or the scale leaves its type): Q8_0, 4 lanes a block.
// roundf(t): t + the number before 1/2 with t's sign, cut (|t| <= 127.5: the sum
// of a fraction of 1/2 or more rounds to the next integer, of less stays below).
__device__ __forceinline__ void mm_codes_q8_0(const float (&v)[8], uint2 &c, float &d) {
    uint32_t m = mm_amax8(v);
    m = dpp_max_u<0xB1>(m);
    m = dpp_max_u<0x4E>(m);
    const float df = __builtin_bit_cast(float, m) / 127.0f;
    const float id = df != 0.0f ? 1.0f / df : 0.0f;
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t = v[j] * id;
        q[j] = (uint32_t)(int)(t + __builtin_copysignf(0.49999997f, t));
    }
    c = mm_bytes8(q);
    d = (float)(_Float16)df;
    if (m >= 0x7f800000u || !(d <= 65504.f)) d = __builtin_nanf("");
}
// Q8_K, 32 lanes a block.  d and the codes change sign together with the sign
// that ggml gives them (of the first largest |x|): their products are the same.
// rint by the sum with 1.5 * 2^23, whose low bits hold the integer.
__device__ __forceinline__ void mm_codes_q8_K(const float (&v)[8], uint2 &c, float &d) {
    uint32_t m = mm_amax8(v);
    m = dpp_max_u<0xB1>(m);
    m = dpp_max_u<0x4E>(m);
    m = dpp_max_u<0x141>(m);
    m = dpp_max_u<0x140>(m);
    uint32_t o = m;
    swap16(m, o);
    m = o > m ? o : m;
    const bool zero = m == 0u, bad = m >= 0x7f800000u;
    const float is = zero || bad ? 0.f : 127.f / __builtin_bit_cast(float, m);
    d = bad ? __builtin_nanf("") : zero ? 0.f : 1 / is;
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __builtin_bit_cast(uint32_t, bad ? 12582912.f : is * v[i] + 12582912.f);
    c = mm_bytes8(q);
}

// A piece: 8 of a row's values, as they are read (SRC 1: fp32; 2: codes and the
// scale of an 8-bit block, NaN where it is not finite).  fetch only loads, so
// several go out before the first is used.  Zeros where the piece is not live.
template <int SRC> struct MmPiece;
template <> struct MmPiece<1> {
    float v[8];
    // values at x, the second four gap values behind the first
    __device__ __forceinline__ void fetch(const float *x, int gap, bool live) {
        float4_t a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if (live) {
            a = *(const float4_a4 *)x;
            b = *(const float4_a4 *)(x + gap);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
    }
};
template <> struct MmPiece<2> {
    uint2 c;
    float d;
};
// order of a piece in its block: Q4_0 operands of k_mm take values 4 g .. 4 g + 3
// and 16 + 4 g .. (g = p % 4: what the nibbles of a dword of the table hold), all
// others 8 in a row
template <int TYPE, int SRC, bool SPLIT>
__device__ __forceinline__ void mm_fetch(MmPiece<SRC> &r, const uint8_t *row, int p, bool live) {
    if constexpr (SRC == 1) {
        if constexpr (SPLIT) r.fetch((const float *)row + 32 * (p >> 2) + 4 * (p & 3), 16, live);
        else r.fetch((const float *)row + 8 * (int64_t)p, 4, live);
    } else {
        r.c = make_uint2(0u, 0u);
        r.d = 0.f;
        if (!live) return;
        if constexpr (TYPE == 2) {
            const uint8_t *b = row + 34 * (int64_t)(p >> 2);
            const int o = SPLIT ? 4 * (p & 3) : 8 * (p & 3);
            r.c = make_uint2(*(const u32_a2 *)(b + 2 + o), *(const u32_a2 *)(b + 2 + o + (SPLIT ? 16 : 4)));
            r.d = h2f(*(const uint16_t *)b);
        } else {
            const uint8_t *b = row + 292 * (int64_t)(p >> 5) + 4;
            r.c = make_uint2(*(const uint32_t *)(b + 8 * (p & 31)), *(const uint32_t *)(b + 8 * (p & 31) + 4));
            r.d = *(const float *)(b - 4);
        }
    }
}
// its codes and scale; the lanes that share a block (4 or 32, aligned) call it together
template <int TYPE, int SRC>
__device__ __forceinline__ void mm_codes(const MmPiece<SRC> &r, uint2 &c, float &d) {
    if constexpr (SRC == 1) {
        if constexpr (TYPE == 2) mm_codes_q8_0(r.v, c, d);
        else mm_codes_q8_K(r.v, c, d);
    } else {
        c = r.c;
        d = fabsf(r.d) <= 3.402823466e38f ? r.d : __builtin_nanf("");   // (an fp16 infinity is one here)
    }
}

// piece p of token row m of a tile into the tile's record at o
template <int TYPE, int SRC>
__device__ __forceinline__ void mm_put(const MmPiece<SRC> &r, int p, int m, uint8_t *o) {
    uint2 c;
    float d;
    mm_codes<TYPE, SRC>(r, c, d);
    if constexpr (TYPE == 2) {
        const int j = (p >> 2) & 3, g = p & 3;
        *(uint2 *)(o + 16 * (64 * (j >> 1) + 16 * g + m) + 8 * (j & 1)) = c;
        if (g == 0) *(float *)(o + 2048 + 64 * j + 4 * m) = d * 0.0625f;
    } else {
        const int e = p & 31, j = e >> 2, g = e & 3;   // sub-block and quarter
        *(uint2 *)(o + 16 * (64 * (j >> 1) + 16 * g + m) + 8 * (j & 1)) = c;
        int s = __builtin_amdgcn_sdot4(0x01010101, (int)c.x, __builtin_amdgcn_sdot4(0x01010101, (int)c.y, 0, false), false);
        s += dpp_i<0xB1>(s);
        // sum of values 16 (e / 2) ..: lane quarter e / 8, slot e / 2 % 4
        if (!(e & 1)) *(_Float16 *)(o + 4096 + 8 * (16 * (e >> 3) + m) + 2 * ((e >> 1) & 3)) = (_Float16)s;
        if (e == 0) *(float *)(o + 4608 + 4 * m) = d;
    }
}

// records of a call's rows: ws + ((tile of 16 tokens) * nsets + set) * BYTES
template <int TYPE, int SRC>
__global__ void __launch_bounds__(256) k_mm_rows(const uint8_t *b, int64_t ldb, int64_t T, int K, int nsets, uint8_t *ws) {
    using R = MmRec<TYPE>;
    const int64_t t = blockIdx.y;
    const int p = blockIdx.x * 256 + threadIdx.x, set = p / (R::VALUES / 8);
    if (set >= nsets) return;   // whole sets of lanes
    MmPiece<SRC> r;
    mm_fetch<TYPE, SRC, TYPE == 2>(r, b + t * ldb, p, 8 * (int64_t)p < K);
    mm_put<TYPE, SRC>(r, p, (int)(t & 15), ws + ((t >> 4) * nsets + set) * R::BYTES);
}

struct MmPlan {
    int src;       // operands: 0 records at ws, 1 fp32 rows (fewer than MM_PREP_T), 2 rows in 8 bits
    int nsets;     // sets of a row
    int chunks, cs;  // chunks of cs sets whose operands lie in LDS at a time
    int wk;        // waves that share a row tile, each taking every wk-th step of sets
    int ntiles;    // row tiles of 16
};

// ---------------------------------------------------------------- one set
template <int TYPE> struct MmRaw;
template <> struct MmRaw<2> { u32x4 q; uint32_t d; };
template <> struct MmRaw<12> { u32x4 h; uint2 q[4]; };

template <int TYPE>
__device__ __forceinline__ void mm_load(MmRaw<TYPE> &r, const uint8_t *row, int set, int nb, int g) {
    if constexpr (TYPE == 2) {
        const int b = imin(4 * set + g, nb - 1);
        const uint8_t *p = row + 18 * b;
        r.q = *(const u32x4_a2 *)(p + 2);
        r.d = *(const uint16_t *)p;
    } else {
        const uint8_t *p = row + 144 * (int64_t)set;
        r.h = *(const u32x4 *)p;
#pragma unroll
        for (int c = 0; c < 4; ++c) r.q[c] = *(const uint2 *)(p + 16 + 32 * c + 8 * g);
    }
}

// a b + c, |a|, |b| < 2^23, one instruction (the empty statement keeps a chain of
// them from being regrouped into products and three-operand additions)
__device__ __forceinline__ int mad24(int a, int b, int c) {
    int r = __mul24(a, b) + c;
    asm("" : "+v"(r));
    return r;
}
__device__ __forceinline__ long mm_u64(uint32_t lo, uint32_t hi) { return (long)(((uint64_t)hi << 32) | lo); }
// acc[mt] += the set's part for token tile mt; x: the set's record of tile 0,
// xs: bytes from a tile's record to the next tile's.  NI: rows of a lane group's
// four that hold tokens.
template <int TYPE, int MT, int NI>
__device__ __forceinline__ void mm_set(const MmRaw<TYPE> &r, const uint8_t *x, int xs, int set, int nb, int lane,
                                       float (&acc)[MT][NI]) {
    const int g = lane >> 4;
    const i32x4 z = {0, 0, 0, 0};
    typedef float fNI __attribute__((ext_vector_type(NI)));
    if constexpr (TYPE == 2) {
        // lane group g holds block g of the set; the products want dword g of
        // block j in group g: a 4 x 4 transpose over the groups
        uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
        swap16(w[0], w[1]);
        swap16(w[2], w[3]);
        swap32(w[0], w[2]);
        swap32(w[1], w[3]);
        // block j's scale in every group
        uint32_t d[4];
        d[0] = d[1] = 4 * set + g < nb ? r.d : 0u;
        swap16(d[0], d[1]);
        d[2] = d[0];
        d[3] = d[1];
        swap32(d[0], d[2]);
        swap32(d[1], d[3]);
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
            u32x4 xv[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) xv[m] = *(const u32x4 *)(x + m * xs + 1024 * jj + 16 * lane);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = 2 * jj + h;
                const float da = h2f((uint16_t)d[j]);
                // 16 (q - 8) as signed bytes: the nibble on top, its highest bit turned
                const uint32_t lo = ((w[j] << 4) & 0xF0F0F0F0u) ^ 0x80808080u, hi = (w[j] & 0xF0F0F0F0u) ^ 0x80808080u;
                const long wb = mm_u64(lo, hi);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const long xa = h ? mm_u64(xv[m].z, xv[m].w) : mm_u64(xv[m].x, xv[m].y);
                    const i32x4 c = __builtin_amdgcn_mfma_i32_16x16x32_i8(xa, wb, z, 0, 0, 0);
                    const fNI db = *(const fNI *)(x + m * xs + 2048 + 64 * j + 16 * g);
#pragma unroll
                    for (int i = 0; i < NI; ++i) acc[m][i] = fmaf((float)c[i], da * db[i], acc[m][i]);
                }
                if constexpr (MT > 2) __builtin_amdgcn_sched_barrier(0);   // (keeps the operands of later blocks in LDS)
            }
        }
    } else {
        const uint32_t w0 = r.h.y, w1 = r.h.z, w2 = r.h.w;
        const float d = h2f((uint16_t)(r.h.x & 0xffff)), dm = h2f((uint16_t)(r.h.x >> 16));
        const uint32_t sc[2] = {w0 & 0x3F3F3F3Fu, (w2 & 0x0F0F0F0Fu) | ((w0 >> 2) & 0x30303030u)};
        const uint32_t mn[2] = {w1 & 0x3F3F3F3Fu, ((w2 >> 4) & 0x0F0F0F0Fu) | ((w1 >> 2) & 0x30303030u)};
        // the minima of sub-blocks 2 g, 2 g + 1, twice each (a sub-block has two sums of 16 codes)
        const uint32_t mg = (g & 2 ? mn[1] : mn[0]) >> (16 * (g & 1));
        const _Float16 m0 = (_Float16)(float)(mg & 0xffu), m1 = (_Float16)(float)((mg >> 8) & 0xffu);
        const half4_t mb = {m0, m0, m1, m1};
        int s[MT][NI];
        if constexpr (MT == 1) {
            // a sub-block a MFMA, its scale on the sums
#pragma unroll
            for (int i = 0; i < NI; ++i) s[0][i] = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const long lo = mm_u64(r.q[c].x & 0x0F0F0F0Fu, r.q[c].y & 0x0F0F0F0Fu);
                const long hi = mm_u64((r.q[c].x >> 4) & 0x0F0F0F0Fu, (r.q[c].y >> 4) & 0x0F0F0F0Fu);
                const int s0 = (int)((sc[c >> 1] >> (16 * (c & 1))) & 0xffu), s1 = (int)((sc[c >> 1] >> (16 * (c & 1) + 8)) & 0xffu);
                const u32x4 xv = *(const u32x4 *)(x + 1024 * c + 16 * lane);
                const i32x4 a = __builtin_amdgcn_mfma_i32_16x16x32_i8(mm_u64(xv.x, xv.y), lo, z, 0, 0, 0);
                const i32x4 b = __builtin_amdgcn_mfma_i32_16x16x32_i8(mm_u64(xv.z, xv.w), hi, z, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < NI; ++i) s[0][i] = mad24(b[i], s1, mad24(a[i], s0, s[0][i]));   // |a| < 2^16, scales below 64
            }
        } else {
            // scale times code as 8 h + l, both digits in 8 bits (15 * 7 = 105): two sub-blocks
            // a MFMA, the whole block's sums of either digit with no other instruction between
            const uint32_t dl[2] = {sc[0] & 0x07070707u, sc[1] & 0x07070707u};
            const uint32_t dh[2] = {(sc[0] >> 3) & 0x07070707u, (sc[1] >> 3) & 0x07070707u};
            i32x4 sl[MT], sh[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) sl[m] = sh[m] = z;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t q[4] = {r.q[c].x & 0x0F0F0F0Fu, r.q[c].y & 0x0F0F0F0Fu, (r.q[c].x >> 4) & 0x0F0F0F0Fu,
                                       (r.q[c].y >> 4) & 0x0F0F0F0Fu};
                i32x4 wl, wh;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    // the sub-block's digits in both halves of a word; bytes stay below 256 in a product
                    const uint32_t sel = 0x0C000C00u + 0x00010001u * (2 * (c & 1) + (k >> 1));
                    const ushort2_t l = __builtin_bit_cast(ushort2_t, __builtin_amdgcn_perm(0u, dl[c >> 1], sel));
                    const ushort2_t h = __builtin_bit_cast(ushort2_t, __builtin_amdgcn_perm(0u, dh[c >> 1], sel));
                    const ushort2_t v = __builtin_bit_cast(ushort2_t, q[k]);
                    wl[k] = __builtin_bit_cast(int, v * l);
                    wh[k] = __builtin_bit_cast(int, v * h);
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const i32x4 xv = *(const i32x4 *)(x + m * xs + 1024 * c + 16 * lane);
                    sl[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv, wl, sl[m], 0, 0, 0);
                    sh[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv, wh, sh[m], 0, 0, 0);
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < NI; ++i) s[m][i] = sl[m][i] + 8 * sh[m][i];
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const half4_t bs = *(const half4_t *)(x + m * xs + 4096 + 8 * lane);
            const float4_t zf = {0.f, 0.f, 0.f, 0.f};
            const float4_t mm = __builtin_amdgcn_mfma_f32_16x16x16f16(bs, mb, zf, 0, 0, 0);
            const fNI db = *(const fNI *)(x + m * xs + 4608 + 16 * g);
#pragma unroll
            for (int i = 0; i < NI; ++i) acc[m][i] = fmaf(fmaf(d, (float)s[m][i], -(dm * mm[i])), db[i], acc[m][i]);
        }
    }
}

// sets of a step (their loads go together): 256 values
template <int TYPE> constexpr int MM_U = TYPE == 2 ? 2 : 1;

// Work-group (x, y) of W waves: tokens 16 MT y .. (NI < 4: 4 NI tokens at most,
// token t in row 4 (t / NI) + t % NI of the MFMA's), row tiles x (W / wk), +
// gridDim.x (W / wk) ..
// Waves of a SIMD: two (one work-group a CU).  Told two or three, the compiler
// orders the steps of 64 tokens as it does with more registers in use (65536 x 2048,
// 1024 rows, Q4_0 564 -> 543 us, Q4_K 375 -> 363; told two only, Q4_0 617).
template <int TYPE, int MT, int NI>
__global__ void __launch_bounds__(64 * MM_W) __attribute__((amdgpu_waves_per_eu(2, 3))) k_mm(MmArgs g, MmPlan p) {
    using R = MmRec<TYPE>;
    constexpr int U = MM_U<TYPE>, W = MM_W;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wk = p.wk, wn = W / wk, kw = wave % wk, nw = wave / wk;
    const int64_t t0 = (int64_t)blockIdx.y * 16 * MT;
    const int nt = (int)(g.T - t0 < 16 * MT ? g.T - t0 : 16 * MT);   // tokens here
    const int nb = (int)(g.K / 32);
    const int xs = p.cs * R::BYTES;   // a token tile's records in LDS
    float *red = (float *)(lds + MT * xs);   // [2][W][MT][64][NI]

    // the operands of chunk ch
    auto fill = [&](int ch) __attribute__((always_inline)) {
        const int s0 = ch * p.cs, ns = imin(p.cs, p.nsets - s0);
        if (p.src == 0) {
            const int per = ns * (R::BYTES / 16);
            for (int m = 0; m < MT && 16 * m < nt; ++m) {
                const uint8_t *src = (const uint8_t *)g.ws + ((t0 / 16 + m) * p.nsets + s0) * R::BYTES;
                for (int i = 64 * wave; i < per; i += 64 * W)   // 1 KB a wave, straight into LDS
                    if (i + lane < per)
                        __builtin_amdgcn_global_load_lds((const global_void_t *)(src + 16 * (i + lane)),
                                                         (lds_void_t *)(lds + m * xs + 16 * i), 16, 0, 0);
            }
            vm_drain();
        } else {
            constexpr int PS = R::VALUES / 8;      // pieces of a set: 16 or 32
            const int pt = (ns * PS + 63) & ~63;   // of a token, rounded up to whole waves: a wave's 64 are of one token
            auto make = [&](auto src) __attribute__((always_inline)) {
                constexpr int SRC = decltype(src)::value, NB = 4;   // NB pieces' loads go out together
                int t = 0, i = tid;
                while (t < nt) {
                    MmPiece<SRC> r[NB];
                    int tt[NB], ii[NB];
#pragma unroll
                    for (int n = 0; n < NB; ++n, i += 64 * W) {
                        while (i >= pt && t < nt) {
                            i -= pt;
                            ++t;
                        }
                        tt[n] = i < ns * PS ? t : nt;   // (else past the row's sets: whole groups of lanes that share a block)
                        ii[n] = i;
                        if (tt[n] < nt)
                            mm_fetch<TYPE, SRC, TYPE == 2>(r[n], (const uint8_t *)g.b + (t0 + t) * g.ldb, s0 * PS + i,
                                                           8 * (int64_t)(s0 * PS + i) < g.K);
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        if (tt[n] >= nt) continue;
                        const int m = NI == 4 ? tt[n] & 15 : 4 * (tt[n] / NI) + tt[n] % NI;
                        mm_put<TYPE, SRC>(r[n], ii[n], m, lds + (NI == 4 ? tt[n] >> 4 : 0) * xs + ii[n] / PS * R::BYTES);
                    }
                }
            };
            // (fp32 rows from MM_PREP_T on always come as records)
            if constexpr (NI < 4) {
                if (p.src == 1) make(std::integral_constant<int, 1>{});
                else make(std::integral_constant<int, 2>{});
            } else {
                make(std::integral_constant<int, 2>{});
            }
        }
    };

    const int stride = (int)gridDim.x * wn;   // tiles from one round to the next
    // the step whose loads are issued next: its tile, chunk end and first set
    int ltile = (int)blockIdx.x * wn + nw, lch = 0, lset = kw * U;
    MmRaw<TYPE> nxt[U];
    const uint8_t *lrow = nullptr;
    auto row_of = [&]() __attribute__((always_inline)) {
        const int64_t n = 16 * (int64_t)imin(ltile, p.ntiles - 1) + (lane & 15);
        lrow = g.a + (n < g.N ? n : g.N - 1) * g.row_bytes;
    };
    // (clamped in the rows and in K: what lies past them is loaded again and dropped)
    auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) mm_load<TYPE>(nxt[u], lrow, imin(lset + u, p.nsets - 1), nb, lane >> 4);
    };
    auto advance = [&]() __attribute__((always_inline)) {
        lset += wk * U;
        if (lset >= imin((lch + 1) * p.cs, p.nsets)) {
            if (++lch == p.chunks) {
                lch = 0;
                ltile += stride;
                row_of();
            }
            lset = lch * p.cs + kw * U;
        }
    };
    row_of();
    load();
    if (p.chunks == 1) {
        fill(0);
        __syncthreads();
    }
    int par = 0;
    for (int tb = (int)blockIdx.x * wn; tb < p.ntiles; tb += stride) {   // the work-group's tiles tb .. tb + wn - 1
        float acc[MT][NI];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < NI; ++i) acc[m][i] = 0.f;
        for (int ch = 0; ch < p.chunks; ++ch) {
            if (p.chunks > 1) {
                __syncthreads();
                fill(ch);
                __syncthreads();
            }
            const int end = imin((ch + 1) * p.cs, p.nsets);
            int set = ch * p.cs + kw * U;
            if (set >= end) advance(), load();   // no step here: the cursor moves with the loops
            for (; set < end; set += wk * U) {
                MmRaw<TYPE> cur[U];
#pragma unroll
                for (int u = 0; u < U; ++u) cur[u] = nxt[u];
                advance();
                load();
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (set + u < end)
                        mm_set<TYPE, MT, NI>(cur[u], lds + (set + u - ch * p.cs) * R::BYTES, xs, set + u, nb, lane, acc);
            }
        }
        if (wk == 1) {
            const int64_t n = 16 * (int64_t)(tb + nw) + (lane & 15);
            if (n < g.N) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        const int t = 16 * m + NI * (lane >> 4) + i;
                        if (t < nt) g.y[(t0 + t) * g.ldy + n] = acc[m][i];
                    }
            }
        } else {
            // the tiles' parts, one buffer per parity: a wave that writes a buffer
            // again is past the barrier after its last use
            float *rb = red + par * (W * MT * 64 * NI);
            par ^= 1;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < NI; ++i) rb[((wave * MT + m) * 64 + lane) * NI + i] = acc[m][i];
            __syncthreads();
            for (int e = tid; e < wn * MT * 64 * NI; e += 64 * W) {
                const int i = e % NI, l = (e / NI) & 63, m = e / (NI * 64) % MT, w = e / (NI * 64 * MT);
                const int t = 16 * m + NI * (l >> 4) + i;
                const int64_t n = 16 * (int64_t)(tb + w) + (l & 15);
                if (t >= nt || n >= g.N) continue;
                float v = rb[((w * wk) * MT + m) * 64 * NI + l * NI + i];
                for (int k = 1; k < wk; ++k) v += rb[((w * wk + k) * MT + m) * 64 * NI + l * NI + i];
                g.y[(t0 + t) * g.ldy + n] = v;
            }
        }
    }
}

// ---------------------------------------------------------------- up to 8 rows
// One lane per 32 values of a row of the matrix (Q4_0: a block; Q4_K: 16 bytes
// of codes, 16 values of one sub-block and 16 of the next), 2^lg lanes per
// row: a wave's loads are runs of whole rows.  The dots run on v_dot4_i32_i8.
//
// The tokens' operands per unit of 32 values, in LDS: the codes of the low
// nibbles (16 bytes), of the high ones (16 bytes), and {scale f32, Q4_0: -8 times
// the codes' sum; Q4_K: the two sums of 16 codes, as halves of a word}.
struct MvPlan {
    int src;           // as MmPlan (1 or 2)
    int nu;            // units of a row
    int lg, chunks;    // lanes per row (log2), units of a row / lanes, rounded up
    int64_t batches;   // of R * 64 / lanes rows
};

// piece p of a token's row into its operands
template <int TYPE, int SRC>
__device__ __forceinline__ void mv_put(const MmPiece<SRC> &r, int p, bool live, uint8_t *lo, uint8_t *hi, uint2 *sc) {
    uint2 c;
    float d;
    mm_codes<TYPE, SRC>(r, c, d);
    int s = __builtin_amdgcn_sdot4(0x01010101, (int)c.x, __builtin_amdgcn_sdot4(0x01010101, (int)c.y, 0, false), false);
    s += dpp_i<0xB1>(s);
    if constexpr (TYPE == 2) {
        s += dpp_i<0x4E>(s);
        if (!live) return;
        *(uint2 *)((p & 2 ? hi : lo) + 16 * (p >> 2) + 8 * (p & 1)) = c;
        if ((p & 3) == 0) sc[p >> 2] = make_uint2(__builtin_bit_cast(uint32_t, d), (uint32_t)(-8 * s));
    } else {
        if (!live) return;
        // sub-block j = p / 4 % 8: bits of chunk j / 2, low or high nibbles by j & 1; half p / 2 & 1
        const int j = (p >> 2) & 7, unit = 8 * (p >> 5) + 2 * (j >> 1) + ((p >> 1) & 1);
        *(uint2 *)((j & 1 ? hi : lo) + 16 * unit + 8 * (p & 1)) = c;
        if (!(p & 1)) {
            ((int16_t *)(sc + unit))[2 + (j & 1)] = (int16_t)s;
            if (!(j & 1)) *(float *)(sc + unit) = d;
        }
    }
}

// sum over aligned groups of 2^lg lanes (8 .. 64)
__device__ __forceinline__ float mv_sum(float v, int lg) {
    v += dpp_f<0xB1>(v);
    v += dpp_f<0x4E>(v);
    v += dpp_f<0x141>(v);
    if (lg > 3) v += dpp_f<0x140>(v);
    if (lg > 4) {
        uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
        swap16(a, b);
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    if (lg > 5) {
        uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
        swap32(a, b);
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    return v;
}

template <int TYPE> struct MvRaw;
template <> struct MvRaw<2> { u32x4 q; uint32_t d; };
template <> struct MvRaw<12> { u32x4 h, q; };

template <int TYPE, int T, int R, int W>
__global__ void __launch_bounds__(64 * W) k_mv(MmArgs g, MvPlan p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nl = 1 << p.lg, l = lane & (nl - 1), rw = 64 >> p.lg;   // lanes of a row, rows of a load
    const int64_t step = (int64_t)gridDim.x * W;
    int64_t b = (int64_t)blockIdx.x * W + wave, lb = b;
    int lch = 0;
    MvRaw<TYPE> nxt[R];
    // (clamped in the rows and in K: what lies past them is loaded again and dropped)
    auto load = [&]() __attribute__((always_inline)) {
        const int u = imin((lch << p.lg) + l, p.nu - 1);
        const int64_t n0 = (lb < p.batches ? lb : p.batches - 1) * (R * rw) + (lane >> p.lg);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t n = n0 + r * rw;
            const uint8_t *a = g.a + (n < g.N ? n : g.N - 1) * g.row_bytes;
            if constexpr (TYPE == 2) {
                nxt[r].q = *(const u32x4_a2 *)(a + 18 * u + 2);
                nxt[r].d = *(const uint16_t *)(a + 18 * u);
            } else {
                a += 144 * (int64_t)(u >> 3);
                nxt[r].h = *(const u32x4 *)a;
                nxt[r].q = *(const u32x4 *)(a + 16 + 16 * (u & 7));
            }
        }
        if (++lch == p.chunks) {
            lch = 0;
            lb += step;
        }
    };
    load();
    const int pieces = 4 * p.nu, pt = (pieces + 63) & ~63;
    const int xb = 40 * p.nu;   // a token's operands
    auto make = [&](auto src) __attribute__((always_inline)) {
        constexpr int SRC = decltype(src)::value, NB = T > 2 ? 2 : 1;   // NB pieces' loads go out together
        int t = 0, i = tid;
        while (t < T) {
            MmPiece<SRC> r[NB];
            int tt[NB], ii[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n, i += 64 * W) {
                while (i >= pt && t < T) {
                    i -= pt;
                    ++t;
                }
                tt[n] = t;
                ii[n] = i;
                if (t < T) mm_fetch<TYPE, SRC, false>(r[n], (const uint8_t *)g.b + t * g.ldb, i, i < pieces);
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                if (tt[n] >= T) continue;   // (whole waves: a wave's 64 pieces are of one token)
                uint8_t *o = lds + tt[n] * xb;
                mv_put<TYPE, SRC>(r[n], ii[n], ii[n] < pieces, o, o + 16 * p.nu, (uint2 *)(o + 32 * p.nu));
            }
        }
    };
    if (p.src == 1) make(std::integral_constant<int, 1>{});
    else make(std::integral_constant<int, 2>{});
    __syncthreads();
    for (; b < p.batches; b += step) {
        float acc[R][T];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < T; ++t) acc[r][t] = 0.f;
        for (int ch = 0; ch < p.chunks; ++ch) {
            MvRaw<TYPE> cur[R];
#pragma unroll
            for (int r = 0; r < R; ++r) cur[r] = nxt[r];
            load();
            const int u0 = (ch << p.lg) + l, u = imin(u0, p.nu - 1);
            const bool live = u0 < p.nu;
            u32x4 xl[T], xh[T];
            uint2 xs[T];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const uint8_t *o = lds + t * xb;
                xl[t] = *(const u32x4 *)(o + 16 * u);
                xh[t] = *(const u32x4 *)(o + 16 * p.nu + 16 * u);
                xs[t] = *(const uint2 *)(o + 32 * p.nu + 8 * u);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if constexpr (TYPE == 2) {
                    const float da = live ? h2f((uint16_t)cur[r].d) : 0.f;
                    int s[T];
#pragma unroll
                    for (int t = 0; t < T; ++t) s[t] = (int)xs[t].y;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int lo = (int)(cur[r].q[j] & 0x0F0F0F0Fu), hi = (int)((cur[r].q[j] >> 4) & 0x0F0F0F0Fu);
#pragma unroll
                        for (int t = 0; t < T; ++t)
                            s[t] = __builtin_amdgcn_sdot4(hi, (int)xh[t][j], __builtin_amdgcn_sdot4(lo, (int)xl[t][j], s[t], false), false);
                    }
#pragma unroll
                    for (int t = 0; t < T; ++t)
                        acc[r][t] = fmaf((float)s[t], da * __builtin_bit_cast(float, xs[t].x), acc[r][t]);
                } else {
                    const uint32_t w0 = cur[r].h.y, w1 = cur[r].h.z, w2 = cur[r].h.w;
                    const float d = live ? h2f((uint16_t)(cur[r].h.x & 0xffff)) : 0.f;
                    const float dm = live ? h2f((uint16_t)(cur[r].h.x >> 16)) : 0.f;
                    // scales and minima of sub-blocks 2 c, 2 c + 1, c = u / 2 % 4
                    const uint32_t sc = (l & 4 ? (w2 & 0x0F0F0F0Fu) | ((w0 >> 2) & 0x30303030u) : w0 & 0x3F3F3F3Fu) >> (8 * (l & 2));
                    const uint32_t mn = (l & 4 ? ((w2 >> 4) & 0x0F0F0F0Fu) | ((w1 >> 2) & 0x30303030u) : w1 & 0x3F3F3F3Fu) >> (8 * (l & 2));
                    int s0[T], s1[T];
#pragma unroll
                    for (int t = 0; t < T; ++t) s0[t] = s1[t] = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int lo = (int)(cur[r].q[j] & 0x0F0F0F0Fu), hi = (int)((cur[r].q[j] >> 4) & 0x0F0F0F0Fu);
#pragma unroll
                        for (int t = 0; t < T; ++t) {
                            s0[t] = __builtin_amdgcn_sdot4(lo, (int)xl[t][j], s0[t], false);
                            s1[t] = __builtin_amdgcn_sdot4(hi, (int)xh[t][j], s1[t], false);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < T; ++t) {
                        const int s = __mul24(s0[t], (int)(sc & 0xffu)) + __mul24(s1[t], (int)((sc >> 8) & 0xffu));
                        const int m = __mul24((int)(int16_t)xs[t].y, (int)(mn & 0xffu)) + __mul24((int)xs[t].y >> 16, (int)((mn >> 8) & 0xffu));
                        acc[r][t] = fmaf(fmaf(d, (float)s, -(dm * (float)m)), __builtin_bit_cast(float, xs[t].x), acc[r][t]);
                    }
                }
            }
        }
        const int64_t n0 = b * (R * rw) + (lane >> p.lg);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const float v = mv_sum(acc[r][t], p.lg);
                const int64_t n = n0 + r * rw;
                if (l == 0 && n < g.N) g.y[t * g.ldy + n] = v;
            }
    }
}

// Two work-groups of 8 waves a CU (one of 16): every work-group makes the
// operands for itself, so few walk over many rows (65536 x 2048 Q4_K, one row:
// 8 work-groups of 4 waves a CU 17.2 us, 2 of 8 16.4).
constexpr int MV_WAVES = 4096;   // waves of the device at a time

// log2 of the lanes of a row: the fewest rounds of loads, over the chunks of a
// row and the batches of a wave; the most lanes (the longest runs of a load)
// among equals
static int mv_lg(int64_t nu, int64_t N, int R) {
    int best = 6;
    int64_t rounds = INT64_MAX;
    for (int lg = 6; lg >= 3; --lg) {
        const int64_t chunks = (nu + (1 << lg) - 1) >> lg, rows = R * (64 >> lg), batches = (N + rows - 1) / rows;
        const int64_t c = chunks * ((batches + MV_WAVES - 1) / MV_WAVES);
        if (c < rounds) rounds = c, best = lg;
    }
    return best;
}

template <int TYPE, int T, int R, int W>
static int mv_go(const MmArgs &g, hipStream_t st) {
    MvPlan p = {};
    p.src = g.btype != 0 ? 2 : 1;
    p.nu = (int)(g.K / 32);
    p.lg = mv_lg(p.nu, g.N, R);
    p.chunks = (p.nu + (1 << p.lg) - 1) >> p.lg;
    const int64_t rows = R * (64 >> p.lg);   // of a wave
    p.batches = (g.N + rows - 1) / rows;
    const int64_t most = (p.batches + W - 1) / W, cap = MV_WAVES / W;
    const dim3 grid((unsigned)(most < cap ? most : cap)), block(64 * W);
    hipLaunchKernelGGL((k_mv<TYPE, T, R, W>), grid, block, (size_t)T * 40 * p.nu, st, g, p);
    return hip_check_launch();
}

// Rows of a lane: one where few, and work-groups of 16 waves, which share the
// operands (8192 x 2048 Q4_0, one row of b: 4 waves 6.2 us, 16 4.3); more loads in
// flight where many: two (16384 x 2048 Q4_0: 7.0 -> 6.1 us), four, as far as the
// registers allow (65536 x 2048 Q4_0 from memory: two 23.7 us, four 21.9; 16384: 6.1 and 8.0)
template <int TYPE, int T>
static int mv_launch(const MmArgs &g, hipStream_t st) {
    if constexpr (T <= 2)
        if (g.N >= 12 * MV_WAVES) return mv_go<TYPE, T, 4, 8>(g, st);
    if (g.N >= 4 * MV_WAVES) return mv_go<TYPE, T, (T <= 4 ? 2 : 1), 8>(g, st);
    return mv_go<TYPE, T, 1, 16>(g, st);
}

// Up to 8 rows of b, while the dots are not what bounds it: the time of these
// kernels grows with the rows of b, that of k_mm hardly does, but for its operands
// (columns of 2048, us here and there: Q4_0 6 rows 8192 x 2048 8.5 and 9.8, 16384
// 13.6 and 12.7, 4 rows 65536 30.7 and 30.9; Q4_K 4 rows 8192 7.4 and 8.0, 16384 11.8
// and 10.1, 2 rows 65536 22.7 and 24.3).
template <int TYPE>
static bool mv_ok(const MmArgs &g) {
    if (g.T > 8 || g.T * 40 * (g.K / 32) > MM_LDS) return false;
    return g.T <= (TYPE == 2 ? 4 : 2) || g.T * g.N * g.K <= (int64_t)9 << (TYPE == 2 ? 24 : 23);
}

constexpr int64_t MM_PASS_T = 32768;   // rows of one pass (grid dimensions)
// From so many rows on (8 rows: where k_mv does not take them) their records are
// written by a launch of their own, else every work-group makes them for itself (2048
// columns, in the work-groups and with the launch: 13 fp32 rows 2048 x Q4_0 9.5 and
// 8.4 us, Q4_K 9.2 and 7.6; 9 rows 8192 x Q4_0 10.3 and 9.9, 32768 20.2 and 19.8; norm
// and product of 200 rows in 8 bits, 8192 x Q4_K 32.7 and 22.3, 64 rows of 8192
// columns, 2048 x Q4_0 50 and 23)
constexpr int64_t MM_PREP_T = 8;
static_assert(MM_PREP_T <= 9, "NI 2 holds 8 rows");

size_t mm_ws_bytes(int type, int64_t T, int64_t K) {
    if (T < MM_PREP_T) return 0;
    return type == 2 ? (size_t)((T + 15) / 16 * ((K + 127) / 128) * MmRec<2>::BYTES)
                     : (size_t)((T + 15) / 16 * (K / 256) * MmRec<12>::BYTES);
}

template <int TYPE, int MT, int NI>
static int mm_go(const MmArgs &g, MmPlan p, hipStream_t st) {
    using R = MmRec<TYPE>;
    constexpr int W = MM_W;
    const int64_t slices = (g.T + 16 * MT - 1) / (16 * MT);
    // waves that share a row tile: the fewest that give every CU eight (8192 x 2048
    // Q4_0, 16 rows: 9.9 us, sixteen 11.8; 128 rows Q4_K: 16.7 and 18.1)
    p.wk = 1;
    while (p.wk < (MT > 2 ? 1 : 8) && p.ntiles * slices * p.wk < 256 * 8) p.wk *= 2;
    const int red = p.wk > 1 ? 2 * W * MT * 64 * NI * 4 : 0;
    const int fit = (MM_LDS - red) / (MT * R::BYTES) / MM_U<TYPE> * MM_U<TYPE>;
    p.chunks = (p.nsets + fit - 1) / fit;
    p.cs = (p.nsets + p.chunks - 1) / p.chunks;
    p.cs = (p.cs + MM_U<TYPE> - 1) / MM_U<TYPE> * MM_U<TYPE>;
    p.chunks = (p.nsets + p.cs - 1) / p.cs;
    const int lds = MT * p.cs * R::BYTES + red;
    const int wn = W / p.wk;
    // work-groups of a slice: one a CU, which then makes or copies the operands once,
    // and none more (2048 x 2048 Q4_0, 700 rows: 24 a slice 49 us, 23 36; 160: 17.9, 15.0).
    // A slice's share is a whole number: of long batches it leaves up to half the CUs
    // idle (8192 x 2048 Q4_0: 8192 rows, 128 slices of two, 575 us; 8193, 129 of one, 1082)
    const int64_t want = slices < 256 ? 256 / slices : 1;
    const int64_t most = (p.ntiles + wn - 1) / wn;
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)slices), block(64 * W);
    hipLaunchKernelGGL((k_mm<TYPE, MT, NI>), grid, block, lds, st, g, p);
    return hip_check_launch();
}

template <int TYPE>
static int mm_launch(const MmArgs &g, hipStream_t st) {
    using R = MmRec<TYPE>;
    if (mv_ok<TYPE>(g)) {
        if (g.T == 1) return mv_launch<TYPE, 1>(g, st);
        if (g.T == 2) return mv_launch<TYPE, 2>(g, st);
        if (g.T == 3) return mv_launch<TYPE, 3>(g, st);
        if (g.T == 4) return mv_launch<TYPE, 4>(g, st);
        if (g.T == 5) return mv_launch<TYPE, 5>(g, st);
        if (g.T == 6) return mv_launch<TYPE, 6>(g, st);
        if (g.T == 7) return mv_launch<TYPE, 7>(g, st);
        return mv_launch<TYPE, 8>(g, st);
    }
    MmPlan p = {};
    p.nsets = (int)((g.K + R::VALUES - 1) / R::VALUES);
    p.ntiles = (int)((g.N + 15) / 16);
    p.src = g.btype != 0 ? 2 : 1;
    if (g.T >= MM_PREP_T && mm_ws_bytes(g.type, g.T, g.K) <= g.ws_bytes) {
        const dim3 grid((unsigned)((p.nsets * (R::VALUES / 8) + 255) / 256), (unsigned)g.T);
        hipLaunchKernelGGL((g.btype == 0 ? k_mm_rows<TYPE, 1> : k_mm_rows<TYPE, 2>), grid, dim3(256), 0, st, (const uint8_t *)g.b, g.ldb,
                           g.T, (int)g.K, p.nsets, (uint8_t *)g.ws);
        const int rc = hip_check_launch();
        if (rc) return rc;
        p.src = 0;
    } else if (g.T >= MM_PREP_T && g.btype == 0) {
        return -4;   // (mi_mul_mat looks before: no such call comes here)
    }
    // (by rows alone, not by b's type: a plan's order of sums is the same for both)
    if (g.T <= 4) return mm_go<TYPE, 1, 1>(g, p, st);
    if (g.T < MM_PREP_T) return mm_go<TYPE, 1, 2>(g, p, st);
    // 16 tokens of a work-group also while one round of the CUs takes all tiles (64
    // rows: 1024 x 8192 Q4_0 14.5 us against 18.3 with 32 tokens, 512 x 4096 10.5 and 12.6)
    if (g.T <= 16 || p.ntiles * ((g.T + 15) / 16) <= 256) return mm_go<TYPE, 1, 4>(g, p, st);
    // 32 tokens of a work-group until 64 leave three waves for every two SIMDs (8192
    // x 2048 Q4_K: 128 rows 16.7 us against 18.4 with 64, 200 rows 31.8 against 19.5)
    if (g.T <= 32 || p.ntiles * ((g.T + 63) / 64) < 1536) return mm_go<TYPE, 2, 4>(g, p, st);
    return mm_go<TYPE, 4, 4>(g, p, st);
}

int launch_mm(const MmArgs &g, hipStream_t st) {
    for (int64_t t = 0; t < g.T; t += MM_PASS_T) {
        MmArgs a = g;
        a.b = (const uint8_t *)g.b + t * g.ldb;
        a.y = g.y + t * g.ldy;
        a.T = g.T - t < MM_PASS_T ? g.T - t : MM_PASS_T;
        const int rc = g.type == 2 ? mm_launch<2>(a, st) : mm_launch<12>(a, st);
        if (rc) return rc;
    }
    return 0;
}

}  // namespace mimoe
