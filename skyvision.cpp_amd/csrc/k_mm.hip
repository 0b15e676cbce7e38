// k_mm.hip - dense products of 4-bit matrices and rows in 8 bits (mi_mul_mat):
//   y[t][n] = sum over blocks of (a's block . b's block), b in a's 8-bit form.
//   Q4_0 . Q8_0: d_a d_b sum (q - 8) c                                      (32 values)
//   Q4_K . Q8_K: d_b (d sum_j sc_j sum_j q c - dmin sum_j m_j sum_j c)     (256, j: 32 values)
// The sums over codes are exact integers, the blocks are added in fp32.
//
// The codes' products run on v_mfma_i32_16x16x32_i8, whose 32 products are one
// 32-value block: 16 tokens x 16 rows of the matrix, one group of 16 lanes per
// quarter of the block.  A lane holds a row's codes straight from the table's
// bytes; the tokens' operands lie in LDS in the lanes' order (MM records) for
// the whole K, written once per work-group, which then walks over row tiles:
// the matrix is read once and nothing else is.
#include "b32.hpp"
#include "common.hpp"
#include "launch.hpp"
#include "wave_ops.hpp"

namespace mimoe {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));

constexpr int MM_W = 8;                // waves of a work-group
constexpr int MM_THREADS = 64 * MM_W;
constexpr int MM_LDS = 160 * 1024;

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

__device__ __forceinline__ bool mm_bad8(const float (&v)[8]) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) bad |= !(fabsf(v[j]) <= 3.402823466e38f);
    return bad;
}
__device__ __forceinline__ uint2 mm_pack8(const int (&q)[8]) {
    uint32_t c[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j >> 2] |= (uint32_t)(q[j] & 0xff) << (8 * (j & 3));
    return make_uint2(c[0], c[1]);
}

// piece p (8 values of token row m of the tile) of the tile's operands into its
// record at o: Q4_0: block p / 4, quarter p % 4; Q4_K: values 8 p ..  The lanes
// that share a block's largest value (4 or 32, aligned) call it together.
// SRC 1: row of fp32 values; 2: of 8-bit blocks.  live: the piece is in the row.
template <int TYPE, int SRC>
__device__ __forceinline__ void mm_piece(const uint8_t *row, int p, int m, bool vec, bool live, uint8_t *o) {
    if constexpr (TYPE == 2) {
        const int blk = p >> 2, g = p & 3;
        uint2 c = make_uint2(0u, 0u);
        float d = 0.f;
        if constexpr (SRC == 1) {
            float v[8];
            const float *x = (const float *)row + 32 * blk + 4 * g;
            if (live) {
                if (vec) {
                    const float4 a = *(const float4 *)x, b = *(const float4 *)(x + 16);
                    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = x[(j & 3) + 16 * (j >> 2)];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = 0.f;
            }
            int bad = mm_bad8(v);
            bad |= dpp_i<0xB1>(bad);
            bad |= dpp_i<0x4E>(bad);
            int q[8];
            uint32_t dh;
            b32_q8_codes(v, q, dh);
            c = mm_pack8(q);
            d = h2f((uint16_t)dh);
            if (bad || !(d <= 65504.f)) d = __builtin_nanf("");
        } else if (live) {
            const uint8_t *b = row + 34 * blk;
            c.x = *(const u32_a2 *)(b + 2 + 4 * g);
            c.y = *(const u32_a2 *)(b + 18 + 4 * g);
            d = h2f(*(const uint16_t *)b);
            if (!(fabsf(d) <= 65504.f)) d = __builtin_nanf("");
        }
        const int j = blk & 3;
        *(uint2 *)(o + 16 * (64 * (j >> 1) + 16 * g + m) + 8 * (j & 1)) = c;
        if (g == 0) *(float *)(o + 2048 + 64 * j + 4 * m) = d * 0.0625f;
    } else {
        const int e = p & 31, j = e >> 2, g = e & 3;   // sub-block and quarter
        uint2 c = make_uint2(0u, 0u);
        float d = 0.f;
        if constexpr (SRC == 1) {
            float v[8];
            const float *x = (const float *)row + 8 * p;
            if (live) {
                if (vec) {
                    const float4 a = *(const float4 *)x, b = *(const float4 *)(x + 4);
                    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = x[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.f;
            }
            const unsigned long long bb = __ballot(mm_bad8(v));
            const bool bad = (uint32_t)(threadIdx.x & 32 ? bb >> 32 : bb) != 0u;
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) t = fmaxf(t, fabsf(v[i]));
            t = fmaxf(t, dpp_f<0xB1>(t));
            t = fmaxf(t, dpp_f<0x4E>(t));
            t = fmaxf(t, dpp_f<0x141>(t));
            t = fmaxf(t, dpp_f<0x140>(t));
            t = fmaxf(t, __shfl_xor(t, 16, 64));
            // d and the codes change sign together with the sign ggml gives them
            // (of the first largest |x|): their products are the same
            const bool zero = t == 0.f;
            const float is = zero ? 0.f : 127.f / t;
            d = zero ? 0.f : 1 / is;
            int q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = bad || zero ? 0 : (int)__builtin_rintf(is * v[i]);
            if (bad) d = __builtin_nanf("");
            c = mm_pack8(q);
        } else if (live) {
            const uint8_t *b = row + 292 * (p >> 5);
            c = make_uint2(*(const uint32_t *)(b + 4 + 8 * e), *(const uint32_t *)(b + 8 + 8 * e));
            d = *(const float *)b;
            if (!(fabsf(d) <= 3.402823466e38f)) d = __builtin_nanf("");
        }
        *(uint2 *)(o + 16 * (64 * (j >> 1) + 16 * g + m) + 8 * (j & 1)) = c;
        int s = __builtin_amdgcn_sdot4(0x01010101, (int)c.x, __builtin_amdgcn_sdot4(0x01010101, (int)c.y, 0, false), false);
        s += dpp_i<0xB1>(s);
        // sum of values 16 (e / 2) ..: lane quarter e / 8, slot e / 2 % 4
        if (!(e & 1)) *(_Float16 *)(o + 4096 + 8 * (16 * (e >> 3) + m) + 2 * ((e >> 1) & 3)) = (_Float16)s;
        if (e == 0) *(float *)(o + 4608 + 4 * m) = d;
    }
}

// records of a call's rows: ws + ((tile of 16 tokens) * nsets + set) * BYTES
template <int TYPE>
__global__ void __launch_bounds__(256) k_mm_rows(const uint8_t *b, int64_t ldb, int64_t T, int K, int nsets, int vec, uint8_t *ws) {
    using R = MmRec<TYPE>;
    const int64_t t = blockIdx.y;
    const int p = blockIdx.x * 256 + threadIdx.x, set = p / (R::VALUES / 8);
    if (set >= nsets) return;   // whole waves (64 pieces: whole sets)
    mm_piece<TYPE, 1>(b + t * ldb, p, (int)(t & 15), vec, 8 * p < K, ws + ((t >> 4) * nsets + set) * R::BYTES);
}

struct MmPlan {
    int src;       // operands: 0 records at ws, 1 fp32 rows, 2 rows in 8 bits
    int vec;       // fp32 rows 16-byte aligned
    int nsets;     // sets of a row
    int chunks, cs;  // chunks of cs sets whose operands lie in LDS at a time
    int wk;        // waves that share a row tile, each taking every wk-th set
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

__device__ __forceinline__ long mm_u64(uint32_t lo, uint32_t hi) { return (long)(((uint64_t)hi << 32) | lo); }
__device__ __forceinline__ void swap16(uint32_t &a, uint32_t &b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void swap32(uint32_t &a, uint32_t &b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// acc[mt] += the set's part for token tile mt; x: the set's record of tile 0,
// xs: bytes from a tile's record to the next tile's
template <int TYPE, int MT>
__device__ __forceinline__ void mm_set(const MmRaw<TYPE> &r, const uint8_t *x, int xs, int set, int nb, int lane,
                                       float4_t (&acc)[MT]) {
    const int g = lane >> 4;
    const i32x4 z = {0, 0, 0, 0};
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
        u32x4 xc[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            xc[m][0] = *(const u32x4 *)(x + m * xs + 16 * lane);
            xc[m][1] = *(const u32x4 *)(x + m * xs + 1024 + 16 * lane);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float da = h2f((uint16_t)d[j]);
            // 16 (q - 8) as signed bytes: the nibble on top, its highest bit turned
            const uint32_t lo = ((w[j] << 4) & 0xF0F0F0F0u) ^ 0x80808080u, hi = (w[j] & 0xF0F0F0F0u) ^ 0x80808080u;
            const long wb = mm_u64(lo, hi);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const u32x4 xv = xc[m][j >> 1];
                const long xa = j & 1 ? mm_u64(xv.z, xv.w) : mm_u64(xv.x, xv.y);
                const i32x4 c = __builtin_amdgcn_mfma_i32_16x16x32_i8(xa, wb, z, 0, 0, 0);
                const float4_t db = *(const float4_t *)(x + m * xs + 2048 + 64 * j + 16 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][i] = fmaf((float)c[i], da * db[i], acc[m][i]);
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
        i32x4 s[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) s[m] = z;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const long lo = mm_u64(r.q[c].x & 0x0F0F0F0Fu, r.q[c].y & 0x0F0F0F0Fu);
            const long hi = mm_u64((r.q[c].x >> 4) & 0x0F0F0F0Fu, (r.q[c].y >> 4) & 0x0F0F0F0Fu);
            const int s0 = (int)((sc[c >> 1] >> (16 * (c & 1))) & 0xffu), s1 = (int)((sc[c >> 1] >> (16 * (c & 1) + 8)) & 0xffu);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const u32x4 xv = *(const u32x4 *)(x + m * xs + 1024 * c + 16 * lane);
                const i32x4 a = __builtin_amdgcn_mfma_i32_16x16x32_i8(mm_u64(xv.x, xv.y), lo, z, 0, 0, 0);
                const i32x4 b = __builtin_amdgcn_mfma_i32_16x16x32_i8(mm_u64(xv.z, xv.w), hi, z, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[m][i] += __mul24(a[i], s0) + __mul24(b[i], s1);
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const half4_t bs = *(const half4_t *)(x + m * xs + 4096 + 8 * lane);
            const float4_t zf = {0.f, 0.f, 0.f, 0.f};
            const float4_t mm = __builtin_amdgcn_mfma_f32_16x16x16f16(bs, mb, zf, 0, 0, 0);
            const float4_t db = *(const float4_t *)(x + m * xs + 4608 + 16 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(fmaf(d, (float)s[m][i], -(dm * mm[i])), db[i], acc[m][i]);
        }
    }
}

// Work-group (x, y): tokens 16 MT y .., row tiles x (W / wk), + gridDim.x (W / wk) ..
template <int TYPE, int MT>
__global__ void __launch_bounds__(MM_THREADS) k_mm(MmArgs g, MmPlan p) {
    using R = MmRec<TYPE>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wk = p.wk, wn = MM_W / wk, kw = wave % wk, nw = wave / wk;
    const int64_t t0 = (int64_t)blockIdx.y * 16 * MT;
    const int nt = (int)(g.T - t0 < 16 * MT ? g.T - t0 : 16 * MT);   // tokens here
    const int nb = (int)(g.K / 32);
    const int xs = p.cs * R::BYTES;   // a token tile's records in LDS
    float4_t *red = (float4_t *)(lds + MT * xs);   // [2][W][MT][64]

    // the operands of chunk ch
    auto fill = [&](int ch) __attribute__((always_inline)) {
        const int s0 = ch * p.cs, ns = imin(p.cs, p.nsets - s0);
        if (p.src == 0) {
            const int per = ns * (R::BYTES / 16);
            for (int m = 0; m < MT && 16 * m < nt; ++m) {
                const u32x4 *src = (const u32x4 *)((const uint8_t *)g.ws + ((t0 / 16 + m) * p.nsets + s0) * R::BYTES);
                u32x4 *dst = (u32x4 *)(lds + m * xs);
                for (int i = tid; i < per; i += MM_THREADS) dst[i] = src[i];
            }
        } else {
            // pieces of 8 values; a wave's 64 pieces are of one token
            constexpr int PS = R::VALUES / 8;   // pieces of a set: 16 or 32
            const int pt = (ns * PS + 63) & ~63;   // of a token, rounded up to whole waves
            for (int i = tid; i < pt * nt; i += MM_THREADS) {
                const int t = i / pt, q = i - t * pt, set = q / PS, pc = s0 * PS + q;
                if (set >= ns) continue;   // (whole groups of lanes that share a block)
                const uint8_t *row = (const uint8_t *)g.b + (t0 + t) * g.ldb;
                uint8_t *o = lds + (t >> 4) * xs + set * R::BYTES;
                if (p.src == 1) mm_piece<TYPE, 1>(row, pc, t & 15, p.vec, 8 * pc < g.K, o);
                else mm_piece<TYPE, 2>(row, pc, t & 15, false, 8 * pc < g.K, o);
            }
        }
    };

    const int spc = (p.cs + wk - 1) / wk;              // steps of a chunk
    const int spt = spc * p.chunks;                    // of a row tile
    const int stride = (int)gridDim.x * wn;
    const int first = (int)blockIdx.x * wn;            // the work-group's first tile
    const int iters = (p.ntiles - first + stride - 1) / stride;
    const int total = iters * spt;

    auto step_of = [&](int st, int &tile, int &set) __attribute__((always_inline)) {
        const int it = st / spt, s = st - it * spt, ch = s / spc;
        tile = first + nw + it * stride;
        set = ch * p.cs + (s - ch * spc) * wk + kw;
        if ((s - ch * spc) * wk + kw >= p.cs || tile >= p.ntiles) set = p.nsets;   // nothing here
    };
    auto load = [&](MmRaw<TYPE> &r, int st) __attribute__((always_inline)) {
        int tile, set;
        step_of(st, tile, set);
        // (clamped: a step that holds nothing loads some row's set and drops it)
        const int64_t n = 16 * (int64_t)imin(tile, p.ntiles - 1) + (lane & 15);
        mm_load<TYPE>(r, g.a + (n < g.N ? n : g.N - 1) * g.row_bytes, imin(set, p.nsets - 1), nb, lane >> 4);
    };

    float4_t acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = {0.f, 0.f, 0.f, 0.f};
    MmRaw<TYPE> cur, nxt;
    load(cur, 0);
    if (p.chunks == 1) {
        fill(0);
        __syncthreads();
    }
    for (int st = 0; st < total; ++st) {
        if (st + 1 < total) load(nxt, st + 1);
        const int it = st / spt, s = st - it * spt, ch = s / spc;
        if (p.chunks > 1 && s == ch * spc) {
            __syncthreads();
            fill(ch);
            __syncthreads();
        }
        int tile, set;
        step_of(st, tile, set);
        if (set < p.nsets) mm_set<TYPE, MT>(cur, lds + (set - ch * p.cs) * R::BYTES, xs, set, nb, lane, acc);
        if (s == spt - 1) {
            const int n = 16 * tile + (lane & 15);
            if (wk == 1) {
                if (tile < p.ntiles && n < g.N) {
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int t = 16 * m + 4 * (lane >> 4) + i;
                            if (t < nt) g.y[(t0 + t) * g.ldy + n] = acc[m][i];
                        }
                }
            } else {
                // the tile's parts, one buffer per parity: a wave that is through
                // with this one is past the barrier after its last use
                float4_t *rb = red + (it & 1) * MM_W * MT * 64;
#pragma unroll
                for (int m = 0; m < MT; ++m) rb[(wave * MT + m) * 64 + lane] = acc[m];
                __syncthreads();
                const float *rf = (const float *)rb;
                for (int e = tid; e < wn * MT * 256; e += MM_THREADS) {
                    const int i = e & 3, l = (e >> 2) & 63, m = (e >> 8) % MT, w = (e >> 8) / MT;
                    const int t = 16 * m + 4 * (l >> 4) + i, tl = first + w + it * stride;
                    const int64_t nn = 16 * (int64_t)tl + (l & 15);
                    if (t >= nt || tl >= p.ntiles || nn >= g.N) continue;
                    float v = rf[((w * wk) * MT + m) * 256 + 4 * l + i];
                    for (int k = 1; k < wk; ++k) v += rf[((w * wk + k) * MT + m) * 256 + 4 * l + i];
                    g.y[(t0 + t) * g.ldy + nn] = v;
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = {0.f, 0.f, 0.f, 0.f};
        }
        cur = nxt;
    }
}

constexpr int64_t MM_PREP_T = 8;   // fp32 rows from so many on: their records in a launch of their own

size_t mm_ws_bytes(int type, int btype, int64_t T, int64_t K) {
    if (btype != 0 || T < MM_PREP_T) return 0;
    return type == 2 ? (size_t)((T + 15) / 16 * ((K + 127) / 128) * MmRec<2>::BYTES)
                     : (size_t)((T + 15) / 16 * (K / 256) * MmRec<12>::BYTES);
}

template <int TYPE>
static int mm_launch(const MmArgs &g, hipStream_t st) {
    using R = MmRec<TYPE>;
    MmPlan p = {};
    p.nsets = (int)((g.K + R::VALUES - 1) / R::VALUES);
    p.ntiles = (int)((g.N + 15) / 16);
    p.vec = (uintptr_t)g.b % 16 == 0 && g.ldb % 16 == 0;
    p.src = g.btype != 0 ? 2 : 1;
    if (g.btype == 0 && g.T >= MM_PREP_T) {
        const dim3 grid((unsigned)((p.nsets * (R::VALUES / 8) + 255) / 256), (unsigned)g.T);
        hipLaunchKernelGGL(k_mm_rows<TYPE>, grid, dim3(256), 0, st, (const uint8_t *)g.b, g.ldb, g.T, (int)g.K, p.nsets, p.vec, (uint8_t *)g.ws);
        const int rc = hip_check_launch();
        if (rc) return rc;
        p.src = 0;
    }
    const int mt = g.T <= 16 ? 1 : g.T <= 32 ? 2 : 4;
    const int64_t slices = (g.T + 16 * mt - 1) / (16 * mt);
    if (slices > 65535) return -6;
    p.wk = mt == 4 ? 1 : MM_W;
    const int red = p.wk > 1 ? 2 * MM_W * mt * 1024 : 0;
    const int fit = (MM_LDS - red) / (mt * R::BYTES);
    p.chunks = (p.nsets + fit - 1) / fit;
    p.cs = (p.nsets + p.chunks - 1) / p.chunks;
    const int lds = mt * p.cs * R::BYTES + red;
    const int per_cu = imin(4, imax(1, MM_LDS / lds));
    const int wn = MM_W / p.wk;
    const int64_t want = (256 * per_cu + slices - 1) / slices;   // work-groups of a slice
    const int64_t most = (p.ntiles + wn - 1) / wn;
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)slices), block(MM_THREADS);
    if (mt == 1) hipLaunchKernelGGL((k_mm<TYPE, 1>), grid, block, lds, st, g, p);
    else if (mt == 2) hipLaunchKernelGGL((k_mm<TYPE, 2>), grid, block, lds, st, g, p);
    else hipLaunchKernelGGL((k_mm<TYPE, 4>), grid, block, lds, st, g, p);
    return hip_check_launch();
}

int launch_mm(const MmArgs &g, hipStream_t st) {
    if (g.T <= 0) return 0;
    return g.type == 2 ? mm_launch<2>(g, st) : mm_launch<12>(g, st);
}

}  // namespace mimoe
