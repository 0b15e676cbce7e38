// k_router.hip - routing to experts on given logits (mi_moe_route,
// mi_moe_forward_router): scores, a bias for the choice, groups of experts of
// which the best are kept, top-k, renormalized weights.
//
//   s = fl32(1 / (1 + exp(-l))) or the softmax over all E as ggml_soft_max
//   (e = fl32(exp(fl32(l - max))), p = e * fl32(1 / sum)), every exp and sum in fp64
//   (the sum over the lanes, not in expert order);
//   c = s + bias; a group's value: the sum of its 1 or 2 largest c; the best
//   groups stay; K rounds of the largest c left, lowest id on ties;
//   w = s [/ (fl32(sum of the K in fp64, slot order) + eps)] * scaling [* scale].
// Values that are no numbers never win (NaN; experts of groups that are out and
// lanes past E are NaN too); slots left take the lowest ids and the weight NaN.
#include "common.hpp"
#include "lanes.hpp"
#include "launch.hpp"
#include "wave_ops.hpp"

namespace mimoe {

// A float's place among all others as an integer; NaN (and what is out of the
// race) below every number.  + 0: -0 is 0.
constexpr int KEY_NONE = (int)0x80000000;
__device__ __forceinline__ int key_of(float c) {
    const int b = __builtin_bit_cast(int, c + 0.f);
    return c == c ? b ^ ((b >> 31) & 0x7fffffff) : KEY_NONE;
}
__device__ __forceinline__ float value_of(int k) { return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff)); }

// exp(x) for |x| <= 700 in fp64, off by at most 1.4e-16 of the value (30 million
// values between): n = rint(x log2 e), the Taylor series of exp(x - n ln 2) to the
// 13th power (|.| <= ln 2 / 2: the next term is below 2^-57), times 2^n.  ln 2 in two
// parts (Cody and Waite's reduction): to a multiple of 2^-42, n times which is
// exact, and the rest
__device__ __forceinline__ double exp_f64(double x) {
    const double n = __builtin_rint(x * 1.4426950408889634074);
    const double r = fma(-n, 0x1.ef35793c7673p-45, fma(-n, 0x1.62e42fefa38p-1, x));
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)n);
}
// 1 / x, x from 1 to 2^1011: the hardware's estimate and two Newton steps
__device__ __forceinline__ double rcp_f64(double x) {
    double r = __builtin_amdgcn_rcp(x);
    r = fma(fma(-x, r, 1.0), r, r);
    return fma(fma(-x, r, 1.0), r, r);
}
// x held to +-700, NaN kept
__device__ __forceinline__ double held700(float x) {
    x = x < -700.f ? -700.f : x;
    return (double)(x > 700.f ? 700.f : x);
}
// fl32(1 / (1 + exp(-x))); past +-700 the result is 0 or 1 in 32 bits
__device__ __forceinline__ float sigmoid_f32(float x) { return (float)rcp_f64(1.0 + exp_f64(-held700(x))); }
// fl32(exp(x)), x <= 0 (or NaN)
__device__ __forceinline__ float exp_f32(float x) { return (float)exp_f64(held700(x)); }

// the wave's largest, uniform
__device__ __forceinline__ int wave_max_i(int m) {
    int o = dpp_i<0xB1>(m);
    m = o > m ? o : m;
    o = dpp_i<0x4E>(m);
    m = o > m ? o : m;
    o = dpp_i<0x141>(m);
    m = o > m ? o : m;
    o = dpp_i<0x140>(m);
    m = o > m ? o : m;
    // (the smallest where no lane reads: the move and the comparison are one instruction)
    o = __builtin_amdgcn_update_dpp(KEY_NONE, m, 0x142, 0xA, 0xF, false);   // rows 0 -> 1, 2 -> 3
    m = o > m ? o : m;
    o = __builtin_amdgcn_update_dpp(KEY_NONE, m, 0x143, 0xC, 0xF, false);   // row 1 -> 2, 3
    m = o > m ? o : m;
    return __builtin_amdgcn_readlane(m, 63);
}

struct RoutePlan {
    int gs;          // experts of a group
    int magic;       // e / gs = e magic >> 20 for e < 1024
    int ls;          // log2 of the lanes that find a group's value
    int whole;       // a lane's experts are of one group
    int vec;         // rows of whole pieces of NPER
};

constexpr int RT_W = 4;   // waves (tokens) of a work-group

// One wave per token, lane l holding the experts NPER l .. NPER l + NPER - 1 as
// sortable integers; a group's value is found by 2^ls lanes from a copy in LDS
// (groups of any size), the groups' places by counting, the experts by K rounds
// of the wave's largest, each lane offering its best.
// Bound by its vector instructions (some 620 a token of 256 experts, 130 of them
// the sigmoids; issued in 77 % of the CUs' time): 8192 tokens of 256 experts in 8
// groups 12.7 us, of 128 without groups (softmax) 7.6; the bytes alone would take 2.
// One token 4.5 us: the rounds' latency.
template <int NPER>
__global__ void __launch_bounds__(64 * RT_W) k_route(const float *__restrict__ logits, int64_t ldl, int64_t T, int E, int K,
                                                     RouterParams p, RoutePlan q, int32_t *__restrict__ sel, float *__restrict__ w) {
    __shared__ float s_score[RT_W][64 * NPER];
    __shared__ int s_key[RT_W][64 * NPER];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = (int64_t)blockIdx.x * RT_W + wave;
    if (t >= T) return;   // whole waves, each on its own
    const float *l = logits + t * ldl;
    const int e0 = NPER * lane;
    float s[NPER], bias[NPER];
    typedef float fN __attribute__((ext_vector_type(NPER)));
    typedef fN fN_a4 __attribute__((aligned(4)));   // (at any float's address)
#pragma unroll
    for (int i = 0; i < NPER; ++i) s[i] = -INFINITY, bias[i] = 0.f;
    if (q.vec) {
        if (e0 < E) {
            const fN v = *(const fN_a4 *)(l + e0);
#pragma unroll
            for (int i = 0; i < NPER; ++i) s[i] = v[i];
            if (p.sel_bias) {
                const fN b = *(const fN_a4 *)(p.sel_bias + e0);
#pragma unroll
                for (int i = 0; i < NPER; ++i) bias[i] = b[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NPER; ++i)
            if (e0 + i < E) {
                s[i] = l[e0 + i];
                if (p.sel_bias) bias[i] = p.sel_bias[e0 + i];
            }
    }
    if (p.score == 1) {
#pragma unroll
        for (int i = 0; i < NPER; ++i) s[i] = sigmoid_f32(s[i]);
    } else {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < NPER; ++i) mx = fmaxf(mx, s[i]);
        mx = wave_max_uniform(mx);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NPER; ++i) {
            s[i] = exp_f32(s[i] - mx);   // (past E: -inf, 0 unless the whole row is NaN)
            sum += (double)s[i];
        }
        sum = wave_sum_d(sum);
        const float inv = (float)(1.0 / sum);
#pragma unroll
        for (int i = 0; i < NPER; ++i) s[i] = s[i] * inv;
    }
    int k[NPER];
#pragma unroll
    for (int i = 0; i < NPER; ++i) {
        s_score[wave][e0 + i] = s[i];
        k[i] = e0 + i >= E ? KEY_NONE : key_of(p.sel_bias ? s[i] + bias[i] : s[i]);
    }
    if (p.n_group > 1) {
#pragma unroll
        for (int i = 0; i < NPER; ++i) s_key[wave][e0 + i] = k[i];
        wave_lds_sync();
        // the group's two largest, over its 2^ls lanes
        const int S = 1 << q.ls, g = lane >> q.ls;
        int a = KEY_NONE, b = KEY_NONE;
        if (g < p.n_group) {
            const int *gk = &s_key[wave][g * q.gs];
            for (int i = lane & (S - 1); i < q.gs; i += S) {
                const int v = gk[i], lo = v < a ? v : a;
                b = lo > b ? lo : b;
                a = v > a ? v : a;
            }
        }
        for (int o = 1; o < S; o <<= 1) {
            int a2, b2;
            if (o == 1) a2 = dpp_i<0xB1>(a), b2 = dpp_i<0xB1>(b);
            else if (o == 2) a2 = dpp_i<0x4E>(a), b2 = dpp_i<0x4E>(b);
            else if (o == 4) a2 = dpp_i<0x141>(a), b2 = dpp_i<0x141>(b);
            else if (o == 8) a2 = dpp_i<0x140>(a), b2 = dpp_i<0x140>(b);
            else a2 = __shfl_xor(a, o, 64), b2 = __shfl_xor(b, o, 64);
            const int lo = a < a2 ? a : a2;
            b = b > b2 ? b : b2;
            b = lo > b ? lo : b;
            a = a > a2 ? a : a2;
        }
        int val = p.group_top == 1 || a == KEY_NONE ? a
                  : key_of(b == KEY_NONE ? -INFINITY : value_of(a) + value_of(b));
        // a group's place: those before it, larger, or equal and lower (larger than
        // the integer below; no number: still above the smallest integer)
        val = val > KEY_NONE ? val : KEY_NONE + 1;
        int before = 0;
        for (int o = 0; o < p.n_group; ++o)
            before += __builtin_amdgcn_readlane(val, o << q.ls) > (o < g ? val - 1 : val) ? 1 : 0;
        const unsigned long long kept = __ballot(g < p.n_group && before < p.n_kept);
        bool in = true;
#pragma unroll
        for (int i = 0; i < NPER; ++i) {
            if (i == 0 || !q.whole) {   // (uniform)
                const uint32_t ge = __umul24((uint32_t)(e0 + i), (uint32_t)q.magic) >> 20;
                in = (kept >> ((ge << q.ls) & 63)) & 1;
            }
            k[i] = in ? k[i] : KEY_NONE;
        }
    }
    // each lane's experts, best first (neighbours change places only for a larger
    // one: equal ones stay in order); up to four: their numbers in the lane as the
    // bytes of a word
    uint32_t ord = 0;
    if constexpr (NPER <= 4) {
        int id[NPER];
#pragma unroll
        for (int i = 0; i < NPER; ++i) id[i] = i;
#pragma unroll
        for (int n = NPER - 1; n > 0; --n)
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const bool sw = k[i + 1] > k[i];
                const int kh = sw ? k[i + 1] : k[i], kl = sw ? k[i] : k[i + 1];
                const int ih = sw ? id[i + 1] : id[i], il = sw ? id[i] : id[i + 1];
                k[i] = kh; k[i + 1] = kl;
                id[i] = ih; id[i + 1] = il;
            }
#pragma unroll
        for (int i = 0; i < NPER; ++i) ord |= (uint32_t)id[i] << (8 * i);
    }
    int mysel = -1;
    for (int r = 0; r < K; ++r) {
        int best = k[0], at = (int)ord;   // (up to four: the lane's best is the lowest byte)
        if constexpr (NPER > 4) {
            at = 0;
#pragma unroll
            for (int i = 1; i < NPER; ++i) {
                const bool up = k[i] > best;
                best = up ? k[i] : best;
                at = up ? i : at;
            }
        }
        const int m = wave_max_i(best);
        if (m == KEY_NONE) break;   // (uniform) no number left
        const int win = (int)__builtin_ctzll(__ballot(best == m));   // lanes hold ascending ids
        const int e = NPER * win + (__builtin_amdgcn_readlane(at, win) & 0xff);
        mysel = lane == r ? e : mysel;
        if constexpr (NPER <= 4) {
            const bool mine = lane == win;
            ord = mine ? ord >> 8 : ord;
#pragma unroll
            for (int i = 0; i + 1 < NPER; ++i) k[i] = mine ? k[i + 1] : k[i];
            k[NPER - 1] = mine ? KEY_NONE : k[NPER - 1];
        } else {
#pragma unroll
            for (int i = 0; i < NPER; ++i) k[i] = e0 + i == e ? KEY_NONE : k[i];
        }
    }
    wave_lds_sync();
    float v = lane < K ? (mysel < 0 ? __builtin_nanf("") : s_score[wave][mysel]) : 0.f;
    const unsigned long long none = __ballot(lane < K && mysel < 0);
    if (none) {
        for (int r = (int)__builtin_ctzll(none); r < K; ++r) {
            int e = 0;
            while (__ballot(lane < r && mysel == e)) ++e;   // (r < K <= E ids are taken)
            if (lane == r) mysel = e;
        }
    }
    if (p.renorm) {
        double sum = 0.0;
        for (int j = 0; j < K; ++j) sum = sum + (double)lane_f(v, j);
        v = v / ((float)sum + p.eps);
    }
    v = v * p.scaling;
    if (lane < K) {
        if (p.expert_scale) v = v * p.expert_scale[mysel];
        sel[t * K + lane] = mysel;
        w[t * K + lane] = v;
    }
}

int launch_route(const float *logits, int64_t ldl, int64_t T, int E, int K, const RouterParams &p, int32_t *sel,
                 float *w, hipStream_t st) {
    if (T <= 0) return 0;
    if (E <= 0 || E > ROUTER_MAX_E || K <= 0 || K > ROUTER_MAX_K || K > E) return -6;
    if (p.n_group < 1 || p.n_group > ROUTER_MAX_GROUPS || E % p.n_group || p.n_kept < 1 || p.n_kept > p.n_group) return -6;
    const int nper = E <= 64 ? 1 : E <= 128 ? 2 : E <= 256 ? 4 : E <= 512 ? 8 : 16;
    RoutePlan q;
    q.gs = E / p.n_group;
    q.magic = ((1 << 20) + q.gs - 1) / q.gs;   // e (magic gs - 2^20) < 1024 * 512 < 2^20: exact
    q.whole = q.gs % nper == 0;
    q.ls = 0;
    while (p.n_group << (q.ls + 1) <= 64) ++q.ls;
    q.vec = E % nper == 0;
    constexpr int64_t PASS = 1 << 24;   // tokens of a launch (it covers fewer than 2^32 threads)
    for (int64_t t = 0; t < T; t += PASS) {
        const int64_t n = T - t < PASS ? T - t : PASS;
        const dim3 grid((unsigned)((n + RT_W - 1) / RT_W)), block(64 * RT_W);
#define ROUTE(N) hipLaunchKernelGGL(k_route<N>, grid, block, 0, st, logits + t * ldl, ldl, n, E, K, p, q, sel + t * K, w + t * K)
        if (nper == 1) ROUTE(1);
        else if (nper == 2) ROUTE(2);
        else if (nper == 4) ROUTE(4);
        else if (nper == 8) ROUTE(8);
        else ROUTE(16);
#undef ROUTE
        const int rc = hip_check_launch();
        if (rc) return rc;
    }
    return 0;
}

}  // namespace mimoe
