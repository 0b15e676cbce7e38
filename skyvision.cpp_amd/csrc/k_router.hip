// k_router.hip - routing to experts on given logits (mi_moe_route,
// mi_moe_forward_router): scores, a bias for the choice, groups of experts of
// which the best are kept, top-k, renormalized weights.
//
//   s = fl32(1 / (1 + exp(-l))) or the softmax over all E as ggml_soft_max
//   (e = fl32(exp(fl32(l - max))), p = e * fl32(1 / sum)), every exp in fp64;
//   c = s + bias; a group's value: the sum of its 1 or 2 largest c; the best
//   groups stay; K rounds of the largest c left, lowest id on ties;
//   w = s [/ (fl32(sum of the K in fp64, slot order) + eps)] * scaling [* scale].
// Values that are no numbers never win (NaN; experts of groups that are out and
// lanes past E are NaN too); slots left take the lowest ids and the weight NaN.
#include "common.hpp"
#include "launch.hpp"
#include "wave_ops.hpp"

namespace mimoe {

// One wave per token, lane l holding the experts 64 i + l.
template <int NPER>
__global__ void __launch_bounds__(256) k_route(const float *__restrict__ logits, int64_t ldl, int64_t T, int E, int K,
                                               RouterParams p, int32_t *__restrict__ sel, float *__restrict__ w) {
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T) return;   // whole waves
    const float *l = logits + t * ldl;
    const float NaN = __builtin_nanf("");
    float s[NPER], c[NPER];
#pragma unroll
    for (int i = 0; i < NPER; ++i) s[i] = lane + 64 * i < E ? l[lane + 64 * i] : -INFINITY;
    if (p.score == 1) {
#pragma unroll
        for (int i = 0; i < NPER; ++i) s[i] = gating_sigmoid(s[i]);
    } else {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < NPER; ++i) mx = fmaxf(mx, s[i]);
        mx = wave_max(mx);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NPER; ++i) {
            s[i] = lane + 64 * i < E ? (float)exp((double)(s[i] - mx)) : 0.f;
            sum += (double)s[i];
        }
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        const float inv = (float)(1.0 / sum);
#pragma unroll
        for (int i = 0; i < NPER; ++i) s[i] = s[i] * inv;
    }
#pragma unroll
    for (int i = 0; i < NPER; ++i) {
        const int e = lane + 64 * i;
        c[i] = e >= E ? NaN : p.sel_bias ? s[i] + p.sel_bias[e] : s[i];
    }
    if (p.n_group > 1) {
        const int gs = E / p.n_group;
        float val = NaN;   // lane g: group g's value
        for (int g = 0; g < p.n_group; ++g) {
            // the two largest numbers of the group (NaN: none)
            float a = NaN, b = NaN;
#pragma unroll
            for (int i = 0; i < NPER; ++i) {
                const int e = lane + 64 * i;
                const float v = e >= g * gs && e < (g + 1) * gs ? c[i] : NaN;
                b = fmaxf(b, fminf(a, v) == fminf(a, v) && a == a && v == v ? fminf(a, v) : NaN);
                a = fmaxf(a, v);
            }
            for (int o = 32; o > 0; o >>= 1) {
                const float a2 = __shfl_xor(a, o, 64), b2 = __shfl_xor(b, o, 64);
                const float lo = a == a && a2 == a2 ? fminf(a, a2) : NaN;
                b = fmaxf(fmaxf(b, b2), lo);
                a = fmaxf(a, a2);
            }
            const float v = p.group_top == 1 ? a : a == a ? (b == b ? a + b : -INFINITY) : NaN;
            if (lane == g) val = v;
        }
        // the best n_kept groups (no numbers: behind, lowest first)
        unsigned long long kept = 0;
        for (int r = 0; r < p.n_kept; ++r) {
            const float m = wave_max_uniform(val);
            unsigned long long b = __ballot(val == m && !(kept >> lane & 1));
            if (b == 0) b = __ballot(lane < p.n_group && !(kept >> lane & 1));
            const int g = (int)__builtin_ctzll(b);
            kept |= 1ull << g;
            if (lane == g) val = NaN;
        }
#pragma unroll
        for (int i = 0; i < NPER; ++i)
            if (lane + 64 * i < E && !(kept >> ((lane + 64 * i) / gs) & 1)) c[i] = NaN;
    }
    int mysel = -1;
    float mys = NaN;   // lane k: the k-th expert's score
    for (int r = 0; r < K; ++r) {
        float m = c[0];
#pragma unroll
        for (int i = 1; i < NPER; ++i) m = fmaxf(m, c[i]);
        m = wave_max_uniform(m);
        int e = -1;
#pragma unroll
        for (int i = 0; i < NPER; ++i) {
            const unsigned long long b = __ballot(c[i] == m);
            if (e < 0 && b != 0ull) e = 64 * i + (int)__builtin_ctzll(b);
        }
        if (e < 0) break;   // (uniform) no number left
        float sv = 0.f;
#pragma unroll
        for (int i = 0; i < NPER; ++i) {
            if (e == 64 * i + lane) c[i] = NaN;
            const float x = lane_f(s[i], e & 63);
            if (i == (e >> 6)) sv = x;
        }
        if (lane == r) {
            mysel = e;
            mys = sv;
        }
    }
    const unsigned long long none = __ballot(lane < K && mysel < 0);
    if (none) {
        for (int r = (int)__builtin_ctzll(none); r < K; ++r) {
            int e = 0;
            while (__ballot(lane < r && mysel == e)) ++e;   // (r < K <= E ids are taken)
            if (lane == r) mysel = e;
        }
    }
    float v = lane < K ? mys : 0.f;
    if (p.renorm) {
        double sum = 0.0;
        for (int k = 0; k < K; ++k) sum = sum + (double)lane_f(v, k);
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
    if ((T + 3) / 4 > 0x7fffffff) return -6;
    const dim3 grid((unsigned)((T + 3) / 4)), block(256);
#define ROUTE(N) hipLaunchKernelGGL(k_route<N>, grid, block, 0, st, logits, ldl, T, E, K, p, sel, w)
    if (E <= 64) ROUTE(1);
    else if (E <= 128) ROUTE(2);
    else if (E <= 256) ROUTE(4);
    else if (E <= 512) ROUTE(8);
    else ROUTE(16);
#undef ROUTE
    return hip_check_launch();
}

}  // namespace mimoe
