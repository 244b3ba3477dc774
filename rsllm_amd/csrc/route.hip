// Expert routing: router logits -> the ids and weights of each token's experts.
//
// An expert's place in the order is its key (score + bias), or its logit itself
// where there is no bias (the scores rise with the logits); equal places go to
// the lower id. Which of two near experts is chosen is settled by 64-bit scores,
// and the weights are 64-bit until their one rounding. Keys are looked at in 32
// bits first, with a bound on their error: only what lies closer together than
// that is worked out again.
// Bound by its instructions for many tokens (16384 x 256 bf16, 8 of 4 of 8 groups:
// 17.4 to 18.3 us, 1012 vector instructions a wavefront of two tokens; reading 8.4 MB
// would take 1.3; up to 24 us where a token or two is done over in 64 bits), by the
// launch and one chain of loads, reductions and 64-bit scores for few (1 x 256: 5.7 us).
#include "kernels.h"

#include <type_traits>

namespace rsllm_hip {

namespace {

__device__ __forceinline__ float route_load(const void *p, size_t i, uint32_t dtype) {
    // + 0.0: -0 and 0 are one place in the order
    if (dtype == T_F32) return static_cast<const float *>(p)[i] + 0.0f;
    const uint16_t b = static_cast<const uint16_t *>(p)[i];
    return (dtype == T_F16 ? f16_to_f32(b) : __builtin_bit_cast(float, (uint32_t)b << 16)) + 0.0f;
}

// exp(x) to some 2^-52: x = n log 2 + r, |r| < 0.35, and the power series of exp(r)
// up to r^12 / 12!, after Cody and Waite's reduction. (Short, where the library's
// is long: most calls of these kernels pay for fetching their code.)
__device__ __forceinline__ double route_exp64(double x) {
    x = fmin(fmax(x, -1000.0), 1000.0);
    const double n = rint(x * 0x1.71547652b82fep+0);  // log2 e
    // log 2 in two parts, the first of few enough bits that n times it is exact
    const double r = fma(n, -0x1.7f7d1cf79abcap-20, fma(n, -0x1.62e4p-1, x));
    double p = 1.0 / 479001600.0;
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
    return ldexp(p, (int)n);
}
// log(1 + e), 0 <= e <= 1: 2 atanh(z), z = e / (2 + e) <= 1/3, to z^33.
__device__ __forceinline__ double route_log1p(double e) {
    const double z = e / (2.0 + e), q = z * z;
    double p = 2.0 / 33.0;
    p = fma(p, q, 2.0 / 31.0);
    p = fma(p, q, 2.0 / 29.0);
    p = fma(p, q, 2.0 / 27.0);
    p = fma(p, q, 2.0 / 25.0);
    p = fma(p, q, 2.0 / 23.0);
    p = fma(p, q, 2.0 / 21.0);
    p = fma(p, q, 2.0 / 19.0);
    p = fma(p, q, 2.0 / 17.0);
    p = fma(p, q, 2.0 / 15.0);
    p = fma(p, q, 2.0 / 13.0);
    p = fma(p, q, 2.0 / 11.0);
    p = fma(p, q, 2.0 / 9.0);
    p = fma(p, q, 2.0 / 7.0);
    p = fma(p, q, 2.0 / 5.0);
    p = fma(p, q, 2.0 / 3.0);
    p = fma(p, q, 2.0);
    return p * z;
}

// exp(l - m) with m the largest logit: the limit where both are +inf.
__device__ __forceinline__ double route_exp(float l, float m) {
    return l == m ? 1.0 : route_exp64((double)l - (double)m);
}

// The score of logit l; softmax: m the row's largest logit, sum its total.
__device__ __forceinline__ double route_score(float l, int score, float m, double sum) {
    if (score == ROUTE_SOFTMAX) return route_exp(l, m) / sum;
    const double x = (double)l, e = route_exp64(score == ROUTE_SIGMOID ? -x : -fabs(x));
    if (score == ROUTE_SIGMOID) return 1.0 / (1.0 + e);
    return sqrt(fmax(x, 0.0) + route_log1p(e));
}

constexpr double kNever = -__builtin_inf();  // an expert that is not to be chosen

// (a, ia) comes before (b, ib): the larger, then the lower index.
__device__ __forceinline__ bool route_before(double a, int ia, double b, int ib) {
    return a > b || (a == b && ia < ib);
}

__device__ __forceinline__ void route_best(double &v, int &i, double v2, int i2) {
    if (route_before(v2, i2, v, i)) {
        v = v2;
        i = i2;
    }
}

}  // namespace

// One workgroup per token, any number of experts: every round looks through all
// keys again, made anew from the logits, for the best that comes after the last
// one chosen. LDS: n_group doubles.
__global__ __launch_bounds__(256) void k_route_any(RouteArgs a) {
    extern __shared__ double gsum[];
    __shared__ double red_v[4];
    __shared__ int red_i[4];
    __shared__ double chosen_s[64];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const size_t row = (size_t)t * a.stride;
    const int per = a.n_expert / a.n_group;

    // the best (value, index) of the workgroup, at every thread
    auto block_best = [&](double v, int i, double &bv, int &bi) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1)
            route_best(v, i, __shfl_xor(v, off, 64), __shfl_xor(i, off, 64));
        __syncthreads();
        if (lane == 0) {
            red_v[wv] = v;
            red_i[wv] = i;
        }
        __syncthreads();
        bv = red_v[0];
        bi = red_i[0];
        for (int w = 1; w < 4; w++) route_best(bv, bi, red_v[w], red_i[w]);
    };

    float m = -__builtin_inff();
    double sum = 0.0;
    if (a.score == ROUTE_SOFTMAX) {
        double v = kNever, bv;
        int bi;
        for (int e = tid; e < a.n_expert; e += 256) {
            const float l = route_load(a.logits, row + e, a.dtype);
            if ((double)l > v) v = (double)l;  // (a NaN is not)
        }
        block_best(v, 0, bv, bi);
        m = (float)bv;
        double s = 0.0;
        for (int e = tid; e < a.n_expert; e += 256) {
            const float l = route_load(a.logits, row + e, a.dtype);
            if (l > -__builtin_inff()) s += route_exp(l, m);
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
        __syncthreads();
        if (lane == 0) red_v[wv] = s;
        __syncthreads();
        sum = (red_v[0] + red_v[1]) + (red_v[2] + red_v[3]);
        __syncthreads();
    }
    // an expert's place; kNever where it is not to be chosen
    auto place = [&](int e) {
        const float l = route_load(a.logits, row + e, a.dtype);
        if (!(l > -__builtin_inff())) return kNever;
        if (!a.bias) return (double)l;
        const double k = route_score(l, a.score, m, sum) + (double)a.bias[e];
        return k > kNever ? k : kNever;
    };
    if (a.n_group > 1) {
        for (int g = tid; g < a.n_group; g += 256) {
            double b0 = kNever, b1 = kNever;
            for (int e = g * per; e < (g + 1) * per; e++) {
                double v = place(e);
                if (!a.bias && v > kNever)
                    v = route_score(route_load(a.logits, row + e, a.dtype), a.score, m, sum);
                if (v > b0) {
                    b1 = b0;
                    b0 = v;
                } else if (v > b1) {
                    b1 = v;
                }
            }
            gsum[g] = a.group_top == 2 && b1 > kNever ? b0 + b1 : b0;
        }
        __syncthreads();
        // the topk_group best groups get NaN, the others are left as they are
        for (int r = 0; r < a.topk_group; r++) {
            double v = kNever, bv;
            int i = a.n_group, bi;
            for (int g = tid; g < a.n_group; g += 256) route_best(v, i, gsum[g], g);
            block_best(v, i, bv, bi);
            if (!(bv > kNever)) break;  // (the same at every thread)
            if (tid == 0) gsum[bi] = __builtin_nan("");
            __syncthreads();
        }
    }
    double last_v = __builtin_inf(), total = 0.0;
    int last_i = -1, found = 0;
    for (int r = 0; r < a.k; r++) {
        double v = kNever, bv;
        int i = a.n_expert, bi;
        for (int e = tid; e < a.n_expert; e += 256) {
            if (a.n_group > 1 && gsum[e / per] == gsum[e / per]) continue;
            const double p = place(e);
            if (p > kNever && route_before(last_v, last_i, p, e)) route_best(v, i, p, e);
        }
        block_best(v, i, bv, bi);
        if (!(bv > kNever)) break;
        const double s = route_score(route_load(a.logits, row + bi, a.dtype), a.score, m, sum);
        total += s;
        if (tid == 0) {
            chosen_s[r] = s;
            a.ids[(size_t)t * a.k + r] = bi;
        }
        last_v = bv;
        last_i = bi;
        found = r + 1;
    }
    __syncthreads();
    if (tid < a.k) {
        const size_t at = (size_t)t * a.k + tid;
        double w = 0.0;
        if (tid < found) {
            w = chosen_s[tid] * (double)a.scale;
            if (a.renormalise) w = total == 0.0 ? 0.0 : w / total;
        } else {
            a.ids[at] = -1;
        }
        a.weights[at] = (float)w;
    }
}

namespace {

// ---- W lanes per token --------------------------------------------------------
//
// Lane l of a token's W holds R neighbouring experts of group l / LG (LG lanes a
// group), so lanes, and a lane's own places, stand in the order of the ids. A
// lane keeps the three best of its R at hand; every round takes the best of the W
// lanes' first ones, and only a lane that gave three looks through its R again.
// The choice is made in f32. Which of two keys is larger is certain there when
// they are further apart than f32 can be off (route_apart). The chosen experts'
// scores are wanted in 64 bits for the weights anyhow: where two neighbours among
// them, or the last of them and up to four behind it, are close, those settle it.
// More that are close there, or a kept group close to one left out, and not the
// same logit and bias: the token's choice is made again in 64 bits.
// Several tokens a wavefront share its instructions, and the best of 16 lanes is
// four steps within a DPP row; more experts a lane cost more looks through them.

// A float's place in the order of all floats as a number (no NaN); 0, below that of
// -inf: none.
__device__ __forceinline__ uint32_t route_order(float v) {
    const int b = __builtin_bit_cast(int, v);
    return (uint32_t)b ^ ((uint32_t)(b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float route_value(uint32_t o) {
    return __builtin_bit_cast(float, o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
// The largest of a token's W lanes' values, at each of them: rotations within the
// DPP rows of 16 lanes, then rows exchanged.
template <int W> __device__ __forceinline__ uint32_t route_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true));  // row_ror:8
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x122, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x121, 0xf, 0xf, true));
    if constexpr (W >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max((uint32_t)s[0], (uint32_t)s[1]);
    }
    if constexpr (W >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max((uint32_t)s[0], (uint32_t)s[1]);
    }
    return v;
}
// The first of a token's W lanes (0..W - 1) where `yes`, W or more if none.
template <int W> __device__ __forceinline__ int route_first(bool yes) {
    const unsigned long long all = __ballot(yes);
    const int lane = threadIdx.x & 63;
    if constexpr (W == 64) return all ? __ffsll(all) - 1 : 64;
    uint32_t half = lane < 32 ? (uint32_t)all : (uint32_t)(all >> 32);
    if constexpr (W == 16) half = lane & 16 ? half >> 16 : half & 0xFFFFu;
    return half ? __ffs((int)half) - 1 : 64;
}
template <int W> __device__ __forceinline__ double route_sum(double v) {
#pragma unroll
    for (int off = W / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

__device__ __forceinline__ float route_score32(float l, int score, float m, float inv) {
    if (score == ROUTE_SOFTMAX) return (l == m ? 1.0f : __expf(l - m)) * inv;
    if (score == ROUTE_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + __expf(-l));
    // log(1 + e) with what the sum 1 + e lost put back
    const float e = __expf(-fabsf(l)), u = 1.0f + e;
    const float g = e < 0.01f ? e * (1.0f - e * (0.5f - e * (1.0f / 3.0f)))
                              : __logf(u) + (e - (u - 1.0f)) * __builtin_amdgcn_rcpf(u);
    return __builtin_amdgcn_sqrtf(fmaxf(l, 0.0f) + g);
}

// Whether f32 keys a >= b are certainly in that order. With u = 2^-24, exp(x) from
// v_exp_f32 is (|x| + 2) u off (the product with log2 e, the instruction's step).
//   sigmoid: s (1 - s) (|x| + 2) u < 0.73 u, and 3 u for 1 + e and v_rcp_f32
//   sqrt(log(1 + e) + max(l, 0)): 1 + e is made good, so the logarithm is within
//     (|l| + 5) u relative, its root within half of that and 2 u: s |l| < 1 where
//     l < 0, so 5 u for s < 1, and 5 u relative above
//   softmax: s <= 1 / S, and relative (|x| + 2) u, and 31 u for S (22 additions
//     one after the other, its terms' own) and its inverse: 36 u / S
// and the sum with the bias u relative. off: twice that and some more, for the two,
// of the token's largest score (from its largest logit).
__device__ __forceinline__ bool route_apart(float a, float b, float off) {
    return a - b > off + 0x1p-22f * fmaxf(fabsf(a), fabsf(b));
}
__device__ __forceinline__ float route_off(int score, float top, float inv) {
    if (score == ROUTE_SOFTMAX) return 0x1.4p-18f * inv;
    if (score == ROUTE_SIGMOID) return 0x1p-21f;
    return 0x1.8p-21f * fmaxf(1.0f, sqrtf(top + 0.7f));
}

// Lane `sub` of a token's: the R experts from id `first` on, logits -inf where
// there is none or it cannot be chosen.
template <int R> struct RouteLane {
    float l[R], b[R];  // logits and biases
    int first;
};

// What the host works out of a call's sizes.
struct RouteForm {
    int per, LG;  // experts a group, lanes a group
    int whole;    // every lane holds R experts, at 16-byte aligned addresses
};
// A token's chosen experts in LDS: id and f32 key (as route_order), the r-th at [r].
struct RoutePick {
    int id;
    uint32_t key;
};

// The k best (and what is close behind them: `taken` in all) of each of the
// wavefront's tokens by their f32 keys (inv: the inverse of
// the softmax's divisor; off: route_off) to `pick`, id -1 behind the last. False at the tokens where
// f32 cannot tell which they are.
template <int W, int R>
__device__ __forceinline__ bool route_choose(const RouteArgs &a, const RouteForm &f, const RouteLane<R> &x,
                                             int g, float m, float inv, float off, RoutePick *pick, int &taken) {
    const int lane = threadIdx.x & 63, sub = lane % W;
    const float none = -__builtin_inff();
    bool sure = true;
    uint32_t place[R];
#pragma unroll
    for (int j = 0; j < R; j++) place[j] = x.l[j] > none ? route_order(x.l[j]) : 0;
    if (a.bias || a.n_group > 1) {
        uint32_t key[R];
#pragma unroll
        for (int j = 0; j < R; j++) {
            const float s = route_score32(x.l[j], a.score, m, inv) + (a.bias ? x.b[j] : 0.0f);
            // (+ 0.0: keys of -0; a NaN is not chosen)
            key[j] = place[j] && s > none ? route_order(s + 0.0f) : 0;
            place[j] = a.bias ? key[j] : place[j];
        }
        if (a.n_group > 1) {
            // the lane's two best keys, then those of the group at its first
            // lane: every step adds the lanes behind those gathered so far
            uint32_t b0 = 0, b1 = 0;
#pragma unroll
            for (int j = 0; j < R; j++) {
                b1 = max(b1, min(key[j], b0));
                b0 = max(b0, key[j]);
            }
            const int head = g * f.LG, in_group = sub - head;
            for (int d = 1; d < f.LG; d <<= 1) {
                const uint32_t c0 = (uint32_t)__shfl_down((int)b0, d, 64), c1 = (uint32_t)__shfl_down((int)b1, d, 64);
                if (in_group + d < f.LG) {
                    b1 = max(max(b1, c1), min(b0, c0));
                    b0 = max(b0, c0);
                }
            }
            // What the group counts, and how far that may be off: its two scores (off),
            // and with K its larger key 2^-24 K for each key's rounding and twice that
            // for the sum's and for the edge's below. K, not the sum: of keys of opposite
            // signs little may be left.
            const bool two = a.group_top == 2 && b1, first = in_group == 0 && g < a.n_group && b0;
            const float v0 = route_value(b0), v1 = two ? route_value(b1) : 0.0f;
            const float count = v0 + v1 + 0.0f, far = off + 0x1.9p-22f * fmaxf(fabsf(v0), fabsf(v1));
            uint32_t sum = first ? route_order(count) : 0;
            bool kept = false;
            for (int r = 0; r < a.topk_group; r++) {
                const uint32_t best = route_max<W>(sum);
                const int who = route_first<W>(sum == best && best != 0);
                kept |= who == head;
                if (who == sub) sum = 0;
            }
            // the least that a kept group may count against the most of one left out (a
            // count beyond f32: anything)
            const float to = kept ? -far : far;
            const uint32_t edge = route_order(fabsf(count) < -none ? count + to : kept ? none : -none);
            const uint32_t low = ~route_max<W>(first && kept ? ~edge : 0), high = route_max<W>(first && !kept ? edge : 0);
            const bool near = high && low <= high;
            if (__ballot(near)) {
                // groups of one key each are equal where the logits and biases are
                bool unsure = near && a.group_top == 2;
                const uint32_t last = ~route_max<W>(first && kept ? ~route_order(count) : 0);
                uint32_t l = 0, b = 0;
#pragma unroll
                for (int j = 0; j < R; j++)
                    if (key[j] == last) {
                        l = max(l, route_order(x.l[j]));
                        b = max(b, a.bias ? route_order(x.b[j]) : 1u);
                    }
                l = route_max<W>(l);
                b = route_max<W>(b);
#pragma unroll
                for (int j = 0; j < R; j++)
                    if (near && key[j] && !route_apart(route_value(max(key[j], last)), route_value(min(key[j], last)), off))
                        unsure |= !(route_order(x.l[j]) == l && (!a.bias || route_order(x.b[j]) == b));
                sure = route_first<W>(unsure) >= W;
            }
#pragma unroll
            for (int j = 0; j < R; j++) place[j] = kept ? place[j] : 0;
        }
    }
    uint32_t h0, h1, h2;
    int a0, a1, a2;
    // the lane's three best of those below `under`, and behind j = from of those
    // that equal it
    auto scan = [&](uint32_t under, int from) __attribute__((always_inline)) {
        h0 = h1 = h2 = 0;
        a0 = a1 = a2 = 0;
#pragma unroll
        for (int j = 0; j < R; j++) {
            const uint32_t v = place[j] < under || (place[j] == under && j > from) ? place[j] : 0;
            const bool g0 = v > h0, g1 = v > h1, g2 = v > h2;
            h2 = g1 ? h1 : g2 ? v : h2;
            a2 = g1 ? a1 : g2 ? j : a2;
            h1 = g0 ? h0 : g1 ? v : h1;
            a1 = g0 ? a0 : g1 ? j : a1;
            h0 = g0 ? v : h0;
            a0 = g0 ? j : a0;
        }
    };
    scan(0xFFFFFFFFu, -1);
    for (int r = sub; r < min(a.k + 4, 64); r += W) pick[r] = RoutePick{-1, 0};
    __builtin_amdgcn_wave_barrier();
    int gave = 0;
    // the best one left, as pick[r], at the tokens where `take` lets it
    auto round = [&](int r, auto take) __attribute__((always_inline)) {
        const uint32_t best = route_max<W>(h0);
        const bool in = best != 0 && take(best);
        const int who = route_first<W>(h0 == best && in);
        const int from = a0;
        if (who == sub) {
            pick[r] = RoutePick{x.first + a0, best};
            gave++;
            h0 = h1;
            a0 = a1;
            h1 = h2;
            a1 = a2;
            h2 = 0;
        }
        if (R > 3 && __ballot(gave == 3)) {
            const uint32_t k0 = h0, k1 = h1, k2 = h2;
            const int i0 = a0, i1 = a1, i2 = a2;
            scan(best, from);  // what comes after the one it just gave
            if (gave == 3) {
                gave = 0;
            } else {
                h0 = k0; h1 = k1; h2 = k2;
                a0 = i0; a1 = i1; a2 = i2;
            }
        }
        return best;
    };
    uint32_t last = 0;
    for (int r = 0; r < a.k; r++) {
        const uint32_t best = round(r, [](uint32_t) { return true; });
        last = best ? best : last;
    }
    taken = a.k;
    if (a.bias) {
        // up to four more that are close to the last chosen, for the 64-bit keys
        auto close = [&](uint32_t k) { return k && !route_apart(route_value(last), route_value(k), off); };
        while (__ballot(close(route_max<W>(h0))) && taken < a.k + 4 && taken < 64) {
            (void)round(taken, close);
            taken++;
        }
        const bool near = close(route_max<W>(h0));
        if (__ballot(near)) {
            // still more: chosen or not, whatever is close to the last chosen has
            // to be its equal then, the same logit and bias
            bool unsure = false;
            uint32_t l = 0, b = 0;
#pragma unroll
            for (int j = 0; j < R; j++)
                if (place[j] == last) {
                    l = max(l, route_order(x.l[j]));
                    b = max(b, route_order(x.b[j]));
                }
            l = route_max<W>(l);
            b = route_max<W>(b);
#pragma unroll
            for (int j = 0; j < R; j++)
                if (near && place[j] && !route_apart(route_value(max(place[j], last)), route_value(min(place[j], last)), off))
                    unsure |= !(route_order(x.l[j]) == l && route_order(x.b[j]) == b);
            sure = sure && route_first<W>(unsure) >= W;
        }
    }
    return sure;
}

// A double's place in the order of all doubles (no NaN).
__device__ __forceinline__ uint64_t route_order64(double v) {
    const long long b = __builtin_bit_cast(long long, v + 0.0);
    return (uint64_t)b ^ ((uint64_t)(b >> 63) | 0x8000000000000000ull);
}

// One token's choice in 64 bits by a whole wavefront, the r-th's id at lane r. Rarely
// run, so its code is kept short: what it costs is fetching it. keys, gsum: LDS for
// n_expert and n_group values; keys are kept as places in the order, 0 for an
// expert that is not to be chosen.
__device__ __forceinline__ int route_exact(const RouteArgs &a, size_t row, double *keys, double *gsum) {
    const int lane = threadIdx.x & 63, per = a.n_expert / a.n_group;
    float m = -__builtin_inff();
    double sum = 0.0;
    if (a.score == ROUTE_SOFTMAX) {
#pragma unroll 1
        for (int e = lane; e < a.n_expert; e += 64) {
            const float l = route_load(a.logits, row + e, a.dtype);
            m = l > m ? l : m;
        }
        m = route_value(route_max<64>(route_order(m)));
#pragma unroll 1
        for (int e = lane; e < a.n_expert; e += 64) {
            const float l = route_load(a.logits, row + e, a.dtype);
            if (l > -__builtin_inff()) sum += route_exp(l, m);
        }
        sum = route_sum<64>(sum);
    }
#pragma unroll 1
    for (int e = lane; e < a.n_expert; e += 64) {
        const float l = route_load(a.logits, row + e, a.dtype);
        double k = kNever;
        if (l > -__builtin_inff()) {
            k = route_score(l, a.score, m, sum) + (a.bias ? (double)a.bias[e] : 0.0);
            k = k > kNever ? k : kNever;
        }
        keys[e] = k;
    }
    __syncthreads();  // (one wavefront a workgroup)
    if (a.n_group > 1) {
        // (at most 64 groups, a lane each)
        double b0 = kNever, b1 = kNever;
        if (lane < a.n_group) {
#pragma unroll 4
            for (int e = lane * per; e < (lane + 1) * per; e++) {
                const double k = keys[e];
                b1 = k > b0 ? b0 : k > b1 ? k : b1;
                b0 = k > b0 ? k : b0;
            }
            b0 = a.group_top == 2 && b1 > kNever ? b0 + b1 : b0;
            gsum[lane] = b0;
        }
        __syncthreads();
        int before = 0;
#pragma unroll 4
        for (int g = 0; g < a.n_group; g++) before += route_before(gsum[g], g, b0, lane);
        if (lane < a.n_group && before >= a.topk_group) {
#pragma unroll 1
            for (int e = lane * per; e < (lane + 1) * per; e++) keys[e] = kNever;
        }
        __syncthreads();
    }
    int id = -1;
    uint64_t *const place = reinterpret_cast<uint64_t *>(keys);
#pragma unroll 1
    for (int e = lane; e < a.n_expert; e += 64) {
        // without a bias the logits are the order
        double k = keys[e];
        if (!a.bias && k > kNever) k = (double)route_load(a.logits, row + e, a.dtype);
        place[e] = k > kNever ? route_order64(k) : 0;
    }
#pragma unroll 1
    for (int r = 0; r < a.k; r++) {
        uint64_t v = 0;
        int i = 0;
#pragma unroll 4
        for (int e = lane; e < a.n_expert; e += 64) {
            const uint64_t k = place[e];
            i = k > v ? e : i;
            v = k > v ? k : v;
        }
        // the upper halves first, then the lower among those, then the ids
        const uint32_t hi = route_max<64>((uint32_t)(v >> 32));
        bool in = (uint32_t)(v >> 32) == hi;
        const uint32_t lo = route_max<64>(in ? (uint32_t)v : 0);
        if (hi == 0) break;
        in = in && (uint32_t)v == lo;
        const int won = (int)~route_max<64>(in ? ~(uint32_t)i : 0);
        if (lane == r) id = won;
        if (in && i == won) place[won] = 0;
    }
    __syncthreads();
    return id;
}

template <int W, int R>
__global__ __launch_bounds__(64) void k_route(RouteArgs a, RouteForm f, int n_tok) {
    constexpr int KS = 64 / W;  // chosen experts a lane
    __shared__ double keys[W * R], gsum[64];
    __shared__ RoutePick picks[KS][64];
    const int lane = threadIdx.x & 63, sub = lane % W;
    const int t = min((int)blockIdx.x * KS + lane / W, n_tok - 1);
    const bool mine = (int)blockIdx.x * KS + lane / W < n_tok;
    const size_t row = (size_t)t * a.stride;
    const float none = -__builtin_inff();
    const int g = a.n_group == 1 ? 0 : sub / f.LG, e0 = (sub - g * f.LG) * R;
    RoutePick *const pick = picks[lane / W];
    RouteLane<R> x;
    x.first = g * f.per + e0;
    // all loads before the first use
    if (f.whole) {
        float4 b[R / 4];
        if (a.bias) {
#pragma unroll
            for (int j = 0; j < R / 4; j++) b[j] = reinterpret_cast<const float4 *>(a.bias + x.first)[j];
        }
        if (a.dtype == T_F32) {
            const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.logits) + row + x.first);
            float4 v[R / 4];
#pragma unroll
            for (int j = 0; j < R / 4; j++) v[j] = p[j];
#pragma unroll
            for (int j = 0; j < R / 4; j++) {
                x.l[4 * j] = v[j].x; x.l[4 * j + 1] = v[j].y; x.l[4 * j + 2] = v[j].z; x.l[4 * j + 3] = v[j].w;
            }
        } else {
            const uint2 *p = reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.logits) + row + x.first);
            uint2 v[R / 4];
#pragma unroll
            for (int j = 0; j < R / 4; j++) v[j] = p[j];
#pragma unroll
            for (int j = 0; j < R; j++) {
                const uint32_t w = j & 2 ? v[j / 4].y : v[j / 4].x;
                x.l[j] = a.dtype == T_F16 ? f16_to_f32(j & 1 ? w >> 16 : w & 0xFFFFu)
                                          : __builtin_bit_cast(float, j & 1 ? w & 0xFFFF0000u : w << 16);
            }
        }
        if (a.bias) {
#pragma unroll
            for (int j = 0; j < R / 4; j++) {
                x.b[4 * j] = b[j].x; x.b[4 * j + 1] = b[j].y; x.b[4 * j + 2] = b[j].z; x.b[4 * j + 3] = b[j].w;
            }
        }
    } else {
        // past the end the row's last expert
        auto at = [&](int j) { return min(x.first + j, a.n_expert - 1); };
        if (a.dtype == T_F32) {
            const float *p = static_cast<const float *>(a.logits) + row;
#pragma unroll
            for (int j = 0; j < R; j++) x.l[j] = p[at(j)];
        } else {
            const uint16_t *p = static_cast<const uint16_t *>(a.logits) + row;
            uint32_t b[R];
#pragma unroll
            for (int j = 0; j < R; j++) b[j] = p[at(j)];
#pragma unroll
            for (int j = 0; j < R; j++)
                x.l[j] = a.dtype == T_F16 ? f16_to_f32(b[j]) : __builtin_bit_cast(float, b[j] << 16);
        }
        if (a.bias) {
#pragma unroll
            for (int j = 0; j < R; j++) x.b[j] = a.bias[at(j)];
        }
#pragma unroll
        for (int j = 0; j < R; j++) x.l[j] = g < a.n_group && e0 + j < f.per ? x.l[j] : none;
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < R; j++) {
        // (+ 0.0: -0 and 0 are one place; a NaN is not to be chosen)
        x.l[j] = x.l[j] > none ? x.l[j] + 0.0f : none;
        top = max(top, route_order(x.l[j]));
    }
    const bool softmax = a.score == ROUTE_SOFTMAX, keyed = a.bias || a.n_group > 1;
    float m = none, inv = 1.0f;
    if (softmax || keyed) {
        m = route_value(route_max<W>(top));
        if (softmax && keyed) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < R; j++)
                if (x.l[j] > none) s += x.l[j] == m ? 1.0f : __expf(x.l[j] - m);
#pragma unroll
            for (int off = W / 2; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
            inv = 1.0f / s;
        }
    }
    auto sum64 = [&]() {
        double s = 0.0;
#pragma unroll 2
        for (int e = sub; e < a.n_expert; e += W) {
            const float l = route_load(a.logits, row + e, a.dtype);
            const double v = route_exp(l, m);
            s += l > none ? v : 0.0;
        }
        return route_sum<W>(s);
    };
    double sum = 1.0;
    if (softmax && !a.renormalise) sum = sum64();
    const float off = route_off(a.score, m, inv);
    int taken;
    const bool sure = route_choose<W, R>(a, f, x, g, m, inv, off, pick, taken);
    bool settled = false;  // by 64-bit keys
    unsigned long long todo = __ballot(!sure);
    while (todo) {
        const int first = (__ffsll(todo) - 1) & ~(W - 1);  // the token's first lane
        todo &= ~(~0ull >> (64 - W) << first);
        const size_t its = ((size_t)__builtin_amdgcn_readlane((int)(row >> 32), first) << 32) |
                           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)row, first);
        const int exact = route_exact(a, its, keys, gsum);
        if (lane < taken) picks[first / W][lane].id = lane < a.k ? exact : -1;
        settled |= (lane & ~(W - 1)) == first;
    }
    __syncthreads();
    int id[KS];
    uint32_t place[KS];
#pragma unroll
    for (int i = 0; i < KS; i++) {
        const RoutePick p = i * W + sub < taken ? pick[i * W + sub] : RoutePick{-1, 0};
        id[i] = p.id;
        place[i] = settled ? 0 : p.key;
    }
    // their scores in 64 bits (renormalised, the softmax's divisor leaves the
    // weights as they are)
    double w[KS];
#pragma unroll
    for (int i = 0; i < KS; i++) {
        w[i] = 0.0;
        if (i * W < taken) {
            const float l = route_load(a.logits, row + max(id[i], 0), a.dtype);
            const double s = route_score(l, a.score, m, sum);
            w[i] = id[i] >= 0 ? s : 0.0;
        }
    }
    int rank[KS];
#pragma unroll
    for (int i = 0; i < KS; i++) rank[i] = i * W + sub;
    if (a.bias) {
        // neighbours in the order that f32 cannot tell apart
        bool near = false;
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const int r = i * W + sub;
            if (r + 1 < taken && place[i]) {
                const uint32_t next = pick[r + 1].key;
                near |= next && !route_apart(route_value(place[i]), route_value(next), off);
            }
        }
        if (__ballot(near)) {
            // all by their keys in 64 bits (the softmax's with its divisor)
            const double norm = softmax && a.renormalise ? sum64() : 1.0;
            double key[KS];
#pragma unroll
            for (int i = 0; i < KS; i++) {
                key[i] = id[i] >= 0 ? w[i] / norm + (double)a.bias[max(id[i], 0)] : kNever;
                rank[i] = 0;
            }
            for (int r = 0; r < taken; r++) {
                const int from = (lane & ~(W - 1)) + r % W;
                double o = key[0];
                int oi = id[0];
#pragma unroll
                for (int i = 1; i < KS; i++) {
                    o = r / W == i ? key[i] : o;
                    oi = r / W == i ? id[i] : oi;
                }
                o = __shfl(o, from, 64);
                oi = __shfl(oi, from, 64);
#pragma unroll
                for (int i = 0; i < KS; i++)
                    rank[i] += id[i] >= 0 ? (oi >= 0 && route_before(o, oi, key[i], id[i])) : i * W + sub > r;
            }
        }
    }
    double total = 0.0;
    if (a.renormalise) {
#pragma unroll
        for (int i = 0; i < KS; i++) total += rank[i] < a.k ? w[i] : 0.0;
        total = route_sum<W>(total);
    }
#pragma unroll
    for (int i = 0; i < KS; i++) {
        if (rank[i] >= a.k || !mine) continue;
        double v = w[i] * (double)a.scale;
        if (a.renormalise) v = total == 0.0 ? 0.0 : v / total;
        const size_t at = (size_t)t * a.k + rank[i];
        a.ids[at] = id[i];
        a.weights[at] = (float)v;
    }
}

template <int W, int R> hipError_t route_go(const RouteArgs &a, int n_tok, int LG, hipStream_t s) {
    constexpr int per_wg = 64 / W;
    const int per = a.n_expert / a.n_group;
    const size_t piece = 4 * (a.dtype == T_F32 ? 4 : 2);  // bytes of a load
    const bool whole = LG * R == per && LG * a.n_group == W && (uintptr_t)a.logits % piece == 0 &&
                       a.stride % 4 == 0 && (uintptr_t)a.bias % 16 == 0;
    k_route<W, R><<<(unsigned)((n_tok + per_wg - 1) / per_wg), 64, 0, s>>>(a, RouteForm{per, LG, whole}, n_tok);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_route(const RouteArgs &a, int n_tok, hipStream_t s) {
    if (n_tok <= 0) return hipSuccess;
    // the fewest lanes a token that hold its groups with 4, then 8 experts each
    // (256 experts, 8 of them, no bias, us at 512 / 4095 / 16384 tokens: 32 lanes
    // of 8 6.4 / 7.7 / 15.6, 64 of 4 6.2 / 7.5 / 21.6, 16 of 16 9.2 / 9.1 / 18.3;
    // 64 experts at 16384: 16 lanes of 4 9.8, 32 of 8 21.7)
    const int per = a.n_expert / a.n_group;
    struct Form {
        int w, r;
        hipError_t (*go)(const RouteArgs &, int, int, hipStream_t);
    };
    static const Form forms[] = {{16, 4, route_go<16, 4>}, {16, 8, route_go<16, 8>}, {32, 8, route_go<32, 8>},
                                 {64, 8, route_go<64, 8>}, {64, 16, route_go<64, 16>}};
    for (const Form &f : forms) {
        const int LG = (per + f.r - 1) / f.r;
        if ((long long)LG * a.n_group <= f.w) return f.go(a, n_tok, LG, s);
    }
    k_route_any<<<(unsigned)n_tok, 256, (size_t)a.n_group * sizeof(double), s>>>(a);
    return hipGetLastError();
}

}  // namespace rsllm_hip
