// Expert routing: router logits -> the ids and weights of each token's experts.
//
// Scores, keys and group sums are 64-bit, so which of two near experts is
// chosen does not hang on a 32-bit rounding of exp; the weights are rounded
// once at the end. An expert's place in the order is its key (score + bias), or
// its logit itself where there is no bias (the scores rise with the logits);
// equal places go to the lower id.
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

// exp(l - m) with m the largest logit: the limit where both are +inf.
__device__ __forceinline__ double route_exp(float l, float m) {
    return l == m ? 1.0 : exp((double)l - (double)m);
}

// The score of logit l; softmax: m the row's largest logit, sum its total.
__device__ __forceinline__ double route_score(float l, int score, float m, double sum) {
    if (score == ROUTE_SOFTMAX) return route_exp(l, m) / sum;
    if (score == ROUTE_SIGMOID) return 1.0 / (1.0 + exp(-(double)l));
    const double x = (double)l;
    return sqrt((x > 0.0 ? x : 0.0) + log1p(exp(-fabs(x))));
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

// ---- one wavefront per token -----------------------------------------------
//
// Lane l holds R neighbouring experts of group l / LG (LG lanes a group), so
// lanes, and a lane's own places, stand in the order of the ids. The choice is
// made in f32 and certain wherever two neighbours in the order are further apart
// than twice what f32 can be off (kRouteOff relative to the larger, or to 1), or
// have the same logit and bias; a token with another close pair goes
// through the same steps in 64 bits. 256 experts with biases of 0.05: about 1
// token in 300 does.

// How far an f32 key may be off, relative to max(1, |key|). exp(x) from v_exp_f32
// is (|x| + 3) 2^-24 off; sigmoid'(x) |x| < 1/4 and exp(x) |x| < 0.4, so the two
// scores within [0, 1] are within 2^-21 (the softmax's sum adds 16 roundings);
// sqrt(log(1 + e)) with e >= 0.01 (below it a series) halves the relative error
// of a logarithm that is within 2^-22 absolute, and is at least 0.1: 2^-19.7.
constexpr float kRouteOff = 0x1p-19f;

// The largest of 64 lanes' values, at every lane (uniform).
__device__ __forceinline__ float route_wave_max(float v) {
    auto step = [](float x, auto ctrl, auto rows) {
        const int lo = __builtin_bit_cast(int, -__builtin_inff());
        return fmaxf(x, __builtin_bit_cast(
                            float, __builtin_amdgcn_update_dpp(lo, __builtin_bit_cast(int, x),
                                                               decltype(ctrl)::value,
                                                               decltype(rows)::value, 0xf, false)));
    };
    using std::integral_constant;
    v = step(v, integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr:1
    v = step(v, integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    v = step(v, integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    v = step(v, integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    v = step(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast:15
    v = step(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row_bcast:31
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ double route_wave_max(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = fmax(v, __shfl_xor(v, off, 64));
    return v;
}

__device__ __forceinline__ float route_score32(float l, int score, float m, float inv) {
    if (score == ROUTE_SOFTMAX) return (l == m ? 1.0f : __expf(l - m)) * inv;
    if (score == ROUTE_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + __expf(-l));
    const float e = __expf(-fabsf(l));
    const float g = e < 0.01f ? e * (1.0f - e * (0.5f - e * (1.0f / 3.0f))) : __logf(1.0f + e);
    return __builtin_amdgcn_sqrtf(fmaxf(l, 0.0f) + g);
}

// Whether a before b is certain in f32.
__device__ __forceinline__ bool route_apart(float a, float b) {
    return a - b > 2.0f * kRouteOff * fmaxf(1.0f, fmaxf(fabsf(a), fabsf(b)));
}

// Lane `lane` of a token's wavefront: the R experts from id `first` on, live
// where they exist and can be chosen.
template <int R> struct RouteLane {
    float l[R];  // logits; -inf where there is nothing to choose
    int first;
};

// The k best of the token in the order of the keys (T: float or double; norm:
// the softmax's divisor, or its inverse in float), lane i getting the i-th's id,
// -1 behind the last. False where T cannot tell.
template <class T, int R>
__device__ __forceinline__ bool route_choose(const RouteArgs &a, size_t row, const RouteLane<R> &x,
                                             int LG, float m, T norm, int &id) {
    constexpr bool kFast = sizeof(T) == 4;
    const int lane = threadIdx.x & 63;
    const T never = -(T)__builtin_inff();
    T key[R], place[R];
#pragma unroll
    for (int j = 0; j < R; j++) {
        key[j] = never;
        if (x.l[j] > -__builtin_inff()) {
            if (a.bias || a.n_group > 1) {
                if constexpr (kFast) key[j] = route_score32(x.l[j], a.score, m, norm);
                else key[j] = route_score(x.l[j], a.score, m, norm);
                if (a.bias) key[j] += (T)a.bias[x.first + j];
                key[j] = key[j] > never ? key[j] : never;  // (a NaN is not)
            }
        }
        place[j] = a.bias ? key[j] : (T)x.l[j];
    }
    if (a.n_group > 1) {
        // the lane's two best keys, then those of the group at its first lane:
        // every step adds the lanes behind those gathered so far
        T b0 = never, b1 = never;
#pragma unroll
        for (int j = 0; j < R; j++) {
            b1 = key[j] > b0 ? b0 : key[j] > b1 ? key[j] : b1;
            b0 = key[j] > b0 ? key[j] : b0;
        }
        const int in_group = lane % LG;
        for (int off = 1; off < LG; off <<= 1) {
            const T c0 = __shfl_down(b0, off, 64), c1 = __shfl_down(b1, off, 64);
            if (in_group + off < LG) {
                const T lo = b0 < c0 ? b0 : c0, hi = b1 > c1 ? b1 : c1;
                b0 = b0 > c0 ? b0 : c0;
                b1 = lo > hi ? lo : hi;
            }
        }
        const bool head = in_group == 0 && lane < LG * a.n_group;
        T sum = !head ? never : a.group_top == 2 && b1 > never ? b0 + b1 : b0;
        unsigned long long kept = 0;
        T last = never;
        for (int r = 0; r < a.topk_group; r++) {
            const T best = route_wave_max(sum);
            if (!(best > never)) break;
            const int who = __ffsll(__ballot(sum == best)) - 1;
            kept |= 1ull << who;
            last = best;
            if (lane == who) sum = never;
        }
        if constexpr (kFast) {
            const T next = route_wave_max(sum);
            // (half the gap: sums of two)
            if (next > never && !route_apart(0.5f * last, 0.5f * next)) return false;
        }
        if (!(kept >> (lane - in_group) & 1)) {
#pragma unroll
            for (int j = 0; j < R; j++) place[j] = never;
        }
    }
    id = -1;
    T last = never;
    int last_id = 0;
    const int rounds = kFast && a.bias ? a.k + 1 : a.k;  // the last against the next
    for (int r = 0; r < rounds; r++) {
        T top = place[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < R; j++) {
            at = place[j] > top ? j : at;
            top = place[j] > top ? place[j] : top;
        }
        const T best = route_wave_max(top);
        if (!(best > never)) break;
        const int who = __ffsll(__ballot(top == best)) - 1;
        const int won = __builtin_amdgcn_readlane(x.first + at, who);
        if constexpr (kFast) {
            // whatever is near the one before has to be its equal in 64 bits
            // too: the same logit and bias
            if (a.bias && r > 0 && !route_apart(last, best)) {
                const float l = route_load(a.logits, row + last_id, a.dtype), b = a.bias[last_id];
                bool unsure = false;
#pragma unroll
                for (int j = 0; j < R; j++)
                    if (place[j] > never && !route_apart(last, place[j]))
                        unsure |= !(x.l[j] == l && a.bias[x.first + j] == b);
                if (__ballot(unsure)) return false;
            }
        }
        if (lane == r && r < a.k) id = won;
        if (lane == who) {
#pragma unroll
            for (int j = 0; j < R; j++)
                if (j == at) place[j] = never;
        }
        last = best;
        last_id = won;
    }
    return true;
}

__device__ __forceinline__ double route_wave_sum(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

template <int R, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_route_wave(RouteArgs a, int n_tok, int LG) {
    const int lane = threadIdx.x & 63;
    const int t = blockIdx.x * WAVES + (int)(threadIdx.x >> 6);
    if (t >= n_tok) return;  // the whole wavefront; no barriers
    const size_t row = (size_t)t * a.stride;
    const float none = -__builtin_inff();
    const int per = a.n_expert / a.n_group, g = lane / LG, e0 = (lane - g * LG) * R;
    RouteLane<R> x;
    x.first = g * per + e0;
    float top = none;
#pragma unroll
    for (int j = 0; j < R; j++) {
        x.l[j] = g < a.n_group && e0 + j < per ? route_load(a.logits, row + x.first + j, a.dtype) : none;
        x.l[j] = x.l[j] > none ? x.l[j] : none;  // (a NaN is not)
        top = fmaxf(top, x.l[j]);
    }
    const bool softmax = a.score == ROUTE_SOFTMAX, keys = a.bias || a.n_group > 1;
    float m = none, inv = 1.0f;
    if (softmax) {
        m = route_wave_max(top);
        if (keys) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < R; j++)
                if (x.l[j] > none) s += x.l[j] == m ? 1.0f : __expf(x.l[j] - m);
            inv = 1.0f / wave_sum(s);
        }
    }
    auto sum64 = [&]() {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < R; j++)
            if (x.l[j] > none) s += route_exp(x.l[j], m);
        return route_wave_sum(s);
    };
    double sum = 1.0;
    if (softmax && !a.renormalise) sum = sum64();
    int id;
    if (!route_choose<float, R>(a, row, x, LG, m, inv, id)) {
        const double total = softmax ? sum64() : 1.0;
        (void)route_choose<double, R>(a, row, x, LG, m, total, id);
    }
    // the weights in 64 bits, a lane each (renormalised, the softmax's divisor
    // leaves them as they are)
    double w = id >= 0 ? route_score(route_load(a.logits, row + max(id, 0), a.dtype), a.score, m, sum) : 0.0;
    if (a.renormalise) {
        const double total = route_wave_sum(w);
        w = total == 0.0 ? 0.0 : w * (double)a.scale / total;
    } else {
        w *= (double)a.scale;
    }
    if (lane < a.k) {
        const size_t at = (size_t)t * a.k + lane;
        a.ids[at] = id;
        a.weights[at] = (float)w;
    }
}

template <int R> static hipError_t route_wave_go(const RouteArgs &a, int n_tok, int LG, hipStream_t s) {
    // a wavefront a workgroup while that leaves CUs to fill
    if (n_tok <= 2048) k_route_wave<R, 1><<<(unsigned)n_tok, 64, 0, s>>>(a, n_tok, LG);
    else k_route_wave<R, 4><<<(unsigned)((n_tok + 3) / 4), 256, 0, s>>>(a, n_tok, LG);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_route(const RouteArgs &a, int n_tok, hipStream_t s) {
    if (n_tok <= 0) return hipSuccess;
    // the fewest experts a lane that bring every group's lanes into a wavefront
    const int per = a.n_expert / a.n_group;
    for (int r = 1; r <= 16; r *= 2) {
        const int LG = (per + r - 1) / r;
        if ((long long)LG * a.n_group > 64) continue;
        switch (r) {
        case 1: return route_wave_go<1>(a, n_tok, LG, s);
        case 2: return route_wave_go<2>(a, n_tok, LG, s);
        case 4: return route_wave_go<4>(a, n_tok, LG, s);
        case 8: return route_wave_go<8>(a, n_tok, LG, s);
        default: return route_wave_go<16>(a, n_tok, LG, s);
        }
    }
    k_route_any<<<(unsigned)n_tok, 256, (size_t)a.n_group * sizeof(double), s>>>(a);
    return hipGetLastError();
}

}  // namespace rsllm_hip
