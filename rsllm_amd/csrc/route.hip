// Expert routing: router logits -> the ids and weights of each token's experts.
//
// Scores, keys and group sums are 64-bit, so which of two near experts is
// chosen does not hang on a 32-bit rounding of exp; the weights are rounded
// once at the end. An expert's place in the order is its key (score + bias), or
// its logit itself where there is no bias (the scores rise with the logits);
// equal places go to the lower id.
#include "kernels.h"

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

hipError_t launch_moe_route(const RouteArgs &a, int n_tok, hipStream_t s) {
    if (n_tok <= 0) return hipSuccess;
    k_route_any<<<(unsigned)n_tok, 256, (size_t)a.n_group * sizeof(double), s>>>(a);
    return hipGetLastError();
}

}  // namespace rsllm_hip
