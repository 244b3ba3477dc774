// Log-probability, rank, entropy and most likely alternatives of each row of
// vocabulary logits.
//   m = max l, S = sum exp(l - m), D = sum exp(l - m) (l - m)
//   logprob = l_tok - m - log S,  entropy = log S - D / S
#include "kernels.h"

namespace rsllm_hip {

namespace {

__device__ __forceinline__ float lp_load(const void *p, size_t i, uint32_t dtype) {
    if (dtype == T_F32) return static_cast<const float *>(p)[i];
    const uint16_t b = static_cast<const uint16_t *>(p)[i];
    return dtype == T_F16 ? f16_to_f32(b) : __builtin_bit_cast(float, (uint32_t)b << 16);
}

constexpr float kInf = __builtin_inff();

// l - m; the limit 0 where both are +inf.
__device__ __forceinline__ float lp_diff(float l, float m) { return l == m ? 0.0f : l - m; }

}  // namespace

// One workgroup per row; every listed alternative is one more look through the
// row.
__global__ __launch_bounds__(256) void k_logprobs_row(LogprobArgs a) {
    __shared__ float red[4][3];
    __shared__ int red_i[4][2];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const size_t row = (size_t)t * a.stride;
    const int tok = a.tokens ? a.tokens[t] : -1;
    const bool has = tok >= 0 && tok < a.vocab;
    const float mine = has ? lp_load(a.logits, row + tok, a.dtype) : 0.0f;

    auto best = [&](float v, int i, float &bv, int &bi) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            const float v2 = __shfl_xor(v, off, 64);
            const int i2 = __shfl_xor(i, off, 64);
            if (v2 > v || (v2 == v && i2 < i)) {
                v = v2;
                i = i2;
            }
        }
        __syncthreads();
        if (lane == 0) {
            red[wv][0] = v;
            red_i[wv][0] = i;
        }
        __syncthreads();
        bv = red[0][0];
        bi = red_i[0][0];
        for (int w = 1; w < 4; w++)
            if (red[w][0] > bv || (red[w][0] == bv && red_i[w][0] < bi)) {
                bv = red[w][0];
                bi = red_i[w][0];
            }
    };

    float v = -kInf, m;
    int above = 0, bad = 0, unused;
    for (int i = tid; i < a.vocab; i += 256) {
        const float l = lp_load(a.logits, row + i, a.dtype);
        if (l > v) v = l;
        above += has && l > mine ? 1 : 0;
        bad |= l != l ? 1 : 0;
    }
    best(v, 0, m, unused);
    float s = 0.0f, d = 0.0f;
    for (int i = tid; i < a.vocab; i += 256) {
        const float l = lp_load(a.logits, row + i, a.dtype);
        if (l > -kInf) {
            const float x = lp_diff(l, m), e = __expf(x);
            s += e;
            if (e > 0.0f) d += e * x;
        }
    }
    s = wave_sum(s);
    d = wave_sum(d);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        above += __shfl_xor(above, off, 64);
        bad |= __shfl_xor(bad, off, 64);
    }
    __syncthreads();
    if (lane == 0) {
        red[wv][1] = s;
        red[wv][2] = d;
        red_i[wv][0] = above;
        red_i[wv][1] = bad;
    }
    __syncthreads();
    s = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
    d = (red[0][2] + red[1][2]) + (red[2][2] + red[3][2]);
    above = red_i[0][0] + red_i[1][0] + red_i[2][0] + red_i[3][0];
    bad = red_i[0][1] | red_i[1][1] | red_i[2][1] | red_i[3][1];
    __syncthreads();
    const bool none = m == -kInf;  // nothing but -inf (and NaN)
    const float log_s = none ? 0.0f : logf(s), nan = __builtin_nanf("");
    auto logprob = [&](float l) { return bad ? nan : none ? -kInf : lp_diff(l, m) - log_s; };
    if (tid == 0) {
        if (a.tokens) {
            a.logprob[t] = has ? logprob(mine) : nan;
            if (a.rank) a.rank[t] = has && mine == mine ? above + 1 : 0;
        }
        if (a.entropy) a.entropy[t] = bad ? nan : none ? 0.0f : log_s - d / s;
    }
    float last = kInf;
    int last_i = -1;
    for (int r = 0; r < a.n_top; r++) {
        float bv = -kInf, cv;
        int bi = a.vocab, ci;
        for (int i = tid; i < a.vocab; i += 256) {
            const float l = lp_load(a.logits, row + i, a.dtype);
            if ((l < last || (l == last && i > last_i)) && l > bv) {
                bv = l;
                bi = i;
            }
        }
        best(bv, bi, cv, ci);
        const bool empty = !(cv > -kInf);
        if (tid == 0) {
            a.top_ids[(size_t)t * a.n_top + r] = empty ? -1 : ci;
            a.top_logprobs[(size_t)t * a.n_top + r] = empty ? (bad ? nan : -kInf) : logprob(cv);
        }
        last = cv;
        last_i = ci;
    }
}

size_t logprobs_scratch_bytes(int n_tok, int vocab, int n_top) { return 0; }

hipError_t launch_logprobs(const LogprobArgs &a, uint8_t *work, int n_tok, hipStream_t s) {
    if (n_tok <= 0) return hipSuccess;
    k_logprobs_row<<<(unsigned)n_tok, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace rsllm_hip
