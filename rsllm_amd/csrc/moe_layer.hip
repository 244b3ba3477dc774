// A mixture-of-experts layer with MXFP4 experts for a few tokens: router, choice,
// gate and up products, SwiGLU, down product, weighted sum.
//
// The weights' codes are widened to bf16 (exactly: a code has two significant bits, a
// scale none), x and h are sums of bf16 terms: one for bf16 x, two for f16, three for
// f32 (8 significant bits each, so 24), so that the products on the matrix cores are
// exact and the sums f32.
#include "fp4_common.h"
#include "route_scores.h"

#include <algorithm>

namespace rsllm_hip {

namespace {

size_t pad256(size_t n) { return (n + 255) / 256 * 256; }
__host__ __device__ inline int pad128(int n) { return (n + 127) / 128 * 128; }

// The caller's work: logits (f64), x and h as bf16 terms, a flag a token.
struct MoeWork {
    double *logits;  // [n_tok, n_expert]
    __bf16 *x;       // [n_tok][3][pad128(n_embd)]
    __bf16 *h;       // [n_tok * (k + n_shared)][3][pad128(n_ff)], weighted
    int *bad;        // [n_tok]: x is not finite
};
size_t moe_parts(int n_tok, int n_embd, int n_ff, int n_expert, int k, int n_shared, uint8_t *base, MoeWork *w) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += pad256(bytes);
        return base + here;
    };
    uint8_t *const logits = take((size_t)n_tok * n_expert * 8);
    uint8_t *const x = take((size_t)n_tok * 3 * pad128(n_embd) * 2);
    uint8_t *const h = take((size_t)n_tok * (k + n_shared) * 3 * pad128(n_ff) * 2);
    uint8_t *const bad = take((size_t)n_tok * 4);
    if (w) *w = {reinterpret_cast<double *>(logits), reinterpret_cast<__bf16 *>(x), reinterpret_cast<__bf16 *>(h),
                 reinterpret_cast<int *>(bad)};
    return at;
}

template <uint32_t DT> constexpr int kTerms = DT == T_F32 ? 3 : DT == T_F16 ? 2 : 1;

__device__ __forceinline__ float moe_load(const void *p, size_t i, uint32_t dtype) {
    return dtype == T_F32 ? mx_load<T_F32>(p, i) : dtype == T_F16 ? mx_load<T_F16>(p, i) : mx_load<T_BF16>(p, i);
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }

// f64 counterparts of the routing's scores.
__device__ __forceinline__ double route_exp(double l, double m) { return l == m ? 1.0 : route_exp64(l - m); }
__device__ __forceinline__ double route_score(double l, int score, double m, double sum) {
    if (score == ROUTE_SOFTMAX) return route_exp(l, m) / sum;
    const double e = route_exp64(score == ROUTE_SIGMOID ? -l : -fabs(l));
    if (score == ROUTE_SIGMOID) return 1.0 / (1.0 + e);
    return sqrt(fmax(l, 0.0) + route_log1p(e));
}

}  // namespace

// Workgroup e < n_expert: the 64-bit logits of expert e for every token; the others: a
// token's x as bf16 terms, zeros behind it, and whether it is finite.
__global__ __launch_bounds__(256) void k_moe_in(MoeLayerArgs a, MoeWork w, int terms) {
    __shared__ double red[4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    if ((int)blockIdx.x < a.n_expert) {
        const int e = blockIdx.x;
        for (int t = 0; t < a.n_tok; t++) {
            double s = 0.0;
            for (int i = tid; i < a.n_embd; i += 256)
                s = fma((double)moe_load(a.x, (size_t)t * a.x_stride + i, a.dtype_x),
                        (double)moe_load(a.router, (size_t)e * a.n_embd + i, a.dtype_router), s);
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
            __syncthreads();
            if (lane == 0) red[wv] = s;
            __syncthreads();
            if (tid == 0) w.logits[(size_t)t * a.n_expert + e] = (red[0] + red[1]) + (red[2] + red[3]);
        }
        return;
    }
    const int t = blockIdx.x - a.n_expert, row = pad128(a.n_embd);
    __bf16 *const dst = w.x + (size_t)t * 3 * row;
    bool ok = true;
    for (int i = tid; i < row; i += 256) {
        float v = i < a.n_embd ? moe_load(a.x, (size_t)t * a.x_stride + i, a.dtype_x) : 0.0f;
        ok &= finite(v);
        for (int j = 0; j < terms; j++) {
            const __bf16 b = (__bf16)v;
            dst[j * row + i] = b;
            v -= (float)b;
        }
    }
    const int all = __syncthreads_and(ok);
    if (tid == 0) w.bad[t] = !all;
}

// A workgroup a token: the experts with the best places, one after the other, as
// k_route_any, from 64-bit logits.
__global__ __launch_bounds__(256) void k_moe_choose(MoeLayerArgs a, MoeWork w) {
    __shared__ double key[1024], gsum[1024], score[32], red_v[4];
    __shared__ int red_i[4], chosen[32];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const double *const l = w.logits + (size_t)t * a.n_expert;
    const int per = a.n_expert / a.n_group;
    auto block_best = [&](double v, int i, double &bv, int &bi) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) route_best(v, i, __shfl_xor(v, off, 64), __shfl_xor(i, off, 64));
        __syncthreads();
        if (lane == 0) {
            red_v[wv] = v;
            red_i[wv] = i;
        }
        __syncthreads();
        bv = red_v[0];
        bi = red_i[0];
        for (int k = 1; k < 4; k++) route_best(bv, bi, red_v[k], red_i[k]);
    };
    double m = kNever, sum = 0.0;
    if (a.score == ROUTE_SOFTMAX) {
        double v = kNever;
        int bi;
        for (int e = tid; e < a.n_expert; e += 256)
            if (l[e] > v) v = l[e];
        block_best(v, 0, m, bi);
        double s = 0.0;
        for (int e = tid; e < a.n_expert; e += 256)
            if (l[e] > kNever) s += route_exp(l[e], m);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
        __syncthreads();
        if (lane == 0) red_v[wv] = s;
        __syncthreads();
        sum = (red_v[0] + red_v[1]) + (red_v[2] + red_v[3]);
    }
    for (int e = tid; e < a.n_expert; e += 256) {
        double p = kNever;
        if (l[e] > kNever) {
            p = a.bias || a.n_group > 1 ? route_score(l[e], a.score, m, sum) + (a.bias ? (double)a.bias[e] : 0.0) : l[e];
            if (!(p > kNever)) p = kNever;
        }
        key[e] = p;
    }
    __syncthreads();
    if (a.n_group > 1) {
        for (int g = tid; g < a.n_group; g += 256) {
            double b0 = kNever, b1 = kNever;
            for (int e = g * per; e < (g + 1) * per; e++) {
                const double v = key[e];
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
            if (!(bv > kNever)) break;
            if (tid == 0) gsum[bi] = __builtin_nan("");
            __syncthreads();
        }
        for (int e = tid; e < a.n_expert; e += 256) {
            const double g = gsum[e / per];
            if (g == g) key[e] = kNever;
            else if (!a.bias && key[e] > kNever) key[e] = l[e];
        }
        __syncthreads();
    }
    int found = 0;
    for (int r = 0; r < a.k; r++) {
        double v = kNever, bv;
        int i = a.n_expert, bi;
        for (int e = tid; e < a.n_expert; e += 256) route_best(v, i, key[e], e);
        block_best(v, i, bv, bi);
        if (!(bv > kNever)) break;
        if (tid == 0) {
            chosen[r] = bi;
            score[r] = route_score(l[bi], a.score, m, sum);
            key[bi] = kNever;
        }
        found = r + 1;
        __syncthreads();
    }
    if (tid < a.k) {
        const size_t at = (size_t)t * a.k + tid;
        double v = 0.0, total = 0.0;
        if (tid < found) {
            for (int r = 0; r < found; r++) total += score[r];
            v = score[tid] * (double)a.scale;
            if (a.renormalise) v = total == 0.0 ? 0.0 : v / total;
        }
        a.ids[at] = tid < found ? chosen[tid] : -1;
        a.weights[at] = (float)v;
    }
}

namespace {

// The expert and weight of a token's slot i (those behind the k-th: the shared ones);
// false where there is none.
__device__ __forceinline__ bool moe_slot(const MoeLayerArgs &a, int t, int i, int &e, float &wt) {
    if (i >= a.k) {
        e = a.n_expert + i - a.k;
        wt = 1.0f;
        return true;
    }
    e = a.ids[t * a.k + i];
    wt = a.weights[t * a.k + i];
    return e >= 0 && wt != 0.0f;
}

// Rows r0 .. r0 + 15 of a code matrix (n rows of `in` from `codes`) times the `terms` rows
// of v, summed over steps st0, st0 + by, ..: the matrix cores' 16 x 16 sums.
__device__ __forceinline__ void moe_rows(const uint8_t *codes, const uint8_t *scales, int r0, int n, int in,
                                         const __bf16 *v, int terms, int st0, int by, mx_v4f &acc) {
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, blocks = (in + 31) / 32, row = pad128(in);
    const size_t rb = mx_row_bytes(in), sb = mx_scale_bytes(in), at = (size_t)min(r0 + r, n - 1);
    const __bf16 *const col = v + (size_t)min(r, terms - 1) * row;
    for (int st = st0; st < row / 128; st += by) {
        const int b = 4 * st + q;
        const uint4 c = *reinterpret_cast<const uint4 *>(codes + at * rb + 16 * (size_t)b);
        const float unit = mx_unit(b < blocks ? scales[at * sb + b] : 127u);
        const uint32_t d[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            mx_bf8 f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                mx_bf2 p;
                if (i == 0) p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[j], unit, 0);
                else if (i == 1) p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[j], unit, 1);
                else if (i == 2) p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[j], unit, 2);
                else p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[j], unit, 3);
                f[2 * i] = p[0];
                f[2 * i + 1] = p[1];
            }
            const mx_bf8 x = *reinterpret_cast<const mx_bf8 *>(col + 32 * b + 8 * j);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, x, acc, 0, 0, 0);
        }
    }
}

// The sum over the first `terms` of every 16 lanes (columns), at column 0's lane.
__device__ __forceinline__ float moe_terms(float v, int terms) {
    const float b = __shfl_down(v, 1, 64), c = __shfl_down(v, 2, 64);
    return terms == 3 ? v + (b + c) : terms == 2 ? v + b : v;
}

}  // namespace

// A wavefront per token, slot and 16 rows of gate and up.
__global__ __launch_bounds__(64) void k_moe_up(MoeLayerArgs a, MoeWork w, int terms, int hterms) {
    const int lane = threadIdx.x, slots = a.k + a.n_shared, t = blockIdx.y / slots, i = blockIdx.y % slots;
    int e;
    float wt;
    if (!moe_slot(a, t, i, e, wt)) return;  // the whole wavefront
    const int r0 = blockIdx.x * 16, ff = a.n_ff, frow = pad128(ff), erow = pad128(a.n_embd);
    const size_t rb = mx_row_bytes(a.n_embd), sb = mx_scale_bytes(a.n_embd), base = (size_t)e * ff;
    mx_v4f g = {0, 0, 0, 0}, u = {0, 0, 0, 0};
    moe_rows(a.gate + base * rb, a.gate_s + base * sb, r0, ff, a.n_embd, w.x + (size_t)t * 3 * erow, terms, 0, 1, g);
    moe_rows(a.up + base * rb, a.up_s + base * sb, r0, ff, a.n_embd, w.x + (size_t)t * 3 * erow, terms, 0, 1, u);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        float gv = moe_terms(g[k], terms), uv = moe_terms(u[k], terms);
        const int r = r0 + 4 * (lane >> 4) + k;
        if ((lane & 15) == 0 && r < frow) {
            if (a.clamp > 1e-6f) {
                gv = gv > a.clamp ? a.clamp : gv;
                uv = uv > a.clamp ? a.clamp : uv < -a.clamp ? -a.clamp : uv;
            }
            float h = r < ff ? gv / (1.0f + expf(-gv)) * uv * wt : 0.0f;
            __bf16 *const dst = w.h + (size_t)blockIdx.y * 3 * frow + r;
            for (int j = 0; j < hterms; j++) {
                const __bf16 b = (__bf16)h;
                dst[j * frow] = b;
                h = finite(h) ? h - (float)b : 0.0f;
            }
        }
    }
}

// A wavefront per token and 16 rows of down, over the token's slots.
__global__ __launch_bounds__(64) void k_moe_down(MoeLayerArgs a, MoeWork w, int hterms) {
    const int lane = threadIdx.x, slots = a.k + a.n_shared, t = blockIdx.y;
    const int r0 = blockIdx.x * 16, frow = pad128(a.n_ff);
    const size_t rb = mx_row_bytes(a.n_ff), sb = mx_scale_bytes(a.n_ff);
    mx_v4f y = {0, 0, 0, 0};
    for (int i = 0; i < slots; i++) {
        int e;
        float wt;
        if (!moe_slot(a, t, i, e, wt)) continue;
        const size_t base = (size_t)e * a.n_embd;
        moe_rows(a.down + base * rb, a.down_s + base * sb, r0, a.n_embd, a.n_ff,
                 w.h + ((size_t)t * slots + i) * 3 * frow, hterms, 0, 1, y);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float v = moe_terms(y[k], hterms);
        const int r = r0 + 4 * (lane >> 4) + k;
        if ((lane & 15) == 0 && r < a.n_embd)
            mx_store(a.out, (size_t)t * a.out_stride + r, w.bad[t] ? __builtin_nanf("") : v, a.dtype_out);
    }
}

size_t moe_layer_work_bytes(int n_tok, int n_embd, int n_ff, int n_expert, int k, int n_shared) {
    return moe_parts(n_tok, n_embd, n_ff, n_expert, k, n_shared, nullptr, nullptr);
}

hipError_t launch_moe_layer(const MoeLayerArgs &a, uint8_t *work, hipStream_t s) {
    if (a.n_tok <= 0) return hipSuccess;
    MoeWork w;
    moe_parts(a.n_tok, a.n_embd, a.n_ff, a.n_expert, a.k, a.n_shared, work, &w);
    const int terms = a.dtype_x == T_F32 ? 3 : a.dtype_x == T_F16 ? 2 : 1, hterms = a.dtype_out == T_F32 ? 3 : 2;
    k_moe_in<<<a.n_expert + a.n_tok, 256, 0, s>>>(a, w, terms);
    k_moe_choose<<<a.n_tok, 256, 0, s>>>(a, w);
    k_moe_up<<<dim3((unsigned)(pad128(a.n_ff) / 16), (unsigned)(a.n_tok * (a.k + a.n_shared))), 64, 0, s>>>(a, w, terms, hterms);
    k_moe_down<<<dim3((unsigned)((a.n_embd + 15) / 16), (unsigned)a.n_tok), 64, 0, s>>>(a, w, hterms);
    return hipGetLastError();
}

}  // namespace rsllm_hip
