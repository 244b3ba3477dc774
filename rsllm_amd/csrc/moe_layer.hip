// A mixture-of-experts layer with MXFP4 experts for a few tokens: router, choice,
// gate and up products, SwiGLU, down product, weighted sum.
//
// The weights' codes are widened to bf16 (exactly: a code has two significant bits, a
// scale none), x and h are sums of bf16 terms: one for bf16 x, two for f16, three for
// f32 (8 significant bits each, so 24), so that the products on the matrix cores are
// exact and the sums f32. A term of a token is a column of the 16-wide products.
#include "fp4_common.h"
#include "route_scores.h"

#include <algorithm>
#include <type_traits>

namespace rsllm_hip {

namespace {

constexpr int kMoeMaxExpert = 1024, kMoeMaxShared = 8, kMoeMaxSlots = 40;
constexpr int kMoeMaxPairs = kMoeMaxTok * kMoeMaxSlots, kMoeMaxAll = kMoeMaxExpert + kMoeMaxShared;

size_t pad256(size_t n) { return (n + 255) / 256 * 256; }
__host__ __device__ constexpr int pad128(int n) { return (n + 127) / 128 * 128; }

// What the tokens chose: every token's slots (the k chosen experts, then the shared ones;
// -1: none, or of weight 0), and the jobs: an expert, in rising order, and the tokens that
// take it, a bit each, as many jobs as it takes with at most `cap` tokens.
struct MoePlan {
    int n_jobs;
    uint32_t tokens[kMoeMaxPairs];
    float weight[kMoeMaxPairs];
    int16_t expert[kMoeMaxPairs];
    uint16_t job[kMoeMaxPairs];
};

// The caller's work: logits and scores (f64), x and h as bf16 terms, a flag a token, the plan.
struct MoeWork {
    double *logits;  // [n_tok, n_expert]
    double *scores;  // [n_tok, n_expert], not of softmax
    __bf16 *x;       // [n_tok][3][pad128(n_embd)]
    __bf16 *h;       // [n_tok * (k + n_shared)][3][pad128(n_ff)], weighted
    int *bad;        // [n_tok]: x is not finite
    MoePlan *plan;
};
size_t moe_parts(int n_tok, int n_embd, int n_ff, int n_expert, int k, int n_shared, uint8_t *base, MoeWork *w) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += pad256(bytes);
        return base + here;
    };
    uint8_t *const logits = take((size_t)n_tok * n_expert * 8);
    uint8_t *const scores = take((size_t)n_tok * n_expert * 8);
    uint8_t *const x = take((size_t)n_tok * 3 * pad128(n_embd) * 2);
    uint8_t *const h = take((size_t)n_tok * (k + n_shared) * 3 * pad128(n_ff) * 2);
    uint8_t *const bad = take((size_t)n_tok * 4);
    uint8_t *const plan = take(n_tok ? sizeof(MoePlan) : 0);
    if (w) *w = {reinterpret_cast<double *>(logits), reinterpret_cast<double *>(scores), reinterpret_cast<__bf16 *>(x),
                 reinterpret_cast<__bf16 *>(h), reinterpret_cast<int *>(bad), reinterpret_cast<MoePlan *>(plan)};
    return at;
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

// ---- the router's product -------------------------------------------------------------

// TB tokens' sums over the wavefronts' lanes: lane `i` of the first TB ends up with token i's.
template <int TB> __device__ __forceinline__ double moe_wave_sums(double (&s)[TB]) {
    const int lane = threadIdx.x & 63;
    // the upper half of the lanes takes over the upper half of the sums, and so on
#pragma unroll
    for (int n = TB, off = 32; n > 1; n >>= 1, off >>= 1) {
        const bool up = (lane & off) != 0;
#pragma unroll
        for (int i = 0; i < n / 2; i++) {
            const double mine = up ? s[n / 2 + i] : s[i], other = up ? s[i] : s[n / 2 + i];
            s[i] = mine + __shfl_xor(other, off, 64);
        }
    }
#pragma unroll
    for (int off = 32 / TB; off >= 1; off >>= 1) s[0] += __shfl_xor(s[0], off, 64);
    return s[0];  // of token i at the lanes whose upper bits are i
}

// Logits of expert e for tokens t0 .. t0 + TB - 1 (those behind the last repeat it).
template <uint32_t DX, uint32_t DR, int TB>
__device__ __forceinline__ void moe_logits(const MoeLayerArgs &a, const MoeWork &w, int e, int t0, bool vx, bool vr,
                                           double (*red)[TB]) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    double s[TB];
#pragma unroll
    for (int t = 0; t < TB; t++) s[t] = 0.0;
    for (int i = 8 * tid; i < a.n_embd; i += 8 * 256) {
        float r[8], x[TB][8];
        mx_load8<DR>(a.router, (size_t)e * a.n_embd, i, a.n_embd, vr, r);
#pragma unroll
        for (int t = 0; t < TB; t++)
            mx_load8<DX>(a.x, (size_t)min(t0 + t, a.n_tok - 1) * a.x_stride, i, a.n_embd, vx, x[t]);
#pragma unroll
        for (int t = 0; t < TB; t++)
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (vr || i + k < a.n_embd) s[t] = fma((double)x[t][k], (double)r[k], s[t]);
    }
    const double sum = moe_wave_sums<TB>(s);
    __syncthreads();
    if (lane % (64 / TB) == 0) red[wv][lane / (64 / TB)] = sum;
    __syncthreads();
    if (tid < TB && t0 + tid < a.n_tok) {
        const size_t at = (size_t)(t0 + tid) * a.n_expert + e;
        const double l = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
        w.logits[at] = l;
        if (a.score != ROUTE_SOFTMAX) w.scores[at] = route_score(l, a.score, 0.0, 1.0);
    }
}

}  // namespace

// Workgroup e < n_expert: the 64-bit logits (and scores) of expert e for every token; the others: a
// token's x as bf16 terms, zeros behind it, and whether it is finite.
template <uint32_t DX, uint32_t DR>
__global__ __launch_bounds__(256) void k_moe_in(MoeLayerArgs a, MoeWork w, int vx, int vr) {
    constexpr int kTerms = DX == T_F32 ? 3 : DX == T_F16 ? 2 : 1;
    __shared__ double red1[4][1], red4[4][4];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < a.n_expert) {
        const int e = blockIdx.x;
        if (a.n_tok == 1) {
            moe_logits<DX, DR, 1>(a, w, e, 0, vx, vr, red1);
        } else {
            for (int t0 = 0; t0 < a.n_tok; t0 += 4) moe_logits<DX, DR, 4>(a, w, e, t0, vx, vr, red4);
        }
        return;
    }
    const int t = blockIdx.x - a.n_expert, row = pad128(a.n_embd);
    __bf16 *const dst = w.x + (size_t)t * 3 * row;
    bool ok = true;
    for (int i = 8 * tid; i < row; i += 8 * 256) {
        float v[8];
        mx_load8<DX>(a.x, (size_t)t * a.x_stride, i, a.n_embd, vx, v);
#pragma unroll
        for (int k = 0; k < 8; k++) ok &= finite(v[k]);
#pragma unroll
        for (int j = 0; j < kTerms; j++) {
            mx_bf8 b;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                b[k] = (__bf16)v[k];
                v[k] -= (float)b[k];
            }
            *reinterpret_cast<mx_bf8 *>(dst + j * row + i) = b;
        }
    }
    const int all = __syncthreads_and(ok);
    if (tid == 0) w.bad[t] = !all;
}

namespace {

// ---- the choice -------------------------------------------------------------------------

// A double's place in the order of all doubles as a number (no NaN); -inf: 0x000F...F.
__device__ __forceinline__ uint64_t order64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
// The lane (0..63) that holds the wavefront's largest key, the lowest `id` among equals;
// -1 if no key is above kNever's.
__device__ __forceinline__ int moe_best(uint64_t key, int id) {
    const uint32_t hi = (uint32_t)(key >> 32), lo = (uint32_t)key;
    const uint32_t mh = wave_max_u32(hi);
    const uint32_t ml = wave_max_u32(hi == mh ? lo : 0u);
    const bool in = hi == mh && lo == ml;
    if (((uint64_t)mh << 32 | ml) <= order64(kNever)) return -1;
    const uint32_t mi = wave_max_u32(in ? ~(uint32_t)id : 0u);
    return __ffsll((unsigned long long)__ballot(in && ~(uint32_t)id == mi)) - 1;
}

// A wavefront's choice for token t: ids and weights of its k slots, -1 and 0 where there is
// none, at lane r the r-th. key: n_expert doubles of LDS, gsum: n_group.
__device__ __forceinline__ void moe_choose(const MoeLayerArgs &a, const double *l, const double *scores, double *key, double *gsum, int &id,
                                           float &weight) {
    const int lane = threadIdx.x & 63, per = a.n_expert / a.n_group;
    double m = kNever, sum = 0.0;
    auto score = [&](int e) { return a.score == ROUTE_SOFTMAX ? route_exp(l[e], m) / sum : scores[e]; };
    if (a.score == ROUTE_SOFTMAX) {
        for (int e = lane; e < a.n_expert; e += 64)
            if (l[e] > m) m = l[e];  // (a NaN is not)
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) m = fmax(m, __shfl_xor(m, off, 64));
        for (int e = lane; e < a.n_expert; e += 64)
            if (l[e] > kNever) sum += route_exp(l[e], m);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    }
    for (int e = lane; e < a.n_expert; e += 64) {
        const double le = l[e];
        double p = kNever;
        if (le > kNever) {
            p = a.bias || a.n_group > 1 ? score(e) + (a.bias ? (double)a.bias[e] : 0.0) : le;
            if (!(p > kNever)) p = kNever;
        }
        key[e] = p;
    }
    __builtin_amdgcn_wave_barrier();
    if (a.n_group > 1) {
        for (int g = lane; g < a.n_group; g += 64) {
            double b0 = kNever, b1 = kNever;
            for (int e = g * per; e < (g + 1) * per; e++) {
                const double v = key[e];
                b1 = fmax(b1, fmin(v, b0));
                b0 = fmax(b0, v);
            }
            gsum[g] = a.group_top == 2 && b1 > kNever ? b0 + b1 : b0;
        }
        __builtin_amdgcn_wave_barrier();
        // the topk_group best groups get NaN, the others are left as they are
        for (int r = 0; r < a.topk_group; r++) {
            double v = kNever;
            int i = a.n_group;
            for (int g = lane; g < a.n_group; g += 64) route_best(v, i, gsum[g], g);
            const int who = moe_best(order64(v), i);
            if (who < 0) break;
            if (lane == who) gsum[i] = __builtin_nan("");
            __builtin_amdgcn_wave_barrier();
        }
        for (int e = lane; e < a.n_expert; e += 64) {
            const double g = gsum[e / per];
            if (g == g) key[e] = kNever;
            else if (!a.bias && key[e] > kNever) key[e] = l[e];
        }
        __builtin_amdgcn_wave_barrier();
    }
    // every lane's best of its keys; the one that gives it looks for its next
    double v = kNever;
    int i = a.n_expert;
    for (int e = lane; e < a.n_expert; e += 64) route_best(v, i, key[e], e);
    id = -1;
    for (int r = 0; r < a.k; r++) {
        const int who = moe_best(order64(v), i);
        if (who < 0) break;
        const int best = __shfl(i, who, 64);
        if (lane == r) id = best;
        if (lane == who) {
            key[i] = kNever;
            v = kNever;
            i = a.n_expert;
            for (int e = lane; e < a.n_expert; e += 64) route_best(v, i, key[e], e);
        }
    }
    const double s = id >= 0 ? score(id) : 0.0;
    double total = s;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) total += __shfl_xor(total, off, 64);
    double out = s * (double)a.scale;
    if (a.renormalise) out = total == 0.0 ? 0.0 : out / total;
    weight = id >= 0 ? (float)out : 0.0f;
}

// The whole workgroup's choice for every token, to `plan` in LDS; workgroup 0 writes ids
// and weights, and the plan for the launch that follows. keys: (n_expert + n_group)
// doubles for each of the first `choosers` wavefronts, who choose. takes: a word an expert.
template <int W> __device__ __forceinline__ void moe_plan(const MoeLayerArgs &a, const MoeWork &w, MoePlan &plan, int cap,
                                                          double *keys, uint32_t *takes, int choosers) {
    __shared__ int part[W];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, slots = a.k + a.n_shared;
    const int all = a.n_expert + a.n_shared;
    for (int e = tid; e < all; e += 64 * W)
        takes[e] = e < a.n_expert ? 0u : a.n_tok == 32 ? 0xFFFFFFFFu : (1u << a.n_tok) - 1u;
    __syncthreads();
    double *const key = keys + wv * (a.n_expert + a.n_group);
    for (int t = wv < choosers ? wv : a.n_tok; t < a.n_tok; t += choosers) {
        int id;
        float weight;
        moe_choose(a, w.logits + (size_t)t * a.n_expert, w.scores + (size_t)t * a.n_expert, key, key + a.n_expert, id, weight);
        if (lane < a.k) {
            if (blockIdx.x == 0) {
                a.ids[t * a.k + lane] = id;
                a.weights[t * a.k + lane] = weight;
            }
            const bool on = id >= 0 && weight != 0.0f;
            plan.expert[t * slots + lane] = (int16_t)(on ? id : -1);
            plan.weight[t * slots + lane] = weight;
            if (on) atomicOr(&takes[id], 1u << t);
        } else if (lane < slots) {
            plan.expert[t * slots + lane] = (int16_t)(a.n_expert + lane - a.k);
            plan.weight[t * slots + lane] = 1.0f;
        }
    }
    __syncthreads();
    // the jobs of a run of experts a thread, behind those of the threads before it
    const int run = (all + 64 * W - 1) / (64 * W), e0 = min(all, tid * run), e1 = min(all, e0 + run);
    int n = 0;
    for (int e = e0; e < e1; e++) n += (__popc(takes[e]) + cap - 1) / cap;
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int add = __shfl_up(inc, (unsigned)d, 64);
        if (lane >= d) inc += add;
    }
    if (lane == 63) part[wv] = inc;
    __syncthreads();
    int at = inc - n;
    for (int i = 0; i < wv; i++) at += part[i];
    for (int e = e0; e < e1; e++) {
        for (uint32_t left = takes[e]; left; at++) {
            uint32_t mine = 0;
            for (int i = 0; i < cap && left; i++) {
                mine |= left & -left;
                left &= left - 1;
            }
            plan.job[at] = (uint16_t)e;
            plan.tokens[at] = mine;
        }
    }
    if (tid == 64 * W - 1) plan.n_jobs = at;
    __syncthreads();
}
// As much of a plan as there is, from LDS to memory or back, by a workgroup of N threads.
template <int N> __device__ __forceinline__ void moe_copy_plan(MoePlan &to, const MoePlan &from, int pairs, int n_jobs) {
    for (int i = threadIdx.x; i < pairs; i += N) {
        to.weight[i] = from.weight[i];
        to.expert[i] = from.expert[i];
    }
    for (int i = threadIdx.x; i < n_jobs; i += N) {
        to.job[i] = from.job[i];
        to.tokens[i] = from.tokens[i];
    }
    if (threadIdx.x == 0) to.n_jobs = n_jobs;
}

// ---- the products -----------------------------------------------------------------------
//
// v_mfma_f32_16x16x32_bf16: rows of weights by columns of terms: column c of a job's tile of
// 16 is term c % terms of its (c / terms)-th token (16 / terms of them a tile), columns
// behind its last token bring zeros.

// 512 codes of FR times 16 rows, a lane's 16 codes' bytes of each step of 128 and its row's
// 16 scale bytes.
template <int FR> struct MoePiece {
    uint4 c[FR][4], s[FR];
};
struct MoeRows {
    const uint8_t *c, *s;  // this lane's row
};
template <int FR>
__device__ __forceinline__ void moe_fetch(MoePiece<FR> &p, const MoeRows (&rows)[FR], int i, int steps) {
#pragma unroll
    for (int f = 0; f < FR; f++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            p.c[f][j] = make_uint4(0, 0, 0, 0);
            if (4 * i + j < steps) p.c[f][j] = *reinterpret_cast<const uint4 *>(rows[f].c + 256 * (size_t)i + 64 * j);
        }
        p.s[f] = *reinterpret_cast<const uint4 *>(rows[f].s + 16 * (size_t)i);
    }
}
__device__ __forceinline__ mx_bf8 moe_widen(uint32_t d, float unit) {
    mx_bf8 f;
    const mx_bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, unit, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, unit, 1);
    const mx_bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, unit, 2), e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, unit, 3);
    f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
    f[4] = c[0]; f[5] = c[1]; f[6] = e[0]; f[7] = e[1];
    return f;
}
// acc += the piece's rows times the terms at `at` (bytes; this lane's column and block of
// step 0, beyond the buffer where the column brings zeros) of the first `tiles` tiles.
template <int FR, int NT>
__device__ __forceinline__ void moe_multiply(const MoePiece<FR> &p, __amdgpu_buffer_rsrc_t terms, const uint32_t (&at)[NT],
                                             int tiles, int i, int steps, int blocks, mx_v4f (&acc)[FR][NT]) {
    const int q = (threadIdx.x & 63) >> 4;
    mx_bf8 x[NT][4], next[NT][4];
    auto get = [&](mx_bf8 (&d)[NT][4], int j) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NT; n++)
            if (n < tiles) {
#pragma unroll
                for (int m = 0; m < 4; m++)
                    d[n][m] = __builtin_bit_cast(mx_bf8, bload16(terms, at[n] + 1024u * (uint32_t)i + 256u * (uint32_t)j + 16u * (uint32_t)m, 0));
            }
    };
    get(x, 0);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (4 * i + j >= steps) break;
        if (j < 3) get(next, j + 1);  // (behind the row's end: the next row's, or zeros; not used)
        // (scales behind a row's last block may be anything: there 1)
        const bool in = 16 * i + 4 * j + q < blocks;
        float unit[FR];
#pragma unroll
        for (int f = 0; f < FR; f++) {
            const uint32_t s = j == 0 ? p.s[f].x : j == 1 ? p.s[f].y : j == 2 ? p.s[f].z : p.s[f].w;
            unit[f] = mx_unit(in ? s >> (8 * q) & 255u : 127u);
        }
#pragma unroll
        for (int m = 0; m < 4; m++) {
#pragma unroll
            for (int f = 0; f < FR; f++) {
                const uint4 &c = p.c[f][j];
                const mx_bf8 w = moe_widen(m == 0 ? c.x : m == 1 ? c.y : m == 2 ? c.z : c.w, unit[f]);
#pragma unroll
                for (int n = 0; n < NT; n++)
                    if (n < tiles) acc[f][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[n][m], acc[f][n], 0, 0, 0);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int m = 0; m < 4; m++) x[n][m] = next[n][m];
    }
}
constexpr uint32_t kMoeNone = 0x80000000u;  // an offset beyond any buffer of terms
// The slot of token t that takes expert e (which it does).
__device__ __forceinline__ int moe_slot_of(const MoeLayerArgs &a, const MoePlan &plan, int t, int e) {
    if (e >= a.n_expert) return a.k + e - a.n_expert;
    int at = 0;
    for (int i = 0; i < a.k; i++) at = plan.expert[t * (a.k + a.n_shared) + i] == e ? i : at;
    return at;
}
// The n-th (from 0) bit of a mask, -1 if there are fewer.
__device__ __forceinline__ int moe_token(uint32_t mask, int n) {
    for (int i = 0; i < n; i++) mask &= mask - 1;
    return mask ? __ffs((int)mask) - 1 : -1;
}

constexpr int kUpWaves = 4, kDownWaves = 8, kUpRows = 4;

}  // namespace

// Gate and up products of RU = 8 FR rows of a job a turn, K in pieces of 512 over the
// wavefronts, and the weighted SwiGLU of their sums as bf16 terms. Jobs of at most `cap`
// tokens, NT tiles.
template <int NT> __global__ __launch_bounds__(64 * kUpWaves, 2)
void k_moe_up(MoeLayerArgs a, MoeWork w, int terms, int hterms, int cap, int choosers) {
    constexpr int W = kUpWaves, FR = kUpRows, RU = 8 * FR, H = FR / 2;  // fragments 0 .. H - 1: gate
    extern __shared__ __align__(16) uint8_t smem[];  // keys of the choice, then the wavefronts' sums
    __shared__ MoePlan plan;
    __shared__ uint32_t takes[kMoeMaxAll];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slots = a.k + a.n_shared, ff = a.n_ff, frow = pad128(ff), erow = pad128(a.n_embd);
    moe_plan<W>(a, w, plan, cap, reinterpret_cast<double *>(smem), takes, choosers);
    if (blockIdx.x == 0) moe_copy_plan<64 * W>(*w.plan, plan, a.n_tok * slots, plan.n_jobs);
    const size_t rb = mx_row_bytes(a.n_embd), sb = mx_scale_bytes(a.n_embd);
    const int steps = (int)(rb / 64), pieces = (int)(sb / 16), blocks = (a.n_embd + 31) / 32;
    const int per = (ff + RU - 1) / RU, units = plan.n_jobs * per, tpt = 16 / terms;
    const __amdgpu_buffer_rsrc_t xt = make_rsrc(w.x, (uint32_t)a.n_tok * 3u * (uint32_t)erow * 2u);
    float *const red = reinterpret_cast<float *>(smem);  // [W][FR][NT][64][4]
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int job = u / per, e = plan.job[job], r0 = u % per * RU;
        const uint32_t mask = plan.tokens[job];
        const int count = __popc(mask), tiles = (count + tpt - 1) / tpt;
        uint32_t at[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int t = r < tpt * terms ? moe_token(mask, n * tpt + r / terms) : -1;
            at[n] = t >= 0 ? (uint32_t)((t * 3 + r % terms) * erow + 32 * q) * 2u : kMoeNone;
        }
        MoeRows rows[FR];
#pragma unroll
        for (int f = 0; f < FR; f++) {
            const size_t row = (size_t)e * ff + min(r0 + 16 * (f % H) + r, ff - 1);
            rows[f].c = (f < H ? a.gate : a.up) + row * rb + 16 * q;
            rows[f].s = (f < H ? a.gate_s : a.up_s) + row * sb;
        }
        mx_v4f acc[FR][NT];
#pragma unroll
        for (int f = 0; f < FR; f++)
#pragma unroll
            for (int n = 0; n < NT; n++) acc[f][n] = mx_v4f{0.0f, 0.0f, 0.0f, 0.0f};
        MoePiece<FR> p;
        if (wv < pieces) moe_fetch<FR>(p, rows, wv, steps);
        for (int i = wv; i < pieces; i += W) {
            const MoePiece<FR> now = p;
            if (i + W < pieces) moe_fetch<FR>(p, rows, i + W, steps);
            moe_multiply<FR, NT>(now, xt, at, tiles, i, steps, blocks, acc);
        }
        __syncthreads();  // (the last turn's sums are read)
        mx_v4f *const part = reinterpret_cast<mx_v4f *>(red);
#pragma unroll
        for (int f = 0; f < FR; f++)
#pragma unroll
            for (int n = 0; n < NT; n++)
                if (n < tiles) part[((wv * FR + f) * NT + n) * 64 + lane] = acc[f][n];
        __syncthreads();
        // a thread's row, a token a turn
        const int row = tid % RU, lanes = 16 * ((row & 15) >> 2), k = row & 3;
        for (int n = tid / RU; n < count; n += 64 * W / RU) {
            const int t = moe_token(mask, n), i = moe_slot_of(a, plan, t, e);
            float g = 0.0f, v = 0.0f;
            for (int j = 0; j < terms; j++) {
                const int c = n % tpt * terms + j;
                const float *const src = red + ((row >> 4) * NT + n / tpt) * 256 + (c + lanes) * 4 + k;
#pragma unroll
                for (int x = 0; x < W; x++) {
                    g += src[x * FR * NT * 256];
                    v += src[(x * FR + H) * NT * 256];
                }
            }
            if (a.clamp > 1e-6f) {
                g = g > a.clamp ? a.clamp : g;
                v = v > a.clamp ? a.clamp : v < -a.clamp ? -a.clamp : v;
            }
            float h = r0 + row < ff ? g / (1.0f + expf(-g)) * v * plan.weight[t * slots + i] : 0.0f;
            __bf16 *const dst = w.h + (size_t)(t * slots + i) * 3 * frow + r0 + row;
            for (int j = 0; j < hterms; j++) {
                const __bf16 b = (__bf16)h;
                if (r0 + row < frow) dst[j * frow] = b;
                h = finite(h) ? h - (float)b : 0.0f;
                if (r0 + RU >= ff)  // zeros up to whole steps
                    for (int z = RU; r0 + row + z < frow; z += RU) dst[j * frow + z] = (__bf16)0.0f;
            }
        }
    }
}

// The down products of 16 rows a turn over all jobs, their pieces over the wavefronts, every
// one of which adds its jobs' columns to sums of its own for each token.
template <int NT> __global__ __launch_bounds__(64 * kDownWaves) void k_moe_down(MoeLayerArgs a, MoeWork w, int hterms) {
    constexpr int W = kDownWaves;
    __shared__ MoePlan plan;
    extern __shared__ __align__(16) uint8_t smem[];  // sums [W][n_tok][16]
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slots = a.k + a.n_shared, frow = pad128(a.n_ff), n_jobs = w.plan->n_jobs;
    moe_copy_plan<64 * W>(plan, *w.plan, a.n_tok * slots, n_jobs);
    float *const sums = reinterpret_cast<float *>(smem), *const mine = sums + wv * a.n_tok * 16;
    const size_t rb = mx_row_bytes(a.n_ff), sb = mx_scale_bytes(a.n_ff);
    const int steps = (int)(rb / 64), pieces = (int)(sb / 16), blocks = (a.n_ff + 31) / 32, tpt = 16 / hterms;
    const __amdgpu_buffer_rsrc_t ht = make_rsrc(w.h, (uint32_t)(a.n_tok * slots) * 3u * (uint32_t)frow * 2u);
    const int total = n_jobs * pieces;
    const int from = (int)((long long)total * wv / W), to = (int)((long long)total * (wv + 1) / W);
    for (int r0 = blockIdx.x * 16; r0 < a.n_embd; r0 += gridDim.x * 16) {
        __syncthreads();  // (the plan is there, the last turn's sums are read)
        for (int i = lane; i < a.n_tok * 16; i += 64) mine[i] = 0.0f;
        const size_t row = (size_t)min(r0 + r, a.n_embd - 1);
        MoePiece<1> next;
        auto fetch = [&](int c) __attribute__((always_inline)) {
            if (c < to) {
                const size_t e = plan.job[c / pieces];
                const MoeRows rows[1] = {{a.down + (e * a.n_embd + row) * rb + 16 * q, a.down_s + (e * a.n_embd + row) * sb}};
                moe_fetch<1>(next, rows, c % pieces, steps);
            }
        };
        fetch(from);
        for (int c = from; c < to;) {
            const int job = c / pieces, e = plan.job[job], end = min(to, (job + 1) * pieces);
            const uint32_t mask = plan.tokens[job];
            const int tiles = (__popc(mask) + tpt - 1) / tpt;
            int tok[NT];
            uint32_t at[NT];
            mx_v4f acc[1][NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                tok[n] = r < tpt * hterms ? moe_token(mask, n * tpt + r / hterms) : -1;
                at[n] = tok[n] >= 0 ? (uint32_t)(((tok[n] * slots + moe_slot_of(a, plan, tok[n], e)) * 3 + r % hterms) * frow + 32 * q) * 2u
                                    : kMoeNone;
                acc[0][n] = mx_v4f{0.0f, 0.0f, 0.0f, 0.0f};
            }
            for (; c < end; c++) {
                const MoePiece<1> now = next;
                fetch(c + 1);
                moe_multiply<1, NT>(now, ht, at, tiles, c % pieces, steps, blocks, acc);
            }
            // a token's terms stand in neighbouring lanes: to the first of them, and to its sums
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if (n >= tiles) continue;
                mx_v4f y = acc[0][n];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float v1 = __shfl_down(acc[0][n][k], 1, 64), v2 = __shfl_down(acc[0][n][k], 2, 64);
                    y[k] += hterms == 3 ? v1 + v2 : v1;
                }
                if (tok[n] >= 0 && r % hterms == 0) *reinterpret_cast<mx_v4f *>(mine + tok[n] * 16 + 4 * q) += y;
            }
        }
        __syncthreads();
        for (int i = tid; i < a.n_tok * 16; i += 64 * W) {
            const int t = i >> 4, o = r0 + (i & 15);
            float y = 0.0f;
#pragma unroll
            for (int x = 0; x < W; x++) y += sums[x * a.n_tok * 16 + i];
            if (o < a.n_embd) mx_store(a.out, (size_t)t * a.out_stride + o, w.bad[t] ? __builtin_nanf("") : y, a.dtype_out);
        }
    }
}

size_t moe_layer_work_bytes(int n_tok, int n_embd, int n_ff, int n_expert, int k, int n_shared) {
    return moe_parts(n_tok, n_embd, n_ff, n_expert, k, n_shared, nullptr, nullptr);
}

namespace {

template <uint32_t DX> void moe_in_go(const MoeLayerArgs &a, const MoeWork &w, hipStream_t s) {
    const int size = DX == T_F32 ? 4 : 2, rsize = a.dtype_router == T_F32 ? 4 : 2;
    const int vx = (uintptr_t)a.x % 16 == 0 && a.x_stride * size % 16 == 0;
    const int vr = (uintptr_t)a.router % 16 == 0 && (size_t)a.n_embd * rsize % 16 == 0;
    const dim3 g((unsigned)(a.n_expert + a.n_tok));
    if (a.dtype_router == T_F32) k_moe_in<DX, T_F32><<<g, 256, 0, s>>>(a, w, vx, vr);
    else if (a.dtype_router == T_F16) k_moe_in<DX, T_F16><<<g, 256, 0, s>>>(a, w, vx, vr);
    else k_moe_in<DX, T_BF16><<<g, 256, 0, s>>>(a, w, vx, vr);
}

template <int NT> hipError_t moe_go(const MoeLayerArgs &a, const MoeWork &w, int terms, int hterms, hipStream_t s) {
    const int cap = NT * (16 / std::max(terms, hterms));
    // 48 KB at most for the choice's keys and the sums
    const size_t keys = (size_t)(a.n_expert + a.n_group) * 8, sums = (size_t)kUpWaves * kUpRows * NT * 1024;
    static_assert(kUpWaves * kUpRows * NT <= 48, "LDS");
    const int choosers = (int)std::min((size_t)kUpWaves, (size_t)48 * 1024 / keys);
    const int pairs = a.n_tok * (a.k + a.n_shared);  // at most as many jobs
    const long long units = (long long)pairs * ((a.n_ff + 8 * kUpRows - 1) / (8 * kUpRows));
    k_moe_up<NT><<<(unsigned)std::min(units, (long long)512), 64 * kUpWaves, std::max(choosers * keys, sums), s>>>(
        a, w, terms, hterms, cap, choosers);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_moe_down<NT><<<(unsigned)std::min((a.n_embd + 15) / 16, 512), 64 * kDownWaves, (size_t)kDownWaves * a.n_tok * 64, s>>>(a, w, hterms);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_layer(const MoeLayerArgs &a, uint8_t *work, hipStream_t s) {
    if (a.n_tok <= 0) return hipSuccess;
    MoeWork w;
    moe_parts(a.n_tok, a.n_embd, a.n_ff, a.n_expert, a.k, a.n_shared, work, &w);
    const int terms = a.dtype_x == T_F32 ? 3 : a.dtype_x == T_F16 ? 2 : 1, hterms = a.dtype_out == T_F32 ? 3 : 2;
    if (a.dtype_x == T_F32) moe_in_go<T_F32>(a, w, s);
    else if (a.dtype_x == T_F16) moe_in_go<T_F16>(a, w, s);
    else moe_in_go<T_BF16>(a, w, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // one tile where it holds every token
    return a.n_tok <= 16 / std::max(terms, hterms) ? moe_go<1>(a, w, terms, hterms, s) : moe_go<2>(a, w, terms, hterms, s);
}

}  // namespace rsllm_hip
