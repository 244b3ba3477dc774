// A mixture-of-experts layer with MXFP4 experts for a few tokens: router, choice,
// gate and up products, SwiGLU, down product, weighted sum.
//
// The weights' codes are widened to bf16 (exactly: a code has two significant bits, a
// scale none; codes of scales 253 and 254 can be infinite there, which moe_again mends), x and
// h are sums of bf16 terms: one for bf16 x, two for f16, three for f32 (8 significant bits
// each, so 24), so that the products on the matrix cores are exact and the sums f32. A term of
// a token is a column of the 16-wide products. The second and third terms are held times 2^7
// and 2^15, and their columns' sums divided by it: bf16 has nothing below 2^-133, where the
// low bits of small numbers lie.
//
// The chosen experts' weights bound everything. An expert's are read once a job, which holds 16
// / terms of its tokens in the up kernel (5 of f32 x) and three or four in the down kernel: once
// where experts are many and tokens few, seven and eleven times for an expert that 32 tokens of
// f32 take. (8 of 8 experts of the layer below, 32 tokens, take 212 us for 107 MB, 8 of 64 294 for
// 843.) 98 MB for one token of a 4096-wide layer with n_ff 2048, 6 of 256 experts and a shared
// one, 1.83 GB for 32 (137 experts). Three launches (four beyond 8 tokens): 42.7 us and 408 us,
// of which the up kernel is 25.5 and 235 (63 MB and 1.2 GB: 2.5 and 5.2 TB/s), the down kernel
// 13.6 and 146 (31 and 610 MB: 2.3 and 4.2 TB/s), the router 4.9 and 18. A launch that only reads
// gets 4.3 TB/s of 31 MB and 5.7 of 400. One token's up kernel is a chain before the stream, which takes 12 us
// of it: the choice 4 us, its jobs 1, the first loads; and behind it 3 us for the last sums.
#include "fp4_common.h"
#include "route_scores.h"

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

namespace rsllm_hip {

namespace {

constexpr int kInWaves = 16, kWaves = 8;
constexpr int kBatch = 4;  // turns of the up kernel finished at once
// Tokens (one a wavefront) and experts (keys in registers) up to which the up kernel's
// workgroups make the choice for themselves, in place of a launch: 47.0 against 48.7 us for
// one token of a 4096-wide layer of 256 experts, 168.0 against 169.7 for eight. From nine on
// a wavefront has two tokens to choose for: 284 against 283 us for 16.
constexpr int kChooseTok = kWaves, kChooseExperts = 256;
// Columns of a job of the down kernel: three tokens of three terms, four of two. An expert's
// rows are read again for more: with three columns 465 us for 32 tokens of the layer above,
// with six 431, with nine 422, with twelve 421 (and 169.3 and 170.0 with the last two for
// eight tokens).
constexpr int kDownColumns = 9;
constexpr int kMoeMaxExpert = 1024, kMoeMaxShared = 8, kMoeMaxSlots = 40;
constexpr int kMoeMaxPairs = kMoeMaxTok * kMoeMaxSlots, kMoeMaxAll = kMoeMaxExpert + kMoeMaxShared;

size_t pad256(size_t n) { return (n + 255) / 256 * 256; }
__host__ __device__ constexpr int pad128(int n) { return (n + 127) / 128 * 128; }

// What the tokens chose, in LDS: every token's slots (the k chosen experts, then the shared
// ones; -1: none, or of weight 0), and the jobs: an expert and the tokens that take it, a bit
// each, as many jobs as it takes with at most `cap` tokens, experts in rising order (one
// token's in the order of its slots).
struct MoePlan {
    int n_jobs;
    uint32_t tokens[kMoeMaxPairs];
    float weight[kMoeMaxPairs];
    int16_t expert[kMoeMaxPairs];
    uint16_t job[kMoeMaxPairs];
    uint32_t takes[kMoeMaxAll];
};

// The caller's work: logits and scores (f64), x and h as bf16 terms, a flag a token.
struct MoeWork {
    double *logits;  // [n_tok, n_expert]
    double *scores;  // [n_tok, n_expert], not of softmax
    __bf16 *x;       // [n_tok][3][pad128(n_embd)]
    __bf16 *h;       // [n_tok * (k + n_shared)][3][pad128(n_ff)], weighted
    int *bad;        // [n_tok]: x is not finite
    float *part;     // [parts][n_tok][n_embd]: the down kernel's sums, if more than one
};
// Parts of the jobs that workgroups of the down kernel take for each 16 rows: one, unless so
// few rows leave half of the chip idle and a wavefront would still have four items of
// each part (if every token chose experts of its own). The sums then take a launch more, 4
// to 5 us: in all 23 in place of 90 us for 22 tokens of a 408-wide layer with n_ff 2687 (8 of
// 32 experts, 9 parts), 24 in place of 28 for 8 tokens of 2048 / 1024 (8 of 128, 2 parts). Below
// that a launch costs what it saves: 4 tokens of 1536 / 768 (6 of 64) take 13 undivided.
int moe_down_parts(int n_tok, int n_embd, int n_ff, int slots) {
    const long long tiles = (n_embd + 15) / 16, pieces = (long long)mx_scale_bytes(n_ff) / 16;
    const long long most = std::min(256 / std::min(tiles, 256ll), 16ll);
    return (int)std::max(1ll, std::min(most, n_tok * slots * pieces / (4 * kWaves)));
}
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
    const int parts = moe_down_parts(n_tok, n_embd, n_ff, k + n_shared);
    uint8_t *const part = take(parts > 1 ? (size_t)parts * n_tok * n_embd * 4 : 0);
    if (w) *w = {reinterpret_cast<double *>(logits), reinterpret_cast<double *>(scores), reinterpret_cast<__bf16 *>(x),
                 reinterpret_cast<__bf16 *>(h), reinterpret_cast<int *>(bad), reinterpret_cast<float *>(part)};
    return at;
}

constexpr float kFltMax = 0x1.fffffep127f, kBf16Max = 0x1.fep127f;
// What a sum of term j's is multiplied by. (2^7 and 2^15, not 2^8 and 2^16: a held term is
// then no larger than the first one, so no sum overflows before its number does.)
__device__ __forceinline__ constexpr float moe_unit_of(int j) { return j == 0 ? 1.0f : j == 1 ? 0x1p-7f : 0x1p-15f; }
// From what is left behind term j to the next one.
__device__ __forceinline__ constexpr float moe_next(int j) { return j == 0 ? 0x1p7f : 0x1p8f; }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }
// The first eight significant bits of v, cut off and not rounded: rounded, what lies above
// bf16's largest number would be an infinity.
__device__ __forceinline__ __bf16 moe_cut(float v) {
    return __builtin_bit_cast(__bf16, (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16));
}

// f64 counterparts of the routing's scores.
__device__ __forceinline__ double route_exp(double l, double m) { return l == m ? 1.0 : route_exp64(l - m); }
__device__ __forceinline__ double route_score(double l, int score, double m, double sum) {
    if (score == ROUTE_SOFTMAX) return route_exp(l, m) / sum;
    const double e = route_exp64(score == ROUTE_SIGMOID ? -l : -fabs(l));
    if (score == ROUTE_SIGMOID) return 1.0 / (1.0 + e);
    return sqrt(fmax(l, 0.0) + route_log1p(e));
}

// ---- the router's product -------------------------------------------------------------

// N sums over the lanes of a wavefront: the upper half of the lanes (bit OFF) takes over the
// upper half of the sums, and so on, so lanes whose upper bits are i end up with sum i.
template <int N, int OFF, int TB> __device__ __forceinline__ void moe_halve(double (&s)[TB]) {
    if constexpr (N > 1) {
        const bool up = (threadIdx.x & OFF) != 0;
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const double mine = up ? s[N / 2 + i] : s[i], other = up ? s[i] : s[N / 2 + i];
            s[i] = mine + __shfl_xor(other, OFF, 64);
        }
        moe_halve<N / 2, OFF / 2>(s);
    } else if constexpr (OFF > 0) {
        s[0] += __shfl_xor(s[0], OFF, 64);
        moe_halve<1, OFF / 2>(s);
    }
}

// Part `part` of `parts` of expert e's logits for tokens t0 .. t0 + TB - 1 (those behind the
// last repeat it), a wavefront's work, to red[token][part].
template <uint32_t DX, uint32_t DR, int TB>
__device__ __forceinline__ void moe_logits(const MoeLayerArgs &a, int e, int t0, int part, int parts, bool vx, bool vr,
                                           double (*red)[kInWaves]) {
    const int lane = threadIdx.x & 63;
    double s[TB];
#pragma unroll
    for (int t = 0; t < TB; t++) s[t] = 0.0;
    for (int i = 512 * part + 8 * lane; i < a.n_embd; i += 512 * parts) {
        float r[8], x[TB][8];
        mx_load8<DR>(a.router, (size_t)e * a.n_embd, i, a.n_embd, vr, r);
#pragma unroll
        for (int t = 0; t < TB; t++)
            mx_load8<DX>(a.x, (size_t)min(t0 + t, a.n_tok - 1) * a.x_stride, i, a.n_embd, vx, x[t]);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const double rk = (double)r[k];  // (behind the row's end both are 0)
#pragma unroll
            for (int t = 0; t < TB; t++) s[t] = fma((double)x[t][k], rk, s[t]);
        }
    }
    moe_halve<TB, 32>(s);
    if (lane % (64 / TB) == 0) red[t0 + lane / (64 / TB)][part] = s[0];
}

}  // namespace

// Workgroup e < n_expert: the 64-bit logits (and scores) of expert e for every token, groups
// of up to 8 tokens and parts of K over the wavefronts (4096-wide, 256 experts: 4.9 us for one
// token, which is the latency of one chain; 18 for 32, whose rows every workgroup reads again,
// 134 MB from L2, and widens to 64 bits); the others: a token's x as bf16
// terms, zeros behind it, and whether it is finite.
template <uint32_t DX, uint32_t DR>
__global__ __launch_bounds__(64 * kInWaves) void k_moe_in(MoeLayerArgs a, MoeWork w, int vx, int vr) {
    constexpr int kTerms = DX == T_F32 ? 3 : DX == T_F16 ? 2 : 1;
    __shared__ double red[kMoeMaxTok][kInWaves];
    const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    if ((int)blockIdx.x < a.n_expert) {
        const int e = blockIdx.x, groups = a.n_tok <= 8 ? 1 : a.n_tok <= 16 ? 2 : 4, parts = kInWaves / groups;
        if (a.n_tok == 1) moe_logits<DX, DR, 1>(a, e, 0, wv, parts, vx, vr, red);
        else if (a.n_tok <= 4) moe_logits<DX, DR, 4>(a, e, 0, wv, parts, vx, vr, red);
        else moe_logits<DX, DR, 8>(a, e, wv / parts * 8, wv % parts, parts, vx, vr, red);
        __syncthreads();
        if (tid < a.n_tok) {
            double l = 0.0;
            for (int i = 0; i < parts; i++) l += red[tid][i];
            const size_t at = (size_t)tid * a.n_expert + e;
            w.logits[at] = l;
            if (a.score != ROUTE_SOFTMAX) w.scores[at] = route_score(l, a.score, 0.0, 1.0);
        }
        return;
    }
    const int t = blockIdx.x - a.n_expert, row = pad128(a.n_embd);
    __bf16 *const dst = w.x + (size_t)t * 3 * row;
    bool ok = true;
    for (int i = 8 * tid; i < row; i += 8 * 64 * kInWaves) {
        float v[8];
        mx_load8<DX>(a.x, (size_t)t * a.x_stride, i, a.n_embd, vx, v);
#pragma unroll
        for (int k = 0; k < 8; k++) ok &= finite(v[k]);
#pragma unroll
        for (int j = 0; j < kTerms; j++) {
            mx_bf8 b;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                b[k] = moe_cut(v[k]);
                v[k] = (v[k] - (float)b[k]) * moe_next(j);
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
    bool in = hi == mh;
    unsigned long long who = __ballot(in);
    if (who & (who - 1)) {  // rarely: the lower halves, then the ids
        const uint32_t ml = wave_max_u32(in ? lo : 0u);
        in = in && lo == ml;
        who = __ballot(in);
        if (who & (who - 1)) {
            const uint32_t mi = wave_max_u32(in ? ~(uint32_t)id : 0u);
            who = __ballot(in && ~(uint32_t)id == mi);
        }
    }
    const int lane = __ffsll(who) - 1;
    const uint64_t best = (uint64_t)mh << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, lane);
    return best <= order64(kNever) ? -1 : lane;
}

// A wavefront's choice for a token of logits l: id and weight of slot r at lane r, -1 and 0
// where there is none. With R > 0 lane `sub` holds the keys of experts sub, sub + 64, .. in
// registers (n_expert <= 64 R), else in `key`. gsum: n_group doubles of LDS, key: n_expert.
template <int R>
__device__ __forceinline__ void moe_choose(const MoeLayerArgs &a, const double *l, const double *scores, double *key,
                                           double *gsum, int &id, float &weight) {
    constexpr int N = R > 0 ? R : 1;
    const int lane = threadIdx.x & 63, per = a.n_expert / a.n_group;
    const bool soft = a.score == ROUTE_SOFTMAX, scored = a.bias || a.n_group > 1;
    double m = kNever, sum = 0.0, own[N], lg[N], sc[N];
    float bias[N];
    if constexpr (R > 0) {  // (all of them asked for at once)
#pragma unroll
        for (int j = 0; j < R; j++) {
            const int e = min(lane + 64 * j, a.n_expert - 1);
            lg[j] = l[e];
            sc[j] = soft ? 0.0 : scores[e];
            bias[j] = a.bias ? a.bias[e] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < R; j++) lg[j] = lane + 64 * j < a.n_expert ? lg[j] : kNever;
    }
    if (soft) {
        if constexpr (R > 0) {
#pragma unroll
            for (int j = 0; j < R; j++) m = lg[j] > m ? lg[j] : m;  // (a NaN is not)
        } else {
            for (int e = lane; e < a.n_expert; e += 64) m = l[e] > m ? l[e] : m;
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) m = fmax(m, __shfl_xor(m, off, 64));
        if constexpr (R > 0) {
#pragma unroll
            for (int j = 0; j < R; j++) {
                sc[j] = lg[j] > kNever ? route_exp(lg[j], m) : 0.0;
                sum += sc[j];
            }
        } else {
            for (int e = lane; e < a.n_expert; e += 64)
                if (l[e] > kNever) sum += route_exp(l[e], m);
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        if constexpr (R > 0) {
#pragma unroll
            for (int j = 0; j < R; j++) sc[j] /= sum;
        }
    }
    auto score = [&](int e) { return soft ? route_exp(l[e], m) / sum : scores[e]; };
    auto place = [&](double le, double s, float b) {
        const double p = scored ? s + (double)b : le;
        return le > kNever && p > kNever ? p : kNever;
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int j = 0; j < R; j++) own[j] = place(lg[j], sc[j], bias[j]);
        if (a.n_group > 1) {
#pragma unroll
            for (int j = 0; j < R; j++)
                if (lane + 64 * j < a.n_expert) key[lane + 64 * j] = own[j];
        }
    } else {
        for (int e = lane; e < a.n_expert; e += 64)
            key[e] = place(l[e], scored ? score(e) : 0.0, a.bias ? a.bias[e] : 0.0f);
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
        auto kept = [&](int e, double k, double le) {
            const double g = gsum[e / per];
            return g == g ? kNever : !a.bias && k > kNever ? le : k;
        };
        if constexpr (R > 0) {
#pragma unroll
            for (int j = 0; j < R; j++)
                if (lane + 64 * j < a.n_expert) own[j] = kept(lane + 64 * j, own[j], lg[j]);
        } else {
            for (int e = lane; e < a.n_expert; e += 64) key[e] = kept(e, key[e], l[e]);
            __builtin_amdgcn_wave_barrier();
        }
    }
    // every lane's best of its keys (and its score); the one that gives it looks for its next
    double v, vs = 0.0, s = 0.0;
    int i;
    auto best = [&]() __attribute__((always_inline)) {
        v = kNever;
        i = a.n_expert;
        if constexpr (R > 0) {
#pragma unroll
            for (int j = 0; j < R; j++) {
                if (route_before(own[j], lane + 64 * j, v, i)) {
                    v = own[j];
                    vs = sc[j];
                    i = lane + 64 * j;
                }
            }
        } else {
            for (int e = lane; e < a.n_expert; e += 64) route_best(v, i, key[e], e);
        }
    };
    best();
    id = -1;
    for (int r = 0; r < a.k; r++) {
        const int who = moe_best(order64(v), i);
        if (who < 0) break;
        const int chosen = __builtin_amdgcn_readlane(i, who);
        const uint64_t bits = __builtin_bit_cast(uint64_t, vs);
        const uint32_t s0 = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, who);
        const uint32_t s1 = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), who);
        if (lane == r) {
            id = chosen;
            s = __builtin_bit_cast(double, (uint64_t)s1 << 32 | s0);
        }
        if (lane == who) {
            if constexpr (R > 0) {
#pragma unroll
                for (int j = 0; j < R; j++) own[j] = lane + 64 * j == chosen ? kNever : own[j];
            } else {
                key[chosen] = kNever;
            }
            best();
        }
    }
    if constexpr (R == 0) s = id >= 0 ? score(id) : 0.0;
    double out = s * (double)a.scale;
    if (a.renormalise) {
        double total = s;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) total += __shfl_xor(total, off, 64);
        out = total == 0.0 ? 0.0 : out / total;
    }
    weight = id >= 0 ? (float)out : 0.0f;
}
// A slot of the plan.
__device__ __forceinline__ void moe_slot(const MoeLayerArgs &a, MoePlan &plan, int t, int i, int id, float weight) {
    const bool on = id >= 0 && weight != 0.0f;
    plan.expert[t * (a.k + a.n_shared) + i] = (int16_t)(on ? id : -1);
    plan.weight[t * (a.k + a.n_shared) + i] = weight;
    if (on) atomicOr(&plan.takes[id], 1u << t);
}
// Token t's choice by this wavefront, slot r's at lane r (-1 and 0 behind the k-th); ids and
// weights written if `write`. keys: n_expert + n_group doubles of LDS.
template <int R>
__device__ __forceinline__ void moe_choose_token(const MoeLayerArgs &a, const MoeWork &w, int t, double *keys, bool write,
                                                 int &id, float &weight) {
    const double *const l = w.logits + (size_t)t * a.n_expert, *const s = w.scores + (size_t)t * a.n_expert;
    const int lane = threadIdx.x & 63;
    moe_choose<R>(a, l, s, keys, keys + a.n_expert, id, weight);
    if (write && lane < a.k) {
        a.ids[t * a.k + lane] = id;
        a.weights[t * a.k + lane] = weight;
    }
}

// The workgroup's plan, jobs of at most cap tokens. `choose`: the first `choose` wavefronts
// make the tokens' choice themselves (workgroup 0 writes it), keys: n_expert + n_group doubles
// for each; 0: it is read.
template <int W> __device__ __forceinline__ void moe_plan(const MoeLayerArgs &a, const MoeWork &w, MoePlan &plan, int cap,
                                                          double *keys, int choose) {
    __shared__ int part[W];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, slots = a.k + a.n_shared;
    const int all = a.n_expert + a.n_shared;
    const bool one = a.n_tok == 1;  // whose slots are its jobs, as they come
    if (!one) {
        for (int e = tid; e < all; e += 64 * W)
            plan.takes[e] = e < a.n_expert ? 0u : a.n_tok == 32 ? 0xFFFFFFFFu : (1u << a.n_tok) - 1u;
        for (int i = tid; i < a.n_tok * a.n_shared; i += 64 * W) {
            const int t = i / a.n_shared, j = i - t * a.n_shared;
            plan.expert[t * slots + a.k + j] = (int16_t)(a.n_expert + j);
            plan.weight[t * slots + a.k + j] = 1.0f;
        }
        __syncthreads();
    }
    int id = -1;
    float weight = 0.0f;
    if (choose) {
        for (int t = wv < choose ? wv : a.n_tok; t < a.n_tok; t += choose) {
            moe_choose_token<kChooseExperts / 64>(a, w, t, keys + wv * (a.n_expert + a.n_group), blockIdx.x == 0, id, weight);
            if (!one && lane < a.k) moe_slot(a, plan, t, lane, id, weight);
        }
    } else if (one) {
        if (tid < a.k) {
            id = a.ids[tid];
            weight = a.weights[tid];
        }
    } else {
        for (int i = tid; i < a.n_tok * a.k; i += 64 * W) {
            const int t = i / a.k;
            moe_slot(a, plan, t, i - t * a.k, a.ids[i], a.weights[i]);
        }
    }
    if (one) {
        if (wv == 0) {
            if (lane >= a.k) {
                id = lane < slots ? a.n_expert + lane - a.k : -1;
                weight = 1.0f;
            }
            const bool on = id >= 0 && weight != 0.0f;
            const unsigned long long mask = __ballot(on);
            if (lane < slots) {
                plan.expert[lane] = (int16_t)(on ? id : -1);
                plan.weight[lane] = weight;
            }
            if (on) {
                const int at = __popcll(mask & ((1ull << lane) - 1));
                plan.job[at] = (uint16_t)id;
                plan.tokens[at] = 1u;
            }
            if (lane == 0) plan.n_jobs = __popcll(mask);
        }
        __syncthreads();
        return;
    }
    __syncthreads();
    // the jobs of a run of experts a thread, behind those of the threads before it
    const int run = (all + 64 * W - 1) / (64 * W), e0 = min(all, tid * run), e1 = min(all, e0 + run);
    int n = 0;
    for (int e = e0; e < e1; e++) n += (__popc(plan.takes[e]) + cap - 1) / cap;
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
        for (uint32_t left = plan.takes[e]; left; at++) {
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

// ---- the products -----------------------------------------------------------------------
//
// v_mfma_f32_16x16x32_bf16: rows of weights by columns of terms: column c of a job is term
// c % terms of its (c / terms)-th token (16 / terms of them a job), columns behind its last
// token bring zeros.

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
// A job's terms for a piece: this lane's column, its block of each step (`at`: bytes of that
// of step 0, beyond the buffer where the column brings zeros; behind a row's end the next
// row's or zeros come, which are not used).
struct MoeTerms {
    mx_bf8 v[4][4];
};
__device__ __forceinline__ void moe_terms(MoeTerms &x, __amdgpu_buffer_rsrc_t terms, uint32_t at, int i) {
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int m = 0; m < 4; m++)
            x.v[j][m] = __builtin_bit_cast(mx_bf8, bload16(terms, at + 1024u * (uint32_t)i + 256u * (uint32_t)j + 16u * (uint32_t)m, 0));
}
// acc[f] += the piece's rows times the terms; term(j, m): 8 of them of step j
template <int FR, class F>
__device__ __forceinline__ void moe_multiply(const MoePiece<FR> &p, F &&term, int i, int steps, int blocks, mx_v4f (&acc)[FR]) {
    const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (4 * i + j >= steps) break;
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
            const mx_bf8 x = term(j, m);
#pragma unroll
            for (int f = 0; f < FR; f++) {
                const uint4 &c = p.c[f][j];
                acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(moe_widen(m == 0 ? c.x : m == 1 ? c.y : m == 2 ? c.z : c.w, unit[f]), x,
                                                                 acc[f], 0, 0, 0);
            }
        }
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
// A row of weights times a row of terms (`pitch` elements from one term to the next, zeros behind
// its end) in 64 bits: for the rare sum that came out infinite or NaN. That happens where f32 is
// left on the way, and where codes of scales 253 and 254, which no quantiser makes, passed bf16's
// range. One lane's work, eight elements at a time; a NaN scale ends it. (With an expert of NaN
// weights that three of 32 tokens take, the 4096-wide layer takes 0.65 in place of 0.41 ms.)
template <int TERMS>
__device__ __forceinline__ double moe_again(const uint8_t *codes, const uint8_t *scales, const __bf16 *terms, int pitch, int n) {
    bool nan = false;
#pragma unroll 8
    for (int b = 0; b < (n + 31) / 32; b++) nan |= scales[b] == 255u;
    double sum = nan ? __builtin_nan("") : 0.0;
#pragma unroll 1
    for (int i = 0; i < n && sum == sum; i += 8) {  // (a NaN stays one)
        const uint32_t c = *reinterpret_cast<const uint32_t *>(codes + i / 2);
        mx_bf8 x[TERMS];
#pragma unroll
        for (int j = 0; j < TERMS; j++) x[j] = *reinterpret_cast<const mx_bf8 *>(terms + j * pitch + i);
        const auto c0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), c1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
        const auto c2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), c3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
        const float w[8] = {c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
        double part = 0.0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            double v = 0.0;
#pragma unroll
            for (int j = 0; j < TERMS; j++) v = fma((double)(float)x[j][k], (double)moe_unit_of(j), v);
            part = fma((double)w[k], v, part);
        }
        sum = fma(part, __builtin_bit_cast(double, (uint64_t)(scales[i / 32] + 1023u - 127u) << 52), sum);
    }
    return sum;
}
// The pairs (token, slot) of every job, CAP a job, 0xFFFF behind its last token.
template <int W, int CAP> __device__ __forceinline__ void moe_pairs(const MoeLayerArgs &a, const MoePlan &plan, uint16_t *pairs) {
    const int slots = a.k + a.n_shared;
    for (int i = threadIdx.x; i < plan.n_jobs * CAP; i += 64 * W) {
        const int job = i / CAP, t = moe_token(plan.tokens[job], i - job * CAP);
        pairs[i] = t >= 0 ? (uint16_t)(t * slots + moe_slot_of(a, plan, t, plan.job[job])) : 0xFFFFu;
    }
}

}  // namespace

// A token's choice a wavefront, for more tokens or experts than the up kernel's workgroups make
// it of for themselves. 6.8 us for 32 tokens of 256 experts: one chain of loads, 64-bit scores
// and k reductions over the lanes.
template <int R> __global__ __launch_bounds__(64) void k_moe_choose(MoeLayerArgs a, MoeWork w) {
    extern __shared__ __align__(16) uint8_t smem[];
    int id;
    float weight;
    moe_choose_token<R>(a, w, blockIdx.x, reinterpret_cast<double *>(smem), true, id, weight);
}

// Gate and up products, and the weighted SwiGLU of their sums as bf16 terms. The pieces of K
// go over `kw` of the wavefronts, XP each, whose terms a wavefront keeps while it goes through
// a run of (job, 16 rows): its loads are the weights' alone, NB turns ahead. (Loads return in
// order: terms fetched for every turn would wait for weights asked for before them.) With
// XP = 0 there are more pieces than that, and their terms come with every turn: at sizes that
// XP = 1 holds (32 tokens of 4096, f32) that takes the layer from 433 to 589 us, where XP = 2
// does (8 of 7168, bf16) from 244 to 269. The wavefronts' sums meet in LDS, where kBatch turns
// are finished at once (one by one the layer took 506 in place of 464 us, two barriers a turn).
template <int XP, int TERMS> __global__ __launch_bounds__(64 * kWaves)
void k_moe_up(MoeLayerArgs a, MoeWork w, int hterms, int kw, int choose) {
    constexpr int W = kWaves, NB = XP == 1 ? 3 : 2, TPT = 16 / TERMS, NX = XP > 0 ? XP : 1;
    extern __shared__ __align__(16) uint8_t smem[];  // keys of the choice, then sums [kBatch][W][2][64][4]
    __shared__ MoePlan plan;
    __shared__ uint16_t pairs[kMoeMaxPairs * TPT];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slots = a.k + a.n_shared, ff = a.n_ff, frow = pad128(ff), erow = pad128(a.n_embd);
    __shared__ int again;  // whether a sum is to be made again, which h of NaN marks
    if (tid == 0) again = 0;
    moe_plan<W>(a, w, plan, TPT, reinterpret_cast<double *>(smem), choose);
    const size_t rb = mx_row_bytes(a.n_embd), sb = mx_scale_bytes(a.n_embd);
    const int steps = (int)(rb / 64), pieces = (int)(sb / 16), blocks = (a.n_embd + 31) / 32;
    const int per = (ff + 15) / 16, turns = plan.n_jobs * per;
    const __amdgpu_buffer_rsrc_t xt = make_rsrc(w.x, (uint32_t)a.n_tok * 3u * (uint32_t)erow * 2u);
    float *const red = reinterpret_cast<float *>(smem);
    // this wavefront's pieces (from `k` on, kw apart) and its group's run of turns
    const int k = wv % kw, group = wv / kw, groups = W / kw, streams = (int)gridDim.x * groups;
    const int stream = (int)blockIdx.x * groups + group;
    const int from = (int)((long long)turns * stream / streams), to = (int)((long long)turns * (stream + 1) / streams);
    const int rounds = (turns + streams - 1) / streams;  // of every wavefront, for the barriers
    const int np = XP > 0 ? XP : (pieces + kw - 1) / kw;
    MoeTerms x[NX];
    MoePiece<2> p[NB];
    auto fetch = [&](MoePiece<2> &d, int m) __attribute__((always_inline)) {  // piece m % np of turn m / np
        const int turn = from + m / np, i = k + kw * (m % np);
        if (turn < to && i < pieces) {
            const size_t row = (size_t)plan.job[turn / per] * ff + min(turn % per * 16 + r, ff - 1);
            const MoeRows rows[2] = {{a.gate + row * rb + 16 * q, a.gate_s + row * sb}, {a.up + row * rb + 16 * q, a.up_s + row * sb}};
            moe_fetch<2>(d, rows, i, steps);
        }
    };
    auto column = [&](int job) {  // this lane's
        const int t = r < TPT * TERMS ? moe_token(plan.tokens[job], r / TERMS) : -1;
        return t >= 0 ? (uint32_t)((t * 3 + r % TERMS) * erow + 32 * q) * 2u : kMoeNone;
    };
    int mine = -1;  // the job whose terms are held
    uint32_t at = kMoeNone;
    auto keep = [&](int job) __attribute__((always_inline)) {
        if (job != mine) {
            mine = job;
            at = column(job);
            if constexpr (XP > 0) {
#pragma unroll
                for (int n = 0; n < XP; n++) moe_terms(x[n], xt, at, k + kw * n);
            }
        }
    };
    if (from < to) keep(from / per);
#pragma unroll
    for (int b = 0; b < NB; b++) fetch(p[b], b);
    moe_pairs<W, TPT>(a, plan, pairs);  // (for finish(), behind its barrier)
    // h of a pair's row r0 + r, from its sums
    auto put = [&](float g, float v, int pair, int r0) __attribute__((always_inline)) {
        if (a.clamp > 1e-6f) {
            g = g > a.clamp ? a.clamp : g;
            v = v > a.clamp ? a.clamp : v < -a.clamp ? -a.clamp : v;
        }
        g = g < -kFltMax ? -kFltMax : g;  // (a sum below f32's range: silu is 0 there, not inf / inf)
        float h = r0 + r < ff ? g / (1.0f + expf(-g)) * v * plan.weight[pair] : 0.0f;
        __bf16 *const dst = w.h + (size_t)pair * 3 * frow + r0 + r;
        for (int j = 0; j < hterms; j++) {
            // (an infinity stays one; a number has no term that is rounded to one)
            const __bf16 b16 = (__bf16)(finite(h) ? fminf(fmaxf(h, -kBf16Max), kBf16Max) : h);
            dst[j * frow] = b16;
            h = finite(h) ? (h - (float)b16) * moe_next(j) : 0.0f;
            if (r0 + 16 >= ff)  // zeros up to whole steps
                for (int z = 16; r0 + r + z < frow; z += 16) dst[j * frow + z] = (__bf16)0.0f;
        }
    };
    int held = 0;  // rounds whose sums are in LDS
    // The last `held` rounds up to b0 + held: a token of one of them for every 16 lanes (rows).
    // (LDS alone is waited for, not the weights on their way.)
    auto finish = [&](int b0) __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        for (int task = wv * 4 + q; task < held * groups * TPT; task += W * 4) {
            const int c0 = task % TPT, g0 = task / TPT % groups, b = task / TPT / groups;
            const int s0 = (int)blockIdx.x * groups + g0;
            const int turn = (int)((long long)turns * s0 / streams) + b0 + b;
            if (turn >= (int)((long long)turns * (s0 + 1) / streams)) continue;
            const int job = turn / per, r0 = turn % per * 16, pair = pairs[job * TPT + c0];
            if (pair == 0xFFFF) continue;
            const float *const src = red + ((b * W + g0 * kw) * 2 * 64 + c0 * TERMS + 16 * (r >> 2)) * 4 + (r & 3);
            float g = 0.0f, v = 0.0f;
#pragma unroll 2
            for (int y = 0; y < kw; y++) {
#pragma unroll
                for (int j = 0; j < TERMS; j++) {
                    g = fmaf(src[(y * 2 * 64 + j) * 4], moe_unit_of(j), g);
                    v = fmaf(src[((y * 2 + 1) * 64 + j) * 4], moe_unit_of(j), v);
                }
            }
            if (!(finite(g) && finite(v))) {
                g = __builtin_nanf("");
                if (!w.bad[pair / slots]) again = 1;
            }
            put(g, v, pair, r0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        held = 0;
    };
    mx_v4f acc[2];
    // one of the NB buffers' turn (or, of more pieces, part of one)
    auto part = [&](auto b_c, int m) __attribute__((always_inline)) {
        constexpr int b = decltype(b_c)::value;
        const int round = m / np, n = m % np, turn = from + round, i = k + kw * n;
        const bool on = turn < to;
        if (n == 0) {
            acc[0] = acc[1] = mx_v4f{0.0f, 0.0f, 0.0f, 0.0f};
            if (on) keep(turn / per);
        }
        if (on && i < pieces) {
            if constexpr (XP > 0) {
                auto mul = [&](const MoeTerms &t) __attribute__((always_inline)) {
                    moe_multiply<2>(p[b], [&](int j, int h) { return t.v[j][h]; }, i, steps, blocks, acc);
                };
                mul(x[XP == 2 ? b : 0]);  // (buffer b: piece b of a turn)
            } else {
                moe_terms(x[0], xt, at, i);
                moe_multiply<2>(p[b], [&](int j, int h) { return x[0].v[j][h]; }, i, steps, blocks, acc);
            }
        }
        fetch(p[b], m + NB);
        if (n == np - 1) {
            mx_v4f *const sums = reinterpret_cast<mx_v4f *>(red) + held * W * 128;
            sums[(wv * 2) * 64 + lane] = acc[0];
            sums[(wv * 2 + 1) * 64 + lane] = acc[1];
            held++;
        }
    };
    const int total = rounds * np;
    for (int m = 0; m < total; m += NB) {
        part(std::integral_constant<int, 0>{}, m);
        if (m + 1 < total) part(std::integral_constant<int, 1>{}, m + 1);
        if constexpr (NB == 3) {
            if (m + 2 < total) part(std::integral_constant<int, 2>{}, m + 2);
        }
        const int end = min(total, m + NB);
        if (held + (XP == 1 ? NB : 1) > kBatch || end == total) finish(end / np - held);
    }
    // The sums to make again: here, where nothing of the loop is live (in finish() it spills).
    if (__builtin_expect(!again, 1)) return;  // (everyone's: finish() ends with a barrier)
    __syncthreads();                          // (h has been written)
    const int first = (int)((long long)turns * (int)blockIdx.x * groups / streams);
    const int last = (int)((long long)turns * ((int)blockIdx.x + 1) * groups / streams);
    for (int turn = first + wv; turn < last; turn += W) {  // (this workgroup's own h)
        const int job = turn / per, r0 = turn % per * 16;
        for (int c0 = q; c0 < TPT; c0 += 4) {
            const int pair = pairs[job * TPT + c0];
            if (pair == 0xFFFF || w.bad[pair / slots] || r0 + r >= ff) continue;
            const float h = (float)w.h[(size_t)pair * 3 * frow + r0 + r];
            if (h == h) continue;
            const size_t row = (size_t)plan.job[job] * ff + r0 + r;
            const __bf16 *const terms = w.x + (size_t)(pair / slots) * 3 * erow;
            const float g = (float)moe_again<TERMS>(a.gate + row * rb, a.gate_s + row * sb, terms, erow, a.n_embd);
            const float v = g == g ? (float)moe_again<TERMS>(a.up + row * rb, a.up_s + row * sb, terms, erow, a.n_embd) : 0.0f;
            put(g, v, pair, r0);
        }
    }
}

// The value of the N-th lane after this one, of the same 16.
template <int N> __device__ __forceinline__ float moe_lane_after(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x100 + N, 0xf, 0xf, true));
}

// The down products of 16 rows a turn over all jobs: the pieces of K over kw of the
// wavefronts, runs of jobs over the groups of so many; which split is a rule on the numbers
// of both (32 tokens of 64 experts with n_ff 1300, three pieces: 214 us for the layer with the
// jobs alone split, 294 with eight wavefronts a job). Every wavefront adds its jobs' columns
// to sums of its own for each token. An item's weights and its terms of h, a row of h (a
// column) a load, are asked for NB items ahead (three and four were no faster) and in the
// order they are used in; the terms then go through LDS, the wavefront's own, to the lanes
// that hold them for the products. With 32 tokens (145 us, 4.2 TB/s of weights) h comes to
// as many bytes from L2 as the weights, and a workgroup a CU keeps its vector units busy a
// third of the time; the rest are waits.
template <int TERMS> __global__ __launch_bounds__(64 * kWaves, 2)
void k_moe_down(MoeLayerArgs a, MoeWork w, int parts) {
    static_assert(kWaves == 8, "the split");
    constexpr int W = kWaves, NB = 2, CAP = kDownColumns / TERMS, C = CAP * TERMS, PITCH = 1024 + 16;  // (16: no bank conflicts)
    __shared__ MoePlan plan;
    __shared__ uint16_t pairs[kMoeMaxPairs * CAP];
    extern __shared__ __align__(16) uint8_t smem[];  // [W][C + 1][PITCH], sums [W][n_tok][16]
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slots = a.k + a.n_shared, frow = pad128(a.n_ff);
    uint8_t *const mine = smem + wv * (C + 1) * PITCH;
    float *const sums = reinterpret_cast<float *>(smem + W * (C + 1) * PITCH), *const own = sums + wv * a.n_tok * 16;
    *reinterpret_cast<uint4 *>(mine + C * PITCH + 16 * lane) = make_uint4(0, 0, 0, 0);  // a column of zeros
    moe_plan<W>(a, w, plan, CAP, nullptr, 0);
    moe_pairs<W, CAP>(a, plan, pairs);
    const size_t rb = mx_row_bytes(a.n_ff), sb = mx_scale_bytes(a.n_ff);
    const int steps = (int)(rb / 64), pieces = (int)(sb / 16), blocks = (a.n_ff + 31) / 32;
    // this workgroup's jobs, of which this wavefront's, and its pieces: the split whose longest
    // share is the shortest
    const int tiles = (int)gridDim.x / parts, me = (int)blockIdx.x / tiles;
    const int all = __builtin_amdgcn_readfirstlane(plan.n_jobs), first = all * me / parts, n_jobs = all * (me + 1) / parts - first;
    int kw = 1, least = INT_MAX;
#pragma unroll
    for (int b = 3; b >= 0; b--) {
        const int share = ((n_jobs + (W >> b) - 1) >> (3 - b)) * ((pieces + (1 << b) - 1) >> b);
        kw = share < least ? 1 << b : kw;
        least = min(share, least);
    }
    const int k = wv % kw, group = wv / kw, groups = W / kw;
    const int from = first + n_jobs * group / groups, to = k < pieces ? first + n_jobs * (group + 1) / groups : from;
    const int total = (to - from) * ((pieces - k + kw - 1) / kw);
    struct At {
        int job, i;
    };
    auto next = [&](At &at) __attribute__((always_inline)) {
        at.i += kw;
        if (at.i >= pieces) {
            at.i = k;
            at.job++;
        }
    };
    struct Item {
        MoePiece<1> p;
        uint4 h[C];
    };
    for (int r0 = ((int)blockIdx.x - me * tiles) * 16; r0 < a.n_embd; r0 += tiles * 16) {
        __syncthreads();  // (pairs are there, the last turn's sums are read)
        for (int i = lane; i < a.n_tok * 16; i += 64) own[i] = 0.0f;
        const size_t row = (size_t)min(r0 + r, a.n_embd - 1);
        Item item[NB];
        At ahead = {from, k}, here = ahead;
        auto fetch = [&](Item &d) __attribute__((always_inline)) {
            const int job = ahead.job, i = ahead.i;
            if (job >= to) return;
            next(ahead);
            const size_t e = (size_t)__builtin_amdgcn_readfirstlane((int)plan.job[job]);
            const MoeRows rows[1] = {{a.down + (e * a.n_embd + row) * rb + 16 * q, a.down_s + (e * a.n_embd + row) * sb}};
            moe_fetch<1>(d.p, rows, i, steps);
            const int col = 512 * i + 8 * lane;
#pragma unroll
            for (int n = 0; n < CAP; n++) {
                const int pair = __builtin_amdgcn_readfirstlane((int)pairs[job * CAP + n]);
                if (pair == 0xFFFF) break;
#pragma unroll
                for (int j = 0; j < TERMS; j++) {
                    d.h[n * TERMS + j] = make_uint4(0, 0, 0, 0);
                    if (col < frow)
                        d.h[n * TERMS + j] = *reinterpret_cast<const uint4 *>(w.h + ((size_t)pair * 3 + j) * frow + col);
                }
            }
        };
        int tok = -1, columns = 0;
        const uint8_t *src = mine;
        mx_v4f acc[1] = {mx_v4f{0.0f, 0.0f, 0.0f, 0.0f}};
        // a token's terms stand in neighbouring lanes: to the first of them, and to its sums
        auto flush = [&]() __attribute__((always_inline)) {
            mx_v4f y = acc[0];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                y[i] = fmaf(moe_lane_after<1>(acc[0][i]), moe_unit_of(1), y[i]);
                if (TERMS == 3) y[i] = fmaf(moe_lane_after<2>(acc[0][i]), moe_unit_of(2), y[i]);
            }
            if (tok >= 0 && r % TERMS == 0) *reinterpret_cast<mx_v4f *>(own + tok * 16 + 4 * q) += y;
            acc[0] = mx_v4f{0.0f, 0.0f, 0.0f, 0.0f};
        };
#pragma unroll
        for (int b = 0; b < NB; b++) fetch(item[b]);
        auto part = [&](auto b_c) __attribute__((always_inline)) {
            Item &d = item[decltype(b_c)::value];
            const int i = here.i;
            if (i == k) {
                const int pair = r < C ? pairs[here.job * CAP + min(r / TERMS, CAP - 1)] : 0xFFFF;
                tok = pair == 0xFFFF ? -1 : pair / slots;
                columns = __builtin_amdgcn_readfirstlane(__popc(plan.tokens[here.job])) * TERMS;
                src = mine + (tok >= 0 ? r : C) * PITCH + 64 * q;
            }
#pragma unroll
            for (int n = 0; n < C; n++)
                if (n < columns) *reinterpret_cast<uint4 *>(mine + n * PITCH + 16 * lane) = d.h[n];
            __builtin_amdgcn_wave_barrier();
            moe_multiply<1>(d.p, [&](int j, int m) { return *reinterpret_cast<const mx_bf8 *>(src + 256 * j + 16 * m); },
                            i, steps, blocks, acc);
            __builtin_amdgcn_wave_barrier();
            fetch(d);
            next(here);
            if (here.i == k) flush();
        };
        for (int c = 0; c < total; c += NB) {
            part(std::integral_constant<int, 0>{});
            if (c + 1 < total) part(std::integral_constant<int, 1>{});
        }
        __syncthreads();
        for (int i = tid; i < a.n_tok * 16; i += 64 * W) {
            const int t = i >> 4, o = r0 + (i & 15), bad = w.bad[t];
            float y = 0.0f;
#pragma unroll
            for (int v = 0; v < W; v++) y += sums[v * a.n_tok * 16 + i];
            if (o >= a.n_embd) continue;
            if (__builtin_expect(!finite(y) && !bad, 0)) {
                double again = 0.0;
                for (int j = first * CAP; j < (first + n_jobs) * CAP && again == again; j++) {
                    if (pairs[j] == 0xFFFF || pairs[j] / slots != t) continue;
                    const size_t row = (size_t)plan.job[j / CAP] * a.n_embd + o;
                    again += moe_again<TERMS>(a.down + row * rb, a.down_s + row * sb, w.h + (size_t)pairs[j] * 3 * frow, frow, a.n_ff);
                }
                y = (float)again;
            }
            if (parts > 1) w.part[((size_t)me * a.n_tok + t) * a.n_embd + o] = y;
            else mx_store(a.out, (size_t)t * a.out_stride + o, bad ? __builtin_nanf("") : y, a.dtype_out);
        }
    }
}

// The sum of the down kernel's parts, in their order: one chain of loads, 4 to 5 us.
__global__ __launch_bounds__(256) void k_moe_sum(MoeLayerArgs a, MoeWork w, int parts) {
    const int t = blockIdx.y, o = blockIdx.x * 256 + threadIdx.x;
    if (o >= a.n_embd) return;
    float y = 0.0f;
    for (int i = 0; i < parts; i++) y += w.part[((size_t)i * a.n_tok + t) * a.n_embd + o];
    mx_store(a.out, (size_t)t * a.out_stride + o, w.bad[t] ? __builtin_nanf("") : y, a.dtype_out);
}

size_t moe_layer_work_bytes(int n_tok, int n_embd, int n_ff, int n_expert, int k, int n_shared) {
    return moe_parts(n_tok, n_embd, n_ff, n_expert, k, n_shared, nullptr, nullptr);
}

namespace {

template <uint32_t DX> void moe_in_go(const MoeLayerArgs &a, const MoeWork &w, hipStream_t s) {
    const int size = DX == T_F32 ? 4 : 2, rsize = a.dtype_router == T_F32 ? 4 : 2;
    const int vx = (uintptr_t)a.x % 16 == 0 && a.x_stride * size % 16 == 0;
    const int vr = (uintptr_t)a.router % 16 == 0 && (size_t)a.n_embd * rsize % 16 == 0;
    const dim3 g((unsigned)(a.n_expert + a.n_tok)), n(64 * kInWaves);
    if (a.dtype_router == T_F32) k_moe_in<DX, T_F32><<<g, n, 0, s>>>(a, w, vx, vr);
    else if (a.dtype_router == T_F16) k_moe_in<DX, T_F16><<<g, n, 0, s>>>(a, w, vx, vr);
    else k_moe_in<DX, T_BF16><<<g, n, 0, s>>>(a, w, vx, vr);
}

// More LDS than a kernel gets unasked, asked for until the runtime has granted it once on
// the current device: a refusal is that call's error alone.
template <int KERNEL> hipError_t moe_allow_lds(const void *kernel, size_t bytes) {
    static std::atomic<uint64_t> granted{0};  // a bit a device; beyond 64 it is asked every time
    int dev;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (granted.load(std::memory_order_acquire) & bit) return hipSuccess;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess) granted.fetch_or(bit, std::memory_order_release);
    else (void)hipGetLastError();  // (or the next launch would report it)
    return e;
}

template <int XP, int TERMS>
hipError_t moe_up_go(const MoeLayerArgs &a, const MoeWork &w, int hterms, int kw, hipStream_t s) {
    // sums, or the choice's keys (32 KB at most)
    const size_t keys = (size_t)(a.n_expert + a.n_group) * 8;
    int choose = 0;
    if (a.n_tok <= kChooseTok && a.n_expert <= kChooseExperts) {
        choose = kWaves;
    } else {
        if (a.n_expert <= kChooseExperts) k_moe_choose<kChooseExperts / 64><<<(unsigned)a.n_tok, 64, keys, s>>>(a, w);
        else k_moe_choose<0><<<(unsigned)a.n_tok, 64, keys, s>>>(a, w);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    // a workgroup a CU, no more than there can be turns
    const long long turns = (long long)a.n_tok * (a.k + a.n_shared) * ((a.n_ff + 15) / 16);
    const long long wgs = (turns * kw + kWaves - 1) / kWaves;
    constexpr size_t sums = (size_t)kBatch * kWaves * 2048;
    const hipError_t e = moe_allow_lds<16 * XP + TERMS + 8>(reinterpret_cast<const void *>(&k_moe_up<XP, TERMS>), sums);
    if (e != hipSuccess) return e;
    k_moe_up<XP, TERMS><<<(unsigned)std::min(wgs, (long long)256), 64 * kWaves, std::max(choose * keys, sums), s>>>(
        a, w, hterms, kw, choose);
    return hipGetLastError();
}
template <int TERMS> hipError_t moe_up(const MoeLayerArgs &a, const MoeWork &w, int hterms, hipStream_t s) {
    const int pieces = (int)mx_scale_bytes(a.n_embd) / 16;
    if (pieces > 2 * kWaves) return moe_up_go<0, TERMS>(a, w, hterms, kWaves, s);
    if (pieces > kWaves) return moe_up_go<2, TERMS>(a, w, hterms, kWaves, s);
    // (Wavefronts idle at 3, 5 to 7 and 9 to 15 pieces. 32 tokens of 6 of 256 experts and a shared
    // one, n_ff 2048, bytes of weights over the layer's time: 3.4 TB/s 2048 wide, 3.1 at 2560, 4.0
    // at 4096, 3.1 and 3.3 at 4608 and 5120, 4.0 at 7168.)
    const int kw = pieces > 4 ? 8 : pieces > 2 ? 4 : pieces;
    return moe_up_go<1, TERMS>(a, w, hterms, kw, s);
}

template <int TERMS> hipError_t moe_down(const MoeLayerArgs &a, const MoeWork &w, hipStream_t s) {
    constexpr size_t columns = (size_t)kWaves * (kDownColumns + 1) * 1040, sums = (size_t)kWaves * 64;
    const hipError_t e = moe_allow_lds<TERMS>(reinterpret_cast<const void *>(&k_moe_down<TERMS>), columns + sums * kMoeMaxTok);
    if (e != hipSuccess) return e;
    const int tiles = std::min((a.n_embd + 15) / 16, 512), parts = moe_down_parts(a.n_tok, a.n_embd, a.n_ff, a.k + a.n_shared);
    k_moe_down<TERMS><<<(unsigned)(tiles * parts), 64 * kWaves, columns + sums * a.n_tok, s>>>(a, w, parts);
    const hipError_t d = hipGetLastError();
    if (d != hipSuccess || parts == 1) return d;
    k_moe_sum<<<dim3((unsigned)(a.n_embd + 255) / 256, (unsigned)a.n_tok), 256, 0, s>>>(a, w, parts);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_layer(const MoeLayerArgs &a, uint8_t *work, hipStream_t s) {
    if (a.n_tok <= 0) return hipSuccess;
    MoeWork w;
    moe_parts(a.n_tok, a.n_embd, a.n_ff, a.n_expert, a.k, a.n_shared, work, &w);
    // h as 16 bits where the output has 8 or 11: an output then differs by a rounding now and then
    // (bf16, 7168 / 2048, 8 of 64 experts, 8 tokens: 0.29% of the elements, 0.06% with 24 bits), the
    // error against 64 bits is the same to four digits. 24 bits take 236 in place of 229 us there,
    // 417 in place of 397 for 32 tokens of 4096 / 2048.
    const int hterms = a.dtype_out == T_F32 ? 3 : 2;
    if (a.dtype_x == T_F32) moe_in_go<T_F32>(a, w, s);
    else if (a.dtype_x == T_F16) moe_in_go<T_F16>(a, w, s);
    else moe_in_go<T_BF16>(a, w, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    e = a.dtype_x == T_F32 ? moe_up<3>(a, w, hterms, s) : a.dtype_x == T_F16 ? moe_up<2>(a, w, hterms, s) : moe_up<1>(a, w, hterms, s);
    if (e != hipSuccess) return e;
    return hterms == 3 ? moe_down<3>(a, w, s) : moe_down<2>(a, w, s);
}

}  // namespace rsllm_hip
