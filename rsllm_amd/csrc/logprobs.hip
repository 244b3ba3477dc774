// Log-probability, rank, entropy and most likely alternatives of each row of
// vocabulary logits, in one pass over them.
//   m = max l, S = sum exp(l - m), D = sum exp(l - m) (l - m)
//   logprob = l_tok - m - log S,  entropy = log S - D / S
// Every lane keeps m, S and D of what it has seen (S and D rescaled when m
// rises: S' = r S, D' = r (D + (m - m') S), r = exp(m - m')), so a row is read
// once; parts meet by the same rule. What bounds it: the read of the logits for
// prompts (1000 x 129280 f32, 5 best: 94 us, 5.5 TB/s), two launches and the
// lists' sorting and merging for few rows (1 x 129280, 8 best: 10.8 us; 32 x 32000
// bf16, 20 best: 14.3, without a list 7.0).
// Alternatives: a wavefront keeps its n_top best in order, one a lane. A logit
// is only looked at where it beats the last of them, which in rows of no
// particular order soon is rare (n_top (1 + log(n / n_top)) times in n); many
// that do at once are sorted and merged in.
#include "kernels.h"

namespace rsllm_hip {

namespace {

constexpr float kInf = __builtin_inff();
constexpr int kLpWaves = 4;         // wavefronts a workgroup
constexpr int kLpFew = 8;           // chunks whose lists are merged one after another
constexpr int kLpTurn = 16 * 64 * kLpWaves;  // elements of a turn: 16 a lane

__device__ __forceinline__ float lp_one(const void *p, size_t i, uint32_t dtype) {
    if (dtype == T_F32) return static_cast<const float *>(p)[i];
    const uint16_t b = static_cast<const uint16_t *>(p)[i];
    return dtype == T_F16 ? f16_to_f32(b) : __builtin_bit_cast(float, (uint32_t)b << 16);
}

template <uint32_t DT> struct LpVec {
    static constexpr int N = DT == T_F32 ? 4 : 8;  // of 16 bytes
    static constexpr int L = 16 / N;               // loads of a turn
    static __device__ __forceinline__ void unpack(const uint4 &u, float *v) {
        const uint32_t d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == T_F32) {
                v[i] = __builtin_bit_cast(float, d[i]);
            } else if constexpr (DT == T_BF16) {
                v[2 * i] = __builtin_bit_cast(float, d[i] << 16);
                v[2 * i + 1] = __builtin_bit_cast(float, d[i] & 0xFFFF0000u);
            } else {
                v[2 * i] = f16_to_f32(d[i] & 0xFFFFu);
                v[2 * i + 1] = f16_to_f32(d[i] >> 16);
            }
        }
    }
};

// Running sums of some logits; m -inf: none but -inf so far. NaN in s: a NaN seen.
struct LpSums {
    float m, s, d;
};
// exp(x), x <= 0. (e x is wanted with e = 0 at x = -inf: hence the floor, far
// below where e vanishes.)
__device__ __forceinline__ float lp_exp(float x) { return __expf(x); }
__device__ __forceinline__ float lp_floor(float x) { return fmaxf(x, -200.0f); }

// What `a` and `b` saw together. +inf: the limit, in which only +inf counts (s
// their number).
__device__ __forceinline__ LpSums lp_join(const LpSums &a, const LpSums &b) {
    const float m = fmaxf(a.m, b.m);
    const float xa = a.m == m ? 0.0f : a.m - m, xb = b.m == m ? 0.0f : b.m - m;
    const float ra = lp_exp(xa), rb = lp_exp(xb);
    return LpSums{m, ra * a.s + rb * b.s,
                  ra * (a.d + lp_floor(xa) * a.s) + rb * (b.d + lp_floor(xb) * b.s)};
}

// A listed logit as one number: the value's place in the order of all floats
// above the complement of its id, so that the larger comes before, and of equals
// the lower id; 0: none. A wavefront's list stands in order, the i-th at lane i.
struct LpKey {
    uint32_t hi, lo;
    __device__ __forceinline__ uint64_t n() const { return (uint64_t)hi << 32 | lo; }
};
__device__ __forceinline__ LpKey lp_key(float v, int i) {
    const int b = __builtin_bit_cast(int, v + 0.0f);  // (-0 and 0 are equal)
    return LpKey{(uint32_t)b ^ ((uint32_t)(b >> 31) | 0x80000000u), ~(uint32_t)i};
}
__device__ __forceinline__ float lp_value(uint32_t hi) {
    return __builtin_bit_cast(float, hi & 0x80000000u ? hi ^ 0x80000000u : ~hi);
}
template <int CTRL> __device__ __forceinline__ uint32_t lp_dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
// Lane l gets lane l ^ X's: within rows of 16 lanes by DPP, across by a shuffle.
template <int X> __device__ __forceinline__ uint32_t lp_xor(uint32_t x) {
    if constexpr (X == 1) return lp_dpp<0xB1>(x);                  // quad_perm
    else if constexpr (X == 2) return lp_dpp<0x4E>(x);
    else if constexpr (X == 4) return lp_dpp<0x1B>(lp_dpp<0x141>(x));  // row_half_mirror (^ 7), ^ 3
    else if constexpr (X == 8) return lp_dpp<0x128>(x);            // row_ror:8
    else return (uint32_t)__shfl_xor((int)x, X, 64);
}
// One step of a bitonic network: of lanes l and l ^ X, those where `first` says
// so keep the one that comes before.
template <int X> __device__ __forceinline__ void lp_step(LpKey &t, bool first) {
    const LpKey o{lp_xor<X>(t.hi), lp_xor<X>(t.lo)};
    if ((o.n() > t.n()) == first) t = o;
}
// Runs of 2 X lanes that fall and then rise (or the reverse), into order: falling
// where `down`.
template <int X> __device__ __forceinline__ void lp_merge_from(LpKey &t, bool down) {
    const int lane = threadIdx.x & 63;
    lp_step<X>(t, ((lane & X) == 0) == down);
    if constexpr (X > 1) lp_merge_from<X / 2>(t, down);
}
__device__ __forceinline__ void lp_sort(LpKey &t) {
    const int lane = threadIdx.x & 63;
    lp_merge_from<1>(t, (lane & 2) == 0);
    lp_merge_from<2>(t, (lane & 4) == 0);
    lp_merge_from<4>(t, (lane & 8) == 0);
    lp_merge_from<8>(t, (lane & 16) == 0);
    lp_merge_from<16>(t, (lane & 32) == 0);
    lp_merge_from<32>(t, true);
}
// The 64 best of two lists in order: the better of a's i-th and b's 63 - i-th
// fall and rise once.
__device__ __forceinline__ void lp_merge(LpKey &top, const LpKey &b) {
    const LpKey o{lp_xor<63>(b.hi), lp_xor<63>(b.lo)};
    if (o.n() > top.n()) top = o;
    lp_merge_from<32>(top, true);
}

// A wavefront's list and its n-th (uniform).
struct LpList {
    LpKey top{0, 0}, edge{0, 0};
    __device__ __forceinline__ void set_edge(int n) {
        edge.hi = (uint32_t)__builtin_amdgcn_readlane((int)top.hi, n - 1);
        edge.lo = (uint32_t)__builtin_amdgcn_readlane((int)top.lo, n - 1);
    }
    // Takes every lane's candidate that is among the n best, and says whether
    // there was one: a few one by one, more of them sorted (kSorted: they come so)
    // and merged.
    template <bool kSorted> __device__ __forceinline__ bool take(int n, const LpKey &c) {
        const int lane = threadIdx.x & 63;
        const bool beats = c.n() > edge.n();
        unsigned long long todo = __ballot(beats);
        if (!todo) return false;
        if (__popcll(todo) > (kSorted ? 3 : 8)) {
            if (!kSorted && edge.n() == 0 && __ballot(top.n() != 0) == 0) {
                top = c;  // the first candidates
                lp_sort(top);
            } else {
                LpKey o{beats ? c.hi : 0, beats ? c.lo : 0};
                if (!kSorted) lp_sort(o);
                lp_merge(top, o);
            }
            set_edge(n);
            return true;
        }
        do {
            const int who = __ffsll(todo) - 1;
            todo &= todo - 1;
            const LpKey w{(uint32_t)__builtin_amdgcn_readlane((int)c.hi, who),
                          (uint32_t)__builtin_amdgcn_readlane((int)c.lo, who)};
            const int at = __popcll(__ballot(top.n() > w.n()));
            const LpKey prev{lp_dpp<0x138>(top.hi), lp_dpp<0x138>(top.lo)};  // wave_shr:1
            top = lane < at ? top : lane == at ? w : prev;
            set_edge(n);
            todo &= __ballot(c.n() > edge.n());
        } while (todo);
        return true;
    }
};

// One part of a row: sums, the number of logits above the token's, and its list.
struct LpPart {
    LpSums sums;
    int above;
};

__device__ __forceinline__ LpPart lp_wave_join(LpPart p) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const LpSums o{__shfl_xor(p.sums.m, off, 64), __shfl_xor(p.sums.s, off, 64),
                       __shfl_xor(p.sums.d, off, 64)};
        p.sums = lp_join(p.sums, o);
        p.above += __shfl_xor(p.above, off, 64);
    }
    return p;
}

// A row's outputs, by one wavefront that holds its sums and list.
__device__ __forceinline__ void lp_finish(const LogprobArgs &a, int t, const LpPart &p, const LpKey &top) {
    const int lane = threadIdx.x & 63;
    const float m = p.sums.m, nan = __builtin_nanf("");
    const bool bad = p.sums.s != p.sums.s, empty = m == -kInf;
    const float log_s = empty ? 0.0f : logf(p.sums.s);
    auto logprob = [&](float l) {
        return bad ? nan : empty ? -kInf : (l == m ? 0.0f : l - m) - log_s;
    };
    if (lane == 0) {
        if (a.tokens) {
            const int tok = a.tokens[t];
            const bool has = tok >= 0 && tok < a.vocab;
            const float l = has ? lp_one(a.logits, (size_t)t * a.stride + tok, a.dtype) : nan;
            a.logprob[t] = has ? logprob(l) : nan;
            if (a.rank) a.rank[t] = l == l ? p.above + 1 : 0;
        }
        if (a.entropy) a.entropy[t] = bad ? nan : empty ? 0.0f : log_s - p.sums.d / p.sums.s;
    }
    if (lane < a.n_top) {
        const size_t at = (size_t)t * a.n_top + lane;
        a.top_ids[at] = top.hi ? (int)~top.lo : -1;
        a.top_logprobs[at] = top.hi ? logprob(lp_value(top.hi)) : bad ? nan : -kInf;
    }
}

}  // namespace

// Where the parts of a row lie in the caller's workspace.
struct LpWork {
    LpPart *parts;  // [n_tok x chunks]
    LpKey *tops;    // [n_tok x chunks x n_top]
};

// Workgroup (chunk, row): `turns` turns, each kLpWaves * L pieces of 64 lanes x
// 16 bytes of the row, counted from the 16 bytes that the row starts in. With one
// chunk a row it writes the row's outputs, else its part.
template <uint32_t DT>
__global__ __launch_bounds__(64 * kLpWaves) void k_logprobs(LogprobArgs a, LpWork w, int chunks,
                                                            int turns) {
    using V = LpVec<DT>;
    constexpr int N = V::N, L = V::L, M = N * L;
    __shared__ LpPart part[kLpWaves];
    __shared__ LpKey list[kLpWaves][64];
    const int t = blockIdx.x / chunks, c = blockIdx.x - t * chunks;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const size_t row = (size_t)t * a.stride;
    const uint8_t *const p = static_cast<const uint8_t *>(a.logits) + row * (16 / N);
    const int head = (int)((uintptr_t)p & 15) / (16 / N);  // elements of the first line before the row

    const int tok = a.tokens ? a.tokens[t] : -1;
    // (NaN: nothing is above)
    const float mine = tok >= 0 && tok < a.vocab ? lp_one(a.logits, row + tok, DT) : __builtin_nanf("");
    LpSums sum{-kInf, 0.0f, 0.0f};
    int above = 0;
    LpList best;
    float edge_v = -kInf;

    const int pieces = turns * (kLpWaves * L);
    const int all = (int)(((long long)head + a.vocab + 64 * N - 1) / (64 * N));
    const int p1 = min(all, (c + 1) * pieces);
    for (int q0 = c * pieces + wv * L; q0 < p1; q0 += kLpWaves * L) {
        float v[M];
        // (piece q0's first element may be before the row: only in its first piece)
        const long long e0 = (long long)q0 * (64 * N) - head;
        if (e0 >= 0 && q0 + L <= p1 && e0 + 64 * M <= a.vocab) {
            const uint4 *src = reinterpret_cast<const uint4 *>(p + e0 * (16 / N)) + lane;
            uint4 u[L];
#pragma unroll
            for (int k = 0; k < L; k++) u[k] = src[64 * k];
#pragma unroll
            for (int k = 0; k < L; k++) V::unpack(u[k], v + N * k);
        } else {
#pragma unroll
            for (int k = 0; k < L; k++)
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const long long e = e0 + 64 * N * k + N * lane + i;
                    const bool in = q0 + k < p1 && e >= 0 && e < a.vocab;
                    v[N * k + i] = in ? lp_one(a.logits, row + (size_t)e, DT) : -kInf;
                }
        }
        float big = v[0];
#pragma unroll
        for (int i = 1; i < M; i++) big = fmaxf(big, v[i]);  // (a NaN is passed over)
        const float m = fmaxf(sum.m, big);
        if (__builtin_expect(__ballot(m == kInf) != 0, 0)) {
            // +inf - +inf is no number: the limit, one element at a time
#pragma unroll
            for (int i = 0; i < M; i++) {
                above += v[i] > mine ? 1 : 0;
                sum = lp_join(sum, v[i] != v[i] ? LpSums{-kInf, v[i], 0.0f}
                                                : LpSums{v[i], v[i] > -kInf ? 1.0f : 0.0f, 0.0f});
            }
        } else {
            const float base = m == -kInf ? 0.0f : m;  // (-inf - -inf is none either)
            const float x = sum.m - base, r = lp_exp(x);
            float s = 0.0f, d = 0.0f;
#pragma unroll
            for (int i = 0; i < M; i++) {
                above += v[i] > mine ? 1 : 0;
                const float y = v[i] - base, e = lp_exp(y);
                s += e;
                d = fmaf(e, lp_floor(y), d);
            }
            sum.d = r * (sum.d + lp_floor(x) * sum.s) + d;
            sum.s = r * sum.s + s;
            sum.m = m;
        }
        // (edge_v: the list's n-th value, -inf before there is one)
        if (a.n_top && __ballot(big >= edge_v && big > -kInf)) {
            const int i0 = (int)(e0 + N * lane);
            auto key = [&](float l, int j) {
                return l > -kInf ? lp_key(l, i0 + j / N * (64 * N) + j % N) : LpKey{0, 0};
            };
            if (best.edge.hi == 0) {
                // the first turns: every lane's largest first, which leaves
                // little of the rest to take
                int at = 0;
                float one = -kInf;
#pragma unroll
                for (int j = 0; j < M; j++) {
                    at = v[j] > one ? j : at;
                    one = fmaxf(one, v[j]);
                }
                best.take<false>(a.n_top, key(one, at));
#pragma unroll
                for (int j = 0; j < M; j++) v[j] = j == at ? -kInf : v[j];
                edge_v = best.edge.hi ? lp_value(best.edge.hi) : -kInf;
            }
#pragma unroll
            for (int j = 0; j < M; j++)
                if (__ballot(v[j] >= edge_v)) {
                    best.take<false>(a.n_top, key(v[j], j));
                    edge_v = best.edge.hi ? lp_value(best.edge.hi) : -kInf;
                }
        }
    }
    const LpPart mypart = lp_wave_join(LpPart{sum, above});
    if (lane == 0) part[wv] = mypart;
    if (a.n_top) list[wv][lane] = lane < a.n_top ? best.top : LpKey{0, 0};
    __syncthreads();
    if (wv != 0) return;
    LpPart all_part = part[0];
#pragma unroll
    for (int k = 1; k < kLpWaves; k++) {
        all_part.sums = lp_join(all_part.sums, part[k].sums);
        all_part.above += part[k].above;
        if (a.n_top) {
            best.take<true>(a.n_top, list[k][lane]);
        }
    }
    if (chunks == 1) {
        lp_finish(a, t, all_part, best.top);
    } else {
        const size_t at = (size_t)t * chunks + c;
        if (lane == 0) w.parts[at] = all_part;
        if (lane < a.n_top) w.tops[at * a.n_top + lane] = best.top;
    }
}

// One wavefront per row: its chunks' parts and lists.
__global__ __launch_bounds__(64) void k_logprobs_join(LogprobArgs a, LpWork w, int chunks) {
    const int t = blockIdx.x, lane = threadIdx.x;
    const size_t at = (size_t)t * chunks;
    LpPart p{{-kInf, 0.0f, 0.0f}, 0};
    for (int c = lane; c < chunks; c += 64) {
        const LpPart o = w.parts[at + c];
        p.sums = lp_join(p.sums, o.sums);
        p.above += o.above;
    }
    p = lp_wave_join(p);
    LpList best;
    if (chunks <= kLpFew && a.n_top > chunks) {
        // few and long: whole lists in order, all on their way before the first
        // is merged in (us, so / as below: 8 x 8000, 64 best 16.4 / 26.9, 8 best
        // 10.2 / 11.1; 32 x 32000 bf16, 64 best 21.4 / 26.8, 20 best 14.0 / 14.8,
        // 5 best 11.6 / 11.4)
        LpKey o[kLpFew];
#pragma unroll
        for (int c = 0; c < kLpFew; c++)
            o[c] = w.tops[(at + min(c, chunks - 1)) * a.n_top + min(lane, a.n_top - 1)];
        if (lane < a.n_top) best.top = o[0];
        best.set_edge(a.n_top);
#pragma unroll
        for (int c = 1; c < kLpFew; c++)
            if (c < chunks) best.take<true>(a.n_top, lane < a.n_top ? o[c] : LpKey{0, 0});
        lp_finish(a, t, p, best.top);
        return;
    }
    // a chunk's list a lane, their i-th entries together: as soon as none of those
    // is among the best, none behind them is
    for (int c0 = 0; c0 < chunks && a.n_top; c0 += 64) {
        const bool in = c0 + lane < chunks;
        const LpKey *src = w.tops + (at + min(c0 + lane, chunks - 1)) * a.n_top;
        LpKey next = src[0];
        for (int r = 0; r < a.n_top; r++) {
            const LpKey o = next;
            next = src[min(r + 1, a.n_top - 1)];
            if (!best.take<false>(a.n_top, in ? o : LpKey{0, 0})) break;
        }
    }
    lp_finish(a, t, p, best.top);
}

namespace {

// Chunks of a row. A workgroup takes a whole row where the rows alone keep the
// CUs busy (four workgroups each); fewer rows are cut up to that many, but no
// finer than one turn of a workgroup's loads.
struct LpPlan {
    int chunks, turns;  // turns of a chunk
};
LpPlan lp_plan(int n_tok, int vocab) {
    // (8: the elements before the row in its first 16 bytes at most, so that the
    // plan depends on n_tok and vocab alone)
    const long long turns = ((long long)vocab + 8 + kLpTurn - 1) / kLpTurn;
    const long long want = std::min<long long>(turns, std::max(1, 1024 / std::max(n_tok, 1)));
    const long long per = (turns + want - 1) / want;
    return {(int)((turns + per - 1) / per), (int)per};
}
size_t lp_round(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

size_t logprobs_scratch_bytes(int n_tok, int vocab, int n_top) {
    const LpPlan p = lp_plan(n_tok, vocab);
    if (p.chunks == 1 || n_tok == 0) return 0;
    const size_t n = (size_t)n_tok * p.chunks;
    return lp_round(n * sizeof(LpPart)) + lp_round(n * n_top * sizeof(LpKey));
}

hipError_t launch_logprobs(const LogprobArgs &a, uint8_t *work, int n_tok, hipStream_t s) {
    if (n_tok <= 0) return hipSuccess;
    const LpPlan p = lp_plan(n_tok, a.vocab);
    LpWork w{};
    if (p.chunks > 1) {
        w.parts = reinterpret_cast<LpPart *>(work);
        w.tops = reinterpret_cast<LpKey *>(work + lp_round((size_t)n_tok * p.chunks * sizeof(LpPart)));
    }
    const dim3 g((unsigned)n_tok * (unsigned)p.chunks);
    if (a.dtype == T_F32) k_logprobs<T_F32><<<g, 64 * kLpWaves, 0, s>>>(a, w, p.chunks, p.turns);
    else if (a.dtype == T_F16) k_logprobs<T_F16><<<g, 64 * kLpWaves, 0, s>>>(a, w, p.chunks, p.turns);
    else k_logprobs<T_BF16><<<g, 64 * kLpWaves, 0, s>>>(a, w, p.chunks, p.turns);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.chunks == 1) return e;
    k_logprobs_join<<<(unsigned)n_tok, 64, 0, s>>>(a, w, p.chunks);
    return hipGetLastError();
}

}  // namespace rsllm_hip
