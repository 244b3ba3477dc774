// The int8 product with a scale per token and per channel, and its quantiser.
#include "buffer_lds.h"
#include "kernels.h"

#include <atomic>
#include <type_traits>

namespace rsllm_hip {

namespace {

__device__ __forceinline__ float i8_load(const void *p, size_t i, uint32_t dtype) {
    if (dtype == T_F32) return static_cast<const float *>(p)[i];
    const uint16_t b = static_cast<const uint16_t *>(p)[i];
    return dtype == T_F16 ? f16_to_f32(b) : __builtin_bit_cast(float, (uint32_t)b << 16);
}

// One f32 rounded to the output's type (half to even), NaN kept.
__device__ __forceinline__ void i8_store(void *p, size_t i, float v, uint32_t dtype) {
    if (dtype == T_F32) {
        static_cast<float *>(p)[i] = v;
    } else if (dtype == T_F16) {
        static_cast<_Float16 *>(p)[i] = (_Float16)v;
    } else {
        static_cast<__bf16 *>(p)[i] = (__bf16)v;
    }
}

// A row's quantisation: the scale, and what a value is multiplied with to be
// near its code. Scales below 2^-100 are worked with 2^64 times as large, values
// too (both exactly), where 1 / d still fits.
struct I8Scale {
    float d, up, d_up, inv, quick;  // quick: 1 / d, or 0 where up is not 1
};
__device__ __forceinline__ I8Scale i8_scale(float amax) {
    I8Scale s;
    s.d = amax / 127.0f;
    s.up = s.d < 0x1p-100f ? 0x1p64f : 1.0f;
    s.d_up = s.d * s.up;
    s.inv = s.d > 0.0f ? 1.0f / s.d_up : 0.0f;
    s.quick = s.up == 1.0f ? s.inv : 0.0f;
    return s;
}
// v / d to the nearest integer, halves to even: the product with 1 / d is off by
// less than one from the exact quotient, and what is left over, v - r d, is
// exact in one FMA, so comparing it with d / 2 settles the rounding.
__device__ __forceinline__ int i8_code(float v, const I8Scale &s) {
#pragma clang fp contract(off)
    const float x = v * s.up;
    float r = rintf(x * s.inv);
    const float left = __builtin_fmaf(-r, s.d_up, x), two = 2.0f * fabsf(left);
    const bool odd = ((int)r & 1) != 0;
    if (two > s.d_up || (two == s.d_up && odd)) r += left > 0.0f ? 1.0f : -1.0f;
    r = fminf(fmaxf(r, -127.0f), 127.0f);  // a subnormal scale can be 1/3 too small
    return s.d > 0.0f ? (int)r : 0;
}

// 16 bytes of a row as floats; elements behind the row's end are 0.
template <uint32_t DT> struct I8Vec {
    static constexpr int N = DT == T_F32 ? 4 : 8;
};
// Elements [i, i + N) of the row at `row` (vec: 16-byte aligned there).
template <uint32_t DT>
__device__ __forceinline__ void i8_load_vec(const void *x, size_t row, int i, int in_dim, bool vec, float *v) {
    constexpr int N = I8Vec<DT>::N;
    if (vec && i + N <= in_dim) {
        const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(x) + (row + i) * (16 / N));
        const uint32_t d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (DT == T_F32) {
                v[k] = __builtin_bit_cast(float, d[k]);
            } else if constexpr (DT == T_BF16) {
                v[2 * k] = __builtin_bit_cast(float, d[k] << 16);
                v[2 * k + 1] = __builtin_bit_cast(float, d[k] & 0xFFFF0000u);
            } else {
                v[2 * k] = f16_to_f32(d[k] & 0xFFFFu);
                v[2 * k + 1] = f16_to_f32(d[k] >> 16);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = i + k < in_dim ? i8_load(x, row + i + k, DT) : 0.0f;
    }
}
// The N codes of v, packed, to 4-byte aligned memory. Adding 1.5 * 2^23 to v / d
// leaves the nearest integer in the low bits of the sum; what is left over is
// below d / 2 for all of them but once in some 2^17, and then v is taken one by
// one (as in rows of tiny scales, whose `quick` is 0).
template <int N> __device__ __forceinline__ void i8_store_codes(int8_t *dst, const float *v, const I8Scale &s) {
#pragma clang fp contract(off)
    uint32_t b[N], w[N / 4];
    float left = 0.0f;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const float sum = __builtin_fmaf(v[k], s.quick, 0x1.8p23f), r = sum - 0x1.8p23f;
        left = fmaxf(left, fabsf(__builtin_fmaf(-r, s.d, v[k])));
        b[k] = __builtin_bit_cast(uint32_t, sum);
    }
    if (!(2.0f * left < s.d)) {
#pragma unroll
        for (int k = 0; k < N; k++) b[k] = (uint32_t)i8_code(v[k], s);
    }
#pragma unroll
    for (int k = 0; k < N / 4; k++)  // the low bytes of four
        w[k] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[4 * k + 3], b[4 * k + 2], 0x0C0C0400u),
                                     __builtin_amdgcn_perm(b[4 * k + 1], b[4 * k], 0x0C0C0400u), 0x05040100u);
    if constexpr (N == 4) *reinterpret_cast<uint32_t *>(dst) = w[0];
    else *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
}
// A largest magnitude that remembers what is not finite: the bits of |v| in
// order, in which inf and NaN are above every number.
__device__ __forceinline__ uint32_t i8_abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }
__device__ __forceinline__ bool i8_finite_bits(uint32_t b) { return b < 0x7F800000u; }

}  // namespace

// A workgroup per row; the first kHeld vectors of a lane stay in registers
// between the search for the largest magnitude and the codes, longer rows are
// read again. Bound by reading x (2048 x 4096 bf16: 8.2 us for 25 MB, 3.1 TB/s).
template <uint32_t DT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_i8_quantize(const void *__restrict__ x, size_t stride,
                                                         int8_t *__restrict__ xq,
                                                         float *__restrict__ scale, int in_dim,
                                                         int row_bytes, int vec) {
    constexpr int N = I8Vec<DT>::N, kHeld = DT == T_F32 ? 4 : 2, W = THREADS / 64;
    __shared__ uint32_t red[W];
    const int t = blockIdx.x, tid = threadIdx.x;
    const size_t row = (size_t)t * stride;
    float held[kHeld][N];
    uint32_t big = 0;
#pragma unroll
    for (int h = 0; h < kHeld; h++) {
        const int i = (h * THREADS + tid) * N;
#pragma unroll
        for (int k = 0; k < N; k++) held[h][k] = 0.0f;
        if (i < in_dim) i8_load_vec<DT>(x, row, i, in_dim, vec, held[h]);
    }
#pragma unroll
    for (int h = 0; h < kHeld; h++)
#pragma unroll
        for (int k = 0; k < N; k++) big = max(big, i8_abs_bits(held[h][k]));
    for (int i = (kHeld * THREADS + tid) * N; i < in_dim; i += THREADS * N) {
        float v[N];
        i8_load_vec<DT>(x, row, i, in_dim, vec, v);
#pragma unroll
        for (int k = 0; k < N; k++) big = max(big, i8_abs_bits(v[k]));
    }
    big = wave_max_u32(big);
    if constexpr (W > 1) {
        if ((tid & 63) == 0) red[tid >> 6] = big;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; w++) big = max(big, red[w]);
    }
    const bool ok = i8_finite_bits(big);
    const I8Scale s = i8_scale(ok ? __builtin_bit_cast(float, big) : 0.0f);
    int8_t *const dst = xq + (size_t)t * row_bytes;
#pragma unroll
    for (int h = 0; h < kHeld; h++) {
        const int i = (h * THREADS + tid) * N;
        if (i < row_bytes) i8_store_codes<N>(dst + i, held[h], s);
    }
    for (int i = (kHeld * THREADS + tid) * N; i < row_bytes; i += THREADS * N) {
        float v[N];
        i8_load_vec<DT>(x, row, i, in_dim, vec, v);
        i8_store_codes<N>(dst + i, v, s);
    }
    if (tid == 0) scale[t] = ok ? s.d : __builtin_nanf("");
}

// ---- one token: one launch, the weights streamed through dot products -----------
//
// A wavefront multiplies R rows: a lane holds 16 bytes of every KB of a row, so the
// weights are read in whole lines, and its R sums are added across the wavefront at
// the end. The workgroup quantises x itself (x is small and in L2), its first
// weights already on the way. Bound by the weight stream (14336 x 4096: see the
// launcher). From two tokens on, every workgroup's quantising costs more than the
// launch it saves (4096 x 4096 f32, us, one launch against two: 1 token 6.9 / 7.9;
// with a form of this kernel for more, 2 tokens 10.2 / 8.2, 4 tokens 15.1 / 8.4).
template <uint32_t DT>
__global__ __launch_bounds__(256) void k_i8_one(I8Args a, const void *__restrict__ x, int in_dim, int kp,
                                                int vec) {
    constexpr int R = 4, P = 4, N = I8Vec<DT>::N, kHeld = 16 / N;  // P: 1 KB pieces of a row in flight
    extern __shared__ __align__(16) int8_t codes[];  // [kp], zero behind in_dim
    __shared__ uint32_t red[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int o0 = blockIdx.x * (4 * R), rb = a.row_bytes;
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(a.w + (size_t)o0 * rb, (uint32_t)min(4 * R, a.out_dim - o0) * (uint32_t)rb);
    uint4 w[P][R];
    // piece k0 of the rows (behind a row's end the next row's bytes or, past the
    // last, zeros: the codes there are zero)
    auto load = [&](uint4 (&d)[R], int k0) {
        if (k0 < rb) {
#pragma unroll
            for (int r = 0; r < R; r++) d[r] = bload16(rw, (uint32_t)((wv * R + r) * rb + k0 + 16 * lane), 0);
        }
    };
    // x, then the first weights behind it: loads return in order
    float held[kHeld][N];
#pragma unroll
    for (int h = 0; h < kHeld; h++) {
        const int i = (h * 256 + tid) * N;
#pragma unroll
        for (int k = 0; k < N; k++) held[h][k] = 0.0f;
        if (i < in_dim) i8_load_vec<DT>(x, 0, i, in_dim, vec, held[h]);
    }
    uint32_t big = 0;
    if (in_dim > kHeld * 256 * N) {
        for (int i = (kHeld * 256 + tid) * N; i < in_dim; i += 256 * N) {
            float v[N];
            i8_load_vec<DT>(x, 0, i, in_dim, vec, v);
#pragma unroll
            for (int k = 0; k < N; k++) big = max(big, i8_abs_bits(v[k]));
        }
    }
#pragma unroll
    for (int p = 0; p < P; p++) load(w[p], 1024 * p);
#pragma unroll
    for (int h = 0; h < kHeld; h++)
#pragma unroll
        for (int k = 0; k < N; k++) big = max(big, i8_abs_bits(held[h][k]));
    big = wave_max_u32(big);
    if (lane == 0) red[wv] = big;
    __syncthreads();
    big = max(max(red[0], red[1]), max(red[2], red[3]));
    const bool ok = i8_finite_bits(big);
    const I8Scale sc = i8_scale(ok ? __builtin_bit_cast(float, big) : 0.0f);
#pragma unroll
    for (int h = 0; h < kHeld; h++) {
        const int i = (h * 256 + tid) * N;
        if (i < kp) i8_store_codes<N>(codes + i, held[h], sc);
    }
    for (int i = (kHeld * 256 + tid) * N; i < kp; i += 256 * N) {
        float v[N];
        i8_load_vec<DT>(x, 0, i, in_dim, vec, v);
        i8_store_codes<N>(codes + i, v, sc);
    }
    __syncthreads();
    int acc[R] = {0, 0, 0, 0};
    for (int k0 = 0; k0 < rb; k0 += 1024 * P) {
#pragma unroll
        for (int p = 0; p < P; p++) {
            const int k = k0 + 1024 * p;
            if (k >= rb) break;
            const uint4 c = *reinterpret_cast<const uint4 *>(codes + k + 16 * lane);
#pragma unroll
            for (int r = 0; r < R; r++) {
                acc[r] = __builtin_amdgcn_sdot4((int)w[p][r].x, (int)c.x, acc[r], false);
                acc[r] = __builtin_amdgcn_sdot4((int)w[p][r].y, (int)c.y, acc[r], false);
                acc[r] = __builtin_amdgcn_sdot4((int)w[p][r].z, (int)c.z, acc[r], false);
                acc[r] = __builtin_amdgcn_sdot4((int)w[p][r].w, (int)c.w, acc[r], false);
            }
            load(w[p], k + 1024 * P);
        }
    }
    // the upper 32 lanes go on with rows 2 and 3, the odd DPP rows with 1 and 3
    const auto s0 = __builtin_amdgcn_permlane32_swap((uint32_t)acc[0], (uint32_t)acc[2], false, false);
    const auto s1 = __builtin_amdgcn_permlane32_swap((uint32_t)acc[1], (uint32_t)acc[3], false, false);
    const auto s = __builtin_amdgcn_permlane16_swap((uint32_t)(s0[0] + s0[1]), (uint32_t)(s1[0] + s1[1]), false, false);
    int sum = (int)(s[0] + s[1]);
    sum += __builtin_amdgcn_mov_dpp(sum, 0x128, 0xf, 0xf, true);  // row_ror:8
    sum += __builtin_amdgcn_mov_dpp(sum, 0x124, 0xf, 0xf, true);
    sum += __builtin_amdgcn_mov_dpp(sum, 0x122, 0xf, 0xf, true);
    sum += __builtin_amdgcn_mov_dpp(sum, 0x121, 0xf, 0xf, true);
    const int o = o0 + wv * R + (lane >> 4);
    if ((lane & 15) == 0 && o < a.out_dim) {
        float y = ((float)sum * (ok ? sc.d : __builtin_nanf(""))) * a.wscale[o];
        if (a.bias) y += a.bias[o];
        i8_store(a.out, (size_t)o, y, a.dtype_out);
    }
}

namespace {

// A row of a slice in LDS is 8 places of 16 bytes; byte 16 c of it lies at place
// c ^ i8_key(row), so that the 16 rows that an operand read takes at one c are
// spread over all banks (no bank conflicts counted).
__device__ __forceinline__ constexpr int i8_key(int row) { return (row >> 1) & 7; }
// ---- the product on the matrix cores -------------------------------------------

typedef int i8_v4 __attribute__((ext_vector_type(4)));

// A workgroup's tile: BM = 16 MF WM channels x BN = 16 NF WN tokens, each
// wavefront 16 MF x 16 NF of it; with WK > 1 the K slices of 128 bytes go round
// the WK groups of wavefronts, whose whole-number sums are added at the end.
// Slices of both operands are copied to LDS ST deep. For few tokens, where the
// weights' stream is the floor (32 x 16 tiles, 32 tokens of 4096 x 4096: 6.0 us for
// 17 MB, 2.8 TB/s).
template <int WM_, int WN_, int WK_, int MF_, int NF_, int ST_> struct I8Tile {
    static constexpr int WM = WM_, WN = WN_, WK = WK_, MF = MF_, NF = NF_, ST = ST_;
    static constexpr int BM = 16 * MF * WM, BN = 16 * NF * WN, kThreads = 64 * WM * WN * WK;
    static constexpr int kSlice = (BM + BN) * 128;          // bytes of one slice
    static constexpr int kCopies = (BM + BN) / 8;           // of 1 KB (8 rows) each
    static constexpr int D = (kCopies + WM * WN - 1) / (WM * WN);  // a wavefront's
    static constexpr int kRed = WK > 1 ? WK * WM * WN * MF * NF * 1024 : 0;
    static constexpr int kRing = WK * ST * kSlice;
    static constexpr int kLds = kRing > kRed ? kRing : kRed;
    static_assert(kLds <= 160 * 1024 && D * (ST - 2) <= 63, "tile");
};

// Four consecutive channels of one token.
__device__ __forceinline__ void i8_finish(const I8Args &a, const i8_v4 &acc, int o, int t, bool vec) {
    if (t >= a.n_tok || o >= a.out_dim) return;
    const float xs = a.xscale[t];
    const size_t at = (size_t)t * a.out_stride + o;
    if (vec && o + 3 < a.out_dim) {
        const float4 ws = *reinterpret_cast<const float4 *>(a.wscale + o);
        float y[4] = {((float)acc[0] * xs) * ws.x, ((float)acc[1] * xs) * ws.y,
                      ((float)acc[2] * xs) * ws.z, ((float)acc[3] * xs) * ws.w};
        if (a.bias) {
            const float4 b = *reinterpret_cast<const float4 *>(a.bias + o);
            y[0] += b.x; y[1] += b.y; y[2] += b.z; y[3] += b.w;
        }
        if (a.dtype_out == T_F32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) =
                make_float4(y[0], y[1], y[2], y[3]);
        } else {
            uint32_t lo, hi;
            if (a.dtype_out == T_F16) {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                lo = __builtin_bit_cast(uint32_t, h2{(_Float16)y[0], (_Float16)y[1]});
                hi = __builtin_bit_cast(uint32_t, h2{(_Float16)y[2], (_Float16)y[3]});
            } else {
                typedef __bf16 b2 __attribute__((ext_vector_type(2)));
                lo = __builtin_bit_cast(uint32_t, b2{(__bf16)y[0], (__bf16)y[1]});
                hi = __builtin_bit_cast(uint32_t, b2{(__bf16)y[2], (__bf16)y[3]});
            }
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + at) = make_uint2(lo, hi);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (o + i >= a.out_dim) return;
        float y = ((float)acc[i] * xs) * a.wscale[o + i];
        if (a.bias) y += a.bias[o + i];
        i8_store(a.out, at + i, y, a.dtype_out);
    }
}

template <class G>
__global__ __launch_bounds__(G::kThreads) void k_i8_tile(I8Args a, int n_ct, int n_tt) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int MF = G::MF, NF = G::NF, ST = G::ST, D = G::D;
    // Workgroups go round the 8 XCDs: each takes a run of tiles, token tiles
    // fastest, so the tiles that share a weight row are behind one L2.
    const int total = n_ct * n_tt, per = (total + 7) / 8;
    const int L = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || L >= total) return;  // the whole workgroup
    const int tt = L % n_tt, ct = L / n_tt;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wn = wv % G::WN, wm = wv / G::WN % G::WM, wk = wv / (G::WN * G::WM);
    const int o0 = ct * G::BM, t0 = tt * G::BN, rb = a.row_bytes;

    const int w_rows = min(G::BM, a.out_dim - o0), x_rows = min(G::BN, a.n_tok - t0);
    const bl_rsrc rw = bl_make_rsrc(a.w + (size_t)o0 * rb, (uint32_t)w_rows * (uint32_t)rb);
    const bl_rsrc rx = bl_make_rsrc(a.xq + (size_t)t0 * rb, (uint32_t)x_rows * (uint32_t)rb);
    // Copy c of a slice: 8 rows of the channels (c < BM / 8) or the tokens;
    // lane i brings row i / 8, and to place i % 8 of it the 16 bytes that the
    // operand reads look for there: (i % 8) ^ key(row).
    const uint32_t lds0 = bl_lds(smem) + (uint32_t)(wk * ST * G::kSlice);
    const int me = wm * G::WN + wn;  // among the wavefronts of one K group
    const int steps = ((rb + 127) / 128 + G::WK - 1) / G::WK;
    auto copy = [&](int i, int buf) {
        const int k0 = (wk + G::WK * i) * 128;
#pragma unroll
        for (int p = 0; p < D; p++) {
            const int c = min(me + G::WM * G::WN * p, G::kCopies - 1);
            const bool is_w = c < G::BM / 8;
            const int row = (is_w ? 8 * c : 8 * c - G::BM) + (lane >> 3);
            const int k = k0 + 16 * ((lane & 7) ^ i8_key(row));
            // behind the row's end: an offset past any resource, which brings zeros
            const uint32_t off = k < rb ? (uint32_t)row * (uint32_t)rb + (uint32_t)k : 0xFFFFFFF0u;
            const uint32_t dst = lds0 + (uint32_t)(buf * G::kSlice + c * 1024);
            if (is_w) bl_dma16(rw, off, 0, dst);
            else bl_dma16(rx, off, 0, dst);
        }
    };
    i8_v4 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) acc[m][n] = i8_v4{0, 0, 0, 0};

    const int r16 = lane & 15, q = lane >> 4;
    const uint8_t *const lw = smem + wk * ST * G::kSlice + (wm * 16 * MF + r16) * 128;
    const uint8_t *const lx = smem + wk * ST * G::kSlice + (G::BM + wn * 16 * NF + r16) * 128;
    const int s0 = 16 * (q ^ i8_key(r16)), s1 = 16 * ((4 + q) ^ i8_key(r16));

#pragma unroll
    for (int i = 0; i < ST - 1; i++) copy(i, i);
    int buf = 0, nbuf = ST - 1;
    for (int i = 0; i < steps; i++) {
        // slice i has landed everywhere, and everyone has read slice i - 1
        if constexpr (G::WM * G::WN * G::WK > G::WK) bl_barrier<D *(ST - 2)>();
        else bl_wait<D *(ST - 2)>();
        copy(i + ST - 1, nbuf);
        const uint8_t *const bw = lw + buf * G::kSlice, *const bx = lx + buf * G::kSlice;
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            const int so = kk ? s1 : s0;
            i8_v4 fw[MF], fx[NF];
#pragma unroll
            for (int n = 0; n < NF; n++) fx[n] = *reinterpret_cast<const i8_v4 *>(bx + n * 2048 + so);
#pragma unroll
            for (int m = 0; m < MF; m++) fw[m] = *reinterpret_cast<const i8_v4 *>(bw + m * 2048 + so);
#pragma unroll
            for (int m = 0; m < MF; m++)
#pragma unroll
                for (int n = 0; n < NF; n++)
                    acc[m][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[m], fx[n], acc[m][n], 0, 0, 0);
        }
        buf = buf + 1 == ST ? 0 : buf + 1;
        nbuf = nbuf + 1 == ST ? 0 : nbuf + 1;
    }
    bl_wait<0>();  // (the copies past the last slice, zeros, land in the ring too)
    const uint32_t esz = a.dtype_out == T_F32 ? 4u : 2u;
    const bool vec = ((uintptr_t)a.out % (4 * esz)) == 0 && a.out_stride % 4 == 0 &&
                     ((uintptr_t)a.wscale % 16) == 0 && ((uintptr_t)a.bias % 16) == 0;
    if constexpr (G::WK == 1) {
#pragma unroll
        for (int n = 0; n < NF; n++)
#pragma unroll
            for (int m = 0; m < MF; m++)
                i8_finish(a, acc[m][n], o0 + 16 * (wm * MF + m) + 4 * q, t0 + 16 * (wn * NF + n) + r16, vec);
    } else {
        bl_barrier<0>();
        i8_v4 *red = reinterpret_cast<i8_v4 *>(smem);
        constexpr int F = G::WM * G::WN * MF * NF;  // 16 x 16 pieces of the tile
#pragma unroll
        for (int m = 0; m < MF; m++)
#pragma unroll
            for (int n = 0; n < NF; n++)
                red[(wk * F + (me * MF + m) * NF + n) * 64 + lane] = acc[m][n];
        __syncthreads();
        for (int f = wv; f < F; f += G::WM * G::WN * G::WK) {
            i8_v4 s = red[f * 64 + lane];
#pragma unroll
            for (int k = 1; k < G::WK; k++) s += red[(k * F + f) * 64 + lane];
            const int n = f % NF, m = f / NF % MF, w = f / (NF * MF), fn = w % G::WN, fm = w / G::WN;
            i8_finish(a, s, o0 + 16 * (fm * MF + m) + 4 * q, t0 + 16 * (fn * NF + n) + r16, vec);
        }
    }
}

// More LDS than a kernel gets unasked, asked for until the runtime has granted it once
// on the current device: a refusal is that call's error alone.
template <class G> hipError_t i8_allow_lds(const void *kernel) {
    static std::atomic<uint64_t> granted{0};  // a bit a device; beyond 64 it is asked every time
    int dev;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (granted.load(std::memory_order_acquire) & bit) return hipSuccess;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, G::kLds);
    if (e == hipSuccess) granted.fetch_or(bit, std::memory_order_release);
    else (void)hipGetLastError();  // (or the next launch would report it)
    return e;
}

template <class G> hipError_t i8_tile_go(const I8Args &a, hipStream_t s) {
    const hipError_t e = i8_allow_lds<G>(reinterpret_cast<const void *>(&k_i8_tile<G>));
    if (e != hipSuccess) return e;
    const int n_ct = (a.out_dim + G::BM - 1) / G::BM, n_tt = (a.n_tok + G::BN - 1) / G::BN;
    const long long wgs = ((long long)n_ct * n_tt + 7) / 8 * 8;
    k_i8_tile<G><<<(unsigned)wgs, G::kThreads, G::kLds, s>>>(a, n_ct, n_tt);
    return hipGetLastError();
}

// The same product for many tokens: WM x WN wavefronts, ST slices in LDS, and
// the operands of the next half slice read into registers while the matrix
// cores work on this one. One barrier a slice, in its middle: behind it the
// next slice has landed, and every wavefront holds what is left of this one in
// registers, so the slice after the next can be copied over it. (64 x 64 tiles, 300
// tokens of 2048 x 4096: 9.4 us, 530 TOP/s: 160 tiles leave 96 CUs idle.)
template <int WM_, int WN_, int MF_, int NF_, int ST_ = 2> struct I8Big {
    static constexpr int WM = WM_, WN = WN_, MF = MF_, NF = NF_, ST = ST_;
    static constexpr int BM = 16 * MF * WM, BN = 16 * NF * WN, kThreads = 64 * WM * WN;
    static constexpr int kSlice = (BM + BN) * 128, kCopies = (BM + BN) / 8;
    static constexpr int D = (kCopies + WM * WN - 1) / (WM * WN);
    static constexpr int kLds = ST * kSlice;
    static_assert(kLds <= 160 * 1024 && D * (ST - 1) <= 63, "tile");
};

template <class G>
__global__ __launch_bounds__(G::kThreads) void k_i8_big(I8Args a, int n_ct, int n_tt) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int MF = G::MF, NF = G::NF, D = G::D, NW = G::WM * G::WN, ST = G::ST;
    const int total = n_ct * n_tt, per = (total + 7) / 8;
    const int L = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || L >= total) return;  // the whole workgroup
    const int tt = L % n_tt, ct = L / n_tt;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wn = wv % G::WN, wm = wv / G::WN;
    const int o0 = ct * G::BM, t0 = tt * G::BN, rb = a.row_bytes;

    const int w_rows = min(G::BM, a.out_dim - o0), x_rows = min(G::BN, a.n_tok - t0);
    const bl_rsrc rw = bl_make_rsrc(a.w + (size_t)o0 * rb, (uint32_t)w_rows * (uint32_t)rb);
    const bl_rsrc rx = bl_make_rsrc(a.xq + (size_t)t0 * rb, (uint32_t)x_rows * (uint32_t)rb);
    const uint32_t lds0 = bl_lds(smem);
    // copy c: 8 rows of channels (c < BM / 8) or tokens; rows behind the last
    // repeat it (their products are not stored)
    uint32_t off[D];
#pragma unroll
    for (int p = 0; p < D; p++) {
        const int c = min(wv + NW * p, G::kCopies - 1);
        const bool is_w = c < G::BM / 8;
        const int row = (is_w ? 8 * c : 8 * c - G::BM) + (lane >> 3);
        off[p] = (uint32_t)min(row, (is_w ? w_rows : x_rows) - 1) * (uint32_t)rb +
                 16u * (uint32_t)((lane & 7) ^ i8_key(row));
    }
    const int n_sl = (rb + 127) / 128;
    auto copy1 = [&](int i, int buf, int p) {
        const int c = min(wv + NW * p, G::kCopies - 1);
        const bool is_w = c < G::BM / 8;
        uint32_t o = off[p] + 128u * (uint32_t)i;
        if (128 * i + 128 > rb) {  // half a slice: zeros behind the row
            const int row = (is_w ? 8 * c : 8 * c - G::BM) + (lane >> 3);
            if (((lane & 7) ^ i8_key(row)) >= 4) o = 0xFFFFFFF0u;
        }
        const bl_rsrc r = is_w ? rw : rx;
        bl_dma16(bl_rsrc{r[0], r[1], i < n_sl ? r[2] : 0u, r[3]}, o, 0,
                 lds0 + (uint32_t)(buf * G::kSlice + c * 1024));
    };
    i8_v4 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) acc[m][n] = i8_v4{0, 0, 0, 0};
    const int r16 = lane & 15, q = lane >> 4;
    const uint8_t *const lw = smem + (wm * 16 * MF + r16) * 128;
    const uint8_t *const lx = smem + (G::BM + wn * 16 * NF + r16) * 128;
    const int s0 = 16 * (q ^ i8_key(r16)), s1 = s0 ^ 64;
    i8_v4 f[2][MF + NF];  // operands of a half slice: NF of tokens, MF of channels
    auto read1 = [&](int h, int buf, int j) {
        const int so = (h ? s1 : s0) + buf * G::kSlice;
        f[h][j] = j < NF ? *reinterpret_cast<const i8_v4 *>(lx + j * 2048 + so)
                         : *reinterpret_cast<const i8_v4 *>(lw + (j - NF) * 2048 + so);
    };
    // the MFMAs of half h; between them the reads of the other half's next
    // operands (from slice buffer rbuf) and, with `cp`, the copies of slice i
    auto phase = [&](auto h_c, int rbuf, bool rd, int i, int cbuf, bool cp) __attribute__((always_inline)) {
        constexpr int h = decltype(h_c)::value;
#pragma unroll
        for (int m = 0; m < MF; m++) {
            if (rd) {
#pragma unroll
                for (int j = m * (MF + NF) / MF; j < (m + 1) * (MF + NF) / MF; j++) read1(h ^ 1, rbuf, j);
            }
            if (cp) {
#pragma unroll
                for (int p = m * D / MF; p < (m + 1) * D / MF; p++) copy1(i, cbuf, p);
            }
#pragma unroll
            for (int n = 0; n < NF; n++)
                acc[m][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[h][NF + m], f[h][n], acc[m][n], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int i = 0; i < ST; i++)
#pragma unroll
        for (int p = 0; p < D; p++) copy1(i, i, p);
    bl_barrier<D *(ST - 1)>();
#pragma unroll
    for (int j = 0; j < MF + NF; j++) read1(0, 0, j);
    int buf = 0;
    for (int i = 0; i < n_sl; i++) {
        const int next = buf + 1 == ST ? 0 : buf + 1;
        phase(std::integral_constant<int, 0>{}, buf, true, 0, 0, false);
        bl_barrier<D *(ST - 2)>();
        phase(std::integral_constant<int, 1>{}, next, true, i + ST, buf, true);
        buf = next;
    }
    bl_wait<0>();  // (the copies past the last slice, zeros, land in the ring too)
    const uint32_t esz = a.dtype_out == T_F32 ? 4u : 2u;
    const bool vec = ((uintptr_t)a.out % (4 * esz)) == 0 && a.out_stride % 4 == 0 &&
                     ((uintptr_t)a.wscale % 16) == 0 && ((uintptr_t)a.bias % 16) == 0;
#pragma unroll
    for (int n = 0; n < NF; n++)
#pragma unroll
        for (int m = 0; m < MF; m++)
            i8_finish(a, acc[m][n], o0 + 16 * (wm * MF + m) + 4 * q, t0 + 16 * (wn * NF + n) + r16, vec);
}

template <class G> hipError_t i8_big_go(const I8Args &a, hipStream_t s) {
    const hipError_t e = i8_allow_lds<G>(reinterpret_cast<const void *>(&k_i8_big<G>));
    if (e != hipSuccess) return e;
    const int n_ct = (a.out_dim + G::BM - 1) / G::BM, n_tt = (a.n_tok + G::BN - 1) / G::BN;
    const long long wgs = ((long long)n_ct * n_tt + 7) / 8 * 8;
    k_i8_big<G><<<(unsigned)wgs, G::kThreads, G::kLds, s>>>(a, n_ct, n_tt);
    return hipGetLastError();
}

// The same with the ring cut finer: five units of one operand's slice, so that
// the channels, which come from memory, are copied two slices ahead and the
// tokens, which other workgroups read as well, one. (224 x 256, 2048 tokens of
// 14336 x 4096: 117 us with bf16 outputs, 2.06 POP/s; matrix cores busy in 47% of
// the cycles. With two slices of 256 x 256 and f32 outputs, 28 of 133 us went with
// the stores and another 18 with the copies to LDS.)
template <int WM_, int WN_, int MF_, int NF_> struct I8Wide {
    static constexpr int WM = WM_, WN = WN_, MF = MF_, NF = NF_;
    static constexpr int BM = 16 * MF * WM, BN = 16 * NF * WN, kThreads = 64 * WM * WN;
    static constexpr int kUnit = (BM > BN ? BM : BN) * 128, kLds = 5 * kUnit;
    static constexpr int DW = (BM / 8 + WM * WN - 1) / (WM * WN), DX = (BN / 8 + WM * WN - 1) / (WM * WN);
    static_assert(kLds <= 160 * 1024, "tile");
};

template <class G>
__global__ __launch_bounds__(G::kThreads) void k_i8_wide(I8Args a, int n_ct, int n_tt) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int MF = G::MF, NF = G::NF, NW = G::WM * G::WN, DW = G::DW, DX = G::DX;
    const int total = n_ct * n_tt, per = (total + 7) / 8;
    const int L = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || L >= total) return;  // the whole workgroup
    const int tt = L % n_tt, ct = L / n_tt;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wn = wv % G::WN, wm = wv / G::WN;
    const int o0 = ct * G::BM, t0 = tt * G::BN, rb = a.row_bytes;

    const int w_rows = min(G::BM, a.out_dim - o0), x_rows = min(G::BN, a.n_tok - t0);
    const bl_rsrc rw = bl_make_rsrc(a.w + (size_t)o0 * rb, (uint32_t)w_rows * (uint32_t)rb);
    const bl_rsrc rx = bl_make_rsrc(a.xq + (size_t)t0 * rb, (uint32_t)x_rows * (uint32_t)rb);
    const uint32_t lds0 = bl_lds(smem);
    // copy p of an operand: 8 rows; rows behind the last repeat it (their
    // products are not stored)
    uint32_t ow[DW], ox[DX];
    auto at = [&](int p, int copies, int rows) {
        const int row = 8 * min(wv + NW * p, copies - 1) + (lane >> 3);
        return (uint32_t)min(row, rows - 1) * (uint32_t)rb + 16u * (uint32_t)((lane & 7) ^ i8_key(row));
    };
#pragma unroll
    for (int p = 0; p < DW; p++) ow[p] = at(p, G::BM / 8, w_rows);
#pragma unroll
    for (int p = 0; p < DX; p++) ox[p] = at(p, G::BN / 8, x_rows);
    const int n_sl = (rb + 127) / 128;
    auto copy1 = [&](const bl_rsrc &r, uint32_t o, int copies, int i, int unit, int p) {
        const int c = min(wv + NW * p, copies - 1);
        o += 128u * (uint32_t)i;
        if (128 * i + 128 > rb && ((lane & 7) ^ i8_key(8 * c + (lane >> 3))) >= 4) o = 0xFFFFFFF0u;
        bl_dma16(bl_rsrc{r[0], r[1], i < n_sl ? r[2] : 0u, r[3]}, o, 0, lds0 + (uint32_t)(unit * G::kUnit + c * 1024));
    };
    auto copy_w = [&](int i, int unit, int p) { copy1(rw, ow[p], G::BM / 8, i, unit, p); };
    auto copy_x = [&](int i, int unit, int p) { copy1(rx, ox[p], G::BN / 8, i, unit, p); };
    i8_v4 acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) acc[m][n] = i8_v4{0, 0, 0, 0};
    const int r16 = lane & 15, q = lane >> 4;
    const uint8_t *const lw = smem + (wm * 16 * MF + r16) * 128;
    const uint8_t *const lx = smem + (wn * 16 * NF + r16) * 128;
    const int s0 = 16 * (q ^ i8_key(r16)), s1 = s0 ^ 64;
    i8_v4 f[2][MF + NF];  // operands of a half slice: NF of tokens, MF of channels
    auto read1 = [&](int h, int uw, int ux, int j) {
        const int so = h ? s1 : s0;
        f[h][j] = j < NF ? *reinterpret_cast<const i8_v4 *>(lx + j * 2048 + so + ux * G::kUnit)
                         : *reinterpret_cast<const i8_v4 *>(lw + (j - NF) * 2048 + so + uw * G::kUnit);
    };
    // phase h: its MFMAs, the other half's next operands read from (uw, ux), and
    // behind the barrier (h = 1) the copies of tokens i + 2 and channels i + 3
    auto phase = [&](auto h_c, int uw, int ux, int i, int fx, int fw) __attribute__((always_inline)) {
        constexpr int h = decltype(h_c)::value;
#pragma unroll
        for (int m = 0; m < MF; m++) {
#pragma unroll
            for (int j = m * (MF + NF) / MF; j < (m + 1) * (MF + NF) / MF; j++) read1(h ^ 1, uw, ux, j);
            if constexpr (h == 1) {
#pragma unroll
                for (int p = m * (DW + DX) / MF; p < (m + 1) * (DW + DX) / MF; p++) {
                    if (p < DX) copy_x(i + 2, fx, p);
                    else copy_w(i + 3, fw, p - DX);
                }
            }
#pragma unroll
            for (int n = 0; n < NF; n++)
                acc[m][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[h][NF + m], f[h][n], acc[m][n], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int i = 0; i < 3; i++) {
#pragma unroll
        for (int p = 0; p < DW; p++) copy_w(i, 2 * i, p);
        if (i < 2) {
#pragma unroll
            for (int p = 0; p < DX; p++) copy_x(i, 2 * i + 1, p);
        }
    }
    bl_barrier<2 * DW + DX>();
#pragma unroll
    for (int j = 0; j < MF + NF; j++) read1(0, 0, 1, j);
    int uw = 0, ux = 1;
    for (int i = 0; i < n_sl; i++) {
        const int nw = uw >= 3 ? uw - 3 : uw + 2, nx = ux >= 3 ? ux - 3 : ux + 2;
        phase(std::integral_constant<int, 0>{}, uw, ux, 0, 0, 0);
        bl_barrier<DW>();
        phase(std::integral_constant<int, 1>{}, nw, nx, i, uw, ux);
        uw = nw;
        ux = nx;
    }
    bl_wait<0>();  // (the copies past the last slice, zeros, land in the ring too)
    const uint32_t esz = a.dtype_out == T_F32 ? 4u : 2u;
    const bool vec = ((uintptr_t)a.out % (4 * esz)) == 0 && a.out_stride % 4 == 0 &&
                     ((uintptr_t)a.wscale % 16) == 0 && ((uintptr_t)a.bias % 16) == 0;
#pragma unroll
    for (int n = 0; n < NF; n++)
#pragma unroll
        for (int m = 0; m < MF; m++)
            i8_finish(a, acc[m][n], o0 + 16 * (wm * MF + m) + 4 * q, t0 + 16 * (wn * NF + n) + r16, vec);
}

template <class G> hipError_t i8_wide_go(const I8Args &a, hipStream_t s) {
    const hipError_t e = i8_allow_lds<G>(reinterpret_cast<const void *>(&k_i8_wide<G>));
    if (e != hipSuccess) return e;
    const int n_ct = (a.out_dim + G::BM - 1) / G::BM, n_tt = (a.n_tok + G::BN - 1) / G::BN;
    const long long wgs = ((long long)n_ct * n_tt + 7) / 8 * 8;
    k_i8_wide<G><<<(unsigned)wgs, G::kThreads, G::kLds, s>>>(a, n_ct, n_tt);
    return hipGetLastError();
}

}  // namespace

namespace {

bool i8_vec_ok(const void *x, size_t stride, uint32_t dtype) {
    const size_t n = dtype == T_F32 ? 4 : 2;
    return (uintptr_t)x % 16 == 0 && stride * n % 16 == 0;
}

template <int THREADS>
hipError_t i8_quantize_go(const void *x, size_t stride, int8_t *xq, float *scale, int n_tok, int in_dim,
                          uint32_t dtype, hipStream_t s) {
    const int rb = (int)i8_row_bytes(in_dim), vec = i8_vec_ok(x, stride, dtype);
    const dim3 g((unsigned)n_tok);
    if (dtype == T_F32) k_i8_quantize<T_F32, THREADS><<<g, THREADS, 0, s>>>(x, stride, xq, scale, in_dim, rb, vec);
    else if (dtype == T_F16) k_i8_quantize<T_F16, THREADS><<<g, THREADS, 0, s>>>(x, stride, xq, scale, in_dim, rb, vec);
    else k_i8_quantize<T_BF16, THREADS><<<g, THREADS, 0, s>>>(x, stride, xq, scale, in_dim, rb, vec);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_i8_quantize(const void *x, size_t stride, int8_t *xq, float *scale, int n_tok,
                              int in_dim, uint32_t dtype, hipStream_t s) {
    if (n_tok <= 0) return hipSuccess;
    // a lane holds 16 elements of its row between the two looks at it
    if (in_dim <= 1024) return i8_quantize_go<64>(x, stride, xq, scale, n_tok, in_dim, dtype, s);
    if (in_dim <= 4096) return i8_quantize_go<256>(x, stride, xq, scale, n_tok, in_dim, dtype, s);
    return i8_quantize_go<512>(x, stride, xq, scale, n_tok, in_dim, dtype, s);
}

bool i8_one_supported(int in_dim) { return in_dim <= 60 * 1024; }  // its codes in LDS

// One token, us, against the quantiser and a tile product, the weights from memory:
// 14336 x 4096 f32 14.4 / 17.1 (59 MB: 4.1 TB/s; 13.0 where three matrices take turns,
// which the cache behind L2 holds in part; a launch that only reads as much 10.2 and
// 9.2), 4096 x 14336 18.4 / 18.7 (bf16 15.7 / 17.4), 4096 x 4096 bf16 5.7 / 7.5,
// 1024 x 1024 2.9 / 5.3.
hipError_t launch_i8_one(const I8Args &a, const void *x, int in_dim, uint32_t dtype, hipStream_t s) {
    if (!i8_one_supported(in_dim) || a.n_tok != 1) return hipErrorNotSupported;
    const int kp = (in_dim + 1023) / 1024 * 1024, vec = i8_vec_ok(x, 0, dtype);
    const dim3 g((unsigned)((a.out_dim + 15) / 16));
    if (dtype == T_F32) k_i8_one<T_F32><<<g, 256, kp, s>>>(a, x, in_dim, kp, vec);
    else if (dtype == T_F16) k_i8_one<T_F16><<<g, 256, kp, s>>>(a, x, in_dim, kp, vec);
    else k_i8_one<T_BF16><<<g, 256, kp, s>>>(a, x, in_dim, kp, vec);
    return hipGetLastError();
}

namespace {

// A kernel of the product and what it takes, by an estimate in us:
//   us = c0 + r c1 + (L per CU or r) slices c2
// with L workgroups a CU, r of them one after the other (at most `occ` run at
// once), `slices` of 128 bytes a wavefront. The constants are fitted to 122 sizes (3
// to 2048 tokens, weights from memory), those of the two widest tiles set by hand
// from a few products. Slower than the fastest of the thirteen: 1.4% on average and
// 12% at most at those sizes; at sizes that no constant was taken from, 1.7% and 15%
// (70 sizes, 2 to 3000 tokens) and 0.2% and 3% (40 products of 20 to 900 GOP).
struct I8Kernel {
    hipError_t (*go)(const I8Args &, hipStream_t);
    int bm, bn, wk, occ;
    float c0, c1, c2;
    float us(int n_tok, int out_dim, int row_bytes) const {
        const long long tiles = (long long)((out_dim + bm - 1) / bm) * ((n_tok + bn - 1) / bn);
        const long long L = (tiles + 255) / 256, r = (L + occ - 1) / occ;
        const int slices = ((row_bytes + 127) / 128 + wk - 1) / wk;
        return c0 + (float)r * c1 + (float)(occ > 1 ? L : r) * (float)slices * c2;
    }
};
template <int WM, int WN, int WK, int MF, int NF, int ST>
constexpr I8Kernel i8_tile(int occ, float c0, float c1, float c2) {
    using G = I8Tile<WM, WN, WK, MF, NF, ST>;
    return {&i8_tile_go<G>, G::BM, G::BN, WK, occ, c0, c1, c2};
}
template <int WM, int WN, int MF, int NF>
constexpr I8Kernel i8_wide(int occ, float c0, float c1, float c2) {
    using G = I8Wide<WM, WN, MF, NF>;
    return {&i8_wide_go<G>, G::BM, G::BN, 1, occ, c0, c1, c2};
}
template <int WM, int WN, int MF, int NF, int ST>
constexpr I8Kernel i8_big(int occ, float c0, float c1, float c2) {
    using G = I8Big<WM, WN, MF, NF, ST>;
    return {&i8_big_go<G>, G::BM, G::BN, 1, occ, c0, c1, c2};
}
const I8Kernel kI8Kernels[] = {
    i8_tile<1, 1, 4, 1, 1, 3>(3, 1.64f, 1.30f, 0.180f),  // 16 channels x 16 tokens
    i8_tile<1, 1, 4, 2, 1, 3>(2, 1.37f, 1.46f, 0.271f),  // 32 x 16
    i8_tile<1, 1, 4, 2, 2, 3>(1, 1.10f, 1.62f, 0.382f),  // 32 x 32
    i8_tile<1, 1, 4, 2, 3, 3>(1, 0.81f, 2.33f, 0.458f),  // 32 x 48
    i8_tile<1, 1, 4, 2, 4, 3>(1, 1.02f, 2.58f, 0.528f),  // 32 x 64
    i8_big<4, 2, 1, 2, 5>(2, 0.0f, 3.22f, 0.207f),       // 64 x 64
    i8_big<2, 4, 2, 2, 4>(1, 0.0f, 3.83f, 0.311f),       // 64 x 128
    i8_big<2, 4, 4, 2, 4>(1, 0.0f, 5.12f, 0.400f),       // 128 x 128
    i8_big<4, 2, 3, 4, 3>(1, 0.0f, 5.14f, 0.562f),       // 192 x 128
    i8_big<2, 4, 8, 2, 3>(1, 0.0f, 6.81f, 0.696f),       // 256 x 128
    i8_big<2, 4, 6, 3, 3>(1, 0.0f, 6.48f, 0.727f),       // 192 x 192
    i8_wide<2, 4, 7, 4>(1, 0.0f, 6.4f, 1.08f),           // 224 x 256
    i8_wide<2, 4, 8, 4>(1, 0.0f, 6.7f, 1.18f),           // 256 x 256
};

}  // namespace

hipError_t launch_i8_matmul(const I8Args &a, hipStream_t s) {
    if (a.n_tok <= 0) return hipSuccess;
    const I8Kernel *best = nullptr;
    float us = 0.0f;
    for (const I8Kernel &k : kI8Kernels) {
        const float t = k.us(a.n_tok, a.out_dim, a.row_bytes);
        if (!best || t < us) {
            best = &k;
            us = t;
        }
    }
    return best->go(a, s);
}

}  // namespace rsllm_hip
