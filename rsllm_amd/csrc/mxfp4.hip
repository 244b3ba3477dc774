// MXFP4 rows: quantising, decoding, and the product of two code matrices.
#include "buffer_lds.h"
#include "mxfp4_product.h"

#include <algorithm>
#include <climits>
#include <atomic>
#include <type_traits>

namespace rsllm_hip {

namespace {

// A magnitude's bits: in the order of the magnitudes, inf and NaN above every number.
__device__ __forceinline__ uint32_t mx_abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

// The largest of four neighbouring lanes' values, at each of them.
__device__ __forceinline__ uint32_t mx_max4(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));  // quad_perm 2 3 0 1
}

// A block's scale byte from its largest magnitude's bits: the exponent less 2, at
// least 0 (subnormal magnitudes are below 2^-125 as well), 255 where not finite.
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t big) {
    const uint32_t e = big >> 23;
    return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// n / groups: in 32 bits where they do.
__device__ __forceinline__ size_t mx_row_of(size_t n, int groups) {
    return n >> 32 ? n / (size_t)groups : (size_t)((uint32_t)n / (uint32_t)groups);
}

// Eight elements (four neighbouring lanes hold a block) as codes; s: the block's scale.
__device__ __forceinline__ uint32_t mx_quantize8(const float (&v)[8], uint32_t &s) {
    uint32_t big = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) big = max(big, mx_abs_bits(v[k]));
    s = mx_scale_of(mx_max4(big));
    uint32_t c = 0;
    if (s != 255u) {
        const float unit = mx_unit(s);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], unit, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], unit, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], unit, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], unit, 3);
    }
    return c;
}

}  // namespace

// A lane's eight elements at a time, four lanes a block: `groups` of eight a row (its
// padding included). The block's largest magnitude is found among its four lanes by DPP,
// and one instruction then divides two elements by the block's power of two, rounds them
// to nearest even and saturates. One read and one write of everything, so the bytes bound
// it: 14336 x 4096 bf16 (149 MB in and out) 32.8 us, 4.5 TB/s, a large copy's rate. One
// row of 4096 f32: 1.8 us, a launch.
template <uint32_t DT>
__global__ __launch_bounds__(256) void k_mx_quantize(const void *__restrict__ x, size_t stride,
                                                     uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                     size_t total, int groups, int in_dim, int vec) {
    const size_t rb = (size_t)groups * 4, sb = mx_scale_bytes(in_dim);
    for (size_t n = (size_t)blockIdx.x * 256 + threadIdx.x; n < total; n += (size_t)gridDim.x * 256) {
        const size_t row = mx_row_of(n, groups);
        const int g = (int)(n - row * (size_t)groups), i = 8 * g;
        float v[8];
        mx_load8<DT>(x, row * stride, i, in_dim, vec, v);
        uint32_t s;
        const uint32_t c = mx_quantize8(v, s);
        *reinterpret_cast<uint32_t *>(codes + row * rb + 4 * g) = c;
        uint8_t *const sr = scales + row * sb;
        if ((g & 3) == 0) sr[g >> 2] = (uint8_t)s;
        if (g == groups - 1)
            for (size_t b = (size_t)groups / 4; b < sb; b++) sr[b] = 0;
    }
}

// 2^(s - 127) in f32, which holds 2^-127 too; 255: NaN.
__device__ __forceinline__ float mx_unit_f32(uint32_t s) {
    return __builtin_bit_cast(float, s == 0 ? 0x00400000u : s == 255u ? 0x7FC00000u : s << 23);
}

// A lane's eight elements at a time, decoded by the conversion instruction and multiplied
// by the block's power of two in f32, which rounds only what is below 2^-126 and
// overflows only above f32's range, as the definition does. vec: rows of out are 16-byte
// aligned. The bytes bound it: 14336 x 4096 to bf16 (149 MB) 24 us where the codes were
// written just before and come from a cache, 117 MB of writes at 4.9 TB/s; an element a lane,
// a table and ldexp took 86 us. One row of 4096 f32: 1.9 us, a launch.
template <uint32_t DT>
__global__ __launch_bounds__(256) void k_mx_dequantize(const uint8_t *__restrict__ codes,
                                                       const uint8_t *__restrict__ scales, void *__restrict__ out,
                                                       size_t stride, size_t total, int groups, int in_dim, int vec) {
    const size_t rb = mx_row_bytes(in_dim), sb = mx_scale_bytes(in_dim);
    for (size_t n = (size_t)blockIdx.x * 256 + threadIdx.x; n < total; n += (size_t)gridDim.x * 256) {
        const size_t row = mx_row_of(n, groups);
        const int g = (int)(n - row * (size_t)groups);
        const uint32_t c = *reinterpret_cast<const uint32_t *>(codes + row * rb + 4 * g);
        const float unit = mx_unit_f32(scales[row * sb + (g >> 2)]);
        float v[8];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            typedef float f2 __attribute__((ext_vector_type(2)));
            f2 p;
            if (k == 0) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
            else if (k == 1) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
            else if (k == 2) p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
            else p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
            v[2 * k] = p[0] * unit;
            v[2 * k + 1] = p[1] * unit;
        }
        const size_t at = row * stride + 8 * g;
        if (vec && 8 * g + 8 <= in_dim) {
            const mx_v4f lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
            const float4 zero = make_float4(-0.0f, -0.0f, -0.0f, -0.0f);  // (-0 + -0 is -0, and +0 + -0 is +0)
            if constexpr (DT == T_F32) {
                float4 *const d = reinterpret_cast<float4 *>(static_cast<float *>(out) + at);
                d[0] = make_float4(v[0], v[1], v[2], v[3]);
                d[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                const uint2 a = mx_pack<DT>(lo, zero), b = mx_pack<DT>(hi, zero);
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + at) = make_uint4(a.x, a.y, b.x, b.y);
            }
        } else {
            for (int k = 0; k < 8 && 8 * g + k < in_dim; k++) mx_store(out, at + k, v[k], DT);
        }
    }
}

// ---- the product -------------------------------------------------------------------

namespace {

// ---- few tokens: the weights streamed into registers ----------------------------------
//
// A workgroup's tile: 16 MF channels x 16 NF tokens; its WK wavefronts take every WK-th
// piece of 512 codes, and their sums are added through LDS. A lane reads 16 codes' bytes
// of a row for each step of 128 and the 16 scale bytes of its row for the piece's four
// steps; the operands of the next piece are on their way while this one is multiplied. The
// weights' bytes bound it, for small ones the latency of a launch, one piece a wavefront and
// the sums' join: 14336 x 4096, one token, 31 MB, 9.6 to 10.7 us in traces' medians, 10.0 a
// call in a graph (a launch that only reads them 7.5); 4096 x 4096, 32 tokens, 6.5; 1001 x 2000, 77 tokens, 4.6. K is split over
// the wavefronts since few channels a workgroup fill the chip (4096 channels: 256 or 128
// workgroups), and since a lane that streams rows into registers needs no LDS and no barrier.
template <int MF_, int NF_, int WK_> struct MxFew {
    static constexpr int MF = MF_, NF = NF_, WK = WK_, BM = 16 * MF, BN = 16 * NF;
};
struct MxPiece {
    mx_v4u c[4], s;
};

// DX: kMxCodes, or the type of float tokens (up to kMxFloatTok, a.xf), of which every
// wavefront quantises its pieces for itself, through LDS, before it multiplies them: the same
// codes, and one launch less. With one and two tokens that takes 4.5 and 4.8 us at 4096 x
// 4096 f32 in place of 6.6 and 6.7, 10.0 and 10.8 in place of 12.6 and 12.9 at 14336 x 4096.
// Every workgroup repeats it, though, and a wavefront waits for each piece's codes: with four
// tokens (in a build of up to eight) 5.7 in place of 6.9 and 12.9 in place of 13.4, but 14.3
// in place of 12.0 where rows are 14336 long, with eight 7.5 and 7.1, 16.5 and 13.8.
constexpr uint32_t kMxCodes = ~0u;
constexpr int kMxFloatTok = 2, kMxFloatPitch = 256 + 16;  // (16: the row's scales)

template <class G, uint32_t DX> __global__ __launch_bounds__(64 * G::WK) void k_mx_few(MxArgs a, int n_ct) {
    constexpr int MF = G::MF, NF = G::NF, WK = G::WK;
    constexpr bool kFloat = DX != kMxCodes;
    static_assert(!kFloat || NF == 1, "few tokens");
    constexpr int kRed = WK * MF * NF * 1024, kTok = kFloat ? WK * kMxFloatTok * kMxFloatPitch : 0;
    __shared__ __align__(16) uint8_t red[kRed > kTok ? kRed : kTok];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int o0 = (blockIdx.x % n_ct) * G::BM, t0 = (blockIdx.x / n_ct) * G::BN;
    const size_t rb = mx_row_bytes(a.in_dim), sb = mx_scale_bytes(a.in_dim);
    const int blocks = (a.in_dim + 31) / 32, pieces = (int)(sb / 16), steps = (int)(rb / 64);
    const uint8_t *w[MF], *ws[MF], *x[NF], *xs[NF];
#pragma unroll
    for (int m = 0; m < MF; m++) {
        const size_t row = (size_t)min(o0 + 16 * m + r, a.out_dim - 1);
        w[m] = a.w + row * rb + 16 * q;
        ws[m] = a.ws + row * sb;
    }
#pragma unroll
    for (int n = 0; n < NF; n++) {
        const size_t row = (size_t)min(t0 + 16 * n + r, a.n_tok - 1);
        x[n] = a.x + row * rb + 16 * q;
        xs[n] = a.xs + row * sb;
    }
    auto load = [&](MxPiece &p, const uint8_t *c, const uint8_t *s, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            p.c[j] = mx_v4u{0, 0, 0, 0};
            if (4 * i + j < steps) p.c[j] = *reinterpret_cast<const mx_v4u *>(c + 256 * (size_t)i + 64 * j);
        }
        p.s = *reinterpret_cast<const mx_v4u *>(s + 16 * (size_t)i);
    };
    mx_v4f acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) acc[m][n] = mx_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    MxPiece pw[MF], px[NF];
    float xf[kFloat ? kMxFloatTok : 1][8];
    auto fetch = [&](int i) __attribute__((always_inline)) {
        if (i < pieces) {
            if constexpr (kFloat) {  // (first: loads return in order, and these come from near)
#pragma unroll
                for (int t = 0; t < kMxFloatTok; t++)
                    if (t < a.n_tok) mx_load8<DX>(a.xf, (size_t)t * a.x_stride, 512 * i + 8 * lane, a.in_dim, a.x_vec, xf[t]);
            }
#pragma unroll
            for (int m = 0; m < MF; m++) load(pw[m], w[m], ws[m], i);
            if constexpr (!kFloat) {
#pragma unroll
                for (int n = 0; n < NF; n++) load(px[n], x[n], xs[n], i);
            }
        }
    };
    uint8_t *const mine = red + wv * kMxFloatTok * kMxFloatPitch;  // this wavefront's tokens
    fetch(wv);
    for (int i = wv; i < pieces; i += WK) {
        MxPiece cw[MF], cx[NF];
#pragma unroll
        for (int m = 0; m < MF; m++) cw[m] = pw[m];
        if constexpr (kFloat) {
#pragma unroll
            for (int t = 0; t < kMxFloatTok; t++) {
                if (t < a.n_tok) {
                    uint32_t s;
                    const uint32_t c = mx_quantize8(xf[t], s);
                    *reinterpret_cast<uint32_t *>(mine + t * kMxFloatPitch + 4 * lane) = c;
                    if (lane % 4 == 0) mine[t * kMxFloatPitch + 256 + lane / 4] = (uint8_t)s;
                }
            }
            __builtin_amdgcn_wave_barrier();
            // (columns behind the last token repeat one)
            const uint8_t *const src = mine + (r < a.n_tok ? r : 0) * kMxFloatPitch;
#pragma unroll
            for (int j = 0; j < 4; j++) cx[0].c[j] = *reinterpret_cast<const mx_v4u *>(src + 64 * j + 16 * q);
            cx[0].s = *reinterpret_cast<const mx_v4u *>(src + 256);
            __builtin_amdgcn_wave_barrier();
        } else {
#pragma unroll
            for (int n = 0; n < NF; n++) cx[n] = px[n];
        }
        fetch(i + WK);
        // (scales behind a row's last block may be anything: there 1)
        const bool tail = 16 * i + 16 > blocks;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (4 * i + j < steps) {
                const bool in = !tail || 16 * i + 4 * j + q < blocks;
                int sw[MF], sx[NF];
#pragma unroll
                for (int m = 0; m < MF; m++) sw[m] = in ? (int)(cw[m].s[j] >> (8 * q)) : 127;
#pragma unroll
                for (int n = 0; n < NF; n++) sx[n] = in ? (int)(cx[n].s[j] >> (8 * q)) : 127;
#pragma unroll
                for (int m = 0; m < MF; m++)
#pragma unroll
                    for (int n = 0; n < NF; n++) acc[m][n] = mx_mfma(cw[m].c[j], cx[n].c[j], acc[m][n], sw[m], sx[n]);
            }
        }
    }
    if constexpr (kFloat) __syncthreads();
    mx_v4f *const part = reinterpret_cast<mx_v4f *>(red);
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) part[(wv * MF * NF + m * NF + n) * 64 + lane] = acc[m][n];
    __syncthreads();
    const bool vec = mx_vec(a);
    for (int f = wv; f < MF * NF; f += WK) {
        mx_v4f s = part[f * 64 + lane];
#pragma unroll
        for (int k = 1; k < WK; k++) s += part[(k * MF * NF + f) * 64 + lane];
        const int o = o0 + 16 * (f / NF) + 4 * q;
        mx_finish(a, s, mx_bias(a, o), o, t0 + 16 * (f % NF) + r, vec);
    }
}

template <class G> hipError_t mx_few_go(const MxArgs &a, hipStream_t s) {
    const int n_ct = (a.out_dim + G::BM - 1) / G::BM, n_tt = (a.n_tok + G::BN - 1) / G::BN;
    k_mx_few<G, kMxCodes><<<(unsigned)n_ct * (unsigned)n_tt, 64 * G::WK, 0, s>>>(a, n_ct);
    return hipGetLastError();
}
// Of a.xf, dtype_x.
template <class G> hipError_t mx_few_float_go(const MxArgs &a, uint32_t dtype_x, hipStream_t s) {
    const unsigned n_ct = (unsigned)((a.out_dim + G::BM - 1) / G::BM), n = 64 * G::WK;
    if (dtype_x == T_F32) k_mx_few<G, T_F32><<<n_ct, n, 0, s>>>(a, (int)n_ct);
    else if (dtype_x == T_F16) k_mx_few<G, T_F16><<<n_ct, n, 0, s>>>(a, (int)n_ct);
    else k_mx_few<G, T_BF16><<<n_ct, n, 0, s>>>(a, (int)n_ct);
    return hipGetLastError();
}

// ---- many tokens: both operands through LDS -------------------------------------------
//
// A workgroup's tile: BM = 16 MF WM channels x BN = 16 NF WN tokens, a wavefront 16 MF x
// 16 NF of it. Slices of 128 bytes (256 codes) of both operands are copied to LDS ST deep;
// the scales, 16 bytes a row for two slices, into a ring of their own. The operands of a
// slice's next half are read into registers while the matrix cores work on this one. One
// barrier a slice, in its middle: behind it the next slice has landed, and every
// wavefront holds what is left of this one in registers, so the slice ST further on can be
// copied over it. 300 tokens of 4096 to 2048 channels: 11.4 us with 64 x 64 (160 workgroups;
// half a us a slice, most of it waits: deeper rings of 6 and 8 slices were no faster);
// 1000 of 4100 to 5000: 26 with 192 x 128 (1.6 PFLOP/s), 2048 of 2048 to 2048: 12.2 with
// 128 x 128 (1.4 PFLOP/s).
template <int WM_, int WN_, int MF_, int NF_, int ST_> struct MxBig {
    static constexpr int WM = WM_, WN = WN_, MF = MF_, NF = NF_, ST = ST_, NW = WM * WN;
    static constexpr int BM = 16 * MF * WM, BN = 16 * NF * WN, kThreads = 64 * NW;
    static constexpr int kSlice = (BM + BN) * 128, kCopies = (BM + BN) / 8;
    static constexpr int D = (kCopies + NW - 1) / NW;
    // scales: a copy brings 64 rows of 16 bytes; the channels' with the even slices, the
    // tokens' of the next two slices with the odd ones
    static constexpr int kRows = BM > BN ? BM : BN, kScaleCopies = (kRows + 63) / 64;
    static constexpr int DS = (kScaleCopies + NW - 1) / NW, kPairs = ST / 2 + 2;
    static constexpr int kScaleSlot = kScaleCopies * 1024;  // of one operand, two slices
    static constexpr int kRing = ST * kSlice, kLds = kRing + kPairs * 2 * kScaleSlot;
    // P fragments' rows interleaved, so that a lane ends up with 4 P consecutive channels
    static constexpr int P = MF % 4 == 0 ? 4 : MF % 2 == 0 ? 2 : 1;
    static_assert(kLds <= 160 * 1024 && (D + DS) * (ST - 1) <= 63, "tile");
};
// Where byte 16 c of a row's slice lies: at place c ^ key, so that the 16 rows which an
// operand read takes at one c are spread over all banks.
template <int P> __device__ __forceinline__ constexpr int mx_key(int row) {
    return ((row >> 1) & 1) | ((row / (4 * P)) & 3) << 1;
}

template <class G> __global__ __launch_bounds__(G::kThreads) void k_mx_big(MxArgs a, int n_ct, int n_tt) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int MF = G::MF, NF = G::NF, D = G::D, DS = G::DS, NW = G::NW, ST = G::ST, P = G::P;
    // Workgroups go round the 8 XCDs: each takes a run of tiles, token tiles fastest, so
    // the tiles that share a weight row are behind one L2.
    const int total = n_ct * n_tt, per = (total + 7) / 8;
    const int L = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || L >= total) return;  // the whole workgroup
    const int tt = L % n_tt, ct = L / n_tt;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wn = wv % G::WN, wm = wv / G::WN;
    const int o0 = ct * G::BM, t0 = tt * G::BN;
    const uint32_t rb = (uint32_t)mx_row_bytes(a.in_dim), sb = (uint32_t)mx_scale_bytes(a.in_dim);
    const int blocks = (a.in_dim + 31) / 32, n_sl = (int)((rb + 127) / 128);

    const int w_rows = min(G::BM, a.out_dim - o0), x_rows = min(G::BN, a.n_tok - t0);
    const bl_rsrc rw = bl_make_rsrc(a.w + (size_t)o0 * rb, (uint32_t)w_rows * rb);
    const bl_rsrc rx = bl_make_rsrc(a.x + (size_t)t0 * rb, (uint32_t)x_rows * rb);
    const bl_rsrc rws = bl_make_rsrc(a.ws + (size_t)o0 * sb, (uint32_t)w_rows * sb);
    const bl_rsrc rxs = bl_make_rsrc(a.xs + (size_t)t0 * sb, (uint32_t)x_rows * sb);
    const uint32_t lds0 = bl_lds(smem);
    // copy c: 8 rows of channels (c < BM / 8) or tokens; rows behind the last repeat it
    // (their products are not stored)
    uint32_t off[D];
    bool half[D];  // this lane's 16 bytes lie in the slice's second half
#pragma unroll
    for (int p = 0; p < D; p++) {
        const int c = min(wv + NW * p, G::kCopies - 1);
        const bool is_w = c < G::BM / 8;
        const int row = (is_w ? 8 * c : 8 * c - G::BM) + (lane >> 3);
        const int at = (lane & 7) ^ (is_w ? mx_key<P>(row) : mx_key<1>(row));
        off[p] = (uint32_t)min(row, (is_w ? w_rows : x_rows) - 1) * rb + 16u * (uint32_t)at;
        half[p] = at >= 4;
    }
    auto copy1 = [&](int i, int buf, int p) __attribute__((always_inline)) {
        const int c = min(wv + NW * p, G::kCopies - 1);
        const bool is_w = c < G::BM / 8;
        uint32_t o = off[p] + 128u * (uint32_t)i;
        if (128u * (uint32_t)i + 128u > rb && half[p]) o = 0xFFFFFFF0u;  // zeros behind the row
        const bl_rsrc r = is_w ? rw : rx;
        bl_dma16(bl_rsrc{r[0], r[1], i < n_sl ? r[2] : 0u, r[3]}, o, 0, lds0 + (uint32_t)(buf * G::kSlice + c * 1024));
    };
    // the scales of pair j (slices 2 j and 2 j + 1) of the channels or the tokens
    auto copy_scales = [&](bool is_w, int j, int p) __attribute__((always_inline)) {
        const int c = min(wv + NW * p, G::kScaleCopies - 1), row = 64 * c + lane;
        const uint32_t o = (uint32_t)min(row, (is_w ? w_rows : x_rows) - 1) * sb + 16u * (uint32_t)j;
        const bl_rsrc r = is_w ? rws : rxs;
        bl_dma16(bl_rsrc{r[0], r[1], 2 * j < n_sl ? r[2] : 0u, r[3]}, o, 0,
                 lds0 + (uint32_t)(G::kRing + (j % G::kPairs * 2 + (is_w ? 0 : 1)) * G::kScaleSlot + c * 1024));
    };
    mx_v4f acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) acc[m][n] = mx_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int r16 = lane & 15, q = lane >> 4;
    // rows of this lane: of fragment m of the channels, n of the tokens
    const int wrow0 = wm * 16 * MF + mx_frag_row<P>(0, r16), xrow0 = wn * 16 * NF + r16;
    const uint8_t *const lw = smem + wrow0 * 128, *const lx = smem + (G::BM + xrow0) * 128;
    const uint8_t *const sw0 = smem + G::kRing + wrow0 * 16 + q, *const sx0 = smem + G::kRing + G::kScaleSlot + xrow0 * 16 + q;
    // (the key of every fragment's row r16 is that of fragment 0's)
    const int pw0 = 16 * (q ^ mx_key<P>(wrow0)), px0 = 16 * (q ^ mx_key<1>(xrow0));
    mx_v4u f[2][MF + NF];  // operands of a half slice: NF of tokens, MF of channels
    int sc[2][MF + NF];
    auto read1 = [&](int h, int buf, int i, int j) __attribute__((always_inline)) {
        const int slot = i / 2 % G::kPairs * 2 * G::kScaleSlot + 8 * (i & 1) + 4 * h;
        if (j < NF) {
            f[h][j] = *reinterpret_cast<const mx_v4u *>(lx + j * 2048 + (px0 ^ (64 * h)) + buf * G::kSlice);
            sc[h][j] = sx0[slot + j * 256];
        } else {
            const int row = mx_frag_row<P>(j - NF, 0);
            f[h][j] = *reinterpret_cast<const mx_v4u *>(lw + row * 128 + (pw0 ^ (64 * h)) + buf * G::kSlice);
            sc[h][j] = sw0[slot + row * 16];
        }
    };
    // the MFMAs of half h of slice i; between them the reads of the other half's next
    // operands (slice ri in buffer rbuf) and, with `cp`, the copies of slice i + ST
    auto phase = [&](auto h_c, int i, int rbuf, int ri, int cbuf, bool cp) __attribute__((always_inline)) {
        constexpr int h = decltype(h_c)::value;
        // (scales behind a row's last block may be anything: there 1)
        if (8 * i + 8 > blocks) {
#pragma unroll
            for (int j = 0; j < MF + NF; j++) sc[h][j] = 8 * i + 4 * h + q < blocks ? sc[h][j] : 127;
        }
#pragma unroll
        for (int m = 0; m < MF; m++) {
#pragma unroll
            for (int j = m * (MF + NF) / MF; j < (m + 1) * (MF + NF) / MF; j++) read1(h ^ 1, rbuf, ri, j);
            if (cp) {
#pragma unroll
                for (int p = m * D / MF; p < (m + 1) * D / MF; p++) copy1(i + ST, cbuf, p);
                if (m == MF - 1) {
                    const int s = i + ST;
#pragma unroll
                    for (int p = 0; p < DS; p++) copy_scales((s & 1) == 0, (s + 1) / 2, p);
                }
            }
#pragma unroll
            for (int n = 0; n < NF; n++)
                acc[m][n] = mx_mfma(f[h][NF + m], f[h][n], acc[m][n], sc[h][NF + m], sc[h][n]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int p = 0; p < DS; p++) copy_scales(false, 0, p);
#pragma unroll
    for (int i = 0; i < ST; i++) {
#pragma unroll
        for (int p = 0; p < D; p++) copy1(i, i, p);
#pragma unroll
        for (int p = 0; p < DS; p++) copy_scales((i & 1) == 0, (i + 1) / 2, p);
    }
    bl_barrier<(D + DS) * (ST - 1)>();
#pragma unroll
    for (int j = 0; j < MF + NF; j++) read1(0, 0, 0, j);
    int buf = 0;
    for (int i = 0; i < n_sl; i++) {
        const int next = buf + 1 == ST ? 0 : buf + 1;
        phase(std::integral_constant<int, 0>{}, i, buf, i, 0, false);
        bl_barrier<(D + DS) * (ST - 2)>();
        phase(std::integral_constant<int, 1>{}, i, next, i + 1, buf, true);
        buf = next;
    }
    bl_wait<0>();  // (the copies past the last slice, zeros, land in the ring too)
    mx_write_tile<MF, NF, G::WM, G::WN, P, G::kLds>(a, acc, smem, o0, t0, wm, wn);
}

template <class G> hipError_t mx_big_go(const MxArgs &a, hipStream_t s) {
    const hipError_t e = mx_allow_lds<G>(reinterpret_cast<const void *>(&k_mx_big<G>));
    if (e != hipSuccess) return e;
    const int n_ct = (a.out_dim + G::BM - 1) / G::BM, n_tt = (a.n_tok + G::BN - 1) / G::BN;
    const long long wgs = ((long long)n_ct * n_tt + 7) / 8 * 8;
    k_mx_big<G><<<(unsigned)wgs, G::kThreads, G::kLds, s>>>(a, n_ct, n_tt);
    return hipGetLastError();
}

}  // namespace

namespace {

bool mx_rows_vec(const void *p, size_t stride, uint32_t dtype) {
    return (uintptr_t)p % 16 == 0 && stride * (dtype == T_F32 ? 4 : 2) % 16 == 0;
}
// Workgroups of 256 for `total` threads' work, in turns behind 2^20 of them.
unsigned mx_grid(size_t total) { return (unsigned)std::min<size_t>((total + 255) / 256, (size_t)1 << 20); }

}  // namespace

hipError_t launch_mx_quantize(const void *x, size_t stride, uint8_t *codes, uint8_t *scales, int n_rows,
                              int in_dim, uint32_t dtype, hipStream_t s) {
    if (n_rows <= 0) return hipSuccess;
    const int groups = (int)mx_row_bytes(in_dim) / 4;
    const size_t total = (size_t)n_rows * groups;
    const int vec = mx_rows_vec(x, stride, dtype);
    const unsigned g = mx_grid(total);
    if (dtype == T_F32) k_mx_quantize<T_F32><<<g, 256, 0, s>>>(x, stride, codes, scales, total, groups, in_dim, vec);
    else if (dtype == T_F16) k_mx_quantize<T_F16><<<g, 256, 0, s>>>(x, stride, codes, scales, total, groups, in_dim, vec);
    else k_mx_quantize<T_BF16><<<g, 256, 0, s>>>(x, stride, codes, scales, total, groups, in_dim, vec);
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const uint8_t *codes, const uint8_t *scales, void *out, size_t stride,
                                int n_rows, int in_dim, uint32_t dtype, hipStream_t s) {
    if (n_rows <= 0) return hipSuccess;
    const int groups = (in_dim + 7) / 8;
    const size_t total = (size_t)n_rows * groups;
    const int vec = mx_rows_vec(out, stride, dtype);
    const unsigned g = mx_grid(total);
    if (dtype == T_F32) k_mx_dequantize<T_F32><<<g, 256, 0, s>>>(codes, scales, out, stride, total, groups, in_dim, vec);
    else if (dtype == T_F16) k_mx_dequantize<T_F16><<<g, 256, 0, s>>>(codes, scales, out, stride, total, groups, in_dim, vec);
    else k_mx_dequantize<T_BF16><<<g, 256, 0, s>>>(codes, scales, out, stride, total, groups, in_dim, vec);
    return hipGetLastError();
}

namespace {

// A kernel of the product and what it takes, by an estimate in us:
//   us = c0 + r c1 + (L c2 + r c3) slices
// with L workgroups a CU, r of them one after the other (`occ` run at once) and `slices`
// pieces of `unit` codes a wavefront, fitted to 150 sizes (1 to 2048 tokens, weights from
// memory; 64 x 64's constants by nine of them, later). At 200 other sizes the kernel it takes is
// slower than the fastest of the twelve by 5.5% on average up to 32 tokens (60 sizes; 49% at
// most: 4.9 in place of 3.3 us for 6 of 226 x 426), 3.6% from 33 to 300 (80; 66%: 26.2 in place of
// 15.8 us for 83 of 6656 x 6848), and 0.0% beyond (60; 0.8%). One or two float tokens, which the
// product quantises, are estimated alike: 2.4% on average at 38 sizes, 13.5% at most. From 129
// tokens on the tiles
// without LDS, which read the tokens' codes for every 16 or 32 channels, lose and are not
// looked at: 14.6 us at best in place of 10.5 for 129 tokens of 4096 x 4096, 58 in place of
// 19 for 200 of 14336 x 4096.
struct MxKernel {
    hipError_t (*go)(const MxArgs &, hipStream_t);
    hipError_t (*go_float)(const MxArgs &, uint32_t, hipStream_t);  // or null
    int bm, bn, wk, unit, occ, max_tok, threads;
    float c0, c1, c2, c3;
    bool fits(const MxArgs &a) const {  // a launch holds less than 2^32 threads
        const long long tiles = (long long)((a.out_dim + bm - 1) / bm) * ((a.n_tok + bn - 1) / bn);
        return a.n_tok <= max_tok && (tiles + 8) * threads < (1ll << 32);
    }
    float us(const MxArgs &a) const {
        const long long tiles = (long long)((a.out_dim + bm - 1) / bm) * ((a.n_tok + bn - 1) / bn);
        const long long L = (tiles + 255) / 256, r = (L + occ - 1) / occ;
        const int slices = ((a.in_dim + unit - 1) / unit + wk - 1) / wk;
        return c0 + (float)r * c1 + ((float)L * c2 + (float)r * c3) * (float)slices;
    }
};
template <int MF, int NF, int WK> constexpr MxKernel mx_few(int occ, float c0, float c1, float c2, float c3) {
    using G = MxFew<MF, NF, WK>;
    hipError_t (*go_float)(const MxArgs &, uint32_t, hipStream_t) = nullptr;
    if constexpr (NF == 1) go_float = &mx_few_float_go<G>;
    return {&mx_few_go<G>, go_float, G::BM, G::BN, WK, 512, occ, 128, 64 * WK, c0, c1, c2, c3};
}
template <int WM, int WN, int MF, int NF, int ST> constexpr MxKernel mx_big(int occ, float c0, float c1, float c2, float c3 = 0.0f) {
    using G = MxBig<WM, WN, MF, NF, ST>;
    return {&mx_big_go<G>, nullptr, G::BM, G::BN, 1, 256, occ, INT_MAX, G::kThreads, c0, c1, c2, c3};
}
const MxKernel kMxKernels[] = {
    mx_few<1, 1, 8>(2, 4.57f, 0.0f, 0.434f, 0.328f),  // 16 channels x 16 tokens
    mx_few<2, 1, 8>(1, 4.26f, 0.0f, 1.196f, 0.0f),    // 32 x 16
    mx_few<2, 1, 4>(3, 4.33f, 0.0f, 0.547f, 0.308f),
    mx_few<2, 2, 8>(1, 3.66f, 0.0f, 1.834f, 0.0f),    // 32 x 32
    mx_few<2, 2, 4>(2, 4.03f, 0.0f, 1.105f, 0.066f),
    mx_few<2, 4, 4>(1, 3.34f, 0.23f, 1.938f, 0.0f),   // 32 x 64
    mx_big<2, 2, 2, 2, 4>(2, 2.5f, 2.0f, 0.22f, 0.18f),  // 64 x 64 (eight wavefronts of 16 x 32: 10 to 25% slower)
    mx_big<2, 4, 2, 2, 4>(1, 0.39f, 4.36f, 0.499f),   // 64 x 128
    mx_big<2, 4, 4, 2, 3>(1, 0.0f, 5.10f, 0.768f),    // 128 x 128
    mx_big<4, 2, 3, 4, 2>(1, 0.54f, 4.50f, 1.153f),   // 192 x 128
    mx_big<2, 4, 8, 2, 2>(1, 2.66f, 4.56f, 1.351f),   // 256 x 128
    {&mx_wide_224, nullptr, 224, 256, 1, 256, 1, INT_MAX, 256, 0.0f, 10.26f, 1.216f, 0.0f},
};

const MxKernel *mx_choose(const MxArgs &a) {
    const MxKernel *best = nullptr;
    float us = 0.0f;
    for (const MxKernel &k : kMxKernels) {
        if (!k.fits(a)) continue;
        const float t = k.us(a);
        if (!best || t < us) {
            best = &k;
            us = t;
        }
    }
    return best;
}

}  // namespace

hipError_t launch_mx_matmul(const MxArgs &a, hipStream_t s) {
    if (a.n_tok <= 0) return hipSuccess;
    const MxKernel *const k = mx_choose(a);
    return k ? k->go(a, s) : hipErrorInvalidValue;
}

hipError_t launch_mx_matmul_float(MxArgs a, const void *x, size_t x_stride, uint32_t dtype_x, uint8_t *codes,
                                  uint8_t *scales, hipStream_t s) {
    if (a.n_tok <= 0) return hipSuccess;
    const MxKernel *const k = mx_choose(a);
    if (!k) return hipErrorInvalidValue;
    if (k->go_float && a.n_tok <= kMxFloatTok) {
        a.xf = x;
        a.x_stride = x_stride;
        a.x_vec = mx_rows_vec(x, x_stride, dtype_x);
        return k->go_float(a, dtype_x, s);
    }
    a.x = codes;
    a.xs = scales;
    const hipError_t e = launch_mx_quantize(x, x_stride, codes, scales, a.n_tok, a.in_dim, dtype_x, s);
    return e == hipSuccess ? k->go(a, s) : e;
}

}  // namespace rsllm_hip
