// The product of 4-bit codes for many tokens: the widest tiles.
#include "mxfp4_product.h"

#include <type_traits>
#include <utility>

namespace rsllm_hip {

namespace {

// A workgroup's tile: BM = 32 MF channels x BN = 32 NF tokens, four wavefronts, 16 MF x
// 16 NF each, one a SIMD: so wide that an operand read from LDS feeds NF or MF matrix
// instructions and the reads stay below LDS' rate. Slices of 256 codes (128 bytes a row,
// whole lines: half ones halve what L2 delivers) of both operands are copied to LDS two
// deep, multiplied in two steps of 128 codes; while a step is multiplied, the next one's
// operands are read into registers. One barrier a slice, before its second step: behind it
// the next slice has landed, and everyone holds what is left of this one in registers, so
// the slice after the next is copied over it.
// With one wavefront a SIMD the matrix cores wait for whatever is not issued in their
// shadow, so every product (16 cycles) is followed by its share of everything else, at
// most some three instructions. Wavefronts 0 and 1 copy channels, 2 and 3 tokens, each
// from one buffer; the scales, 16 bytes a row for two slices, come as two more copies a
// slice of wavefronts 0 (the channels') and 1.
// 2048 tokens, 14336 x 4096, bf16 out: 75 us, 3.2 PFLOP/s, in two rounds of 256 workgroups. Of
// a tile's some 32 us 3 pass before the first product, 23 in the loop (70% of the matrix
// cores' rate at the 1.7 GHz that they get under this load) and 5 with the stores, in which
// nothing multiplies. k_mx_big's widest tiles (128 x 128, 256 x 128) take 128 us here.
template <int MF_, int NF_> struct MxWide {
    static constexpr int MF = MF_, NF = NF_, BM = 32 * MF, BN = 32 * NF;
    static constexpr int D = 2 * MF;  // a wavefront's copies of 8 rows x 128 bytes a slice
    static constexpr int X = 2;       // and of scales, or what tokens are left
    static constexpr int kSlice = (BM + BN) * 128, kRing = 2 * kSlice;
    static constexpr int kScales = 4096, kPair = 2 * kScales;  // 256 rows' scales of two slices
    static constexpr int kLds = kRing + 2 * kPair;
    static constexpr int P = MF % 4 == 0 ? 4 : MF % 2 == 0 ? 2 : 1;
    static_assert(kLds <= 160 * 1024 && BM <= 256 && BN <= 256 && (2 * NF == D || 2 * NF == D + X) && 3 * (D + X) <= MF * NF, "tile");
};

// Byte 16 c of a row's 128 lies at place c ^ key: the 16 rows of an operand read are
// spread over all banks.
template <int P> __device__ __forceinline__ constexpr int mx_key8(int row) {
    return ((row >> 1) & 1) | ((row / (4 * P)) & 3) << 1;
}

// acc += w x in place, with byte U of the scales, the accumulators in the accumulation
// registers, the operands in the others: left to itself the compiler mixes the two and
// spills. What it does not know of is the wait between the last of these and the first
// other use of a sum.
template <int U> __device__ __forceinline__ void mx_mfma_acc(mx_v4f &acc, const mx_v4u &w, const mx_v4u &x, uint32_t sw, uint32_t sx) {
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4 blgp:4"
                 : "+a"(acc)
                 : "v"(w), "v"(x), "v"(sw), "v"(sx), "n"(U & 1), "n"(U >> 1));
}

// A copy in two parts with a product between them (which stands in for the wait state
// that M0 needs): where in LDS, then 16 bytes a lane from voff of the buffer there.
// M0 is not restored: nothing else in this file uses it (LDS needs none, and the compiler
// sets it before each use of its own; it takes no declaration of it as overwritten). Between
// the two parts nothing may be added that needs it.
__device__ __forceinline__ void mx_dma_to(uint32_t lds, int at) {
    asm volatile("s_add_u32 m0, %0, %1" ::"s"(__builtin_amdgcn_readfirstlane((int)lds)), "s"(at) : "memory", "scc");
}
__device__ __forceinline__ void mx_dma(const bl_rsrc &r, uint32_t voff) {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r) : "memory");
}
// The buffer `by` bytes further on, with its end where it was; nothing of it if not `any`.
// (Not the load's scalar offset: which offsets the check against the end counts would have
// to be known.)
__device__ __forceinline__ bl_rsrc mx_ahead(const bl_rsrc &r, uint32_t by, bool any) {
    const uint64_t p = ((uint64_t)r[1] << 32 | r[0]) + by;
    return bl_rsrc{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p),
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32)),
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)(any ? r[2] - by : 0u)), r[3]};
}

template <class F, int... K> __device__ __forceinline__ void mx_each_(F &&f, std::integer_sequence<int, K...>) {
    (f(std::integral_constant<int, K>{}), ...);
}
// f(0), .., f(N - 1) with constants
template <int N, class F> __device__ __forceinline__ void mx_each(F &&f) {
    mx_each_(f, std::make_integer_sequence<int, N>{});
}

template <class G> __global__ __launch_bounds__(256, 1) void k_mx_wide(MxArgs a, int n_ct, int n_tt) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int MF = G::MF, NF = G::NF, D = G::D, X = G::X, P = G::P, NO = MF + NF, NM = MF * NF;
    // Workgroups go round the 8 XCDs: each takes a run of tiles, token tiles fastest, so
    // the tiles that share a weight row are behind one L2.
    const int total = n_ct * n_tt, per = (total + 7) / 8;
    const int L = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || L >= total) return;  // the whole workgroup
    const int tt = L % n_tt, ct = L / n_tt;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wn = wv & 1, wm = wv >> 1;
    const int o0 = ct * G::BM, t0 = tt * G::BN;
    const uint32_t rb = (uint32_t)mx_row_bytes(a.in_dim), sb = (uint32_t)mx_scale_bytes(a.in_dim);
    const int blocks = (a.in_dim + 31) / 32, n_sl = (int)((rb + 127) / 128);

    // This wavefront's copies: D (and, of tokens, up to X) times 8 rows; rows behind the last
    // repeat it (their products are not stored).
    const bool is_w = wv < 2;
    const int rows = is_w ? min(G::BM, a.out_dim - o0) : min(G::BN, a.n_tok - t0);
    const int mine = is_w ? 2 * MF : 2 * NF, first = (wv & 1) * mine;
    const size_t r0 = (size_t)(is_w ? o0 : t0);
    const bl_rsrc rc = bl_make_rsrc((is_w ? a.w : a.x) + r0 * rb, (uint32_t)rows * rb);
    const uint32_t lds0 = bl_lds(smem), lds_c = lds0 + (uint32_t)((is_w ? 0 : G::BM * 128) + first * 1024);
    auto offset = [&](int c) {
        const int row = 8 * (first + c) + (lane >> 3);
        const int at = (lane & 7) ^ (is_w ? mx_key8<P>(row) : mx_key8<1>(row));
        return (uint32_t)min(row, rows - 1) * rb + 16u * (uint32_t)at;
    };
    uint32_t off[D], offx[2][X];  // offx: by the parity of the slice
#pragma unroll
    for (int p = 0; p < D; p++) off[p] = offset(p);
    // the scales' rows: wavefront 0 the channels', 1 the tokens'; two copies of 64 rows with
    // every slice (odd s: the first two of the next pair of slices, even s: the last two)
    const int s_rows = wv == 0 ? min(G::BM, a.out_dim - o0) : min(G::BN, a.n_tok - t0);
    const bl_rsrc rs = bl_make_rsrc(wv == 0 ? a.ws + (size_t)o0 * sb : a.xs + (size_t)t0 * sb, (uint32_t)s_rows * sb);
#pragma unroll
    for (int odd = 0; odd < 2; odd++)
#pragma unroll
        for (int x = 0; x < X; x++)
            offx[odd][x] = is_w ? (uint32_t)min(64 * (odd ? x : x + 2) + lane, s_rows - 1) * sb : offset(min(D + x, mine - 1));
    const uint32_t lds_s = lds0 + (uint32_t)(G::kRing + (wv & 1) * G::kScales);
    // what the copies of slice s need beside their offsets
    struct Set {
        bl_rsrc r, rx;
        uint32_t ldsx;
    };
    auto make_set = [&](int s, int odd) __attribute__((always_inline)) {
        const int g = (s + 1) >> 1;  // the pair of slices whose scales come
        Set t;
        t.r = mx_ahead(rc, 128u * (uint32_t)s, s < n_sl);
        t.rx = is_w ? mx_ahead(rs, 16u * (uint32_t)g, 2 * g < n_sl) : t.r;
        t.ldsx = is_w ? lds_s + (uint32_t)((g & 1) * G::kPair + (odd ? 0 : 2048)) : lds_c + (uint32_t)(odd * G::kSlice + D * 1024);
        return t;
    };
    // copy c of D + X of a slice: where to, and from where. (Half a slice at the row's end:
    // what is copied behind it is the next row's start or zeros, and is not used.)
    auto copy_to = [&](auto c_c, const Set &t, int odd) __attribute__((always_inline)) {
        constexpr int c = decltype(c_c)::value;
        if constexpr (c < D) mx_dma_to(lds_c, odd * G::kSlice + c * 1024);
        else if constexpr (2 * NF == D) mx_dma_to(t.ldsx, is_w ? (c - D) * 1024 : -1024);  // (tokens: the last again)
        else mx_dma_to(t.ldsx, (c - D) * 1024);
    };
    auto copy_from = [&](auto c_c, const Set &t, int odd) __attribute__((always_inline)) {
        constexpr int c = decltype(c_c)::value;
        if constexpr (c < D) mx_dma(t.r, off[c]);
        else mx_dma(t.rx, offx[odd][c - D]);
    };
    mx_v4f acc[MF][NF];
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) {
            acc[m][n] = mx_v4f{0.0f, 0.0f, 0.0f, 0.0f};
            asm volatile("" : "+a"(acc[m][n]));  // (written here, long before the first product)
        }
    const int r16 = lane & 15, q = lane >> 4;
    const int wrow = wm * 16 * MF + mx_frag_row<P>(0, r16), xrow = wn * 16 * NF + r16;
    // Where this lane's operands lie in slice buffer 0 and 1, first half; the second is 64
    // bytes off by xor. (The key of every fragment's row r16 is that of fragment 0's.)
    uint32_t at_w = (uint32_t)(wrow * 128 + 16 * (q ^ mx_key8<P>(wrow)));
    uint32_t at_x = (uint32_t)((G::BM + xrow) * 128 + 16 * (q ^ mx_key8<1>(xrow)));
    const uint8_t *pw[2][2], *px[2][2];  // [buffer][half]
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t ow = (at_w ^ (64u * h)) + b * G::kSlice, ox = (at_x ^ (64u * h)) + b * G::kSlice;
            asm volatile("" : "+v"(ow), "+v"(ox));  // (registers of their own: an LDS read's immediate reaches 64 KB)
            pw[b][h] = smem + ow;
            px[b][h] = smem + ox;
        }
    const uint8_t *const sw0 = smem + G::kRing + wrow * 16, *const sx0 = smem + G::kRing + G::kScales + xrow * 16;
    mx_v4u f[2][NO];  // a step's operands: NF of tokens, MF of channels
    uint32_t sc[NO], sn[NO];  // scales of four steps (two slices), a byte each; the next ones
    mx_v4u raw[NO];
    auto read1 = [&](int b, int h, int j) __attribute__((always_inline)) {
        if (j < NF) f[h][j] = *reinterpret_cast<const mx_v4u *>(px[b][h] + j * 2048);
        else f[h][j] = *reinterpret_cast<const mx_v4u *>(pw[b][h] + mx_frag_row<P>(j - NF, 0) * 128);
    };
    // operand j's scales of pair g of slices: byte q of four dwords
    const uint32_t pick = (uint32_t)q | (uint32_t)(q + 4) << 8;
    auto scales1 = [&](int g, int j) __attribute__((always_inline)) {
        const uint8_t *const p = j < NF ? sx0 + j * 256 : sw0 + mx_frag_row<P>(j < NF ? 0 : j - NF, 0) * 16;
        raw[j] = *reinterpret_cast<const mx_v4u *>(p + (g & 1) * G::kPair);
    };
    auto scales2 = [&](int j) __attribute__((always_inline)) {
        // (v_perm_b32 counts the bytes of its second operand first)
        const mx_v4u v = raw[j];
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], pick), __builtin_amdgcn_perm(v[1], v[0], pick), 0x05040100u);
    };
    // Step (half H of a slice, its parity ODD) over the operands in f[H] with byte 2 ODD + H
    // of the scales; behind product k its share of: the reads of the next step's operands
    // (buffer rb_), with H = 1 the copies of slice s + 2, and with that and ODD the reads of
    // the next pair's scales.
    auto step = [&](auto odd_c, auto h_c, int s) __attribute__((always_inline)) {
        constexpr int odd = decltype(odd_c)::value, H = decltype(h_c)::value;
        constexpr int C = D + X;
        Set t;
        if constexpr (H == 1) t = make_set(s + 2, odd);
        mx_each<NM>([&](auto k_c) __attribute__((always_inline)) {
            constexpr int k = decltype(k_c)::value;
            mx_mfma_acc<2 * odd + H>(acc[k / NF][k % NF], f[H][NF + k / NF], f[H][k % NF], sc[NF + k / NF], sc[k % NF]);
            if constexpr (k % 2 == 0 && k / 2 < NO) read1(H ? odd ^ 1 : odd, H ^ 1, k / 2);
            if constexpr (H == 1) {
                // copy c's two parts behind products 3 c + 1 and 3 c + 2
                if constexpr (k % 3 == 1 && k / 3 < C) copy_to(std::integral_constant<int, k / 3>{}, t, odd);
                if constexpr (k % 3 == 2 && k / 3 < C) copy_from(std::integral_constant<int, k / 3>{}, t, odd);
                if constexpr (odd == 1) {
                    constexpr int k0 = 2 * NO < NM - NO - 6 ? 2 * NO : NM - NO - 6;
                    if constexpr (k >= k0 && k < k0 + NO) scales1((s + 1) >> 1, k - k0);
                    if constexpr (k >= k0 + 5 && k < k0 + 5 + NO) sn[k - k0 - 5] = scales2(k - k0 - 5);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // the next pair's scales take the place of this one's; those behind a row's last block
    // may be anything: there 1
    auto settle = [&](int s) __attribute__((always_inline)) {
        uint32_t keep = 0xFFFFFFFFu;
        if (8 * s + 16 > blocks) {
            keep = 0;
#pragma unroll
            for (int u = 0; u < 4; u++) keep |= 8 * s + 4 * u + q < blocks ? 0xFFu << (8 * u) : 0u;
        }
#pragma unroll
        for (int j = 0; j < NO; j++) {
            sc[j] = (sn[j] & keep) | (0x7F7F7F7Fu & ~keep);
            asm volatile("" : "+v"(sc[j]));
        }
        // (written some cycles before a product, which the compiler does not see, reads them)
        asm volatile("s_nop 3" ::: "memory");
    };
    auto set = [&](int s, int odd) __attribute__((always_inline)) {
        const Set t = make_set(s, odd);
        mx_each<D + X>([&](auto c_c) __attribute__((always_inline)) {
            copy_to(c_c, t, odd);
            asm volatile("s_nop 0" ::: "memory");
            copy_from(c_c, t, odd);
        });
    };
    if (is_w) {  // the first pair's first scales
#pragma unroll
        for (int x = 0; x < X; x++) {
            mx_dma_to(lds_s, x * 1024);
            asm volatile("s_nop 0" ::: "memory");
            mx_dma(rs, offx[1][x]);
        }
    }
    set(0, 0);
    set(1, 1);
    bl_barrier<D + X>();
#pragma unroll
    for (int j = 0; j < NO; j++) {
        read1(0, 0, j);
        scales1(0, j);
    }
#pragma unroll
    for (int j = 0; j < NO; j++) sn[j] = scales2(j);
    const int steps = (int)(rb / 64);
    for (int s = 0; s < n_sl; s += 2) {
        settle(s);
        step(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{}, s);
        bl_barrier<0>();
        if (2 * s + 1 >= steps) break;
        step(std::integral_constant<int, 0>{}, std::integral_constant<int, 1>{}, s);
        if (s + 1 >= n_sl) break;
        step(std::integral_constant<int, 1>{}, std::integral_constant<int, 0>{}, s + 1);
        bl_barrier<0>();
        if (2 * s + 3 >= steps) break;
        step(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}, s + 1);
    }
    bl_wait<0>();  // (the copies past the last slice, zeros, land in the ring too)
    // every sum written before it is read: 16 passes of 4 cycles at most
    asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int m = 0; m < MF; m++)
#pragma unroll
        for (int n = 0; n < NF; n++) asm volatile("" : "+a"(acc[m][n]));
    mx_write_tile<MF, NF, 2, 2, P, G::kLds>(a, acc, smem, o0, t0, wm, wn);
}

template <class G> hipError_t mx_wide_go(const MxArgs &a, hipStream_t s) {
    const hipError_t e = mx_allow_lds<G>(reinterpret_cast<const void *>(&k_mx_wide<G>));
    if (e != hipSuccess) return e;
    const int n_ct = (a.out_dim + G::BM - 1) / G::BM, n_tt = (a.n_tok + G::BN - 1) / G::BN;
    const long long wgs = ((long long)n_ct * n_tt + 7) / 8 * 8;
    k_mx_wide<G><<<(unsigned)wgs, 256, G::kLds, s>>>(a, n_ct, n_tt);
    return hipGetLastError();
}

}  // namespace

hipError_t mx_wide_224(const MxArgs &a, hipStream_t s) { return mx_wide_go<MxWide<7, 8>>(a, s); }

}  // namespace rsllm_hip
