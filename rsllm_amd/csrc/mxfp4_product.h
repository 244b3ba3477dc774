// What the product kernels of 4-bit codes share.
//
// v_mfma_scale_f32_16x16x128: lane l holds 32 codes (16 bytes) and a scale byte of row
// l % 16 of either operand, block l / 16 of the step's four; its four sums are rows
// 4 (l / 16) + i of the first operand (channels) at row l % 16 of the second (tokens).
#pragma once

#include <atomic>
#include <type_traits>

#include "buffer_lds.h"
#include "fp4_common.h"

namespace rsllm_hip {

typedef uint32_t mx_v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ mx_v4f mx_mfma(const mx_v4u &w, const mx_v4u &x, const mx_v4f &acc, int sw, int sx) {
    const mx_v8i a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const mx_v8i b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, sw, 0, sx);
}

// The biases of four channels, 0 where there are none.
__device__ __forceinline__ float4 mx_bias(const MxArgs &a, int o) {
    float b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = a.bias && o + i < a.out_dim ? a.bias[o + i] : 0.0f;
    return make_float4(b[0], b[1], b[2], b[3]);
}
// Whether four channels of an output row, from a multiple of 4 on, can be stored at once.
__device__ __forceinline__ bool mx_vec(const MxArgs &a) {
    return (uintptr_t)a.out % (a.dtype_out == T_F32 ? 16 : 8) == 0 && a.out_stride % 4 == 0;
}

// Row r of fragment m of a wavefront's channels: P fragments' rows interleaved, so that a
// lane ends up with 4 P consecutive channels.
template <int P> __device__ __forceinline__ constexpr int mx_frag_row(int m, int r) {
    return 16 * P * (m / P) + 4 * P * (r >> 2) + 4 * (m % P) + (r & 3);
}

// Four sums as `dtype`, packed.
template <uint32_t DT> struct MxPack {
    typedef uint2 type;
};
template <> struct MxPack<T_F32> {
    typedef float4 type;
};
template <uint32_t DT> __device__ __forceinline__ typename MxPack<DT>::type mx_pack(const mx_v4f &v, const float4 &b) {
    const float y[4] = {v[0] + b.x, v[1] + b.y, v[2] + b.z, v[3] + b.w};
    if constexpr (DT == T_F32) {
        return make_float4(y[0], y[1], y[2], y[3]);
    } else if constexpr (DT == T_F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return make_uint2(__builtin_bit_cast(uint32_t, h2{(_Float16)y[0], (_Float16)y[1]}),
                          __builtin_bit_cast(uint32_t, h2{(_Float16)y[2], (_Float16)y[3]}));
    } else {
        return make_uint2(__builtin_bit_cast(uint32_t, mx_bf2{(__bf16)y[0], (__bf16)y[1]}),
                          __builtin_bit_cast(uint32_t, mx_bf2{(__bf16)y[2], (__bf16)y[3]}));
    }
}

// Four consecutive channels from o on of token t, bias b. vec: bias and out aligned for them.
__device__ __forceinline__ void mx_finish(const MxArgs &a, const mx_v4f &acc, const float4 &b, int o, int t, bool vec) {
    if (t >= a.n_tok || o >= a.out_dim) return;
    const size_t at = (size_t)t * a.out_stride + o;
    if (vec && o + 4 <= a.out_dim) {
        uint8_t *const p = static_cast<uint8_t *>(a.out) + at * (a.dtype_out == T_F32 ? 4 : 2);
        if (a.dtype_out == T_F32) *reinterpret_cast<float4 *>(p) = mx_pack<T_F32>(acc, b);
        else *reinterpret_cast<uint2 *>(p) = a.dtype_out == T_F16 ? mx_pack<T_F16>(acc, b) : mx_pack<T_BF16>(acc, b);
        return;
    }
    const float y[4] = {acc[0] + b.x, acc[1] + b.y, acc[2] + b.z, acc[3] + b.w};
    for (int i = 0; i < 4; i++)
        if (o + i < a.out_dim) mx_store(a.out, at + i, y[i], a.dtype_out);
}

// A workgroup's sums to out: BM channels from o0 on, WN 16 NF tokens from t0 on; wavefront
// (wm, wn) of NW holds MF x NF fragments. They go through LDS (`kLds` bytes at smem, free
// for it), some token fragments at a time, so that whole lines are written. The loops are
// kept short: every workgroup has to fetch this code (with the edges' cases in them, 224 x
// 256 sums of four wavefronts took 9 us).
template <int MF, int NF, int WM, int WN, int P, int kLds>
__device__ __forceinline__ void mx_write_tile(const MxArgs &a, const mx_v4f (&acc)[MF][NF], uint8_t *smem, int o0,
                                              int t0, int wm, int wn) {
    constexpr int BM = 16 * MF * WM, NW = WM * WN, kPitch = BM + 4;  // (4 floats: no bank conflicts)
    constexpr auto fits = [](int d) { return NF % d == 0 && WN * 16 * d * kPitch * 4 <= kLds; };
    constexpr int PF = fits(NF) ? NF : NF % 2 == 0 && fits(NF / 2) ? NF / 2 : 1;  // fragments a pass
    static_assert(fits(PF), "tile");
    constexpr int kLanes = BM / 4, kTok = 64 / kLanes;  // lanes a token, tokens a wavefront's turn
    constexpr int kTurns = 16 * PF / (NW * kTok), U = kTurns % 8 == 0 ? 8 : kTurns % 4 == 0 ? 4 : kTurns % 2 == 0 ? 2 : 1;
    static_assert(kTurns * NW * kTok == 16 * PF, "tile");  // (a wavefront column's tokens)
    float *const tile = reinterpret_cast<float *>(smem);
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, wv = wm * WN + wn;
    const int sub = lane / kLanes, c0 = lane % kLanes;
    const bool four = mx_vec(a), mine = kTok * kLanes == 64 || sub < kTok;
    // a lane's four channels at once; WHOLE: no token behind the last
    auto rows = [&](auto dt_c, auto whole_c, int n0) __attribute__((always_inline)) {
        typedef typename MxPack<decltype(dt_c)::value>::type pack;
        const int o = o0 + 4 * c0;
        if (!mine || o + 4 > a.out_dim) return;
        const float4 b = mx_bias(a, o);
        const size_t step = (size_t)(NW * kTok) * a.out_stride;
#pragma unroll 1
        for (int g = 0; g < WN; g++) {  // the wavefronts' tokens, one after the other
            int t = t0 + g * 16 * NF + 16 * n0 + wv * kTok + sub;
            const float *src = tile + (g * 16 * PF + wv * kTok + sub) * kPitch + 4 * c0;
            pack *dst = reinterpret_cast<pack *>(static_cast<uint8_t *>(a.out) + ((size_t)t * a.out_stride + o) * (sizeof(pack) / 4));
#pragma unroll 1
            for (int i = 0; i < kTurns; i += U, src += U * NW * kTok * kPitch) {
                mx_v4f v[U];
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = *reinterpret_cast<const mx_v4f *>(src + u * NW * kTok * kPitch);
#pragma unroll
                for (int u = 0; u < U; u++, t += NW * kTok) {
                    if (decltype(whole_c)::value || t < a.n_tok) *dst = mx_pack<decltype(dt_c)::value>(v[u], b);
                    dst = reinterpret_cast<pack *>(reinterpret_cast<uint8_t *>(dst) + step * (sizeof(pack) / 4));
                }
            }
        }
    };
    // channels one by one, from c on kLanes apart
    auto ones = [&](int n0, int c) __attribute__((always_inline)) {
        if (!mine) return;
#pragma unroll 1
        for (; c < BM && o0 + c < a.out_dim; c += kLanes) {
            const float b = a.bias ? a.bias[o0 + c] : 0.0f;
#pragma unroll 1
            for (int i = 0; i < WN * kTurns; i += U) {
                const int g = i / kTurns, k = wv * kTok + sub + i % kTurns * NW * kTok;
                float v[U];
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = tile[(g * 16 * PF + k + u * NW * kTok) * kPitch + c];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int t = t0 + g * 16 * NF + 16 * n0 + k + u * NW * kTok;
                    if (t < a.n_tok) mx_store(a.out, (size_t)t * a.out_stride + o0 + c, v[u] + b, a.dtype_out);
                }
            }
        }
    };
#pragma unroll 1
    for (int n0 = 0; n0 < NF; n0 += PF) {
        __syncthreads();
#pragma unroll
        for (int p = 0; p < NF; p += PF) {
            if (p == n0) {
#pragma unroll
                for (int n = 0; n < PF; n++)
#pragma unroll
                    for (int m = 0; m < MF; m++)
                        *reinterpret_cast<mx_v4f *>(tile + ((wn * PF + n) * 16 + r) * kPitch + wm * 16 * MF +
                                                    mx_frag_row<P>(m, 4 * q)) = acc[m][p + n];
            }
        }
        __syncthreads();
        if (!four) {
            ones(n0, c0);
            continue;
        }
        auto typed = [&](auto whole_c) __attribute__((always_inline)) {
            if (a.dtype_out == T_F32) rows(std::integral_constant<uint32_t, T_F32>{}, whole_c, n0);
            else if (a.dtype_out == T_F16) rows(std::integral_constant<uint32_t, T_F16>{}, whole_c, n0);
            else rows(std::integral_constant<uint32_t, T_BF16>{}, whole_c, n0);
        };
        if (t0 + 16 * NF * WN <= a.n_tok) typed(std::true_type{});
        else typed(std::false_type{});
        // what is left of the last channels
        const int left = a.out_dim - o0;
        if (left < BM && left % 4 != 0 && c0 < left % 4) ones(n0, left - left % 4 + c0);
    }
}

// More LDS than a kernel gets unasked, asked for until the runtime has granted it once
// on the current device: a refusal is that call's error alone.
template <class G> hipError_t mx_allow_lds(const void *kernel) {
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

// mxfp4_wide.hip: tiles of 224 channels x 256 tokens
hipError_t mx_wide_224(const MxArgs &a, hipStream_t s);

}  // namespace rsllm_hip
