// MXFP4 rows: quantising, decoding, and the product of two code matrices.
#include "fp4_common.h"

#include <algorithm>

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

}  // namespace

// A lane's eight elements at a time, four lanes a block: `groups` of eight a row (its
// padding included).
template <uint32_t DT>
__global__ __launch_bounds__(256) void k_mx_quantize(const void *__restrict__ x, size_t stride,
                                                     uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                     size_t total, int groups, int in_dim, int vec) {
    const size_t rb = (size_t)groups * 4, sb = mx_scale_bytes(in_dim);
    for (size_t n = (size_t)blockIdx.x * 256 + threadIdx.x; n < total; n += (size_t)gridDim.x * 256) {
        const size_t row = n / (size_t)groups;
        const int g = (int)(n - row * (size_t)groups), i = 8 * g;
        float v[8];
        mx_load8<DT>(x, row * stride, i, in_dim, vec, v);
        uint32_t big = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) big = max(big, mx_abs_bits(v[k]));
        const uint32_t s = mx_scale_of(mx_max4(big));
        uint32_t c = 0;
        if (s != 255u) {
            const float unit = mx_unit(s);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], unit, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], unit, 1);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], unit, 2);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], unit, 3);
        }
        *reinterpret_cast<uint32_t *>(codes + row * rb + 4 * g) = c;
        uint8_t *const sr = scales + row * sb;
        if ((g & 3) == 0) sr[g >> 2] = (uint8_t)s;
        if (g == groups - 1)
            for (size_t b = (size_t)groups / 4; b < sb; b++) sr[b] = 0;
    }
}

__global__ __launch_bounds__(256) void k_mx_dequantize(const uint8_t *__restrict__ codes,
                                                       const uint8_t *__restrict__ scales, void *__restrict__ out,
                                                       size_t stride, size_t total, int groups, int in_dim,
                                                       uint32_t dtype) {
    const size_t rb = mx_row_bytes(in_dim), sb = mx_scale_bytes(in_dim);
    for (size_t n = (size_t)blockIdx.x * 256 + threadIdx.x; n < total; n += (size_t)gridDim.x * 256) {
        const size_t row = n / (size_t)groups;
        const int g = (int)(n - row * (size_t)groups);
        const uint32_t c = *reinterpret_cast<const uint32_t *>(codes + row * rb + 4 * g);
        const uint32_t s = scales[row * sb + (g >> 2)];
        constexpr float kValue[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
        for (int k = 0; k < 8 && 8 * g + k < in_dim; k++) {
            const uint32_t q = c >> (4 * k);
            const float m = (q & 8u) ? -kValue[q & 7u] : kValue[q & 7u];
            mx_store(out, row * stride + 8 * g + k, s == 255u ? __builtin_nanf("") : ldexpf(m, (int)s - 127), dtype);
        }
    }
}

// ---- the product -------------------------------------------------------------------
//
// v_mfma_scale_f32_16x16x128: lane l holds 32 codes (16 bytes) and a scale byte of row
// l % 16 of either operand, block l / 16 of the step's four; its four sums are rows
// 4 (l / 16) + i of the first operand (channels) at row l % 16 of the second (tokens).
// A wavefront per 16 x 16 outputs.
__global__ __launch_bounds__(64) void k_mx_simple(MxArgs a) {
    const int lane = threadIdx.x, r = lane & 15, q = lane >> 4;
    const int o0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
    const size_t rb = mx_row_bytes(a.in_dim), sb = mx_scale_bytes(a.in_dim);
    const int blocks = (a.in_dim + 31) / 32;
    const size_t wr = (size_t)min(o0 + r, a.out_dim - 1), xr = (size_t)min(t0 + r, a.n_tok - 1);
    mx_v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int st = 0; st < (int)(rb / 64); st++) {
        const int b = 4 * st + q;
        const uint4 cw = *reinterpret_cast<const uint4 *>(a.w + wr * rb + 16 * (size_t)b);
        const uint4 cx = *reinterpret_cast<const uint4 *>(a.x + xr * rb + 16 * (size_t)b);
        // (a weight row's scales behind its last block may be anything)
        const int sw = b < blocks ? a.ws[wr * sb + b] : 127, sx = b < blocks ? a.xs[xr * sb + b] : 127;
        const mx_v8i fw = {(int)cw.x, (int)cw.y, (int)cw.z, (int)cw.w, 0, 0, 0, 0};
        const mx_v8i fx = {(int)cx.x, (int)cx.y, (int)cx.z, (int)cx.w, 0, 0, 0, 0};
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw, fx, acc, 4, 4, 0, sw, 0, sx);
    }
    if (t0 + r >= a.n_tok) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int o = o0 + 4 * q + i;
        if (o < a.out_dim)
            mx_store(a.out, (size_t)(t0 + r) * a.out_stride + o, a.bias ? acc[i] + a.bias[o] : acc[i], a.dtype_out);
    }
}

namespace {

// Workgroups of 256 for `total` threads' work, in turns behind 2^20 of them.
unsigned mx_grid(size_t total) { return (unsigned)std::min<size_t>((total + 255) / 256, (size_t)1 << 20); }

}  // namespace

hipError_t launch_mx_quantize(const void *x, size_t stride, uint8_t *codes, uint8_t *scales, int n_rows,
                              int in_dim, uint32_t dtype, hipStream_t s) {
    if (n_rows <= 0) return hipSuccess;
    const int groups = (int)mx_row_bytes(in_dim) / 4;
    const size_t total = (size_t)n_rows * groups;
    const int vec = (uintptr_t)x % 16 == 0 && stride * (dtype == T_F32 ? 4 : 2) % 16 == 0;
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
    k_mx_dequantize<<<mx_grid(total), 256, 0, s>>>(codes, scales, out, stride, total, groups, in_dim, dtype);
    return hipGetLastError();
}

hipError_t launch_mx_matmul(const MxArgs &a, hipStream_t s) {
    if (a.n_tok <= 0) return hipSuccess;
    // (the second grid dimension holds 65535: more tokens go in turns)
    for (int t = 0; t < a.n_tok; t += 65535 * 16) {
        MxArgs part = a;
        part.n_tok = std::min(a.n_tok - t, 65535 * 16);
        part.x += (size_t)t * mx_row_bytes(a.in_dim);
        part.xs += (size_t)t * mx_scale_bytes(a.in_dim);
        part.out = static_cast<uint8_t *>(a.out) + (size_t)t * a.out_stride * (a.dtype_out == T_F32 ? 4 : 2);
        k_mx_simple<<<dim3((a.out_dim + 15) / 16, (part.n_tok + 15) / 16), 64, 0, s>>>(part);
    }
    return hipGetLastError();
}

}  // namespace rsllm_hip
