// The int8 product with a scale per token and per channel, and its quantiser.
#include "kernels.h"

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
    float d, up, d_up, inv;
};
__device__ __forceinline__ I8Scale i8_scale(float amax) {
    I8Scale s;
    s.d = amax / 127.0f;
    s.up = s.d < 0x1p-100f ? 0x1p64f : 1.0f;
    s.d_up = s.d * s.up;
    s.inv = s.d > 0.0f ? 1.0f / s.d_up : 0.0f;
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

}  // namespace

__global__ __launch_bounds__(256) void k_i8_quantize(const void *__restrict__ x, size_t stride,
                                                     int8_t *__restrict__ xq,
                                                     float *__restrict__ scale, int in_dim,
                                                     int row_bytes, uint32_t dtype) {
    __shared__ float red[4];
    __shared__ int red_bad[4];
    const int t = blockIdx.x, tid = threadIdx.x;
    const size_t row = (size_t)t * stride;
    float amax = 0.0f;
    int bad = 0;
    for (int i = tid; i < in_dim; i += 256) {
        const float v = i8_load(x, row + i, dtype);
        amax = fmaxf(amax, fabsf(v));
        bad |= !__builtin_isfinite(v);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        amax = fmaxf(amax, __shfl_xor(amax, off, 64));
        bad |= __shfl_xor(bad, off, 64);
    }
    if ((tid & 63) == 0) {
        red[tid >> 6] = amax;
        red_bad[tid >> 6] = bad;
    }
    __syncthreads();
    amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    bad = red_bad[0] | red_bad[1] | red_bad[2] | red_bad[3];
    const I8Scale s = i8_scale(bad ? 0.0f : amax);
    for (int i = tid; i < row_bytes; i += 256) {
        const int q = i < in_dim && !bad ? i8_code(i8_load(x, row + i, dtype), s) : 0;
        xq[(size_t)t * row_bytes + i] = (int8_t)q;
    }
    if (tid == 0) scale[t] = bad ? __builtin_nanf("") : s.d;
}

// One thread per output.
__global__ __launch_bounds__(256) void k_i8_simple(I8Args a) {
    const int o = blockIdx.x * 64 + (threadIdx.x & 63), t = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (o >= a.out_dim || t >= a.n_tok) return;
    const uint4 *w = reinterpret_cast<const uint4 *>(a.w + (size_t)o * a.row_bytes);
    const uint4 *x = reinterpret_cast<const uint4 *>(a.xq + (size_t)t * a.row_bytes);
    int acc = 0;
    for (int i = 0; i < a.row_bytes / 16; i++) {
        const uint4 p = w[i], q = x[i];
        acc = __builtin_amdgcn_sdot4((int)p.x, (int)q.x, acc, false);
        acc = __builtin_amdgcn_sdot4((int)p.y, (int)q.y, acc, false);
        acc = __builtin_amdgcn_sdot4((int)p.z, (int)q.z, acc, false);
        acc = __builtin_amdgcn_sdot4((int)p.w, (int)q.w, acc, false);
    }
    float y = ((float)acc * a.xscale[t]) * a.wscale[o];
    if (a.bias) y += a.bias[o];
    i8_store(a.out, (size_t)t * a.out_stride + o, y, a.dtype_out);
}

hipError_t launch_i8_quantize(const void *x, size_t stride, int8_t *xq, float *scale, int n_tok,
                              int in_dim, uint32_t dtype, hipStream_t s) {
    if (n_tok <= 0) return hipSuccess;
    k_i8_quantize<<<(unsigned)n_tok, 256, 0, s>>>(x, stride, xq, scale, in_dim,
                                                 (int)i8_row_bytes(in_dim), dtype);
    return hipGetLastError();
}

size_t i8_split_bytes(int n_tok, int in_dim, int out_dim) { return 0; }

hipError_t launch_i8_matmul(const I8Args &a, uint8_t *split, hipStream_t s) {
    if (a.n_tok <= 0) return hipSuccess;
    const dim3 grid((unsigned)((a.out_dim + 63) / 64), (unsigned)((a.n_tok + 3) / 4));
    k_i8_simple<<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace rsllm_hip
