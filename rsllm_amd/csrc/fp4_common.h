// What the kernels of 4-bit codes share: loads and stores of the three float types,
// scale bytes, decoding.
#pragma once

#include "kernels.h"

namespace rsllm_hip {

typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef float mx_v4f __attribute__((ext_vector_type(4)));
typedef __bf16 mx_bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf8 __attribute__((ext_vector_type(8)));

template <uint32_t DT> __device__ __forceinline__ float mx_load(const void *p, size_t i) {
    if constexpr (DT == T_F32) return static_cast<const float *>(p)[i];
    const uint16_t b = static_cast<const uint16_t *>(p)[i];
    return DT == T_F16 ? f16_to_f32(b) : __builtin_bit_cast(float, (uint32_t)b << 16);
}
// One f32 rounded to the type (half to even), NaN kept.
__device__ __forceinline__ void mx_store(void *p, size_t i, float v, uint32_t dtype) {
    if (dtype == T_F32) {
        static_cast<float *>(p)[i] = v;
    } else if (dtype == T_F16) {
        static_cast<_Float16 *>(p)[i] = (_Float16)v;
    } else {
        static_cast<__bf16 *>(p)[i] = (__bf16)v;
    }
}
// Eight values of a row from element i on; those behind its end are 0. vec: the row
// is 16-byte aligned there.
template <uint32_t DT>
__device__ __forceinline__ void mx_load8(const void *x, size_t row, int i, int in_dim, bool vec, float *v) {
    if (vec && i + 8 <= in_dim) {
        if constexpr (DT == T_F32) {
            const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(x) + row + i);
            const float4 a = p[0], b = p[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + row + i);
            const uint32_t d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[2 * k] = DT == T_F16 ? f16_to_f32(d[k] & 0xFFFFu) : __builtin_bit_cast(float, d[k] << 16);
                v[2 * k + 1] = DT == T_F16 ? f16_to_f32(d[k] >> 16) : __builtin_bit_cast(float, d[k] & 0xFFFF0000u);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = i + k < in_dim ? mx_load<DT>(x, row + i + k) : 0.0f;
    }
}
// 2^(s - 127) as the scaled conversions read it: they take a float's exponent bits
// alone (0 counts as 2^-127, 255 as NaN).
__device__ __forceinline__ float mx_unit(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

}  // namespace rsllm_hip
