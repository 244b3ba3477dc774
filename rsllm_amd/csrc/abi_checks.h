// Argument checks that the device-pointer entry points of the serving and 4-bit calls
// share.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/rsllm_hip.h"
#include "abi_internal.h"
#include "kernels.h"

namespace rsllm_hip::abi {

#define HIP_TRY(expr, where)                                  \
    do {                                                      \
        hipError_t e_ = (expr);                               \
        if (e_ != hipSuccess) return abi::device_error(e_, where); \
    } while (0)

inline int invalid(const char *m) { return set_error(RSLLM_HIP_ERR_INVALID_ARGUMENT, m); }
inline int mismatch(const char *m) { return set_error(RSLLM_HIP_ERR_SHAPE_MISMATCH, m); }

inline bool float_type(uint32_t t) { return t == T_F32 || t == T_F16 || t == T_BF16; }
inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline size_t elem_bytes(uint32_t t) { return t == T_F32 ? 4 : 2; }

// rows of `row` elements, `stride` apart, inside len elements (0 rows: any)
inline bool span_ok(size_t rows, size_t row, size_t stride, size_t len) {
    size_t n;
    return rows == 0 || (!__builtin_mul_overflow(rows - 1, stride, &n) &&
                         !__builtin_add_overflow(n, row, &n) && n <= len);
}
inline bool product_is(size_t a, size_t b, size_t len) {
    size_t n;
    return !__builtin_mul_overflow(a, b, &n) && n == len;
}
// Rows or channels of one call. A launch holds less than 2^32 threads: these with
// up to 512 a row, and the int8 product's tiles of as many rows and channels as
// fit memory (below 2^31 threads, over all such sizes).
constexpr size_t kMaxRows = ((size_t)1 << 23) - 1;
inline bool counts_ok(size_t n) { return n <= kMaxRows; }

inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace rsllm_hip::abi
