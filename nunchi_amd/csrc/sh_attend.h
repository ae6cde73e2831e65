// What the attention kernels over pages share (sh_page_attn.hip, sh_tree_attn.hip): the matrix instructions of either type, the
// rounding and rescaling of weights, and the request of a row.
#pragma once
#include <hip/hip_runtime.h>

#include "sh_device.h"
#include "sh_serve.h"

namespace sh {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <class T> struct mat;
template <> struct mat<_Float16> {
    static constexpr unsigned EXP = 0x7C00u;   // the exponent bits of one value: all set in infinities and NaN
    static constexpr unsigned ONE = 0x3C00u;
    static constexpr float SLACK = 4.0f, LIFT = 11.0f;   // weights up to 2^15; their last place is 2^-35 of the largest
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct mat<__bf16> {
    static constexpr unsigned EXP = 0x7F80u, ONE = 0x3F80u;
    static constexpr float SLACK = 8.0f, LIFT = 0.0f;    // (eight bits of exponent hold any weight)
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <class T> __device__ __forceinline__ unsigned pack2(float x, float y) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    const t2 v = {(T)x, (T)y};   // to nearest
    return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// e^(from - to) in powers of two for maxima that may be -inf (nothing seen yet)
__device__ __forceinline__ float rescale(float from, float to) { return from == -INFINITY ? 0.0f : exp2_(from - to); }

// the request whose rows hold `row` (the last k with cu[k] <= row)
__device__ __forceinline__ int request_of(const int32_t* cu, int n, int row) {
    int x = 0, y = n;
    while (y - x > 1) {
        const int mid = (x + y) >> 1;
        if (cu[mid] <= row) x = mid;
        else y = mid;
    }
    return x;
}

}  // namespace
}  // namespace sh
