// half_types.hpp -- the 16-bit types that the differential attention and the
// projections with an epilogue take (binary16 and bfloat16), their MFMA and
// the split of a float32 weight into two of them.
#pragma once

#include "attn_common.hpp"

namespace f3s {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// kRange: weights have to be scaled into the type's range (binary16 ends at
// 65,504 and thins out below 2^-14; bfloat16 has float32's exponents).
template <typename T>
struct Half;

template <>
struct Half<_Float16> {
    typedef h8 v8;
    typedef h4 v4;
    typedef h2 v2;
    static constexpr bool kRange = true;
    static __device__ __forceinline__ f4 mfma(v8 a, v8 b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

template <>
struct Half<__bf16> {
    typedef b8 v8;
    typedef b4 v4;
    typedef b2 v2;
    static constexpr bool kRange = false;
    static __device__ __forceinline__ f4 mfma(v8 a, v8 b, f4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// w = hi + lo: the rounded value and what the rounding left, rounded in its
// turn.  A product with both has 2^-22 of w left (binary16; 2^-18 bfloat16, and
// never under 2^-25 in binary16's subnormals) where one rounding leaves 2^-11.
template <typename T>
__device__ __forceinline__ void split8(const float (&w)[8], typename Half<T>::v8& hi,
                                       typename Half<T>::v8& lo)
{
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const f2 x = {w[j], w[j + 1]};
        const typename Half<T>::v2 h = __builtin_convertvector(x, typename Half<T>::v2);
        hi[j] = h[0];
        hi[j + 1] = h[1];
        const f2 rest = {w[j] - (float)h[0], w[j + 1] - (float)h[1]};
        const typename Half<T>::v2 l = __builtin_convertvector(rest, typename Half<T>::v2);
        lo[j] = l[0];
        lo[j + 1] = l[1];
    }
}

}  // namespace f3s
