// edge_stream.hpp -- what the trainable attentions over a graph's edges share
// (diff_attention.hip, edge_attention.hip): rows of strided tensors, LDS accesses by
// address, row masks of a chunk's slots, the scaling of weights into binary16.
#pragma once

#include "attn_plan.hpp"
#include "half_types.hpp"

namespace f3s {

// The lane again, for the compiler a new value: what is derived from it is then made
// where it is used and not held in registers through the chunk loop.
__device__ __forceinline__ int anew(int lane)
{
    asm volatile("" : "+v"(lane));
    return lane;
}

// Rows r of a tensor start `stride` bytes apart; a head's values are
// contiguous, heads adjacent.
struct EdgeRows {
    const char* ptr;
    uint64_t stride;
    uint32_t bytes;   // narrow launches: end of the last row (loads past it read 0)
};

typedef __attribute__((address_space(3))) char* LdsPtr;
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at)
{
    return *(__attribute__((address_space(3))) V*)(LdsPtr)(uintptr_t)at;
}
template <typename V>
__device__ __forceinline__ void lds_write(uint32_t at, V v)
{
    *(__attribute__((address_space(3))) V*)(LdsPtr)(uintptr_t)at = v;
}

// Which of the lane's eight slots row r attends: all bits or none.
typedef uint32_t Attends[8];
__device__ __forceinline__ float where(uint32_t on, float x, float other)
{
    return __uint_as_float((__float_as_uint(x) & on) | (__float_as_uint(other) & ~on));
}
__device__ __forceinline__ float where(uint32_t on, float x)
{
    return __uint_as_float(__float_as_uint(x) & on);
}

// From a record's masks at `masks`, anew wherever they are used: two LDS reads,
// where eight registers would be held.
__device__ __forceinline__ void attends(uint32_t masks, int lane, Attends& on)
{
    const int l = anew(lane), r = l & 15, rbit = (r & 1) ? 16 + (r >> 1) : (r >> 1);
    const uint32_t at = masks + 16 * (l >> 4);   // slots 4 g .. and 16 + 4 g ..
    const u4 a = lds_read<u4>(at), b = lds_read<u4>(at + 64);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        on[j] = (uint32_t)__builtin_amdgcn_sbfe((int)(j < 4 ? a[j & 3] : b[j & 3]), rbit, 1);
}

// The same of slots 16 t + 4 g .. alone.
__device__ __forceinline__ void attends_half(uint32_t masks, int t, int lane, uint32_t (&on)[4])
{
    const int l = anew(lane), r = l & 15, rbit = (r & 1) ? 16 + (r >> 1) : (r >> 1);
    const u4 a = lds_read<u4>(masks + 64 * t + 16 * (l >> 4));
#pragma unroll
    for (int j = 0; j < 4; ++j) on[j] = (uint32_t)__builtin_amdgcn_sbfe((int)a[j], rbit, 1);
}

// Weights of a size of 1 at most, in binary16: with |w| <= 2 they stay below 2^15, and
// their halves end at 2^-39.  (A node that a row hardly attends, or that only rows of
// very many edges do, has weights of 2^-17 and less alone: unscaled, 2^-20 was off by
// 2^-6 of itself.)
// (In the rows' pass as an addend of the exponent: all its sums are divided by the
// weights' own.  A row of 10^5 equal edges has weights of 2^-17, all rounded the same
// way: dq, a difference of two sums of them, was off by 2^-8 of either.)
template <typename T>
constexpr float kLift = Half<T>::kRange ? 16384.f : 1.f;
template <typename T>
constexpr float kLiftLog2 = Half<T>::kRange ? 14.f : 0.f;
// Such a weight's exponent.  A weight is at most 1, but for what a log-sum-exp of 24
// bits leaves (logits past 2^24 come out as 2^2 and more): kept at 2 (rows, lifted) and
// at 1 (columns), inside the type.  NaN stays.
template <typename T>
__device__ __forceinline__ float lifted(float x, float most)
{
    return Half<T>::kRange ? __builtin_elementwise_minimum(x, most) : x;
}

__device__ __forceinline__ float over_groups(float x)
{
    x += __shfl_xor(x, 16, kWave);
    return x + __shfl_xor(x, 32, kWave);
}

__device__ __forceinline__ float uniform(float x)
{
    return __uint_as_float(__builtin_amdgcn_readfirstlane((int)__float_as_uint(x)));
}

template <typename V>
__device__ __forceinline__ V scalar_load(const V* at)
{
    typedef const __attribute__((address_space(4))) V* Constant;
    return *(Constant)(uintptr_t)at;
}

static inline size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

static inline EdgeRows rows_of(const void* ptr, int64_t stride)
{
    return EdgeRows{static_cast<const char*>(ptr), (uint64_t)stride * 2, 0};
}

}  // namespace f3s
