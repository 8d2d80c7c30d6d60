// exl3_attn8.h -- what the attention kernels over a paged cache in 8 bits share.
#pragma once
#include "exl3_cache8.h"

namespace exl3 {

struct Attn8Args : AttnArgs {
    Cache8 c;
};

__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }   // base 2

// A row's factor of its scores: never 0, which would make NaN of a masked score's infinity, and next to nothing where it would be
__device__ __forceinline__ float row_scale_of(float scale, float qs)
{
    const float f = scale * qs;
    return f < 1e-37f ? 1e-37f : f;
}

// Rows of q as fp16, the products' type; all of a row's lanes call it with their pieces, and row_max gives each the largest value
// over the row's.  fp16 ones stay as they are.  A bf16 row is divided by the power of two that leaves its largest finite element in
// [2^14, 2^15), which fp16's 11 bits hold without rounding down to 2^-28 of it; the power is returned, to go into the scores'
// factor.
template <class T, int N, class RowMax>
__device__ __forceinline__ float fp16_rows(u32x4 (&q)[N], RowMax&& row_max)
{
    if constexpr (std::is_same_v<T, f16>) {
        return 1.f;
    } else {
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = fabsf((float) __builtin_bit_cast(bf16x8, q[c])[i]);
                m = fmaxf(m, x < INFINITY ? x : 0.f);
            }
        m = row_max(m);
        // both powers are to be normal numbers
        const int e = min(max((int) ((uint32_t) __float_as_int(m) >> 23) - 127, -112), 127);
        const float f = __int_as_float((127 + 14 - e) << 23);
#pragma unroll
        for (int c = 0; c < N; ++c) {
            f16x8 y;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (f16) ((float) __builtin_bit_cast(bf16x8, q[c])[i] * f);
            q[c] = __builtin_bit_cast(u32x4, y);
        }
        return __int_as_float((127 - 14 + e) << 23);
    }
}

// many rows a request, `rows` for each kv head on average (exl3_attn8_prefill.hip)
void launch_attn8_prefill(const Attn8Args& a, int64_t rows, int dtype, hipStream_t s);

}  // namespace exl3
