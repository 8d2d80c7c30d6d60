// exl3_rope.h -- rotary angles and the rotation of a head's elements, for the kernels that write a paged cache.
#pragma once
#include "exl3_attn.h"

namespace exl3 {

// position * freq / (2 pi) less its whole turns.  1 / (2 pi) in two doubles, and each product's rounding error by
// fma: what is lost is below 2^-100 of the angle, so the fraction is good to 32 bits for any position below 2^53.
__device__ __forceinline__ double turn_fraction(double position, double freq)
{
#pragma clang fp contract(off)                          // a product that a subtraction absorbs has no error to add
    constexpr double C_HI = 0x1.45f306dc9c883p-3, C_LO = -0x1.6b01ec5417056p-57;
    const double g = freq * C_HI, g_err = fma(freq, C_HI, -g) + freq * C_LO;
    const double turns = position * g, err = fma(position, g, -turns) + position * g_err;
    const double x = (turns - floor(turns)) + err;
    return x - floor(x);
}

// What 8 elements of a head from column c on pair with (half layout with whole pieces; else nothing): requested with them, so
// that it is there when the angles are.
template <class T, int LAYOUT>
__device__ __forceinline__ u32x4 partner8(const uint16_t* head, int c, int rot)
{
    if constexpr (LAYOUT == ROPE_HALF)
        if (c < rot) return *reinterpret_cast<gc_u32x4*>(as_global(head) + (c < rot / 2 ? c + rot / 2 : c - rot / 2));
    return u32x4{0u, 0u, 0u, 0u};
}

// The rotated ones of 8 elements x of a head from column c on: put(i, value), values in fp32.  other: partner8's; cs: the
// token's (cos, sin) per frequency.
template <class T, int LAYOUT, class Put>
__device__ __forceinline__ void rotate8(u32x4 xb, u32x4 other, const uint16_t* head, int c, int rot, const float2* cs, Put&& put)
{
    using V = typename Elem<T>::x8;
    const V x = __builtin_bit_cast(V, xb);
    const int half = rot / 2;
    if constexpr (LAYOUT == ROPE_HALF) {               // half % 8 == 0: the whole piece pairs with one piece
        if (c < rot) {
            const bool low = c < half;
            const V o = __builtin_bit_cast(V, other);
            const float2* f = cs + (low ? c : c - half);
#pragma unroll
            for (int i = 0; i < 8; ++i) put(i, (float) x[i] * f[i].x + (low ? -(float) o[i] : (float) o[i]) * f[i].y);
        }
    } else if constexpr (LAYOUT == ROPE_PAIRS) {       // pairs side by side
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if (c + i < rot) {
                const float2 f = cs[(c + i) / 2];
                const float u = (float) x[i], w = (float) x[i + 1];
                put(i, u * f.x - w * f.y);
                put(i + 1, w * f.x + u * f.y);
            }
    } else {                                           // half layout with an odd boundary: element by element
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = c + i;
            if (e < rot) {
                const bool low = e < half;
                const float o = (float) __builtin_bit_cast(T, (uint16_t) *(as_global(head) + (low ? e + half : e - half)));
                const float2 f = cs[low ? e : e - half];
                put(i, (float) x[i] * f.x + (low ? -o : o) * f.y);
            }
        }
    }
}

// ... rounded to the element type, the others as they were
template <class T, int LAYOUT>
__device__ __forceinline__ u32x4 rotated8(u32x4 xb, u32x4 other, const uint16_t* head, int c, int rot, const float2* cs)
{
    auto y = __builtin_bit_cast(typename Elem<T>::x8, xb);
    rotate8<T, LAYOUT>(xb, other, head, c, rot, cs, [&](int i, float v) __attribute__((always_inline)) { y[i] = (T) v; });
    return __builtin_bit_cast(u32x4, y);
}

}  // namespace exl3
