// exl3_attn.h -- what the paged-cache kernels share: element types, argument checks, limits.
#pragma once
#include "exl3_device.h"
#include <algorithm>
#include <initializer_list>

namespace exl3 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <class T> struct Elem;
template <> struct Elem<f16> { typedef f16x8 x8; };
template <> struct Elem<__bf16> { typedef bf16x8 x8; };

enum { ROPE_HALF, ROPE_PAIRS, ROPE_ANY };
constexpr int ROPE_GROUP = 4;                           // most tokens of a rotary workgroup

inline bool paged_head_dim(int d) { return d == 64 || d == 128 || d == 256; }
inline bool paged_dtype(int t) { return t == EXL3_FP16 || t == EXL3_BF16; }
inline bool aligned16(std::initializer_list<const void*> ps)
{
    return std::all_of(ps.begin(), ps.end(), [](const void* p) { return ((uintptr_t) p & 15u) == 0; });
}
inline bool multiples_of_8(std::initializer_list<int64_t> ld)
{
    return std::all_of(ld.begin(), ld.end(), [](int64_t s) { return s >= 0 && s % 8 == 0; });
}

}  // namespace exl3
