// exl3_cache8.h -- the paged cache in 8 bits: what the kernels that write it, read it back and attend over it share.
//
// A value is code * scale: the code a whole number in 8 bits, the scale one fp32 number for each 16 tokens of a page and kv head
// (2048 codes at 128 columns: 0.2 % more bytes).  The writer's scales are powers of two, so that every product and quotient by one is
// exact: a value has one right code, whatever the order of the arithmetic, and rows that are rounded anew when their block's
// scale doubles are rounded from what they stood for.  A scale that fits the largest value exactly would have steps two thirds
// as large on average; but tokens come one at a time, and each that raises a block's largest value would round its other rows
// once more.
// Every byte is a finite number, so what lies in rows that nobody sees (old codes, memory never written) needs no masking in
// products: a probability of 0 hides it.  Scales there may be anything, and are clamped where they are read.
#pragma once
#include "exl3_attn.h"

namespace exl3 {

constexpr int C8_BLOCK = EXL3_CACHE8_BLOCK;
constexpr int C8_LEAST = -40, C8_MOST = 40;             // exponents of the writer's scales

struct Cache8 {
    int8_t *k, *v;
    float *ks, *vs;
    int64_t k_ldp, k_ldt, k_ldh, v_ldp, v_ldt, v_ldh, ks_ldp, ks_ldb, ks_ldh, vs_ldp, vs_ldb, vs_ldh;
    int pages, page, hkv, d;
    UDiv d_page;
};

// The host's checks of a caller's cache, and its strides: one that addresses nothing may be anything.  False: refused.
inline bool cache8_of(const exl3_cache8* c, Cache8& o)
{
    if (!c || c->kv_heads < 1 || c->kv_heads > EXL3_PAGED_MAX_HEADS || !paged_head_dim(c->head_dim)) return false;
    if (c->pages < 0 || c->page_size < C8_BLOCK || c->page_size % C8_BLOCK || c->page_size > EXL3_PAGED_MAX_PAGE) return false;
    if ((int64_t) c->pages * c->page_size > INT32_MAX) return false;
    if (c->pages && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return false;
    o = Cache8{(int8_t*) c->k, (int8_t*) c->v, (float*) c->k_scale, (float*) c->v_scale, c->k_ldp, c->k_ldt, c->k_ldh, c->v_ldp, c->v_ldt, c->v_ldh,
               c->ks_ldp, c->ks_ldb, c->ks_ldh, c->vs_ldp, c->vs_ldb, c->vs_ldh, c->pages, c->page_size, c->kv_heads, c->head_dim,
               UDiv::of((uint32_t) c->page_size)};
    if (o.pages <= 1) o.k_ldp = o.v_ldp = o.ks_ldp = o.vs_ldp = 0;
    if (o.hkv == 1) o.k_ldh = o.v_ldh = o.ks_ldh = o.vs_ldh = 0;
    if (o.page == C8_BLOCK) o.ks_ldb = o.vs_ldb = 0;
    for (int64_t s : {o.k_ldp, o.k_ldt, o.k_ldh, o.v_ldp, o.v_ldt, o.v_ldh})
        if (s < 0 || s % 16) return false;
    for (int64_t s : {o.ks_ldp, o.ks_ldb, o.ks_ldh, o.vs_ldp, o.vs_ldb, o.vs_ldh})
        if (s < 0) return false;
    if (o.k_ldt > EXL3_ATTN_MAX_LDT || o.v_ldt > EXL3_ATTN_MAX_LDT) return false;
    return aligned16({o.k, o.v}) && (((uintptr_t) o.ks | (uintptr_t) o.vs) & 3u) == 0;
}

// a scale as it is used: between the writer's least and most, whatever the memory holds (NaN: the least)
__device__ __forceinline__ float scale8(float s)
{
    return fminf(fmaxf(s, __builtin_ldexpf(1.f, C8_LEAST)), __builtin_ldexpf(1.f, C8_MOST));
}

// Two codes as fp16 numbers.  0x6400 + b is 1024 + b in fp16 for a byte b, and a code with its sign bit flipped is the byte
// code + 128, so 1152 too much: the subtraction is exact.
constexpr uint32_t C8_FLIP = 0x80808080u, C8_ONE = 0x64646464u;
__device__ __forceinline__ uint32_t less_1152(uint32_t x)
{
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - f16x2{(f16) 1152.f, (f16) 1152.f});
}
// bytes 2 h and 2 h + 1 of w ^ C8_FLIP
__device__ __forceinline__ uint32_t codes2(uint32_t flipped_w, int h)
{
    return less_1152(__builtin_amdgcn_perm(C8_ONE, flipped_w, h ? 0x04030402u : 0x04010400u));
}
// byte e of lo and of hi
__device__ __forceinline__ uint32_t codes2_of(uint32_t lo, uint32_t hi, int e)
{
    return less_1152(__builtin_amdgcn_perm(hi, lo, 0x0C000C00u | (uint32_t) (4 + e) << 16 | (uint32_t) e) ^ 0x64806480u);
}

}  // namespace exl3
