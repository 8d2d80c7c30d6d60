// exl3_paged8.hip -- the paged cache in 8 bits: rotary embedding with k and v quantised into it (exl3_rope_kv_write8), and
// tokens read back from it (exl3_kv_read8).
#include "exl3_cache8.h"
#include "exl3_rope.h"

using namespace exl3;

namespace {

typedef __attribute__((address_space(1))) u32x2 g_u32x2;

struct Write8Args {
    const uint16_t *q, *k, *v;
    int64_t q_ldt, q_ldh, k_ldt, k_ldh, v_ldt, v_ldh;
    const int64_t *pos, *slots;
    uint16_t* out;
    Cache8 c;
    const double* inv_freq;
    float mscale;
    int tokens, hq, rot;
    int rows, heads, head_parts, turns, turn_wgs;                 // a k/v workgroup's rows of the batch, its kv heads, workgroups over the heads; workgroups that take a window's blocks in turn
    int kv_wgs, q_parts;                                // k/v workgroups in front of the q ones; workgroups of a token's q
};

// The smallest exponent e of a scale with 127 * 2^e >= most, within the writer's.
__device__ __forceinline__ int exponent8(float most)
{
    const uint32_t b = (uint32_t) __float_as_int(most);
    const int e = (int) (b >> 23) - 127 - 6 + ((b & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);     // 127 / 64 = 1.984375: the mantissa 0x7E0000
    return min(max(e, C8_LEAST), C8_MOST);
}
__device__ __forceinline__ float power2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ float reciprocal8(float s)      // of a scale: from its exponent where it is a power of two
{
    const int b = __float_as_int(s);
    return b & 0x7FFFFF ? 1.f / s : __int_as_float((254 << 23) - b);
}

__device__ __forceinline__ float finite_abs(float x)
{
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;                      // NaN compares false
}

// Codes of 8 values, whose quotient by the scale is exact (a power of two).  Values of at most 127 steps are rounded to even by the
// addition of 1.5 2^23, which leaves the whole number in the sum's low bits; `odd`: some may be more, infinite or NaN.
// middle: bit i if value i may be, as far as values off by up to `off` tell, on the other side of the middle between two codes.
__device__ __forceinline__ u32x2 codes_of(const float (&x)[8], float inv, bool odd, float off, uint32_t& middle)
{
    constexpr float MAGIC = 12582912.f;
    const float limit = fmaf(off, -inv, 0.5f);
    uint32_t b[8];
    middle = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float sum = fmaf(x[i], inv, MAGIC), rest = fmaf(x[i], inv, -(sum - MAGIC));
        b[i] = (uint32_t) __float_as_int(sum);
        middle |= fabsf(rest) >= limit ? 1u << i : 0u;
    }
    if (__builtin_expect(odd, 0)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = x[i] == x[i] ? (uint32_t) (int) rintf(fminf(fmaxf(x[i] * inv, -127.f), 127.f)) : 0u;
    }
    u32x2 r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        r[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x0C0C0400u),
                                     __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0C0C0400u), 0x05040100u);
    return r;
}

// A rotated element in float64: element e of the head at `head`, in the token at position pos.  Called, not inlined: its two uses' constants
// would spill what the block has under way (128 decodes, 40 heads over 8 of 128, 8.7 us instead of 8.0; 8192 tokens of heads of 256 70 instead of 61).
template <class T, int LAYOUT>
__device__ __attribute__((noinline)) double rotated_f64(const uint16_t* head, int e, int rot, int64_t pos, const double* freq, float mscale)
{
    auto at = [&](int i) __attribute__((always_inline)) { return (double) (float) __builtin_bit_cast(T, (uint16_t) *(as_global(head) + i)); };
    const int half = rot / 2;
    const bool first = LAYOUT == ROPE_PAIRS ? e % 2 == 0 : e < half;
    const double x = at(e), y = at(LAYOUT == ROPE_PAIRS ? e ^ 1 : first ? e + half : e - half);
    double s, c;
    sincospi(2.0 * turn_fraction((double) pos, freq[LAYOUT == ROPE_PAIRS ? e / 2 : first ? e : e - half]), &s, &c);
    return (x * c + (first ? -y : y) * s) * mscale;
}
// The largest finite one of 8 elements of a head from column c on, the rotated ones in float64 and rounded up: it passes 127 of a scale if and
// only if one of them does.  x: the elements before the rotation.
template <class T, int LAYOUT>
__device__ __forceinline__ float exact_top(u32x4 x, const uint16_t* head, int c, int rot, int64_t pos, const double* freq, float mscale)
{
    const auto e = __builtin_bit_cast(typename Elem<T>::x8, x);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, c + i < rot ? 0.f : finite_abs((float) e[i]));
#pragma unroll 1
    for (int i = 0; i < min(rot - c, 8); ++i) {
        const double y = fabs(rotated_f64<T, LAYOUT>(head, c + i, rot, pos, freq, mscale));
        const float z = (float) y;
        top = fmaxf(top, z < INFINITY ? (double) z < y ? __int_as_float(__float_as_int(z) + 1) : z : 0.f);
    }
    return top;
}
// codes of a row whose block's scale grew by 1 / f
__device__ __forceinline__ u32x2 rounded_anew(u32x2 old, float f)
{
    u32x2 r = u32x2{0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = (int) (int8_t) (uint8_t) (old[i >> 2] >> (8 * (i & 3)));
        r[i >> 2] |= ((uint32_t) (int) rintf((float) c * f) & 0xFFu) << (8 * (i & 3));
    }
    return r;
}

// The largest of a wave's 64 values, in every lane.
__device__ __forceinline__ float wave_max(float x)
{
    auto with = [&](auto CTRL) __attribute__((always_inline)) {
        x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(CTRL)::value, 0xF, 0xF, true)));
    };
    with(std::integral_constant<int, 0xB1>{});          // quad_perm 1 0 3 2
    with(std::integral_constant<int, 0x4E>{});          // quad_perm 2 3 0 1
    with(std::integral_constant<int, 0x141>{});         // row_half_mirror
    with(std::integral_constant<int, 0x140>{});         // row_mirror
    return max_quads(x);
}

// One launch, two kinds of workgroups.  The first kv_wgs quantise k and v: workgroup (w, p) takes the blocks whose first row
// in the batch is one of [rows w, rows (w + 1)), for the kv heads of part p.  A block's rows are consecutive in the batch, so one
// workgroup has all of a block's new tokens, and its scale needs no second pass and no other workgroup.  A thread
// holds 8 elements of k and v of one of the block's 16 rows: new rows from the batch, the others' codes from the cache, requested at
// once whether the scale will grow or not, with the angles formed meanwhile: a block takes two trips to memory (its slots and
// positions, then all else), and a further head's is under way while the head before is computed.  The other workgroups rotate q.
// A rotated k has the scale and code of its exact value: fp32 decides, but for blocks whose largest it leaves next to 127 steps of a scale, and
// elements next to the middle between two codes; these are rotated again in float64 (rotating all of them in float64 takes 8192 tokens 79 us
// instead of 49).
// Prompts are bound by memory: 8192 tokens of 40 heads over 8 of 128 (218 MB) in 47 us one after the other, 4.6 TB/s, and 60 among other
// launches; of 24 over 4 of 256 (252 MB) 79 to 87 (pairs side by side: 61), 3.0 TB/s (two tokens a q workgroup: 78.5 instead of 81, but 2048 tokens
// 26.7 instead of 25.8).  Decodes are
// bound by a chain of waits: 32 in 5.8 us (q alone 2.8, slots 0.3, the rest of the block's loads 1.0, codes and stores 1.5; the exact
// ones 0.2).  The 16-bit cache's kernel, which needs no block's maximum, takes 2.8.
template <class T, int D, int LAYOUT>
__global__ void __launch_bounds__(2 * D, 4) rope_kv_write8_kernel(Write8Args a)
{
    constexpr int PIECES = D / 8, THREADS = C8_BLOCK * PIECES, WAVES = THREADS / 64;
    constexpr int FREQS = (D / 2 + 63) / 64;            // frequencies of a lane
    constexpr int QN = 3;                               // pieces of q that a thread has under way
    __shared__ float2 cs[C8_BLOCK][D / 2];
    __shared__ int src[C8_BLOCK];                       // the block's rows: their token in the batch, -1 none
    __shared__ int64_t pos[C8_BLOCK];                   // ... and its position
    __shared__ double freqs[D / 2];
    __shared__ float tops[2][WAVES][2];                 // largest values of k and v of each wave; heads take turns
    using V8 = typename Elem<T>::x8;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto cos_sin = [&](int64_t pos, double freq) __attribute__((always_inline)) {
        float s, c;
        sincospif(2.f * (float) turn_fraction((double) pos, freq), &s, &c);
        return make_float2(c * a.mscale, s * a.mscale);
    };

    if ((int) blockIdx.x >= a.kv_wgs) {
        const int b = (int) blockIdx.x - a.kv_wgs, tok = b / a.q_parts, part = b - tok * a.q_parts, items = a.hq * PIECES;
        for (int i0 = part * THREADS + tid; i0 - tid < items; i0 += QN * THREADS * a.q_parts) {
            u32x4 x[QN], o[QN];
            auto head_of = [&](int i) __attribute__((always_inline)) { return a.q + (int64_t) tok * a.q_ldt + (int64_t) (i / PIECES) * a.q_ldh; };
#pragma unroll
            for (int j = 0; j < QN; ++j) {
                const int i = i0 + j * THREADS * a.q_parts;
                if (i < items) {
                    x[j] = *reinterpret_cast<gc_u32x4*>(as_global(head_of(i)) + 8 * (i % PIECES));
                    o[j] = partner8<T, LAYOUT>(head_of(i), 8 * (i % PIECES), a.rot);
                }
            }
            if (i0 == part * THREADS + tid) {
                for (int f = tid; f < a.rot / 2; f += THREADS) cs[0][f] = cos_sin(a.pos[tok], a.inv_freq[f]);
                __syncthreads();
            }
#pragma unroll
            for (int j = 0; j < QN; ++j) {
                const int i = i0 + j * THREADS * a.q_parts, c = 8 * (i % PIECES);
                if (i < items) *reinterpret_cast<g_u32x4*>(as_global(a.out) + ((int64_t) tok * items + i) * 8) = rotated8<T, LAYOUT>(x[j], o[j], head_of(i), c, a.rot, cs[0]);
            }
        }
        return;
    }

    const int my_turn = (int) blockIdx.x / a.turn_wgs, z = (int) blockIdx.x - my_turn * a.turn_wgs;
    const int w = z / a.head_parts, h0 = (z - w * a.head_parts) * a.heads, h1 = min(h0 + a.heads, a.c.hkv), row0 = w * a.rows;
    const int64_t cache_slots = (int64_t) a.c.pages * a.c.page;
    auto slot_of = [&](int t) __attribute__((always_inline)) {                       // -1: a row of the batch that goes nowhere
        if (t < 0 || t >= a.tokens) return -1;
        const int64_t s = a.slots[t];
        return s >= 0 && s < cache_slots ? (int) s : -1;
    };
    // lane l: rows row0 + l and the one before.  A block begins where the row before belongs to another (-1 >> 4 is -1: none).
    const int slot = slot_of(row0 + lane), mine = slot >> 4, prior = slot_of(row0 + lane - 1) >> 4;
    static_assert(C8_BLOCK == 16);
    double freq[FREQS];
#pragma unroll
    for (int i = 0; i < FREQS; ++i) freq[i] = lane + 64 * i < a.rot / 2 ? a.inv_freq[lane + 64 * i] : 0.0;
    if (wave == 0)
#pragma unroll
        for (int i = 0; i < FREQS; ++i)
            if (lane + 64 * i < D / 2) freqs[lane + 64 * i] = freq[i];
    uint64_t begins = __ballot(lane < a.rows && mine >= 0 && mine != prior);
    for (int i = 0; begins; begins &= begins - 1, ++i) {
        if (i % a.turns != my_turn) continue;
        const int at = __builtin_ctzll(begins), block = __builtin_amdgcn_readlane(mine, at);
        __syncthreads();                                // of the block before: src, cs and tops are free
        if (tid < C8_BLOCK) src[tid] = -1;
        __syncthreads();
        if (wave == 0) {
            // a slot that comes twice in a block's rows: the last one counts
            uint64_t run = __ballot(mine == block) >> at;
            int n = ~run ? __builtin_ctzll(~run) : 64;
            if (lane >= at && lane < at + n) atomicMax(&src[slot & 15], row0 + lane);
            for (int t = row0 + 64; at + n >= 64; t += 64) {       // more than the lanes' rows
                const int s = slot_of(t + lane);
                run = __ballot(s >> 4 == block);
                n = ~run ? __builtin_ctzll(~run) : 64;
                if (lane < n) atomicMax(&src[s & 15], t + lane);
                if (n < 64) break;
            }
        }
        __syncthreads();
        const bool anew = src[0] >= 0;
        const int page = (int) a.c.d_page.div((uint32_t) block * C8_BLOCK), in = block * C8_BLOCK - page * a.c.page;
        const int row = tid / PIECES, c = 8 * (tid % PIECES), tok = src[row];
        float* ks = a.c.ks + ((int64_t) page * a.c.ks_ldp + (int64_t) (in / C8_BLOCK) * a.c.ks_ldb + (int64_t) h0 * a.c.ks_ldh);
        float* vs = a.c.vs + ((int64_t) page * a.c.vs_ldp + (int64_t) (in / C8_BLOCK) * a.c.vs_ldb + (int64_t) h0 * a.c.vs_ldh);
        int8_t* kc = a.c.k + ((int64_t) page * a.c.k_ldp + (int64_t) (in + row) * a.c.k_ldt + (int64_t) h0 * a.c.k_ldh + c);
        int8_t* vc = a.c.v + ((int64_t) page * a.c.v_ldp + (int64_t) (in + row) * a.c.v_ldt + (int64_t) h0 * a.c.v_ldh + c);
        const uint16_t* k = a.k + ((int64_t) tok * a.k_ldt + (int64_t) h0 * a.k_ldh);
        const uint16_t* v = a.v + ((int64_t) tok * a.v_ldt + (int64_t) h0 * a.v_ldh);
        struct Piece {
            u32x4 k, v, o;                              // new elements and k's partners; or in half of it the codes of a row that stays
            float ks, vs;
        };
        auto request = [&](Piece& x, int d) __attribute__((always_inline)) {       // of head h + d
            u32x4 xk = u32x4{0u, 0u, 0u, 0u}, xv = xk, xo = xk;
            if (tok >= 0) {
                xk = *reinterpret_cast<gc_u32x4*>(as_global(k + d * a.k_ldh) + c);
                xv = *reinterpret_cast<gc_u32x4*>(as_global(v + d * a.v_ldh) + c);
                xo = partner8<T, LAYOUT>(k + d * a.k_ldh, c, a.rot);
            } else if (!anew) {
                const u32x2 ko = *reinterpret_cast<gc_u32x2*>(as_global(kc + d * a.c.k_ldh)), vo = *reinterpret_cast<gc_u32x2*>(as_global(vc + d * a.c.v_ldh));
                xk = u32x4{ko[0], ko[1], 0u, 0u};
                xv = u32x4{vo[0], vo[1], 0u, 0u};
            }
            x = Piece{xk, xv, xo, *as_global(ks + d * a.c.ks_ldh), *as_global(vs + d * a.c.vs_ldh)};
        };
        Piece now, next;
        request(now, 0);
        for (int r = wave; r < C8_BLOCK; r += WAVES) {
            const int t = src[r];
            if (t < 0) continue;
            const int64_t p = a.pos[t];
            if (lane == 0) pos[r] = p;
#pragma unroll
            for (int i = 0; i < FREQS; ++i)
                if (lane + 64 * i < a.rot / 2) cs[r][lane + 64 * i] = cos_sin(p, freq[i]);
        }
        __syncthreads();
        for (int h = h0; h < h1; ++h) {
            if (h + 1 < h1) request(next, 1);
            float x[8], y[8], top_k = 0.f, top_v = 0.f, top_in = 0.f;
            bool odd = false;                           // some of the thread's elements are infinite, NaN or past all scales
            if (tok >= 0) {
                const V8 e = __builtin_bit_cast(V8, now.k), g = __builtin_bit_cast(V8, now.v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = (float) e[i];
                    y[i] = (float) g[i];
                    top_in = fmaxf(top_in, fabsf(x[i]));
                }
                if constexpr (LAYOUT == ROPE_HALF) {
                    const V8 o = __builtin_bit_cast(V8, now.o);
#pragma unroll
                    for (int i = 0; i < 8; ++i) top_in = fmaxf(top_in, fabsf((float) o[i]));
                } else if constexpr (LAYOUT == ROPE_ANY) {
                    top_in = INFINITY;                  // its partners lie anywhere: all are rotated again
                }
                rotate8<T, LAYOUT>(now.k, now.o, k, c, a.rot, cs[row], [&](int i, float z) __attribute__((always_inline)) { x[i] = z; });
                float any = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    top_k = fmaxf(top_k, fabsf(x[i]));
                    top_v = fmaxf(top_v, fabsf(y[i]));
                    any = fmaf(x[i], 0.f, fmaf(y[i], 0.f, any));
                }
                odd = any != any || fmaxf(top_k, top_v) > 127.f * power2(C8_MOST);
                if (__builtin_expect(any != any, 0)) {
                    top_k = top_v = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        top_k = fmaxf(top_k, finite_abs(x[i]));
                        top_v = fmaxf(top_v, finite_abs(y[i]));
                    }
                }
            }
            const int turn = (h - h0) & 1;
            top_k = wave_max(top_k);
            top_v = wave_max(top_v);
            if (lane == 0) {
                tops[turn][wave][0] = top_k;
                tops[turn][wave][1] = top_v;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                top_k = fmaxf(top_k, tops[turn][i][0]);
                top_v = fmaxf(top_v, tops[turn][i][1]);
            }
            // A pair's larger element is at least its length over 2^1/2, so fp32's error is below 2^-20 of the block's largest: it tells the
            // scale unless that lies within 32 units of its last place (2^-19) of 127 steps.
            if (a.rot && __builtin_expect(abs((__float_as_int(top_k) & 0x7FFFFF) - 0x7E0000) <= 32, 0)) {
                top_k = wave_max(tok >= 0 ? exact_top<T, LAYOUT>(now.k, k, c, a.rot, pos[row], freqs, a.mscale) : 0.f);
                __syncthreads();
                if (lane == 0) tops[turn][wave][0] = top_k;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < WAVES; ++i) top_k = fmaxf(top_k, tops[turn][i][0]);
            }
            // A rotated pair (a, b) in fp32 is off by at most 2^-21 (|a| + |b|) mscale: cosine and sine by 2^-22, products and sum by 2^-23.
            const float off = 0x1p-20f * top_in * fabsf(a.mscale);
            // The codes of 8 elements or of a row that stays, under the block's scale: of k, then of v by the same code (two copies of it:
            // 2048 tokens of 4 heads of 256 27.2 us instead of 25.8, 128 decodes over 8 of 128 8.2 instead of 7.8).
            float top = top_k, was = now.ks, *scale = ks;
            int8_t* to = kc;
            u32x4 old = now.k;
#pragma unroll 1
            for (bool is_k = true;; is_k = false) {
                const float need = power2(exponent8(top)), had = scale8(was);
                const bool grown = anew || need > had;
                const float is = grown ? need : had, inv = reciprocal8(is);
                if (tid == 0 && grown) *as_global(scale) = is;
                auto* const dst = reinterpret_cast<g_u32x2*>(as_global(to));
                if (tok >= 0) {
                    uint32_t middle;
                    u32x2 codes = codes_of(x, inv, odd, off, middle);
                    // what fp32 leaves next to the middle between two codes (never infinities and NaN); v and what is not rotated are exact
                    middle &= !is_k ? 0u : (1u << min(max(a.rot - c, 0), 8)) - 1u;
                    for (; __builtin_expect(middle != 0, 0); middle &= middle - 1u) {
                        const int i = __builtin_ctz(middle);
                        const double q = rint(rotated_f64<T, LAYOUT>(k, c + i, a.rot, pos[row], freqs, a.mscale) * (double) inv);
                        const uint32_t m = 0xFFu << (8 * (i & 3)), b = ((uint32_t) (int) fmin(fmax(q, -127.0), 127.0) & 0xFFu) << (8 * (i & 3));
                        codes[0] = i < 4 ? (codes[0] & ~m) | b : codes[0];
                        codes[1] = i < 4 ? codes[1] : (codes[1] & ~m) | b;
                    }
                    *dst = codes;
                } else if (anew) *dst = u32x2{0u, 0u};
                else if (grown) *dst = rounded_anew(u32x2{old[0], old[1]}, had * inv);
                if (!is_k) break;
                top = top_v, was = now.vs, scale = vs, to = vc, old = now.v;
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = y[i];
            }
            now = next;
            ks += a.c.ks_ldh, vs += a.c.vs_ldh, kc += a.c.k_ldh, vc += a.c.v_ldh, k += a.k_ldh, v += a.v_ldh;
        }
    }
}

template <class T, int D>
void launch_write8(const Write8Args& a, int layout, int wgs, hipStream_t s)
{
    auto* kern = layout == ROPE_HALF ? rope_kv_write8_kernel<T, D, ROPE_HALF>
                 : layout == ROPE_PAIRS ? rope_kv_write8_kernel<T, D, ROPE_PAIRS> : rope_kv_write8_kernel<T, D, ROPE_ANY>;
    hipLaunchKernelGGL(kern, dim3((unsigned) wgs), dim3(2 * D), 0, s, a);
}

struct Read8Args {
    Cache8 c;
    const int64_t* slots;
    uint16_t *k, *v;
    int tokens, items;                                  // 16-code pieces of a token's k and v
    UDiv d_items;
};

// Tokens' k and v as fp16 or bf16 values: a thread turns 16 codes into 32 bytes.  Bound by memory: 120641 tokens of 4 heads of 256 (370 MB) in
// 72 us, 5.1 TB/s; two and four pieces a thread, all requested at once: 79 and 83.
template <class T, int D>
__global__ void __launch_bounds__(256) kv_read8_kernel(Read8Args a)
{
    constexpr int PIECES = D / 16;
    using V8 = typename Elem<T>::x8;
    const int64_t first = (int64_t) blockIdx.x * 256, cache_slots = (int64_t) a.c.pages * a.c.page;
    const int t0 = (int) (first / a.items);             // uniform
    const uint32_t z = (uint32_t) (first - (int64_t) t0 * a.items) + threadIdx.x, dt = a.d_items.div(z);
    const int t = t0 + (int) dt, i = (int) (z - dt * (uint32_t) a.items), p = i % PIECES, y = i / PIECES;
    if (t >= a.tokens) return;
    const bool is_v = y >= a.c.hkv;
    const int h = is_v ? y - a.c.hkv : y;
    u32x4 codes = u32x4{0u, 0u, 0u, 0u};
    float s = 1.f;
    const int64_t slot = a.slots[t];
    if (slot >= 0 && slot < cache_slots) {
        const int page = (int) a.c.d_page.div((uint32_t) slot), in = (int) slot - page * a.c.page;
        codes = *reinterpret_cast<gc_u32x4*>(as_global(is_v ? a.c.v + page * a.c.v_ldp + in * a.c.v_ldt + h * a.c.v_ldh
                                                            : a.c.k + page * a.c.k_ldp + in * a.c.k_ldt + h * a.c.k_ldh) + 16 * p);
        s = *as_global(is_v ? a.c.vs + page * a.c.vs_ldp + in / C8_BLOCK * a.c.vs_ldb + h * a.c.vs_ldh
                            : a.c.ks + page * a.c.ks_ldp + in / C8_BLOCK * a.c.ks_ldb + h * a.c.ks_ldh);
    }
    auto* const dst = as_global(is_v ? a.v : a.k) + ((int64_t) t * a.c.hkv + h) * D + 16 * p;
    const float f = scale8(s);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        V8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (T) ((float) (int8_t) (uint8_t) (codes[2 * j + (e >> 2)] >> (8 * (e & 3))) * f);
        *reinterpret_cast<g_u32x4*>(dst + 8 * j) = __builtin_bit_cast(u32x4, x);
    }
}

template <class T>
void launch_read8(const Read8Args& a, hipStream_t s)
{
    auto* kern = a.c.d == 64 ? kv_read8_kernel<T, 64> : a.c.d == 128 ? kv_read8_kernel<T, 128> : kv_read8_kernel<T, 256>;
    hipLaunchKernelGGL(kern, dim3((unsigned) (((int64_t) a.tokens * a.items + 255) / 256)), dim3(256), 0, s, a);
}

}  // namespace

extern "C" int exl3_rope_kv_write8(const void* q, int64_t q_ldt, int64_t q_ldh, const void* k, int64_t k_ldt, int64_t k_ldh,
                                   const void* v, int64_t v_ldt, int64_t v_ldh, const int64_t* positions, const int64_t* slots,
                                   void* q_out, const exl3_cache8* cache, const double* inv_freq, float mscale, int tokens, int q_heads,
                                   int rot_dim, int interleaved, int dtype, void* stream)
{
    Write8Args a{};
    if (!cache8_of(cache, a.c)) return EXL3_EINVAL;
    const int d = a.c.d, hkv = a.c.hkv;
    if (tokens < 0 || tokens > EXL3_PAGED_MAX_TOKENS || q_heads < hkv || q_heads > EXL3_PAGED_MAX_HEADS) return EXL3_EINVAL;
    if (rot_dim < 0 || rot_dim > d || (rot_dim & 1) || !paged_dtype(dtype)) return EXL3_EINVAL;
    if (tokens == 0) return EXL3_OK;
    if (!q || !k || !v || !positions || !slots || !q_out || (rot_dim && !inv_freq)) return EXL3_EINVAL;
    if (tokens == 1) q_ldt = k_ldt = v_ldt = 0;
    if (q_heads == 1) q_ldh = 0;
    if (hkv == 1) k_ldh = v_ldh = 0;
    if (!aligned16({q, k, v, q_out}) || !multiples_of_8({q_ldt, q_ldh, k_ldt, k_ldh, v_ldt, v_ldh})) return EXL3_EINVAL;
    a.q = (const uint16_t*) q, a.k = (const uint16_t*) k, a.v = (const uint16_t*) v;
    a.q_ldt = q_ldt, a.q_ldh = q_ldh, a.k_ldt = k_ldt, a.k_ldh = k_ldh, a.v_ldt = v_ldt, a.v_ldh = v_ldh;
    a.pos = positions, a.slots = slots, a.out = (uint16_t*) q_out, a.inv_freq = inv_freq, a.mscale = mscale;
    a.tokens = tokens, a.hq = q_heads, a.rot = rot_dim;
    // Few tokens: a workgroup for each row and head, so that all blocks of a batch of decodes are under way at once.  More: windows
    // of 16 rows, in which a prompt begins one or two blocks, and four workgroups that take them in turn; so many heads a
    // workgroup that about 1024 have work, since its angles serve all of them.  One row / 16 rows a window, us, 40 + 8 heads of 128, in a row: a prompt's
    // 128 tokens 9.5 / 6.9, 128 decodes 8.2 / 14.6; 512 tokens 14.7 / 8.3, 512 decodes 24.6 / 21.7; 32 decodes 5.8 / 14.  One, two,
    // four and eight heads of 8192 tokens: 79, 61, 53, 47; of 1000 tokens: 12.2, 11.6, 14.9, 22.8.
    const bool few = (int64_t) tokens * hkv <= 1024;
    a.rows = few ? 1 : C8_BLOCK;
    a.turns = few ? 1 : 4;
    const int windows = (tokens + a.rows - 1) / a.rows;
    a.heads = few ? 1 : (int) std::min((int64_t) hkv, ((int64_t) windows * hkv + 255) / 256);
    a.head_parts = (hkv + a.heads - 1) / a.heads;
    a.turn_wgs = windows * a.head_parts;
    a.kv_wgs = a.turn_wgs * a.turns;                    // with the q ones fewer than 2^32 threads for 2^22 tokens
    a.q_parts = tokens <= 512 ? std::min(64, (q_heads * (d / 8) + 2 * d - 1) / (2 * d)) : 1;
    const int layout = interleaved ? ROPE_PAIRS : rot_dim % 16 == 0 ? ROPE_HALF : ROPE_ANY, wgs = a.kv_wgs + tokens * a.q_parts;
    hipStream_t s = (hipStream_t) stream;
    if (dtype == EXL3_FP16) {
        if (d == 64) launch_write8<f16, 64>(a, layout, wgs, s);
        else if (d == 128) launch_write8<f16, 128>(a, layout, wgs, s);
        else launch_write8<f16, 256>(a, layout, wgs, s);
    } else {
        if (d == 64) launch_write8<__bf16, 64>(a, layout, wgs, s);
        else if (d == 128) launch_write8<__bf16, 128>(a, layout, wgs, s);
        else launch_write8<__bf16, 256>(a, layout, wgs, s);
    }
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}

extern "C" int exl3_kv_read8(const exl3_cache8* cache, const int64_t* slots, void* k_out, void* v_out, int tokens, int dtype, void* stream)
{
    Read8Args a{};
    if (!cache8_of(cache, a.c) || tokens < 0 || tokens > EXL3_PAGED_MAX_TOKENS || !paged_dtype(dtype)) return EXL3_EINVAL;
    if (tokens == 0) return EXL3_OK;
    if (!slots || !k_out || !v_out || !aligned16({k_out, v_out})) return EXL3_EINVAL;
    a.slots = slots, a.k = (uint16_t*) k_out, a.v = (uint16_t*) v_out, a.tokens = tokens;
    a.items = 2 * a.c.hkv * (a.c.d / 16);
    a.d_items = UDiv::of((uint32_t) a.items);
    if ((int64_t) tokens * a.items > UINT32_MAX - 256) return EXL3_EINVAL;         // a launch has fewer than 2^32 threads: 137 GB of values
    if (dtype == EXL3_FP16) launch_read8<f16>(a, (hipStream_t) stream);
    else launch_read8<__bf16>(a, (hipStream_t) stream);
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}
