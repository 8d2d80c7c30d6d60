// exl3_attn.h -- what the paged-cache kernels share: element types, argument checks, limits.
#pragma once
#include "exl3_device.h"
#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace exl3 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <class T> struct Elem;
template <> struct Elem<f16> { typedef f16x8 x8; };
template <> struct Elem<__bf16> { typedef bf16x8 x8; };

enum { ROPE_HALF, ROPE_PAIRS, ROPE_ANY };

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

__device__ __forceinline__ uint64_t uniform(uint64_t x)
{
    return (uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) x) |
           (uint64_t) (uint32_t) __builtin_amdgcn_readfirstlane((int) (uint32_t) (x >> 32)) << 32;
}

typedef __attribute__((address_space(1))) const char gc_char;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 0xFFFF in each half of x that is an infinity or NaN: adding one to an exponent of all ones reaches the sign's place
// (integer arithmetic: 64 compares at once would take the scalar registers of 64 results)
template <class T>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x)
{
    constexpr uint32_t ONE = std::is_same_v<T, f16> ? 0x04000400u : 0x00800080u;
    const uint32_t n = ((x & 0x7FFF7FFFu) + ONE) & 0x80008000u;
    return n | (n - (n >> 15));
}

template <class T> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<f16>(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<__bf16>(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// max / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float max_quads(float x)
{
    float lo, hi;
    halves_x(x, lo, hi);
    x = fmaxf(lo, hi);
    const auto w = __builtin_amdgcn_permlane16_swap((uint32_t) __float_as_int(x), (uint32_t) __float_as_int(x), false, false);
    return fmaxf(__int_as_float((int) w[0]), __int_as_float((int) w[1]));
}
__device__ __forceinline__ float sum_quads(float x)
{
    float lo, hi;
    halves_x(x, lo, hi);
    x = lo + hi;
    const auto w = __builtin_amdgcn_permlane16_swap((uint32_t) __float_as_int(x), (uint32_t) __float_as_int(x), false, false);
    return __int_as_float((int) w[0]) + __int_as_float((int) w[1]);
}

constexpr float LOWEST = -3.0e38f;                      // a running maximum that no key has raised

__device__ __forceinline__ u32x4 flipped(u32x4 x, uint32_t f) { return u32x4{x[0] ^ f, x[1] ^ f, x[2] ^ f, x[3] ^ f}; }

// out = sum / l of four columns; a row that saw nothing (l = 0) is 0
template <class T>
__device__ __forceinline__ void store_out(__attribute__((address_space(1))) uint16_t* at, f32x4 sum, float l)
{
    typedef T T4 __attribute__((ext_vector_type(4)));
    const float r = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<__attribute__((address_space(1))) T4*>(at) = T4{(T) (sum[0] * r), (T) (sum[1] * r), (T) (sum[2] * r), (T) (sum[3] * r)};
}

// ---- attention: one launch's arguments, and the work that its workgroups share ------------------------------
struct AttnArgs {
    const uint16_t *q, *k, *v;
    int64_t q_ldt, q_ldh, k_ldp, k_ldt, k_ldh, v_ldp, v_ldt, v_ldh, o_ldt, o_ldh, ld_table;
    const int *table, *cu_q, *seq;
    uint16_t* out;
    int tokens, requests, group, hkv, pages, page, window;
    int cap;                                            // positions that a row of the table holds
    float scale;                                        // its size times log2(e): above 0
    uint32_t flip;                                      // sign bits of two halves of q: 0 but for a negative scale
    UDiv d_page, d_group;
    uint32_t* counters;                                 // one per workgroup, zero between calls
    float* part;                                        // partial tiles: two a workgroup
};

// a partial tile, floats: rows x D outputs, then (maximum, sum) a row; two for each workgroup of a grid
constexpr int attn_slot(int rows, int d) { return rows * (d + 2); }
constexpr int ATTN_COUNTERS = EXL3_ATTN_COUNTER_BYTES / 4;                      // the largest grid
constexpr size_t ATTN_PART_BYTES = (size_t) 2 * 512 * attn_slot(128, 130) * 4;  // the largest grid times slot (all kernels assert it)

// A request's new rows for one kv head, (token, head of the group) in token order, are cut into tiles of `rows`; a tile
// reads the keys that any of its rows sees, in steps of KEYS.  A launch's work is the steps of every (kv head,
// request, tile) in that order, and each workgroup takes an equal, contiguous share of it (at least `least` steps), so
// the launch is balanced for any mix of lengths, none of which the host knows.
struct AttnTile {
    int first, last;                                    // new tokens of its first and last row
    int lo, hi;                                         // keys [lo, hi) that any row sees
    int step0, steps;                                   // its steps; one (of no key) where no row sees any
};

template <int ROWS, int KEYS, int GRID>
struct AttnWork {
    const AttnArgs& a;
    int r, t, h;                                        // request, tile, kv head
    int tok0, n, pos0;                                  // the request's first row of q, new tokens, first position
    AttnTile tile;

    __device__ __forceinline__ AttnWork(const AttnArgs& args) : a(args) {}

    __device__ __forceinline__ void request(int req)
    {
        r = req;
        tok0 = min(max(a.cu_q[r], 0), a.tokens);
        const int all = max(a.cu_q[r + 1] - tok0, 0);
        n = min(all, a.tokens - tok0);
        pos0 = max(a.seq[r], 0) - all;
    }
    __device__ __forceinline__ int tiles() const { return (n * a.group + ROWS - 1) / ROWS; }
    __device__ __forceinline__ AttnTile tile_of(int i) const
    {
        AttnTile x;
        x.first = (int) a.d_group.div((uint32_t) (i * ROWS));
        x.last = (int) a.d_group.div((uint32_t) (min((i + 1) * ROWS, n * a.group) - 1));
        x.hi = max(0, min(pos0 + x.last + 1, a.cap));
        x.lo = a.window ? min(max(pos0 + x.first + 1 - a.window, 0), x.hi) : 0;
        x.step0 = x.lo / KEYS;
        x.steps = max(1, (x.hi + KEYS - 1) / KEYS - x.step0);
        return x;
    }

    // Every thread sums the steps of its range of requests; a scan gives the total and finds the tile of this
    // workgroup's first step.  lds: THREADS / 64 + 4 64-bit words.  False: this workgroup has no share.  off: the first
    // step's place in its tile; left: the steps of the share (64 bits: long contexts times heads pass 2^32); per: those of
    // a whole share, as far as a tile's steps can tell (below 2^30).  All but the sums is uniform, in scalar registers.
    template <int THREADS>
    __device__ __forceinline__ bool find(int wg, int least, uint64_t* lds, int& off, int64_t& left, uint32_t& per)
    {
        // few requests: several threads each, a range of its tiles a thread (2^share_log of them)
        const int tid = threadIdx.x, each = (a.requests + THREADS - 1) / THREADS;
        int share_log = 0;
        while ((a.requests << (share_log + 1)) <= THREADS && share_log < 8) ++share_log;
        const int r0 = min(share_log ? tid >> share_log : tid * each, a.requests), r1 = min(r0 + max(each, 1), a.requests);
        auto tiles_from = [&](int m, int& j, int& end) __attribute__((always_inline)) {
            const int c = (m + (1 << share_log) - 1) >> share_log;
            j = min((tid & ((1 << share_log) - 1)) * c, m);
            end = min(j + c, m);
        };
        uint64_t sum = 0;
        for (int i = r0; i < r1; ++i) {
            request(i);
            int j, end;
            for (tiles_from(tiles(), j, end); j < end; ++j) sum += (uint64_t) tile_of(j).steps;
        }
        uint64_t upto = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t x = __shfl_up(upto, d);
            if ((tid & 63) >= d) upto += x;
        }
        if ((tid & 63) == 63) lds[tid >> 6] = upto;
        __syncthreads();
        uint64_t sums = 0;
#pragma unroll 4
        for (int i = 0; i < THREADS / 64; ++i) {
            if (i < (tid >> 6)) upto += lds[i];
            sums += lds[i];
        }
        const uint64_t total = uniform(sums), all = total * (uint64_t) a.hkv;
        const uint64_t share = max((all + GRID - 1) / GRID, (uint64_t) least);
        uint64_t u = (uint64_t) wg * share;
        if (u >= all) return false;
        per = (uint32_t) min(share, (uint64_t) 1 << 30);
        left = (int64_t) min(share, all - u);
        h = 0;
        for (; u >= total; u -= total) ++h;
        if (u >= upto - sum && u < upto) {
            uint64_t x = u - (upto - sum);
            for (int i = r0;; ++i) {
                request(i);
                int j, end;
                for (tiles_from(tiles(), j, end); j < end; ++j) {
                    const uint64_t steps = (uint64_t) tile_of(j).steps;
                    if (x < steps) break;
                    x -= steps;
                }
                if (j == end) continue;
                int* o = reinterpret_cast<int*>(lds + THREADS / 64);
                o[0] = i;
                o[1] = j;
                o[2] = (int) x;
                o[3] = tok0;
                o[4] = n;
                o[5] = pos0;
                break;
            }
        }
        __syncthreads();
        const int* o = reinterpret_cast<const int*>(lds + THREADS / 64);
        r = o[0];
        t = o[1];
        off = __builtin_amdgcn_readfirstlane(o[2]);
        tok0 = o[3];
        n = o[4];
        pos0 = o[5];
        return true;
    }
    // all of it into scalar registers (the compiler keeps values that went through a loop or LDS in vector ones)
    __device__ __forceinline__ void settle()
    {
        r = __builtin_amdgcn_readfirstlane(r);
        t = __builtin_amdgcn_readfirstlane(t);
        h = __builtin_amdgcn_readfirstlane(h);
        tok0 = __builtin_amdgcn_readfirstlane(tok0);
        n = __builtin_amdgcn_readfirstlane(n);
        pos0 = __builtin_amdgcn_readfirstlane(pos0);
        tile = tile_of(t);
    }
    // The tile after this one (there is one).  Requests without new tokens are passed one by one, 0.1 us each: eight decodes over 4000
    // tokens (40 heads over 8 of 128) take 29 us, as the first of 256 slots 54, spread over 256 slots 32.
    __device__ __forceinline__ void next()
    {
        if (++t < tiles()) return;
        t = 0;
        int i = r;
        do {
            if (++i == a.requests) {
                i = 0;
                ++h;
            }
            request(i);
        } while (__builtin_amdgcn_readfirstlane(n) == 0);
    }
};

// A split tile's parts, summed in the order of their workgroups: part c of workgroup c lies in slot 2 c, the first
// one's in 2 c + 1; B of them are in flight.
template <class T, int D, int ROWS, int THREADS, int SLOT, int B, class At>
__device__ __forceinline__ void join_parts(__amdgpu_buffer_rsrc_t prs, int first, int last, int rows, At&& out_at)
{
    auto slot = [&](int c) __attribute__((always_inline)) { return (uint32_t) (2 * c + (c == first ? 1 : 0)) * (uint32_t) SLOT; };
    for (int z = threadIdx.x; z < rows * (D / 4); z += THREADS) {
        const int x = z / (D / 4), col = 4 * (z % (D / 4));
        const uint32_t at = (uint32_t) (x * D + col), ml = (uint32_t) (ROWS * D + 2 * x);
        float m = LOWEST, l = 0.f;
        f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int c0 = first; c0 <= last; c0 += B) {
            u32x2 mls[B];
            f32x4 v[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const uint32_t s = slot(min(c0 + i, last));
                mls[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(prs, (s + ml) * 4u, 0, SC1));
                v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, (s + at) * 4u, 0, SC1));
            }
            float top = m;
#pragma unroll
            for (int i = 0; i < B; ++i) top = fmaxf(top, __int_as_float((int) mls[i][0]));
            const float c = exp2_fast(m - top);
            l *= c;
            sum *= c;
            m = top;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const float f = c0 + i <= last ? exp2_fast(__int_as_float((int) mls[i][0]) - m) : 0.f;
                l += f * __int_as_float((int) mls[i][1]);
                sum += v[i] * f;
            }
        }
        store_out<T>(out_at(x) + col, sum, l);
    }
}

// many rows a request (exl3_attn_prefill.hip)
void launch_attn_prefill(const AttnArgs& a, int dtype, int head_dim, hipStream_t s);

}  // namespace exl3
