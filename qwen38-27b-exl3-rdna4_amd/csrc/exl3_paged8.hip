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
    int rows, heads, head_parts;                        // a k/v workgroup's rows of the batch, its kv heads, workgroups over the heads
    int kv_wgs, q_parts;                                // k/v workgroups in front of the q ones; workgroups of a token's q
};

constexpr int MOST_KV_WGS = 1 << 21;                    // a launch has fewer than 2^32 threads

// The smallest exponent e of a scale with 127 * 2^e >= most, within the writer's.
__device__ __forceinline__ int exponent8(float most)
{
    const uint32_t b = (uint32_t) __float_as_int(most);
    const int e = (int) (b >> 23) - 127 - 6 + ((b & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);     // 127 / 64 = 1.984375: the mantissa 0x7E0000
    return min(max(e, C8_LEAST), C8_MOST);
}
__device__ __forceinline__ float power2(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float finite_abs(float x)
{
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;                      // NaN compares false
}

// codes of 8 values, whose quotient by the scale is exact (a power of two): rounded to even, infinities to +-127, NaN to 0
__device__ __forceinline__ u32x2 codes_of(const float (&x)[8], float inv)
{
    u32x2 r = u32x2{0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = fminf(fmaxf(rintf(x[i] * inv), -127.f), 127.f);
        const int q = x[i] == x[i] ? (int) y : 0;
        r[i >> 2] |= ((uint32_t) q & 0xFFu) << (8 * (i & 3));
    }
    return r;
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

// One launch, two kinds of workgroups.  The first kv_wgs quantise k and v: workgroup (w, p) takes the blocks whose first row
// in the batch is one of [rows w, rows (w + 1)), for the kv heads of part p.  A block's rows are consecutive in the batch, so one
// workgroup has all of a block's new tokens, and its scale needs no second pass and no other workgroup.  Its 256 threads
// hold the 16 rows of k and v of one head (8 elements a piece): new rows from the batch, the others' codes from the cache, requested
// at once whether the scale will grow or not, so a block takes one trip to memory.  The others rotate q.
template <class T, int D, int LAYOUT>
__global__ void __launch_bounds__(256) rope_kv_write8_kernel(Write8Args a)
{
    constexpr int PIECES = D / 8, KIND = C8_BLOCK * PIECES, N = 2 * KIND / 256;      // pieces of a row, of k or v; a thread's
    __shared__ float2 cs[C8_BLOCK][D / 2];
    __shared__ int src[C8_BLOCK];                       // the block's rows: their token in the batch, -1 none
    __shared__ float tops[2][4][2];                     // largest values of k and v of each wave; heads take turns
    using V8 = typename Elem<T>::x8;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    auto angles = [&](int row, int tok) __attribute__((always_inline)) {
        float s, c;
        for (int f = lane; f < a.rot / 2; f += 64) {
            sincospif(2.f * turn_fraction((double) a.pos[tok], a.inv_freq[f]), &s, &c);
            cs[row][f] = make_float2(c * a.mscale, s * a.mscale);
        }
    };

    if ((int) blockIdx.x >= a.kv_wgs) {
        const int b = (int) blockIdx.x - a.kv_wgs, tok = b / a.q_parts, part = b - tok * a.q_parts;
        for (int f = tid; f < a.rot / 2; f += 256) {
            float s, c;
            sincospif(2.f * turn_fraction((double) a.pos[tok], a.inv_freq[f]), &s, &c);
            cs[0][f] = make_float2(c * a.mscale, s * a.mscale);
        }
        __syncthreads();
        for (int i = part * 256 + tid; i < a.hq * PIECES; i += 256 * a.q_parts) {
            const int h = i / PIECES, c = 8 * (i % PIECES);
            const uint16_t* head = a.q + (int64_t) tok * a.q_ldt + (int64_t) h * a.q_ldh;
            const u32x4 x = *reinterpret_cast<gc_u32x4*>(as_global(head) + c);
            *reinterpret_cast<g_u32x4*>(as_global(a.out) + ((int64_t) tok * a.hq + h) * D + c) = rotated8<T, LAYOUT>(x, head, c, a.rot, cs[0]);
        }
        return;
    }

    const int w = (int) blockIdx.x / a.head_parts, h0 = ((int) blockIdx.x - w * a.head_parts) * a.heads, h1 = min(h0 + a.heads, a.c.hkv);
    const int row0 = w * a.rows;
    const int64_t cache_slots = (int64_t) a.c.pages * a.c.page;
    auto block_of = [&](int t) __attribute__((always_inline)) {                      // -1: a row of the batch that goes nowhere
        if (t < 0 || t >= a.tokens) return -1;
        const int64_t s = a.slots[t];
        return s >= 0 && s < cache_slots ? (int) (s / C8_BLOCK) : -1;
    };
    // lane l: row row0 + l; rows a block begins at (rows <= 64)
    const int mine = lane < a.rows ? block_of(row0 + lane) : -1, prior = block_of(row0 + lane - 1);
    uint64_t begins = __ballot(mine >= 0 && mine != prior);
    for (; begins; begins &= begins - 1) {
        const int first = row0 + __builtin_ctzll(begins), block = block_of(first);
        __syncthreads();                                // of the block before: src, cs and tops are free
        if (tid < C8_BLOCK) src[tid] = -1;
        __syncthreads();
        if (wave == 0) {
            // a slot that comes twice in a block's rows: the last one counts
            for (int t = first;; t += 64) {
                const uint64_t run = __ballot(block_of(t + lane) == block);
                const int n = ~run ? __builtin_ctzll(~run) : 64;
                if (lane < n) atomicMax(&src[a.slots[t + lane] % C8_BLOCK], t + lane);
                if (n < 64) break;
            }
        }
        __syncthreads();
        for (int r = wave; r < C8_BLOCK; r += 4)
            if (src[r] >= 0) angles(r, src[r]);
        __syncthreads();
        const bool anew = src[0] >= 0;
        const int page = (int) a.c.d_page.div((uint32_t) block * C8_BLOCK), in = block * C8_BLOCK - page * a.c.page;
        for (int h = h0; h < h1; ++h) {
            float* const ks = a.c.ks + (int64_t) page * a.c.ks_ldp + (int64_t) (in / C8_BLOCK) * a.c.ks_ldb + (int64_t) h * a.c.ks_ldh;
            float* const vs = a.c.vs + (int64_t) page * a.c.vs_ldp + (int64_t) (in / C8_BLOCK) * a.c.vs_ldb + (int64_t) h * a.c.vs_ldh;
            int8_t* const kc = a.c.k + (int64_t) page * a.c.k_ldp + (int64_t) in * a.c.k_ldt + (int64_t) h * a.c.k_ldh;
            int8_t* const vc = a.c.v + (int64_t) page * a.c.v_ldp + (int64_t) in * a.c.v_ldt + (int64_t) h * a.c.v_ldh;
            const float was[2] = {*as_global(ks), *as_global(vs)};
            u32x4 raw[N];
            u32x2 old[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int p = tid + 256 * j, r = p % KIND / PIECES, c = 8 * (p % PIECES), t = src[r];
                const bool is_v = p >= KIND;
                if (t >= 0) {
                    const uint16_t* head = is_v ? a.v + (int64_t) t * a.v_ldt + (int64_t) h * a.v_ldh : a.k + (int64_t) t * a.k_ldt + (int64_t) h * a.k_ldh;
                    raw[j] = *reinterpret_cast<gc_u32x4*>(as_global(head) + c);
                } else if (!anew) {
                    old[j] = *reinterpret_cast<gc_u32x2*>(as_global(is_v ? vc + (int64_t) r * a.c.v_ldt + c : kc + (int64_t) r * a.c.k_ldt + c));
                }
            }
            float x[N][8], top[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int p = tid + 256 * j, r = p % KIND / PIECES, c = 8 * (p % PIECES), t = src[r];
                const bool is_v = p >= KIND;
                if (t < 0) continue;
                const V8 e = __builtin_bit_cast(V8, raw[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = (float) e[i];
                if (!is_v) {
                    const uint16_t* head = a.k + (int64_t) t * a.k_ldt + (int64_t) h * a.k_ldh;
                    rotate8<T, LAYOUT>(e, head, c, a.rot, cs[r], [&](int i, float y) __attribute__((always_inline)) { x[j][i] = y; });
                }
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(x[j][i]));
                top[0] = fmaxf(top[0], is_v ? 0.f : m);
                top[1] = fmaxf(top[1], is_v ? m : 0.f);
            }
            const int turn = (h - h0) & 1;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) top[i] = fmaxf(top[i], __shfl_xor(top[i], m));
                if (lane == 0) tops[turn][wave][i] = top[i];
            }
            __syncthreads();
            float now[2];
            bool grown[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float m = tops[turn][0][i];
#pragma unroll
                for (int y = 1; y < 4; ++y) m = fmaxf(m, tops[turn][y][i]);
                const float need = power2(exponent8(m)), had = scale8(was[i]);
                grown[i] = anew || need > had;
                now[i] = grown[i] ? need : had;
            }
            if (tid < 2 && grown[tid]) *as_global(tid ? vs : ks) = now[tid];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int p = tid + 256 * j, r = p % KIND / PIECES, c = 8 * (p % PIECES), t = src[r];
                const bool is_v = p >= KIND;
                auto* const dst = reinterpret_cast<g_u32x2*>(as_global(is_v ? vc + (int64_t) r * a.c.v_ldt + c : kc + (int64_t) r * a.c.k_ldt + c));
                if (t >= 0) *dst = codes_of(x[j], 1.f / now[is_v]);
                else if (anew) *dst = u32x2{0u, 0u};
                else if (grown[is_v]) *dst = rounded_anew(old[j], scale8(was[is_v]) / now[is_v]);
            }
        }
    }
}

template <class T, int D>
void launch_write8(const Write8Args& a, int layout, int wgs, hipStream_t s)
{
    auto* kern = layout == ROPE_HALF ? rope_kv_write8_kernel<T, D, ROPE_HALF>
                 : layout == ROPE_PAIRS ? rope_kv_write8_kernel<T, D, ROPE_PAIRS> : rope_kv_write8_kernel<T, D, ROPE_ANY>;
    hipLaunchKernelGGL(kern, dim3((unsigned) wgs), dim3(256), 0, s, a);
}

struct Read8Args {
    Cache8 c;
    const int64_t* slots;
    uint16_t *k, *v;
    int tokens, rows;                                   // rows of the batch that a workgroup reads
};

// Tokens' k and v as fp16 or bf16 values: a thread turns 16 codes into 32 bytes.
template <class T, int D>
__global__ void __launch_bounds__(256) kv_read8_kernel(Read8Args a)
{
    constexpr int PIECES = D / 16;
    using V8 = typename Elem<T>::x8;
    const int items = 2 * a.c.hkv * PIECES, t0 = (int) blockIdx.x * a.rows, t1 = min(t0 + a.rows, a.tokens);
    const int64_t cache_slots = (int64_t) a.c.pages * a.c.page;
    for (int t = t0; t < t1; ++t) {
        const int64_t slot = a.slots[t];
        const bool held = slot >= 0 && slot < cache_slots;
        const int page = held ? (int) a.c.d_page.div((uint32_t) slot) : 0, in = held ? (int) slot - page * a.c.page : 0;
        for (int i = threadIdx.x; i < items; i += 256) {
            const int p = i % PIECES, y = i / PIECES;
            const bool is_v = y >= a.c.hkv;
            const int h = is_v ? y - a.c.hkv : y;
            u32x4 codes = u32x4{0u, 0u, 0u, 0u};
            float s = 1.f;
            if (held) {
                const int8_t* src = is_v ? a.c.v + page * a.c.v_ldp + in * a.c.v_ldt + h * a.c.v_ldh : a.c.k + page * a.c.k_ldp + in * a.c.k_ldt + h * a.c.k_ldh;
                codes = *reinterpret_cast<gc_u32x4*>(as_global(src) + 16 * p);
                s = scale8(*as_global(is_v ? a.c.vs + page * a.c.vs_ldp + in / C8_BLOCK * a.c.vs_ldb + h * a.c.vs_ldh
                                           : a.c.ks + page * a.c.ks_ldp + in / C8_BLOCK * a.c.ks_ldb + h * a.c.ks_ldh));
            }
            auto* const dst = as_global(is_v ? a.v : a.k) + ((int64_t) t * a.c.hkv + h) * D + 16 * p;
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                V8 x;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (T) ((float) (int8_t) (uint8_t) (codes[2 * z + (e >> 2)] >> (8 * (e & 3))) * s);
                *reinterpret_cast<g_u32x4*>(dst + 8 * z) = __builtin_bit_cast(u32x4, x);
            }
        }
    }
}

template <class T>
void launch_read8(const Read8Args& a, hipStream_t s)
{
    auto* kern = a.c.d == 64 ? kv_read8_kernel<T, 64> : a.c.d == 128 ? kv_read8_kernel<T, 128> : kv_read8_kernel<T, 256>;
    hipLaunchKernelGGL(kern, dim3((unsigned) ((a.tokens + a.rows - 1) / a.rows)), dim3(256), 0, s, a);
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
    const bool few = tokens <= 512;
    a.rows = few ? 1 : C8_BLOCK;
    const int windows = (tokens + a.rows - 1) / a.rows;
    a.heads = (int) (((int64_t) windows * hkv + MOST_KV_WGS - 1) / MOST_KV_WGS);
    a.head_parts = (hkv + a.heads - 1) / a.heads;
    a.kv_wgs = windows * a.head_parts;
    a.q_parts = few ? std::min(64, (q_heads * (d / 8) + 255) / 256) : 1;
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
    a.rows = 1;
    if (dtype == EXL3_FP16) launch_read8<f16>(a, (hipStream_t) stream);
    else launch_read8<__bf16>(a, (hipStream_t) stream);
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}
