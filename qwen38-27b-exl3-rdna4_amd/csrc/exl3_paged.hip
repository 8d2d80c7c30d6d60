// exl3_paged.hip -- a decoder step's bookkeeping over a paged key/value cache (exl3_batch_plan), and the
// rotary embedding of q and k with the cache's write (exl3_rope_kv_write).
#include "exl3_device.h"
#include "exl3_attn.h"

using namespace exl3;

namespace {

constexpr int PLAN_TOKENS = 2048;                      // tokens of one request that a workgroup writes

// Counts come from the caller's GPU memory, where nothing has checked them: sums stop at 2^31 - 1 instead of passing it, in
// any order alike, so no index formed from them is negative.
__device__ __forceinline__ int add_count(int a, int b) { return (int) min((uint32_t) a + (uint32_t) b, (uint32_t) INT32_MAX); }

// sum over the workgroup's 256 threads of two counts
__device__ __forceinline__ int2 block_sum2(int a, int b, int* lds)
{
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        a = add_count(a, __shfl_xor(a, m));
        b = add_count(b, __shfl_xor(b, m));
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        lds[2 * wave] = a;
        lds[2 * wave + 1] = b;
    }
    __syncthreads();
    return make_int2(add_count(add_count(lds[0], lds[2]), add_count(lds[4], lds[6])), add_count(add_count(lds[1], lds[3]), add_count(lds[5], lds[7])));
}

struct PlanArgs {
    const int* ctx;
    const int* add;
    int* table;
    int64_t ld_table;
    const int* free_pages;
    const int* free_count;
    int* cu_q;
    int* seq;
    int64_t* pos;
    int64_t* slots;
    int* left;
    int requests, cols, n_free, page, tokens;
    UDiv d_page;
};

// Request r's first token and first new page are sums over the requests before it.  Workgroup (r, c) forms
// both sums by itself from the lengths (r / 256 loads a thread, all in cache after the first workgroups),
// so no workgroup waits for another and one launch does it all; then it writes the request's tokens
// [2048 c, 2048 (c + 1)) and, for c = 0, its new table entries.  Row r = requests writes the tokens past the
// last request.  A step is bound by the latency of one launch and three dependent accesses (lengths, page, stores): 3.3 us
// for 48 decodes, 4.7 for 300 requests of 10419 tokens.
__global__ void __launch_bounds__(256) batch_plan_kernel(PlanArgs a)
{
    __shared__ int lds[8];
    const int r = blockIdx.x, t0 = (int) blockIdx.y * PLAN_TOKENS;
    const bool tail = r == a.requests;
    const int ctx = tail ? 0 : max(a.ctx[r], 0);
    int add = tail ? 0 : min(max(a.add[r], 0), INT32_MAX - ctx);
    if (!tail && t0 > 0 && t0 >= add) return;
    const int count = min(a.free_count[0], a.n_free);
    auto pages = [&](int tokens) __attribute__((always_inline)) {   // columns of the table that `tokens` fill
        return min((int) a.d_page.div((uint32_t) tokens + (uint32_t) (a.page - 1)), a.cols);
    };
    int before = 0, taken = 0;
    for (int s = threadIdx.x; s < r; s += 256) {
        const int c = max(a.ctx[s], 0), n = min(max(a.add[s], 0), INT32_MAX - c);
        before = add_count(before, n);
        taken = add_count(taken, n ? pages(c + n) - pages(c) : 0);
    }
    const int2 sums = block_sum2(before, taken, lds);
    const int first = sums.x, had = pages(ctx), need = add ? pages(ctx + add) - had : 0, top = max(count, 0) - 1 - sums.y;
    if (t0 == 0) {
        if (threadIdx.x == 0) {
            a.cu_q[r] = first;
            if (tail) a.left[0] = (int) max((int64_t) count - sums.y, (int64_t) INT32_MIN);
            else a.seq[r] = ctx + add;
        }
        for (int j = threadIdx.x; j < need; j += 256)
            a.table[(int64_t) r * a.ld_table + had + j] = j <= top ? a.free_pages[top - j] : -1;
    }
    if (tail) {
        for (int i = t0 + (int) threadIdx.x; i < min(a.tokens - first, t0 + PLAN_TOKENS); i += 256) {
            a.pos[first + i] = 0;
            a.slots[first + i] = -1;
        }
        return;
    }
    add = min(add, t0 + PLAN_TOKENS);
    for (int i = t0 + (int) threadIdx.x; i < add; i += 256) {
        if (i >= a.tokens - first) break;
        const int t = first + i, p = ctx + i, col = (int) a.d_page.div((uint32_t) p);
        int page = -1;
        if (col < had) page = a.table[(int64_t) r * a.ld_table + col];
        else if (col < a.cols && col - had <= top) page = a.free_pages[top - (col - had)];
        a.pos[t] = p;
        a.slots[t] = page < 0 ? -1 : (int64_t) page * a.page + (p - col * a.page);
    }
}

// position * freq / (2 pi) less its whole turns.  1 / (2 pi) in two doubles, and each product's rounding error by
// fma: what is lost is below 2^-100 of the angle, so the fraction is good to 32 bits for any position below 2^53.
__device__ __forceinline__ float turn_fraction(double position, double freq)
{
#pragma clang fp contract(off)                          // a product that a subtraction absorbs has no error to add
    constexpr double C_HI = 0x1.45f306dc9c883p-3, C_LO = -0x1.6b01ec5417056p-57;
    const double g = freq * C_HI, g_err = fma(freq, C_HI, -g) + freq * C_LO;
    const double turns = position * g, err = fma(position, g, -turns) + position * g_err;
    const double x = (turns - floor(turns)) + err;
    return (float) (x - floor(x));
}

struct RopeArgs {
    const uint16_t *q, *k, *v;
    int64_t q_ldt, q_ldh, k_ldt, k_ldh, v_ldt, v_ldh;
    const int64_t *pos, *slots;
    uint16_t *out, *kc, *vc;
    int64_t kc_ldp, kc_ldt, kc_ldh, vc_ldp, vc_ldt, vc_ldh;
    const double* inv_freq;
    float mscale;
    int tokens, hq, hkv, rot, page;
    int64_t cache_slots;
    int items;                                          // 8-element pieces of a token: (hq + 2 hkv) D / 8
    UDiv d_page;
};

// 8 elements of a head from column c on, rotated.  x: those elements; other: the elements they pair with (half
// layout); cs: the token's (cos, sin) per frequency.
template <class T, int LAYOUT>
__device__ __forceinline__ u32x4 rotate8(u32x4 xb, const uint16_t* head, int c, int rot, const float2* cs)
{
    using V = typename Elem<T>::x8;
    const V x = __builtin_bit_cast(V, xb);
    V y = x;
    const int half = rot / 2;
    if constexpr (LAYOUT == ROPE_HALF) {               // half % 8 == 0: the whole piece pairs with one piece
        if (c < rot) {
            const bool low = c < half;
            const V o = __builtin_bit_cast(V, *reinterpret_cast<gc_u32x4*>(as_global(head) + (low ? c + half : c - half)));
            const float2* f = cs + (low ? c : c - half);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (T) ((float) x[i] * f[i].x + (low ? -(float) o[i] : (float) o[i]) * f[i].y);
        }
    } else if constexpr (LAYOUT == ROPE_PAIRS) {       // pairs side by side
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if (c + i < rot) {
                const float2 f = cs[(c + i) / 2];
                const float u = (float) x[i], w = (float) x[i + 1];
                y[i] = (T) (u * f.x - w * f.y);
                y[i + 1] = (T) (w * f.x + u * f.y);
            }
    } else {                                           // half layout with an odd boundary: element by element
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = c + i;
            if (e < rot) {
                const bool low = e < half;
                const float o = (float) __builtin_bit_cast(T, (uint16_t) *(as_global(head) + (low ? e + half : e - half)));
                const float2 f = cs[low ? e : e - half];
                y[i] = (T) ((float) x[i] * f.x + (low ? -o : o) * f.y);
            }
        }
    }
    return __builtin_bit_cast(u32x4, y);
}

// theta = position x frequency is reduced to a fraction of a turn before it is rounded to 32 bits, so a position of a
// million turns as exactly as position 0 (32-bit angles are 0.06 off there).  A workgroup forms the cosines and sines of
// its token once, in LDS, and uses them for every head; k goes straight to its cache slot.  Bound by memory: 8192 tokens
// of 40 + 8 heads of 128 (235 MB) in 47 us, 5.0 TB/s, where calls write two outputs in turn, 40 us where all write the same
// one (a large copy: 4.6 TB/s); 32 tokens in 2.6 to 3.1.
template <class T, int D, int LAYOUT>
__global__ void __launch_bounds__(256) rope_kv_write_kernel(RopeArgs a)
{
    __shared__ float2 cs[D / 2];
    const int64_t tok = blockIdx.x;
    for (int f = threadIdx.x; f < a.rot / 2; f += 256) {
        float s, c;
        sincospif(2.f * turn_fraction((double) a.pos[tok], a.inv_freq[f]), &s, &c);
        cs[f] = make_float2(c * a.mscale, s * a.mscale);
    }
    __syncthreads();
    constexpr int PIECES = D / 8;
    for (int i = (int) blockIdx.y * 256 + (int) threadIdx.x; i < a.items; i += 256 * (int) gridDim.y) {
        int h = i / PIECES;
        const int c = 8 * (i % PIECES);
        if (h < a.hq) {
            const uint16_t* head = a.q + tok * a.q_ldt + h * a.q_ldh;
            const u32x4 x = *reinterpret_cast<gc_u32x4*>(as_global(head) + c);
            *reinterpret_cast<g_u32x4*>(as_global(a.out) + (tok * a.hq + h) * D + c) = rotate8<T, LAYOUT>(x, head, c, a.rot, cs);
            continue;
        }
        const int64_t slot = a.slots[tok];
        if (slot < 0 || slot >= a.cache_slots) continue;
        const int64_t page = a.d_page.div((uint32_t) slot), off = slot - page * a.page;
        h -= a.hq;
        if (h < a.hkv) {
            const uint16_t* head = a.k + tok * a.k_ldt + h * a.k_ldh;
            const u32x4 x = *reinterpret_cast<gc_u32x4*>(as_global(head) + c);
            *reinterpret_cast<g_u32x4*>(as_global(a.kc) + page * a.kc_ldp + off * a.kc_ldt + h * a.kc_ldh + c) =
                rotate8<T, LAYOUT>(x, head, c, a.rot, cs);
        } else {
            h -= a.hkv;
            const u32x4 x = *reinterpret_cast<gc_u32x4*>(as_global(a.v) + tok * a.v_ldt + h * a.v_ldh + c);
            *reinterpret_cast<g_u32x4*>(as_global(a.vc) + page * a.vc_ldp + off * a.vc_ldt + h * a.vc_ldh + c) = x;
        }
    }
}

template <class T, int D>
void launch_rope(const RopeArgs& a, int layout, dim3 grid, hipStream_t s)
{
    auto* kern = layout == ROPE_HALF ? rope_kv_write_kernel<T, D, ROPE_HALF>
                 : layout == ROPE_PAIRS ? rope_kv_write_kernel<T, D, ROPE_PAIRS> : rope_kv_write_kernel<T, D, ROPE_ANY>;
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, a);
}

}  // namespace

extern "C" int exl3_batch_plan(const int* ctx_lens, const int* new_lens, int* block_table, int64_t ld_table, int table_cols,
                               const int* free_pages, int n_free, const int* free_count, int* cu_q, int* seq_lens,
                               int64_t* positions, int64_t* slots, int* free_left, int requests, int page_size, int tokens,
                               void* stream)
{
    if (requests < 0 || tokens < 0 || table_cols < 0 || n_free < 0 || page_size < 1 || page_size > EXL3_PAGED_MAX_PAGE) return EXL3_EINVAL;
    if (requests > EXL3_PAGED_MAX_REQUESTS || tokens > EXL3_PAGED_MAX_TOKENS || ld_table < table_cols) return EXL3_EINVAL;
    if (!free_count || !cu_q || !free_left || (n_free && !free_pages)) return EXL3_EINVAL;
    if (requests && (!ctx_lens || !new_lens || !seq_lens || (table_cols && !block_table))) return EXL3_EINVAL;
    if (tokens && (!positions || !slots)) return EXL3_EINVAL;
    PlanArgs a{ctx_lens, new_lens, block_table, ld_table, free_pages, free_count, cu_q, seq_lens, positions, slots, free_left,
               requests, table_cols, n_free, page_size, tokens, UDiv::of((uint32_t) page_size)};
    const dim3 grid((unsigned) requests + 1u, (unsigned) std::max(1, (tokens + PLAN_TOKENS - 1) / PLAN_TOKENS));
    hipLaunchKernelGGL(batch_plan_kernel, grid, dim3(256), 0, (hipStream_t) stream, a);
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}

extern "C" int exl3_rope_kv_write(const void* q, int64_t q_ldt, int64_t q_ldh, const void* k, int64_t k_ldt, int64_t k_ldh,
                                  const void* v, int64_t v_ldt, int64_t v_ldh, const int64_t* positions, const int64_t* slots,
                                  void* q_out, void* k_cache, int64_t kc_ldp, int64_t kc_ldt, int64_t kc_ldh, void* v_cache,
                                  int64_t vc_ldp, int64_t vc_ldt, int64_t vc_ldh, const double* inv_freq, float mscale, int tokens,
                                  int q_heads, int kv_heads, int head_dim, int rot_dim, int interleaved, int pages, int page_size,
                                  int dtype, void* stream)
{
    if (tokens < 0 || tokens > EXL3_PAGED_MAX_TOKENS || q_heads < 1 || kv_heads < 1 || q_heads > EXL3_PAGED_MAX_HEADS || kv_heads > q_heads)
        return EXL3_EINVAL;
    if (!paged_head_dim(head_dim) || rot_dim < 0 || rot_dim > head_dim || (rot_dim & 1) || !paged_dtype(dtype)) return EXL3_EINVAL;
    if (pages < 0 || page_size < 1 || page_size > EXL3_PAGED_MAX_PAGE || (int64_t) pages * page_size > INT32_MAX) return EXL3_EINVAL;
    if (tokens == 0) return EXL3_OK;
    if (!q || !k || !v || !positions || !slots || !q_out || !k_cache || !v_cache || (rot_dim && !inv_freq)) return EXL3_EINVAL;
    // a stride that addresses nothing may be anything
    if (tokens == 1) q_ldt = k_ldt = v_ldt = 0;
    if (q_heads == 1) q_ldh = 0;
    if (kv_heads == 1) k_ldh = v_ldh = kc_ldh = vc_ldh = 0;
    if (pages <= 1) kc_ldp = vc_ldp = 0;
    if (page_size == 1) kc_ldt = vc_ldt = 0;
    if (!aligned16({q, k, v, q_out, k_cache, v_cache}) ||
        !multiples_of_8({q_ldt, q_ldh, k_ldt, k_ldh, v_ldt, v_ldh, kc_ldp, kc_ldt, kc_ldh, vc_ldp, vc_ldt, vc_ldh}))
        return EXL3_EINVAL;
    RopeArgs a{(const uint16_t*) q, (const uint16_t*) k, (const uint16_t*) v, q_ldt, q_ldh, k_ldt, k_ldh, v_ldt, v_ldh, positions, slots,
               (uint16_t*) q_out, (uint16_t*) k_cache, (uint16_t*) v_cache, kc_ldp, kc_ldt, kc_ldh, vc_ldp, vc_ldt, vc_ldh, inv_freq, mscale,
               tokens, q_heads, kv_heads, rot_dim, page_size, (int64_t) pages * page_size, (q_heads + 2 * kv_heads) * (head_dim / 8),
               UDiv::of((uint32_t) page_size)};
    // a vector piece of 8 pairs with one other piece where half the rotated part is a multiple of 8
    const int layout = interleaved ? ROPE_PAIRS : rot_dim % 16 == 0 ? ROPE_HALF : ROPE_ANY;
    // Few tokens: a token's pieces over several workgroups, so that all heads' loads go out together; many fill the GPU
    // without, and forming the angles once is cheaper.  Several workgroups a token / one, us, in a graph of calls that write one
    // output, 40 + 8 heads of 128: 32 tokens 2.6 / 3.3, 256 3.4 / 3.8, 512 4.8 / 4.7, 768 6.2 / 6.2, 2048 11.8 / 10.9,
    // 8192 50 / 38; 24 + 4 of 256, a quarter rotated: 2.8 / 4.0, 3.5 / 4.1, 4.7 / 5.0, 6.4 / 6.3, 12.8 / 11.9, 56 / 46.
    const dim3 grid((unsigned) tokens, tokens <= 512 ? (unsigned) std::min(64, (a.items + 255) / 256) : 1u);
    hipStream_t s = (hipStream_t) stream;
    if (dtype == EXL3_FP16) {
        if (head_dim == 64) launch_rope<f16, 64>(a, layout, grid, s);
        else if (head_dim == 128) launch_rope<f16, 128>(a, layout, grid, s);
        else launch_rope<f16, 256>(a, layout, grid, s);
    } else {
        if (head_dim == 64) launch_rope<__bf16, 64>(a, layout, grid, s);
        else if (head_dim == 128) launch_rope<__bf16, 128>(a, layout, grid, s);
        else launch_rope<__bf16, 256>(a, layout, grid, s);
    }
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}
