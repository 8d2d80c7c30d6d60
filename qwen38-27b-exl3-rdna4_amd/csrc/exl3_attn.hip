// exl3_attn.hip -- causal attention of each request's new tokens over its paged key/value cache.
#include "exl3_attn.h"

using namespace exl3;

namespace {

struct AttnArgs {
    const uint16_t *q, *k, *v;
    int64_t q_ldt, q_ldh, k_ldp, k_ldt, k_ldh, v_ldp, v_ldt, v_ldh, o_ldt, o_ldh, ld_table;
    const int *table, *cu_q, *seq;
    uint16_t* out;
    int tokens, requests, hq, hkv, pages, cols, page, window;
    float scale;
    UDiv d_page, d_group;
};

// One wave per (token, query head): a lane scores one key of 64, the running maximum and sum follow, then every lane
// sums its D / 64 columns over the 64 keys.
template <class T, int D>
__global__ void __launch_bounds__(64) attn_simple_kernel(AttnArgs a)
{
    constexpr int E = D / 64;
    __shared__ float qs[D];
    __shared__ float ps[64];
    __shared__ int slots[64];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, hk = (int) a.d_group.div((uint32_t) h);
    for (int e = lane; e < D; e += 64) qs[e] = (float) __builtin_bit_cast(T, a.q[(int64_t) t * a.q_ldt + h * a.q_ldh + e]) * a.scale;
    // the last request that starts at or before the token
    int lo = 0, hi = a.requests;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.cu_q[mid] <= t) lo = mid;
        else hi = mid;
    }
    int first = 0, end = 0;
    if (a.requests > 0 && t >= a.cu_q[lo] && t < a.cu_q[lo + 1]) {
        const int n = a.cu_q[lo + 1] - a.cu_q[lo], p = a.seq[lo] - n + (t - a.cu_q[lo]);
        end = min(p + 1, a.cols * a.page);
        if (a.window > 0) first = max(0, p + 1 - a.window);
    }
    float m = -INFINITY, l = 0.f, acc[E] = {};
    for (int j0 = first; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        float s = -INFINITY;
        int slot = -1;
        if (j < end) {
            const int col = (int) a.d_page.div((uint32_t) j), page = a.table[(int64_t) lo * a.ld_table + col];
            if ((unsigned) page < (unsigned) a.pages) {
                slot = page * a.page + (j - col * a.page);
                const uint16_t* kp = a.k + (int64_t) page * a.k_ldp + (int64_t) (j - col * a.page) * a.k_ldt + hk * a.k_ldh;
                s = 0.f;
                for (int e = 0; e < D; e += 8) {
                    const auto kv = __builtin_bit_cast(typename Elem<T>::x8, *reinterpret_cast<const u32x4*>(kp + e));
#pragma unroll
                    for (int i = 0; i < 8; ++i) s = fmaf(qs[e + i], (float) kv[i], s);
                }
            }
        }
        float mx = s;
        for (int x = 1; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
        mx = fmaxf(mx, m);
        if (mx == -INFINITY) continue;                  // nothing seen so far (uniform)
        const float p = slot < 0 ? 0.f : __expf(s - mx), c = __expf(m - mx);
        float sum = p;
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        l = l * c + sum;
        m = mx;
        __syncthreads();
        ps[lane] = p;
        slots[lane] = slot;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= c;
        for (int i = 0; i < 64; ++i) {
            const int sl = slots[i];
            if (sl < 0) continue;
            const int page = (int) a.d_page.div((uint32_t) sl);
            const uint16_t* vp = a.v + (int64_t) page * a.v_ldp + (int64_t) (sl - page * a.page) * a.v_ldt + hk * a.v_ldh;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(ps[i], (float) __builtin_bit_cast(T, vp[lane + 64 * e]), acc[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        a.out[(int64_t) t * a.o_ldt + h * a.o_ldh + lane + 64 * e] = __builtin_bit_cast(uint16_t, (T) (l == 0.f ? 0.f : acc[e] / l));
}

template <class T>
void launch_simple(const AttnArgs& a, int d, hipStream_t s)
{
    auto* kern = d == 64 ? attn_simple_kernel<T, 64> : d == 128 ? attn_simple_kernel<T, 128> : attn_simple_kernel<T, 256>;
    hipLaunchKernelGGL(kern, dim3((unsigned) a.tokens, (unsigned) a.hq), dim3(64), 0, s, a);
}

}  // namespace

extern "C" size_t exl3_paged_attention_workspace_size(int tokens, int requests, int q_heads, int kv_heads, int head_dim)
{
    return 0;
}

extern "C" int exl3_paged_attention(const void* q, int64_t q_ldt, int64_t q_ldh, const void* k_cache, int64_t k_ldp, int64_t k_ldt,
                                    int64_t k_ldh, const void* v_cache, int64_t v_ldp, int64_t v_ldt, int64_t v_ldh,
                                    const int* block_table, int64_t ld_table, int table_cols, const int* cu_q, const int* seq_lens,
                                    void* out, int64_t o_ldt, int64_t o_ldh, int tokens, int requests, int q_heads, int kv_heads,
                                    int head_dim, int pages, int page_size, float scale, int window, int dtype, void* workspace,
                                    size_t ws_bytes, void* stream)
{
    if (tokens < 0 || tokens > EXL3_PAGED_MAX_TOKENS || requests < 0 || requests > EXL3_PAGED_MAX_REQUESTS) return EXL3_EINVAL;
    if (q_heads < 1 || q_heads > EXL3_PAGED_MAX_HEADS || kv_heads < 1 || q_heads % kv_heads || !paged_head_dim(head_dim) || !paged_dtype(dtype))
        return EXL3_EINVAL;
    if (pages < 0 || page_size < 16 || page_size % 16 || page_size > EXL3_PAGED_MAX_PAGE || (int64_t) pages * page_size > INT32_MAX) return EXL3_EINVAL;
    if (table_cols < 0 || ld_table < table_cols || (int64_t) table_cols * page_size > INT32_MAX || window < 0) return EXL3_EINVAL;
    if (tokens == 0) return EXL3_OK;
    if (!q || !out || !cu_q || (pages && (!k_cache || !v_cache)) || (requests && !seq_lens) || (requests && table_cols && !block_table)) return EXL3_EINVAL;
    if (!aligned16({q, k_cache, v_cache, out}) ||
        !multiples_of_8({q_ldt, q_ldh, k_ldp, k_ldt, k_ldh, v_ldp, v_ldt, v_ldh, o_ldt, o_ldh}))
        return EXL3_EINVAL;
    AttnArgs a{(const uint16_t*) q, (const uint16_t*) k_cache, (const uint16_t*) v_cache, q_ldt, q_ldh, k_ldp, k_ldt, k_ldh, v_ldp, v_ldt,
               v_ldh, o_ldt, o_ldh, ld_table, block_table, cu_q, seq_lens, (uint16_t*) out, tokens, requests, q_heads, kv_heads, pages,
               table_cols, page_size, window, scale, UDiv::of((uint32_t) page_size), UDiv::of((uint32_t) (q_heads / kv_heads))};
    if (dtype == EXL3_FP16) launch_simple<f16>(a, head_dim, (hipStream_t) stream);
    else launch_simple<__bf16>(a, head_dim, (hipStream_t) stream);
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}
