// exl3_attn.hip -- causal attention of each request's new tokens over its paged key/value cache: the entry point, and
// the kernel for few rows per request (decodes and drafts).
#include "exl3_attn.h"
#include <cmath>

using namespace exl3;

namespace {

template <int N> struct Words;
template <> struct Words<4> { typedef u32x4 T; typedef gc_u32x4 G; };
template <> struct Words<2> { typedef u32x2 T; typedef gc_u32x2 G; };

// ---- few rows: 16 rows a tile, bound by the reading of K and V --------------------------------------------
// Every wave takes whole steps of 32 keys of its tile, with a softmax of its own (running maximum, sum, output), and
// loads their K and V from memory straight into matrix operands, so the loop has no LDS traffic for them and no
// barrier.  The next step's K is requested once this one's scores are formed, its V once this one's products are, so a
// wave has about a step (128 D bytes) in flight at all times and each buffer is there once:
//   S^T = K Q^T  (16x16x32): lane l gives key l & 15 of a page's 16, elements 32 c + 8 (l >> 4) .. + 7
//   O^T = V^T P^T: S^T leaves lane l with keys 4 (l >> 4) + i (i < 4) of both 16s, row l & 15.  Taken as operand elements
//         8 (l >> 4) + j that is already P^T, if V^T's lane holds the same keys: its loads are 16 bytes of 8 rows
//         of V (a row's 16 lanes read it whole), paired by v_perm, and column 8 (l & 15) + e is row l & 15 of product e
// A lane's row of S^T and of O^T is the same (l & 15), so maxima, sums and corrections never leave the lane's column.
// Bound by memory: two sequences of 90000 and 129226 tokens (24 heads over 4 of 256) 173 us, 5.4 TB/s; 48 of 100 to 16000 (40
// over 8 of 128) 92 us, 4.5 TB/s; one of 1500 13.4 us, the latency of its dependent loads and the join.
template <class T, int D, int WAVES>
struct Decode {
    static constexpr int ROWS = 16, THREADS = 64 * WAVES;
    static constexpr int KC = D / 32;                   // 16-byte pieces of a K row that a lane holds
    static constexpr int VW = D >= 128 ? 16 : 8;        // bytes of a V row that a lane loads at once
    static constexpr int VC = D * 2 / (16 * VW);        // ... and how many times
    static constexpr int E = VW / 2;                    // V columns of one load: its products
    static constexpr int LEAST = 4;                     // steps of a share at least
    static constexpr int PAD = D + 4;                   // LDS row (floats) of the waves' outputs
    static constexpr bool Q_LDS = KC > 4;               // Q would take more than 16 registers: read from LDS at each step
    static constexpr int Q_PAD = D + 8;                 // its LDS row (halves)
    static constexpr int GRID = 256;                    // workgroups: one a CU
    static constexpr int SLOT = attn_slot(ROWS, D);
    static_assert(GRID <= ATTN_COUNTERS && (size_t) 2 * GRID * SLOT * 4 <= ATTN_PART_BYTES);
    // Probabilities are rounded to the element type for their product with V, after the 32-bit sum has taken them as they are:
    // the matrix unit's operands have 16 bits, and a second product for what the rounding cuts off would double those with V.
    // The output's error against 64 bits grows by 4 to 11 % in fp16 and 8 to 18 % in bf16 over 32-bit probabilities, most of it
    // being the output's own rounding.  fp16 ones are held times 2^8: the smallest that a key keeps is then 2^-33 of its
    // row's largest.
    static constexpr float SHIFT = std::is_same_v<T, f16> ? 8.f : 0.f;
    using V = typename Words<VW / 4>::T;
    using GV = typename Words<VW / 4>::G;
    using K2 = u32x4[2][KC];
    using V8 = V[8][VC];

    struct Shared {
        float o[WAVES][16][PAD];
        float m[WAVES][ROWS], l[WAVES][ROWS];
        uint16_t q[Q_LDS ? ROWS : 1][Q_PAD];
        uint64_t find[WAVES + 4];
        int last;
    };

    // operand element j of product e of piece u: column e of the lane's piece, key 16 (j >> 2) + 4 (l >> 4) + (j & 3)
    static __device__ __forceinline__ u32x4 column(const V8& v, int u, int e)
    {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_perm(v[2 * j + 1][u][e / 2], v[2 * j][u][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
        return r;
    }
};

template <class T, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, 1) attn_decode_kernel(AttnArgs a)
{
    using X = Decode<T, D, WAVES>;
    constexpr int KC = X::KC, VC = X::VC, E = X::E, ROWS = X::ROWS;
    __shared__ typename X::Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g4 = lane >> 4;
    const int wg = blockIdx.x;

    // rows of no request
    const int used = a.requests ? min(max(a.cu_q[a.requests], 0), a.tokens) : 0;
    for (int t = used + wg; t < a.tokens; t += X::GRID)
        for (int i = tid; i < a.group * a.hkv * (D / 8); i += X::THREADS)
            *reinterpret_cast<g_u32x4*>(as_global(a.out) + (int64_t) t * a.o_ldt + (i / (D / 8)) * a.o_ldh + 8 * (i % (D / 8))) = u32x4{0u, 0u, 0u, 0u};

    AttnWork<ROWS, 32, X::GRID> wk(a);
    int64_t left;
    int off;
    uint32_t per;
    if (!wk.template find<X::THREADS>(wg, X::LEAST, sh.find, off, left, per)) return;

    const uint32_t k_lane = (uint32_t) (c16 * (int) a.k_ldt + 8 * g4) * 2u;
    uint32_t v_lane[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v_lane[i] = (uint32_t) ((4 * g4 + i) * (int) a.v_ldt) * 2u + (uint32_t) (X::VW * c16);

    while (true) {
        wk.settle();
        const AttnTile tile = wk.tile;
        const int n_steps = __builtin_amdgcn_readfirstlane((int) min((int64_t) (tile.steps - off), left));
        const int s0 = tile.step0 + off, s1 = s0 + n_steps;
        const int* const row = a.table + (int64_t) wk.r * a.ld_table;
        const char* const kh = reinterpret_cast<const char*>(a.k + (int64_t) wk.h * a.k_ldh);
        const char* const vh = reinterpret_cast<const char*>(a.v + (int64_t) wk.h * a.v_ldh);

        // Q^T: lane's row c16 of the tile, elements 32 c + 8 g4 ..; and the position of the row's token
        const int rows = wk.n * a.group;
        auto q_at = [&](int x) __attribute__((always_inline)) {
            const int y = min(wk.t * ROWS + x, rows - 1), tok = (int) a.d_group.div((uint32_t) y);
            return as_global(a.q) + (int64_t) (wk.tok0 + tok) * a.q_ldt + (int64_t) (wk.h * a.group + y - tok * a.group) * a.q_ldh;
        };
        u32x4 q[X::Q_LDS ? 1 : KC];
        const int xl = wk.t * ROWS + c16, pos = xl < rows ? wk.pos0 + (int) a.d_group.div((uint32_t) xl) : -1;  // a row past the tile's sees nothing
        const int upto = min(pos, a.cap - 1), from = a.window ? pos - a.window : -1;                            // the row sees from < key <= upto
        if constexpr (!X::Q_LDS) {
            auto* const src = q_at(c16) + 8 * g4;
#pragma unroll
            for (int c = 0; c < KC; ++c) q[c] = flipped(*reinterpret_cast<gc_u32x4*>(src + 32 * c), a.flip);
        }
        if constexpr (X::Q_LDS) {
            for (int z = tid; z < ROWS * D / 8; z += X::THREADS)
                *reinterpret_cast<u32x4*>(&sh.q[z / (D / 8)][8 * (z % (D / 8))]) =
                    flipped(*reinterpret_cast<gc_u32x4*>(q_at(z / (D / 8)) + 8 * (z % (D / 8))), a.flip);
            __syncthreads();
        }
        f32x4 o[VC][E];
        float m = LOWEST, l = 0.f;
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) o[c][e] = f32x4{0.f, 0.f, 0.f, 0.f};

        // pages of this wave's next 32 steps, lane 2 x + y: the y-th 16 keys of its x-th step; -1: none
        auto pages_from = [&](int s) __attribute__((always_inline)) {
            const int key = 32 * (s + WAVES * (lane >> 1)) + 16 * (lane & 1);
            int p = -1;
            if (key < tile.hi) {
                p = row[a.d_page.div((uint32_t) key)];
                if ((unsigned) p >= (unsigned) a.pages) p = -1;
            }
            return p;
        };
        // the first of 16 keys from `key` on of page p of a cache; -1 reads page 0, and its keys are seen by nobody
        auto keys_at = [&](const char* base, int64_t ldp, int64_t ldt, int p, int key) __attribute__((always_inline)) {
            const int in = key - (int) a.d_page.div((uint32_t) key) * a.page;
            return as_global(base) + ((int64_t) max(p, 0) * ldp + (int64_t) in * ldt) * 2;
        };
        auto load_k = [&](typename X::K2& x, int s, int p0, int p1) __attribute__((always_inline)) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                gc_char* const kp = keys_at(kh, a.k_ldp, a.k_ldt, y ? p1 : p0, 32 * s + 16 * y);
#pragma unroll
                for (int c = 0; c < KC; ++c) x[y][c] = *reinterpret_cast<gc_u32x4*>(kp + k_lane + 64 * c);
            }
        };
        auto load_v = [&](typename X::V8& x, int s, int p0, int p1) __attribute__((always_inline)) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                gc_char* const vp = keys_at(vh, a.v_ldp, a.v_ldt, y ? p1 : p0, 32 * s + 16 * y);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < VC; ++c) x[4 * y + i][c] = *reinterpret_cast<typename X::GV*>(vp + v_lane[i] + 16 * X::VW * c);
            }
        };

        int s = s0 + wave;
        if (s < s1 && tile.lo < tile.hi) {
            typename X::K2 k;
            typename X::V8 v;
            int pg = pages_from(s), at = 0, p0 = __builtin_amdgcn_readlane(pg, 0), p1 = __builtin_amdgcn_readlane(pg, 1);
            load_k(k, s, p0, p1);
            load_v(v, s, p0, p1);
            int pg_next = pages_from(s + 32 * WAVES);
            while (true) {
                const int next = s + WAVES;
                int n0 = 0, n1 = 0;
                if (next < s1) {
                    if (++at == 32) {
                        pg = pg_next;
                        pg_next = pages_from(next + 32 * WAVES);
                        at = 0;
                    }
                    n0 = __builtin_amdgcn_readlane(pg, 2 * at);
                    n1 = __builtin_amdgcn_readlane(pg, 2 * at + 1);
                }
                // whether every row sees every key of the step
                const bool whole = p0 >= 0 && p1 >= 0 && 32 * s + 31 <= wk.pos0 + tile.first && (!a.window || 32 * s > wk.pos0 + tile.last - a.window) &&
                                   32 * s + 32 <= a.cap;
                f32x4 st[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    u32x4 qc;
                    if constexpr (X::Q_LDS) qc = *reinterpret_cast<const u32x4*>(&sh.q[c16][32 * c + 8 * g4]);
                    else qc = q[c];
#pragma unroll
                    for (int y = 0; y < 2; ++y) st[y] = mfma16<T>(k[y][c], qc, st[y]);
                }
                if (next < s1) load_k(k, next, n0, n1);
                float mx = m;
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = st[y][e] * a.scale;
                        if (!whole) {
                            const int key = 32 * s + 16 * y + 4 * g4 + e, end = (y ? p1 : p0) >= 0 ? upto : -1;
                            x = ((key <= end) & (key > from)) ? x : -INFINITY;
                        }
                        st[y][e] = x;
                        mx = fmaxf(mx, x);
                    }
                mx = max_quads(mx);
                if (__any(mx > m)) {
                    const float c = exp2_fast(m - mx);
                    l *= c;
#pragma unroll
                    for (int u = 0; u < VC; ++u)
#pragma unroll
                        for (int e = 0; e < E; ++e) o[u][e] *= c;
                    m = mx;
                }
                const float base = m - X::SHIFT;
                typename Elem<T>::x8 p8;
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = exp2_fast(st[y][e] - base);
                        l += x;
                        p8[4 * y + e] = (T) x;
                    }
                const u32x4 pb = __builtin_bit_cast(u32x4, p8);
                // What V holds for keys that a row does not see must not reach it, and a probability of 0 does not hide
                // an infinity or NaN: V of keys that no row sees is zeroed, and where rows of several tokens differ in what
                // they see, such elements are zeroed too and added afterwards to the rows that see them.
                bool odd = false;
                if (!whole) {
                    uint32_t f = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int key = 32 * s + 16 * (i >> 2) + 4 * g4 + (i & 3);
                        const bool live = (key >= tile.lo) & (key < ((i < 4 ? p0 : p1) >= 0 ? tile.hi : 0));
#pragma unroll
                        for (int c = 0; c < VC; ++c)
#pragma unroll
                            for (int e = 0; e < E / 2; ++e) {
                                v[i][c][e] = live ? v[i][c][e] : 0u;
                                f |= nonfinite2<T>(v[i][c][e]);
                            }
                    }
                    odd = tile.first != tile.last && __any(f != 0u);
                    if (odd) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int c = 0; c < VC; ++c)
#pragma unroll
                                for (int e = 0; e < E / 2; ++e) v[i][c][e] &= ~nonfinite2<T>(v[i][c][e]);
                    }
                }
#pragma unroll
                for (int u = 0; u < VC; ++u)
#pragma unroll
                    for (int e = 0; e < E; ++e) o[u][e] = mfma16<T>(X::column(v, u, e), pb, o[u][e]);
                if (odd) {
#pragma unroll 1
                    for (int y = 0; y < 32; ++y) {
                        const int key = 32 * s + y, j = 2 * (y >> 4) + ((y & 3) >> 1);
                        if (key < tile.lo || key >= tile.hi || (y < 16 ? p0 : p1) < 0) continue;
                        gc_u16* const vr = reinterpret_cast<gc_u16*>(keys_at(vh, a.v_ldp, a.v_ldt, y < 16 ? p0 : p1, 32 * s + (y & 16)) + (int64_t) (y & 15) * a.v_ldt * 2);
                        uint32_t pw = j == 0 ? pb[0] : j == 1 ? pb[1] : j == 2 ? pb[2] : pb[3];
                        pw = (uint32_t) __shfl((int) pw, 16 * ((y >> 2) & 3) + c16);
                        const float p = (float) __builtin_bit_cast(T, (uint16_t) (y & 1 ? pw >> 16 : pw));
                        const uint32_t seen = ((key <= upto) & (key > from)) ? 0xFFFFu : 0u;
#pragma unroll
                        for (int u = 0; u < VC; ++u)
#pragma unroll
                            for (int e = 0; e < E; ++e)
#pragma unroll
                                for (int d = 0; d < 4; ++d) {
                                    const uint32_t b = vr[16 * E * u + E * (4 * g4 + d) + e];
                                    o[u][e][d] += p * (float) __builtin_bit_cast(T, (uint16_t) (b & seen & nonfinite2<T>(b)));
                                }
                    }
                }
                if (next >= s1) break;
                load_v(v, next, n0, n1);
                s = next;
                p0 = n0;
                p1 = n1;
            }
        }

        // the waves' outputs joined: maxima first, then sums and outputs scaled to their maximum
        const bool starts = off == 0, ends = off + n_steps == tile.steps, split = !(starts && ends);
        if (g4 == 0) sh.m[wave][c16] = m;
        __syncthreads();
        const int first_wg = wg - (int) (((uint32_t) off + per - 1u) / per);        // workgroups back to the tile's first step
        const uint32_t slot = 2u * (uint32_t) wg + (starts ? 1u : 0u);
        const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(a.part, 0, (int) ATTN_PART_BYTES, RAW_BUFFER_FLAGS);
        auto out_at = [&](int x) __attribute__((always_inline)) {                  // row x of the tile
            const int y = wk.t * ROWS + x, tok = (int) a.d_group.div((uint32_t) y);
            return as_global(a.out) + (int64_t) (wk.tok0 + tok) * a.o_ldt + (int64_t) (wk.h * a.group + y - tok * a.group) * a.o_ldh;
        };
        const int live_rows = min(ROWS, rows - wk.t * ROWS);
        float top = LOWEST;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) top = fmaxf(top, sh.m[x][c16]);
        const float c = exp2_fast(m - top), lt = sum_quads(l) * c;
        if (g4 == 0) sh.l[wave][c16] = lt;
#pragma unroll
        for (int u = 0; u < VC; ++u)
#pragma unroll
            for (int y = 0; y < 4; ++y)                // product e holds columns E (4 g4 + y) + e of piece u
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    *reinterpret_cast<f32x4*>(&sh.o[wave][c16][16 * E * u + E * (4 * g4 + y) + e]) =
                        f32x4{o[u][e][y] * c, o[u][e + 1][y] * c, o[u][e + 2][y] * c, o[u][e + 3][y] * c};
        __syncthreads();
        for (int z = tid; z < live_rows * (D / 4); z += X::THREADS) {
            const int x = z / (D / 4), col = 4 * (z % (D / 4));
            float lx = 0.f;
            f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int y = 0; y < WAVES; ++y) {
                lx += sh.l[y][x];
                sum += *reinterpret_cast<const f32x4*>(&sh.o[y][x][col]);
            }
            if (!split) {
                store_out<T>(out_at(x) + col, sum, lx);
            } else {
                const uint32_t at = (slot * X::SLOT + (uint32_t) (x * D + col)) * 4u;
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), prs, at, 0, SC1);
                if (col == 0) {
                    float mx = LOWEST;
#pragma unroll 4
                    for (int y = 0; y < WAVES; ++y) mx = fmaxf(mx, sh.m[y][x]);
                    const u32x2 ml = u32x2{(uint32_t) __float_as_int(mx), (uint32_t) __float_as_int(lx)};
                    __builtin_amdgcn_raw_buffer_store_b64(ml, prs, (slot * X::SLOT + (uint32_t) (ROWS * D + 2 * x)) * 4u, 0, SC1);
                }
            }
        }
        if (split) {
            // the workgroup that counts last joins the tile's parts, in the order of the workgroups
            const int last_wg = wg + (int) (((uint32_t) (tile.steps - off - n_steps) + per - 1u) / per);
            __builtin_amdgcn_s_waitcnt(0x0F70);        // vmcnt(0): the part has landed
            __syncthreads();
            if (tid == 0) {
                const uint32_t before = __hip_atomic_fetch_add(&a.counters[first_wg], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                sh.last = before == (uint32_t) (last_wg - first_wg);
                if (sh.last) __hip_atomic_store(&a.counters[first_wg], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (sh.last) join_parts<T, D, ROWS, X::THREADS, X::SLOT, 8>(prs, first_wg, last_wg, live_rows, out_at);
        }
        __syncthreads();
        left -= n_steps;
        if (left <= 0) break;
        off = 0;
        wk.next();
    }
}

template <class T>
void launch(const AttnArgs& a, int d, hipStream_t s)
{
    if (d == 64) hipLaunchKernelGGL((attn_decode_kernel<T, 64, 8>), dim3(Decode<T, 64, 8>::GRID), dim3(512), 0, s, a);
    else if (d == 128) hipLaunchKernelGGL((attn_decode_kernel<T, 128, 8>), dim3(Decode<T, 128, 8>::GRID), dim3(512), 0, s, a);
    else hipLaunchKernelGGL((attn_decode_kernel<T, 256, 4>), dim3(Decode<T, 256, 4>::GRID), dim3(256), 0, s, a);
}

}  // namespace

extern "C" size_t exl3_paged_attention_workspace_size(void)
{
    return EXL3_ATTN_COUNTER_BYTES + (size_t) (int) ATTN_PART_BYTES;
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
    if ((int64_t) tokens * (q_heads / kv_heads) > INT32_MAX - 1024) return EXL3_EINVAL;
    if (pages < 0 || page_size < 16 || page_size % 16 || page_size > EXL3_PAGED_MAX_PAGE || (int64_t) pages * page_size > INT32_MAX) return EXL3_EINVAL;
    if (table_cols < 0 || ld_table < table_cols || (int64_t) table_cols * page_size > INT32_MAX - 65536 || window < 0) return EXL3_EINVAL;
    if (window > EXL3_ATTN_MAX_WINDOW) return EXL3_EINVAL;
    // a stride that addresses nothing may be anything
    if (tokens == 1) q_ldt = o_ldt = 0;
    if (q_heads == 1) q_ldh = o_ldh = 0;
    if (kv_heads == 1) k_ldh = v_ldh = 0;
    if (pages <= 1) k_ldp = v_ldp = 0;
    if (k_ldt > EXL3_ATTN_MAX_LDT || v_ldt > EXL3_ATTN_MAX_LDT) return EXL3_EINVAL;
    if (tokens == 0) return EXL3_OK;
    if (!q || !out || !cu_q || (pages && (!k_cache || !v_cache)) || (requests && !seq_lens) || (requests && table_cols && !block_table)) return EXL3_EINVAL;
    if (!aligned16({q, k_cache, v_cache, out}) ||
        !multiples_of_8({q_ldt, q_ldh, k_ldp, k_ldt, k_ldh, v_ldp, v_ldt, v_ldh, o_ldt, o_ldh}))
        return EXL3_EINVAL;
    if (!workspace || ((uintptr_t) workspace & 15u) || ws_bytes < exl3_paged_attention_workspace_size()) return EXL3_EWORKSPACE;
    AttnArgs a{(const uint16_t*) q, (const uint16_t*) k_cache, (const uint16_t*) v_cache, q_ldt, q_ldh, k_ldp, k_ldt, k_ldh, v_ldp, v_ldt,
               v_ldh, o_ldt, o_ldh, ld_table, block_table, cu_q, seq_lens, (uint16_t*) out, tokens, requests, q_heads / kv_heads, kv_heads,
               pages, page_size, window, pages ? table_cols * page_size : 0, std::max(std::fabs(scale) * 1.44269504f, 1e-30f), scale < 0.f ? 0x80008000u : 0u, UDiv::of((uint32_t) page_size),
               UDiv::of((uint32_t) (q_heads / kv_heads)), (uint32_t*) workspace,
               reinterpret_cast<float*>((char*) workspace + EXL3_ATTN_COUNTER_BYTES)};
    // Rows of an average request and kv head: up to 16 are one tile of the decode kernel.  Eight requests of 16000 tokens, 40 heads
    // over 8 of 128, decode / chunk kernel in us: 100 / 125 at 15 rows, 141 / 125 at 20, 169 / 127 at 40; 24 over 4 of 256:
    // 105 / 130 at 12, 174 / 129 at 18; 32 over 8 of 64: 46 / 68 at 16, 68 / 69 at 24; two of 2000 tokens: 19 / 29 at 15 rows
    // of 128, 36 / 29 at 20.  The host knows the average alone, not the lengths, so a batch of unlike requests takes the kernel
    // of the many: a 512-token prompt beside 255 empty requests (40 heads over 8 of 128) 141 us in the decode kernel, which
    // reads its keys for each 16 rows, 30 us by itself; beside 255 decodes over 2000 tokens 575 us there, the two by themselves
    // 30 and 366; with 24 heads over 4 of 256 (18 rows on average) 587 us in the chunk kernel, by themselves 44 and 360.
    if (requests && (int64_t) tokens * a.group / requests > 16) launch_attn_prefill(a, dtype, head_dim, (hipStream_t) stream);
    else if (dtype == EXL3_FP16) launch<f16>(a, head_dim, (hipStream_t) stream);
    else launch<__bf16>(a, head_dim, (hipStream_t) stream);
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}
