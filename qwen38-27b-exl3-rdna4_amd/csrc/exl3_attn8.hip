// exl3_attn8.hip -- causal attention of each request's new tokens over its paged key/value cache in 8 bits: the entry point,
// and the kernel for few rows per request (decodes and drafts).
#include "exl3_attn8.h"
#include <cmath>

using namespace exl3;

namespace {

typedef __attribute__((address_space(1))) const uint32_t gc_w1;

template <int N> struct Codes;
template <> struct Codes<1> { typedef uint32_t T __attribute__((ext_vector_type(1))); typedef __attribute__((address_space(1))) const T G; };
template <> struct Codes<2> { typedef u32x2 T; typedef gc_u32x2 G; };
template <> struct Codes<4> { typedef u32x4 T; typedef gc_u32x4 G; };

// ---- few rows: 16 rows a tile, bound by the reading of K and V --------------------------------------------
// out = sum_j p_j sv_j cv_j / sum_j p_j, p_j = 2^(s_j - m), s_j = (q . ck_j) sk_j scale log2(e), where sk and sv are one number for
// each 16 keys and the codes ck and cv are fp16 numbers without rounding.  So the products are between q (fp16) and codes,
// a block's sk is a factor of its scores, and its sv goes into the exponent: with r the row's running maximum of
// s_j + log2 sv_j, the kernel sums e_j cv_j and e_j / sv_j, e_j = 2^(s_j + log2 sv_j - r), a multiplication a block and no
// more operations an element than without scales.  e is in [0, 1], so fp16 holds it (times 2^8, as in the 16-bit kernel),
// and scales within 2^-40 .. 2^40 leave the sums of e / sv in fp32's range.
// Layout of the products as in the 16-bit cache's kernel: S^T = K Q^T leaves P^T as the next product's operand, a wave takes whole
// steps with a softmax of its own, K and V go from memory into registers and are made operands there.
//   K: a lane holds key l & 15, bytes 64 c + 16 (l >> 4) .. + 15: two products' 8 elements each, so q's lane holds the same columns
//   V: a lane holds E = D / 16 columns E (l & 15) .. of its keys, and product e is made of column e of pairs of keys
template <class T, int D, int WAVES, int KEYS>
struct Decode8 {
    static constexpr int ROWS = 16, THREADS = 64 * WAVES;
    static constexpr int NB = KEYS / C8_BLOCK;          // blocks of a step
    static constexpr int AHEAD = 64 / NB;               // steps whose pages and scales a wave's lanes hold
    static constexpr int KC = D / 64;                   // 16-byte pieces of a K row that a lane holds: two products each
    static constexpr int E = D / 16;                    // V columns of a lane: its products
    static constexpr int LEAST = 4;                     // steps of a share at least
    static constexpr int PAD = D + 4;                   // LDS row (floats) of the waves' outputs
    static constexpr bool Q_LDS = D > 128;              // Q would take more than 16 registers: read from LDS at each step
    static constexpr int Q_PAD = D + 8;                 // its LDS row (halves)
    static constexpr int GRID = 256;                    // workgroups: one a CU
    static constexpr int SLOT = attn_slot(ROWS, D);
    static_assert(GRID <= ATTN_COUNTERS && (size_t) 2 * GRID * SLOT * 4 <= ATTN_PART_BYTES);
    static constexpr float SHIFT = 8.f;                 // fp16 probabilities are held times 2^8
    using V = typename Codes<E / 4>::T;
    using GV = typename Codes<E / 4>::G;
    using KS = u32x4[NB][KC];
    using VS = V[4 * NB];

    struct Shared {
        float o[WAVES][16][PAD];
        float m[WAVES][ROWS], l[WAVES][ROWS];
        uint16_t q[Q_LDS ? ROWS : 1][Q_PAD];
        float grown[ROWS];
        uint64_t find[WAVES + 4];
        int last;
    };
};

template <class T, int D, int WAVES, int KEYS>
__global__ void __launch_bounds__(64 * WAVES, 1) attn8_decode_kernel(Attn8Args a)
{
    using X = Decode8<T, D, WAVES, KEYS>;
    constexpr int KC = X::KC, E = X::E, ROWS = X::ROWS, NB = X::NB, AHEAD = X::AHEAD;
    __shared__ typename X::Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g4 = lane >> 4;
    const int wg = blockIdx.x;

    // rows of no request
    const int used = a.requests ? min(max(a.cu_q[a.requests], 0), a.tokens) : 0;
    for (int t = used + wg; t < a.tokens; t += X::GRID)
        for (int i = tid; i < a.group * a.hkv * (D / 8); i += X::THREADS)
            *reinterpret_cast<g_u32x4*>(as_global(a.out) + (int64_t) t * a.o_ldt + (i / (D / 8)) * a.o_ldh + 8 * (i % (D / 8))) = u32x4{0u, 0u, 0u, 0u};

    AttnWork<ROWS, KEYS, X::GRID> wk(a);
    int64_t left;
    int off;
    uint32_t per;
    if (!wk.template find<X::THREADS>(wg, X::LEAST, sh.find, off, left, per)) return;

    const uint32_t k_lane = (uint32_t) (c16 * (int) a.c.k_ldt + 16 * g4);
    uint32_t v_lane[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v_lane[i] = (uint32_t) ((4 * g4 + i) * (int) a.c.v_ldt + E * c16);

    while (true) {
        wk.settle();
        const AttnTile tile = wk.tile;
        const int n_steps = __builtin_amdgcn_readfirstlane((int) min((int64_t) (tile.steps - off), left));
        const int s0 = tile.step0 + off, s1 = s0 + n_steps;
        const int* const row = a.table + (int64_t) wk.r * a.ld_table;
        const int8_t* const kh = a.c.k + (int64_t) wk.h * a.c.k_ldh;
        const int8_t* const vh = a.c.v + (int64_t) wk.h * a.c.v_ldh;
        const float* const ksh = a.c.ks + (int64_t) wk.h * a.c.ks_ldh;
        const float* const vsh = a.c.vs + (int64_t) wk.h * a.c.vs_ldh;

        // Q^T in fp16: lane's row c16 of the tile, elements 64 c + 16 g4 + 8 h ..; and the position of the row's token
        const int rows = wk.n * a.group;
        auto q_at = [&](int x) __attribute__((always_inline)) {
            const int y = min(wk.t * ROWS + x, rows - 1), tok = (int) a.d_group.div((uint32_t) y);
            return as_global(a.q) + (int64_t) (wk.tok0 + tok) * a.q_ldt + (int64_t) (wk.h * a.group + y - tok * a.group) * a.q_ldh;
        };
        u32x4 q[X::Q_LDS ? 1 : 2 * KC];
        const int xl = wk.t * ROWS + c16, pos = xl < rows ? wk.pos0 + (int) a.d_group.div((uint32_t) xl) : -1;  // a row past the tile's sees nothing
        const int upto = min(pos, a.cap - 1), from = a.window ? pos - a.window : -1;                            // the row sees from < key <= upto
        float qs;                                       // what the row's fp16 elements are to be multiplied by
        if constexpr (!X::Q_LDS) {
            auto* const src = q_at(c16) + 16 * g4;
#pragma unroll
            for (int c = 0; c < 2 * KC; ++c) q[c] = flipped(*reinterpret_cast<gc_u32x4*>(src + 64 * (c / 2) + 8 * (c % 2)), a.flip);
            qs = fp16_rows<T>(q, [](float m) __attribute__((always_inline)) { return max_quads(m); });
        }
        if constexpr (X::Q_LDS) {
            // D / 8 lanes hold a row
            for (int z = tid; z < ROWS * D / 8; z += X::THREADS) {
                u32x4 x[1] = {flipped(*reinterpret_cast<gc_u32x4*>(q_at(z / (D / 8)) + 8 * (z % (D / 8))), a.flip)};
                const float f = fp16_rows<T>(x, [](float m) __attribute__((always_inline)) {
#pragma unroll
                    for (int d = 1; d < D / 8; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
                    return m;
                });
                *reinterpret_cast<u32x4*>(&sh.q[z / (D / 8)][8 * (z % (D / 8))]) = x[0];
                if (z % (D / 8) == 0) sh.grown[z / (D / 8)] = f;
            }
            __syncthreads();
            qs = sh.grown[c16];
        }
        f32x4 o[E];
        float m = LOWEST, l = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float row_scale = row_scale_of(a.scale, qs);

        // pages of this wave's next AHEAD steps, lane NB x + y: block y of its x-th step; -1: none
        auto pages_from = [&](int s) __attribute__((always_inline)) {
            const int key = KEYS * (s + WAVES * (lane / NB)) + C8_BLOCK * (lane % NB);
            int p = -1;
            if (key < tile.hi) {
                p = row[a.d_page.div((uint32_t) key)];
                if ((unsigned) p >= (unsigned) a.pages) p = -1;
            }
            return p;
        };
        // ... and their scales: K's, and V's logarithm
        struct Scales { float k, v; };
        auto scales_of = [&](int s, int p) __attribute__((always_inline)) {
            const int key = KEYS * (s + WAVES * (lane / NB)) + C8_BLOCK * (lane % NB);
            Scales x{1.f, 1.f};
            if (p >= 0) {
                const int in = key - (int) a.d_page.div((uint32_t) key) * a.page;
                x.k = *as_global(ksh + (int64_t) p * a.c.ks_ldp + (int64_t) (in / C8_BLOCK) * a.c.ks_ldb);
                x.v = *as_global(vsh + (int64_t) p * a.c.vs_ldp + (int64_t) (in / C8_BLOCK) * a.c.vs_ldb);
            }
            return x;
        };
        // the first of 16 keys from `key` on of page p of a cache; -1 reads page 0, and its keys are seen by nobody
        auto keys_at = [&](const int8_t* base, int64_t ldp, int64_t ldt, int p, int key) __attribute__((always_inline)) {
            const int in = key - (int) a.d_page.div((uint32_t) key) * a.page;
            return as_global(base) + ((int64_t) max(p, 0) * ldp + (int64_t) in * ldt);
        };
        auto load_k = [&](typename X::KS& x, int s, const int (&p)[NB]) __attribute__((always_inline)) {
#pragma unroll
            for (int y = 0; y < NB; ++y) {
                auto* const kp = keys_at(kh, a.c.k_ldp, a.c.k_ldt, p[y], KEYS * s + C8_BLOCK * y);
#pragma unroll
                for (int c = 0; c < KC; ++c) x[y][c] = *reinterpret_cast<gc_u32x4*>(kp + k_lane + 64 * c);
            }
        };
        auto load_v = [&](typename X::VS& x, int s, const int (&p)[NB]) __attribute__((always_inline)) {
#pragma unroll
            for (int y = 0; y < NB; ++y) {
                auto* const vp = keys_at(vh, a.c.v_ldp, a.c.v_ldt, p[y], KEYS * s + C8_BLOCK * y);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[4 * y + i] = *reinterpret_cast<typename X::GV*>(vp + v_lane[i]);
            }
        };

        int s = s0 + wave;
        if (s < s1 && tile.lo < tile.hi) {
            typename X::KS k;
            typename X::VS v;
            int pg = pages_from(s), at = 0, p[NB];
#pragma unroll
            for (int y = 0; y < NB; ++y) p[y] = __builtin_amdgcn_readlane(pg, y);
            load_k(k, s, p);
            load_v(v, s, p);
            Scales sc = scales_of(s, pg), sc_next = sc;
            int pg_next = pages_from(s + AHEAD * WAVES);
            while (true) {
                const int next = s + WAVES;
                int n[NB];
                float sk[NB], lv[NB];
#pragma unroll
                for (int y = 0; y < NB; ++y) {
                    sk[y] = scale8(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(sc.k), NB * at + y)));
                    lv[y] = log2_fast(scale8(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(sc.v), NB * at + y))));
                    n[y] = 0;
                }
                // the next lanes' scales half way, when their pages have long been there
                if (at == AHEAD / 2) sc_next = scales_of(next + (AHEAD - 1 - at) * WAVES, pg_next);
                if (next < s1) {
                    if (++at == AHEAD) {
                        pg = pg_next;
                        sc = sc_next;
                        pg_next = pages_from(next + AHEAD * WAVES);
                        at = 0;
                    }
#pragma unroll
                    for (int y = 0; y < NB; ++y) n[y] = __builtin_amdgcn_readlane(pg, NB * at + y);
                }
                // whether every row sees every key of the step
                bool whole = KEYS * s + KEYS - 1 <= wk.pos0 + tile.first && (!a.window || KEYS * s > wk.pos0 + tile.last - a.window) && KEYS * s + KEYS <= a.cap;
#pragma unroll
                for (int y = 0; y < NB; ++y) whole = whole && p[y] >= 0;
                f32x4 st[NB];
#pragma unroll
                for (int y = 0; y < NB; ++y) st[y] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2 * KC; ++c) {
                    u32x4 qc;
                    if constexpr (X::Q_LDS) qc = *reinterpret_cast<const u32x4*>(&sh.q[c16][64 * (c / 2) + 16 * g4 + 8 * (c % 2)]);
                    else qc = q[c];
#pragma unroll
                    for (int y = 0; y < NB; ++y) {
                        const uint32_t w0 = k[y][c / 2][2 * (c % 2)] ^ C8_FLIP, w1 = k[y][c / 2][2 * (c % 2) + 1] ^ C8_FLIP;
                        st[y] = mfma16<f16>(u32x4{codes2(w0, 0), codes2(w0, 1), codes2(w1, 0), codes2(w1, 1)}, qc, st[y]);
                    }
                }
                if (next < s1) load_k(k, next, n);
                float mx = m;
#pragma unroll
                for (int y = 0; y < NB; ++y) {
                    const float f = row_scale * sk[y];
                    const int end = p[y] >= 0 ? upto : -1;
                    float top = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = st[y][e] * f;
                        if (!whole) {
                            const int key = KEYS * s + C8_BLOCK * y + 4 * g4 + e;
                            x = ((key <= end) & (key > from)) ? x : -INFINITY;
                        }
                        st[y][e] = x;
                        top = fmaxf(top, x);
                    }
                    mx = fmaxf(mx, top + lv[y]);
                }
                mx = max_quads(mx);
                if (__any(mx > m)) {
                    const float c = exp2_fast(m - mx);
                    l *= c;
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] *= c;
                    m = mx;
                }
                u32x4 pb[NB / 2];
#pragma unroll
                for (int b = 0; b < NB / 2; ++b) {
                    f16x8 p8;
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const int y = 2 * b + z;
                        const float base = m - X::SHIFT - lv[y];
                        float sum = 0.f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = exp2_fast(st[y][e] - base);
                            sum += x;
                            p8[4 * z + e] = (f16) x;
                        }
                        l += sum * exp2_fast(-lv[y]);
                    }
                    pb[b] = __builtin_bit_cast(u32x4, p8);
                }
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int b = 0; b < NB / 2; ++b) {
                        u32x4 x;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int i = 4 * (2 * b + j / 2) + 2 * (j % 2);
                            x[j] = codes2_of(v[i][e / 4], v[i + 1][e / 4], e % 4);
                        }
                        o[e] = mfma16<f16>(x, pb[b], o[e]);
                    }
                if (next >= s1) break;
                load_v(v, next, n);
                s = next;
#pragma unroll
                for (int y = 0; y < NB; ++y) p[y] = n[y];
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
        for (int y = 0; y < 4; ++y)                    // product e holds columns E (4 g4 + y) + e
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<f32x4*>(&sh.o[wave][c16][E * (4 * g4 + y) + e]) = f32x4{o[e][y] * c, o[e + 1][y] * c, o[e + 2][y] * c, o[e + 3][y] * c};
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

template <class T, int D, int WAVES, int KEYS>
void launch_one(const Attn8Args& a, hipStream_t s)
{
    using X = Decode8<T, D, WAVES, KEYS>;
    hipLaunchKernelGGL((attn8_decode_kernel<T, D, WAVES, KEYS>), dim3(X::GRID), dim3(X::THREADS), 0, s, a);
}

template <class T>
void launch(const Attn8Args& a, hipStream_t s)
{
    if (a.c.d == 64) launch_one<T, 64, 8, 64>(a, s);
    else if (a.c.d == 128) launch_one<T, 128, 8, 64>(a, s);
    else launch_one<T, 256, 4, 64>(a, s);
}

}  // namespace

extern "C" int exl3_paged_attention8(const void* q, int64_t q_ldt, int64_t q_ldh, const exl3_cache8* cache, const int* block_table,
                                     int64_t ld_table, int table_cols, const int* cu_q, const int* seq_lens, void* out, int64_t o_ldt,
                                     int64_t o_ldh, int tokens, int requests, int q_heads, float scale, int window, int dtype,
                                     void* workspace, size_t ws_bytes, void* stream)
{
    Attn8Args a{};
    if (!cache8_of(cache, a.c)) return EXL3_EINVAL;
    const int hkv = a.c.hkv, page = a.c.page;
    if (tokens < 0 || tokens > EXL3_PAGED_MAX_TOKENS || requests < 0 || requests > EXL3_PAGED_MAX_REQUESTS) return EXL3_EINVAL;
    if (q_heads < 1 || q_heads > EXL3_PAGED_MAX_HEADS || q_heads % hkv || !paged_dtype(dtype)) return EXL3_EINVAL;
    if ((int64_t) tokens * (q_heads / hkv) > INT32_MAX - 1024) return EXL3_EINVAL;
    if (table_cols < 0 || ld_table < table_cols || (int64_t) table_cols * page > INT32_MAX - 65536) return EXL3_EINVAL;
    if (window < 0 || window > EXL3_ATTN_MAX_WINDOW) return EXL3_EINVAL;
    // a stride that addresses nothing may be anything
    if (tokens == 1) q_ldt = o_ldt = 0;
    if (q_heads == 1) q_ldh = o_ldh = 0;
    if (tokens == 0) return EXL3_OK;
    if (!q || !out || !cu_q || (requests && !seq_lens) || (requests && table_cols && !block_table)) return EXL3_EINVAL;
    if (!aligned16({q, out}) || !multiples_of_8({q_ldt, q_ldh, o_ldt, o_ldh})) return EXL3_EINVAL;
    if (!workspace || ((uintptr_t) workspace & 15u) || ws_bytes < exl3_paged_attention_workspace_size()) return EXL3_EWORKSPACE;
    a.q = (const uint16_t*) q, a.q_ldt = q_ldt, a.q_ldh = q_ldh, a.o_ldt = o_ldt, a.o_ldh = o_ldh, a.ld_table = ld_table;
    a.table = block_table, a.cu_q = cu_q, a.seq = seq_lens, a.out = (uint16_t*) out;
    a.tokens = tokens, a.requests = requests, a.group = q_heads / hkv, a.hkv = hkv, a.pages = a.c.pages, a.page = page, a.window = window;
    a.cap = a.pages ? table_cols * page : 0;
    a.scale = std::fabs(scale) * 1.44269504f;
    a.flip = scale < 0.f ? 0x80008000u : 0u;
    a.d_page = a.c.d_page, a.d_group = UDiv::of((uint32_t) a.group);
    a.counters = (uint32_t*) workspace;
    a.part = reinterpret_cast<float*>((char*) workspace + EXL3_ATTN_COUNTER_BYTES);
    if (requests && (int64_t) tokens * a.group / requests > 16) launch_attn8_prefill(a, dtype, (hipStream_t) stream);
    else if (dtype == EXL3_FP16) launch<f16>(a, (hipStream_t) stream);
    else launch<__bf16>(a, (hipStream_t) stream);
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}
