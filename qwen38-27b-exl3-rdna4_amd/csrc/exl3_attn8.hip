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
// More than 16 rows: a tile is S sets of 16, and S workgroups on one XCD, each with a set, work through the same keys at
// the same time, so that all but the first read them from its L2 (12 requests of 24 rows: 198 MB of memory traffic for 188 MB of keys).
// Layout of the products as in the 16-bit cache's kernel: S^T = K Q^T leaves P^T as the next product's operand, a wave takes whole
// steps with a softmax of its own, K and V go from memory into registers and are made operands there.
//   K: a lane holds key l & 15, bytes 64 c + 16 (l >> 4) .. + 15: two products' 8 elements each, so q's lane holds the same columns
//   V: a lane holds E = D / 16 columns E (l & 15) .. of its keys, and product e is made of column e of pairs of keys
// 16 rows: bound by memory.  96 decodes of 100 to 16000 tokens, 40 heads over 8 of 128 (535 MB), 117 us, 4.6 TB/s (ends of tiles);
// two of 131000, 24 over 4 of 256 (728 MB), 127 us, 5.8 TB/s.  17 to 32 rows: by waits and issue, 12 requests' drafts (189 MB, 24 rows of
// 256) 65 us, 2.9 TB/s; vector instructions take 34 % of the cycles, waits 40 % of the waves' time.
template <class T, int D, int WAVES, int KEYS, int S>
struct Decode8 {
    static constexpr int ROWS = 16, TILE = ROWS * S, THREADS = 64 * WAVES;
    static constexpr int NB = KEYS / C8_BLOCK;          // blocks of a step
    static constexpr int AHEAD = 64 / NB;               // steps whose pages and scales a wave's lanes hold
    static constexpr int KC = D / 64;                   // 16-byte pieces of a K row that a lane holds: two products each
    static constexpr int E = D / 16;                    // V columns of a lane: its products
    static constexpr int LEAST = 256 / KEYS;            // steps of a share at least
    static constexpr int PAD = D + 4;                   // LDS row (floats) of the waves' outputs
    static constexpr bool Q_LDS = D > 128;              // Q would take more than 16 registers: read from LDS at each step
    static constexpr int Q_PAD = D + 8;                 // its LDS row (halves)
    static constexpr int WGS = 8 / WAVES, GRID = 256 * WGS;             // workgroups: WGS a CU
    static constexpr int SHARES = GRID / S;             // S workgroups have a share of the work, 16 rows of its tiles each
    static constexpr int SLOT = attn_slot(ROWS, D);
    static_assert(GRID <= ATTN_COUNTERS / 2 && (size_t) 2 * GRID * SLOT * 4 <= ATTN_PART_BYTES);
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

// Parts of a tile summed in order: part i at slot_at(i) (floats), rows x D outputs, then (maximum, sum) a row.  Z elements of a thread
// and B parts of each are in flight (16 parts: the same time).
template <int D, int ROWS, int THREADS, class SlotAt, class Put>
__device__ __forceinline__ void join8(__amdgpu_buffer_rsrc_t prs, int parts, int rows, SlotAt&& slot_at, Put&& put)
{
    constexpr int Z = 2, B = 8;
    const int all = rows * (D / 4);
    for (int z0 = threadIdx.x; z0 < all; z0 += Z * THREADS) {
        uint32_t at[Z], ml[Z];
        float m[Z], l[Z];
        f32x4 sum[Z];
#pragma unroll
        for (int i = 0; i < Z; ++i) {
            const int z = min(z0 + i * THREADS, all - 1);
            at[i] = 16u * (uint32_t) z;
            ml[i] = (uint32_t) (ROWS * D + 2 * (z / (D / 4))) * 4u;
            m[i] = LOWEST;
            l[i] = 0.f;
            sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll 1
        for (int c0 = 0; c0 < parts; c0 += B) {
            u32x2 mls[Z][B];
            f32x4 v[Z][B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const uint32_t s = 4u * (uint32_t) __builtin_amdgcn_readfirstlane((int) slot_at(min(c0 + b, parts - 1)));
#pragma unroll
                for (int i = 0; i < Z; ++i) {
                    mls[i][b] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(prs, ml[i], s, SC1));
                    v[i][b] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, at[i], s, SC1));
                }
            }
#pragma unroll
            for (int i = 0; i < Z; ++i) {
                float top = m[i];
#pragma unroll
                for (int b = 0; b < B; ++b) top = fmaxf(top, __int_as_float((int) mls[i][b][0]));
                const float c = exp2_fast(m[i] - top);
                l[i] *= c;
                sum[i] *= c;
                m[i] = top;
#pragma unroll
                for (int b = 0; b < B; ++b) {
                    const float f = c0 + b < parts ? exp2_fast(__int_as_float((int) mls[i][b][0]) - top) : 0.f;
                    l[i] += f * __int_as_float((int) mls[i][b][1]);
                    sum[i] += v[i][b] * f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < Z; ++i) {
            const int z = z0 + i * THREADS;
            if (z < all) put(z / (D / 4), 4 * (z % (D / 4)), sum[i], m[i], l[i]);
        }
    }
}

template <class T, int D, int WAVES, int KEYS, int S>
__global__ void __launch_bounds__(64 * WAVES, 2) attn8_decode_kernel(Attn8Args a)
{
    using X = Decode8<T, D, WAVES, KEYS, S>;
    constexpr int KC = X::KC, E = X::E, ROWS = X::ROWS, NB = X::NB, AHEAD = X::AHEAD;
    __shared__ typename X::Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g4 = lane >> 4;
    // workgroups go round the 8 XCDs: b and b + 8 are on one
    const int set = S == 1 ? 0 : (int) blockIdx.x / 8 % S, wg = S == 1 ? (int) blockIdx.x : (int) blockIdx.x / (8 * S) * 8 + (int) blockIdx.x % 8;

    // rows of no request
    const int used = a.requests ? min(max(a.cu_q[a.requests], 0), a.tokens) : 0;
    for (int t = used + (int) blockIdx.x; t < a.tokens; t += X::GRID)
        for (int i = tid; i < a.group * a.hkv * (D / 8); i += X::THREADS)
            *reinterpret_cast<g_u32x4*>(as_global(a.out) + (int64_t) t * a.o_ldt + (i / (D / 8)) * a.o_ldh + 8 * (i % (D / 8))) = u32x4{0u, 0u, 0u, 0u};

    using Work = AttnWork<X::TILE, KEYS, X::SHARES>;
    Work wk(a);
    int64_t left;
    int off;
    uint32_t per;
    if (!wk.template find<X::THREADS>(wg, X::LEAST, sh.find, off, left, per)) return;

    const uint32_t k_lane = (uint32_t) (c16 * (int) a.c.k_ldt + 16 * g4);
    uint32_t v_lane[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v_lane[i] = (uint32_t) ((4 * g4 + i) * (int) a.c.v_ldt + E * c16);

    // What a tile's first steps need is requested before the tile before is done, so that its trips to memory (lengths, table, then
    // keys) pass beside the other's work; `x` is a tile's work in all of these.
    auto rows_of = [&](const Work& x) __attribute__((always_inline)) { return x.n * a.group; };
    // pages of this wave's next AHEAD steps, lane NB x + y: block y of its x-th step; -1: none
    auto pages_from = [&](const Work& x, int s) __attribute__((always_inline)) {
        const int key = KEYS * (s + WAVES * (lane / NB)) + C8_BLOCK * (lane % NB);
        int p = -1;
        if (key < x.tile.hi) {
            p = (a.table + (int64_t) x.r * a.ld_table)[a.d_page.div((uint32_t) key)];
            if ((unsigned) p >= (unsigned) a.pages) p = -1;
        }
        return p;
    };
    // ... and their scales
    struct Scales { float k, v; };
    auto scales_of = [&](const Work& x, int s, int p) __attribute__((always_inline)) {
        const int key = KEYS * (s + WAVES * (lane / NB)) + C8_BLOCK * (lane % NB);
        float k = 1.f, v = 1.f;
        if (p >= 0) {
            const int b = (key - (int) a.d_page.div((uint32_t) key) * a.page) / C8_BLOCK;
            k = *as_global(a.c.ks + (int64_t) x.h * a.c.ks_ldh + (int64_t) p * a.c.ks_ldp + (int64_t) b * a.c.ks_ldb);
            v = *as_global(a.c.vs + (int64_t) x.h * a.c.vs_ldh + (int64_t) p * a.c.vs_ldp + (int64_t) b * a.c.vs_ldb);
        }
        return Scales{k, v};
    };
    // the first of 16 keys from `key` on of page p of a cache; -1 reads page 0, and its keys are seen by nobody
    auto keys_at = [&](const int8_t* base, int64_t ldp, int64_t ldt, int p, int key) __attribute__((always_inline)) {
        const int in = key - (int) a.d_page.div((uint32_t) key) * a.page;
        return as_global(base) + ((int64_t) max(p, 0) * ldp + (int64_t) in * ldt);
    };
    // Keys that one workgroup alone reads leave the caches to others: 5 to 12 % faster.
    auto load_once = [&](auto* p) __attribute__((always_inline)) {
        if constexpr (S == 1) return __builtin_nontemporal_load(p);
        else return *p;
    };
    typename X::KS k;
    typename X::VS v;
    auto load_k = [&](const Work& x, int s, const int (&p)[NB]) __attribute__((always_inline)) {
#pragma unroll
        for (int y = 0; y < NB; ++y) {
            auto* const kp = keys_at(a.c.k + (int64_t) x.h * a.c.k_ldh, a.c.k_ldp, a.c.k_ldt, p[y], KEYS * s + C8_BLOCK * y);
#pragma unroll
            for (int c = 0; c < KC; ++c) k[y][c] = load_once(reinterpret_cast<gc_u32x4*>(kp + k_lane + 64 * c));
        }
    };
    auto load_v = [&](const Work& x, int s, const int (&p)[NB]) __attribute__((always_inline)) {
#pragma unroll
        for (int y = 0; y < NB; ++y) {
            auto* const vp = keys_at(a.c.v + (int64_t) x.h * a.c.v_ldh, a.c.v_ldp, a.c.v_ldt, p[y], KEYS * s + C8_BLOCK * y);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * y + i] = load_once(reinterpret_cast<typename X::GV*>(vp + v_lane[i]));
        }
    };
    // Q^T: lane's row c16 of the tile, elements 64 c + 16 g4 + 8 h ..; or a thread's pieces of Q on their way to LDS
    constexpr int NQ = X::Q_LDS ? ROWS * D / 8 / X::THREADS : 2 * KC;
    u32x4 q[NQ];
    auto load_q = [&](const Work& x) __attribute__((always_inline)) {
        auto at = [&](int z) __attribute__((always_inline)) {
            const int y = min(x.t * X::TILE + ROWS * set + z, rows_of(x) - 1), tok = (int) a.d_group.div((uint32_t) y);
            return as_global(a.q) + (int64_t) (x.tok0 + tok) * a.q_ldt + (int64_t) (x.h * a.group + y - tok * a.group) * a.q_ldh;
        };
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
            const int z = tid + X::THREADS * c;
            q[c] = X::Q_LDS ? *reinterpret_cast<gc_u32x4*>(at(z / (D / 8)) + 8 * (z % (D / 8)))
                            : *reinterpret_cast<gc_u32x4*>(at(c16) + 16 * g4 + 64 * (c / 2) + 8 * (c % 2));
        }
    };
    int pg = -1;
    Scales sc{1.f, 1.f};
    auto steps_of = [&](const Work& x, int off, int64_t left) __attribute__((always_inline)) {
        return __builtin_amdgcn_readfirstlane((int) min((int64_t) (x.tile.steps - off), left));
    };
    // the first step of a wave of the tile's steps s0 .. s1 - 1, whose pages are in pg
    auto begin = [&](const Work& x, int s0, int s1) __attribute__((always_inline)) {
        load_q(x);
        const int s = s0 + wave;
        if (s < s1 && x.tile.lo < x.tile.hi) {
            int p[NB];
#pragma unroll
            for (int y = 0; y < NB; ++y) p[y] = __builtin_amdgcn_readlane(pg, y);
            load_k(x, s, p);
            sc = scales_of(x, s, pg);
            load_v(x, s, p);
        }
    };

    wk.settle();
    int n_steps = steps_of(wk, off, left);
    pg = pages_from(wk, wk.tile.step0 + off + wave);
    begin(wk, wk.tile.step0 + off, wk.tile.step0 + off + n_steps);
    while (true) {
        const AttnTile tile = wk.tile;
        const int s0 = tile.step0 + off, s1 = s0 + n_steps, rows = rows_of(wk);
        // the next tile's lengths, and its first pages on their way
        const int64_t after = left - n_steps;
        Work nx(a);
        int pg_nx = -1, n_nx = 0;
        nx.r = wk.r, nx.t = wk.t, nx.h = wk.h, nx.tok0 = wk.tok0, nx.n = wk.n, nx.pos0 = wk.pos0;
        if (after > 0) {
            nx.next();
            nx.settle();
            n_nx = steps_of(nx, 0, after);
            pg_nx = pages_from(nx, nx.tile.step0 + wave);
        }

        const int live_rows = max(min(ROWS, rows - wk.t * X::TILE - ROWS * set), 0);
        // Q in fp16, and the position of the row's token
        const int xl = wk.t * X::TILE + ROWS * set + c16, pos = xl < rows ? wk.pos0 + (int) a.d_group.div((uint32_t) xl) : -1;  // a row past the tile's sees nothing
        const int upto = min(pos, a.cap - 1), from = a.window ? pos - a.window : -1;                            // the row sees from < key <= upto
        float qs;                                       // what the row's fp16 elements are to be multiplied by
#pragma unroll
        for (int c = 0; c < NQ; ++c) q[c] = flipped(q[c], a.flip);
        if constexpr (!X::Q_LDS) qs = fp16_rows<T>(q, [](float m) __attribute__((always_inline)) { return max_quads(m); });
        if constexpr (X::Q_LDS) {
            // D / 8 lanes hold a row
#pragma unroll
            for (int c = 0; c < NQ; ++c) {
                const int z = tid + X::THREADS * c;
                u32x4 x[1] = {q[c]};
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

        int s = s0 + wave;
        if (s < s1 && tile.lo < tile.hi && live_rows > 0) {
            int at = 0, p[NB];
#pragma unroll
            for (int y = 0; y < NB; ++y) p[y] = __builtin_amdgcn_readlane(pg, y);
            int pg_next = pages_from(wk, s + AHEAD * WAVES);
            // a lane's block: K's scale, V's logarithm and 1 / V's
            float ska = scale8(sc.k), lva = log2_fast(scale8(sc.v)), iva = exp2_fast(-lva);
            Scales sc_next{1.f, 1.f};
            while (true) {
                const int next = s + WAVES;
                int n[NB];
                float sk[NB], lv[NB], iv[NB];
                auto of_block = [&](float x, int y) __attribute__((always_inline)) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), NB * at + y)); };
#pragma unroll
                for (int y = 0; y < NB; ++y) {
                    sk[y] = of_block(ska, y);
                    lv[y] = of_block(lva, y);
                    iv[y] = of_block(iva, y);
                    n[y] = 0;
                }
                // the next lanes' scales half way, when their pages have long been there
                if (at == AHEAD / 2) sc_next = scales_of(wk, next + (AHEAD - 1 - at) * WAVES, pg_next);
                if (next < s1) {
                    if (++at == AHEAD) {
                        pg = pg_next;
                        ska = scale8(sc_next.k);
                        lva = log2_fast(scale8(sc_next.v));
                        iva = exp2_fast(-lva);
                        pg_next = pages_from(wk, next + AHEAD * WAVES);
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
                if (next < s1) load_k(wk, next, n);
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
                        l = fmaf(sum, iv[y], l);
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
                load_v(wk, next, n);
                s = next;
#pragma unroll
                for (int y = 0; y < NB; ++y) p[y] = n[y];
            }
        }
        if (after > 0) {
            pg = pg_nx;
            begin(nx, nx.tile.step0, nx.tile.step0 + n_nx);
        }

        // the waves' outputs joined: maxima first, then sums and outputs scaled to their maximum
        const bool starts = off == 0, ends = off + n_steps == tile.steps, split = !(starts && ends);
        if (g4 == 0) sh.m[wave][c16] = m;
        __syncthreads();
        const int first_wg = wg - (int) (((uint32_t) off + per - 1u) / per);        // workgroups back to the tile's first step
        const uint32_t slot = 2u * (uint32_t) (wg + set * X::SHARES) + (starts ? 1u : 0u);
        const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(a.part, 0, (int) ATTN_PART_BYTES, RAW_BUFFER_FLAGS);
        auto out_at = [&](int x) __attribute__((always_inline)) {                  // row x of the tile
            const int y = wk.t * X::TILE + ROWS * set + x, tok = (int) a.d_group.div((uint32_t) y);
            return as_global(a.out) + (int64_t) (wk.tok0 + tok) * a.o_ldt + (int64_t) (wk.h * a.group + y - tok * a.group) * a.o_ldh;
        };
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
        if (split && live_rows > 0) {
            // Who counts last joins, in the order of the workgroups.  Many parts in two levels: groups of about their number's
            // root, joined by the last of each at the same time, then the groups.  (A workgroup's part of one tile and of the
            // next lie in slots 2 c and 2 c + 1 and are counted under the tiles' first workgroups.  What is joined of a group lies in a
            // slot that neither uses: 2 c + 1 of its first workgroup c, which begins no tile, or for a tile's first group of its second.)
            const int last_wg = wg + (int) (((uint32_t) (tile.steps - off - n_steps) + per - 1u) / per), n = last_wg - first_wg + 1;
            const int size = n <= 12 ? n : n <= 64 ? 8 : n <= 256 ? 16 : 24, group = (wg - first_wg) / size, groups = (n + size - 1) / size;
            const int begin_wg = first_wg + group * size, in_group = min(size, last_wg + 1 - begin_wg);
            auto part = [&](int c) __attribute__((always_inline)) { return (uint32_t) (2 * (c + set * X::SHARES) + (c == first_wg ? 1 : 0)) * (uint32_t) X::SLOT; };
            auto joined = [&](int g) __attribute__((always_inline)) {
                const int c = first_wg + g * size;
                return c == last_wg ? part(c) : (uint32_t) (2 * ((g ? c : c + 1) + set * X::SHARES) + 1) * (uint32_t) X::SLOT;
            };
            auto i_am_last = [&](uint32_t* counter, int of) __attribute__((always_inline)) {
                __builtin_amdgcn_s_waitcnt(0x0F70);    // vmcnt(0): the part has landed
                __syncthreads();
                if (tid == 0) {
                    sh.last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t) (of - 1);
                    if (sh.last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                __syncthreads();
                return sh.last != 0;
            };
            bool mine = true;
            if (groups > 1 && in_group > 1) {
                mine = i_am_last(&a.counters[ATTN_COUNTERS / 2 + begin_wg + set * X::SHARES], in_group);
                if (mine) {
                    const uint32_t to = joined(group);
                    join8<D, ROWS, X::THREADS>(prs, in_group, live_rows, [&](int i) __attribute__((always_inline)) { return part(begin_wg + i); },
                                               [&](int x, int col, f32x4 sum, float top, float l) __attribute__((always_inline)) {
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), prs, (to + (uint32_t) (x * D + col)) * 4u, 0, SC1);
                        if (col == 0)
                            __builtin_amdgcn_raw_buffer_store_b64(u32x2{(uint32_t) __float_as_int(top), (uint32_t) __float_as_int(l)}, prs, (to + (uint32_t) (ROWS * D + 2 * x)) * 4u, 0, SC1);
                    });
                }
            }
            if (mine && i_am_last(&a.counters[first_wg + set * X::SHARES], groups > 1 ? groups : n))
                join8<D, ROWS, X::THREADS>(prs, groups > 1 ? groups : n, live_rows,
                                           [&](int i) __attribute__((always_inline)) { return groups > 1 ? joined(i) : part(first_wg + i); },
                                           [&](int x, int col, f32x4 sum, float, float l) __attribute__((always_inline)) { store_out<T>(out_at(x) + col, sum, l); });
        }
        __syncthreads();
        if (after <= 0) break;
        left = after;
        off = 0;
        n_steps = n_nx;
        wk.r = nx.r, wk.t = nx.t, wk.h = nx.h, wk.tok0 = nx.tok0, wk.n = nx.n, wk.pos0 = nx.pos0, wk.tile = nx.tile;
    }
}

template <class T, int D, int WAVES, int KEYS, int S>
void launch_one(const Attn8Args& a, hipStream_t s)
{
    using X = Decode8<T, D, WAVES, KEYS, S>;
    hipLaunchKernelGGL((attn8_decode_kernel<T, D, WAVES, KEYS, S>), dim3(X::GRID), dim3(X::THREADS), 0, s, a);
}

template <class T>
void launch(const Attn8Args& a, int rows, hipStream_t s)
{
    // Four waves a workgroup and two workgroups a CU: one streams while the other ends a tile and begins the next (512 requests of 200
    // tokens, 40 heads over 8 of 128: 64 us, with one workgroup of eight waves 90).  Heads of 256 and few tiles, so that hardly
    // any end, take eight waves: two and four requests' tiles over 131000 tokens 101 us against 112, but 256 requests of 1000 110
    // against 100.  Up to 32 rows on average: two workgroups that share a tile's keys (TILE above).
    if (rows > 16) {
        if (a.c.d == 64) launch_one<T, 64, 4, 64, 2>(a, s);
        else if (a.c.d == 128) launch_one<T, 128, 4, 32, 2>(a, s);
        else launch_one<T, 256, 8, 32, 2>(a, s);
    } else if (a.c.d == 64) launch_one<T, 64, 4, 64, 1>(a, s);
    else if (a.c.d == 128) launch_one<T, 128, 4, 64, 1>(a, s);
    else if ((int64_t) a.requests * a.hkv >= 256) launch_one<T, 256, 4, 32, 1>(a, s);
    else launch_one<T, 256, 8, 32, 1>(a, s);
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
    // Rows of an average request and kv head: up to 16 are one tile of the decode kernel, up to 32 two sets of 16 rows whose workgroups
    // read the same keys at the same time.  Two sets / one set after the other / chunk kernel, us, fp16: 12 requests of 1000 to 32000 tokens,
    // 24 rows, 24 heads over 4 of 256: 77 / 93 / 89; 16 of 4000 46 / 60 / 61, one of 1000 17 / 17 / 24; 20 rows, 40 over 8 of 128: 73 / 91 / 80,
    // 49 / 65 / 59, 12 / 12 / 20; 24 rows, 32 over 8 of 64: 50 / 55 / 57, 36 / 40 / 40, 10 / 10 / 15.  From 33 rows the chunk kernel: eight
    // of 16000 tokens, 40 rows of 128, 119 us against 143 with four sets; 36 rows of 256, 102 against 120, and 64 of 1000 53 against 78.
    // The host knows the average alone, not the lengths, so a batch of unlike requests takes the kernel of the many.  That costs most where a few
    // chunks are among many decodes: 256 decodes over 4000 tokens and 512 tokens over 8000, 40 heads over 8 of 128, 904 us; in two calls 428 + 153.
    const int64_t rows = requests ? (int64_t) tokens * a.group / requests : 0;
    if (rows > 32) launch_attn8_prefill(a, rows, dtype, (hipStream_t) stream);
    else if (dtype == EXL3_FP16) launch<f16>(a, (int) rows, (hipStream_t) stream);
    else launch<__bf16>(a, (int) rows, (hipStream_t) stream);
    return hipGetLastError() == hipSuccess ? EXL3_OK : EXL3_ELAUNCH;
}
