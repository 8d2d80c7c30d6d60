// exl3_attn_prefill.hip -- paged attention for many rows a request (prompt chunks), bound by the matrix products.
#include "exl3_attn.h"

using namespace exl3;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char lchar;
typedef __attribute__((address_space(3))) u32x4 lu32x4;
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class T> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mfma32<f16>(u32x4 a, u32x4 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma32<__bf16>(u32x4 a, u32x4 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// values formed by here: they would be sunk to their first use, past the products that they are to run beside
__device__ __forceinline__ void here(u32x4& a, u32x4& b, float& c)
{
    asm volatile("" : "+v"(a), "+v"(b), "+v"(c));
}

// 128 rows a tile, 64 keys a step.  K and V go through LDS once for all waves: a wave requests its keys (of one page: page
// sizes are multiples of 16) of step s + 2 while step s is computed, and stores those of s + 1 into the other buffer
// after it, so a step has one barrier.  Heads of 64 and 128 take four waves of 32 rows:
//   S^T = K Q^T (32x32x16): lane l gives key l & 31, elements 16 c + 8 (l >> 5) ..; its result holds row l & 31,
//         keys 8 (i >> 2) + 4 (l >> 5) + (i & 3)
//   O^T = V^T P^T: results 8 b .. 8 b + 7 are operand elements of 16 keys as they lie; V^T's lane gets the same keys by
//         transposing LDS reads (16 lanes read 4 keys x 16 columns, lane i gets column i of the 4)
// Heads of 256 take eight waves of 16 rows (16x16x32, row l & 15, keys 4 (l >> 4) + (i & 3) of two 16s: the decode kernel's
// layout): 32 rows' outputs and Q alone would be 192 registers, one wave a SIMD, with nothing to run beside its waits.
// A lane's row is the same in S^T and O^T, as in the decode kernel.  LDS rows are padded so that no bank is met twice: K's by
// 16 bytes (16 keys' reads of one piece), V's by 64 (4 keys' 64 bytes) or, for 16 rows a wave, 32 (16 keys' 32 bytes);
// padded rows, unlike permuted ones, let one address register and the instructions' offsets reach a whole step, and the two
// buffers are two copies of the loop's body for the same reason: at 128 columns the registers are all taken (output 64,
// Q 32, scores 32, K and V on the way 32).  One copy, the buffer a register, takes 1 to 1.5 % longer over long contexts.
// 2048 tokens over 14000 (40 heads over 8 of 128): 786 to 831 us, 755 to 800 TFLOPS (a large library product takes 1160 to 1220); a
// 2048-token prompt 100 us; 8 x 4 tokens over 1000 to 32000 (24 over 4 of 256) 83 us, 3.0 TB/s of K and V.
template <class T, int D>
struct Prefill {
    static constexpr int RW = D == 256 ? 16 : 32;       // rows of a wave
    static constexpr int ROWS = 128, KEYS = 64, WAVES = ROWS / RW, THREADS = 64 * WAVES;
    static constexpr int GRID = D == 256 ? 256 : 512;   // workgroups: one or two a CU
    static constexpr int SLOT = attn_slot(ROWS, D + 128 / RW - 2); // every lane's maximum and sum, also where lanes share a row
    static_assert(GRID <= ATTN_COUNTERS && (size_t) 2 * GRID * SLOT * 4 <= ATTN_PART_BYTES);
    static constexpr int LEAST = 4;                     // steps of a share at least
    static constexpr int CH = D / 8;                    // 16-byte pieces of a row
    static constexpr int KW = KEYS / WAVES;             // keys that a wave moves
    static constexpr int LI = KW * CH / 64;             // ... pieces of them a lane
    static constexpr int KD = RW == 32 ? 16 : 32;       // columns of K that a product takes
    static constexpr int KS = D / KD;                   // products over D
    static constexpr int DT = D / RW;                   // column tiles of the output
    static constexpr int AE = RW == 32 ? 16 : 4;        // results of a product a lane
    static constexpr int TH = 32 / RW;                  // key tiles of a half step (32 keys)
    static constexpr int NB = AE * TH / 8;              // operands of its probabilities
    using Acc = std::conditional_t<RW == 32, f32x16, f32x4>;
    static constexpr float SHIFT = std::is_same_v<T, f16> ? 8.f : 0.f;   // fp16 probabilities are held times 2^8 (Decode::SHIFT)
    static constexpr int K_LD = D + 8, V_LD = RW == 32 ? D + 32 : D + 16;  // LDS rows, halves

    struct alignas(16) Shared {
        alignas(16) uint16_t k[2][KEYS * K_LD];
        alignas(16) uint16_t v[2][KEYS * V_LD];
        uint64_t find[WAVES + 4];
        alignas(16) int page[2][WAVES];                 // of a wave's keys: 1 their page is one, 2 zeroed elements are to be added
        int last;
    };
    static __device__ __forceinline__ Acc product(u32x4 a, u32x4 b, Acc c)
    {
        if constexpr (RW == 32) return mfma32<T>(a, b, c);
        else return mfma16<T>(a, b, c);
    }
    static __device__ __forceinline__ float row_max(float x)
    {
        if constexpr (RW == 16) return max_quads(x);
        float lo, hi;
        halves_x(x, lo, hi);
        return fmaxf(lo, hi);
    }
    static __device__ __forceinline__ float row_sum(float x)
    {
        if constexpr (RW == 16) return sum_quads(x);
        float lo, hi;
        halves_x(x, lo, hi);
        return lo + hi;
    }
    // place of result e of a half step's 32 keys (less 4 (l / RW)), and of quad g of column tile d
    static constexpr int key_of(int e) { return RW == 32 ? 8 * (e >> 2) + (e & 3) : 16 * (e >> 2) + (e & 3); }
    static constexpr int col_of(int d, int g) { return RW * d + 8 * g; }
};

template <class T, int D>
__global__ void __launch_bounds__((Prefill<T, D>::THREADS), (Prefill<T, D>::THREADS == 256 ? 2 : 1)) attn_prefill_kernel(AttnArgs a)
{
    using X = Prefill<T, D>;
    using Acc = typename X::Acc;
    constexpr int LI = X::LI, KS = X::KS, DT = X::DT, CH = X::CH, RW = X::RW, KW = X::KW, AE = X::AE, TH = X::TH, NB = X::NB, QD = AE / 4;
    __shared__ typename X::Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), cr = lane % RW, hg = lane / RW;
    // consecutive shares to one XCD (workgroups go round the 8 XCDs): they read the same head's K and V
    const int wg = (int) (blockIdx.x % 8) * (X::GRID / 8) + (int) blockIdx.x / 8;

    const int used = a.requests ? min(max(a.cu_q[a.requests], 0), a.tokens) : 0;
    for (int t = used + wg; t < a.tokens; t += X::GRID)    // rows of no request
        for (int i = tid; i < a.group * a.hkv * (D / 8); i += X::THREADS)
            *reinterpret_cast<g_u32x4*>(as_global(a.out) + (int64_t) t * a.o_ldt + (i / (D / 8)) * a.o_ldh + 8 * (i % (D / 8))) = u32x4{0u, 0u, 0u, 0u};

    AttnWork<X::ROWS, X::KEYS, X::GRID> wk(a);
    int64_t left;
    int off;
    uint32_t per;
    if (!wk.template find<X::THREADS>(wg, X::LEAST, sh.find, off, left, per)) return;

    // the lane's place in its wave's keys: row st_row + 64 / CH i, piece st_piece
    const int st_row = lane / CH, st_piece = lane % CH;
    // transposing reads: key 4 hg + tr_row, columns 16 tr_half + 4 tr_q ..
    const int s16 = lane & 15, tr_row = s16 >> 2, tr_q = s16 & 3, tr_half = RW == 32 ? (lane >> 4) & 1 : 0;

    const uint32_t k_lane = (uint32_t) (st_row * (int) a.k_ldt + 8 * st_piece) * 2u, v_lane = (uint32_t) (st_row * (int) a.v_ldt + 8 * st_piece) * 2u;
    // LDS addresses of the lane's writes and reads: what the instructions' offsets are added to
    lchar* const k_put = (lchar*) &sh.k[0][(KW * wave + st_row) * X::K_LD + 8 * st_piece];
    lchar* const v_put = (lchar*) &sh.v[0][(KW * wave + st_row) * X::V_LD + 8 * st_piece];
    lchar* const k_get = (lchar*) &sh.k[0][cr * X::K_LD + 8 * hg];
    lchar* const v_get = (lchar*) &sh.v[0][(4 * hg + tr_row) * X::V_LD + 16 * tr_half + 4 * tr_q];

    while (true) {
        wk.settle();
        const AttnTile tile = wk.tile;
        const int n_steps = __builtin_amdgcn_readfirstlane((int) min((int64_t) (tile.steps - off), left));
        const int s0 = tile.step0 + off, s1 = s0 + n_steps, rows = wk.n * a.group;
        const int* const table = a.table + (int64_t) wk.r * a.ld_table;
        const char* const kh = reinterpret_cast<const char*>(a.k + (int64_t) wk.h * a.k_ldh);
        const char* const vh = reinterpret_cast<const char*>(a.v + (int64_t) wk.h * a.v_ldh);

        const int x0 = wk.t * X::ROWS + RW * wave;      // the wave's first row
        const bool rows_here = x0 < rows;
        const int w_first = wk.pos0 + (int) a.d_group.div((uint32_t) x0), w_last = wk.pos0 + (int) a.d_group.div((uint32_t) (min(x0 + RW, rows) - 1));
        const int xl = x0 + cr, tok = (int) a.d_group.div((uint32_t) min(xl, rows - 1)), pos = xl < rows ? wk.pos0 + tok : -1;
        const int upto = min(pos, a.cap - 1), from = a.window ? pos - a.window : -1;
        u32x4 q[KS];
        {
            gc_u16* const src = as_global(a.q) + (int64_t) (wk.tok0 + tok) * a.q_ldt + (int64_t) (wk.h * a.group + min(xl, rows - 1) - tok * a.group) * a.q_ldh + 8 * hg;
#pragma unroll
            for (int c = 0; c < KS; ++c) q[c] = flipped(*reinterpret_cast<gc_u32x4*>(src + X::KD * c), a.flip);
        }
        Acc o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < AE; ++i) o[d][i] = 0.f;
        float m = LOWEST, l = 0.f;

        auto page_of = [&](int s) __attribute__((always_inline)) {
            const int key = X::KEYS * s + KW * wave;
            int p = -1;
            if (key < tile.hi) {
                p = table[a.d_page.div((uint32_t) key)];
                if ((unsigned) p >= (unsigned) a.pages) p = -1;
            }
            return __builtin_amdgcn_readfirstlane(p);
        };
        auto keys_at = [&](const char* base, int64_t ldp, int64_t ldt, int p, int key) __attribute__((always_inline)) {
            const int in = key - (int) a.d_page.div((uint32_t) key) * a.page;
            return as_global(base) + ((int64_t) max(p, 0) * ldp + (int64_t) in * ldt) * 2;
        };
        u32x4 kr[LI], vr[LI];
        auto request = [&](int s, int p) __attribute__((always_inline)) {
            gc_char* const kp = keys_at(kh, a.k_ldp, a.k_ldt, p, X::KEYS * s + KW * wave);
            gc_char* const vp = keys_at(vh, a.v_ldp, a.v_ldt, p, X::KEYS * s + KW * wave);
#pragma unroll
            for (int i = 0; i < LI; ++i) {
                kr[i] = *reinterpret_cast<gc_u32x4*>(kp + (int64_t) (128 / CH * i) * a.k_ldt + k_lane);
                vr[i] = *reinterpret_cast<gc_u32x4*>(vp + (int64_t) (128 / CH * i) * a.v_ldt + v_lane);
            }
        };
        auto store = [&](auto BUF, int s, int p) __attribute__((always_inline)) {
            const int key0 = X::KEYS * s + KW * wave;
            // whether every row of the tile sees these keys; if not, V of keys that no row sees may hold anything and is
            // zeroed, and so are infinities and NaN, which a probability of 0 does not hide from the rows that do not see them
            const bool seen = p >= 0 && key0 + KW - 1 <= wk.pos0 + tile.first && (!a.window || key0 > wk.pos0 + tile.last - a.window) && key0 + KW <= a.cap;
            constexpr int buf = BUF;
            int flags = p >= 0 ? 1 : 0;
            if (!seen) {
                uint32_t f = 0;
#pragma unroll
                for (int i = 0; i < LI; ++i) {
                    const int key = key0 + st_row + 64 / CH * i;
                    const bool live = (key >= tile.lo) & (key < (p >= 0 ? tile.hi : 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x = live ? vr[i][e] : 0u, n = nonfinite2<T>(x);
                        f |= n;
                        vr[i][e] = x & ~n;
                    }
                }
                if (__any(f != 0u)) flags |= 2;
            }
#pragma unroll
            for (int i = 0; i < LI; ++i) {
                *reinterpret_cast<lu32x4*>(k_put + 2 * (buf * X::KEYS + 64 / CH * i) * X::K_LD) = kr[i];
                *reinterpret_cast<lu32x4*>(v_put + 2 * (buf * X::KEYS + 64 / CH * i) * X::V_LD) = vr[i];
            }
            if (lane == 0) sh.page[buf][wave] = flags;
        };
        auto compute = [&](auto BUF, int s) __attribute__((always_inline)) {
            constexpr int buf = BUF;
            const int k0 = X::KEYS * s;
            // nothing for this wave's rows in the step
            if (!rows_here || k0 > w_last || (a.window && k0 + X::KEYS - 1 <= w_first - a.window)) return;
            // of the step's four 16s of keys
            auto flags_of = [&](int i) __attribute__((always_inline)) {
                int f = sh.page[buf][i * (X::WAVES / 4)];
                if constexpr (X::WAVES == 8) f |= sh.page[buf][2 * i + 1];
                return __builtin_amdgcn_readfirstlane(f);
            };
            const int fl0 = flags_of(0), fl1 = flags_of(1), fl2 = flags_of(2), fl3 = flags_of(3);
            const bool whole = (fl0 & fl1 & fl2 & fl3 & 1) && k0 + X::KEYS - 1 <= w_first && (!a.window || k0 > w_last - a.window) && k0 + X::KEYS <= a.cap;
            // Two halves of 32 keys, each of scores, softmax and products with V; the matrix unit works on the second half's scores
            // while the first's exponentials are formed, and on the first's products while the second's are.
            Acc st[2][TH];
            u32x4 kf[TH][KS], pb[2][NB], vf[2][NB];
            auto read_k = [&](int y) __attribute__((always_inline)) {
#pragma unroll
                for (int t = 0; t < TH; ++t)
#pragma unroll
                    for (int c = 0; c < KS; ++c)
                        kf[t][c] = *reinterpret_cast<lu32x4*>(k_get + 2 * ((buf * X::KEYS + 32 * y + RW * t) * X::K_LD + X::KD * c));
            };
            auto read_v = [&](u32x4 (&f)[NB], int y, int d) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s16x4*) (v_get + 2 * ((buf * X::KEYS + 32 * y + X::key_of(8 * b + 4 * x)) * X::V_LD + RW * d))));
                        f[b][2 * x] = w[0];
                        f[b][2 * x + 1] = w[1];
                    }
            };
            auto scores = [&](int y) __attribute__((always_inline)) {
#pragma unroll
                for (int t = 0; t < TH; ++t) {
#pragma unroll
                    for (int i = 0; i < AE; ++i) st[y][t][i] = 0.f;
#pragma unroll
                    for (int c = 0; c < KS; ++c) st[y][t] = X::product(kf[t][c], q[c], st[y][t]);
                }
            };
            // masked scores; the factor by which the row's new maximum shrinks what was summed
            auto maximum = [&](int y) __attribute__((always_inline)) {
                if (!whole) {
                    const int end0 = (y ? fl2 : fl0) & 1 ? upto : -1, end1 = (y ? fl3 : fl1) & 1 ? upto : -1;
#pragma unroll
                    for (int e = 0; e < TH * AE; ++e) {
                        const int key = k0 + 32 * y + X::key_of(e) + 4 * hg;
                        const float x = st[y][e / AE][e % AE];
                        st[y][e / AE][e % AE] = ((key <= (X::key_of(e) < 16 ? end0 : end1)) & (key > from)) ? x : -INFINITY;
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < TH * AE; ++e) mx = fmaxf(mx, st[y][e / AE][e % AE]);
                mx = fmaxf(m, X::row_max(mx) * a.scale); // a.scale > 0
                const float c = exp2_fast(m - mx);
                m = mx;
                return c;
            };
            auto exponentials = [&](int y) __attribute__((always_inline)) {
                const float base = X::SHIFT - m;
                float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    typename Elem<T>::x8 p;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float x = exp2_fast(fmaf(st[y][(8 * b + j) / AE][(8 * b + j) % AE], a.scale, base));
                        ls[j & 3] += x;
                        p[j] = (T) x;
                    }
                    pb[y][b] = __builtin_bit_cast(u32x4, p);
                }
                return (ls[0] + ls[1]) + (ls[2] + ls[3]);
            };
            auto products = [&](int y, int d) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) o[d] = X::product(vf[d & 1][b], pb[y][b], o[d]);
            };
            auto shrink = [&](float c) __attribute__((always_inline)) {
                if (__any(c != 1.f)) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[d] *= c;
                }
            };
            read_k(0);
            __builtin_amdgcn_sched_barrier(0);          // all the reads go out first: left alone, each product waits for its own
            scores(0);
            read_k(1);
            const float c0 = maximum(0);
            shrink(c0);
            float l0 = exponentials(0);
            scores(1);
#pragma unroll
            for (int c = 0; c < TH * KS; ++c) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);       // a product, then what fills its time
                __builtin_amdgcn_sched_group_barrier(0x002, 4 * AE * TH / (TH * KS), 0);
            }
            here(pb[0][0], pb[0][NB - 1], l0);
            l = l * c0 + l0;
            const float c1 = maximum(1);
            read_v(vf[0], 0, 0);
            read_v(vf[1], 0, 1);
            float l1 = exponentials(1);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                products(0, d);
                if (d + 2 < DT) read_v(vf[d & 1], 0, d + 2);
                else read_v(vf[d & 1], 1, d + 2 - DT);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, 4 * NB, 0);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 4 * AE * TH / (DT * NB), 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, 2 * NB, 0);
            }
            here(pb[1][0], pb[1][NB - 1], l1);
            l = l * c1 + l1;
            shrink(c1);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                products(1, d);
                if (d + 2 < DT) read_v(vf[d & 1], 1, d + 2);
            }
            if ((fl0 | fl1 | fl2 | fl3) & 2) {
                // the infinities and NaN that were zeroed, added to the rows that see them
#pragma unroll 1
                for (int z = 0; z < X::KEYS; ++z) {
                    const int key = k0 + z, fl = z < 16 ? fl0 : z < 32 ? fl1 : z < 48 ? fl2 : fl3;
                    if (fl != 3 || key < tile.lo || key >= tile.hi) continue;
                    const int p = table[a.d_page.div((uint32_t) key)], in = key - (int) a.d_page.div((uint32_t) key) * a.page;
                    gc_u16* const vk = reinterpret_cast<gc_u16*>(as_global(vh) + ((int64_t) p * a.v_ldp + (int64_t) in * a.v_ldt) * 2);
                    // where the key's probability lies: result `reg` of a half's, in the lanes of group `in_group`
                    const int zz = z & 31, reg = RW == 32 ? 4 * (zz >> 3) + (zz & 3) : 4 * (zz >> 4) + (zz & 3), in_group = RW == 32 ? (zz >> 2) & 1 : (zz >> 2) & 3;
                    uint32_t pw = 0;
#pragma unroll
                    for (int w = 0; w < 8 * NB; ++w) pw = (z >> 5) * 4 * NB + (reg >> 1) == w ? pb[w / (4 * NB)][(w >> 2) % NB][w & 3] : pw;
                    pw = (uint32_t) __shfl((int) pw, RW * in_group + cr);
                    const float pr = (float) __builtin_bit_cast(T, (uint16_t) (reg & 1 ? pw >> 16 : pw)) * (z < 32 ? c1 : 1.f);
                    const uint32_t mask = ((key <= upto) & (key > from)) ? 0xFFFFu : 0u;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < AE; ++i) {
                            const uint32_t b = vk[X::col_of(d, i >> 2) + 4 * hg + (i & 3)];
                            o[d][i] += pr * (float) __builtin_bit_cast(T, (uint16_t) (b & mask & nonfinite2<T>(b)));
                        }
                }
            }
        };

        if (tile.lo < tile.hi) {
            int p0 = page_of(s0), p1 = page_of(s0 + 1), p2 = page_of(s0 + 2);
            request(s0, p0);
            store(std::integral_constant<int, 0>{}, s0, p0);
            if (s0 + 1 < s1) request(s0 + 1, p1);
            __syncthreads();
            // step s from one buffer, with step s + 1 into the other; false: it was the last
            auto turn = [&](auto BUF, int s) __attribute__((always_inline)) {
                compute(BUF, s);
                if (s + 1 == s1) return false;
                store(std::integral_constant<int, 1 - BUF>{}, s + 1, p1);
                p1 = p2;
                p2 = page_of(s + 3);
                if (s + 2 < s1) request(s + 2, p1);
                __syncthreads();
                return true;
            };
            for (int s = s0; turn(std::integral_constant<int, 0>{}, s) && turn(std::integral_constant<int, 1>{}, s + 1); s += 2) {}
        }

        // a wave's 32 rows, or their part
        const bool starts = off == 0, ends = off + n_steps == tile.steps;
        l = X::row_sum(l);
        // column tiles d0 .. d0 + N - 1 of the output
        auto put = [&](auto D0, auto N, const Acc* sum, float total) __attribute__((always_inline)) {
            if (xl < rows) {
                auto* const dst = as_global(a.out) + (int64_t) (wk.tok0 + tok) * a.o_ldt + (int64_t) (wk.h * a.group + xl - tok * a.group) * a.o_ldh + 4 * hg;
#pragma unroll
                for (int d = 0; d < N; ++d)
#pragma unroll
                    for (int i = 0; i < QD; ++i)
                        store_out<T>(dst + X::col_of(D0 + d, i), f32x4{sum[d][4 * i], sum[d][4 * i + 1], sum[d][4 * i + 2], sum[d][4 * i + 3]}, total);
            }
        };
        if (starts && ends) {
            put(std::integral_constant<int, 0>{}, std::integral_constant<int, DT>{}, o, l);
        } else {
            // A part moves as it lies in the registers (a lane's 16 bytes next to its neighbours').  The workgroup that
            // finds all others' parts written joins them with its own, in the order of the workgroups, and writes none.  Many
            // parts of few rows (drafts over a long context) are all written, and every thread of the last workgroup sums some
            // of the live rows' elements, eight parts in flight: where that takes less than half as many turns of waiting
            // (1.5 us each) as one part after the other.
            constexpr int Z = 2, B = 8;                // elements of a thread at once, parts in flight
            const int first_wg = wg - (int) (((uint32_t) off + per - 1u) / per);
            const int last_wg = wg + (int) (((uint32_t) (tile.steps - off - n_steps) + per - 1u) / per);
            const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(a.part, 0, (int) ATTN_PART_BYTES, RAW_BUFFER_FLAGS);
            // slot 2 c of workgroup c, 2 c + 1 for the tile's first
            auto slot = [&](int c) __attribute__((always_inline)) {
                return (2u * (uint32_t) c + (c == first_wg ? 1u : 0u)) * (uint32_t) (X::SLOT * 4) + (uint32_t) wave * (uint32_t) (X::SLOT * 4 / X::WAVES);
            };
            const uint32_t at = 16u * (uint32_t) lane, ml_at = (uint32_t) (QD * DT * 1024) + 8u * (uint32_t) lane;
            const int live_rows = min(X::ROWS, rows - wk.t * X::ROWS), quads = (live_rows + RW - 1) / RW * (QD * DT * 64);
            const int turns = (quads + Z * X::THREADS - 1) / (Z * X::THREADS) * ((last_wg - first_wg + B) / B);
            const bool few = 2 * turns > last_wg - first_wg;
            if (tid == 0) {
                sh.last = few && __hip_atomic_load(&a.counters[first_wg], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t) (last_wg - first_wg);
            }
            __syncthreads();
            bool mine = sh.last;
            if (!mine) {
                const uint32_t to = slot(wg);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < QD; ++i)
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]}), prs,
                                                               at + 1024u * (uint32_t) (QD * d + i), to, SC1);
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{(uint32_t) __float_as_int(m), (uint32_t) __float_as_int(l)}, prs, ml_at, to, SC1);
                __builtin_amdgcn_s_waitcnt(0x0F70);    // vmcnt(0): the part has landed
                __syncthreads();
                if (tid == 0)
                    sh.last = __hip_atomic_fetch_add(&a.counters[first_wg], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t) (last_wg - first_wg);
                __syncthreads();
                mine = sh.last;
            }
            if (mine) {
                if (tid == 0) __hip_atomic_store(&a.counters[first_wg], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (!few) {
                    for (int z0 = tid; z0 < quads; z0 += Z * X::THREADS) {
                        uint32_t from_wave[Z], at_quad[Z], at_ml[Z];
                        f32x4 sum[Z];
                        float top[Z], total[Z];
#pragma unroll
                        for (int i = 0; i < Z; ++i) {
                            const uint32_t z = (uint32_t) min(z0 + i * X::THREADS, quads - 1), w = z / (QD * DT * 64), r = z % (QD * DT * 64);
                            from_wave[i] = w * (uint32_t) (X::SLOT * 4 / X::WAVES);
                            at_quad[i] = from_wave[i] + 16u * r;
                            at_ml[i] = from_wave[i] + (uint32_t) (QD * DT * 1024) + 8u * (r & 63u);
                            sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                            top[i] = LOWEST;
                            total[i] = 0.f;
                        }
#pragma unroll 1
                        for (int c0 = first_wg; c0 <= last_wg; c0 += B) {
                            u32x2 ml[Z][B];
                            f32x4 v[Z][B];
#pragma unroll
                            for (int b = 0; b < B; ++b) {
                                const uint32_t fr = slot(min(c0 + b, last_wg)) - (uint32_t) wave * (uint32_t) (X::SLOT * 4 / X::WAVES);
#pragma unroll
                                for (int i = 0; i < Z; ++i) {
                                    ml[i][b] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(prs, at_ml[i], fr, SC1));
                                    v[i][b] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, at_quad[i], fr, SC1));
                                }
                            }
#pragma unroll
                            for (int i = 0; i < Z; ++i) {
                                float up = top[i];
#pragma unroll
                                for (int b = 0; b < B; ++b) up = fmaxf(up, __int_as_float((int) ml[i][b][0]));
                                const float f = exp2_fast(top[i] - up);
                                total[i] *= f;
                                sum[i] *= f;
                                top[i] = up;
#pragma unroll
                                for (int b = 0; b < B; ++b) {
                                    const float g = c0 + b <= last_wg ? exp2_fast(__int_as_float((int) ml[i][b][0]) - up) : 0.f;
                                    total[i] += g * __int_as_float((int) ml[i][b][1]);
                                    sum[i] += v[i][b] * g;
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < Z; ++i) {
                            const int z = z0 + i * X::THREADS, w = z / (QD * DT * 64), r = z % (QD * DT * 64), ln = r & 63, x = RW * w + ln % RW;
                            if (z >= quads || x >= live_rows) continue;
                            const int y = wk.t * X::ROWS + x, tk = (int) a.d_group.div((uint32_t) y);
                            store_out<T>(as_global(a.out) + (int64_t) (wk.tok0 + tk) * a.o_ldt + (int64_t) (wk.h * a.group + y - tk * a.group) * a.o_ldh +
                                             X::col_of(r / 64 / QD, r / 64 % QD) + 4 * (ln / RW), sum[i], total[i]);
                        }
                    }
                } else {
                // 64 registers of the output at a time: more would not fit beside the workgroup's own
                constexpr int N = DT * AE < 64 ? DT : 64 / AE;
                static_for(std::make_integer_sequence<int, DT / N>{}, [&](auto P) __attribute__((always_inline)) {
                    Acc sum[N];
                    float top = LOWEST, total = 0.f;
#pragma unroll
                    for (int d = 0; d < N; ++d)
#pragma unroll
                        for (int i = 0; i < AE; ++i) sum[d][i] = 0.f;
#pragma unroll 1
                    for (int c = first_wg; c <= last_wg; ++c) {
                        Acc x[N];
                        float mc = m, lc = l;
                        if (c == wg) {
#pragma unroll
                            for (int d = 0; d < N; ++d) x[d] = o[N * P + d];
                        } else {
                            const uint32_t fr = slot(c);
                            const u32x2 ml = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(prs, ml_at, fr, SC1));
#pragma unroll
                            for (int d = 0; d < N; ++d)
#pragma unroll
                                for (int i = 0; i < QD; ++i) {
                                    const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, at + 1024u * (uint32_t) (QD * (N * P + d) + i), fr, SC1));
#pragma unroll
                                    for (int e = 0; e < 4; ++e) x[d][4 * i + e] = v[e];
                                }
                            mc = __int_as_float((int) ml[0]);
                            lc = __int_as_float((int) ml[1]);
                        }
                        const float up = fmaxf(top, mc), f = exp2_fast(top - up), g = exp2_fast(mc - up);
                        total = total * f + lc * g;
                        top = up;
#pragma unroll
                        for (int d = 0; d < N; ++d) sum[d] = sum[d] * f + x[d] * g;
                    }
                    put(std::integral_constant<int, N * P>{}, std::integral_constant<int, N>{}, sum, total);
                });
                }
            }
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
    if (d == 64) hipLaunchKernelGGL((attn_prefill_kernel<T, 64>), dim3(Prefill<T, 64>::GRID), dim3(256), 0, s, a);
    else if (d == 128) hipLaunchKernelGGL((attn_prefill_kernel<T, 128>), dim3(Prefill<T, 128>::GRID), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_prefill_kernel<T, 256>), dim3(Prefill<T, 256>::GRID), dim3(512), 0, s, a);
}

}  // namespace

namespace exl3 {

void launch_attn_prefill(const AttnArgs& a, int dtype, int head_dim, hipStream_t s)
{
    dtype == EXL3_FP16 ? launch<f16>(a, head_dim, s) : launch<__bf16>(a, head_dim, s);
}

}  // namespace exl3
