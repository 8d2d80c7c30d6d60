// exl3_attn8_prefill.hip -- paged attention over a cache in 8 bits for many rows a request (prompt chunks), bound by the matrix
// products and the vector work beside them.
#include "exl3_attn8.h"

using namespace exl3;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char lchar;
typedef __attribute__((address_space(3))) u32x4 lu32x4;
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// values formed by here: they would be sunk to their first use, past the products that they are to run beside
__device__ __forceinline__ void here(u32x4& a, u32x4& b, float& c)
{
    asm volatile("" : "+v"(a), "+v"(b), "+v"(c));
}

// The 16-bit cache's chunk kernel with codes made fp16 numbers on their way into LDS (1.25 operations a code, once for all of the
// tile's waves), and a factor and an exponent for each 16 keys (exl3_attn8.hip: the formulas).  64 keys a step: a wave requests its
// keys (of one block: it has 8 or 16 of them) of step s + 2 while step s is computed, and stores those of s + 1 into the other
// buffer after it, so a step has one barrier.  Heads of 64 and 128: 32 rows a wave,
//   S^T = K Q^T (32x32x16): lane l gives key l & 31, elements 16 c + 8 (l >> 5) ..; its result holds row l & 31,
//         keys 8 (i >> 2) + 4 (l >> 5) + (i & 3)
//   O^T = V^T P^T: results 8 b .. 8 b + 7 are operand elements of 16 keys (a block) as they lie; V^T's lane gets the same keys by
//         transposing LDS reads (16 lanes read 4 keys x 16 columns, lane i gets column i of the 4)
// Heads of 256: 16 rows a wave (16x16x32, row l & 15, keys 4 (l >> 4) + (i & 3) of two blocks).
// A lane's row is the same in S^T and O^T.  LDS rows are padded so that no bank is met twice.
// 2048 tokens over 12000, 40 heads over 8 of 128 (546 GFLOP): 640 us, 853 TFLOPS, bound by products and vector work that
// overlap little, and waits.  1501 over 9001, 24 over 4 of 256 (360 GFLOP): 495 us, 727 TFLOPS, bound by LDS reads (16 rows a wave).  Not kept:
// the step's halves pipelined over steps 826, two groups of four waves that take products and vector work in turn 729, the next step's
// codes stored beside the last products 796 (spills); 32 rows a wave for heads of 256 (one wave a SIMD, spills) 703.
template <class T, int D, int W>
struct Prefill8 {
    static constexpr int RW = D == 256 ? 16 : 32;       // rows of a wave
    static constexpr int WAVES = W, ROWS = RW * WAVES, KEYS = 64, THREADS = 64 * WAVES;
    static constexpr int GRID = THREADS == 512 ? 256 : 512;             // workgroups: one or two a CU
    static constexpr int SLOT = attn_slot(ROWS, D + 128 / RW - 2); // every lane's maximum and sum, also where lanes share a row
    // two counters a workgroup: of the tile that it begins, and of the group of its parts that it begins
    static_assert(GRID <= ATTN_COUNTERS / 2 && (size_t) 2 * GRID * SLOT * 4 <= ATTN_PART_BYTES);
    static constexpr int LEAST = 4;                     // steps of a share at least
    static constexpr int CH = D / 8;                    // 8-code pieces of a row
    static constexpr int KW = KEYS / WAVES;             // keys that a wave moves
    static constexpr int LI = KW * CH / 64;             // ... pieces of them a lane
    static constexpr int KD = RW == 32 ? 16 : 32;       // columns of K that a product takes
    static constexpr int KS = D / KD;                   // products over D
    static constexpr int DT = D / RW;                   // column tiles of the output
    static constexpr int AE = RW == 32 ? 16 : 4;        // results of a product a lane
    static constexpr int TH = 32 / RW;                  // key tiles of a half step (32 keys)
    static constexpr int NB = AE * TH / 8;              // operands of its probabilities
    static constexpr int HALF = TH * AE / 2;            // a lane's results of each of its two blocks
    static constexpr int VD = RW == 32 ? 2 : 4;         // column tiles of V on their way from LDS (two of heads of 256: 4 % slower)
    using Acc = std::conditional_t<RW == 32, f32x16, f32x4>;
    static constexpr float SHIFT = 8.f;                 // probabilities are held times 2^8
    static constexpr int K_LD = D + 8, V_LD = RW == 32 ? D + 32 : D + 16;  // LDS rows, halves
    static_assert(C8_BLOCK % KW == 0);

    struct alignas(16) Shared {
        alignas(16) uint16_t k[2][KEYS * K_LD];
        alignas(16) uint16_t v[2][KEYS * V_LD];
        uint64_t find[WAVES + 4];
        alignas(16) f32x4 block[2][WAVES];              // of a wave's keys: K's scale, V's logarithm, 1 / V's, 1 if their page is one
        int last;
    };
    static __device__ __forceinline__ Acc product(u32x4 a, u32x4 b, Acc c)
    {
        if constexpr (RW == 32) return mfma32(a, b, c);
        else return mfma16<f16>(a, b, c);
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
    // The columns of K and Q that lanes of group hg have in product c are q_col(hg) + Q_STEP c and the 7 after them; any order of D
    // does.  16 lanes' 16-byte LDS reads pass at once, of two groups where a group has 16: theirs lie 128 columns (all
    // banks) apart.
    static constexpr int Q_STEP = RW == 32 ? 16 : 8;
    static __device__ __forceinline__ int q_col(int hg) { return RW == 32 ? 8 * hg : 128 * (hg & 1) + 64 * (hg >> 1); }
};

template <class T, int D, int W>
__global__ void __launch_bounds__((Prefill8<T, D, W>::THREADS), (Prefill8<T, D, W>::THREADS == 256 ? 2 : 1)) attn8_prefill_kernel(Attn8Args a)
{
    using X = Prefill8<T, D, W>;
    using Acc = typename X::Acc;
    constexpr int LI = X::LI, KS = X::KS, DT = X::DT, CH = X::CH, RW = X::RW, KW = X::KW, AE = X::AE, TH = X::TH, NB = X::NB, HALF = X::HALF, VD = X::VD, QD = AE / 4;
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

    const uint32_t k_lane = (uint32_t) (st_row * (int) a.c.k_ldt + 8 * st_piece), v_lane = (uint32_t) (st_row * (int) a.c.v_ldt + 8 * st_piece);
    // LDS addresses of the lane's writes and reads: what the instructions' offsets are added to
    lchar* const k_put = (lchar*) &sh.k[0][(KW * wave + st_row) * X::K_LD + 8 * st_piece];
    lchar* const v_put = (lchar*) &sh.v[0][(KW * wave + st_row) * X::V_LD + 8 * st_piece];
    lchar* const k_get = (lchar*) &sh.k[0][cr * X::K_LD + X::q_col(hg)];
    lchar* const v_get = (lchar*) &sh.v[0][(4 * hg + tr_row) * X::V_LD + 16 * tr_half + 4 * tr_q];

    while (true) {
        wk.settle();
        const AttnTile tile = wk.tile;
        const int n_steps = __builtin_amdgcn_readfirstlane((int) min((int64_t) (tile.steps - off), left));
        const int s0 = tile.step0 + off, s1 = s0 + n_steps, rows = wk.n * a.group;
        const int* const table = a.table + (int64_t) wk.r * a.ld_table;
        const int8_t* const kh = a.c.k + (int64_t) wk.h * a.c.k_ldh;
        const int8_t* const vh = a.c.v + (int64_t) wk.h * a.c.v_ldh;
        const float* const ksh = a.c.ks + (int64_t) wk.h * a.c.ks_ldh;
        const float* const vsh = a.c.vs + (int64_t) wk.h * a.c.vs_ldh;

        const int x0 = wk.t * X::ROWS + RW * wave;      // the wave's first row
        const bool rows_here = x0 < rows;
        const int w_first = wk.pos0 + (int) a.d_group.div((uint32_t) x0), w_last = wk.pos0 + (int) a.d_group.div((uint32_t) (min(x0 + RW, rows) - 1));
        const int xl = x0 + cr, tok = (int) a.d_group.div((uint32_t) min(xl, rows - 1)), pos = xl < rows ? wk.pos0 + tok : -1;
        const int upto = min(pos, a.cap - 1), from = a.window ? pos - a.window : -1;
        u32x4 q[KS];
        {
            gc_u16* const src = as_global(a.q) + (int64_t) (wk.tok0 + tok) * a.q_ldt + (int64_t) (wk.h * a.group + min(xl, rows - 1) - tok * a.group) * a.q_ldh + X::q_col(hg);
#pragma unroll
            for (int c = 0; c < KS; ++c) q[c] = flipped(*reinterpret_cast<gc_u32x4*>(src + X::Q_STEP * c), a.flip);
        }
        const float row_scale = row_scale_of(a.scale, fp16_rows<T>(q, [](float x) __attribute__((always_inline)) { return X::row_max(x); }));
        Acc o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < AE; ++i) o[d][i] = 0.f;
        float m = LOWEST, l = 0.f;

        // every row of the wave sees every key of the steps whose first keys are whole_from .. whole_to, if their pages are pages
        const int whole_from = a.window ? w_last - a.window + 1 : 0, whole_to = min(w_first - (X::KEYS - 1), a.cap - X::KEYS);
        // a page is looked up a step before it is needed: a wait for it would be a trip to memory each step
        auto look_up = [&](int s) __attribute__((always_inline)) {
            const int key = X::KEYS * s + KW * wave;
            return key < tile.hi ? table[a.d_page.div((uint32_t) key)] : -1;
        };
        auto page_of = [&](int looked_up) __attribute__((always_inline)) {
            const int p = __builtin_amdgcn_readfirstlane(looked_up);
            return (unsigned) p >= (unsigned) a.pages ? -1 : p;
        };
        u32x2 kr[LI], vr[LI];
        float skr, svr;
        auto request = [&](int s, int p) __attribute__((always_inline)) {
            const int key = X::KEYS * s + KW * wave, in = key - (int) a.d_page.div((uint32_t) key) * a.page, pg = max(p, 0);
            auto* const kp = as_global(kh) + ((int64_t) pg * a.c.k_ldp + (int64_t) in * a.c.k_ldt);
            auto* const vp = as_global(vh) + ((int64_t) pg * a.c.v_ldp + (int64_t) in * a.c.v_ldt);
#pragma unroll
            for (int i = 0; i < LI; ++i) {
                kr[i] = *reinterpret_cast<gc_u32x2*>(kp + (int64_t) (64 / CH * i) * a.c.k_ldt + k_lane);
                vr[i] = *reinterpret_cast<gc_u32x2*>(vp + (int64_t) (64 / CH * i) * a.c.v_ldt + v_lane);
            }
            skr = *as_global(ksh + (int64_t) pg * a.c.ks_ldp + (int64_t) (in / C8_BLOCK) * a.c.ks_ldb);
            svr = *as_global(vsh + (int64_t) pg * a.c.vs_ldp + (int64_t) (in / C8_BLOCK) * a.c.vs_ldb);
        };
        auto halves = [&](u32x2 w) __attribute__((always_inline)) {
            const uint32_t w0 = w[0] ^ C8_FLIP, w1 = w[1] ^ C8_FLIP;
            return u32x4{codes2(w0, 0), codes2(w0, 1), codes2(w1, 0), codes2(w1, 1)};
        };
        auto store = [&](auto BUF, int s, int p) __attribute__((always_inline)) {
            constexpr int buf = BUF;
#pragma unroll
            for (int i = 0; i < LI; ++i) {
                *reinterpret_cast<lu32x4*>(k_put + 2 * (buf * X::KEYS + 64 / CH * i) * X::K_LD) = halves(kr[i]);
                *reinterpret_cast<lu32x4*>(v_put + 2 * (buf * X::KEYS + 64 / CH * i) * X::V_LD) = halves(vr[i]);
            }
            const float lv = log2_fast(scale8(svr));
            if (lane == 0) sh.block[buf][wave] = f32x4{scale8(skr), lv, exp2_fast(-lv), p >= 0 ? 1.f : 0.f};
        };
        auto compute = [&](auto BUF, int s) __attribute__((always_inline)) {
            constexpr int buf = BUF;
            const int k0 = X::KEYS * s;
            // nothing for this wave's rows in the step
            if (!rows_here || k0 > w_last || (a.window && k0 + X::KEYS - 1 <= w_first - a.window)) return;
            // of the step's four blocks
            f32x4 bl[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) bl[i] = sh.block[buf][i * (X::WAVES / 4)];
            const int pages = __builtin_amdgcn_readfirstlane(__float_as_int(fminf(fminf(bl[0][3], bl[1][3]), fminf(bl[2][3], bl[3][3]))));
            const bool whole = (int) (pages != 0) & (int) (k0 >= whole_from) & (int) (k0 <= whole_to);
            // Two halves of 32 keys, each of scores, softmax and products with V; the matrix unit works on the second half's scores
            // while the first's exponentials are formed, and on the first's products while the second's are.
            Acc st[2][TH];
            u32x4 kf[TH][KS], pb[2][NB], vf[VD][NB];
            auto read_k = [&](int y) __attribute__((always_inline)) {
#pragma unroll
                for (int t = 0; t < TH; ++t)
#pragma unroll
                    for (int c = 0; c < KS; ++c)
                        kf[t][c] = *reinterpret_cast<lu32x4*>(k_get + 2 * ((buf * X::KEYS + 32 * y + RW * t) * X::K_LD + X::Q_STEP * c));
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
            float f[2][2];
            auto maximum = [&](int y) __attribute__((always_inline)) {
                if (!whole) {
                    const int end0 = bl[2 * y][3] != 0.f ? upto : -1, end1 = bl[2 * y + 1][3] != 0.f ? upto : -1;
#pragma unroll
                    for (int e = 0; e < TH * AE; ++e) {
                        const int key = k0 + 32 * y + X::key_of(e) + 4 * hg;
                        const float x = st[y][e / AE][e % AE];
                        st[y][e / AE][e % AE] = ((key <= (e < HALF ? end0 : end1)) & (key > from)) ? x : -INFINITY;
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float top = -INFINITY;
#pragma unroll
                    for (int e = b * HALF; e < (b + 1) * HALF; ++e) top = fmaxf(top, st[y][e / AE][e % AE]);
                    f[y][b] = fmaxf(row_scale * bl[2 * y + b][0], 1e-37f);  // above 0: a masked score's infinity stays one
                    mx = fmaxf(mx, fmaf(top, f[y][b], bl[2 * y + b][1]));
                }
                mx = fmaxf(m, X::row_max(mx));
                const float c = exp2_fast(m - mx);
                m = mx;
                return c;
            };
            auto exponentials = [&](int y) __attribute__((always_inline)) {
                float ls[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
                const float base[2] = {X::SHIFT - m + bl[2 * y][1], X::SHIFT - m + bl[2 * y + 1][1]};
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    f16x8 p;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int e = 8 * b + j, z = e < HALF ? 0 : 1;
                        const float x = exp2_fast(fmaf(st[y][e / AE][e % AE], f[y][z], base[z]));
                        ls[z][j & 1] += x;
                        p[j] = (f16) x;
                    }
                    pb[y][b] = __builtin_bit_cast(u32x4, p);
                }
                return (ls[0][0] + ls[0][1]) * bl[2 * y][2] + (ls[1][0] + ls[1][1]) * bl[2 * y + 1][2];
            };
            auto products = [&](int y, int d) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) o[d] = X::product(vf[d % VD][b], pb[y][b], o[d]);
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
#pragma unroll
            for (int d = 0; d < VD; ++d) read_v(vf[d], 0, d);
            float l1 = exponentials(1);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                products(0, d);
                if (d + VD < DT) read_v(vf[d % VD], 0, d + VD);
                else read_v(vf[d % VD], 1, d + VD - DT);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * VD * NB, 0);
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
                if (d + VD < DT) read_v(vf[d % VD], 1, d + VD);
            }
        };

        if (tile.lo < tile.hi) {
            const int p0 = page_of(look_up(s0));
            int p1 = page_of(look_up(s0 + 1)), next = look_up(s0 + 2);
            request(s0, p0);
            store(std::integral_constant<int, 0>{}, s0, p0);
            if (s0 + 1 < s1) request(s0 + 1, p1);
            __syncthreads();
            // step s from one buffer, with step s + 1 into the other; false: it was the last
            auto turn = [&](auto BUF, int s) __attribute__((always_inline)) {
                compute(BUF, s);
                if (s + 1 == s1) return false;
                store(std::integral_constant<int, 1 - BUF>{}, s + 1, p1);
                p1 = page_of(next);
                next = look_up(s + 3);
                if (s + 2 < s1) request(s + 2, p1);
                __syncthreads();
                return true;
            };
            for (int s = s0; turn(std::integral_constant<int, 0>{}, s) && turn(std::integral_constant<int, 1>{}, s + 1); s += 2) {}
        }

        // Arguments read anew, and indexes formed anew: kept in registers through the steps, what the join needs pushes out what they need
        // (2048 tokens over 12000, heads of 256: 922 us instead of 874).
        auto* args = (__attribute__((address_space(4))) const Attn8Args*) __builtin_amdgcn_kernarg_segment_ptr();
        int wg_here = wg, tid_here = tid;
        asm volatile("" : "+s"(args), "+s"(wg_here), "+v"(tid_here));
        const int wg = wg_here, tid = tid_here, lane = tid & 63;
        const UDiv d_group{args->d_group.m, args->d_group.s1, args->d_group.s2};
        const int64_t o_ldt = args->o_ldt, o_ldh = args->o_ldh;
        uint16_t* const out = args->out;
        uint32_t* const counters = args->counters;
        const int group_heads = args->group;
        // a wave's 32 rows, or their part
        const bool starts = off == 0, ends = off + n_steps == tile.steps;
        l = X::row_sum(l);
        // column tiles d0 .. d0 + N - 1 of the output
        auto put = [&](auto D0, auto N, const Acc* sum, float total) __attribute__((always_inline)) {
            if (xl < rows) {
                auto* const dst = as_global(out) + (int64_t) (wk.tok0 + tok) * o_ldt + (int64_t) (wk.h * group_heads + xl - tok * group_heads) * o_ldh + 4 * hg;
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
            // A part moves as it lies in the registers (a lane's 16 bytes next to its neighbours').  Few parts of many rows: the workgroup
            // that finds all others' parts written joins them with its own, in the order of the workgroups, and writes none.
            // Else all are written, and every thread of a last workgroup sums some of the live rows' elements, eight parts in flight:
            // where that takes less than half as many turns of waiting (2 us each) as there are parts (1 us each one after the other).  So
            // do two levels, as in the decode kernel (exl3_attn8.hip), with its slots and counters: one request of 40 rows over 100000
            // tokens 103 us against 129, over one kv head 74 against 316, but 640 rows over 8000 84 against 60.  (They cost long chunks 1 to 2 %.)
            constexpr int Z = 2, B = 8;                // elements of a thread at once, parts in flight
            const int first_wg = wg - (int) (((uint32_t) off + per - 1u) / per);
            const int last_wg = wg + (int) (((uint32_t) (tile.steps - off - n_steps) + per - 1u) / per), n = last_wg - first_wg + 1;
            const int live_rows = min(X::ROWS, rows - wk.t * X::ROWS), quads = (live_rows + RW - 1) / RW * (QD * DT * 64);
            const int turns = (quads + Z * X::THREADS - 1) / (Z * X::THREADS);        // of waiting, for B parts
            const int sizes = n <= 64 ? 8 : n <= 256 ? 16 : 24, waits = (sizes + B - 1) / B + ((n + sizes - 1) / sizes + B - 1) / B;
            const bool two = 2 * turns * waits < n && waits < (n + B - 1) / B;
            const int size = two ? sizes : n, groups = (n + size - 1) / size, group = (wg - first_wg) / size;
            const int begin_wg = first_wg + group * size, in_group = min(size, last_wg + 1 - begin_wg);
            const bool few = !two && 2 * turns * ((n + B - 1) / B) >= n;
            const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(args->part, 0, (int) ATTN_PART_BYTES, RAW_BUFFER_FLAGS);
            // slot 2 c of workgroup c, 2 c + 1 for the tile's first; bytes
            auto slot = [&](int c) __attribute__((always_inline)) { return (2u * (uint32_t) c + (c == first_wg ? 1u : 0u)) * (uint32_t) (X::SLOT * 4); };
            auto joined = [&](int g) __attribute__((always_inline)) {
                const int c = first_wg + g * size;
                return c == last_wg ? slot(c) : (2u * (uint32_t) (g ? c : c + 1) + 1u) * (uint32_t) (X::SLOT * 4);
            };
            const uint32_t my_wave = (uint32_t) wave * (uint32_t) (X::SLOT * 4 / X::WAVES);
            const uint32_t at = 16u * (uint32_t) lane, ml_at = (uint32_t) (QD * DT * 1024) + 8u * (uint32_t) lane;
            uint32_t* const counter = &counters[first_wg];
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
            if (tid == 0) {
                sh.last = few && __hip_atomic_load(counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t) (n - 1);
                if (sh.last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            bool mine = sh.last;
            if (!mine) {
                const uint32_t to = slot(wg) + my_wave;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < QD; ++i)
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]}), prs,
                                                               at + 1024u * (uint32_t) (QD * d + i), to, SC1);
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{(uint32_t) __float_as_int(m), (uint32_t) __float_as_int(l)}, prs, ml_at, to, SC1);
                // (a group of one has no counter: that of its workgroup may be the next tile's)
                if (groups > 1) mine = in_group == 1 || i_am_last(&counters[ATTN_COUNTERS / 2 + begin_wg], in_group);
                else mine = i_am_last(counter, n);
            }
            if (mine && !few) {
#pragma unroll 1
                for (bool last = groups == 1 || in_group == 1;; last = true) {
                    if (last && groups > 1 && !i_am_last(counter, groups)) break;
                    const int parts = !last ? in_group : groups > 1 ? groups : n;
                    const uint32_t to = joined(group);
                    for (int z0 = tid; z0 < quads; z0 += Z * X::THREADS) {
                        uint32_t at_quad[Z], at_ml[Z];
                        f32x4 sum[Z];
                        float top[Z], total[Z];
#pragma unroll
                        for (int i = 0; i < Z; ++i) {
                            const uint32_t z = (uint32_t) min(z0 + i * X::THREADS, quads - 1), w = z / (QD * DT * 64), r = z % (QD * DT * 64);
                            const uint32_t from_wave = w * (uint32_t) (X::SLOT * 4 / X::WAVES);
                            at_quad[i] = from_wave + 16u * r;
                            at_ml[i] = from_wave + (uint32_t) (QD * DT * 1024) + 8u * (r & 63u);
                            sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                            top[i] = LOWEST;
                            total[i] = 0.f;
                        }
#pragma unroll 1
                        for (int c0 = 0; c0 < parts; c0 += B) {
                            u32x2 ml[Z][B];
                            f32x4 v[Z][B];
#pragma unroll
                            for (int b = 0; b < B; ++b) {
                                const int c = min(c0 + b, parts - 1);
                                const uint32_t fr = last && groups > 1 ? joined(c) : slot(begin_wg + c);
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
                                    const float g = c0 + b < parts ? exp2_fast(__int_as_float((int) ml[i][b][0]) - up) : 0.f;
                                    total[i] += g * __int_as_float((int) ml[i][b][1]);
                                    sum[i] += v[i][b] * g;
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < Z; ++i) {
                            const int z = z0 + i * X::THREADS, w = z / (QD * DT * 64), r = z % (QD * DT * 64), ln = r & 63, x = RW * w + ln % RW;
                            if (z >= quads) continue;
                            if (!last) {
                                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum[i]), prs, at_quad[i], to, SC1);
                                if (r < 64)
                                    __builtin_amdgcn_raw_buffer_store_b64(u32x2{(uint32_t) __float_as_int(top[i]), (uint32_t) __float_as_int(total[i])}, prs, at_ml[i], to, SC1);
                            } else if (x < live_rows) {
                                const int y = wk.t * X::ROWS + x, tk = (int) d_group.div((uint32_t) y);
                                store_out<T>(as_global(out) + (int64_t) (wk.tok0 + tk) * o_ldt + (int64_t) (wk.h * group_heads + y - tk * group_heads) * o_ldh +
                                                 X::col_of(r / 64 / QD, r / 64 % QD) + 4 * (ln / RW), sum[i], total[i]);
                            }
                        }
                    }
                    if (last) break;
                }
            } else if (mine) {
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
                            const uint32_t fr = slot(c) + my_wave;
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
        __syncthreads();
        left -= n_steps;
        if (left <= 0) break;
        off = 0;
        wk.next();
    }
}

template <class T, int D, int W>
void launch_one(const Attn8Args& a, hipStream_t s)
{
    using X = Prefill8<T, D, W>;
    hipLaunchKernelGGL((attn8_prefill_kernel<T, D, W>), dim3(X::GRID), dim3(X::THREADS), 0, s, a);
}

template <class T>
void launch(const Attn8Args& a, int64_t rows, hipStream_t s)
{
    // Many rows: 256 a tile, whose keys are made fp16 once for eight waves instead of four (2048 tokens over 12000, 40 heads over 8 of
    // 128: 643 us against 732; 512 over none 42 against 37).  Heads of 64 gain as much over a long context (362 against 419, one after the other) but
    // lose without one (512 tokens 26 against 24) and in small chunks beside decodes (32 against 30).
    if (a.c.d == 64) launch_one<T, 64, 4>(a, s);
    else if (a.c.d == 256) launch_one<T, 256, 8>(a, s);
    else if (rows > 4096) launch_one<T, 128, 8>(a, s);
    else launch_one<T, 128, 4>(a, s);
}

}  // namespace

namespace exl3 {

void launch_attn8_prefill(const Attn8Args& a, int64_t rows, int dtype, hipStream_t s)
{
    dtype == EXL3_FP16 ? launch<f16>(a, rows, s) : launch<__bf16>(a, rows, s);
}

}  // namespace exl3
