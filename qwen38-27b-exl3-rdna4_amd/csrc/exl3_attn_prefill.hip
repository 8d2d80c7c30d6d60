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

// 128 rows a tile, 32 a wave, 64 keys a step.  K and V go through LDS once for the four waves: wave w requests keys
// 16 w .. + 15 of step s + 2 (one page: page sizes are multiples of 16) while step s is computed, and stores those of
// s + 1 into the other buffer after it, so a step has one barrier.
//   S^T = K Q^T (32x32x16): lane l gives key l & 31, elements 16 c + 8 (l >> 5) ..; its result holds row l & 31,
//         keys 8 (i >> 2) + 4 (l >> 5) + (i & 3)
//   O^T = V^T P^T: results 8 b .. 8 b + 7 are operand elements of 16 keys as they lie; V^T's lane gets the same keys by
//         transposing LDS reads (16 lanes read 4 keys x 16 columns, lane i gets column i of the 4)
// A lane's row is the same in S^T and O^T, as in the decode kernel.  LDS rows are padded, K's by 16 bytes so that 16
// keys' reads of one piece meet no bank twice, V's by 64 so that 4 keys' 64 bytes do not; padded rows, unlike permuted
// ones, let one address register and the instructions' offsets reach a whole step, and the two buffers are two copies of
// the loop's body for the same reason: the registers are all taken (output 64, Q 32, scores 32, K and V on the way 32).
template <class T, int D>
struct Prefill {
    static constexpr int ROWS = 128, KEYS = 64, WAVES = 4, THREADS = 256;
    static constexpr int GRID = D == 256 ? 256 : 512;   // workgroups: one or two a CU
    static constexpr int SLOT = attn_slot(ROWS, D + 2); // both halves of a wave hold its rows' maxima and sums
    static_assert(GRID <= ATTN_COUNTERS && (size_t) 2 * GRID * SLOT * 4 <= ATTN_PART_BYTES);
    static constexpr int LEAST = 4;                     // steps of a share at least
    static constexpr int CH = D / 8;                    // 16-byte pieces of a row
    static constexpr int LI = D / 32;                   // ... of a wave's 16 keys that a lane moves
    static constexpr int KS = D / 16;                   // products over D
    static constexpr int DT = D / 32;                   // column tiles of the output
    static constexpr float SHIFT = std::is_same_v<T, f16> ? 8.f : 0.f;   // fp16 probabilities are held times 2^8

    static constexpr int K_LD = D + 8, V_LD = D + 32;   // LDS rows, halves

    struct alignas(16) Shared {
        alignas(16) uint16_t k[2][KEYS * K_LD];
        alignas(16) uint16_t v[2][KEYS * V_LD];
        uint64_t find[WAVES + 4];
        alignas(16) int page[2][WAVES];                 // of a wave's 16 keys: 1 its page is one, 2 zeroed elements are to be added
        int last;
    };
};

template <class T, int D>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) attn_prefill_kernel(AttnArgs a)
{
    using X = Prefill<T, D>;
    constexpr int LI = X::LI, KS = X::KS, DT = X::DT, CH = X::CH;
    __shared__ typename X::Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, h2 = lane >> 5;
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

    // the lane's place in its wave's 16 keys: row st_row + 64 / CH i, piece st_piece
    const int st_row = lane / CH, st_piece = lane % CH;
    // transposing reads: key 4 h2 + tr_row of 8, columns 32 dt + 16 tr_half + 4 tr_q ..
    const int s16 = lane & 15, tr_row = s16 >> 2, tr_q = s16 & 3, tr_half = (lane >> 4) & 1;

    const uint32_t k_lane = (uint32_t) (st_row * (int) a.k_ldt + 8 * st_piece) * 2u, v_lane = (uint32_t) (st_row * (int) a.v_ldt + 8 * st_piece) * 2u;
    // LDS addresses of the lane's writes and reads: what the instructions' offsets are added to
    lchar* const k_put = (lchar*) &sh.k[0][(16 * wave + st_row) * X::K_LD + 8 * st_piece];
    lchar* const v_put = (lchar*) &sh.v[0][(16 * wave + st_row) * X::V_LD + 8 * st_piece];
    lchar* const k_get = (lchar*) &sh.k[0][c32 * X::K_LD + 8 * h2];
    lchar* const v_get = (lchar*) &sh.v[0][(4 * h2 + tr_row) * X::V_LD + 16 * tr_half + 4 * tr_q];

    while (true) {
        wk.settle();
        const AttnTile tile = wk.tile;
        const int n_steps = __builtin_amdgcn_readfirstlane((int) min((int64_t) (tile.steps - off), left));
        const int s0 = tile.step0 + off, s1 = s0 + n_steps, rows = wk.n * a.group;
        const int* const table = a.table + (int64_t) wk.r * a.ld_table;
        const char* const kh = reinterpret_cast<const char*>(a.k + (int64_t) wk.h * a.k_ldh);
        const char* const vh = reinterpret_cast<const char*>(a.v + (int64_t) wk.h * a.v_ldh);

        const int x0 = wk.t * X::ROWS + 32 * wave;      // the wave's first row
        const bool rows_here = x0 < rows;
        const int w_first = wk.pos0 + (int) a.d_group.div((uint32_t) x0), w_last = wk.pos0 + (int) a.d_group.div((uint32_t) (min(x0 + 32, rows) - 1));
        const int xl = x0 + c32, tok = (int) a.d_group.div((uint32_t) min(xl, rows - 1)), pos = xl < rows ? wk.pos0 + tok : -1;
        const int upto = min(pos, a.cap - 1), from = a.window ? pos - a.window : -1;
        u32x4 q[KS];
        {
            gc_u16* const src = as_global(a.q) + (int64_t) (wk.tok0 + tok) * a.q_ldt + (int64_t) (wk.h * a.group + min(xl, rows - 1) - tok * a.group) * a.q_ldh + 8 * h2;
#pragma unroll
            for (int c = 0; c < KS; ++c) q[c] = flipped(*reinterpret_cast<gc_u32x4*>(src + 16 * c), a.flip);
        }
        f32x16 o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
        float m = LOWEST, l = 0.f;

        auto page_of = [&](int s) __attribute__((always_inline)) {
            const int key = X::KEYS * s + 16 * wave;
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
            gc_char* const kp = keys_at(kh, a.k_ldp, a.k_ldt, p, X::KEYS * s + 16 * wave);
            gc_char* const vp = keys_at(vh, a.v_ldp, a.v_ldt, p, X::KEYS * s + 16 * wave);
#pragma unroll
            for (int i = 0; i < LI; ++i) {
                kr[i] = *reinterpret_cast<gc_u32x4*>(kp + (int64_t) (128 / CH * i) * a.k_ldt + k_lane);
                vr[i] = *reinterpret_cast<gc_u32x4*>(vp + (int64_t) (128 / CH * i) * a.v_ldt + v_lane);
            }
        };
        auto store = [&](auto BUF, int s, int p) __attribute__((always_inline)) {
            const int key0 = X::KEYS * s + 16 * wave;
            // whether every row of the tile sees these keys; if not, V of keys that no row sees may hold anything and is
            // zeroed, and so are infinities and NaN, which a probability of 0 does not hide from the rows that do not see them
            const bool seen = p >= 0 && key0 + 15 <= wk.pos0 + tile.first && (!a.window || key0 > wk.pos0 + tile.last - a.window) && key0 + 16 <= a.cap;
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
            const int fl0 = __builtin_amdgcn_readfirstlane(sh.page[buf][0]), fl1 = __builtin_amdgcn_readfirstlane(sh.page[buf][1]),
                      fl2 = __builtin_amdgcn_readfirstlane(sh.page[buf][2]), fl3 = __builtin_amdgcn_readfirstlane(sh.page[buf][3]);
            const bool whole = (fl0 & fl1 & fl2 & fl3 & 1) && k0 + X::KEYS - 1 <= w_first && (!a.window || k0 > w_last - a.window) && k0 + X::KEYS <= a.cap;
            // Two halves of 32 keys, each of scores, softmax and products with V; the matrix unit works on the second half's scores
            // while the first's exponentials are formed, and on the first's products while the second's are.
            f32x16 st[2];
            u32x4 kf[KS], pb[2][2], vf[2][2];
            auto read_k = [&](int y) __attribute__((always_inline)) {
#pragma unroll
                for (int c = 0; c < KS; ++c) kf[c] = *reinterpret_cast<lu32x4*>(k_get + 2 * ((buf * X::KEYS + 32 * y) * X::K_LD + 16 * c));
            };
            auto read_v = [&](u32x4 (&f)[2], int y, int d) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s16x4*) (v_get + 2 * ((buf * X::KEYS + 32 * y + 16 * b + 8 * x) * X::V_LD + 32 * d))));
                        f[b][2 * x] = w[0];
                        f[b][2 * x + 1] = w[1];
                    }
            };
            auto scores = [&](int y) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) st[y][i] = 0.f;
#pragma unroll
                for (int c = 0; c < KS; ++c) st[y] = mfma32<T>(kf[c], q[c], st[y]);
            };
            // masked scores; the factor by which the row's new maximum shrinks what was summed
            auto maximum = [&](int y) __attribute__((always_inline)) {
                if (!whole) {
                    const int end0 = (y ? fl2 : fl0) & 1 ? upto : -1, end1 = (y ? fl3 : fl1) & 1 ? upto : -1;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = k0 + 32 * y + 8 * (i >> 2) + 4 * h2 + (i & 3);
                        st[y][i] = ((key <= (i < 8 ? end0 : end1)) & (key > from)) ? st[y][i] : -INFINITY;
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[y][i]);
                float lo, hi;
                halves_x(mx, lo, hi);
                mx = fmaxf(m, fmaxf(lo, hi) * a.scale); // a.scale > 0
                const float c = exp2_fast(m - mx);
                m = mx;
                return c;
            };
            auto exponentials = [&](int y) __attribute__((always_inline)) {
                const float base = X::SHIFT - m;
                float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    typename Elem<T>::x8 p;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float x = exp2_fast(fmaf(st[y][8 * b + j], a.scale, base));
                        ls[j & 3] += x;
                        p[j] = (T) x;
                    }
                    pb[y][b] = __builtin_bit_cast(u32x4, p);
                }
                return (ls[0] + ls[1]) + (ls[2] + ls[3]);
            };
            auto products = [&](int y, int d) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < 2; ++b) o[d] = mfma32<T>(vf[d & 1][b], pb[y][b], o[d]);
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
            for (int c = 0; c < KS; ++c) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);       // a product, then what fills its time
                __builtin_amdgcn_sched_group_barrier(0x002, 60 / KS, 0);
            }
            here(pb[0][0], pb[0][1], l0);
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
            __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 30 / DT, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 30 / DT, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
            }
            here(pb[1][0], pb[1][1], l1);
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
                    const int reg = 4 * (z >> 3) + (z & 3);                    // of the 32 of st
                    uint32_t pw = 0;
#pragma unroll
                    for (int w = 0; w < 16; ++w) pw = reg >> 1 == w ? pb[w >> 3][(w >> 2) & 1][w & 3] : pw;
                    pw = (uint32_t) __shfl((int) pw, 32 * ((z >> 2) & 1) + c32);
                    const float pr = (float) __builtin_bit_cast(T, (uint16_t) (reg & 1 ? pw >> 16 : pw)) * (z < 32 ? c1 : 1.f);
                    const uint32_t mask = ((key <= upto) & (key > from)) ? 0xFFFFu : 0u;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const uint32_t b = vk[32 * d + 8 * (i >> 2) + 4 * h2 + (i & 3)];
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
        float lo, hi;
        halves_x(l, lo, hi);
        l = lo + hi;
        // column tiles d0 .. d0 + N - 1 of the output
        auto put = [&](auto D0, auto N, const f32x16* sum, float total) __attribute__((always_inline)) {
            if (xl < rows) {
                auto* const dst = as_global(a.out) + (int64_t) (wk.tok0 + tok) * a.o_ldt + (int64_t) (wk.h * a.group + xl - tok * a.group) * a.o_ldh + 4 * h2;
#pragma unroll
                for (int d = 0; d < N; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        store_out<T>(dst + 32 * (D0 + d) + 8 * i, f32x4{sum[d][4 * i], sum[d][4 * i + 1], sum[d][4 * i + 2], sum[d][4 * i + 3]}, total);
            }
        };
        if (starts && ends) {
            put(std::integral_constant<int, 0>{}, std::integral_constant<int, DT>{}, o, l);
        } else {
            // A part moves as it lies in the registers (a lane's 16 bytes of 16 d + 4 i .. next to its neighbours').  The workgroup that
            // finds all others' parts written joins them with its own, in the order of the workgroups, and writes none.
            const int first_wg = wg - (int) (((uint32_t) off + per - 1u) / per);
            const int last_wg = wg + (int) (((uint32_t) (tile.steps - off - n_steps) + per - 1u) / per);
            const __amdgpu_buffer_rsrc_t prs = __builtin_amdgcn_make_buffer_rsrc(a.part, 0, (int) ATTN_PART_BYTES, RAW_BUFFER_FLAGS);
            // slot 2 c of workgroup c, 2 c + 1 for the tile's first
            auto slot = [&](int c) __attribute__((always_inline)) {
                return (2u * (uint32_t) c + (c == first_wg ? 1u : 0u)) * (uint32_t) (X::SLOT * 4) + (uint32_t) wave * (uint32_t) (X::SLOT);
            };
            const uint32_t at = 16u * (uint32_t) lane, ml_at = (uint32_t) (4 * DT * 1024) + 8u * (uint32_t) lane;
            if (tid == 0) {
                sh.last = __hip_atomic_load(&a.counters[first_wg], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t) (last_wg - first_wg);
            }
            __syncthreads();
            bool mine = sh.last;
            if (!mine) {
                const uint32_t to = slot(wg);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]}), prs,
                                                               at + 1024u * (uint32_t) (4 * d + i), to, SC1);
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
                // four column tiles at a time: more would not fit beside the workgroup's own
                constexpr int N = DT < 4 ? DT : 4;
                static_for(std::make_integer_sequence<int, DT / N>{}, [&](auto P) __attribute__((always_inline)) {
                    f32x16 sum[N];
                    float top = LOWEST, total = 0.f;
#pragma unroll
                    for (int d = 0; d < N; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum[d][i] = 0.f;
#pragma unroll 1
                    for (int c = first_wg; c <= last_wg; ++c) {
                        f32x16 x[N];
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
                                for (int i = 0; i < 4; ++i) {
                                    const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(prs, at + 1024u * (uint32_t) (4 * (N * P + d) + i), fr, SC1));
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

template <class T>
void launch(const AttnArgs& a, int d, hipStream_t s)
{
    if (d == 64) hipLaunchKernelGGL((attn_prefill_kernel<T, 64>), dim3(Prefill<T, 64>::GRID), dim3(256), 0, s, a);
    else if (d == 128) hipLaunchKernelGGL((attn_prefill_kernel<T, 128>), dim3(Prefill<T, 128>::GRID), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_prefill_kernel<T, 256>), dim3(Prefill<T, 256>::GRID), dim3(256), 0, s, a);
}

}  // namespace

namespace exl3 {

void launch_attn_prefill(const AttnArgs& a, int dtype, int head_dim, hipStream_t s)
{
    dtype == EXL3_FP16 ? launch<f16>(a, head_dim, s) : launch<__bf16>(a, head_dim, s);
}

}  // namespace exl3
