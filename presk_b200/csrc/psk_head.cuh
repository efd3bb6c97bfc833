// The loss at the end of a language model, taken through the head in pieces of the vocabulary (PSK_OP_HEAD_XENT,
// PSK_OP_HEAD_DISTILL and their _VJP): the logits l = x·w exist only as accumulators in tensor memory and registers.
//
// Forward. One pass over the vocabulary: a tile of 128 rows by 256 classes is multiplied on the tensor cores, and its
// epilogue reduces each row's 128 columns a thread to a maximum m and z = sum of 2^((l - m)·c), c = log2 e / τ, which
// k_head_join puts together over the tiles: ln sum exp(l / τ) = M / τ + ln sum z·2^((m - M)·c).
// The targets' logits are picked out of the same registers. Backward. The tile is multiplied again, the epilogue
// writes g = ct/τ (2^(l·c - lse) - p) of a piece of the vocabulary, and two more products give dx and dw from it.
//
// Why the sums are kept twice. tcgen05 adds into its f32 accumulator by truncation: measured here, a sum of 4096
// products comes out 4.4e-6 (products of both signs) to 1.4e-5 (of one sign) too small, always towards zero, where a
// loss is the difference of two logits. So the accumulator holds `chunk` steps of the summed axis only, and the
// epilogue's threads add it, rounded to nearest, into registers while the next chunk runs in the other accumulator.
//
// Types. bf16 and binary16 operands are multiplied as they are. f32 operands are two binary16 planes, hi + lo, 22 bits
// of the number, of which three partial products are taken (lo·lo is below 2^-22 of the product): half the tensor
// work of three bf16 planes and their six products, which this was first (333 us at 2044 x 1024 x 16384, against
// 183 us). Binary16's range is met by powers of two: w is scaled by its greatest |element|, x by a row's, g by the greatest
// |ct|, each to the top of the range, 2^14 to 2^15, so that what falls below 2^-24 there is 2^-39 of the greatest.
// g itself is kept in binary16 for f32 and, for many rows, for bf16 operands too, x and w being copied into it (exactly:
// eight bits into eleven): g in bf16 would cost its 2^-9 an entry, as much again as the result's own rounding.
#pragma once
#include <utility>
#include "psk_dev.cuh"
#include "psk_gemm_tc.cuh"

namespace psk {
namespace head {

constexpr int BM = 128, BN = 256, BK = 64;
// Three warpgroups: warp 0 issues the TMA loads, warp 1 the products (2 and 3 idle); warps 4 to 11 are the epilogue, two
// a quadrant of tensor memory, 128 columns each. An epilogue thread keeps its 128 sums in registers, so the first
// warpgroup gives most of its share up: 128·40 + 256·232 = 384·168, what the block is launched with.
constexpr int THREADS = 384;
constexpr int REGS_FEW = 40, REGS_MANY = 232, REGS_LAUNCH = 168;
static_assert(128 * REGS_FEW + 256 * REGS_MANY <= THREADS * REGS_LAUNCH, "setmaxnreg waits for registers that the block does not have");
// MT: 128-row halves of a CTA's tile. One, with the two accumulators taking turns, for sums kept in registers; two,
// both multiplying the same tile of b (a third fewer bytes from the L2 a product), for the plain products dx and dw.
template <int MT>
struct Cfg {
    static constexpr int STAGES = MT == 1 ? 4 : 3;
    static constexpr int A_BYTES = MT * BM * BK * 2, B_BYTES = BN * BK * 2;
    static constexpr int TILE_BYTES = STAGES * (A_BYTES + B_BYTES);
    static constexpr int STAGE_OUT = 8 * 32 * 128;
    static constexpr int SMEM_TOTAL = TILE_BYTES + 256 + STAGE_OUT + 1024;
};
constexpr int COLS = 128; // columns of a tile an epilogue thread holds

enum { MODE_STATS = 0, MODE_GRAD = 1, MODE_OUT = 2 };

// Planes of the partial product q of two operands of two planes: hi·hi, hi·lo, lo·hi.
PSK_DEV int plane_a(int q) { return q == 2; }
PSK_DEV int plane_b(int q) { return q == 1; }

// The greatest finite |element| of the operands, as f32 bits (0: not scaled), and the powers of two made of them.
struct Scales {
    uint32_t max_x, max_w, max_ct, pad;
};

// 2^e as an f32, e within its normal range.
PSK_DEV float pow2(int e) { return __uint_as_float((uint32_t)(127 + (e < -126 ? -126 : e > 127 ? 127 : e)) << 23); }

// The exponent of the power of two that brings a maximum into [2^14, 2^15); 0 for none.
PSK_DEV int scale_of(uint32_t max_bits)
{
    const int e = (int)(max_bits >> 23);
    if (max_bits == 0) return 0;
    const int k = 14 + 127 - (e == 0 ? 1 : e);
    return k > 60 ? 60 : k; // 1/(g·w) and 1/(g·x) are f32 numbers then
}

enum { UN_NONE = 0, UN_DX = 1, UN_DW = 2 }; // what a product's sums are multiplied by: 1, 1/(g·w), 1/(g·x)
PSK_DEV float undo(const Scales *s, int un)
{
    if (!s || un == UN_NONE) return 1.0f;
    return pow2(-scale_of(s->max_ct) - scale_of(un == UN_DX ? s->max_w : s->max_x));
}

struct Params {
    int64_t m, n;                 // rows and columns of the product
    int64_t tiles_m, tiles_n, splits, panel;
    int32_t kb_k, nprod;          // blocks of 64 along the summed axis; partial products a block (1, or 3 of two planes)
    int32_t kb_split;             // blocks of the summed axis a split
    int32_t chunk;                // steps (block, partial product) in one accumulator before it is added into registers
    int32_t in_f16, a_m_major, b_n_major;
    uint32_t *status;
    const Scales *scales;         // or null: every factor 1
    int32_t logits_scaled;        // the operands of the logits are
    // MODE_STATS, MODE_GRAD
    float c;                      // log2 e / τ
    const float *un_x;            // a row's factor that undoes its scale; or null
    int64_t rows;                 // rows with a target list
    int64_t col0;                 // the class of column 0: where the piece begins
    const int32_t *ids;           // rows x top classes in ascending order, absent entries last as 0x7fffffff
    const float *p;               // their weights; or null: 1 (labels)
    const uint16_t *start;        // rows x (parts + 1): a row's first entry of each 128 classes; or null: one entry a row
    int32_t top;
    int64_t parts;                // 128-class parts of the vocabulary
    // MODE_STATS
    float2 *part;                 // [part][row]: (max, sum of 2^((l - max)·c))
    float *hit;                   // rows x top: the entries' logits
    // MODE_GRAD
    const float *lse2, *coef;     // a row's log-sum-exp in base 2, and ct/τ (0 where it has no target)
    uint16_t *g;
    int32_t g_f16;                // g in binary16, scaled by max_ct where there are scales; else bf16
    int64_t g_ld, g_rest;         // row stride; REST: how much further on what the rounding leaves is kept
    // MODE_OUT
    void *out;                    // [split][m][out_ld]
    int64_t out_ld;
    int32_t out_dtype;            // f32, bf16 or binary16 (one split then)
    int32_t out_vec;              // whole 16-byte units: aligned rows, n a multiple of a unit
    int32_t accumulate;           // f32: add to what is there (a later piece of the summed axis)
    int32_t un;                   // UN_DX, UN_DW
    uint32_t *ovf;                // the overflow guard's flag; or null
};

PSK_DEV float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

PSK_DEV float bf16_up(uint32_t h) { return __uint_as_float(h << 16); }

// One of a thread's registers, chosen by a number that only the thread knows: a compare and a predicated operation a
// register, sixteen at a time. The comparison's number is a constant of the instruction: written as an index, or with
// numbers that could be merged, the array would be moved to local memory for every tile (1.5 times the time).
template <int I>
PSK_DEV void pick(float &l, int y, float v)
{
    asm("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, %2;\n\t@p mov.f32 %0, %3;\n\t}" : "+f"(l) : "r"(y), "n"(I), "f"(v));
}
template <int I>
PSK_DEV void take(float &v, int y, float amount)
{
    asm("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, %2;\n\t@p sub.rn.f32 %0, %0, %3;\n\t}" : "+f"(v) : "r"(y), "n"(I), "f"(amount));
}
template <int G, int... I>
PSK_DEV void pick_column(float &l, int y, const float (&v)[COLS], std::integer_sequence<int, I...> s)
{
    if (y >> 4 == G) (pick<G * 16 + I>(l, y, v[G * 16 + I]), ...);
    if constexpr (G + 1 < COLS / 16) pick_column<G + 1>(l, y, v, s);
}
template <int G, int... I>
PSK_DEV void take_column(float (&v)[COLS], int y, float amount, std::integer_sequence<int, I...> s)
{
    if (y >> 4 == G) (take<G * 16 + I>(v[G * 16 + I], y, amount), ...);
    if constexpr (G + 1 < COLS / 16) take_column<G + 1>(v, y, amount, s);
}

// First entry of a row's ascending list that is at least `c`.
PSK_DEV int lower_bound(const int32_t *ids, int n, int32_t c)
{
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ids[mid] < c) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// 128 bytes of each of this warp's 32 rows: from the threads' packed words through a staging tile (16-byte units
// swizzled by the row), so that a store instruction writes whole lines (8 lanes a row, 4 rows an instruction).
// `bytes`: how many of the 128 lie inside the matrix, a multiple of 16.
template <bool ADD>
PSK_DEV void store_rows(uint4 *stage, int lane, const uint32_t (&w)[32], uint8_t *base, int64_t ld_bytes, int rows_live, int bytes)
{
#pragma unroll
    for (int q = 0; q < 8; ++q) stage[lane * 8 + (q ^ (lane & 7))] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    __syncwarp();
    const int unit = lane & 7;
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const int rr = it * 4 + (lane >> 3);
        if (rr < rows_live && unit * 16 < bytes) {
            uint4 v = stage[rr * 8 + (unit ^ (rr & 7))];
            uint4 *dst = reinterpret_cast<uint4 *>(base + rr * ld_bytes + unit * 16);
            if (ADD) {
                const uint4 o = *dst;
                v = make_uint4(__float_as_uint(__fadd_rn(__uint_as_float(o.x), __uint_as_float(v.x))), __float_as_uint(__fadd_rn(__uint_as_float(o.y), __uint_as_float(v.y))),
                               __float_as_uint(__fadd_rn(__uint_as_float(o.z), __uint_as_float(v.z))), __float_as_uint(__fadd_rn(__uint_as_float(o.w), __uint_as_float(v.w))));
            }
            *dst = v;
        }
    }
    __syncwarp();
}

// The same where rows begin at any element: the lanes write neighbouring elements (T: 16 or 32 bits) of one row.
template <class T>
PSK_DEV void store_rows_any(uint4 *stage, int lane, const uint32_t (&w)[32], uint8_t *base, int64_t ld_bytes, int rows_live, int bytes)
{
#pragma unroll
    for (int q = 0; q < 8; ++q) stage[lane * 8 + (q ^ (lane & 7))] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    __syncwarp();
    constexpr int PER = 16 / sizeof(T);
#pragma unroll 4
    for (int rr = 0; rr < rows_live; ++rr) {
        T *dst = reinterpret_cast<T *>(base + rr * ld_bytes);
        const T *src = reinterpret_cast<const T *>(stage + rr * 8);
#pragma unroll
        for (int e = lane; e < 128 / (int)sizeof(T); e += 32)
            if (e * (int)sizeof(T) < bytes) dst[e] = src[((e / PER) ^ (rr & 7)) * PER + e % PER];
    }
    __syncwarp();
}

// The product of a persistent CTA's tiles, and what MODE makes of it. Bounds: the tensor pipe (2·m·n·k flops) for many
// rows; for few, the bytes of the second operand.
template <int MODE, int MT = 1, bool REST = false>
__global__ void __launch_bounds__(THREADS, 1) k_head(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Params P)
{
    static_assert(MT == 1 || MODE == MODE_OUT, "two halves leave no second accumulator to sum in parts with");
    constexpr int STAGES = Cfg<MT>::STAGES, A_BYTES = Cfg<MT>::A_BYTES, B_BYTES = Cfg<MT>::B_BYTES, TILE_BYTES = Cfg<MT>::TILE_BYTES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *smem_a = smem, *smem_b = smem + STAGES * A_BYTES;
    uint64_t *bars = (uint64_t *)(smem + TILE_BYTES);
    // full[STAGES], empty[STAGES], accumulator full[2], accumulator empty[2]
    uint32_t *tmem_slot = (uint32_t *)(bars + 2 * STAGES + 4);
    volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full0 = tc::smem_u32(bars), empty0 = tc::smem_u32(bars + STAGES);
    const uint32_t tfull0 = tc::smem_u32(bars + 2 * STAGES), tempty0 = tc::smem_u32(bars + 2 * STAGES + 2);

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) { tc::mbar_init(full0 + 8 * s, 1); tc::mbar_init(empty0 + 8 * s, 1); }
        for (int s = 0; s < 2; ++s) { tc::mbar_init(tfull0 + 8 * s, 1); tc::mbar_init(tempty0 + 8 * s, 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tmem_slot)), "r"(2 * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;

    const int64_t per_split = P.tiles_m * P.tiles_n, total = per_split * P.splits;
    // the steps of a split: blocks kb_first .. of the summed axis, nprod partial products each
    auto steps_of = [&](int64_t sp, int &kb_first) {
        kb_first = (int)sp * P.kb_split;
        const int left = P.kb_k - kb_first;
        return (left < P.kb_split ? left : P.kb_split) * P.nprod;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
        if (warp == 0 && lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (int64_t t = blockIdx.x; t < total && ok; t += gridDim.x) {
                int64_t mt, nt;
                tc::tile_of(t % per_split, P.tiles_m, P.tiles_n, P.panel, mt, nt);
                const int m0 = (int)mt * BM * MT, n0 = (int)nt * BN;
                int kb0;
                const int steps = steps_of(t / per_split, kb0);
                int kb = kb0, q = 0;
                for (int s = 0; s < steps; ++s) {
                    ok = tc::mbar_wait(empty0 + 8 * stage, phase ^ 1u, abort_flag, P.status, 1u);
                    if (!ok) break;
                    const uint32_t fb = full0 + 8 * stage;
                    tc::mbar_expect_tx(fb, A_BYTES + B_BYTES);
                    const int k0 = kb * BK, pa = P.nprod == 1 ? 0 : plane_a(q), pb = P.nprod == 1 ? 0 : plane_b(q);
                    const uint32_t sa = tc::smem_u32(smem_a + stage * A_BYTES), sb = tc::smem_u32(smem_b + stage * B_BYTES);
                    if (!P.a_m_major) tc::tma_load_4d(sa, &map_a, fb, k0, m0, pa, 0);
                    else
#pragma unroll
                        for (int c = 0; c < BM * MT / 64; ++c) tc::tma_load_4d(sa + c * 8192, &map_a, fb, m0 + c * 64, k0, pa, 0);
                    if (!P.b_n_major) tc::tma_load_4d(sb, &map_b, fb, k0, n0, pb, 0);
                    else
#pragma unroll
                        for (int c = 0; c < BN / 64; ++c) tc::tma_load_4d(sb + c * 8192, &map_b, fb, n0 + c * 64, k0, pb, 0);
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    if (++q == P.nprod) { q = 0; ++kb; }
                }
            }
        }
        if (warp == 1 && lane == 0) {
            const uint32_t idesc = tc::instr_desc(P.in_f16, P.b_n_major, BN, P.a_m_major);
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            for (int64_t t = blockIdx.x; t < total && ok; t += gridDim.x) {
                int kb0;
                const int steps = steps_of(t / per_split, kb0);
                int in_chunk = 0;
                for (int s = 0; s < steps; ++s) {
                    if (MT == 1 && in_chunk == 0) {
                        ok = tc::mbar_wait(tempty0 + 8 * acc, acc_phase ^ 1u, abort_flag, P.status, 2u);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    }
                    ok = tc::mbar_wait(full0 + 8 * stage, phase, abort_flag, P.status, 3u);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t sa = tc::smem_u32(smem_a + stage * A_BYTES), sb = tc::smem_u32(smem_b + stage * B_BYTES);
#pragma unroll
                    for (int h = 0; h < MT; ++h) {
                        if (MT == 2 && s == 0) { // this half's accumulator has to be read out by the tile before
                            ok = tc::mbar_wait(tempty0 + 8 * h, acc_phase ^ 1u, abort_flag, P.status, 2u);
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        }
#pragma unroll
                        for (int k = 0; k < BK / tc::UMMA_K; ++k) {
                            const uint64_t ad = P.a_m_major ? tc::smem_desc(sa + h * (BM * BK * 2) + k * 2048, 8192, 1024) : tc::smem_desc(sa + h * (BM * BK * 2) + k * 32, 16, 1024);
                            const uint64_t bd = P.b_n_major ? tc::smem_desc(sb + k * 2048, 8192, 1024) : tc::smem_desc(sb + k * 32, 16, 1024);
                            tc::umma(tmem_base + (MT == 1 ? acc : (uint32_t)h) * BN, ad, bd, idesc, (in_chunk | k) != 0 ? 1u : 0u);
                        }
                    }
                    if (!ok) break;
                    tc::umma_commit(empty0 + 8 * stage);
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    ++in_chunk;
                    if (MT == 1 && (in_chunk == P.chunk || s + 1 == steps)) {
                        tc::umma_commit(tfull0 + 8 * acc);
                        in_chunk = 0;
                        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
                    }
                }
                if (MT == 2 && ok) { tc::umma_commit(tfull0); acc_phase ^= 1u; }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MANY));
        const int quad = warp & 3, half = (warp - 4) >> 2;
        uint4 *stage_out = reinterpret_cast<uint4 *>(smem + TILE_BYTES + 256) + (warp - 4) * 32 * 8;
        uint32_t acc = 0, acc_phase = 0;
        bool ok = true;
        for (int64_t t = blockIdx.x; t < total && ok; t += gridDim.x) {
            int64_t mt, nt;
            tc::tile_of(t % per_split, P.tiles_m, P.tiles_n, P.panel, mt, nt);
            const int64_t sp = t / per_split, cbase = nt * BN + half * COLS;
            int kb0;
            const int steps = steps_of(sp, kb0), chunks = MT == 1 ? (steps + P.chunk - 1) / P.chunk : 1;
#pragma unroll 1
            for (int mh = 0; mh < MT && ok; ++mh) {
            const int64_t row0 = (mt * MT + mh) * BM + quad * 32, row = row0 + lane;
            // what the row's epilogue reads, asked for while the products still run: its factors and its first target here
            const bool own = MODE != MODE_OUT && row < P.rows && cbase < P.n;
            const int32_t first = (int32_t)(P.col0 + cbase); // the class of v[0]
            int32_t y = 0x7fffffff;                          // the target's column, if it has one here
            float pw = 1.0f, un = 1.0f, lse2 = 0.0f, coef = 0.0f;
            int32_t at = 0, end = 0; // its place in the row's list, and how far the part's entries go
            bool none = true;
            const int32_t *list = nullptr;
            if (MODE != MODE_OUT && own) {
                list = P.ids + row * P.top;
                end = 1;
                none = list[0] == 0x7fffffff; // ascending, absent entries last
                if (P.start) {
                    const uint16_t *sr = P.start + row * (P.parts + 1) + (first / COLS);
                    end = sr[1];
                    at = sr[0];
                }
                if (at < end) {
                    y = list[at] - first;
                    if (P.p) pw = P.p[row * P.top + at];
                }
                if (P.logits_scaled) un = __fmul_rn(pow2(-scale_of(P.scales->max_w)), P.un_x ? P.un_x[row] : 1.0f);
                if (MODE == MODE_GRAD) {
                    lse2 = P.lse2[row];
                    coef = P.coef[row];
                    if (P.scales && P.g_f16) coef = __fmul_rn(coef, pow2(scale_of(P.scales->max_ct)));
                }
            }
            float v[COLS];
#pragma unroll
            for (int i = 0; i < COLS; ++i) v[i] = 0.0f;
            for (int ch = 0; ch < chunks; ++ch) {
                if (MT == 1 || mh == 0) {
                    ok = tc::mbar_wait(MT == 1 ? tfull0 + 8 * acc : tfull0, acc_phase, abort_flag, P.status, 4u);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t ta = tmem_base + ((uint32_t)(quad * 32) << 16) + (MT == 1 ? acc : (uint32_t)mh) * BN + half * COLS;
                // 32 columns at a time, the next 32 on their way while these are added
                uint32_t ra[32], rb[32];
                tc::tmem_ld32(ta, ra);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (g < 3) tc::tmem_ld32(ta + (g + 1) * 32, g & 1 ? ra : rb);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[g * 32 + i] = __fadd_rn(v[g * 32 + i], __uint_as_float(g & 1 ? rb[i] : ra[i]));
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(tempty0 + 8 * (MT == 1 ? acc : (uint32_t)mh));
                if (MT == 1 && ++acc == 2) { acc = 0; acc_phase ^= 1u; }
            }
            if (!ok) break;
            const int rows_live = P.m - row0 < 32 ? (int)(P.m - row0) : 32;
            if (rows_live <= 0 || cbase >= P.n) continue; // the whole warp: the next half, or the next tile
            const int live = P.n - cbase < COLS ? (int)(P.n - cbase) : COLS; // columns inside the matrix
            if constexpr (MODE == MODE_STATS || MODE == MODE_GRAD) {
                if (live < COLS) {
#pragma unroll
                    for (int i = 0; i < COLS; ++i)
                        if (i >= live) v[i] = -INFINITY;
                }
            }
            const float c = MODE == MODE_OUT ? 0.0f : __fmul_rn(P.c, un);
            if constexpr (MODE == MODE_STATS) {
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < COLS; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
                const float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                // (one rounded product m·c instead of the differences would be an instruction less, and wrong by 2^-24 of m·c)
                const float shift = m == -INFINITY ? 0.0f : m;
                // the targets' logits: a column that only its thread knows, found among registers sixteen at a time
                while (y >= 0 && y < live) {
                    float l = 0.0f;
                    pick_column<0>(l, y, v, std::make_integer_sequence<int, 16>());
                    P.hit[row * P.top + at] = __fmul_rn(l, un);
                    y = ++at < end ? list[at] - first : -1;
                }
                float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < COLS; ++i) z[i & 3] = __fadd_rn(z[i & 3], ex2(__fmul_rn(__fsub_rn(v[i], shift), c)));
                if (own) P.part[(int64_t)(first / COLS) * P.rows + row] = make_float2(__fmul_rn(m, un), __fadd_rn(__fadd_rn(z[0], z[1]), __fadd_rn(z[2], z[3])));
            } else if constexpr (MODE == MODE_GRAD) {
#pragma unroll
                for (int i = 0; i < COLS; ++i) v[i] = ex2(__fmaf_rn(v[i], c, -lse2));
                while (y >= 0 && y < live) {
                    take_column<0>(v, y, pw, std::make_integer_sequence<int, 16>());
                    y = -1;
                    if (++at < end) { y = list[at] - first; pw = P.p[row * P.top + at]; }
                }
                // a row without a target: zeros, whatever it holds
#pragma unroll
                for (int i = 0; i < COLS; ++i) v[i] = none ? 0.0f : __fmul_rn(v[i], coef);
                // Rounded for the two products that read it; where the rest of a rounding is kept too (REST: few rows,
                // f32), it is the exact remainder rounded again. Rows are padded to whole lines, the padding zeros.
                uint8_t *base = (uint8_t *)(P.g + row0 * P.g_ld + cbase);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int64_t left = (P.g_ld - cbase - g * 64) * 2;
                    const int bytes = left < 128 ? (int)left : 128;
                    uint32_t w[32];
                    if (P.g_f16) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) w[i] = pack_f16x2_hw(v[g * 64 + 2 * i], v[g * 64 + 2 * i + 1]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) w[i] = pack_bf16x2_hw(v[g * 64 + 2 * i], v[g * 64 + 2 * i + 1]);
                    }
                    store_rows<false>(stage_out, lane, w, base + g * 128, P.g_ld * 2, rows_live, bytes);
                    if constexpr (REST) {
                        if (P.g_f16) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                w[i] = pack_f16x2_hw(__fsub_rn(v[g * 64 + 2 * i], f16_to_f32((uint16_t)(w[i] & 0xffffu))), __fsub_rn(v[g * 64 + 2 * i + 1], f16_to_f32((uint16_t)(w[i] >> 16))));
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                w[i] = pack_bf16x2_hw(__fsub_rn(v[g * 64 + 2 * i], bf16_up(w[i] & 0xffffu)), __fsub_rn(v[g * 64 + 2 * i + 1], bf16_up(w[i] >> 16)));
                        }
                        store_rows<false>(stage_out, lane, w, base + g * 128 + P.g_rest * 2, P.g_ld * 2, rows_live, bytes);
                    }
                }
            } else {
                const float f = undo(P.scales, P.un);
                if (P.out_dtype == PSK_F32) {
                    uint8_t *base = (uint8_t *)((float *)P.out + (sp * P.m + row0) * P.out_ld + cbase);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        uint32_t w[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(__fmul_rn(v[g * 32 + i], f));
                        const int64_t left = (P.n - cbase - g * 32) * 4;
                        const int bytes = left < 128 ? (int)(P.out_vec ? (left + 15) / 16 * 16 : left) : 128; // vec: n a multiple of 4, or rows padded to one
                        if (P.accumulate) store_rows<true>(stage_out, lane, w, base + g * 128, P.out_ld * 4, rows_live, bytes);
                        else if (P.out_vec) store_rows<false>(stage_out, lane, w, base + g * 128, P.out_ld * 4, rows_live, bytes);
                        else store_rows_any<uint32_t>(stage_out, lane, w, base + g * 128, P.out_ld * 4, rows_live, bytes);
                    }
                } else {
                    uint8_t *base = (uint8_t *)((uint16_t *)P.out + row0 * P.out_ld + cbase);
                    uint32_t over = 0;
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        uint32_t w[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float a = __fmul_rn(v[g * 64 + 2 * i], f), b = __fmul_rn(v[g * 64 + 2 * i + 1], f);
                            if (P.out_dtype == PSK_F16) { over |= overflows(a, kF16Overflow) | overflows(b, kF16Overflow); w[i] = pack_f16x2_hw(a, b); }
                            else w[i] = pack_bf16x2_hw(a, b);
                        }
                        const int64_t left = (P.n - cbase - g * 64) * 2;
                        const int bytes = left < 128 ? (int)left : 128;
                        if (P.out_vec) store_rows<false>(stage_out, lane, w, base + g * 128, P.out_ld * 2, rows_live, bytes);
                        else store_rows_any<uint16_t>(stage_out, lane, w, base + g * 128, P.out_ld * 2, rows_live, bytes);
                    }
                    if (P.ovf && over) atomicOr(P.ovf, 1u);
                }
            }
            } // mh
            if (MT == 2) acc_phase ^= 1u;
        }
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BN) : "memory");
    }
}

// ---- what stands around the products -----------------------------------------------------------------------------

// A strided operand over the launch's rows (axes 0 .. no - 1 of `dims`).
struct RowOperand {
    const void *p;
    int32_t dtype;
    int64_t stride[PSK_MAX_AXES];
};

struct RowSpace {
    int32_t no;
    int64_t dims[PSK_MAX_AXES];
    int64_t rows;
};

PSK_DEV int64_t row_offset(const RowSpace &s, const int64_t *stride, int64_t row)
{
    int64_t off = 0;
    for (int a = s.no - 1; a >= 0; --a) {
        off += row % s.dims[a] * stride[a];
        row /= s.dims[a];
    }
    return off;
}

// Labels as lists of one class (0x7fffffff where a row has none) and, backward, a row's factor ct/τ and its log-sum-exp in
// base 2. A class that the vocabulary does not have is reported and counts as no target.
struct LabelParams {
    RowSpace s;
    RowOperand ids, ct, lse;
    int64_t classes;
    float inv_tau;
    int32_t *ids_out;
    float *coef, *lse2;
    uint32_t *status, *ctmax;
};

// ct and lse of a row, for either kind of target. Rows that a launch's weight leaves out keep the value they have.
PSK_DEV void row_factors(const RowSpace &s, const RowOperand &ct, const RowOperand &lse, int64_t row, bool none, float inv_tau, float *coef, float *lse2, uint32_t *ctmax)
{
    if (!coef) return;
    const float c = none ? 0.0f : __fmul_rn(load_real(ct.p, ct.dtype, row_offset(s, ct.stride, row)), inv_tau);
    coef[row] = c;
    lse2[row] = none ? 0.0f : (float)((double)load_real(lse.p, lse.dtype, row_offset(s, lse.stride, row)) * 1.4426950408889634);
    if (ctmax && !none && fabsf(c) <= 3.4e38f) atomicMax(ctmax, __float_as_uint(fabsf(c))); // non-negative floats order as their bits do: no order of the rows changes it
}

static __global__ void __launch_bounds__(256) k_head_labels(const __grid_constant__ LabelParams P)
{
    const int64_t row = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (row >= P.s.rows) return;
    const int64_t y = ((const int64_t *)P.ids.p)[row_offset(P.s, P.ids.stride, row)];
    if (y >= P.classes) atomicOr(P.status, 2u);
    const bool none = y < 0 || y >= P.classes;
    P.ids_out[row] = none ? 0x7fffffff : (int32_t)y;
    row_factors(P.s, P.ct, P.lse, row, none, P.inv_tau, P.coef, P.lse2, P.ctmax);
}

// A teacher's entries of one row a block: p = softmax(t/τ) over those kept (an id of zero or more, a logit above
// minus infinity), sum of p·ln p, and the entries by ascending class (each entry counts those before it: top² integer
// comparisons in shared memory), so that a tile's epilogue finds its own by bisection.
struct TeacherParams {
    RowSpace s;
    RowOperand ids, t, ct, lse;
    int64_t ids_k, t_k; // strides along the list
    int64_t classes;
    int32_t top;
    float inv_tau;
    int32_t *out_ids;
    uint16_t *start; // rows x (parts + 1)
    int64_t parts;
    float *out_p, *plogp;
    float *coef, *lse2;
    uint32_t *status, *ctmax;
};

template <bool MAX>
PSK_DEV float block_all(float x, float *red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float y = __shfl_xor_sync(0xffffffffu, x, o);
        x = MAX ? fmaxf(x, y) : __fadd_rn(x, y);
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    float r = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) r = MAX ? fmaxf(r, red[w]) : __fadd_rn(r, red[w]);
    __syncthreads();
    return r;
}

static __global__ void __launch_bounds__(1024) k_head_teacher(const __grid_constant__ TeacherParams P)
{
    extern __shared__ int32_t list[]; // top ids as they come, then in order
    __shared__ float red[32];
    const int64_t row = blockIdx.x;
    const int j = threadIdx.x;
    int32_t id = 0x7fffffff;
    float t = -INFINITY;
    if (j < P.top) {
        const int64_t raw = ((const int64_t *)P.ids.p)[row_offset(P.s, P.ids.stride, row) + j * P.ids_k];
        if (raw >= P.classes) atomicOr(P.status, 2u);
        if (raw >= 0 && raw < P.classes) {
            t = __fmul_rn(load_real(P.t.p, P.t.dtype, row_offset(P.s, P.t.stride, row) + j * P.t_k), P.inv_tau);
            if (!(t == -INFINITY)) id = (int32_t)raw;
        }
        list[j] = id;
    }
    __syncthreads();
    const bool here = id != 0x7fffffff;
    const float m = block_all<true>(here ? t : -INFINITY, red);
    // a NaN among the entries makes the row NaN: the maximum passes it over, the sum does not
    const float e = here ? expf(__fsub_rn(t, m)) : 0.0f;
    const float z = block_all<false>(e, red);
    const bool none = __syncthreads_count(here) == 0;
    const float p = here ? __fdiv_rn(e, z) : 0.0f;
    const float pl = here && p != 0.0f ? __fmul_rn(p, __fsub_rn(__fsub_rn(t, m), logf(z))) : 0.0f;
    const float sum = block_all<false>(pl, red);
    if (j < P.top) {
        int at = 0;
        for (int i = 0; i < P.top; ++i) at += list[i] < id || (list[i] == id && i < j);
        P.out_ids[row * P.top + at] = id;
        P.out_p[row * P.top + at] = p;
        list[P.top + at] = id;
    }
    __syncthreads();
    for (int64_t c = j; c <= P.parts; c += blockDim.x) P.start[row * (P.parts + 1) + c] = (uint16_t)lower_bound(list + P.top, P.top, c * COLS < 0x7fffffff ? (int32_t)(c * COLS) : 0x7fffffff);
    if (j == 0) {
        P.plogp[row] = sum;
        row_factors(P.s, P.ct, P.lse, row, none, P.inv_tau, P.coef, P.lse2, P.ctmax);
    }
}

// The greatest finite |element| of a matrix, as f32 bits (non-negative floats order as their bits do, so the blocks'
// order changes nothing): rows of `cols` elements `col_stride` apart; rows without a target are passed over.
struct MaxParams {
    RowSpace s;
    RowOperand src;
    int64_t col_stride, cols;
    const int32_t *ids;
    int32_t top, vec; // vec: 16 bytes a load (contiguous, aligned, cols a multiple of a unit)
    uint32_t *out;
};

PSK_DEV bool no_target(const int32_t *ids, int top, int64_t row) { return ids && ids[row * top] == 0x7fffffff; }

PSK_DEV uint32_t finite_bits(float x)
{
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

constexpr int PIECE = 1024; // columns of a row that a warp takes at a time

template <bool F32>
__global__ void __launch_bounds__(256) k_head_max(const __grid_constant__ MaxParams P)
{
    __shared__ uint32_t red[8];
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8, pieces = (P.cols + PIECE - 1) / PIECE;
    uint32_t m = 0;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < P.s.rows * pieces; i += warps) {
        const int64_t row = i / pieces, c0 = (i - row * pieces) * PIECE, c1 = c0 + PIECE < P.cols ? c0 + PIECE : P.cols;
        if (no_target(P.ids, P.top, row)) continue;
        const int64_t off = row_offset(P.s, P.src.stride, row);
        if (P.vec) {
            const uint4 *q = reinterpret_cast<const uint4 *>((const uint8_t *)P.src.p + (off + c0) * (F32 ? 4 : 2));
            const int n = (int)(c1 - c0) / (F32 ? 4 : 8);
#pragma unroll 4
            for (int k = lane; k < n; k += 32) {
                const uint4 u = q[k];
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int k2 = 0; k2 < 4; ++k2) {
                    if (F32) m = max(m, finite_bits(__uint_as_float(w[k2])));
                    else m = max(m, max(finite_bits(bf16_up(w[k2] & 0xffffu)), finite_bits(bf16_up(w[k2] >> 16)))); // bf16: the only 16-bit type that is scaled
                }
            }
        } else {
            const int n = (int)(c1 - c0);
            const int64_t cs = P.col_stride;
            const void *src = (const uint8_t *)P.src.p + (off + c0 * cs) * (F32 ? 4 : 2);
#pragma unroll 8
            for (int c = lane; c < n; c += 32) m = max(m, finite_bits(F32 ? ((const float *)src)[c * cs] : bf16_up(((const uint16_t *)src)[c * cs])));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) m = max(m, red[w]);
        if (m) atomicMax(P.out, m);
    }
}

// The parts' (m, z) of a row put together, and its loss. X neighbouring rows a block, 256 / X threads a row.
struct JoinParams {
    RowSpace s;
    int64_t parts;
    const float2 *part;
    const float *hit;   // rows x top
    const int32_t *ids; // rows x top
    const float *p;     // or null: labels
    const float *plogp;
    int32_t top;
    float c;      // log2 e / τ
    double inv_tau;
    RowOperand loss, lse; // lse.p may be null
    uint32_t *ovf;
    int32_t guarded;
};

template <int X>
__global__ void __launch_bounds__(256) k_head_join(const __grid_constant__ JoinParams P)
{
    constexpr int Y = 256 / X, AHEAD = 8;
    __shared__ float sm[8][X], sz[8][X];
    __shared__ double sh[8][X];
    const int x = threadIdx.x % X, y = threadIdx.x / X, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * X + x;
    float m = -INFINITY, z = 0.0f;
    double h = 0.0; // sum of p·l
    // (m, z) + (am, az) about the greater maximum; an empty part has m = -inf and z = 0
    auto join = [&](float am, float az) {
        const float g = fmaxf(m, am);
        if (!(g == -INFINITY)) z = __fadd_rn(__fmul_rn(z, exp2f(__fmul_rn(__fsub_rn(m, g), P.c))), __fmul_rn(az, exp2f(__fmul_rn(__fsub_rn(am, g), P.c))));
        m = g;
    };
    if (row < P.s.rows) {
        for (int64_t th = y; th < P.parts; th += Y * AHEAD) {
            float2 a[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) a[k] = th + Y * k < P.parts ? P.part[(th + Y * k) * P.s.rows + row] : make_float2(-INFINITY, 0.0f);
            float g = a[0].x, s = 0.0f;
#pragma unroll
            for (int k = 1; k < AHEAD; ++k) g = fmaxf(g, a[k].x);
            if (!(g == -INFINITY)) {
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) s = __fadd_rn(s, __fmul_rn(a[k].y, exp2f(__fmul_rn(__fsub_rn(a[k].x, g), P.c))));
            }
            join(g, s);
        }
        if (P.p)
            for (int j = y; j < P.top; j += Y) {
                const int64_t at = row * P.top + j;
                if (P.ids[at] != 0x7fffffff) h += (double)P.p[at] * (double)P.hit[at];
            }
    }
    if (X < 32) {
#pragma unroll
        for (int o = X; o < 32; o <<= 1) {
            const float am = __shfl_xor_sync(0xffffffffu, m, o), az = __shfl_xor_sync(0xffffffffu, z, o);
            h += __shfl_xor_sync(0xffffffffu, h, o);
            join(am, az);
        }
    }
    if ((threadIdx.x & 31) < X) { sm[warp][x] = m; sz[warp][x] = z; sh[warp][x] = h; }
    __syncthreads();
    if (threadIdx.x >= X || row >= P.s.rows) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        join(sm[i][x], sz[i][x]);
        h += sh[i][x];
    }
    const bool none = no_target(P.ids, P.top, row);
    const double lse = (double)m * P.inv_tau + log((double)z);
    const double loss = P.p ? (double)P.plogp[row] - h * P.inv_tau + lse : lse - (double)P.hit[row];
    const uint32_t ovf = store_real(const_cast<void *>(P.loss.p), P.loss.dtype, row_offset(P.s, P.loss.stride, row), none ? 0.0f : (float)loss);
    if (P.lse.p) store_real(const_cast<void *>(P.lse.p), P.lse.dtype, row_offset(P.s, P.lse.stride, row), none ? 0.0f : (float)lse);
    if (P.guarded && ovf) atomicOr(P.ovf, 1u);
}

// A matrix laid out for the tensor maps: rows of `cols` elements from any strides into rows of `ld` (a multiple of 8),
// the padding zeros, a warp 1024 columns of a row and neighbouring lanes neighbouring elements (both sides whole lines whatever the
// source's alignment). `to`: the same 16 bits; binary16 of bf16, scaled (exact); two binary16 planes of f32, scaled.
// Rows without a target (of x) become zeros, so that nothing they hold reaches dw. `copies`: the rows again below
// themselves (the second operand of a product over g and its remainder).
enum { PACK_SAME = 0, PACK_F16 = 1, PACK_SPLIT = 2 };

struct PackParams {
    RowSpace s; // the rows (for w: one axis)
    RowOperand src;
    int64_t col_stride, cols, ld, plane;
    uint16_t *dst;
    int32_t to, copies;
    const uint32_t *max; // of the whole matrix, for its scale; or null
    float *un;          // PACK_SPLIT: scale every row by its own greatest element instead, and put the factor that undoes it here
    const int32_t *ids;
    int32_t top;
};

template <int TO>
PSK_DEV uint16_t packed(uint16_t w, float f)
{
    return TO == PACK_F16 ? (uint16_t)(pack_f16x2_hw(__fmul_rn(bf16_up(w), f), 0.0f) & 0xffffu) : w;
}

// An f32 number's two planes; an infinity or a NaN stays in the first.
PSK_DEV uint32_t split_f16(float x)
{
    const uint32_t hi = pack_f16x2_hw(x, 0.0f) & 0xffffu;
    const float r = __fsub_rn(x, f16_to_f32((uint16_t)hi));
    return hi | (fabsf(r) < 65504.0f ? pack_f16x2_hw(r, 0.0f) << 16 : 0u);
}

// VEC: the source's rows contiguous and on 16-byte boundaries, cols = ld: eight elements a lane.
template <int TO, bool VEC>
__global__ void __launch_bounds__(256) k_head_pack(const __grid_constant__ PackParams P)
{
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * 8, width = P.un ? P.ld : PIECE, pieces = (P.ld + width - 1) / width, again = P.s.rows * P.ld;
    const float whole = P.max ? pow2(scale_of(*P.max)) : 1.0f;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < P.s.rows * pieces; i += warps) {
        const int64_t row = i / pieces, c0 = (i - row * pieces) * width;
        const int n = (int)((P.ld - c0) < width ? P.ld - c0 : width);                                        // columns to write
        const int live = no_target(P.ids, P.top, row) ? 0 : (int)((P.cols - c0) < n ? P.cols - c0 : n); // of which the matrix has
        const int64_t cs = P.col_stride, off = row_offset(P.s, P.src.stride, row) + c0 * cs;
        uint16_t *dst = P.dst + row * P.ld + c0;
        if constexpr (TO == PACK_SPLIT) {
            const float *src = (const float *)P.src.p + off;
            float f = whole;
            if (P.un) {
                uint32_t m = 0;
#pragma unroll 8
                for (int c = lane; c < live; c += 32) m = max(m, finite_bits(src[c * cs]));
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                const int e = scale_of(m);
                f = pow2(e);
                if (lane == 0) P.un[row] = pow2(-e);
            }
            if constexpr (VEC) {
                for (int cb = lane * 4; cb < n; cb += 4 * 128) {
                    float4 in[4]; // (all loads of a batch before its stores: the compiler cannot tell the buffers apart)
#pragma unroll
                    for (int k = 0; k < 4; ++k) in[k] = live && cb + k * 128 < n ? *reinterpret_cast<const float4 *>(src + cb + k * 128) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                    const int c = cb + k * 128;
                    if (c >= n) break;
                    const float4 x = in[k];
                    const uint32_t w0 = split_f16(__fmul_rn(x.x, f)), w1 = split_f16(__fmul_rn(x.y, f)), w2 = split_f16(__fmul_rn(x.z, f)), w3 = split_f16(__fmul_rn(x.w, f));
                    *reinterpret_cast<uint2 *>(dst + c) = make_uint2((w0 & 0xffffu) | w1 << 16, (w2 & 0xffffu) | w3 << 16);
                    *reinterpret_cast<uint2 *>(dst + P.plane + c) = make_uint2(w0 >> 16 | (w1 & 0xffff0000u), w2 >> 16 | (w3 & 0xffff0000u));
                    }
                }
            } else {
                for (int cb = lane; cb < n; cb += 8 * 32) {
                    float in[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) in[k] = cb + k * 32 < live ? src[(cb + k * 32) * cs] : 0.0f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int c = cb + k * 32;
                        if (c >= n) break;
                        const uint32_t w = split_f16(__fmul_rn(in[k], f));
                        dst[c] = (uint16_t)w;
                        dst[c + P.plane] = (uint16_t)(w >> 16);
                    }
                }
            }
        } else {
            const uint16_t *src = (const uint16_t *)P.src.p + off;
            if constexpr (VEC) {
                uint4 in[PIECE / 256];
#pragma unroll
                for (int k = 0; k < PIECE / 256; ++k) in[k] = live && lane * 8 + k * 256 < n ? *reinterpret_cast<const uint4 *>(src + lane * 8 + k * 256) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int k4 = 0; k4 < PIECE / 256; ++k4) {
                    const int c = lane * 8 + k4 * 256;
                    if (c >= n) break;
                    uint4 u = in[k4];
                    if constexpr (TO == PACK_F16) {
                        uint32_t *w = &u.x;
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] = pack_f16x2_hw(__fmul_rn(bf16_up(w[k] & 0xffffu), whole), __fmul_rn(bf16_up(w[k] >> 16), whole));
                    }
                    *reinterpret_cast<uint4 *>(dst + c) = u;
                    if (P.copies > 1) *reinterpret_cast<uint4 *>(dst + c + again) = u;
                }
            } else {
                for (int cb = lane; cb < n; cb += 16 * 32) {
                    uint16_t in[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) in[k] = cb + k * 32 < live ? src[(cb + k * 32) * cs] : (uint16_t)0;
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int c = cb + k * 32;
                        if (c >= n) break;
                        const uint16_t w = packed<TO>(in[k], whole);
                        dst[c] = w;
                        if (P.copies > 1) dst[c + again] = w;
                    }
                }
            }
        }
    }
}

// A gradient from its f32 partial sums into its place: the splits' sums in their order (and, of few rows, those of g's
// remainder `fold` rows below), times what undoes the scales, rounded once. Four columns a thread.
struct SumParams {
    RowSpace s;
    const float *part;
    int64_t parts, part_rows, ld, fold, cols, col_stride; // ld: a multiple of 4
    const Scales *scales;
    int32_t un; // UN_DX, UN_DW
    RowOperand dst;
    uint32_t *ovf;
    int32_t guarded;
};

static __global__ void __launch_bounds__(256) k_head_sum(const __grid_constant__ SumParams P)
{
    const int64_t quads = (P.cols + 3) / 4, warps = (int64_t)gridDim.x * 8, chunks = (quads + 31) / 32;
    const int lane = threadIdx.x & 31;
    const float un = undo(P.scales, P.un);
    uint32_t ovf = 0;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < P.s.rows * chunks; i += warps) {
        const int64_t row = i / chunks, c = ((i - row * chunks) * 32 + lane) * 4;
        if (c >= P.cols) continue;
        float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float *src = P.part + row * P.ld + c;
#pragma unroll 4
        for (int64_t k = 0; k < P.parts; ++k) {
            const float4 q = *reinterpret_cast<const float4 *>(src + k * P.part_rows * P.ld);
            a[0] = __fadd_rn(a[0], q.x); a[1] = __fadd_rn(a[1], q.y); a[2] = __fadd_rn(a[2], q.z); a[3] = __fadd_rn(a[3], q.w);
            if (P.fold) {
                const float4 r = *reinterpret_cast<const float4 *>(src + (k * P.part_rows + P.fold) * P.ld);
                a[0] = __fadd_rn(a[0], r.x); a[1] = __fadd_rn(a[1], r.y); a[2] = __fadd_rn(a[2], r.z); a[3] = __fadd_rn(a[3], r.w);
            }
        }
        const int64_t off = row_offset(P.s, P.dst.stride, row) + c * P.col_stride;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < P.cols) ovf |= store_real(const_cast<void *>(P.dst.p), P.dst.dtype, off + j * P.col_stride, __fmul_rn(a[j], un));
    }
    if (P.guarded && ovf) atomicOr(P.ovf, 1u);
}

} // namespace head
} // namespace psk
