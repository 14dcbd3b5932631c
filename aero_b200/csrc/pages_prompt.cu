// Attention of several new tokens per sequence over the paged cache
// (include/aero_cuda_pages.h): causal, with a sliding window and first tokens that stay
// visible, one pass over K and V with a running maximum and sum (pages_decode.cu has
// the formulas).
//
// Bound by the tensor cores and, as much, by the exponentials: a step of two row tiles of 128
// rows by 128 positions at head size 128 is 4 x 2.1 M multiply-adds (2048 cycles of an SM's
// tcgen05 pipe) and 2 x 16384 exponentials (2048 cycles at 16 a cycle). Measured: 2600 cycles a
// step; a prompt of 4096 tokens of 32 query heads on 4 kv heads 126 us (1090 TFLOP/s of the causal
// half), of 16384 tokens 1.66 ms cold (1330), 1.81 ms in a row under the power cap. Head size 64, 8192
// tokens: 379 us (725); 256, 16 query heads on 2, 8192 tokens: 514 us (1070).
//
// Layout: a row is one (token, query head); the rows of a sequence's kv head, its group of
// query heads innermost, are cut into tiles of 128, so a K/V tile in shared memory serves
// every query head of the group and a short prompt still fills rows. A CTA takes two row
// tiles (one at head sizes 192 and 256, where two do not fit TMEM) over the tiles of
// positions that any of its tokens sees. Warps: four per row tile (a thread a row) for the
// softmax, one per row tile that issues its products, one that brings K and V by TMA (a box per
// page and 64 columns), one that zeroes V rows no token sees. S = Q K^T goes to TMEM, its
// thread takes the row's scores and writes P to TMEM in the cache's type, O += P V reads P
// there and V from shared memory.
//
// TMEM holds O and P of both row tiles and one S for both: a row tile's S is written when the
// other's has been read, so the two are always half a step apart and one's products run under the
// other's softmax. (With an S of its own for each, which P then overwrites, the two fall into
// step and wait together: 881 against 1100 TFLOP/s at 16384 tokens; with two S of 64 positions
// each, Q is read twice as often from shared memory, whose 128 bytes a cycle then bind: 1000.) One
// row tile has two S buffers instead and writes P over S.
//
// Exactness: scores, m, l and O are f32. A weight meets V rounded to the cache's type, which moves the
// output about as far as its own rounding does, so it comes out up to 1.4 times as far from the exact one
// as rounding that would be (four windowed prompts in bf16 0.0023 against 0.0017 of the output's norm,
// 16384 tokens in f16 0.00027 against 0.00020). Weights as two values of the type, as for single tokens,
// would be half as many products again, and products bind here. O is rescaled only when a row's maximum
// has grown by more than 2^8 since it was last: the weights are as exact relative to their size, but the
// largest is no longer a power of two, which would not round. Rescaled at every growth: 0.0019 and
// 0.00023, for 108 -> 119 us, 1.81 -> 2.11 ms, 4096 tokens 126 -> 148 us and at head size 256 149 -> 239 us;
// with the sum of the rounded weights for l: 0.0021 and 0.00026, for 108 -> 111 us and 1.81 -> 1.96 ms.
//
// Few row tiles over a long cache: the positions of a row tile are split over several
// CTAs that leave (o, m, l); the last to arrive joins them in order.
//
// Positions that no token of the CTA sees are zeroed in the V tile (their memory may
// hold anything, and 0 x NaN is NaN). A position that only some rows see (diagonal, ends of the
// window) may hold values that are not finite; then the rows that do not see it come out not
// finite too. So where a warp ends with such rows, it looks through the V rows that one of its rows
// does not see and another of the CTA does, and computes the rows that do not see one that is not
// finite again, by rows_slow. A row that sees all such values keeps its result.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "pages.h"
#include "pages_mma.cuh"
#include "tc_common.cuh"

namespace aero {
namespace {

constexpr int kTileRows = 128;
// How far a row tile is split: a part more saves the others its tiles and costs the CTA that
// joins the reading of rows * D sums. A tile takes about as long as the sums of kJoinRows
// rows, so nt / parts + parts * rows / kJoinRows is least at sqrt(nt * kJoinRows / rows) parts.
constexpr float kJoinRows = 220.f;
// O is rescaled when a row's maximum has grown by more than this power of two since it was last.
constexpr float kLazy = 8.f;
// At head size 64, where exponentials bind, one of every so many pairs of them is computed on the
// multiply-add pipe (ex2_poly), to relieve the special-function pipe: 8192 tokens, 32 heads, none 404 us,
// every 8th pair 380. Wider heads (4096 tokens, 128, 192 and 256) take the same time without.
constexpr int kPolyEvery = 8;

template <int D>
struct PCfg {
    static constexpr int NQ = D <= 128 ? 2 : 1;        // row tiles of a CTA
    static constexpr int rows = NQ * kTileRows;
    static constexpr int BN = D <= 128 ? 128 : 64;     // positions per tile
    // TMEM columns. Two row tiles share one S buffer and have a P each; one row tile has two S
    // buffers and writes P over S. O last.
    static constexpr bool shared_s = NQ == 2;
    static constexpr int SA = shared_s ? 1 : 2;        // tiles that S runs ahead of P V
    static constexpr int p_col0 = shared_s ? BN : 0;
    static constexpr int o_col0 = 2 * BN;
    static constexpr int tmem = 512;
    static constexpr int PH = D <= 128 ? 2 : 1;        // parts in which a tile's P is handed over
    static constexpr int stages = D == 64 ? 4 : 2;     // of K and of V
    static constexpr int half = BN * 128;              // bytes of a tile's 64-column part
    static constexpr int kv_bytes = (D / 64) * half;
    static constexpr int q_bytes = (D / 64) * kTileRows * 128;  // of one row tile
    static constexpr int smem = NQ * q_bytes + 2 * stages * kv_bytes + 512;
    static constexpr int threads = 32 * (5 * NQ + 2);
};

// What a CTA works on.
struct Work {
    int seq, len;     // the sequence and the positions it holds
    int q0, n_new;    // its first token in q, its number of tokens
    int row0, rows;   // the CTA's first row (of n_new * G) and the rows of the sequence
    int p0, p1;       // positions of the CTA's first and last token
    int lo, sinks;    // window start and first tokens in front of it, of the CTA's first token
    int first, tile0, tiles;  // tiles of positions: `first` of the sinks, then from tile0 on
};

template <int BN>
__device__ __forceinline__ int tile_pos(const Work& w, int t) { return (t < w.first ? t : w.tile0 + t - w.first) * BN; }

// The slot's sequence: slots of sequence i begin at f(i) = q_start[i] * G / R + i, which
// leaves each sequence at least as many slots as it has row tiles.
template <int D>
__device__ __forceinline__ bool find_work(const AttendArgs& a, int slot, Work& w) {
    constexpr int R = PCfg<D>::rows, BN = PCfg<D>::BN;
    const int G = a.H / a.c.HK;
    const auto f = [&](int i) { return (int64_t)a.q_start[i] * G / R + i; };
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (f(mid) <= slot)
            lo = mid;
        else
            hi = mid;
    }
    const int q0 = a.q_start[lo], q1 = a.q_start[lo + 1];
    if (q0 < 0 || q1 < q0 || q1 > a.T) {
        pages_flag(a.c, AERO_CUDA_PAGES_BAD_ROWS);
        return false;
    }
    w.q0 = q0;
    w.n_new = q1 - q0;
    w.rows = w.n_new * G;
    const int64_t r0 = ((int64_t)slot - f(lo)) * R;
    if (r0 < 0 || r0 >= w.rows) return false;
    w.row0 = (int)r0;
    w.seq = a.seqs[lo];
    if (w.seq < 0 || w.seq >= a.c.n_seq) pages_flag(a.c, AERO_CUDA_PAGES_BAD_SEQ);
    w.len = pages_length(a.c, w.seq);
    w.lo = w.sinks = w.first = w.tile0 = w.tiles = 0;
    w.p0 = w.len - w.n_new + w.row0 / G;
    w.p1 = w.len - w.n_new + (min(w.rows, w.row0 + R) - 1) / G;
    if (w.n_new > w.len) {  // its rows come out zero
        pages_flag(a.c, AERO_CUDA_PAGES_BAD_ROWS);
        return true;
    }
    w.lo = a.window ? max(0, w.p0 - a.window + 1) : 0;
    w.sinks = min(a.sinks, w.lo);
    w.tile0 = w.lo / BN;
    w.first = min((w.sinks + BN - 1) / BN, w.tile0);
    w.tiles = w.first + w.p1 / BN + 1 - w.tile0;
    return true;
}

// Shared-memory operand descriptors, 128-byte swizzle, 8-row groups 1024 bytes apart: the low
// word holds the address (in 16 bytes) and, for an operand whose N (the head's columns) is
// contiguous, the distance of its 64-column parts; the high word is the same for all.
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t part) { return (saddr >> 4) | ((part >> 4) << 16); }
__device__ __forceinline__ uint64_t desc(uint32_t low) { return (uint64_t)kDescHigh << 32 | low; }
// D (TMEM) (+)= A B, 16-bit types, A from shared memory or from TMEM.
template <bool ADD>
__device__ __forceinline__ void umma16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(
            d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "n"(ADD ? 1 : 0));
}
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
    return one != 0;
}
// Instruction descriptor: f32 sums, both operands f16 or both bf16; B with N contiguous if bn.
template <bool BF16>
__device__ __forceinline__ uint32_t idesc16(int N, bool bn) {
    return idesc_f16(kTileRows, N) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (bn ? 1u << 16 : 0u);
}

// The lowest n bits set (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

// Pairs of f32 in a 64-bit register, and their packed arithmetic.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
// Largest of three; not a number if one is none.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float v;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
    return v;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float v;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(a), "f"(b));
    return v;
}

// 2^x of a pair on the multiply-add pipe: x = n + f with n the nearest integer and |f| <= 1/2,
// 2^f by a polynomial of degree 5 (least largest relative error with a constant term of 1,
// fitted over [-1/2, 1/2]: 1.1e-7, half of what ex2 may have), n added to the exponent. Below -127, -inf among them,
// exactly 0; x at most 127 and no NaN.
__device__ __forceinline__ void ex2_poly(uint64_t x, float& p0, float& p1) {
    float a, b;
    unpair(x, a, b);
    x = pair(fmaxf(a, -127.f), fmaxf(b, -127.f));
    const uint64_t r = add2(x, pair(12582912.f, 12582912.f));  // 1.5 * 2^23: the sum's last bits are n
    const uint64_t f = fma2(add2(r, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), x);
    uint64_t t = fma2(f, pair(0.001326472731307149f, 0.001326472731307149f), pair(0.009671512991189957f, 0.009671512991189957f));
    t = fma2(t, f, pair(0.05550733581185341f, 0.05550733581185341f));
    t = fma2(t, f, pair(0.24022242426872253f, 0.24022242426872253f));
    t = fma2(t, f, pair(0.6931470036506653f, 0.6931470036506653f));
    t = fma2(t, f, pair(1.f, 1.f));
    float t0, t1, r0, r1;
    unpair(t, t0, t1);
    unpair(r, r0, r1);
    p0 = __uint_as_float(__float_as_uint(t0) + (__float_as_uint(r0) << 23));
    p1 = __uint_as_float(__float_as_uint(t1) + (__float_as_uint(r1) << 23));
}

// The pool's row of position j, or -1 where its page is none.
__device__ __forceinline__ int64_t pool_row(const AttendArgs& a, const Work& w, int h, int j) {
    const int page = a.c.table[(int64_t)w.seq * a.c.max_pages + (j >> a.c.page_shift)];
    if ((uint32_t)page >= (uint32_t)a.c.n_page) return -1;
    return ((((int64_t)a.layer * a.c.n_page + page) * a.c.HK + h) << a.c.page_shift) + (j & ((1 << a.c.page_shift) - 1));
}
// Where piece c (16 bytes) of the CTA's row r lies in Q's place, as the products read it.
template <int D>
__device__ __forceinline__ uint32_t staged(int r, int c) {
    return (uint32_t)((r >> 7) * PCfg<D>::q_bytes + (c >> 3) * (kTileRows * 128) + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4));
}
// 1 / sum of a row's weights: 0 for a row that sees nothing, and no number stays none.
__device__ __forceinline__ float inverse(float sum) { return sum > 0.f ? 1.f / sum : sum == sum ? 0.f : sum; }

// Does position j's V row hold a value that is not finite?
template <int D, bool BF16>
__device__ bool v_not_finite(const AttendArgs& a, const Work& w, int h, int j, const uint16_t* vp) {
    constexpr uint32_t ones = BF16 ? 0x7F807F80u : 0x7C007C00u;  // an exponent of ones, in both halves
    const int64_t row = pool_row(a, w, h, j);
    if (row < 0) return false;
    const uint4* v = reinterpret_cast<const uint4*>(vp + row * D);
    uint32_t any = 0;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
        const uint4 x = v[c];
        any |= __vcmpeq2(x.x & ones, ones) | __vcmpeq2(x.y & ones, ones) | __vcmpeq2(x.z & ones, ones) | __vcmpeq2(x.w & ones, ones);
    }
    return any != 0;
}

// 8 values of a query row in f32.
template <bool BF16>
__device__ __forceinline__ void query8(const uint16_t* q, int vec, float (&f)[8]) {
    uint32_t u[4];
    if (vec) {
        const uint4 x = *reinterpret_cast<const uint4*>(q);
        u[0] = x.x, u[1] = x.y, u[2] = x.z, u[3] = x.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = q[2 * e] | (uint32_t)q[2 * e + 1] << 16;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = to_f32<BF16>((uint16_t)(u[e >> 1] >> (16 * (e & 1))));
}

// kSlowRows rows over the tiles [ta, tb) in f32 by a whole warp: 32 positions' scores at a time, a lane
// each, then the columns of o by lane, 2 (lane + 32 k) and the next in o[.][2 k] and o[.][2 k + 1]. What it
// costs is the way to K and V, which the rows share. One V row in the middle of a
// prompt of 4096, 32 query heads of 128 on 4 kv heads, infinite: 4.3 ms in place of 0.14; of 16384: 19 in
// place of 1.7; every 40th of 4096: 20 ms. Rows that all see such a value take none of this.
constexpr int kSlowRows = 4;
template <int D, bool BF16>
__device__ __noinline__ void rows_slow(const AttendArgs& a, const Work& w, int h, const uint16_t* const (&q)[kSlowRows],
                                       const int (&pos)[kSlowRows], int ta, int tb, const uint16_t* kp, const uint16_t* vp,
                                       float (&o)[kSlowRows][D / 32], float (&m)[kSlowRows], float (&l)[kSlowRows]) {
    const int lane = (int)threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < kSlowRows; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) o[r][k] = 0.f;
    }
    for (int t = ta; t < tb; ++t)
        for (int i0 = 0; i0 < PCfg<D>::BN; i0 += 32) {
            const int j = tile_pos<PCfg<D>::BN>(w, t) + i0 + lane;
            uint32_t seen[kSlowRows], by_any = 0;
#pragma unroll
            for (int r = 0; r < kSlowRows; ++r) {
                seen[r] = __ballot_sync(0xffffffffu, j <= pos[r] && (!a.window || j > pos[r] - a.window || j < a.sinks));
                by_any |= seen[r];
            }
            if (!by_any) continue;
            const int64_t row = by_any >> lane & 1u ? pool_row(a, w, h, j) : -1;
            float s[kSlowRows];
#pragma unroll
            for (int r = 0; r < kSlowRows; ++r) s[r] = 0.f;
            if (row >= 0) {
                const uint4* kr = reinterpret_cast<const uint4*>(kp + row * D);
#pragma unroll 1
                for (int c0 = 0; c0 < D / 8; c0 += 8) {
                    uint4 x[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) x[c] = kr[c0 + c];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint32_t u[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
                        for (int r = 0; r < kSlowRows; ++r) {
                            float f[8];
                            query8<BF16>(q[r] + (c0 + c) * 8, a.vec, f);
#pragma unroll
                            for (int e = 0; e < 8; ++e) s[r] = fmaf(f[e], to_f32<BF16>((uint16_t)(u[e >> 1] >> (16 * (e & 1)))), s[r]);
                        }
                    }
                }
            }
            float p[kSlowRows];
#pragma unroll
            for (int r = 0; r < kSlowRows; ++r) {
                s[r] = seen[r] >> lane & 1u ? s[r] * a.scale_log2 : -INFINITY;  // (0 without a page)
                float x = s[r];
#pragma unroll
                for (int b = 1; b < 32; b <<= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, b));
                const float mn = max_nan(m[r], x), f = mn == -INFINITY ? 1.f : ex2(m[r] - mn), z = mn == -INFINITY ? 0.f : lifted<BF16>(mn, kLazy);
                m[r] = mn;
                p[r] = ex2(s[r] - z);
                float sum = p[r];
#pragma unroll
                for (int b = 1; b < 32; b <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, b);
                l[r] = fmaf(l[r], f, sum);
#pragma unroll
                for (int k = 0; k < D / 32; ++k) o[r][k] *= f;
            }
#pragma unroll 1
            for (int i0 = 0; i0 < 32; i0 += 8) {
                uint32_t u[8][D / 64];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int64_t from = (int64_t)((uint64_t)__shfl_sync(0xffffffffu, (uint32_t)((uint64_t)row >> 32), i0 + i) << 32 |
                                                   __shfl_sync(0xffffffffu, (uint32_t)row, i0 + i));
                    const uint32_t* v = reinterpret_cast<const uint32_t*>(vp + from * D) + lane;
#pragma unroll
                    for (int k = 0; k < D / 64; ++k) u[i][k] = from < 0 ? 0u : v[32 * k];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int r = 0; r < kSlowRows; ++r) {
                        const float y = __shfl_sync(0xffffffffu, p[r], i0 + i);
                        if (!(seen[r] >> (i0 + i) & 1u)) continue;  // (0 x infinity is no number)
#pragma unroll
                        for (int k = 0; k < D / 64; ++k) {
                            o[r][2 * k] = fmaf(y, to_f32<BF16>((uint16_t)u[i][k]), o[r][2 * k]);
                            o[r][2 * k + 1] = fmaf(y, to_f32<BF16>((uint16_t)(u[i][k] >> 16)), o[r][2 * k + 1]);
                        }
                    }
            }
        }
}

// Of a warp's rows (lane: row), those in doubt that do not see a V row which is not finite and which the
// CTA's products read for another row: computed again, to where a row's result is kept (`parts`: the
// CTA's partial results, else Q's place in shared memory). All lanes call it.
template <int D, bool BF16>
__device__ __noinline__ void rows_again(const AttendArgs& a, const Work& w, int h, int pos, bool doubt, int ta, int tb,
                                        const uint16_t* kp, const uint16_t* vp, uint8_t* sm, float* parts, float& m, float& l) {
    using C = PCfg<D>;
    const int lane = (int)threadIdx.x & 31, lrow0 = (int)threadIdx.x & ~31, G = a.H / a.c.HK;
    const int first = __shfl_sync(0xffffffffu, pos, 0), last = __reduce_max_sync(0xffffffffu, pos);
    // the last such V row behind the warp's first position, and the first in front of its last row's window
    const auto bad = [&](int j) {
        const int t = w.first + j / C::BN - w.tile0;
        return t >= ta && t < tb && v_not_finite<D, BF16>(a, w, h, j, vp);
    };
    int behind = -1, before = INT_MAX;
    for (int j = first + 1 + lane; j <= w.p1; j += 32)
        if (bad(j)) behind = j;
    if (a.window)
        for (int j = max(w.lo, min(a.sinks, w.p1 + 1)) + lane; j <= last - a.window; j += 32)
            if (bad(j)) before = min(before, j);
    behind = __reduce_max_sync(0xffffffffu, behind);
    before = __reduce_min_sync(0xffffffffu, before);
    uint32_t again = __ballot_sync(0xffffffffu, doubt && (behind > pos || (a.window && before <= pos - a.window)));
    while (again) {
        int which[kSlowRows], at[kSlowRows], some = 0;
        const uint16_t* q[kSlowRows];
#pragma unroll
        for (int i = 0; i < kSlowRows; ++i) {
            if (again) some = __ffs(again) - 1;  // (the last one again where there are no more)
            again &= again - 1;
            which[i] = some;
            at[i] = __shfl_sync(0xffffffffu, pos, some);
            const int row = w.row0 + lrow0 + some;
            q[i] = static_cast<const uint16_t*>(a.q) + (int64_t)(w.q0 + row / G) * a.q_token + (int64_t)(h * G + row % G) * a.q_head;
        }
        float o[kSlowRows][D / 32], row_m[kSlowRows], row_l[kSlowRows];
        rows_slow<D, BF16>(a, w, h, q, at, ta, tb, kp, vp, o, row_m, row_l);
#pragma unroll
        for (int i = 0; i < kSlowRows; ++i) {
            const int lrow = lrow0 + which[i];
            if (lane == which[i]) m = row_m[i], l = row_l[i];
            const float inv = inverse(row_l[i]);
#pragma unroll
            for (int k = 0; k < D / 64; ++k) {
                const int d = 2 * (lane + 32 * k);
                if (parts) {
                    float* to = parts + (int64_t)d * C::rows + lrow;
                    to[0] = o[i][2 * k];
                    to[C::rows] = o[i][2 * k + 1];
                } else {
                    *reinterpret_cast<uint32_t*>(sm + staged<D>(lrow, d >> 3) + (d & 7) * 2) =
                        pack16<BF16>(o[i][2 * k] * inv, o[i][2 * k + 1] * inv);
                }
            }
        }
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(PCfg<D>::threads, 1)
    prompt_attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                         const __grid_constant__ CUtensorMap vmap, const uint16_t* kp,
                         const uint16_t* vp, int n_slot, int splits) {
    using C = PCfg<D>;
    constexpr int NQ = C::NQ, BN = C::BN, SA = C::SA, PH = C::PH, ST = C::stages, SW = 4 * NQ;  // SW: softmax warps
    extern __shared__ __align__(1024) uint8_t sm[];
    const uint32_t q_s = smem_u32(sm), k_s = q_s + NQ * C::q_bytes, v_s = k_s + ST * C::kv_bytes;
    uint8_t* v_gen = sm + NQ * C::q_bytes + ST * C::kv_bytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + NQ * C::q_bytes + 2 * ST * C::kv_bytes);
    const auto bar = [&](int i) { return smem_u32(bars + i); };
    // S runs SA tiles ahead of P V. A stage holds V of tile i and K of tile i + SA, which one
    // step of the products uses; K of the first SA tiles comes first, to where K of tiles ST and
    // on will be. Barriers: full (F), V's unseen rows zero (V) and empty (E) by stage; K of the first
    // tiles there (KF) and used (KU); S there (SF), S read (SR) and P there by part (PF), by row
    // tile or by S buffer; O added to (OD) and Q there (QF) by row tile; AB: the products of a row
    // tile that is given up.
    enum {
        F = 0, V = F + ST, E = V + ST, KF = E + ST, KU = KF + 2, SF = KU + 2, SR = SF + 2, PF = SR + 2, OD = PF + 4,
        QF = OD + 2, AB = QF + 2, NB = AB + 2
    };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NB);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* last = reinterpret_cast<int*>(tmem_slot + 2);
    static_assert(NB * 8 + 24 <= 512, "barrier area");
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int HK = a.c.HK, G = a.H / HK;
    const int h = (int)blockIdx.x % HK;
    const int slot = n_slot - 1 - (int)blockIdx.x / HK;  // the longest rows first

    stream_turn();
    if (blockIdx.x == 0 && blockIdx.y == 0) check_q_start(a);
    Work w;
    if (!find_work<D>(a, slot, w)) return;
    // this CTA's share of the tiles
    const int most = min(splits, (int)sqrtf((float)w.tiles * kJoinRows / (float)min(C::rows, w.rows - w.row0)) + 1);
    const int per = max(1, (w.tiles + most - 1) / most);
    const int parts = max(1, (w.tiles + per - 1) / per);
    const int part = (int)blockIdx.y;
    if (part >= parts) return;
    const int ta = part * per, tb = min(w.tiles, ta + per), nt = tb - ta;

    if (tid == 0) {
        for (int i = 0; i < NB; ++i) {
            const bool frees = (i >= E && i < KF) || (i >= KU && i < SF), rows = (i >= SR && i < OD) || (i >= QF && i < AB);
            mbar_init(bar(i), frees ? (uint32_t)NQ : rows ? 4u : 1u);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *abort_flag = 0;
    }
    if (warp == SW) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"((uint32_t)C::tmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // the S buffer (and its barriers) of row tile q and tile i, and how often it was used before
    const auto buffer = [](int q, int i) { return C::shared_s ? q : i % C::SA; };
    const auto uses = [](int i) { return C::shared_s ? i : i / C::SA; };
    const auto s_col = [](int i) { return C::shared_s ? 0 : i % C::SA * C::BN; };
    const auto p_col = [](int q, int i) { return C::shared_s ? C::p_col0 + q * (C::BN / 2) : i % C::SA * C::BN; };
    // every position of the tile at j0 is seen by rows at positions first .. last
    const auto all_see = [&](int j0, int first, int last_pos) {
        return j0 + C::BN - 1 <= first && (!a.window || j0 > last_pos - a.window || j0 + C::BN <= a.sinks);
    };
    const auto give_up = [&]() {
        *abort_flag = 1;
        pages_flag(a.c, AERO_CUDA_PAGES_WAIT);
    };

    if (warp == SW + NQ) {
        // ------------------------------------------------------------ K and V tiles by TMA
        const int P = 1 << a.c.page_shift, box = min(P, 64), boxes = BN / box;
        bool good = true;
        // this lane's box of tile i, if a row sees a position in it: the pool's row, kNoPageRow, or -1
        const auto find = [&](int i) {
            const int j0 = tile_pos<BN>(w, ta + i) + lane * box;
            if (i >= nt || lane >= boxes || j0 > w.p1 || (j0 + box <= w.lo && j0 >= w.sinks)) return -1;
            const int page = a.c.table[(int64_t)w.seq * a.c.max_pages + (j0 >> a.c.page_shift)];
            if ((uint32_t)page >= (uint32_t)a.c.n_page) {
                pages_flag(a.c, AERO_CUDA_PAGES_BAD_PAGE);
                return kNoPageRow;
            }
            // < 2^31: checked when the cache was opened
            return (int)(((((int64_t)a.layer * a.c.n_page + page) * HK + h) << a.c.page_shift) + (j0 & (P - 1)));
        };
        const auto load = [&](const CUtensorMap& map, uint32_t tile, int row, int full) {
            if (row == -1) return;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) tma_load_2d(tile + lane * box * 128 + c * C::half, &map, c * 64, row, bar(full));
        };
        const auto expect = [&](int n_box, int full) {
            if (lane == 0) {
                if (n_box)
                    mbar_expect_tx(bar(full), (uint32_t)(n_box * box * D * 2));
                else
                    mbar_arrive(bar(full));
            }
            __syncwarp();
        };
        const auto count = [&](int row) { return __popc(__ballot_sync(0xffffffffu, row != -1)); };
        // rows of the tiles i .. i + SA - 1, whose K is on its way
        int row[SA + 1];
#pragma unroll
        for (int i = 0; i < SA; ++i) {
            row[i] = find(i);
            expect(count(row[i]), KF + i);
            load(kmap, k_s + ((i + ST - SA) % ST) * C::kv_bytes, row[i], KF + i);
        }
        int done = 0;  // stages whose copies were issued
        for (int i = 0; i < nt; ++i) {
            row[SA] = find(i + SA);
            const int st = i % ST;
            // the stage's last use; of the places of the first tiles' K, that use
            if (i >= ST) good = good && warp_wait(bar(E + st), (uint32_t)(i / ST - 1) & 1u, abort_flag);
            if (i + SA < nt && i < ST && i >= ST - SA) good = good && warp_wait(bar(KU + i - (ST - SA)), 0, abort_flag);
            if (!good) break;
            expect(count(row[0]) + count(row[SA]), F + st);
            load(vmap, v_s + st * C::kv_bytes, row[0], F + st);
            load(kmap, k_s + st * C::kv_bytes, row[SA], F + st);
#pragma unroll
            for (int k = 0; k < SA; ++k) row[k] = row[k + 1];
            ++done;
        }
        if (!good) {
            if (lane == 0) give_up();
            // copies in flight land before the memory is given up
            for (int i = 0; i < SA; ++i) mbar_wait_timed(bar(KF + i), 0);
            for (int i = std::max(0, done - ST); i < done; ++i) mbar_wait_timed(bar(F + i % ST), (uint32_t)(i / ST) & 1u);
        }
    } else if (warp == SW + NQ + 1) {
        // ------------------------------------------------------------ V rows that no row sees, to zero
        bool good = true;
        for (int i = 0; i < nt && good; ++i) {
            const int j0 = tile_pos<BN>(w, ta + i);
            good = warp_wait(bar(F + i % ST), (uint32_t)(i / ST) & 1u, abort_flag);
            if (good && !all_see(j0, w.p0, w.p1)) {
                uint8_t* vt = v_gen + (i % ST) * C::kv_bytes;
                for (int r = lane; r < BN; r += 32) {
                    const int j = j0 + r;
                    if (j <= w.p1 && (!a.window || j >= w.lo || j < a.sinks)) continue;
                    for (int c = 0; c < D / 8; ++c)  // (the swizzle only orders a row's pieces)
                        *reinterpret_cast<uint4*>(vt + (c >> 3) * C::half + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                            make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async();
            }
            __syncwarp();
            if (good && lane == 0) mbar_arrive(bar(V + i % ST));
        }
        if (!good && lane == 0) give_up();
    } else if (warp >= SW) {
        // ------------------------------------------------------------ the products of row tile q
        // (a warp each: while one waits for its softmax, the other's products run)
        const int q = warp - SW;
        // The whole warp walks the loop, with values that are visibly the same in every lane, so
        // descriptors are made by the uniform pipe; one lane issues. (With one lane walking it, the
        // arithmetic and its moves took longer than the products.)
        const int n = __shfl_sync(0xffffffffu, nt, 0);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const bool leads = elect_one();
        const uint32_t iqk = idesc16<BF16>(BN, false), ipv = idesc16<BF16>(D, true);
        bool good = true;
        const auto wait = [&](int b, int nth) {  // the nth completion (from 0) of barrier b
            if (good && !warp_wait(bar(b), (uint32_t)nth & 1u, abort_flag)) {
                good = false;
                if (leads) give_up();
            }
        };
        const auto qk = [&](int i) {
            const uint32_t qa = desc_low(q_s + q * C::q_bytes, 16), kb = desc_low(k_s + ((i + ST - SA) % ST) * C::kv_bytes, 16);
            const uint32_t d = tm + s_col(i);
            if (leads) {
                umma16_ss<false>(d, desc(qa), desc(kb), iqk);
#pragma unroll
                for (int ks = 1; ks < D / 16; ++ks)
                    umma16_ss<true>(d, desc(qa + (((ks >> 2) * (kTileRows * 128) + (ks & 3) * 32) >> 4)),
                                    desc(kb + (((ks >> 2) * C::half + (ks & 3) * 32) >> 4)), iqk);
                umma_commit(bar(SF + buffer(q, i)));
            }
            __syncwarp();
        };
        const auto pv = [&](int i, int part) {
            const int k0 = part * (BN / 16 / PH);
            const uint32_t vb = desc_low(v_s + (i % ST) * C::kv_bytes + k0 * 2048, C::half);
            const uint32_t d = tm + C::o_col0 + q * D, p = tm + p_col(q, i) + k0 * 8;
            if (leads) {
#pragma unroll
                for (int k = 0; k < BN / 16 / PH; ++k)
                    umma_ts(d, p + k * 8, desc(vb + (k * 2048 >> 4)), ipv, i > 0 || part > 0 || k > 0);
            }
            __syncwarp();
        };
        const auto commit = [&](int b) {
            if (leads) umma_commit(bar(b));
            __syncwarp();
        };
        if (n > 0) {
            wait(QF + q, 0);
            // S of tile i may be written when the buffer's last S has been read: the other row
            // tile's of this tile or the one before, or (P over S) when P V of tile i - 2, in front
            // of it, has read P
            const auto s_free = [&](int i) {
                if (C::shared_s && (q == 1 || i > 0)) wait(SR + (q ^ 1), q == 1 ? i : i - 1);
            };
            for (int i = 0; i < SA && i < n && good; ++i) {
                wait(KF + i, 0);
                s_free(i);
                if (!good) break;
                tc_fence_after();
                qk(i);
                commit(KU + i);
            }
            for (int i = 0; i < n && good; ++i) {
                wait(V + i % ST, i / ST);
                if (C::shared_s && i + SA < n) {
                    s_free(i + SA);
                    if (!good) break;
                    tc_fence_after();
                    qk(i + SA);
                }
                for (int part = 0; part < PH && good; ++part) {
                    wait(PF + buffer(q, i) * PH + part, uses(i));
                    if (!good) break;
                    tc_fence_after();
                    pv(i, part);
                }
                if (!good) break;
                if (!C::shared_s && i + SA < n) qk(i + SA);
                if (C::shared_s || i + SA >= n) commit(OD + q);
                commit(E + i % ST);
            }
            if (!good) {  // products in flight end before TMEM is given up
                commit(AB + q);
                mbar_wait_timed(bar(AB + q), 0);
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ softmax: a thread a row
        const int q = warp >> 2, lrow = q * kTileRows + (warp & 3) * 32 + lane;  // row within the CTA
        const int row = w.row0 + lrow;
        const bool real = row < w.rows && w.n_new <= w.len;
        const int tok = row / G, head = h * G + row % G;  // (used where real)
        const int pos = real ? w.len - w.n_new + tok : -1;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        // The warp's 32 rows, 16 bytes a lane, neighbouring lanes neighbouring pieces: piece x of the
        // x-th of 32 * D / 8, where it lies in shared memory (as the products read it), and the
        // offset of its row, which the row's own lane knows.
        constexpr int kPieces = D / 8;
        const auto at = [&](int x) { return staged<D>(warp * 32 + x / kPieces, x % kPieces); };
        const auto of_row = [&](int64_t mine, int r) {
            const uint32_t low = __shfl_sync(0xffffffffu, (uint32_t)mine, r), high = __shfl_sync(0xffffffffu, (uint32_t)(mine >> 32), r);
            return (int64_t)((uint64_t)high << 32 | low);
        };
        {
            const int64_t mine = real ? (int64_t)(w.q0 + tok) * a.q_token + (int64_t)head * a.q_head : -1;
            const uint16_t* all = static_cast<const uint16_t*>(a.q);
            constexpr int kLoads = kPieces % 16 == 0 ? 16 : 8;  // in flight a lane
#pragma unroll 1
            for (int x0 = 0; x0 < kPieces; x0 += kLoads) {
                uint4 v[kLoads];
#pragma unroll
                for (int k = 0; k < kLoads; ++k) {
                    const int x = (x0 + k) * 32 + lane;
                    const int64_t row_at = of_row(mine, x / kPieces);
                    v[k] = make_uint4(0u, 0u, 0u, 0u);
                    if (row_at >= 0) {
                        const uint16_t* y = all + row_at + x % kPieces * 8;
                        if (a.vec)
                            v[k] = *reinterpret_cast<const uint4*>(y);
                        else
                            v[k] = make_uint4(y[0] | (uint32_t)y[1] << 16, y[2] | (uint32_t)y[3] << 16,
                                              y[4] | (uint32_t)y[5] << 16, y[6] | (uint32_t)y[7] << 16);
                    }
                }
#pragma unroll
                for (int k = 0; k < kLoads; ++k) *reinterpret_cast<uint4*>(sm + at((x0 + k) * 32 + lane)) = v[k];
            }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(QF + q));

        // positions of this warp's rows (ascending with the row)
        const int pw0 = __shfl_sync(0xffffffffu, pos, 0);
        const int pw1 = __reduce_max_sync(0xffffffffu, pos);
        const bool full_warp = __all_sync(0xffffffffu, real);
        const float sc = a.scale_log2;
        float m = -INFINITY, l = 0.f;
        bool good = true;
        for (int i = 0; i < nt && good; ++i) {
            const int buf = buffer(q, i);
            const int j0 = tile_pos<BN>(w, ta + i);
            if (!warp_wait(bar(SF + buf), (uint32_t)uses(i) & 1u, abort_flag)) {
                good = false;
                break;
            }
            tc_fence_after();
            const uint32_t st = tmem + lanes + s_col(i), pt = tmem + lanes + p_col(q, i);
            uint32_t s[BN / 32][32];
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) tmem_ld32(st + c * 32, s[c]);
            tmem_wait_ld();
            if constexpr (C::shared_s) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(SR + q));
            }
            if (!(full_warp && all_see(j0, pw0, pw1))) {
                // bit k of a word: does the row see position k of its 32?
                const int hi = pos - j0, lo = a.window ? pos - a.window - j0 : -1, sk = a.window ? a.sinks - j0 : 0;
#pragma unroll
                for (int c = 0; c < BN / 32; ++c) {
                    const uint32_t see = low_bits(hi + 1 - 32 * c) & (~low_bits(lo + 1 - 32 * c) | low_bits(sk - 32 * c));
                    if (__all_sync(0xffffffffu, see == 0xFFFFFFFFu)) continue;
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(see >> e & 1u)) s[c][e] = 0xFF800000u;  // -inf
                }
            }
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < BN / 32; ++c)
#pragma unroll
                for (int e = 0; e < 32; e += 2)
                    x[(e >> 1) & 3] = max3(x[(e >> 1) & 3], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
            const float mt = max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3])) * sc;
            // P V of the tile before has ended: O may be rescaled and, where P has a place of its own,
            // P written. With two S buffers O's barrier counts the last two tiles alone, and the
            // first of them is waited for here, before this tile's P lets the second complete: a
            // wait that came after both would take its phase for one still to come.
            if (C::shared_s ? i > 0 : i > 0 && i == nt - 1) {
                if (!warp_wait(bar(OD + q), C::shared_s ? (uint32_t)(i - 1) & 1u : 0u, abort_flag)) {
                    good = false;
                    break;
                }
                tc_fence_after();
            }
            if (i == 0) {
                m = mt;
            } else if (__any_sync(0xffffffffu, !(mt <= m + kLazy) && mt != -INFINITY)) {
                const float mn = max_nan(m, mt);
                const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
                m = mn;
                l *= f;
                if (!C::shared_s && i + 1 < nt) {
                    // P V of the tile before has ended when S of the next tile, issued after it, is there
                    if (!warp_wait(bar(SF + (buf ^ 1)), (uint32_t)uses(i + 1) & 1u, abort_flag)) {
                        good = false;
                        break;
                    }
                    tc_fence_after();
                }
                const uint32_t ot = tmem + lanes + C::o_col0 + q * D;
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16(ot + c * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_st16(ot + c * 16, o);
                }
            }
            // (m + (m - m) is m, or no number where m is infinite or none: then the whole row is
            // none, as its formula says, and ex2_poly's result does not matter)
            const float z = m == -INFINITY ? 0.f : lifted<BF16>(m + (m - m), kLazy);
            const uint64_t sc2 = pair(sc, sc), nz2 = pair(-z, -z);
            uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint64_t y = fma2(pair(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])), sc2, nz2);
                    float p0, p1;
                    if (D == 64 && e % kPolyEvery == kPolyEvery - 1) {
                        ex2_poly(y, p0, p1);
                    } else {
                        unpair(y, p0, p1);
                        p0 = ex2(p0);
                        p1 = ex2(p1);
                    }
                    sum[e & 1] = add2(sum[e & 1], pair(p0, p1));
                    // the weights meet V in its type: a relative rounding of up to 2^-11 (f16) or 2^-8 (bf16)
                    // each, as much as the output's own; their sum l stays f32
                    p[e] = pack16<BF16>(p0, p1);
                }
                tmem_st16(pt + c * 16, p);
                if ((c + 1) % (BN / 32 / PH) == 0) {  // a part of P is there
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(PF + buf * PH + c / (BN / 32 / PH)));
                }
            }
            float l0, l1;
            unpair(add2(sum[0], sum[1]), l0, l1);
            l += l0 + l1;
        }
        if (good && nt > 0)  // the last addition to O
            good = warp_wait(bar(OD + q), C::shared_s ? (uint32_t)(nt - 1) & 1u : (uint32_t)(nt > 1), abort_flag);
        tc_fence_after();
        if (!good) give_up();
        const bool stores = row < w.rows;
        // partial results: columns in front of rows, so a warp's stores are contiguous
        constexpr int64_t slot_f = (int64_t)C::rows * (D + 2);
        const int64_t unit = (int64_t)(blockIdx.x) * splits;
        float* mine = a.part + (unit + part) * slot_f;
        const float k = inverse(l);
        const uint32_t ot = tmem + lanes + C::o_col0 + q * D;
        uint64_t zero = pair(0.f, 0.f);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            if (nt > 0) {
                tmem_ld32(ot + c * 32, o);
                tmem_wait_ld();
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0u;
            }
#pragma unroll
            for (int e = 0; e < 32; e += 2)  // 0 x o is no number where o is infinite or none
                zero = fma2(pair(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), pair(0.f, 0.f), zero);
            if (parts > 1) {
                if (stores)
#pragma unroll
                    for (int e = 0; e < 32; ++e) mine[(int64_t)(c * 32 + e) * C::rows + lrow] = __uint_as_float(o[e]);
            } else {
                // into Q's place, which no product reads any more
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint4 v;
                    v.x = pack16<BF16>(__uint_as_float(o[e]) * k, __uint_as_float(o[e + 1]) * k);
                    v.y = pack16<BF16>(__uint_as_float(o[e + 2]) * k, __uint_as_float(o[e + 3]) * k);
                    v.z = pack16<BF16>(__uint_as_float(o[e + 4]) * k, __uint_as_float(o[e + 5]) * k);
                    v.w = pack16<BF16>(__uint_as_float(o[e + 6]) * k, __uint_as_float(o[e + 7]) * k);
                    *reinterpret_cast<uint4*>(sm + at(lane * kPieces + c * 4 + e / 8)) = v;
                }
            }
        }
        float z0, z1;
        unpair(zero, z0, z1);
        __syncwarp();
        const bool doubt = !(z0 + z1 == 0.f) && real && l == l;  // (a score that is no number leaves none in the whole row)
        if (__any_sync(0xffffffffu, doubt)) {
            float m2 = m, l2 = l;
            rows_again<D, BF16>(a, w, h, pos, doubt, ta, tb, kp, vp, sm, parts > 1 ? mine : nullptr, m2, l2);
            m = m2, l = l2;
            __syncwarp();
        }
        if (parts == 1) {
            const int64_t to = stores ? (int64_t)(w.q0 + tok) * a.o_token + (int64_t)head * a.o_head : -1;
#pragma unroll 1
            for (int x0 = 0; x0 < kPieces; x0 += 8) {
                uint4 v[8];
                int64_t row_at[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int x = (x0 + k) * 32 + lane;
                    row_at[k] = of_row(to, x / kPieces);
                    v[k] = *reinterpret_cast<const uint4*>(sm + at(x));
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (row_at[k] < 0) continue;
                    uint16_t* y = static_cast<uint16_t*>(a.out) + row_at[k] + ((x0 + k) * 32 + lane) % kPieces * 8;
                    if (a.vec) {
                        *reinterpret_cast<uint4*>(y) = v[k];
                    } else {
                        const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
                        for (int b = 0; b < 8; ++b) y[b] = (uint16_t)(u[b >> 1] >> (16 * (b & 1)));
                    }
                }
            }
        }
        if (parts > 1) {
            if (stores) {
                mine[(int64_t)D * C::rows + lrow] = m;
                mine[(int64_t)(D + 1) * C::rows + lrow] = l;
            }
            asm volatile("bar.sync 4, %0;" ::"n"(128 * NQ) : "memory");
            if (tid == 0) {
                __threadfence();  // the CTA's stores, ordered before by the barrier
                *last = atomicAdd(a.counters + blockIdx.x, 1u) == (uint32_t)(parts - 1);
                if (*last) a.counters[blockIdx.x] = 0;  // for the next launch
                __threadfence();
            }
            asm volatile("bar.sync 4, %0;" ::"n"(128 * NQ) : "memory");
            if (*last) {
                // 16 columns of a row a thread, however few rows there are; the loads of kBatch parts are in
                // flight at once (an L2 round trip each batch is what this costs)
                constexpr int kBatch = 4, kCols = 16;
                const int nrows = min(C::rows, w.rows - w.row0);
                for (int x = tid; x < nrows * (D / kCols); x += 128 * NQ) {
                    const int r = x % nrows, d0 = x / nrows * kCols;
                    const float* p0 = a.part + unit * slot_f + r;
                    float M = -INFINITY, L = 0.f, o[kCols];
#pragma unroll
                    for (int e = 0; e < kCols; ++e) o[e] = 0.f;
                    for (int c0 = 0; c0 < parts; c0 += kBatch) {
                        float pm[kBatch], pl[kBatch], v[kBatch][kCols];
#pragma unroll
                        for (int b = 0; b < kBatch; ++b) {
                            const float* p = p0 + min(c0 + b, parts - 1) * slot_f;
                            pm[b] = __ldcg(p + (int64_t)D * C::rows);
                            pl[b] = __ldcg(p + (int64_t)(D + 1) * C::rows);
#pragma unroll
                            for (int e = 0; e < kCols; ++e) v[b][e] = __ldcg(p + (int64_t)(d0 + e) * C::rows);
                        }
                        float N = M;
#pragma unroll
                        for (int b = 0; b < kBatch; ++b) {
                            if (c0 + b >= parts) pm[b] = -INFINITY, pl[b] = 0.f;  // (the last part again, weight 0)
                            N = max_nan(N, pm[b]);
                        }
                        const float z = N == -INFINITY ? 0.f : N, f = ex2(M - z);
                        M = N;
                        L *= f;
#pragma unroll
                        for (int e = 0; e < kCols; ++e) o[e] *= f;
#pragma unroll
                        for (int b = 0; b < kBatch; ++b) {
                            const float y = ex2(pm[b] - z);
                            L = fmaf(pl[b], y, L);
#pragma unroll
                            for (int e = 0; e < kCols; ++e) o[e] = fmaf(v[b][e], y, o[e]);
                        }
                    }
                    const float inv = inverse(L);
                    const int t = (w.row0 + r) / G, hd = h * G + (w.row0 + r) % G;
                    uint16_t* y = static_cast<uint16_t*>(a.out) + (int64_t)(w.q0 + t) * a.o_token + (int64_t)hd * a.o_head + d0;
#pragma unroll
                    for (int e = 0; e < kCols; e += 8) {
                        const uint4 u = make_uint4(pack16<BF16>(o[e] * inv, o[e + 1] * inv), pack16<BF16>(o[e + 2] * inv, o[e + 3] * inv),
                                                   pack16<BF16>(o[e + 4] * inv, o[e + 5] * inv), pack16<BF16>(o[e + 6] * inv, o[e + 7] * inv));
                        if (a.vec) {
                            *reinterpret_cast<uint4*>(y + e) = u;
                        } else {
                            const uint32_t half[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                            for (int b = 0; b < 8; ++b) y[e + b] = (uint16_t)(half[b >> 1] >> (16 * (b & 1)));
                        }
                    }
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == SW) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::tmem));
    }
}

template <int D, bool BF16>
cudaError_t launch(const AttendArgs& a, const CUtensorMap& kmap, const CUtensorMap& vmap, const void* kp, const void* vp,
                   int n_sm, cudaStream_t s) {
    using C = PCfg<D>;
    static thread_local int prepared = -1;  // the device whose attribute this thread has set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (prepared != dev) {
        e = cudaFuncSetAttribute(prompt_attend_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem);
        if (e != cudaSuccess) return e;
        prepared = dev;
    }
    const int G = a.H / a.c.HK;
    const int n_slot = (int)((int64_t)a.T * G / C::rows) + a.n;  // see find_work
    const int64_t ctas = (int64_t)n_slot * a.c.HK;
    // fewer CTAs with work than SMs: split the positions (the kernel splits no further than pays);
    // slots without rows end at once, so they are not counted, up to the workspace's size
    const int64_t busy = std::max<int64_t>(a.n, ((int64_t)a.T * G + C::rows - 1) / C::rows) * a.c.HK;
    const int splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(n_sm / busy, pages_prompt_max_grid(n_sm) / ctas), 64));
    return launch_in_turn(prompt_attend_kernel<D, BF16>, dim3((unsigned)ctas, (unsigned)splits), C::threads, C::smem, s, a, kmap,
                          vmap, static_cast<const uint16_t*>(kp), static_cast<const uint16_t*>(vp), n_slot, splits);
}

}  // namespace

int pages_prompt_max_grid(int n_sm) { return 2 * n_sm; }
size_t pages_prompt_part_floats(int D, int n_sm) {
    return (size_t)pages_prompt_max_grid(n_sm) * (size_t)((D <= 128 ? 2 : 1) * kTileRows) * (size_t)(D + 2);
}

cudaError_t launch_pages_prompt(const AttendArgs& a, bool bf16, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                const void* k, const void* v, int n_sm, cudaStream_t s) {
    switch (a.c.D) {
        case 64: return bf16 ? launch<64, true>(a, kmap, vmap, k, v, n_sm, s) : launch<64, false>(a, kmap, vmap, k, v, n_sm, s);
        case 128: return bf16 ? launch<128, true>(a, kmap, vmap, k, v, n_sm, s) : launch<128, false>(a, kmap, vmap, k, v, n_sm, s);
        case 192: return bf16 ? launch<192, true>(a, kmap, vmap, k, v, n_sm, s) : launch<192, false>(a, kmap, vmap, k, v, n_sm, s);
        case 256: return bf16 ? launch<256, true>(a, kmap, vmap, k, v, n_sm, s) : launch<256, false>(a, kmap, vmap, k, v, n_sm, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace aero
