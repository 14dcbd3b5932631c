// Attention of several new tokens per sequence over the paged cache
// (include/aero_cuda_pages.h): causal, with a sliding window and first tokens that stay
// visible, one pass over K and V with a running maximum and sum (pages_decode.cu has
// the formulas).
//
// Bound by the tensor cores and, as much, by the exponentials: a tile of 128 rows by 128
// positions at head size 128 is 2 x 2.1 M multiply-adds (about 1000 cycles of an SM's
// tcgen05 pipe) and 16384 exponentials (1024 cycles at 16 a cycle).
//
// Layout: a row is one (token, query head); the rows of a sequence's kv head, its group of
// query heads innermost, are cut into tiles of 128, so a K/V tile in shared memory serves
// every query head of the group and a short prompt still fills rows. A CTA takes two row
// tiles (one at head sizes 192 and 256, where two do not fit TMEM) over the tiles of
// positions that any of its tokens sees. Warps: four per row tile (a thread a row) for
// the softmax, one that issues the products, one that brings K and V by TMA (a box per
// page and 64 columns). S = Q K^T goes to TMEM, its thread takes the row's 128 scores,
// writes P over them in the cache's type, and O += P V reads P from TMEM and V from shared
// memory. The two row tiles alternate, so one's products run under the other's softmax;
// with one row tile S has two buffers instead. O stays in TMEM and is rescaled only
// when a row's maximum has grown by more than 2^8 since it was last: until then the
// weights are at most 2^8, which f16, bf16 and the f32 sums hold as exactly as any.
//
// Few row tiles over a long cache: the positions of a row tile are split over several
// CTAs that leave (o, m, l); the last to arrive joins them in order.
//
// Positions that no token of the CTA sees are zeroed in the V tile (their memory may
// hold anything, and 0 x NaN is NaN). Where only some rows see a position (diagonal, ends of
// the window), V tiles are searched for values that are not finite; if there are any, the
// row tile is computed again in f32 by row_slow, position by position: rows that do not see
// them come out as without them.
#include <cuda_runtime.h>

#include <algorithm>

#include "pages.h"
#include "pages_mma.cuh"
#include "tc_common.cuh"

namespace aero {
namespace {

constexpr int kTileRows = 128;

template <int D>
struct PCfg {
    static constexpr int NQ = D <= 128 ? 2 : 1;        // row tiles of a CTA
    static constexpr int BN = D <= 128 ? 128 : 64;     // positions per tile
    static constexpr int rows = NQ * kTileRows;
    static constexpr int stages = D == 64 ? 4 : 2;     // of K and of V
    static constexpr int half = BN * 128;              // bytes of a tile's 64-column part
    static constexpr int kv_bytes = (D / 64) * half;
    static constexpr int q_bytes = (D / 64) * kTileRows * 128;  // of one row tile
    static constexpr int smem = NQ * q_bytes + 2 * stages * kv_bytes + 256;
    static constexpr int threads = 32 * (4 * NQ + 2);
    // TMEM columns: two S buffers (of the two row tiles, or of one), then O
    static constexpr int s_col = BN;
    static constexpr int o_col0 = 2 * BN;
    static constexpr int tmem = 512;
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

// Row-major K x N operand with N (the head's columns) contiguous, 128-byte swizzle: 8-row
// groups 1024 bytes apart, 64-column parts `part` bytes apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t part) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(part >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D (TMEM) += A B, both from shared memory, 16-bit types.
__device__ __forceinline__ void umma16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(
            d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc));
}
// Instruction descriptor: f32 sums, both operands f16 or both bf16; B with N contiguous if bn.
template <bool BF16>
__device__ __forceinline__ uint32_t idesc16(int N, bool bn) {
    return idesc_f16(kTileRows, N) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (bn ? 1u << 16 : 0u);
}

// Any of the 8 16-bit values infinite or not a number?
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint4 v) {
    // the exponent bits alone; adding one step of them to all-ones carries into the sign bit
    constexpr uint32_t ex = BF16 ? 0x7F807F80u : 0x7C007C00u, one = BF16 ? 0x00800080u : 0x04000400u;
    return (((v.x & ex) + one) | ((v.y & ex) + one) | ((v.z & ex) + one) | ((v.w & ex) + one)) & 0x80008000u;
}

template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t v) {
    if constexpr (BF16)
        return __uint_as_float((uint32_t)v << 16);
    else
        return __half2float(__ushort_as_half(v));
}

// One row over the tiles [ta, tb), position by position in f32: 32 columns of o at a time to
// put(d, o, l), then m to done(m, l). For rows that meet values that are not finite.
template <int D, bool BF16, typename Put, typename Done>
__device__ __noinline__ void row_slow(const AttendArgs& a, const Work& w, int h, const uint16_t* q, int pos, int ta,
                                      int tb, const uint16_t* kp, const uint16_t* vp, Put put, Done done) {
    const int P = 1 << a.c.page_shift;
    const auto each = [&](auto f) {  // f(score, V row) for every position that the row sees
        for (int t = ta; t < tb; ++t)
            for (int i = 0; i < PCfg<D>::BN; ++i) {
                const int j = tile_pos<PCfg<D>::BN>(w, t) + i;
                if (j > pos || (a.window && j <= pos - a.window && j >= a.sinks)) continue;
                const int page = a.c.table[(int64_t)w.seq * a.c.max_pages + (j >> a.c.page_shift)];
                if ((uint32_t)page >= (uint32_t)a.c.n_page) continue;
                const int64_t row =
                    ((((int64_t)a.layer * a.c.n_page + page) * a.c.HK + h) << a.c.page_shift) + (j & (P - 1));
                float s = 0.f;
                for (int d = 0; d < D; ++d) s = fmaf(to_f32<BF16>(q[d]), to_f32<BF16>(kp[row * D + d]), s);
                f(s * a.scale_log2, vp + row * D);
            }
    };
    float m = -INFINITY, l = 0.f;
    each([&](float s, const uint16_t*) { m = fmaxf(m, s); });
    const float z = m == -INFINITY ? 0.f : m;
    each([&](float s, const uint16_t*) { l += ex2(s - z); });
    for (int d0 = 0; d0 < D; d0 += 32) {
        float o[32];
        for (int d = 0; d < 32; ++d) o[d] = 0.f;
        each([&](float s, const uint16_t* v) {
            const float p = ex2(s - z);
            for (int d = 0; d < 32; ++d) o[d] = fmaf(p, to_f32<BF16>(v[d0 + d]), o[d]);
        });
        put(d0, o, l);
    }
    done(m, l);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(PCfg<D>::threads, 1)
    prompt_attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                         const __grid_constant__ CUtensorMap vmap, const uint16_t* __restrict__ kp,
                         const uint16_t* __restrict__ vp, int n_slot, int splits) {
    using C = PCfg<D>;
    constexpr int NQ = C::NQ, BN = C::BN, ST = C::stages, SW = 4 * NQ;  // SW: softmax warps
    extern __shared__ __align__(1024) uint8_t sm[];
    const uint32_t q_s = smem_u32(sm), k_s = q_s + NQ * C::q_bytes, v_s = k_s + ST * C::kv_bytes;
    uint8_t* v_gen = sm + NQ * C::q_bytes + ST * C::kv_bytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + NQ * C::q_bytes + 2 * ST * C::kv_bytes);
    const auto bar = [&](int i) { return smem_u32(bars + i); };
    // barriers: K full / empty, V full / empty by stage; S full, P full by S buffer; O done, Q full by row
    // tile; AB: the products of a CTA that gives up
    enum { KF = 0, KE = KF + ST, VF = KE + ST, VE = VF + ST, SF = VE + ST, PF = SF + 2, OD = PF + 2, QF = OD + 2, AB = QF + 2, NB = AB + 1 };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NB);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* poison = reinterpret_cast<int*>(tmem_slot + 2);  // [NQ]
    int* last = poison + 2;
    static_assert(NB * 8 + 24 <= 256, "barrier area");
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int HK = a.c.HK, G = a.H / HK;
    const int h = (int)blockIdx.x % HK;
    const int slot = n_slot - 1 - (int)blockIdx.x / HK;  // the longest rows first

    if (blockIdx.x == 0 && blockIdx.y == 0) {  // the whole of q_start
        bool bad = false;
        for (int i = tid; i < a.n; i += C::threads) bad |= a.q_start[i] > a.q_start[i + 1];
        if (tid == 0) bad |= a.q_start[0] != 0 || a.q_start[a.n] != a.T;
        if (bad) pages_flag(a.c, AERO_CUDA_PAGES_BAD_ROWS);
    }
    Work w;
    if (!find_work<D>(a, slot, w)) return;
    // this CTA's share of the tiles; a share holds at least 4 of them
    const int per = splits > 1 ? max(4, (w.tiles + splits - 1) / splits) : max(w.tiles, 1);
    const int parts = max(1, (w.tiles + per - 1) / per);
    const int part = (int)blockIdx.y;
    if (part >= parts) return;
    const int ta = part * per, tb = min(w.tiles, ta + per), nt = tb - ta;

    if (tid == 0) {
        for (int i = 0; i < NB; ++i) mbar_init(bar(i), (i >= PF && i < OD) || (i >= QF && i < AB) ? 128u : 1u);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *abort_flag = 0;
        poison[0] = poison[1] = 0;
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
    const auto give_up = [&]() {
        *abort_flag = 1;
        pages_flag(a.c, AERO_CUDA_PAGES_WAIT);
    };

    if (warp == SW + 1) {
        // ------------------------------------------------------------ K and V tiles by TMA
        const int P = 1 << a.c.page_shift, box = min(P, 64), boxes = BN / box;
        bool good = true;
        int done = 0;  // tiles whose copies were issued
        for (int i = 0; i < nt && good; ++i) {
            const int j0 = tile_pos<BN>(w, ta + i) + lane * box;
            bool want = lane < boxes && j0 <= w.p1;
            int row = 0;
            if (want) {
                const int page = a.c.table[(int64_t)w.seq * a.c.max_pages + (j0 >> a.c.page_shift)];
                if ((uint32_t)page >= (uint32_t)a.c.n_page) {
                    pages_flag(a.c, AERO_CUDA_PAGES_BAD_PAGE);
                    want = false;
                }
                // < 2^31: checked when the cache was opened
                row = want ? (int)((((int64_t)a.layer * a.c.n_page + page) * HK + h) << a.c.page_shift) + (j0 & (P - 1)) : 0;
            }
            const int n_box = __popc(__ballot_sync(0xffffffffu, want));
            const int st = i % ST;
            const uint32_t ph = (uint32_t)(i / ST) & 1u;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const uint32_t full = bar((kv ? VF : KF) + st);
                if (!mbar_wait(bar((kv ? VE : KE) + st), ph ^ 1u, abort_flag)) {
                    good = false;
                    break;
                }
                if (lane == 0) {
                    if (n_box)
                        mbar_expect_tx(full, (uint32_t)(n_box * box * D * 2));
                    else
                        mbar_arrive(full);
                }
                __syncwarp();
                if (want) {
                    const uint32_t dst = (kv ? v_s : k_s) + (uint32_t)(st * C::kv_bytes + lane * box * 128);
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + c * C::half, kv ? &vmap : &kmap, c * 64, row, full);
                }
                __syncwarp();
            }
            done += good;
        }
        if (!good) {
            if (lane == 0) give_up();
            for (int i = std::max(0, done - ST); i < done; ++i) {  // copies in flight land before the memory is given up
                mbar_wait_timed(bar(KF + i % ST), (uint32_t)(i / ST) & 1u);
                mbar_wait_timed(bar(VF + i % ST), (uint32_t)(i / ST) & 1u);
            }
        }
    } else if (warp == SW) {
        // ------------------------------------------------------------ the products
        if (lane == 0 && nt > 0) {
            const uint32_t iqk = idesc16<BF16>(BN, false), ipv = idesc16<BF16>(D, true);
            bool good = true;
            const auto wait = [&](int b, int n) {  // the n-th completion (from 0) of barrier b
                if (good && !mbar_wait(bar(b), (uint32_t)n & 1u, abort_flag)) {
                    good = false;
                    give_up();
                }
                tc_fence_after();
            };
            const auto qk = [&](int q, int buf, int i) {
                const uint32_t qa = q_s + q * C::q_bytes, kb = k_s + (i % ST) * C::kv_bytes;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma16_ss(tmem + buf * C::s_col, sw128_desc(qa + (ks >> 2) * (kTileRows * 128) + (ks & 3) * 32),
                              sw128_desc(kb + (ks >> 2) * C::half + (ks & 3) * 32), iqk, ks > 0);
                umma_commit(bar(SF + buf));
            };
            const auto pv = [&](int q, int buf, int i) {
                const uint32_t vb = v_s + (i % ST) * C::kv_bytes;
#pragma unroll
                for (int ks = 0; ks < BN / 16; ++ks)
                    umma_ts(tmem + C::o_col0 + q * D, tmem + buf * C::s_col + ks * 8,
                            sw128_mn_desc(vb + ks * 2048, C::half), ipv, i > 0 || ks > 0);
            };
            for (int q = 0; q < NQ; ++q) wait(QF + q, 0);
            wait(KF, 0);
            if (good) {
                for (int q = 0; q < NQ; ++q) qk(q, q, 0);
                umma_commit(bar(KE));
            }
            for (int i = 0; i < nt && good; ++i) {
                const bool next = i + 1 < nt;
                if (next) wait(KF + (i + 1) % ST, (i + 1) / ST);
                if constexpr (NQ == 2) {
                    for (int q = 0; q < 2 && good; ++q) {
                        wait(PF + q, i);
                        if (q == 0) wait(VF + i % ST, i / ST);
                        if (!good) break;
                        pv(q, q, i);
                        if (next)
                            qk(q, q, i + 1);
                        else
                            umma_commit(bar(OD + q));
                    }
                } else {
                    if (next && good) qk(0, (i + 1) & 1, i + 1);
                    wait(PF + (i & 1), i >> 1);
                    wait(VF + i % ST, i / ST);
                    if (!good) break;
                    pv(0, i & 1, i);
                    umma_commit(bar(OD));
                }
                if (!good) break;
                umma_commit(bar(VE + i % ST));
                if (next) umma_commit(bar(KE + (i + 1) % ST));
            }
            if (!good) {  // products in flight end before TMEM is given up
                umma_commit(bar(AB));
                mbar_wait_timed(bar(AB), 0);
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
        const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (int64_t)(w.q0 + tok) * a.q_token + (int64_t)head * a.q_head;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        {
            const uint32_t dst = q_s + q * C::q_bytes + ((warp & 3) * 32 + lane) * 128;
            const int sw = lane & 7;
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (real) {
                    if (a.vec) {
                        v = *reinterpret_cast<const uint4*>(qp + 8 * c);
                    } else {
                        const uint16_t* x = qp + 8 * c;
                        v = make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16,
                                       x[4] | (uint32_t)x[5] << 16, x[6] | (uint32_t)x[7] << 16);
                    }
                }
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(
                                 dst + (uint32_t)((c >> 3) * (kTileRows * 128) + (((c & 7) ^ sw) << 4))),
                             "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                             : "memory");
            }
        }
        fence_proxy_async();
        mbar_arrive(bar(QF + q));

        // positions of this warp's rows (ascending with the row) and of this row tile's
        const int pw0 = __shfl_sync(0xffffffffu, pos, 0);
        const int pw1 = __reduce_max_sync(0xffffffffu, pos);
        const bool full_warp = __all_sync(0xffffffffu, real);
        const int tile_row0 = w.row0 + q * kTileRows;
        const int pt0 = w.len - w.n_new + min(tile_row0, w.rows - 1) / G;
        const int pt1 = w.len - w.n_new + (min(w.rows, tile_row0 + kTileRows) - 1) / G;
        const auto all_see = [&](int j0, int first, int lastp) {  // every position of the tile, for rows at first .. lastp
            return j0 + BN - 1 <= first && (!a.window || j0 > lastp - a.window || j0 + BN <= a.sinks);
        };
        const float sc = a.scale_log2;
        float m = -INFINITY, l = 0.f;
        bool good = true;
        for (int i = 0; i < nt && good; ++i) {
            const int buf = NQ == 2 ? q : i & 1, use = NQ == 2 ? i : i >> 1;
            const int j0 = tile_pos<BN>(w, ta + i);
            if (!mbar_wait(bar(SF + buf), (uint32_t)use & 1u, abort_flag)) {
                good = false;
                break;
            }
            tc_fence_after();
            const uint32_t st = tmem + lanes + buf * C::s_col;
            uint32_t s[BN / 32][32];
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) tmem_ld32(st + c * 32, s[c]);
            tmem_wait_ld();
            if (!(full_warp && all_see(j0, pw0, pw1))) {
                const int hi = pos - j0, lo = a.window ? pos - a.window - j0 : -1, sk = a.window ? a.sinks - j0 : 0;
#pragma unroll
                for (int c = 0; c < BN / 32; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int k = c * 32 + e;
                        if (!(k <= hi && (k > lo || k < sk))) s[c][e] = 0xFF800000u;  // -inf
                    }
            }
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < BN / 32; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e & 3] = fmaxf(x[e & 3], __uint_as_float(s[c][e]));
            const float mt = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * sc;
            if (i == 0) {
                m = mt;
            } else if (__any_sync(0xffffffffu, mt > m + 8.f)) {
                const float mn = fmaxf(m, mt);
                const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
                m = mn;
                l *= f;
                // O += P V of the tile before has ended: with two row tiles it was issued before
                // this tile's S; with one it has a barrier of its own
                if constexpr (NQ == 1) {
                    if (!mbar_wait(bar(OD), (uint32_t)(i - 1) & 1u, abort_flag)) {
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
            const float z = m == -INFINITY ? 0.f : m;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float p0 = ex2(fmaf(__uint_as_float(s[c][e]), sc, -z));
                    const float p1 = ex2(fmaf(__uint_as_float(s[c][e + 1]), sc, -z));
                    sum[e & 2] += p0;
                    sum[(e & 2) + 1] += p1;
                    // the weights meet V in its type: a relative rounding of 2^-11 (f16) or 2^-8
                    // (bf16) each, below the output's own; their sum l stays f32
                    p[e / 2] = pack16<BF16>(p0, p1);
                }
                tmem_st16(st + c * 16, p);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            const bool some = !all_see(j0, pt0, pt1);  // a position of the tile that some row does not see
            if (some) {
                if (!mbar_wait(bar(VF + i % ST), (uint32_t)(i / ST) & 1u, abort_flag)) {
                    good = false;
                    break;
                }
                uint8_t* vt = v_gen + (i % ST) * C::kv_bytes;
                bool odd = false;
                const int r = ((warp & 3) * 32 + lane) % BN;  // the row of V this thread looks after
                const int j = j0 + r;
                const bool dead = j > w.p1 || (a.window && j < w.lo && j >= a.sinks);
                // (the swizzle only orders the 16-byte pieces of a row)
                for (int c = (warp & 3) * 32 + lane >= BN ? D / 16 : 0; c < (BN == 64 && (warp & 3) < 2 ? D / 16 : D / 8); ++c) {
                    uint4* at = reinterpret_cast<uint4*>(vt + (c >> 3) * C::half + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                    if (dead)
                        *at = make_uint4(0u, 0u, 0u, 0u);
                    else
                        odd |= not_finite<BF16>(*at);
                }
                if (odd) poison[q] = 1;
                fence_proxy_async();
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bar(PF + buf));
        }
        if (good && nt > 0 && !mbar_wait(bar(OD + q), NQ == 2 ? 0u : (uint32_t)(nt - 1) & 1u, abort_flag)) good = false;
        tc_fence_after();
        if (!good) give_up();
        // every thread of the row tile has said what it met
        asm volatile("bar.sync %0, 128;" ::"r"(1 + q) : "memory");
        const bool slow = poison[q] != 0;
        uint16_t* out = static_cast<uint16_t*>(a.out) + (int64_t)(w.q0 + tok) * a.o_token + (int64_t)head * a.o_head;
        const bool stores = row < w.rows;
        const auto put_out = [&](int d0, const float* o, float k, int n) {
            for (int e = 0; e < n; e += 8) {
                const uint4 v = make_uint4(pack16<BF16>(o[e] * k, o[e + 1] * k), pack16<BF16>(o[e + 2] * k, o[e + 3] * k),
                                           pack16<BF16>(o[e + 4] * k, o[e + 5] * k), pack16<BF16>(o[e + 6] * k, o[e + 7] * k));
                uint16_t* y = out + d0 + e;
                if (a.vec) {
                    *reinterpret_cast<uint4*>(y) = v;
                } else {
                    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
                    for (int b = 0; b < 8; ++b) y[b] = (uint16_t)(x[b >> 1] >> (16 * (b & 1)));
                }
            }
        };
        const auto inverse = [](float sum) { return sum > 0.f ? 1.f / sum : sum == sum ? 0.f : sum; };
        // partial results: columns in front of rows, so a warp's stores are contiguous
        constexpr int64_t slot_f = (int64_t)C::rows * (D + 2);
        const int64_t unit = (int64_t)(blockIdx.x) * splits;
        float* mine = a.part + (unit + part) * slot_f;
        const auto put_part = [&](int d0, const float* o, int n) {
            for (int e = 0; e < n; ++e) mine[(int64_t)(d0 + e) * C::rows + lrow] = o[e];
        };
        if (slow && real) {
            row_slow<D, BF16>(
                a, w, h, qp, pos, ta, tb, kp, vp,
                [&](int d0, const float* o, float sum) {
                    if (parts == 1)
                        put_out(d0, o, inverse(sum), 32);
                    else
                        put_part(d0, o, 32);
                },
                [&](float sm_, float sl) { m = sm_, l = sl; });
        } else {
            const float k = inverse(l);
            const uint32_t ot = tmem + lanes + C::o_col0 + q * D;
            if (!slow) {
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    if (nt > 0) {
                        tmem_ld16(ot + c * 16, o);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = 0u;
                    }
                    float f[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) f[e] = __uint_as_float(o[e]);
                    if (stores && parts == 1) put_out(c * 16, f, k, 16);
                    if (parts > 1) put_part(c * 16, f, 16);
                }
            }
        }
        if (parts > 1) {
            mine[(int64_t)D * C::rows + lrow] = m;
            mine[(int64_t)(D + 1) * C::rows + lrow] = l;
            __threadfence();
            asm volatile("bar.sync 4, %0;" ::"n"(128 * NQ) : "memory");
            if (tid == 0) {
                *last = atomicAdd(a.counters + blockIdx.x, 1u) == (uint32_t)(parts - 1);
                if (*last) a.counters[blockIdx.x] = 0;  // for the next launch
            }
            asm volatile("bar.sync 4, %0;" ::"n"(128 * NQ) : "memory");
            if (*last) {
                __threadfence();
                const float* p0 = a.part + unit * slot_f + lrow;
                float M = -INFINITY, L = 0.f;
                for (int c = 0; c < parts; ++c) M = fmaxf(M, __ldcg(p0 + c * slot_f + (int64_t)D * C::rows));
                const float z = M == -INFINITY ? 0.f : M;
                for (int c = 0; c < parts; ++c)
                    L += __ldcg(p0 + c * slot_f + (int64_t)(D + 1) * C::rows) *
                         ex2(__ldcg(p0 + c * slot_f + (int64_t)D * C::rows) - z);
                const float k = inverse(L);
                for (int d0 = 0; d0 < D; d0 += 16) {
                    float o[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = 0.f;
                    for (int c = 0; c < parts; ++c) {
                        const float f = ex2(__ldcg(p0 + c * slot_f + (int64_t)D * C::rows) - z);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = fmaf(f, __ldcg(p0 + c * slot_f + (int64_t)(d0 + e) * C::rows), o[e]);
                    }
                    if (stores) put_out(d0, o, k, 16);
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
    // fewer CTAs than SMs: split the positions (the kernel splits no further than they reach)
    const int splits = (int)std::max<int64_t>(1, std::min<int64_t>(n_sm / ctas, 64));
    prompt_attend_kernel<D, BF16><<<dim3((unsigned)ctas, (unsigned)splits), C::threads, C::smem, s>>>(
        a, kmap, vmap, static_cast<const uint16_t*>(kp), static_cast<const uint16_t*>(vp), n_slot, splits);
    return cudaGetLastError();
}

}  // namespace

int pages_prompt_max_grid(int n_sm) { return n_sm; }
size_t pages_prompt_part_floats(int D, int n_sm) {
    return (size_t)n_sm * (size_t)((D <= 128 ? 2 : 1) * kTileRows) * (size_t)(D + 2);
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
