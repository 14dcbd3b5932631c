// Attention over the paged cache (include/aero_cuda_pages.h), token by token: one new
// token per sequence, or few of several. o = sum_j softmax_j(scale q . k_j) v_j over the visible
// positions, one pass over K and V with a running maximum m and sum l:
//   m' = max(m, max_j s_j),  l' = l 2^(m - m') + sum_j 2^(s_j - m'),
//   o' = o 2^(m - m') + sum_j 2^(s_j - m') v_j     (s in powers of two),
// and two partial results join by the same rule.
//
// Bound by HBM: every visible K and V row is read once (up to 16 query heads share it,
// at most 16 operations a byte). Measured, time on the GPU: 48 sequences of 8192 to 32768 positions, 32
// query heads on 4 kv heads of 128, 289 us (1.85 GB: 6.4 TB/s); one sequence of 4096 12.9 us, of 20 5.3 us,
// where a launch, the chain from lengths to pages to rows, and the join set the time. Over listed blocks: 48
// sequences, 32 blocks of 64 positions a kv head, 43.8 us (199 MB: 4.5 TB/s); 2048 of one sequence's 32768
// positions 11.2 us. Lists wider than a sequence: 64 sequences of 20 positions, pages of 16, 6.1 us with lists as long as they are, 6.3
// us with 128 entries, 8.1 us with 1000 (-1 behind).
//
// Split: the work of the call is one line of units, unit = 64 positions of one
// (sequence, kv head); each CTA takes an equal piece of the line, wherever it begins, so
// sequences of any lengths load the GPU evenly and one long sequence is split over all of
// it. A (sequence, head) whose units lie in one CTA is finished there; the others leave
// partial results (o, m, l), and the CTA that arrives last joins them in the line's
// order, so the sums do not depend on timing.
//
// A CTA: one producer warp brings units into a ring of stages by TMA (a page is a run of
// rows per head; a box of min(page, 64) rows by 64 columns, swizzled), four consumer warps
// take 16 positions of each unit as S^T = K Q^T and O^T += V^T P^T in m16n8k16 products, the kv
// head's query heads as the 8 or 16 columns (as rows they would be padded to 16, with twice the
// products and sums: 8 % more for one sequence of 4096, 3 % for the long ones), each warp with its own
// m, l, o until the segment's end. The consumers never wait for one another within a segment. An SM's
// share of HBM takes 1400 cycles for a unit's 32 KB (head size 128); the matrix pipe is active for 15 %
// of them, issue slots for 21 %: the unit's bytes, not its products, set the time, so tcgen05's 128
// rows would not help.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "pages.h"
#include "pages_mma.cuh"
#include "tc_common.cuh"

namespace aero {
namespace {

constexpr int kUnit = 64;          // positions per unit
constexpr int kConsumers = 4;      // warps; each takes 16 positions of a unit
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kWhole = 8, kParts = 16;  // see piece_length
constexpr int kHalf = kUnit * 128; // bytes of a unit's 64-column half
constexpr int kNowhere = 1 << 30;  // a position that no token sees (sequences hold at most 2^30)
constexpr int kNoMore = -1;        // in a stage's first position: this is no unit, and the list has no more
constexpr int kLook = 4;           // entries of a list that a lane looks at at once

template <int D>
struct Cfg {
    // two CTAs of an SM hide one another's segment ends; wide heads fill it alone
    static constexpr int ctas = D <= 128 ? 2 : 1;
    static constexpr int stages = D == 64 ? 6 : D == 128 ? 3 : D == 192 ? 4 : 3;
    static constexpr int stage_bytes = 2 * (D / 64) * kHalf;
    static constexpr int red_bytes = 2 * 16 * D * 4;
    static constexpr int smem = stages * stage_bytes + red_bytes + 1024;
};

// The units of one token's kv head: tiles of 64 positions that hold a visible one,
// first those of the first tokens (sinks), then the window's.
struct Span {
    int seq;
    int n;      // positions that the token may see: its own and those before it
    int lo;     // first position of the window
    int sinks;  // positions visible before it
    int first;  // tiles of the sinks in front of the window's
    int tile0;  // the window's first tile
    int tiles;  // at least 1: an empty sequence has a unit that writes zeros
};

// Over listed blocks (SEL) a kv head's units are the list's: 64 positions of it in its order. The line has
// units for as many entries of it as the token has blocks (`first`): most lists have no others that count. Of a longer list
// whoever takes the last of these units goes on through the entries behind them and takes what they list (blocks
// after -1s, listed again, after some that the token does not see), as units that the line does not know of. A list
// that ends in -1s costs a look at them and no unit, while the units before are on their way.
template <bool SEL>
__device__ __forceinline__ Span span_of(const AttendArgs& a, int e) {
    Span p;
    token_rows(a, e, p.seq, p.n);
    if (p.seq < 0 || p.seq >= a.c.n_seq) pages_flag(a.c, AERO_CUDA_PAGES_BAD_SEQ);
    if constexpr (SEL) {
        p.lo = p.sinks = p.tile0 = 0;
        p.first = p.n > 0 ? min(a.width, ((p.n - 1) >> a.c.page_shift) + 1) : 0;
        p.tiles = p.n > 0 ? (int)((((int64_t)p.first << a.c.page_shift) + kUnit - 1) / kUnit) : 1;
        return p;
    }
    p.lo = a.window && p.n > a.window ? p.n - a.window : 0;
    p.sinks = min(a.sinks, p.lo);
    p.tile0 = p.lo / kUnit;
    p.first = min((p.sinks + kUnit - 1) / kUnit, p.tile0);
    p.tiles = p.n > 0 ? p.first + (p.n - 1) / kUnit + 1 - p.tile0 : 1;
    return p;
}
// Whether entries of a list lie behind units [t0, t0 + cnt) and behind the line's.
__device__ __forceinline__ bool listed_behind(const AttendArgs& a, const Span& p, int t0, int cnt) {
    return cnt > 0 && t0 + cnt == p.tiles && p.first < a.width && p.n > 0;
}
// By a warp: a list's first entry from i on that is a block which the token sees (up to `own`); `width`: none is. (A function of
// its own: inside the producer's loop it costs a call of 11 us that never comes here 0.1 us more.)
__device__ __noinline__ int seen_from(const int32_t* list, int i, int width, int own) {
    const int lane = (int)threadIdx.x & 31;
    for (; i < width; i += 32 * kLook) {
        int block[kLook];
#pragma unroll
        for (int k = 0; k < kLook; ++k) block[k] = i + 32 * k + lane < width ? list[i + 32 * k + lane] : -1;
#pragma unroll
        for (int k = 0; k < kLook; ++k) {
            const uint32_t have = __ballot_sync(0xffffffffu, block[k] >= 0 && block[k] <= own);
            if (have) return i + 32 * k + __ffs((int)have) - 1;
        }
    }
    return width;
}
__device__ __forceinline__ int tile_at(const Span& p, int t) { return t < p.first ? t : p.tile0 + t - p.first; }
__device__ __forceinline__ bool visible(const Span& p, int j) { return j < p.n && (j >= p.lo || j < p.sinks); }

// a / b of numbers >= 0: in 32 bits where they fit (a division in 64 costs some 200 cycles, and those
// of a CTA's beginning were most of its 5000 before the first copy).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// Places of the line that a CTA takes: an equal share, but at least what is worth a part of its own.
// (sequence, head)s of up to kWhole units are left whole: joining parts costs more than those few
// units one after another. Longer ones are cut into about kParts parts, as many as a join reads at
// once, of 2 to 4 units, if possible an even cut, so that no part holds the end of one and the
// beginning of the next (one sequence of 4096, 64 units: parts of 3 take 2.4 us more than of 4).
__device__ __forceinline__ int64_t piece_length(int64_t total, int64_t segments) {
    const int64_t each = quotient(total + segments - 1, segments), share = quotient(total + gridDim.x - 1, gridDim.x);
    if (each <= kWhole) return max(each, share);
    const int least = (int)min((int64_t)4, max((int64_t)2, (each + kParts - 1) / kParts));
    int w = least;
    for (int c = 2 * least - 1; c >= least; --c)
        if (each - quotient(each, c) * c == 0) w = c;
    return max((int64_t)w, share);
}

// What [u, u1) of the line holds of the (sequence, head) at u: on the line each begins with a.over
// places for the cost of having it at all, so that CTAs with more beginnings get fewer units.
struct Piece {
    int h, t0, cnt, line;  // kv head, units [t0, t0 + cnt), places on the line
};
__device__ __forceinline__ Piece piece_at(const AttendArgs& a, const Span& p, int64_t u, int64_t u1, int64_t base) {
    const int line = p.tiles + a.over;
    const int64_t in = u - base;
    Piece c;
    c.h = (int)quotient(in, line);
    const int at = (int)(in - (int64_t)c.h * line);
    c.line = (int)min((int64_t)(line - at), u1 - u);
    c.t0 = max(at - a.over, 0);
    c.cnt = max(at + c.line - a.over, 0) - c.t0;
    return c;
}

// NT: tiles of 8 query heads (a kv head's group is up to 8 or up to 16 of them). SEL: over listed blocks.
template <int D, bool BF16, int NT, bool SEL>
__global__ void __launch_bounds__(kThreads, Cfg<D>::ctas)
    decode_attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap kmap,
                         const __grid_constant__ CUtensorMap vmap) {
    constexpr int ST = Cfg<D>::stages;
    extern __shared__ __align__(1024) uint8_t sm[];
    float* red = reinterpret_cast<float*>(sm + ST * Cfg<D>::stage_bytes);        // [4][8][D] or [2][16][D], columns swizzled by row
    float2* ml = reinterpret_cast<float2*>(sm + ST * Cfg<D>::stage_bytes + Cfg<D>::red_bytes);  // [4][16] (m, l)
    float2* joint = ml + 64;                                                     // [16]
    uint64_t* bars = reinterpret_cast<uint64_t*>(joint + 16);                    // full[ST], empty[ST]
    int64_t* begin_s = reinterpret_cast<int64_t*>(bars + 2 * ST);                // entry base
    int4* joins = reinterpret_cast<int4*>(begin_s + 2);                          // [2]: parts to join (or 0), first CTA, token, head
    int* misc = reinterpret_cast<int*>(joins + 2);                               // entry, abort
    Span* span_s = reinterpret_cast<Span*>(misc + 2);                            // the first entry's
    int* box_at = reinterpret_cast<int*>(span_s + 1);                            // [ST][8]: SEL: a box's first position
    static_assert((64 + 16) * 8 + 2 * ST * 8 + 16 + 32 + 8 + sizeof(Span) + ST * 32 <= 1024, "the last 1024 bytes hold these");
    volatile int* abort_flag = misc + 1;
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int HK = a.c.HK, G = a.H / HK;
    const uint32_t ring = smem_u32(sm);

    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(smem_u32(bars + i), 1);
            mbar_init(smem_u32(bars + ST + i), kConsumers);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *abort_flag = 0;
    }
    stream_turn();
    if (blockIdx.x == 0 && a.q_start) check_q_start(a);
    // ---- this CTA's piece of the line of units
    int64_t total, w;
    {
        int64_t* sums = reinterpret_cast<int64_t*>(red);  // [kThreads / 32]
        const int per = (a.T + kThreads - 1) / kThreads;
        const int e0 = min(a.T, tid * per), e1 = min(a.T, e0 + per);
        int64_t mine = 0;
        for (int e = e0; e < e1; ++e) mine += span_of<SEL>(a, e).tiles + a.over;
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        int64_t before = incl - mine;
        total = 0;
        for (int i = 0; i < kThreads / 32; ++i) {
            if (i < warp) before += sums[i];
            total += sums[i];
        }
        total *= HK;
        w = piece_length(total, (int64_t)a.T * HK);
        const int64_t u0 = w * blockIdx.x;
        if (u0 >= before * HK && u0 < (before + mine) * HK) {
            int64_t base = before * HK;
            int e = e0;
            Span at;
            for (;; ++e) {
                at = span_of<SEL>(a, e);
                const int64_t next = base + (int64_t)(at.tiles + a.over) * HK;
                if (u0 < next) break;
                base = next;
            }
            begin_s[0] = base;
            misc[0] = e;
            *span_s = at;
        }
        __syncthreads();
    }
    const int64_t u0 = w * blockIdx.x, u1 = min(total, u0 + w);
    if (u0 >= u1) return;

    int e = misc[0];
    int64_t base = begin_s[0];
    Span sp = *span_s;
    int stage = 0;
    uint32_t phase = 0;

    if (warp == kConsumers) {
        // ---------------------------------------------------------- producer
        const int P = 1 << a.c.page_shift, rows = min(P, kUnit), boxes = kUnit / rows;
        int64_t loaded = 0;
        bool good = true;
        for (int64_t u = u0; u < u1 && good;) {
            const Piece pc = piece_at(a, sp, u, u1, base);
            const int h = pc.h, t0 = pc.t0, cnt = pc.cnt;
            const int s = sp.seq;
            // SEL: a box's first position and page for each lane, 32 boxes at once (the list and then the table are
            // two reads one after another; for each unit anew they held the first stages up)
            int at32 = kNowhere, page32 = 0;
            const bool behind = SEL && listed_behind(a, sp, t0, cnt);
            const int32_t* const list = SEL ? a.blocks + ((int64_t)e * HK + h) * a.width : nullptr;
            int hand = t0;  // a unit at which 32 boxes were taken in hand
            for (int t = t0; t < t0 + cnt || behind; ++t) {
                // lane i brings box i, if a position in it is visible
                int j0;
                bool want;
                int page = 0;
                if constexpr (SEL) {
                    int slot = (t - hand) * boxes & 31;
                    int left = (t0 + cnt - t) * boxes;  // (beyond the piece: boxes that no unit here takes)
                    if (t >= t0 + cnt && (slot == 0 || t == t0 + cnt)) {
                        // behind the line's units: on to the next one with an entry that counts, if there is one
                        const int i = seen_from(list, (int)(((int64_t)t * kUnit) >> a.c.page_shift), a.width, (sp.n - 1) >> a.c.page_shift);
                        t = max(t, (int)(((int64_t)i << a.c.page_shift) / kUnit));
                        hand = t;
                        slot = 0;
                        left = i < a.width ? 32 : 0;
                    }
                    if (slot == 0) {
                        const int64_t at = (int64_t)t * kUnit + lane * rows;  // in the list's positions
                        const int i = (int)(at >> a.c.page_shift);
                        const int block = i < a.width && lane < left ? list[i] : -1;
                        at32 = kNowhere;
                        if (block >= 0 && block <= (sp.n - 1) >> a.c.page_shift) {
                            const int j = (block << a.c.page_shift) + (int)(at & (P - 1));
                            if (j < sp.n) {
                                at32 = j;
                                page32 = a.c.table[(int64_t)s * a.c.max_pages + block];
                                if ((uint32_t)page32 >= (uint32_t)a.c.n_page) pages_flag(a.c, AERO_CUDA_PAGES_BAD_PAGE);
                            }
                        }
                    }
                    j0 = __shfl_sync(0xffffffffu, at32, slot + (lane & (boxes - 1)));
                    page = __shfl_sync(0xffffffffu, page32, slot + (lane & (boxes - 1)));
                    want = lane < boxes && j0 != kNowhere;
                    if (t >= t0 + cnt && !__any_sync(0xffffffffu, want)) {
                        if (left) continue;  // (nothing of it is seen)
                        j0 = kNoMore;
                    }
                } else {
                    j0 = tile_at(sp, t) * kUnit + lane * rows;
                    want = lane < boxes && j0 < sp.n && (j0 + rows > sp.lo || j0 < sp.sinks);
                    if (want) {
                        page = a.c.table[(int64_t)s * a.c.max_pages + (j0 >> a.c.page_shift)];
                        if ((uint32_t)page >= (uint32_t)a.c.n_page) pages_flag(a.c, AERO_CUDA_PAGES_BAD_PAGE);
                    }
                }
                if (!warp_wait(smem_u32(bars + ST + stage), phase ^ 1u, abort_flag)) {
                    good = false;
                    break;
                }
                const uint32_t full = smem_u32(bars + stage);
                if constexpr (SEL) {
                    if (lane < 8) box_at[stage * 8 + lane] = j0;
                    __syncwarp();  // before lane 0's arrival
                }
                const int n_box = __popc(__ballot_sync(0xffffffffu, want));
                if (lane == 0) {
                    if (n_box)
                        mbar_expect_tx(full, (uint32_t)(n_box * rows * D * 2 * 2));
                    else
                        mbar_arrive(full);
                }
                __syncwarp();
                if (want) {
                    const int64_t row0 = (((int64_t)a.layer * a.c.n_page + page) * HK + h) << a.c.page_shift;
                    // < 2^31: checked when the cache was opened
                    const int row = (uint32_t)page < (uint32_t)a.c.n_page ? (int)row0 + (j0 & (P - 1)) : kNoPageRow;
                    const uint32_t dst = ring + (uint32_t)stage * Cfg<D>::stage_bytes + (uint32_t)(lane * rows * 128);
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + c * kHalf, &kmap, c * 64, row, full);
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + (D / 64 + c) * kHalf, &vmap, c * 64, row, full);
                }
                __syncwarp();
                ++loaded;
                if (++stage == ST) {
                    stage = 0;
                    phase ^= 1u;
                }
                if (SEL && j0 == kNoMore) break;  // (in all lanes)
            }
            u += pc.line;
            if (u == base + (int64_t)(sp.tiles + a.over) * HK && u < u1) {
                base = u;
                sp = span_of<SEL>(a, ++e);
            }
        }
        if (!good) {
            *abort_flag = 1;
            if (lane == 0) pages_flag(a.c, AERO_CUDA_PAGES_WAIT);
            // copies in flight land before the CTA's memory is given up
            for (int i = 0; i < ST && i < loaded; ++i) {
                const int64_t k = loaded - 1 - i;
                mbar_wait_timed(smem_u32(bars + (int)(k % ST)), (uint32_t)((k / ST) & 1));
            }
        }
        return;
    }

    // -------------------------------------------------------------- consumers
    const int g = lane >> 2, tq = lane & 3;
    bool dead = false;
    // rows and columns of the 8x8 blocks this lane addresses. K, keys as the product's rows: blocks
    // (keys 0-7, 8-15) x (columns 0-7), then columns 8-15. V, transposed, columns as the product's
    // rows: blocks (columns 0-7, 8-15) x (keys 0-7), then keys 8-15.
    const int krow = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), kcol = lane >> 4;
    const int vrow = warp * 16 + (lane >> 4) * 8 + (lane & 7), vcol = (lane >> 3) & 1;
    constexpr int kRegions = 4 / NT;  // of `red`, 8 * NT rows each
    constexpr int64_t slot = 16 * (D + 2);  // floats of a partial result
    if (tid < 2) joins[tid] = make_int4(0, 0, 0, 0);  // (read after later barriers)
    const auto out_of = [&](int tok, int h) {
        return static_cast<uint16_t*>(a.out) + (int64_t)tok * a.o_token + (int64_t)(h * G) * a.o_head;
    };
    const auto put = [&](uint16_t* to, int row, int d, float4 v) {
        uint16_t* y = to + (int64_t)row * a.o_head + d;
        const uint32_t w0 = pack16<BF16>(v.x, v.y), w1 = pack16<BF16>(v.z, v.w);
        if (a.vec) {
            *reinterpret_cast<uint2*>(y) = make_uint2(w0, w1);
        } else {
            y[0] = (uint16_t)w0;
            y[1] = (uint16_t)(w0 >> 16);
            y[2] = (uint16_t)w1;
            y[3] = (uint16_t)(w1 >> 16);
        }
    };
    const auto summed = [&](int row, int d) {
        const int col = d ^ (((row >> 1) & 3) * 8);
        float4 x = *reinterpret_cast<const float4*>(red + row * D + col);
#pragma unroll
        for (int i = 1; i < kRegions; ++i) {
            const float4 y = *reinterpret_cast<const float4*>(red + (i * 8 * NT + row) * D + col);
            x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
        return x;
    };
    for (int64_t u = u0; u < u1;) {
        const Piece pc = piece_at(a, sp, u, u1, base);
        const int h = pc.h, t0 = pc.t0, cnt = pc.cnt;
        if (cnt > 0) {
        // the query heads as the products' columns; those past G are zero
        uint32_t qf[D / 16][NT][2];
        {
            const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)e * a.q_token + (int64_t)(h * G) * a.q_head;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i) {
                    const int r = g + (i >> 1) * 8;
                    const uint16_t* x = q + (int64_t)r * a.q_head + ks * 16 + (i & 1) * 8 + 2 * tq;
                    qf[ks][i >> 1][i & 1] = r >= G ? 0u
                                            : a.vec ? *reinterpret_cast<const uint32_t*>(x)
                                                    : (uint32_t)x[0] | ((uint32_t)x[1] << 16);
                }
        }
        // o[i][n]: columns 16 i + g and + 8 (by bit 1) of query heads 8 n + 2 tq and + 1 (by bit 0)
        float o[D / 16][NT][4];
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
        float m[2 * NT], l[2 * NT];
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) m[i] = -INFINITY, l[i] = 0.f;
        const bool behind = SEL && listed_behind(a, sp, t0, cnt);
        for (int t = t0; t < t0 + cnt || behind; ++t) {
            // a warp whose wait gave up goes on without waiting (its results are void, the status
            // says so): the other warps still meet it at the barriers below
            if (!dead && !warp_wait(smem_u32(bars + stage), phase, abort_flag)) {
                dead = true;
                *abort_flag = 1;
                if (lane == 0) pages_flag(a.c, AERO_CUDA_PAGES_WAIT);
            }
            if (SEL && t >= t0 + cnt && (dead || box_at[stage * 8] == kNoMore)) {
                __syncwarp();
                if (lane == 0 && !dead) mbar_arrive(smem_u32(bars + ST + stage));
                if (++stage == ST) {
                    stage = 0;
                    phase ^= 1u;
                }
                break;
            }
            const uint32_t kb = ring + (uint32_t)stage * Cfg<D>::stage_bytes, vb = kb + (D / 64) * kHalf;
            // (two sums each, of the even and the odd steps: a shorter chain of products)
            float s[NT][4], so[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = so[n][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                uint32_t b[4];
                const int c16 = (ks & 3) * 2 + kcol;
                ldsm4<false>(b, kb + (ks >> 2) * kHalf + krow * 128 + ((c16 ^ (krow & 7)) << 4));
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16<BF16>(ks & 1 ? so[n] : s[n], b, qf[ks][n][0], qf[ks][n][1]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = (s[n][i] + so[n][i]) * a.scale_log2;
            // positions that the token does not see: their scores are -inf and their V rows
            // are taken as zero, whatever their memory holds
            int j, j8;  // positions of the warp's first and ninth row (boxes are of 8 rows or more)
            bool partly;
            if constexpr (SEL) {
                const int rows = min(1 << a.c.page_shift, kUnit), r = warp * 16;
                j = box_at[stage * 8 + r / rows] + (r & (rows - 1));
                j8 = box_at[stage * 8 + (r + 8) / rows] + ((r + 8) & (rows - 1));
                partly = j + 8 > sp.n || j8 + 8 > sp.n;
            } else {
                const int j0 = tile_at(sp, t) * kUnit;
                j = j0 + warp * 16;
                j8 = j + 8;
                partly = j0 + kUnit > sp.n || (j0 < sp.lo && j0 + kUnit > sp.sinks);
            }
            uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;
            if (partly) {
                keep0 = (visible(sp, j + 2 * tq) ? 0x0000FFFFu : 0u) | (visible(sp, j + 2 * tq + 1) ? 0xFFFF0000u : 0u);
                keep1 = (visible(sp, j8 + 2 * tq) ? 0x0000FFFFu : 0u) | (visible(sp, j8 + 2 * tq + 1) ? 0xFFFF0000u : 0u);
                const bool see0 = visible(sp, j + g), see1 = visible(sp, j8 + g);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (!see0) s[n][0] = s[n][1] = -INFINITY;
                    if (!see1) s[n][2] = s[n][3] = -INFINITY;
                }
            }
            float x[2 * NT];
            bool grows = false;
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) {
                x[i] = fmaxf(s[i >> 1][i & 1], s[i >> 1][2 + (i & 1)]);
#pragma unroll
                for (int b = 4; b < 32; b <<= 1) x[i] = fmaxf(x[i], __shfl_xor_sync(0xffffffffu, x[i], b));
                grows |= x[i] > m[i];
            }
            if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i) {
                    const float nm = fmaxf(m[i], x[i]);
                    // (a query head without a visible position stays at -inf; its sums are zero)
                    const float f = nm == -INFINITY ? 0.f : ex2(m[i] - nm);
                    m[i] = nm;
                    l[i] *= f;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        o[k][i >> 1][i & 1] *= f;
                        o[k][i >> 1][2 + (i & 1)] *= f;
                    }
                }
            }
            uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float z0 = m[2 * n] == -INFINITY ? 0.f : lifted<BF16>(m[2 * n], 0.f);
                const float z1 = m[2 * n + 1] == -INFINITY ? 0.f : lifted<BF16>(m[2 * n + 1], 0.f);
                const float p0 = ex2(s[n][0] - z0), p1 = ex2(s[n][1] - z1), p2 = ex2(s[n][2] - z0), p3 = ex2(s[n][3] - z1);
                l[2 * n] += p0 + p2;
                l[2 * n + 1] += p1 + p3;
                // P as two values of the cache's type, its rounding and what that leaves: 2^-22 (f16) or 2^-16
                // (bf16) of a weight are lost. (One value would lose 2^-11 or 2^-8, as much as the output's own
                // rounding; the second product costs 0.5 % of the time, 2 % with wide heads in groups of 16.)
                // The sums l stay f32. Transposed: keys as the product's depth.
                const uint32_t h0 = pack16<BF16>(p0, p1), h1 = pack16<BF16>(p2, p3);
                pb[n][0] = transpose8(h0);
                pb[n][1] = transpose8(h1);
                pl[n][0] = transpose8(pack16<BF16>(p0 - low16<BF16>(h0), p1 - low16<BF16>(h0 >> 16)));
                pl[n][1] = transpose8(pack16<BF16>(p2 - low16<BF16>(h1), p3 - low16<BF16>(h1 >> 16)));
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                uint32_t b[4];
                const int c16 = (i & 3) * 2 + vcol;
                ldsm4<true>(b, vb + (i >> 2) * kHalf + vrow * 128 + ((c16 ^ (vrow & 7)) << 4));
                const uint32_t va[4] = {b[0] & keep0, b[1] & keep0, b[2] & keep1, b[3] & keep1};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma16<BF16>(o[i][n], va, pb[n][0], pb[n][1]);
                    mma16<BF16>(o[i][n], va, pl[n][0], pl[n][1]);
                }
            }
            __syncwarp();
            if (lane == 0 && !dead) mbar_arrive(smem_u32(bars + ST + stage));
            if (++stage == ST) {
                stage = 0;
                phase ^= 1u;
            }
        }
        // ---- the four warps' results into one: o[head][d] = the sum of red's regions, (m, l) in joint
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
#pragma unroll
            for (int b = 4; b < 32; b <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], b);
            if (g == 0) ml[warp * 16 + 8 * (i >> 1) + 2 * tq + (i & 1)] = make_float2(m[i], l[i]);
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        {
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) {
                const int row = 8 * (i >> 1) + 2 * tq + (i & 1);
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int k = 0; k < kConsumers; ++k) M = fmaxf(M, ml[k * 16 + row].x);
#pragma unroll
                for (int k = 0; k < kConsumers; ++k) {
                    const float2 v = ml[k * 16 + row];
                    L += v.x == -INFINITY ? 0.f : v.y * ex2(v.x - M);
                }
                if (warp == 0 && g == 0) joint[row] = make_float2(M, L);
                const float f = m[i] == -INFINITY ? 0.f : ex2(m[i] - M);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    o[k][i >> 1][i & 1] *= f;
                    o[k][i >> 1][2 + (i & 1)] *= f;
                }
            }
            // rows 2 tq (+ 1) of a region, columns exchanged in blocks of 8 by tq: no bank twice
            float* r = red + (warp % kRegions) * 8 * NT * D;
            const auto cell = [&](int k, int n, int i) { return r + (8 * n + 2 * tq + (i & 1)) * D + ((16 * k + (i >> 1) * 8 + g) ^ (8 * tq)); };
            if (warp >= kConsumers - kRegions) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) *cell(k, n, i) = o[k][n][i];
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if constexpr (kRegions < kConsumers) {
                if (warp < kConsumers - kRegions) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) *cell(k, n, i) += o[k][n][i];
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
            }
        }
        if (cnt == sp.tiles) {
            for (int i = tid; i < G * (D / 4); i += 32 * kConsumers) {
                const int row = i / (D / 4), d = i % (D / 4) * 4;
                const float L = joint[row].y, k = L > 0.f ? 1.f / L : L == L ? 0.f : L;  // a sum that is no number stays none
                const float4 v = summed(row, d);
                put(out_of(e, h), row, d, make_float4(v.x * k, v.y * k, v.z * k, v.w * k));
            }
        } else {
            // partial results: slot 1 of the CTA where the (sequence, head) begins, slot 0 of the others
            const int which = t0 == 0;
            float* mine = a.part + ((int64_t)blockIdx.x * 2 + which) * slot;
            for (int i = tid; i < G * (D / 4); i += 32 * kConsumers) {
                const int row = i / (D / 4), d = i % (D / 4) * 4;
                *reinterpret_cast<float4*>(mine + row * D + d) = summed(row, d);
            }
            if (tid < G) *reinterpret_cast<float2*>(mine + 16 * D + 2 * tid) = joint[tid];
            const int64_t seg0 = base + (int64_t)h * (sp.tiles + a.over) + a.over;  // its units: [seg0, seg0 + tiles)
            const int64_t c0 = quotient(seg0, w);
            const int parts = (int)(quotient(seg0 + sp.tiles - 1, w) - c0) + 1;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (tid == 0) {
                // the CTA's stores, ordered before by the barrier; what the others stored, ordered by the barrier below for the
                // whole CTA
                uint32_t before;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.counters + c0) : "memory");
                const bool last = before == (uint32_t)(parts - 1);
                if (last) a.counters[c0] = 0;  // for the next launch
                joins[which] = make_int4(last ? parts : 0, (int)c0, e, h);
            }
        }
        }
        u += pc.line;
        if (u == base + (int64_t)(sp.tiles + a.over) * HK && u < u1) {
            base = u;
            sp = span_of<SEL>(a, ++e);
        }
    }
    // ---- joins of the (at most two) shared (sequence, head)s whose last part this CTA wrote; here,
    // so that neither the arrivals nor the joins hold up the units
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int which = 0; which < 2; ++which) {
        const int parts = joins[which].x;
        if (!parts) continue;
        const int64_t c0 = joins[which].y;
        uint16_t* to = out_of(joins[which].z, joins[which].w);
        // part c of the line: the first one's slot is 1, the others' 0
        const float* first = a.part + (c0 * 2 + 1) * slot;
        const float* rest = a.part + (c0 * 2) * slot;
        const auto part_at = [&](int c) { return c == 0 ? first : rest + (int64_t)c * 2 * slot; };
        // four columns of a row a thread; the loads of kBatch parts are in flight at once
        // (an L2 round trip each batch is what this costs)
        constexpr int kBatch = 16;
        for (int i = tid; i < G * (D / 4); i += 32 * kConsumers) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            float M = -INFINITY, L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int b0 = 0; b0 < parts; b0 += kBatch) {
                float2 x[kBatch];
                float4 v[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const float* p = part_at(min(b0 + k, parts - 1));
                    x[k] = __ldcg(reinterpret_cast<const float2*>(p + 16 * D + 2 * row));
                    v[k] = __ldcg(reinterpret_cast<const float4*>(p + row * D + d));
                }
                float N = M;
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    if (b0 + k >= parts) x[k] = make_float2(-INFINITY, 0.f);
                    N = fmaxf(N, x[k].x);
                }
                const float z = N == -INFINITY ? 0.f : N, f = ex2(M - z);
                M = N;
                L *= f;
                acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {  // (past the last part: its values again, weight 0)
                    const float y = ex2(x[k].x - z);
                    L = fmaf(x[k].y, y, L);
                    acc.x = fmaf(v[k].x, y, acc.x);
                    acc.y = fmaf(v[k].y, y, acc.y);
                    acc.z = fmaf(v[k].z, y, acc.z);
                    acc.w = fmaf(v[k].w, y, acc.w);
                }
            }
            const float k = L > 0.f ? 1.f / L : L == L ? 0.f : L;
            put(to, row, d, make_float4(acc.x * k, acc.y * k, acc.z * k, acc.w * k));
        }
    }
}

template <int D, bool BF16, int NT, bool SEL>
cudaError_t launch(AttendArgs a, const CUtensorMap& kmap, const CUtensorMap& vmap, int n_sm, cudaStream_t s) {
    static thread_local int prepared = -1;  // the device whose attribute this thread has set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (prepared != dev) {
        e = cudaFuncSetAttribute(decode_attend_kernel<D, BF16, NT, SEL>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::smem);
        if (e != cudaSuccess) return e;
        prepared = dev;
    }
    // Beginnings and ends of (sequence, head)s cost about three units each, and are counted where they
    // are many (16 sequences of up to 4096 positions, 4 kv heads: 24.3 -> 22.7 us); where a few long ones
    // are split over all CTAs that would only shift the cuts (one sequence of 4096: 12.9 -> 14.5 us).
    a.over = (int64_t)a.T * a.c.HK >= 32 ? 3 : 0;
    // no more CTAs than units the tables can hold
    const int64_t cap = ((int64_t)(SEL ? std::min(a.width, a.c.max_pages) : a.c.max_pages) << a.c.page_shift) / kUnit + 2 + a.over;
    const int64_t units = (int64_t)a.T * a.c.HK * cap;
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>((int64_t)n_sm * Cfg<D>::ctas, units));
    return launch_in_turn(decode_attend_kernel<D, BF16, NT, SEL>, grid, kThreads, Cfg<D>::smem, s, a, kmap, vmap);
}

}  // namespace

int pages_decode_max_grid(int n_sm) { return 2 * n_sm; }
size_t pages_decode_part_floats(int D, int n_sm) { return (size_t)pages_decode_max_grid(n_sm) * 2 * 16 * (size_t)(D + 2); }

cudaError_t launch_pages_decode(const AttendArgs& a, bool bf16, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                int n_sm, cudaStream_t s) {
    const auto typed = [&](auto d, auto bf) {
        constexpr int D = decltype(d)::value;
        constexpr bool B = decltype(bf)::value;
        const bool few = a.H / a.c.HK <= 8;
        if (a.blocks) return few ? launch<D, B, 1, true>(a, kmap, vmap, n_sm, s) : launch<D, B, 2, true>(a, kmap, vmap, n_sm, s);
        return few ? launch<D, B, 1, false>(a, kmap, vmap, n_sm, s) : launch<D, B, 2, false>(a, kmap, vmap, n_sm, s);
    };
    const auto sized = [&](auto d) { return bf16 ? typed(d, std::true_type{}) : typed(d, std::false_type{}); };
    switch (a.c.D) {
        case 64: return sized(std::integral_constant<int, 64>{});
        case 128: return sized(std::integral_constant<int, 128>{});
        case 192: return sized(std::integral_constant<int, 192>{});
        case 256: return sized(std::integral_constant<int, 256>{});
    }
    return cudaErrorInvalidValue;
}

}  // namespace aero
