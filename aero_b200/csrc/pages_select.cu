// Bounds of a paged cache's keys and the choice of blocks by them (include/aero_cuda_pages.h).
//
// Bounds. lo[d] and hi[d], the smallest and the largest value in column d of a page's keys of one kv
// head. Bound by HBM: the page's rows are read once, a warp a (page, kv head), 16 bytes a lane
// (32 sequences of 8192 to 16384 positions, 4 heads of 128: 413 MB in 72 us, 5.7 TB/s).
//
// Choice. score(b) = max over the kv head's query heads g of sum_d max(q_gd lo_bd, q_gd hi_bd): no key
// between the bounds has a larger product with any of these heads' queries. As one product with
// depth 2 D: max(q lo, q hi) = q+ hi + q- lo, where q+ and q- are q's positive and negative parts (the
// bounds are finite, so the part that is zero adds nothing). A wrong order of two scores is a wrong block, so what is
// chosen has to follow from sums in 64 bits; those cost 64 products a cycle and SM at best (m8n8k4 products: 48
// sequences of up to 512 blocks, 32 query heads, 16 us of scores). So every score is computed first in f32 (m16n8k16
// products, the operands as they are), off by at most e = 17 2^-23 D / 8 M, M = max_g sum_d |q_gd| max |bounds|. A score is D / 8
// sums of 17 terms (16 products, which are exact, and the sum so far) one after another, and no term or sum exceeds M. Terms are brought
// to the largest one's exponent and cut there, each by 2^-23 of it at most. A sum with that exponent lies on the same grid and is cut no
// further; of one with a higher exponent each of those cuts is half as much or less, so that with the sum's own they are
// (17 / 2 + 1) 2^-23 of it. Measured on a B200, 4 10^8 sums (terms alike, spread, of one sign, one or the sum so far large): 4.0 2^-23 of the larger of the largest term and the sum, at
// most. Only the blocks whose score lies within 2 e of where the least chosen one can be are computed again in 64 bits, a handful; where
// they are many (blocks alike) all are.
//
// Bound by a chain of steps, not by bytes: one sequence of 2048 blocks, 32 query heads on 4 kv heads of 128, 12.7 us, 48
// sequences of up to 512 blocks 18.6 us, 8 sequences with 1 to 9 tokens each 15.6 us, a launch included (all in 64 bits: 18.8, 38.6
// and 34.8 us). Cycles of the first with its inputs in L2, as where that was measured (and from HBM): lengths and queries 2600
// (4400), page numbers, bounds and products 4800 (7900), ends 2400 (2800), a histogram 3600 (3800), blocks near the border, their
// scores and exchange 5800, their order 2800, the list 1100; in all 23,000 (28,500). So 7400 (12,300) of them, 12,600 of
// 23,400 (23,100 of 34,100) for the 48 sequences, are reads one after another before the scores are there, of which the queries, the
// page numbers and the bounds could be on their way at once; the rest are steps with a barrier each.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "pages.h"
#include "pages_mma.cuh"

namespace aero {
namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ bounds
constexpr int kBoundThreads = 256;

template <bool BF16>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {  // of a number and none: the number
    if constexpr (BF16) {
        const __nv_bfloat162 r = __hmin2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 r = __hmin2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}
template <bool BF16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    if constexpr (BF16) {
        const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

// By one warp: the bounds of `rows` rows of D values at k into out (2 x D). Infinities count as the type's
// largest values, what is no number is passed over (a column of nothing else: 0).
template <bool BF16>
__device__ void page_bounds(const uint16_t* k, int rows, int D, uint16_t* out) {
    constexpr uint32_t kMost = BF16 ? 0x7F7F7F7Fu : 0x7BFF7BFFu, kLeast = kMost | 0x80008000u;
    constexpr int U = 8;  // rows in flight a lane
    const int lane = (int)threadIdx.x & 31, pieces = D / 8, groups = 32 / pieces;
    const int piece = lane % pieces, group = lane / pieces;
    const bool mine = group < groups;
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[i] = kMost, hi[i] = kLeast;
    for (int r0 = group; r0 < rows; r0 += groups * U) {
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * groups;
            x[u] = mine && r < rows ? __ldcs(reinterpret_cast<const uint4*>(k + (int64_t)r * D) + piece) : make_uint4(~0u, ~0u, ~0u, ~0u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t w[4] = {x[u].x, x[u].y, x[u].z, x[u].w};  // (all ones: no numbers)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lo[i] = min2<BF16>(lo[i], w[i]);
                hi[i] = max2<BF16>(hi[i], w[i]);
            }
        }
    }
    __syncwarp();
    for (int o = pieces; o < 32 && groups > 1; o <<= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] = min2<BF16>(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
            hi[i] = max2<BF16>(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
        }
    }
    if (lane >= pieces) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo[i] = max2<BF16>(lo[i], kLeast);
        hi[i] = min2<BF16>(hi[i], kMost);
#pragma unroll
        for (int s = 0; s < 32; s += 16)
            if (low16<BF16>(lo[i] >> s) > low16<BF16>(hi[i] >> s)) {
                lo[i] &= ~(0xFFFFu << s);
                hi[i] &= ~(0xFFFFu << s);
            }
    }
    reinterpret_cast<uint4*>(out)[piece] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    reinterpret_cast<uint4*>(out + D)[piece] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
}

// The bounds of page `page` of kv head h of `layer`, whose first `rows` rows are a sequence's.
template <bool BF16>
__device__ __forceinline__ void bound(const PageView& c, int layer, const uint16_t* k, int page, int h, int rows) {
    const int64_t at = ((int64_t)layer * c.n_page + page) * c.HK + h;
    page_bounds<BF16>(k + (at << c.page_shift) * c.D, rows, c.D, c.bounds + at * 2 * c.D);
}

// Every page of the n listed sequences: (page, kv head)s of one sequence after another, dealt to the warps in turn.
template <bool BF16>
__global__ void __launch_bounds__(kBoundThreads, 4) set_bounds_kernel(PageView c, int layer, const uint16_t* k, const int32_t* seqs, int n) {
    stream_turn();
    const int lane = (int)threadIdx.x & 31;
    const int64_t nw = (int64_t)gridDim.x * (kBoundThreads / 32);
    const int64_t w = (int64_t)blockIdx.x * (kBoundThreads / 32) + (threadIdx.x >> 5);
    int64_t base = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + lane, s = i < n ? seqs[i] : 0;
        if (i < n && (s < 0 || s >= c.n_seq) && w == 0) pages_flag(c, AERO_CUDA_PAGES_BAD_SEQ);
        const int len = i < n ? pages_length(c, s) : 0;
        int64_t incl = (int64_t)(((int64_t)len + (1 << c.page_shift) - 1) >> c.page_shift) * c.HK;
        const int64_t items = incl;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        const int64_t total = __shfl_sync(0xffffffffu, incl, 31), excl = incl - items;
        for (int64_t x = (w + nw - base % nw) % nw; x < total; x += nw) {
            const int j = __popc(__ballot_sync(0xffffffffu, incl <= x));
            const int64_t in = x - __shfl_sync(0xffffffffu, excl, j);
            const int sj = __shfl_sync(0xffffffffu, s, j), lj = __shfl_sync(0xffffffffu, len, j);
            const int slot = (int)(in / c.HK), h = (int)(in % c.HK);
            const int page = c.table[(int64_t)sj * c.max_pages + slot];
            if ((uint32_t)page >= (uint32_t)c.n_page) {
                pages_flag(c, AERO_CUDA_PAGES_BAD_PAGE);
                continue;
            }
            // (a page of several sequences, whose lengths may differ, whole: the warps that take it write the same)
            const int rows = c.refs[page] > 1 ? 1 << c.page_shift : lj - (slot << c.page_shift);
            bound<BF16>(c, layer, k, page, h, min(1 << c.page_shift, rows));
        }
        base += total;
    }
}

// The pages that T appended tokens went to. Of tokens that follow one another in the list and in a page the last
// one's warp takes it, so a prompt's page is read once; what an append refuses is left.
template <bool BF16>
__global__ void __launch_bounds__(kBoundThreads, 4) append_bounds_kernel(PageView c, int layer, const uint16_t* k, const int32_t* seqs,
                                                                       const int32_t* positions, int T) {
    stream_turn();
    const int64_t nw = (int64_t)gridDim.x * (kBoundThreads / 32), all = (int64_t)T * c.HK;
    for (int64_t x = (int64_t)blockIdx.x * (kBoundThreads / 32) + (threadIdx.x >> 5); x < all; x += nw) {
        const int t = (int)(x / c.HK), h = (int)(x % c.HK);
        const int s = seqs[t], p = positions[t], slot = p >> c.page_shift;
        if (t + 1 < T && seqs[t + 1] == s && positions[t + 1] >> c.page_shift == slot && positions[t + 1] < pages_length(c, s)) continue;
        if (s < 0 || s >= c.n_seq || p < 0 || p >= pages_length(c, s)) continue;
        const int page = c.table[(int64_t)s * c.max_pages + slot];
        if ((uint32_t)page >= (uint32_t)c.n_page || c.refs[page] > 1) continue;
        bound<BF16>(c, layer, k, page, h, min(1 << c.page_shift, pages_length(c, s) - (slot << c.page_shift)));
    }
}

// ------------------------------------------------------------------ the choice of blocks
// A cluster of CTAs per (token, kv head), each with an even share of its blocks in their order. Scores become
// 64-bit keys that order as they do and stay in shared memory; the least chosen key is found by histograms over
// the interval that holds it, narrowed by a factor of kBins each time (a cluster barrier each, once
// or twice for scores of a few thousand blocks); then each CTA writes its chosen blocks in order behind
// those of the CTAs before it. Counts are integers and ties go to the lowest block, so timing changes nothing.
constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32;
constexpr int kBins = kSelThreads;  // (reads of peers' memory are slow: two or three levels of 512 rather than of 2048)
constexpr int kSelCluster = 8;
constexpr int kMostKeys = kSelectPages / kSelCluster;
constexpr unsigned long long kAlways = ~0ull;  // the key of a block that is chosen whatever its score (no score has it)

using u64 = unsigned long long;

// D (8x8) += A (8x4) x B (4x8) in 64 bits.
__device__ __forceinline__ void mma64(double (&d)[2], double a, double b) {
    asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};" : "+d"(d[0]), "+d"(d[1]) : "d"(a), "d"(b));
}

// Keys in the order of the scores; -0 as 0, no number as +infinity.
__device__ __forceinline__ u64 key_of(double score) {
    const double s = score == score ? score + 0.0 : (double)INFINITY;
    const u64 b = (u64)__double_as_longlong(s);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

template <int D, int NT>
constexpr int query_bytes() {  // of the query heads' fragments in 64 bits
    return NT * 8 * 2 * D * 8;
}

constexpr int kNear = 64;  // blocks of a CTA whose scores are computed again

// Keys of scores in f32.
__device__ __forceinline__ uint32_t key32_of(float score) {
    const uint32_t b = __float_as_uint(score + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float score32_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7FFFFFFFu : ~key); }
constexpr uint32_t kAlways32 = ~0u;

// What a CTA of the cluster tells the others.
struct Told {
    uint32_t lo, hi;    // keys
    float most;         // the largest bound
    int chosen, sure, near;
    u64 near_key[kNear];
    int near_block[kNear];
};

// NT: tiles of 8 query heads.
template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(kSelThreads, 2) select_kernel(const SelectArgs a) {
    constexpr int KS = D / 32;             // 16-byte pieces of a bound's row a lane takes
    constexpr int NU = D <= 128 ? 2 : 1;   // tiles of 8 blocks a warp has in hand
    extern __shared__ __align__(16) uint8_t smem[];
    double* qf = reinterpret_cast<double*>(smem);                                          // [NT][2][KS][8][32]
    uint32_t* hist = reinterpret_cast<uint32_t*>(smem + query_bytes<D, NT>());             // [2][kBins]
    u64* keys = reinterpret_cast<u64*>(smem + query_bytes<D, NT>() + 2 * kBins * 4);
    __shared__ u64 least[kSelWarps], most64[kSelWarps], range[2];
    __shared__ uint32_t sums[kSelWarps], found[3], mine[1];
    __shared__ float sizes[NT * 8], bounds_of[kSelWarps];
    __shared__ Told told[kSelCluster];
    __shared__ int near;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int HK = a.c.HK, G = a.H / HK, P = 1 << a.c.page_shift;
    const int pair = (int)blockIdx.x / C, t = pair / HK, h = pair % HK;
    cluster_begun(C);
    stream_turn();
    if (blockIdx.x == 0 && a.q_start) check_q_start(a);
    int seq, n;
    token_rows(a, t, seq, n);
    if (tid == 0 && (seq < 0 || seq >= a.c.n_seq)) pages_flag(a.c, AERO_CUDA_PAGES_BAD_SEQ);
    const int W = a.width, nb = n > 0 ? (n + P - 1) >> a.c.page_shift : 0;
    int32_t* list = a.out + (int64_t)pair * W;
    // the blocks that are chosen always: [0, f1) and [r0_, nb)
    const int f1 = min(a.first, nb), r0_ = max(nb - a.recent, f1);
    int need = W - (f1 + nb - r0_);
    if (nb <= W || need <= 0) {
        // all of them, or no others
        for (int i = rank * kSelThreads + tid; i < W; i += C * kSelThreads)
            list[i] = nb <= W ? (i < nb ? i : -1) : i < f1 ? i : r0_ + i - f1;
        cluster_all_begun(C);
        return;
    }
    cluster_all_begun(C);
    const int per = ((nb + C - 1) / C + 15) & ~15;
    const int b0 = min(nb, rank * per), b1 = min(nb, b0 + per);
    const uint16_t* const q = static_cast<const uint16_t*>(a.q) + (int64_t)t * a.q_token + (int64_t)(h * G) * a.q_head;
    const uint16_t* const bounds = a.c.bounds + (int64_t)h * 2 * D;
    const auto page_of = [&](int b) { return b < b1 ? a.c.table[(int64_t)seq * a.c.max_pages + b] : -1; };
    const auto row_of = [&](int page) { return bounds + ((int64_t)a.layer * a.c.n_page + page) * HK * 2 * D; };
    // the sum of the numbers of the threads before this one, and of all
    const auto scan = [&](uint32_t v, uint32_t& all) {
        uint32_t incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = incl;
        __syncthreads();
        uint32_t before = 0;
        all = 0;
#pragma unroll
        for (int i = 0; i < kSelWarps; ++i) {
            before += i < warp ? sums[i] : 0;
            all += sums[i];
        }
        return before + incl - v;
    };
    if (a.vec) {
        // ---- scores in f32. The query heads' parts as the products' columns: a warp a head
        uint2* const frag = reinterpret_cast<uint2*>(smem);  // [NT][2][KS][2][32]
        uint32_t* const keys32 = reinterpret_cast<uint32_t*>(keys);
        for (int i = tid; i < 2 * kBins; i += kSelThreads) hist[i] = 0;
        for (int head = warp; head < NT * 8; head += kSelWarps) {
            float size = 0.f;
            if (lane < D / 8) {
                const uint4 x = *reinterpret_cast<const uint4*>(q + (int64_t)(head % G) * a.q_head + lane * 8);  // (heads past G: the first ones again)
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                uint32_t neg[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    neg[j] = w[j] & ((w[j] >> 15 & 0x10001u) * 0xFFFFu);
                    size += fabsf(low16<BF16>(w[j])) + fabsf(low16<BF16>(w[j] >> 16));
                }
                uint2* to = frag + ((head / 8 * 2) * KS + lane / 4) * 64 + (head % 8) * 4 + lane % 4;
                to[0] = make_uint2(neg[0], neg[1]);  // with the lower bounds
                to[32] = make_uint2(neg[2], neg[3]);
                to[KS * 64] = make_uint2(w[0] ^ neg[0], w[1] ^ neg[1]);  // with the upper ones
                to[KS * 64 + 32] = make_uint2(w[2] ^ neg[2], w[3] ^ neg[3]);
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) size += __shfl_xor_sync(0xffffffffu, size, o);
            if (lane == 0) sizes[head] = size;
        }
        __syncthreads();
        uint32_t lo = ~0u, hi = 0, most = 0;
        for (int base = b0 + warp * 16; base < b1; base += kSelWarps * 16) {
            const int p0 = page_of(base + lane / 4), p1 = page_of(base + 8 + lane / 4);
            const bool g0 = (uint32_t)p0 < (uint32_t)a.c.n_page, g1 = (uint32_t)p1 < (uint32_t)a.c.n_page;
            if ((!g0 && base + lane / 4 < b1) || (!g1 && base + 8 + lane / 4 < b1)) pages_flag(a.c, AERO_CUDA_PAGES_BAD_PAGE);
            const uint4 *r0 = reinterpret_cast<const uint4*>(row_of(p0)) + lane % 4, *r1 = reinterpret_cast<const uint4*>(row_of(p1)) + lane % 4;
            float acc[NT][4];
#pragma unroll
            for (int m = 0; m < NT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
            constexpr int PH = D / 64;  // (four pieces of each row at a time, so that two CTAs fit an SM)
#pragma unroll
            for (int half = 0; half < PH; ++half) {
                constexpr int N = 2 * KS / PH;
                uint4 x[N], y[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    x[i] = g0 ? __ldcg(r0 + 4 * (half * N + i)) : make_uint4(0u, 0u, 0u, 0u);
                    y[i] = g1 ? __ldcg(r1 + 4 * (half * N + i)) : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    constexpr uint32_t kSize = 0x7FFF7FFFu;
                    most = max2<BF16>(most, max2<BF16>(max2<BF16>(x[i].x & kSize, x[i].y & kSize), max2<BF16>(x[i].z & kSize, x[i].w & kSize)));
                    most = max2<BF16>(most, max2<BF16>(max2<BF16>(y[i].x & kSize, y[i].y & kSize), max2<BF16>(y[i].z & kSize, y[i].w & kSize)));
#pragma unroll
                    for (int m = 0; m < NT; ++m) {
                        const uint2* f = frag + ((m * 2) * KS + half * N + i) * 64 + lane;
                        const uint2 f0 = f[0], f1 = f[32];
                        const uint32_t a0[4] = {x[i].x, y[i].x, x[i].y, y[i].y}, a1[4] = {x[i].z, y[i].z, x[i].w, y[i].w};
                        mma16<BF16>(acc[m], a0, f0.x, f0.y);
                        mma16<BF16>(acc[m], a1, f1.x, f1.y);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float v = fmaxf(acc[0][2 * e], acc[0][2 * e + 1]);
#pragma unroll
                for (int m = 1; m < NT; ++m) v = fmaxf(v, fmaxf(acc[m][2 * e], acc[m][2 * e + 1]));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                const int b = base + 8 * e + lane / 4;
                if (lane % 4 == 0 && b < b1) {
                    const bool always = b < f1 || b >= r0_;
                    const uint32_t k = key32_of(v);
                    keys32[b - b0] = always ? kAlways32 : k;
                    if (!always) {
                        lo = min(lo, k);
                        hi = max(hi, k);
                    }
                }
            }
        }
        // ---- all CTAs' ends, and how far the scores may be off
        float bound = fmaxf(low16<BF16>(most), low16<BF16>(most >> 16));
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
        if (lane == 0) least[warp] = lo, most64[warp] = hi, bounds_of[warp] = bound;
        __syncthreads();
        if (tid < C) {
            for (int i = 0; i < kSelWarps; ++i) {
                lo = min(lo, (uint32_t)least[i]);
                hi = max(hi, (uint32_t)most64[i]);
                bound = fmaxf(bound, bounds_of[i]);
            }
            Told& to = cluster.map_shared_rank(told, tid)[rank];
            to.lo = lo;
            to.hi = hi;
            to.most = bound;
        }
        cluster_barrier(C);
        lo = ~0u, hi = 0, bound = 0.f;
        for (int i = 0; i < C; ++i) {
            lo = min(lo, told[i].lo);
            hi = max(hi, told[i].hi);
            bound = fmaxf(bound, told[i].most);
        }
        float size = 0.f;
        bool number = true;
        for (int i = 0; i < NT * 8; ++i) {
            number &= sizes[i] < INFINITY;
            size = fmaxf(size, sizes[i]);
        }
        const float off = size * bound * (5.12e-7f * D) + 2e-35f;  // 2 e (5.07e-7), rounded up, and 2 * 17 * 32 times the least normal number for what underflows
        if (number && off < 1e30f) {
            // ---- an interval that holds the least chosen score: a few blocks' or narrower than what they may be off
            int left = need;
            for (int level = 0; lo != hi; ++level) {
                const int shift = max(0, 23 - __clz((int)(hi - lo)));  // (hi - lo) >> shift < kBins = 2^9
                uint32_t* own = hist + (level & 1) * kBins;
                for (int i = tid; i < b1 - b0; i += kSelThreads) {
                    const uint32_t k = keys32[i];
                    if (k >= lo && k <= hi && k != kAlways32) atomicAdd(own + ((hi - k) >> shift), 1u);
                }
                cluster_barrier(C);
                // the other histogram, read by all before this barrier, is the next one's
                hist[(~level & 1) * kBins + tid] = 0;
                uint32_t v = 0, all;
#pragma unroll 8
                for (int i = 0; i < C; ++i) v += (C > 1 ? cluster.map_shared_rank(own, i) : own)[tid];
                const uint32_t before = scan(v, all);
                if (before < (uint32_t)left && (uint32_t)left <= before + v) {
                    found[0] = (uint32_t)tid;
                    found[1] = before;
                    found[2] = v;
                }
                __syncthreads();
                const uint32_t top = hi - (found[0] << shift), span = (1u << shift) - 1;
                left -= (int)found[1];
                hi = top;
                lo = top - lo > span ? top - span : lo;
                if (found[2] <= 8u * (uint32_t)C || score32_of(hi) - score32_of(lo) <= off) break;
            }
            // ---- blocks above what that leaves open are chosen, those within it computed again
            const uint32_t open_lo = key32_of(score32_of(lo) - off * 1.001f), open_hi = min(key32_of(score32_of(hi) + off * 1.001f), kAlways32 - 1);
            Told& mine = told[rank];
            if (tid == 0) near = 0;
            if (tid < kNear) mine.near_key[tid] = 0;
            __syncthreads();
            uint32_t chosen = 0, sure = 0;
            for (int i = tid; i < b1 - b0; i += kSelThreads) {
                const uint32_t k = keys32[i];
                chosen += k > open_hi;
                sure += k > open_hi && k != kAlways32;
                if (k >= open_lo && k <= open_hi) {
                    const int at = atomicAdd(&near, 1);
                    if (at < kNear) mine.near_block[at] = b0 + i;
                }
            }
            uint32_t both;
            scan(chosen | sure << 16, both);
            const int n = near;
            for (int item = warp; item < min(n, kNear) * G; item += kSelWarps) {
                // a warp a block and query head, columns over the lanes
                const int i = item / G, g = item % G;
                const int page = page_of(mine.near_block[i]);
                const bool good = (uint32_t)page < (uint32_t)a.c.n_page;
                const uint16_t* row = row_of(page);
                double sum = 0.0;
#pragma unroll
                for (int d = 0; d < D / 64; ++d) {
                    const int at = 64 * d + 2 * lane;
                    const uint32_t x = *reinterpret_cast<const uint32_t*>(q + (int64_t)g * a.q_head + at);
                    const uint32_t l = good ? __ldcg(reinterpret_cast<const uint32_t*>(row + at)) : 0u, u = good ? __ldcg(reinterpret_cast<const uint32_t*>(row + D + at)) : 0u;
#pragma unroll
                    for (int e = 0; e < 32; e += 16) {
                        const float y = low16<BF16>(x >> e);
                        sum = fma((double)y, (double)low16<BF16>((y < 0.f ? l : u) >> e), sum);
                    }
                }
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane == 0) atomicMax(&mine.near_key[i], key_of(sum));
            }
            __syncthreads();
            for (int i = tid; i < C * kNear; i += kSelThreads) {
                const int c = i / kNear, e = i % kNear;
                Told& to = C > 1 ? cluster.map_shared_rank(told, c)[rank] : mine;
                if (c != rank && e < min(n, kNear)) {
                    to.near_key[e] = mine.near_key[e];
                    to.near_block[e] = mine.near_block[e];
                }
                if (e == 0) {
                    to.chosen = (int)(both & 0xFFFFu);
                    to.sure = (int)(both >> 16);
                    to.near = n;
                }
            }
            cluster_barrier(C);
            bool few = true;
            int open = need, base = 0;
            for (int i = 0; i < C; ++i) {
                few &= told[i].near <= kNear;
                open -= told[i].sure;
                base += i < rank ? told[i].chosen : 0;
            }
            if (few) {
                // of all CTAs' the `open` highest, equal ones by their number
                if (tid < 2) found[tid] = 0;  // this CTA's, and those before it
                __syncthreads();
                for (int i = tid; i < C * kNear; i += kSelThreads) {
                    const int c = i / kNear, e = i % kNear;
                    if (c > rank || e >= told[c].near) continue;
                    const u64 k = told[c].near_key[e];
                    const int b = told[c].near_block[e];
                    int before = 0;
                    for (int j = 0; j < C; ++j)
                        for (int o = 0; o < told[j].near; ++o) {
                            const u64 other = told[j].near_key[o];
                            before += other > k || (other == k && told[j].near_block[o] < b);
                        }
                    if (before < open) {
                        if (c == rank)
                            keys32[b - b0] = kAlways32;
                        else
                            atomicAdd(found + 1, 1u);
                    }
                }
                __syncthreads();
                base += (int)found[1];
                // ---- the chosen ones, in order: each thread a run of blocks
                const int run = (per + kSelThreads - 1) / kSelThreads;
                const int i0 = min(b1 - b0, tid * run), i1 = min(b1 - b0, i0 + run);
                uint32_t count = 0, all;
                for (int i = i0; i < i1; ++i) count += keys32[i] > open_hi;
                int at = base + (int)scan(count, all);
                for (int i = i0; i < i1; ++i)
                    if (keys32[i] > open_hi) list[at++] = b0 + i;
                return;
            }
        }
    }
    // ---- scores in 64 bits, all of them
    cluster_barrier(C);  // (the memory that others may be reading is written again)
    // ---- the query heads' positive and negative parts, as the products' fragments; heads past G are the first ones again
    {
        for (int i = tid; i < NT * 8 * D; i += kSelThreads) {
            const int head = i / D, d = i % D, c16 = d / 8;
            const float x = to_f32<BF16>(q[(int64_t)(head % G) * a.q_head + d]);
            double* to = qf + (((head / 8 * 2) * KS + c16 / 4) * 8 + d % 8) * 32 + (head % 8) * 4 + c16 % 4;
            to[0] = x > 0.f ? 0.0 : (double)x;               // with the lower bounds
            to[KS * 8 * 32] = x > 0.f ? (double)x : x == x ? 0.0 : (double)x;  // with the upper ones
        }
        for (int i = tid; i < 2 * kBins; i += kSelThreads) hist[i] = 0;
    }
    __syncthreads();
    // ---- scores
    u64 lo = kAlways, hi = 0;
    for (int base = b0 + warp * 8 * NU; base < b1; base += kSelWarps * 8 * NU) {
        uint4 x[NU][2][KS];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int b = base + u * 8 + lane / 4;
            const int page = page_of(b);
            const bool good = (uint32_t)page < (uint32_t)a.c.n_page;
            if (b < b1 && !good) pages_flag(a.c, AERO_CUDA_PAGES_BAD_PAGE);
            const uint16_t* row = row_of(page);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    x[u][p][i] = good ? __ldcg(reinterpret_cast<const uint4*>(row + p * D) + 4 * i + lane % 4) : make_uint4(0u, 0u, 0u, 0u);
        }
        double acc[NU][NT][2];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int m = 0; m < NT; ++m) acc[u][m][0] = acc[u][m][1] = 0.0;
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    double bv[NU];
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        const uint32_t w = j < 2 ? x[u][p][i].x : j < 4 ? x[u][p][i].y : j < 6 ? x[u][p][i].z : x[u][p][i].w;
                        bv[u] = (double)to_f32<BF16>((uint16_t)(w >> 16 * (j & 1)));
                    }
#pragma unroll
                    for (int m = 0; m < NT; ++m) {
                        const double av = qf[(((m * 2 + p) * KS + i) * 8 + j) * 32 + lane];
#pragma unroll
                        for (int u = 0; u < NU; ++u) mma64(acc[u][m], av, bv[u]);
                    }
                }
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                u64 k = key_of(acc[u][0][e]);
#pragma unroll
                for (int m = 1; m < NT; ++m) k = max(k, key_of(acc[u][m][e]));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
                const int b = base + u * 8 + 2 * (lane & 3) + e;
                if (lane < 4 && b < b1) {
                    const bool always = b < f1 || b >= r0_;
                    keys[b - b0] = always ? kAlways : k;
                    if (!always) {
                        lo = min(lo, k);
                        hi = max(hi, k);
                    }
                }
            }
    }
    // ---- the interval of all keys
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (lane == 0) least[warp] = lo, most64[warp] = hi;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kSelWarps; ++i) {
            lo = min(lo, least[i]);
            hi = max(hi, most64[i]);
        }
        range[0] = lo;
        range[1] = hi;
    }
    cluster_barrier(C);
    lo = kAlways, hi = 0;
    for (int i = 0; i < C; ++i) {
        const u64* r = cluster.map_shared_rank(range, i);
        lo = min(lo, r[0]);
        hi = max(hi, r[1]);
    }
    // ---- the need-th key from above: all above `edge` are chosen, and the first `ties` blocks with it
    u64 edge = lo;
    int ties = need;
    for (int level = 0; lo != hi; ++level) {
        const int shift = max(0, 55 - __clzll((long long)(hi - lo)));  // (hi - lo) >> shift < kBins = 2^9
        uint32_t* own = hist + (level & 1) * kBins;
        for (int i = tid; i < b1 - b0; i += kSelThreads) {
            const u64 k = keys[i];
            if (k >= lo && k <= hi) atomicAdd(own + (uint32_t)((hi - k) >> shift), 1u);
        }
        cluster_barrier(C);
        // the other histogram, read by all before this barrier, is the next one's
        hist[(~level & 1) * kBins + tid] = 0;
        uint32_t v = 0, all;
        for (int i = 0; i < C; ++i) v += cluster.map_shared_rank(own, i)[tid];
        const uint32_t before = scan(v, all);
        if (before < (uint32_t)need && (uint32_t)need <= before + v) {
            found[0] = (uint32_t)tid;
            found[1] = before;
            found[2] = v;
        }
        __syncthreads();
        const u64 top = hi - ((u64)found[0] << shift), span = (1ull << shift) - 1;
        need -= (int)found[1];
        hi = top;
        lo = top - lo > span ? top - span : lo;
        edge = lo;
        ties = need;
        if (found[2] == (uint32_t)need) {
            ties = 1 << 30;  // the whole interval: all from `edge` on
            break;
        }
        __syncthreads();  // found and sums may be written again
    }
    // ---- the chosen ones, in order: each thread a run of blocks
    const int run = (per + kSelThreads - 1) / kSelThreads;
    const int i0 = min(b1 - b0, tid * run), i1 = min(b1 - b0, i0 + run);
    uint32_t count = 0;  // above the edge; in the high half, on it
    for (int i = i0; i < i1; ++i) count += (keys[i] > edge) + ((uint32_t)(keys[i] == edge) << 16);
    uint32_t all;
    const uint32_t before = scan(count, all);
    if (tid == 0) mine[0] = all;
    cluster_barrier(C);
    int above = (int)(before & 0xFFFFu), on = (int)(before >> 16);
    for (int i = 0; i < rank; ++i) {
        const uint32_t x = *cluster.map_shared_rank(mine, i);
        above += (int)(x & 0xFFFFu);
        on += (int)(x >> 16);
    }
    for (int i = i0; i < i1; ++i) {
        const u64 k = keys[i];
        if (k > edge) {
            list[above + min(on, ties)] = b0 + i;
            ++above;
        } else if (k == edge) {
            if (on < ties) list[above + on] = b0 + i;
            ++on;
        }
    }
    cluster_barrier(C);  // no CTA ends while another reads its memory
}

template <int D, bool BF16, int NT>
cudaError_t launch(const SelectArgs& a, int n_sm, cudaStream_t s) {
    static thread_local int prepared = -1;  // the device whose attribute this thread has set
    constexpr int kFixed = query_bytes<D, NT>() + 2 * kBins * 4;
    static_assert(kFixed + kMostKeys * 8 + kSelCluster * sizeof(Told) + 512 <= 226 * 1024, "shared memory of a CTA");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (prepared != dev) {
        e = cudaFuncSetAttribute(select_kernel<D, BF16, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + kMostKeys * 8);
        if (e != cudaSuccess) return e;
        prepared = dev;
    }
    // As many CTAs a (token, kv head) as fill the SMs twice, none with less than a round of blocks, and as many
    // as the keys of the longest sequence need.
    const int64_t pairs = (int64_t)a.T * a.c.HK;
    int C = 1;
    while (C < kSelCluster && (a.c.max_pages > 6144 * C || (pairs * C <= n_sm && a.c.max_pages > 128 * C))) C *= 2;
    const int keys = ((a.c.max_pages + C - 1) / C + 15) & ~15;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)C;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(pairs * C));
    c.blockDim = dim3(kSelThreads);
    c.dynamicSmemBytes = (size_t)kFixed + (size_t)keys * 8;
    c.stream = s;
    c.attrs = at;
    c.numAttrs = 2;
    return cudaLaunchKernelEx(&c, select_kernel<D, BF16, NT>, a);
}

}  // namespace

cudaError_t launch_set_bounds(const PageView& c, bool bf16, int layer, const void* k, const int32_t* seqs, int n, int n_sm,
                              cudaStream_t s) {
    const unsigned grid = (unsigned)(n_sm * 4);
    const uint16_t* rows = static_cast<const uint16_t*>(k);
    return bf16 ? launch_in_turn(set_bounds_kernel<true>, grid, kBoundThreads, 0, s, c, layer, rows, seqs, n)
                : launch_in_turn(set_bounds_kernel<false>, grid, kBoundThreads, 0, s, c, layer, rows, seqs, n);
}

cudaError_t launch_append_bounds(const PageView& c, bool bf16, int layer, const void* k, const int32_t* seqs,
                                 const int32_t* positions, int T, int n_sm, cudaStream_t s) {
    const int64_t warps = (int64_t)T * c.HK;
    const unsigned grid = (unsigned)std::min<int64_t>((warps + kBoundThreads / 32 - 1) / (kBoundThreads / 32), (int64_t)n_sm * 4);
    const uint16_t* rows = static_cast<const uint16_t*>(k);
    return bf16 ? launch_in_turn(append_bounds_kernel<true>, grid, kBoundThreads, 0, s, c, layer, rows, seqs, positions, T)
                : launch_in_turn(append_bounds_kernel<false>, grid, kBoundThreads, 0, s, c, layer, rows, seqs, positions, T);
}

cudaError_t launch_select(const SelectArgs& a, bool bf16, int n_sm, cudaStream_t s) {
    const auto typed = [&](auto d, auto bf) {
        constexpr int D = decltype(d)::value;
        constexpr bool B = decltype(bf)::value;
        return a.H / a.c.HK <= 8 ? launch<D, B, 1>(a, n_sm, s) : launch<D, B, 2>(a, n_sm, s);
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
