// A token drawn from each row of a batch's logits (include/aero_cuda_pages.h, aero_cuda_logits_sample).
//
// In falling order of the logits, equal ones by their number, with weights w_j = 2^(-(m - x_j) log2(e) / T): every
// limit (top_k, top_p, min_p) keeps a prefix of that order, so what is kept is said by one number, its sum S, and the
// token is the first whose running sum exceeds u S. Nothing is sorted as a whole and nothing is written but the token:
// each question is "which is the first in the order whose running sum (or number) reaches a limit?", answered by a
// histogram of the row (counts and sums over kBins slices of its values), then by the members of the one slice that
// holds the answer, gathered and sorted by themselves. A slice with more than kMembers is divided again by
// its keys; one of equal keys is answered by arithmetic and its members' order.
//
// Weights are whole numbers, multiples of 2^-B of the largest (B = 44 for a vocabulary of 2^18): their sums
// are exact in any order, so histograms may be made by atomics and the answer does not depend on timing. Each weight is
// computed in 64 bits and off by half of 2^-B at most, so a sum of V of them by V / 2 2^-B of the largest at the
// very most (2^-27 for V = 2^18).
//
// A cluster of CTAs per row, each with an even share of the row, which it reads from HBM once and two to four
// times more from the caches; the first CTA's shared memory holds the row's sums and members.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "../../include/aero_cuda_pages.h"
#include "internal.h"
#include "pages.h"

namespace aero {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleCluster = 8;
constexpr int kBins = 4 * kSampleThreads, kLast = kBins - 1;
constexpr int kMembers = 2048;
constexpr int kFew = kSampleThreads / 4;  // members put in order by counting
constexpr int kMostVocab = 1 << 22;
constexpr float kMostFloat = 3.402823466e38f;
constexpr double kTwo52 = 4503599627370496.0;

struct SampleArgs {
    const void* in;
    int64_t ld;
    int vocab, slice, bits;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int32_t* token;
    float* logprob;
};

// Keys in the values' order, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7FFFFFFFu : ~key); }

template <typename E>
__device__ __forceinline__ float to_f(E v) {
    if constexpr (sizeof(E) == 4)
        return v;
    else if constexpr (std::is_same<E, __half>::value)
        return __half2float(v);
    else
        return __bfloat162float(v);
}
// The j-th value of a 32-bit word.
template <typename E>
__device__ __forceinline__ float value_in(uint32_t w, int j) {
    if constexpr (sizeof(E) == 4)
        return __uint_as_float(w);
    else if constexpr (std::is_same<E, __half>::value)
        return __half2float(__ushort_as_half((uint16_t)(w >> 16 * j)));
    else
        return __uint_as_float(j ? w & 0xFFFF0000u : w << 16);
}

// What all threads know of a row. Its values are divided into kBins slices, slice b around m - b step; the last one holds
// what lies 36 T and more below m, whose weights (e^-36 < 2^-51) are 0 as multiples of 2^-48 or more, and what is never
// drawn (-infinity and no numbers).
struct Row {
    float m;             // the largest logit
    float half_m, scale; // slice = (m / 2 - x / 2) * scale (halves: the difference of any two numbers is one)
    double per_t;        // 1 / T
    double grid;         // step / T
    double least;        // min_p 2^B
    double lift;         // 2^B
    // (as a number beside 2^23, for comparisons)
    __device__ __forceinline__ float slice(float x) const { return fminf(fmaf(x, -0.5f, half_m) * scale, (float)kLast) + 8388608.f; }
    __device__ __forceinline__ int bin(float x) const { return (int)(__float_as_uint(slice(x)) & (kBins - 1)); }
    // 2^B e^((x - m) / T) in 64 bits, for slices but the last: with y = (x - m) / T + b step / T, at most 0.009 either way, the
    // table's value e^(-b step / T) 2^B times e^y by its series, whose first term left out is below 10^-15
    __device__ __forceinline__ double weight(float x, int b, const double* table) const {
        const double t = (double)x - (double)m;
        const double y = fma(t, per_t, (__hiloint2double(0x43300000, b) - kTwo52) * grid);
        double p = fma(y, 1.0 / 120, 1.0 / 24);
        p = fma(p, y, 1.0 / 6);
        p = fma(p, y, 0.5);
        p = fma(p, y, 1.0);
        p = fma(p, y, 1.0);
        return p * table[b];
    }
    // the nearest whole number (2^B is at most 2^48)
    static __device__ __forceinline__ u64 whole(double w) { return (u64)__double_as_longlong(w + kTwo52) & 0xFFFFFFFFFFFFFull; }
};

// what the cluster does next
enum { kNumbers, kSums, kLook, kDivide, kGather, kGatherKeys, kTies, kCrowd, kDone };
// what is looked for: the end of what top_k keeps, of what top_p keeps, the token; or, among members that begin with
// the row's first, the end of what top_k keeps and then the rest; or, among the members of the slices that
// can hold them, the end of what top_p keeps and the token
enum { kTopK, kTopP, kDraw, kPrefix, kBoth };

// Where the search for a row's token is: every CTA of the cluster works it out for itself, but what the members say, which the
// first CTA tells the others.
struct Search {
    int op, goal;
    uint32_t lo, hi;     // kDivide, kGatherKeys: keys
    int shift;           // kDivide: slice = (hi - key) >> shift
    int b0, b1, b2;      // kGather: slices [b0, b1] and b2
    int last;            // kGather: the members have the answer for certain; -1: a slice has too many
    uint32_t nth;        // kTies: which of the tokens with key lo, from 1
    float logprob;       // kTies
    uint32_t count_before;         // tokens before the slice in hand
    u64 limit;                     // the running sum, or number (kTopK, kPrefix), to be reached
    u64 mass_before, more_before;  // sums before the slice in hand; kBoth: and before slice b2
    u64 total, kept, likely;       // sums: of the row, of the kept, of those that min_p keeps
};

struct Shared {
    double table[kBins];
    u64 first_mass[kBins];    // the row's first histogram: sums, and first_count
    u64 more_mass[kBins];     // the row's histogram of a slice; the members' weights
    u64 member[kMembers];     // key, then all ones less the token's number (in the first CTA)
    uint32_t own_low[kBins], own_high[kBins], own_count[kBins];  // this CTA's histogram: sums, numbers; zero when not in use
    uint32_t first_count[kBins], more_count[kBins];
    u64 set_member[kFew], set_weight[kFew];
    double coarse[kBins / 32], fine[32];
    u64 warp_mass[kSampleWarps];
    uint32_t warp_count[kSampleWarps], warp_lo[kSampleWarps], warp_hi[kSampleWarps];
    float2 ends[kSampleCluster], warp_ends[kSampleWarps];  // largest and smallest of the CTAs, of the warps
    u64 likely[kSampleCluster];
    uint32_t ties[kSampleCluster];
    uint32_t members, staged, base;
    Row row;
    Search find;
    float u, p, min_p;
    int k, few, table_made, fresh;
    int at[2];
    u64 at_mass[2], at_own[2], at_one;
    uint32_t at_count[2], at_members[2];
};
static_assert(sizeof(Shared) <= 113 * 1024, "two CTAs an SM");

// Each part below is a function of its own, with the registers it needs: what runs once is bound by fetching its
// instructions, what runs over the row by its own loop.
__device__ __forceinline__ Shared& shared() {
    extern __shared__ __align__(16) uint8_t smem[];
    return *reinterpret_cast<Shared*>(smem);
}
__device__ __noinline__ double exp_of(double x) { return exp(x); }
__device__ __noinline__ double log_of(double x) { return log(x); }
__device__ __forceinline__ float logprob_of(const Row& r, float x, u64 kept) {
    return (float)(((double)x - (double)r.m) * r.per_t - log_of((double)kept / r.lift));
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ void clear(Shared& s) {
#pragma unroll 1
    for (int i = (int)threadIdx.x; i < 3 * kBins / 4; i += kSampleThreads) reinterpret_cast<uint4*>(s.own_low)[i] = make_uint4(0u, 0u, 0u, 0u);
}

// u S as the running sum to be reached: the first above it.
__device__ __forceinline__ u64 drawn(float u, u64 kept) {
    const double v = u > 0.f ? fmin((double)u, 1.0) * (double)kept : 0.0;
    return min((u64)v + 1, kept);
}
// p S, likewise: the kept ones end with the first that reaches it.
__device__ __forceinline__ u64 nucleus(float p, u64 sum) {
    const double v = p > 0.f ? ceil((double)p * (double)sum) : 1.0;
    return min(max((u64)v, 1ull), sum);
}

// The next goal, once a prefix's sum is known.
__device__ __noinline__ void next_goal(u64 kept) {
    Shared& s = shared();
    Search& f = s.find;
    if (f.goal == kTopK && s.p < 1.f) {
        f.goal = kTopP;
        f.limit = nucleus(s.p, kept);
    } else {
        f.goal = kDraw;
        f.kept = min(kept, f.likely);
        f.limit = drawn(s.u, f.kept);
    }
    f.op = kLook;
}

// The lowest key whose slice is at most b (slices do not rise with the key).
__device__ __noinline__ uint32_t lowest_key(int b) {
    const Row r = shared().row;
    uint32_t lo = key_of(-kMostFloat), hi = key_of(r.m);
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (r.bin(value_of(mid)) <= b)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

// (hi - lo) >> shift < kBins = 2^11
__device__ __forceinline__ int shift_of(uint32_t span) { return max(0, 21 - __clz((int)span)); }

// A thread's four slices of a histogram and what lies before them.
struct Slices {
    u64 mass, mass4[4];
    uint32_t count, count4[4];
    // mass, count: of all before the histogram's first; every thread calls it
    __device__ __forceinline__ void scan(Shared& s, u64 mass_before, uint32_t count_before) {
        const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
        const u64 m0 = mass4[0] + mass4[1] + mass4[2] + mass4[3];
        const uint32_t c0 = count4[0] + count4[1] + count4[2] + count4[3];
        u64 m = m0;
        uint32_t c = c0;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const u64 x = __shfl_up_sync(0xffffffffu, m, o);
            const uint32_t y = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) m += x, c += y;
        }
        if (lane == 31) s.warp_mass[warp] = m, s.warp_count[warp] = c;
        __syncthreads();
        mass = m - m0 + mass_before;
        count = c - c0 + count_before;
#pragma unroll 1
        for (int i = 0; i < warp; ++i) mass += s.warp_mass[i], count += s.warp_count[i];
    }
    // the slice that holds the answer to a limit into at[j]
    __device__ __forceinline__ void pick(Shared& s, bool by_count, int j, u64 limit) const {
        u64 m = mass;
        uint32_t c = count;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u64 had = by_count ? c : m, has = by_count ? c + count4[i] : m + mass4[i];
            if (had < limit && limit <= has) {
                s.at[j] = 4 * (int)threadIdx.x + i;
                s.at_mass[j] = m;
                s.at_own[j] = mass4[i];
                s.at_count[j] = c;
                s.at_members[j] = count4[i];
            }
            m += mass4[i];
            c += count4[i];
        }
    }
};

// f(four values, the first one's token) for a CTA's tokens; values past the last one are -infinity. Two 16-byte pieces a
// thread are on their way while two are looked at.
template <typename E, typename F>
__device__ __forceinline__ void each(const E* in, int v0, int nv, F f) {
    constexpr int PER = 4 / (int)sizeof(E), V = 4 * PER;
    const int tid = (int)threadIdx.x, vecs = ((uintptr_t)in & 15) == 0 ? nv / V : 0;
    const uint4* v = reinterpret_cast<const uint4*>(in);
    const auto piece = [&](const uint4& raw, int i) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = value_in<E>(w[(j + e) / PER], (j + e) % PER);
            f(x, v0 + i * V + j);
        }
    };
    uint4 one = make_uint4(0u, 0u, 0u, 0u), two = one;
    if (tid < vecs) one = v[tid];
    if (tid + kSampleThreads < vecs) two = v[tid + kSampleThreads];
#pragma unroll 1
    for (int i = tid; i < vecs; i += 2 * kSampleThreads) {
        const uint4 now = one, then = two;
        if (i + 2 * kSampleThreads < vecs) one = v[i + 2 * kSampleThreads];
        if (i + 3 * kSampleThreads < vecs) two = v[i + 3 * kSampleThreads];
        piece(now, i);
        if (i + kSampleThreads < vecs) piece(then, i + kSampleThreads);
    }
#pragma unroll 1
    for (int i = vecs * V + 4 * tid; i < nv; i += 4 * kSampleThreads) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = i + e < nv ? to_f(in[i + e]) : -INFINITY;
        f(x, v0 + i);
    }
}

// Four weights into this CTA's histogram: a 64-bit sum as two of 32 bits.
__device__ __forceinline__ void add4(Shared& s, const int (&b)[4], const u64 (&n)[4]) {
    uint32_t was[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) was[e] = atomicAdd(&s.own_low[b[e]], (uint32_t)n[e]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t high = (uint32_t)(n[e] >> 32) + (was[e] + (uint32_t)n[e] < was[e]);
        if (high) atomicAdd(&s.own_high[b[e]], high);
    }
}

template <typename E>
__device__ __noinline__ void numbers_pass(const E* in, int nv) {
    Shared& s = shared();
    const Row r = s.row;
    each<E>(in, 0, nv, [&](const float (&x)[4], int) {
#pragma unroll
        for (int e = 0; e < 4; ++e) atomicAdd(&s.own_count[r.bin(x[e])], 1u);
    });
}

// FULL: numbers too, and returns the sum of this thread's weights that min_p keeps.
template <typename E, bool FULL>
__device__ __noinline__ u64 sums_pass(const E* in, int nv) {
    Shared& s = shared();
    const Row r = s.row;
    u64 likely = 0;
    each<E>(in, 0, nv, [&](const float (&x)[4], int) {
        int b[4];
        u64 n[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            b[e] = r.bin(x[e]);
            const double w = r.weight(x[e], b[e], s.table);
            n[e] = b[e] == kLast ? 0 : Row::whole(w);
            if (FULL) {
                if (w >= r.least && b[e] != kLast) likely += n[e];
                atomicAdd(&s.own_count[b[e]], 1u);
            }
        }
        add4(s, b, n);
    });
    return likely;
}

template <typename E>
__device__ __noinline__ void divide_pass(const E* in, int nv) {
    Shared& s = shared();
    const Row r = s.row;
    const uint32_t lo = s.find.lo, hi = s.find.hi;
    const int shift = s.find.shift;
    each<E>(in, 0, nv, [&](const float (&x)[4], int) {
        int b[4];
        u64 n[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t key = key_of(x[e]);
            const bool is = key >= lo && key <= hi;
            const int from = r.bin(x[e]);
            b[e] = is ? (int)((hi - key) >> shift) : 0;
            n[e] = is && from != kLast ? Row::whole(r.weight(x[e], from, s.table)) : 0;
            if (is) atomicAdd(&s.own_count[b[e]], 1u);
        }
        add4(s, b, n);
    });
}

// The members into this CTA's memory (its histogram's place).
template <typename E, bool KEYS>
__device__ __noinline__ void gather_pass(const E* in, int v0, int nv) {
    Shared& s = shared();
    const Row r = s.row;
    const uint32_t lo = s.find.lo, hi = s.find.hi;
    const float f0 = 8388608.f + (float)s.find.b0, f1 = 8388608.f + (float)s.find.b1, f2 = 8388608.f + (float)s.find.b2;
    u64* const stage = reinterpret_cast<u64*>(s.own_low);
    each<E>(in, v0, nv, [&](const float (&x)[4], int token) {
        uint32_t is = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (KEYS) {
                const uint32_t key = key_of(x[e]);
                if (key >= lo && key <= hi) is |= 1u << e;
            } else {
                const float at = r.slice(x[e]);
                if ((at >= f0 && at <= f1) || at == f2) is |= 1u << e;
            }
        }
        if (is) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (is >> e & 1u) {
                    const uint32_t at = atomicAdd(&s.staged, 1u);
                    if (at < (uint32_t)kMembers) stage[at] = (u64)key_of(x[e]) << 32 | (uint32_t)~(token + e);
                }
        }
    });
}

// The largest and the smallest but -infinity, of this thread's values.
template <typename E>
__device__ __noinline__ float2 ends_pass(const E* in, int nv) {
    constexpr int PER = 4 / (int)sizeof(E), V = 4 * PER, U = 4;  // (from HBM: more on their way)
    const int tid = (int)threadIdx.x, vecs = ((uintptr_t)in & 15) == 0 ? nv / V : 0;
    float most = -INFINITY, least = INFINITY;
    const auto see = [&](float x) {
        most = fmaxf(most, x);
        least = fminf(least, x > -INFINITY ? x : INFINITY);
    };
#pragma unroll 1
    for (int i = tid; i < vecs; i += U * kSampleThreads) {
        uint4 raw[U];
#pragma unroll
        for (int j = 0; j < U; ++j) raw[j] = reinterpret_cast<const uint4*>(in)[min(i + j * kSampleThreads, vecs - 1)];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
            for (int e = 0; e < V; ++e) see(value_in<E>(w[e / PER], e % PER));
        }
    }
#pragma unroll 1
    for (int i = vecs * V + tid; i < nv; i += kSampleThreads) see(to_f(in[i]));
    return make_float2(most, least);
}

// The nth token with key find.lo, or (crowd) the one drawn among all with it: a warp's in their order, then the warps', then the CTAs'.
template <typename E>
__device__ __noinline__ void nth_token(const SampleArgs& a, int row, const E* in, int v0, int nv, bool crowd) {
    Shared& s = shared();
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t key = s.find.lo;
    const int part = (nv + kSampleThreads - 1) / kSampleThreads * 32;  // a warp's tokens
    const int i0 = min(nv, warp * part), i1 = min(nv, i0 + part);
    uint32_t have = 0;
#pragma unroll 4
    for (int i = i0 + lane; i - lane < i1; i += 32) {
        const float y = i < i1 ? to_f(in[i]) : -INFINITY;
        have += __popc(__ballot_sync(0xffffffffu, y > -INFINITY && key_of(y) == key));
    }
    if (lane == 0) s.warp_count[warp] = have;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int i = 0; i < kSampleWarps; ++i) {
        before += i < warp ? s.warp_count[i] : 0;
        all += s.warp_count[i];
    }
    if (tid < C) cluster.map_shared_rank(&s, tid)->ties[rank] = all;
    cluster.sync();
    all = 0;
    for (int i = 0; i < C; ++i) {
        before += i < rank ? s.ties[i] : 0;
        all += s.ties[i];
    }
    uint32_t nth = s.find.nth;
    float logprob = s.find.logprob;
    if (crowd) {
        u64 kept = s.k > 0 ? min((u64)s.k, (u64)all) : all;
        if (s.p < 1.f) kept = nucleus(s.p, kept);
        if (s.min_p > 1.f) kept = 1;
        nth = (uint32_t)drawn(s.u, kept);
        logprob = (float)-log_of((double)kept);
    }
    if (before < nth && nth <= before + have)
        for (int i = i0 + lane; i - lane < i1; i += 32) {
            const float y = i < i1 ? to_f(in[i]) : -INFINITY;
            const bool is = y > -INFINITY && key_of(y) == key;
            const uint32_t who = __ballot_sync(0xffffffffu, is);
            if (is && before + __popc(who & ((2u << lane) - 1u)) == nth) {
                a.token[row] = v0 + i;
                if (a.logprob) a.logprob[row] = logprob;
            }
            before += __popc(who);
        }
}

// The CTAs' histograms into the row's, each CTA a part of it for all; and cleared.
__device__ __noinline__ void collect(bool first, bool sums, bool numbers) {
    Shared& s = shared();
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    uint32_t* const counts = first ? s.first_count : s.more_count;
    u64* const masses = first ? s.first_mass : s.more_mass;
    cluster.sync();
#pragma unroll 1
    for (int b = rank * (kBins / C) + (int)threadIdx.x; b < (rank + 1) * (kBins / C); b += kSampleThreads) {
        uint32_t c = 0;
        u64 m = 0;
#pragma unroll 4
        for (int i = 0; i < C; ++i) {
            const Shared* o = cluster.map_shared_rank(&s, i);
            if (numbers) c += o->own_count[b];
            if (sums) m += (u64)o->own_low[b] + ((u64)o->own_high[b] << 32);
        }
#pragma unroll 4
        for (int i = 0; i < C; ++i) {
            if (numbers) *cluster.map_shared_rank(counts + b, i) = c;
            if (sums) *cluster.map_shared_rank(masses + b, i) = m;
        }
    }
    cluster.sync();
    clear(s);
}

// The slice of a histogram that holds the answer, and what to do with it. Every CTA works this out for itself.
__device__ __noinline__ void look(bool first, bool sums, int C) {
    Shared& s = shared();
    Search& f = s.find;
    const int tid = (int)threadIdx.x, k = s.k;
    Slices t;
    {
        const uint32_t* counts = first ? s.first_count : s.more_count;
        const u64* masses = first ? s.first_mass : s.more_mass;
        const bool numbers = !first || k > 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t.mass4[i] = sums ? masses[4 * tid + i] : 0;
            t.count4[i] = numbers ? counts[4 * tid + i] : 0;
        }
        t.scan(s, first ? 0 : f.mass_before, first ? 0 : f.count_before);
        if (s.fresh && tid == kSampleThreads - 1) {
            u64 likely = 0;
            f.total = t.mass + t.mass4[0] + t.mass4[1] + t.mass4[2] + t.mass4[3];
            for (int i = 0; sums && i < C; ++i) likely += s.likely[i];
            // (the first of the order is kept whatever min_p is)
            f.likely = s.row.least > 0.0 ? max(likely, (u64)s.row.lift) : f.total;
            f.goal = kTopK;
            f.last = 0;
            const u64 all = t.count + t.count4[0] + t.count4[1] + t.count4[2] + t.count4[3];  // (the last slice's never drawn too)
            if (k > 1 && (s.few || (u64)k < all))
                f.limit = min((u64)k, all);
            else
                next_goal(f.total);
        }
        __syncthreads();
    }
    const int goal = f.goal;
    const bool by_key = f.last < 0;
    t.pick(s, goal == kTopK, 0, f.limit);
    __syncthreads();
    const int b = s.at[0];
    if (first && goal == kTopP && !by_key) {
        // and the slices that can hold the token, as the kept ones end somewhere in slice b
        const u64 front = s.at_mass[0], own = s.at_own[0], likely = f.likely;
        const float u = s.u;
        __syncthreads();
#pragma unroll 1
        for (int j = 0; j < 2; ++j) t.pick(s, false, j, drawn(u, min(j ? front + own : front + 1, likely)));
        __syncthreads();
        if (tid == 0) {
            f.op = kGather;
            f.b0 = s.at[0];
            f.b1 = s.at[1];
            f.b2 = b;
            f.goal = kBoth;
            f.mass_before = s.at_mass[0];
            f.more_before = front;
            // no slice has more members than its sum has least weights of its (and half a unit each)
            const auto most = [&](u64 sum, int slice) { return (double)sum / fmax(s.table[slice] * 0.98 - 1.0, 1e-9); };
            const u64 middle = f.b1 < b ? s.at_mass[1] + s.at_own[1] - s.at_mass[0] : front - s.at_mass[0];
            f.last = most(middle, min(f.b1, b)) + most(own, b) <= (double)kMembers;
        }
    } else if (tid == 0) {
        const uint32_t before = s.at_count[0], members = s.at_members[0];
        uint32_t lo = 0, hi = 0;
        bool into = false;
        if (!first) {
            hi = f.hi - ((uint32_t)b << f.shift);
            const uint32_t span = (1u << f.shift) - 1;
            lo = hi - f.lo > span ? hi - span : f.lo;
            into = true;
        } else if (goal == kTopK && s.few && (b == kLast ? before : before + members) <= (uint32_t)kMembers) {
            // the kept ones and no more than kMembers in all (those of the last slice have no weight)
            f.goal = kPrefix;
            f.limit = b == kLast ? min(f.limit, (u64)before) : f.limit;
            f.op = kGather;
            f.b0 = 0;
            f.b1 = f.b2 = b == kLast ? b - 1 : b;
            f.last = 1;
        } else if (!sums) {
            f.op = kSums;
        } else if (goal == kTopK && b == kLast) {
            next_goal(f.total);
        } else if (goal == kDraw && !by_key) {
            f.mass_before = s.at_mass[0];
            f.op = kGather;
            f.b0 = f.b1 = f.b2 = b;
            f.last = (double)s.at_own[0] <= (double)kMembers * (s.table[b] * 0.98 - 1.0);
        } else {
            lo = lowest_key(b);
            hi = b ? lowest_key(b - 1) - 1 : key_of(s.row.m);
            into = true;
        }
        if (into) {
            f.mass_before = s.at_mass[0];
            f.count_before = s.at_count[0];
            f.lo = lo;
            f.hi = hi;
            f.last = 0;
            if ((!first || k > 1) && members <= (uint32_t)kMembers) {
                f.op = kGatherKeys;
            } else if (lo < hi) {
                f.op = kDivide;
                f.shift = shift_of(hi - lo);
            } else {
                // equal keys
                const Row r = s.row;
                const float x = value_of(lo);
                const u64 w = Row::whole(r.weight(x, r.bin(x), s.table));
                const u64 nth = goal == kTopK ? f.limit - f.count_before : (f.limit - f.mass_before + w - 1) / max(w, 1ull);
                if (goal == kDraw) {
                    f.op = kTies;
                    f.nth = (uint32_t)nth;
                    f.logprob = logprob_of(r, x, f.kept);
                } else {
                    next_goal(f.mass_before + nth * w);
                }
            }
        }
    }
    s.fresh = 0;
    __syncthreads();
}

// By the first CTA: of the members of slices [lo, hi], before which the row's sum and number are `before` and `number`, the first
// whose running sum, or number, reaches `limit`, into at_one; returns its running sum.
__device__ __noinline__ u64 reach(int lo, int hi, u64 before, uint32_t number, bool by_count, u64 limit) {
    Shared& s = shared();
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31, n = (int)s.members;
    const Row r = s.row;
    const u64* const weight = s.more_mass;
    uint32_t klo = 0, khi = ~0u;
    // f(index, key) for this thread's members of the set; returns the set's size
    const auto members = [&](auto f) {
        int size = 0;
#pragma unroll 1
        for (int base = 0; base < n; base += kSampleThreads) {
            const int i = base + tid;
            const uint32_t key = i < n ? (uint32_t)(s.member[i] >> 32) : 0u;
            bool is = i < n && key >= klo && key <= khi;
            if (is) {
                const int b = r.bin(value_of(key));
                is = b >= lo && b <= hi;
            }
            if (is) f(i, key);
            size += __syncthreads_count(is);
        }
        return size;
    };
    uint32_t least = ~0u, most = 0;
    int size = members([&](int, uint32_t key) {
        least = min(least, key);
        most = max(most, key);
    });
#pragma unroll 1
    while (size > kFew) {
        // the set's keys from lowest to highest, divided
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) s.warp_lo[warp] = least, s.warp_hi[warp] = most;
        __syncthreads();
        klo = __reduce_min_sync(0xffffffffu, s.warp_lo[lane % kSampleWarps]);
        khi = __reduce_max_sync(0xffffffffu, s.warp_hi[lane % kSampleWarps]);
        if (klo == khi) break;
        const int shift = shift_of(khi - klo);
        members([&](int i, uint32_t key) {
            const int to = (int)((khi - key) >> shift);
            const u64 w = weight[i];
            atomicAdd(&s.own_count[to], 1u);
            const uint32_t was = atomicAdd(&s.own_low[to], (uint32_t)w);
            atomicAdd(&s.own_high[to], (uint32_t)(w >> 32) + (was + (uint32_t)w < was));
        });
        Slices t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t.mass4[i] = (u64)s.own_low[4 * tid + i] + ((u64)s.own_high[4 * tid + i] << 32);
            t.count4[i] = s.own_count[4 * tid + i];
        }
        t.scan(s, before, number);
        t.pick(s, by_count, 0, limit);
        __syncthreads();
        before = s.at_mass[0];
        number = s.at_count[0];
        const uint32_t top = khi - ((uint32_t)s.at[0] << shift), span = (1u << shift) - 1;
        klo = top - klo > span ? top - span : klo;
        khi = top;
        clear(s);
        least = ~0u, most = 0;
        size = members([&](int, uint32_t key) {
            least = min(least, key);
            most = max(most, key);
        });
    }
    if (tid == 0) s.staged = 0;
    __syncthreads();
    if (size <= kFew) {
        members([&](int i, uint32_t) {
            const uint32_t at = atomicAdd(&s.staged, 1u);
            s.set_member[at] = s.member[i];
            s.set_weight[at] = weight[i];
        });
        __syncthreads();
        // four threads a member: how many are before it, and their sum
        const int e = min(tid / 4, size - 1);
        const u64 mine = s.set_member[e], own = s.set_weight[e];
        u64 sum = 0;
        int place = 0;
#pragma unroll 2
        for (int i = tid % 4; i < size; i += 4)
            if (s.set_member[i] > mine) {
                ++place;
                sum += s.set_weight[i];
            }
        place += __shfl_xor_sync(0xffffffffu, place, 1);
        place += __shfl_xor_sync(0xffffffffu, place, 2);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum += before;
        if (by_count ? (u64)number + place + 1 == limit : sum < limit && limit <= sum + own) {
            s.at_one = mine;
            s.at_mass[0] = sum + own;
        }
    } else {
        // equal keys, equal weights: the nth of them by their numbers, found bit by bit
        members([&](int i, uint32_t) { s.at_own[0] = weight[i]; });
        const u64 w = s.at_own[0];
        const int nth = (int)(by_count ? limit - number : (limit - before + w - 1) / max(w, 1ull));
        uint32_t token = 0;
#pragma unroll 1
        for (int bit = 21; bit >= 0; --bit) {
            int below = 0;
#pragma unroll 1
            for (int base = 0; base < n; base += kSampleThreads) {
                const int i = base + tid;
                below += __syncthreads_count(i < n && (uint32_t)(s.member[i] >> 32) == klo && (uint32_t)~(uint32_t)s.member[i] < token + (1u << bit));
            }
            if (below < nth) token += 1u << bit;
        }
        if (tid == 0) {
            s.at_one = (u64)klo << 32 | (uint32_t)~token;
            s.at_mass[0] = before + (u64)nth * w;
        }
    }
    __syncthreads();
    const u64 sum = s.at_mass[0];
    __syncthreads();
    return sum;
}

// By the first CTA: what the members say.
__device__ __noinline__ void settle(const SampleArgs& a, int row) {
    Shared& s = shared();
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31, n = (int)s.members;
    const int goal = s.find.goal;
    u64 likely = 0;
    {
        const Row r = s.row;
        const bool table = s.table_made;
#pragma unroll 1
        for (int i = tid; i < n; i += kSampleThreads) {
            const float x = value_of((uint32_t)(s.member[i] >> 32));
            const double y = table ? r.weight(x, r.bin(x), s.table) : exp_of(((double)x - (double)r.m) * r.per_t) * r.lift;
            const u64 w = Row::whole(y);
            s.more_mass[i] = w;
            if (y >= r.least) likely += w;
        }
    }
    if (goal == kPrefix) {
        likely = warp_sum(likely);
        if (lane == 0) s.warp_mass[warp] = likely;
        __syncthreads();
        likely = 0;
        for (int i = 0; i < kSampleWarps; ++i) likely += s.warp_mass[i];
        likely = max(likely, (u64)s.row.lift);  // (the first of the order is kept whatever min_p is)
    }
    __syncthreads();
    const float p = s.p, u = s.u;
    u64 kept = s.find.kept, answer = 0;
    const int questions = goal == kPrefix ? 3 : goal == kBoth ? 2 : 1;
#pragma unroll 1
    for (int q = 0; q < questions; ++q) {
        int lo = 0, hi = kLast;
        u64 before = s.find.mass_before, limit = s.find.limit;
        uint32_t number = 0;
        bool by_count = false;
        if (goal == kPrefix) {
            before = 0;
            by_count = q == 0;
            if (q == 1) {
                if (!(p < 1.f)) continue;
                limit = nucleus(p, kept);
            }
            if (q == 2) {
                kept = min(kept, likely);
                limit = drawn(u, kept);
            }
        } else if (goal == kBoth) {
            if (q == 0) {
                lo = hi = s.find.b2;
                before = s.find.more_before;
            } else {
                hi = s.find.b1;
                kept = min(kept, s.find.likely);
                limit = drawn(u, kept);
            }
        } else if (goal == kTopK) {
            by_count = true;
            number = s.find.count_before;
        }
        answer = reach(lo, hi, before, number, by_count, limit);
        if (q + 1 < questions) kept = answer;
    }
    if (tid != 0) return;
    if (goal == kTopK || goal == kTopP) {
        next_goal(answer);
    } else {
        a.token[row] = (int)~(uint32_t)s.at_one;
        if (a.logprob) a.logprob[row] = logprob_of(s.row, value_of((uint32_t)(s.at_one >> 32)), kept);
        s.find.op = kDone;
    }
}

template <typename E>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
    Shared& s = shared();
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = (int)blockIdx.x / C;
    const int v0 = min(a.vocab, rank * a.slice), nv = min(a.vocab - v0, a.slice);
    const E* in = static_cast<const E*>(a.in) + (int64_t)row * a.ld + v0;
    Shared* const head = cluster.map_shared_rank(&s, 0);
    clear(s);
    stream_turn();
    const float T0 = a.temperature ? a.temperature[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
    const int k = a.top_k ? a.top_k[row] : 0;
    if (tid == 0) {
        s.members = 0;
        s.k = k;
        s.few = k > 1 && k <= kMembers;  // the first histogram needs no sums
        s.p = a.top_p ? a.top_p[row] : 1.f;
        s.u = a.u[row];
        s.min_p = min_p;
        s.table_made = 0;
        s.fresh = 1;
    }
    // ---- the largest and the smallest
    {
        float2 e = ends_pass<E>(in, nv);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            e.x = fmaxf(e.x, __shfl_xor_sync(0xffffffffu, e.x, o));
            e.y = fminf(e.y, __shfl_xor_sync(0xffffffffu, e.y, o));
        }
        if (lane == 0) s.warp_ends[warp] = e;
        __syncthreads();
        if (warp == 0) {
            e = s.warp_ends[lane % kSampleWarps];
#pragma unroll
            for (int o = 1; o < kSampleWarps; o <<= 1) {
                e.x = fmaxf(e.x, __shfl_xor_sync(0xffffffffu, e.x, o));
                e.y = fminf(e.y, __shfl_xor_sync(0xffffffffu, e.y, o));
            }
            if (lane < C) cluster.map_shared_rank(&s, lane)->ends[rank] = e;
        }
        cluster.sync();
    }
    int op;
    {
        Row r;
        float least = INFINITY;
        r.m = -INFINITY;
        for (int i = 0; i < C; ++i) {
            r.m = fmaxf(r.m, s.ends[i].x);
            least = fminf(least, s.ends[i].y);
        }
        if (r.m == -INFINITY) {
            if (rank == 0 && tid == 0) {
                a.token[row] = -1;
                if (a.logprob) a.logprob[row] = -INFINITY;
            }
            return;
        }
        // the first of the order; or, beside +infinity, only what is: tokens of equal weights
        op = !(T0 > 0.f) || k == 1 ? kTies : r.m == INFINITY ? kCrowd : k > 1 && k <= kMembers ? kNumbers : kSums;
        if (tid == 0) {
            const float T = fmaxf(T0, 7.8886091e-31f);  // 2^-100: what follows stays within f32's range
            r.half_m = 0.5f * r.m;
            r.per_t = 1.0 / (double)T;
            r.lift = __longlong_as_double((long long)(1023 + a.bits) << 52);
            r.least = min_p > 0.f ? (double)min_p * r.lift : 0.0;
            // half of the range that the first histogram divides: all values, or those with a weight
            const float range = fminf(fmaf(least, -0.5f, r.half_m), 18.f * T);
            r.scale = range > 0.f ? fminf((float)(kLast - 1) / range, 1e35f) : 0.f;
            r.grid = r.scale > 0.f ? 2.0 / (double)r.scale * r.per_t : 0.0;
            s.row = r;
            s.find.lo = key_of(r.m);
            s.find.nth = 1;
            s.find.logprob = 0.f;
        }
        __syncthreads();
    }
#pragma unroll 1
    for (;;) {
        if (op == kTies || op == kCrowd) {
            nth_token<E>(a, row, in, v0, nv, op == kCrowd);
            return;
        }
        if (op == kGather || op == kGatherKeys) {
            // the members into this CTA's memory, then behind one another into the first CTA's
            const bool last = s.find.last > 0;
            if (tid == 0) s.staged = 0;
            __syncthreads();
            if (op == kGather)
                gather_pass<E, false>(in, v0, nv);
            else
                gather_pass<E, true>(in, v0, nv);
            __syncthreads();
            const uint32_t staged = s.staged;
            if (tid == 0) s.base = atomicAdd(&head->members, staged);
            __syncthreads();
            const uint32_t base = s.base;
            const u64* const stage = reinterpret_cast<const u64*>(s.own_low);
#pragma unroll 1
            for (uint32_t i = tid; i < staged && base + i < (uint32_t)kMembers; i += kSampleThreads) head->member[base + i] = stage[i];
            __syncthreads();
            clear(s);
            cluster.sync();
            if (last && rank != 0) return;
            if (rank == 0) {
                if (s.members > (uint32_t)kMembers) {
                    // (a slice whose tokens were not counted has more than that: by its keys)
                    if (tid == 0) {
                        if (s.find.goal == kBoth) s.find.goal = kTopP;
                        s.find.op = kLook;
                        s.find.last = -1;
                    }
                } else {
                    settle(a, row);
                    if (last) return;
                }
                __syncthreads();
                if (tid == 0) s.members = 0;
            }
            // what it found, to all
            cluster.sync();
            if (rank != 0 && tid == 0) s.find = head->find;
            cluster.sync();
            op = s.find.op;
            if (op == kDone) return;
        }
        if (op == kDivide) {
            divide_pass<E>(in, nv);
        } else if (op == kNumbers) {
            numbers_pass<E>(in, nv);
        } else if (op == kSums) {
            if (tid < kBins / 32 + 32) {
                const int i = tid < kBins / 32 ? 32 * tid : tid - kBins / 32;
                const double e = exp_of(-i * s.row.grid);
                if (tid < kBins / 32)
                    s.coarse[tid] = e * s.row.lift;
                else
                    s.fine[tid - kBins / 32] = e;
            }
            __syncthreads();
            for (int i = tid; i < kBins; i += kSampleThreads) s.table[i] = s.coarse[i / 32] * s.fine[i % 32];
            if (tid == 0) s.table_made = s.fresh = 1;
            __syncthreads();
            if (k > 1 || s.row.least > 0.0) {
                const u64 likely = warp_sum(sums_pass<E, true>(in, nv));
                if (lane == 0) s.warp_mass[warp] = likely;
                __syncthreads();
                if (tid < C) {
                    u64 sum = 0;
                    for (int i = 0; i < kSampleWarps; ++i) sum += s.warp_mass[i];
                    cluster.map_shared_rank(&s, tid)->likely[rank] = sum;
                }
            } else {
                sums_pass<E, false>(in, nv);
            }
        }
        if (op != kLook) collect(op != kDivide, op != kNumbers, op != kSums || k > 1);
        look(op != kDivide, op != kNumbers, C);
        op = s.find.op;
    }
}

template <typename E>
cudaError_t launch_sample(SampleArgs a, int rows, int device, int n_sm, cudaStream_t s) {
    static thread_local int prepared = -1;  // the device whose attribute this thread has set
    if (prepared != device) {
        const cudaError_t e = cudaFuncSetAttribute(sample_kernel<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared));
        if (e != cudaSuccess) return e;
        prepared = device;
    }
    // As many CTAs a row as fill the SMs twice, each with a few thousand tokens or more.
    int C = 1;
    while (C < kSampleCluster && (int64_t)rows * C <= n_sm && a.vocab > 4096 * C) C *= 2;
    a.slice = ((a.vocab + C - 1) / C + 7) & ~7;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)C;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(rows * C));
    c.blockDim = dim3(kSampleThreads);
    c.dynamicSmemBytes = sizeof(Shared);
    c.stream = s;
    c.attrs = at;
    c.numAttrs = 2;
    return cudaLaunchKernelEx(&c, sample_kernel<E>, a);
}

bool refuse(const char* what) {
    set_free_error(what);
    return false;
}

bool sample(const void* logits, int64_t ld, int dtype, int rows, int vocab, const float* u, const float* temperature,
            const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens, float* logprob, void* stream) {
    if (dtype != AERO_CUDA_TYPE_F32 && dtype != AERO_CUDA_TYPE_F16 && dtype != AERO_CUDA_TYPE_BF16)
        return refuse("logits are F32, F16 or BF16");
    if (rows < 0 || rows > (1 << 20) || vocab <= 0 || vocab > kMostVocab)
        return refuse("rows must be from 0 to 2^20 and vocab from 1 to 2^22");
    if (rows == 0) return true;
    if (ld < 0) return refuse("ld must be >= 0");
    const uintptr_t size = dtype == AERO_CUDA_TYPE_F32 ? 4 : 2;
    cudaPointerAttributes where{};
    if (!logits || cudaPointerGetAttributes(&where, logits) != cudaSuccess) {
        cudaGetLastError();
        where.type = cudaMemoryTypeUnregistered;
    }
    if (where.type != cudaMemoryTypeDevice && where.type != cudaMemoryTypeManaged) return refuse("logits must be device memory");
    if ((uintptr_t)logits % size) return refuse("logits must be aligned to their type");
    if (!u || !tokens) return refuse("u and tokens are required");
    const void* arrays[] = {u, temperature, top_k, top_p, min_p, tokens, logprob};
    for (const void* p : arrays)
        if (p && (!is_device_ptr(p) || ((uintptr_t)p & 3))) return refuse("u, the limits and the results must be device memory, aligned to 4 bytes");
    OnDevice on(where.device);
    if (!on.good) return refuse("cudaSetDevice failed");
    int n_sm = 148, bits = 48;
    cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, where.device);
    while (bits > 0 && ((int64_t)vocab << bits) > (1ll << 62)) --bits;
    const SampleArgs a{logits, ld, vocab, 0, bits, u, temperature, top_p, min_p, top_k, tokens, logprob};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == AERO_CUDA_TYPE_F32   ? launch_sample<float>(a, rows, where.device, n_sm, s)
                          : dtype == AERO_CUDA_TYPE_F16 ? launch_sample<__half>(a, rows, where.device, n_sm, s)
                                                        : launch_sample<__nv_bfloat16>(a, rows, where.device, n_sm, s);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_free_error(std::string("logits_sample: ") + cudaGetErrorString(e));
        return false;
    }
    return true;
}

}  // namespace
}  // namespace aero

extern "C" int aero_cuda_logits_sample(const void* logits, int64_t ld, int dtype, int rows, int vocab, const float* u,
                                       const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                       int32_t* tokens, float* logprob, void* stream) {
    try {
        return aero::sample(logits, ld, dtype, rows, vocab, u, temperature, top_k, top_p, min_p, tokens, logprob, stream) ? 0 : -1;
    } catch (...) {
        return -1;
    }
}
