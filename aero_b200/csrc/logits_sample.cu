// A token drawn from each row of a batch's logits (include/aero_cuda_pages.h, aero_cuda_logits_sample).
//
// In falling order of the logits, equal ones by their number, with weights w_j = 2^(-(m - x_j) log2(e) / T): every
// limit (top_k, top_p, min_p) keeps a prefix of that order, so what is kept is said by one number, its sum S, and the
// token is the first whose running sum exceeds u S. Nothing is sorted as a whole and nothing is written but the token:
// each question is "which is the first in the order whose running sum (or number) reaches a limit?", answered by a
// histogram of the row (counts or sums over kBins slices of its values), then by the members of the slices that can hold
// the answer, gathered and put in order by themselves. A slice with more than kMembers is divided again by
// its keys; one of equal keys is answered by arithmetic and its members' order.
//
// Weights are whole numbers, multiples of 2^-B of the largest (B = 44 for a vocabulary of 2^18): their sums
// are exact in any order, so histograms may be made by atomics and the answer does not depend on timing. Each weight is
// computed in 64 bits and off by half of 2^-B and by 2^-50 of the largest at most (y halvings below it by 2^-51 of itself for the
// series, the table and the arithmetic, and by y 2^-52 for 1 / T's rounding), so a sum of V of them by V / 2 2^-B of the
// largest and by 2^-47 of itself (in all 2^-27 of the largest for V = 2^18, if all weigh as much).
//
// A cluster of CTAs per row, each with an even share of the row, which it reads from HBM once, for the largest, and twice more
// from L2, for the sums and for the members; the first CTA's shared memory holds the members. What crosses the cluster is 64
// sums a CTA and 64 slices an answer: reads of another CTA's memory take some 13 cycles a warp's load (all
// slices to all: 4000 to 14000 cycles).
//
// Bound, for many rows, by the weights' 64-bit arithmetic (64 rows of 151936, top-p: 51 us, of which 13 are the sums with 8
// 64-bit operations in 32 instructions a token, 11 the other two passes from L2, some 11 the search, step after step);
// for one row of 32000 by ten steps of some 2000 cycles one after another (11.5 us). Clusters of 16 gain 4 %
// for one row of 151936 and lose 10 % for 16 mixed ones.
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
constexpr int kBins = 8 * kSampleThreads, kLast = kBins - 1, kGroups = 64;
constexpr int kParts = 4 * kSampleThreads;  // of a slice's keys
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

// Keys of numbers in their order, -0 as 0. (What is no number may have any key: the sign of an operation's result is not
// said.)
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

// What all threads know of a row. Its values are divided into kBins slices below m, 64 to each halving of the weights; the last
// one holds what lies 63.99 halvings and more below m, whose weights are 0 as multiples of 2^-48 or more, and what is
// never drawn (-infinity and no numbers).
struct Row {
    float m;             // the largest logit
    float half_m, scale; // slice = (m / 2 - x / 2) * scale (halves: the difference of any two numbers is one)
    float step;          // a slice's width; infinity: m is too large for sums and differences of slices' ends
    float floor;         // a value of the last slice, next to its middle; -infinity: there is none
    double per_t;        // 32 log2(e) / T
    double lift;         // 2^B
    u64 least;           // min_p 2^B
    __device__ __forceinline__ float open_place(float x) const { return fmaf(x, -0.5f, half_m) * scale; }
    __device__ __forceinline__ float place(float x) const { return fminf(open_place(x), (float)kLast); }
    // (as a number beside 2^23, for comparisons)
    __device__ __forceinline__ float slice(float x) const { return place(x) + 8388608.f; }
    __device__ __forceinline__ int bin(float x) const { return (int)(__float_as_uint(slice(x)) & (kBins - 1)); }
    // 2^52 + 2^B e^((x - m) / T), which leaves the weight's nearest whole number in the low bits (2^B is at most 2^48), for
    // slices but the last. at = place(x). In 32nds of a halving x lies z = 32 log2(e) (x - m) / T above m; with i the whole number
    // next to -z and r = z + i, at most a half either way, the weight is 2^-(i / 32) 2^(r / 32): a table's value (2^B's 32 parts,
    // the halvings taken off its exponent) times the series of 2^(r / 32) to r^5, whose term in r^6 is made up for by Chebyshev's
    // polynomial; what is left out is below 2^-52 (with 16 parts 2^-46.6, 2.5 of 2^-48).
    __device__ __forceinline__ double beside(float x, float at, const double* table) const {
        constexpr double L = 0.6931471805599453 / 32, h2 = 0.25, a5 = L * L * L * L * L * L / 720;
        const float i = fmaf(at, 0.5f, 8388608.f);
        const double z = fma((double)x - (double)m, per_t, (double)(i - 8388608.f));
        double p = fma(z, L * L * L * L * L / 120, L * L * L * L / 24 + 1.25 * h2 * a5);
        p = fma(p, z, L * L * L / 6);
        p = fma(p, z, L * L / 2 - 0.3125 * h2 * h2 * a5);
        p = fma(p, z, L);
        p = fma(p, z, 1.0);
        const uint32_t n = __float_as_uint(i);
        const double t = table[n & 31u];
        return fma(p, __hiloint2double(__double2hiint(t) - (int)((n & ~31u) * 32768u), __double2loint(t)), kTwo52);
    }
    static __device__ __forceinline__ u64 whole(double beside) { return (u64)__double_as_longlong(beside) & 0xFFFFFFFFFFFFFull; }
    __device__ __forceinline__ u64 weight(float x, const double* table) const { return whole(beside(x, place(x), table)); }
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
    int by_count;        // kBoth: the first is what top_k keeps
    int k_slice;         // the slice that holds the k-th, or -1: top_k keeps all
    uint32_t k_before, k_members;  // tokens before it and in it
    uint32_t nth;        // kTies: which of the tokens with key lo, from 1
    float logprob;       // kTies
    uint32_t count_before;         // tokens before the slice in hand
    u64 limit;                     // the running sum, or number (kTopK, kPrefix), to be reached
    u64 mass_before, more_before;  // sums before the slice in hand; kBoth: and before slice b2
    u64 kept, likely;              // sums: of the kept, of those that min_p keeps
};

// A CTA's histogram of its tokens: sums as two words (or numbers, as the low one), numbers.
struct Slices {
    uint32_t low[kBins], high[kBins];
};
struct Parts {
    uint32_t low[kParts], high[kParts], count[kParts];
};
// Sums over a 64th of a histogram each.
struct Groups {
    u64 mass[kGroups];
    uint32_t count[kGroups];
};

struct Shared {
    double table[32];
    Slices first;             // of Row's slices
    Parts more;               // of one slice's keys, or of members' keys; the place of members on their way; else zero
    u64 member[kMembers];     // key, then all ones less the token's number (in the first CTA)
    u64 weight[kMembers];     // (in the first CTA)
    Groups from[kSampleCluster];         // what the CTAs' histograms hold
    Groups first_groups, more_groups;    // the row's
    u64 set_member[kFew], set_weight[kFew];
    int set_slice[kFew];
    u64 warp_mass[kSampleWarps];
    uint32_t warp_count[kSampleWarps], warp_lo[kSampleWarps], warp_hi[kSampleWarps];
    float ends[kSampleCluster], warp_ends[kSampleWarps];  // the largest of the CTAs, of the warps
    u64 likely[kSampleCluster];
    uint32_t ties[kSampleCluster];
    uint32_t members, staged, base;
    Row row;
    Search find;
    float u, p, min_p;
    int k, few, fresh;
    int at[3];
    u64 at_mass[3], at_own[3], at_one;
    uint32_t at_count[3], at_members[3];
};
static_assert(sizeof(Shared) <= 113 * 1024, "two CTAs an SM");

// Each part below is a function of its own, with the registers it needs: what runs once is bound by fetching its
// instructions, what runs over the row by its own loop.
__device__ __forceinline__ Shared& shared() {
    extern __shared__ __align__(16) uint8_t smem[];
    return *reinterpret_cast<Shared*>(smem);
}
__device__ __noinline__ double log_of(double x) { return log(x); }
__device__ __forceinline__ float logprob_of(const Row& r, float x, u64 kept) {
    return (float)(((double)x - (double)r.m) * r.per_t * (0.6931471805599453 / 32) - log_of((double)kept / r.lift));
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename H>
__device__ __forceinline__ void clear(H& h) {
#pragma unroll 1
    for (int i = (int)threadIdx.x; i < (int)sizeof(H) / 16; i += kSampleThreads) reinterpret_cast<uint4*>(&h)[i] = make_uint4(0u, 0u, 0u, 0u);
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

// (hi - lo) >> shift < kParts = 2^11
__device__ __forceinline__ int shift_of(uint32_t span) { return max(0, 21 - __clz((int)span)); }

// A histogram's groups; every thread calls it: eight threads a group.
__device__ __forceinline__ void group(const Slices& h, Groups& g) {
    const int t = (int)threadIdx.x;
    u64 m = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 low = reinterpret_cast<const uint4*>(h.low)[2 * t + i], high = reinterpret_cast<const uint4*>(h.high)[2 * t + i];
        m += (u64)low.x + low.y + low.z + low.w + (((u64)high.x + high.y + high.z + high.w) << 32);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    if (t % 8 == 0) g.mass[t / 8] = m;
}
__device__ __forceinline__ void group(const Parts& h, Groups& g) {
    const int t = (int)threadIdx.x;
    const uint4 low = reinterpret_cast<const uint4*>(h.low)[t], high = reinterpret_cast<const uint4*>(h.high)[t];
    const uint4 count = reinterpret_cast<const uint4*>(h.count)[t];
    u64 m = (u64)low.x + low.y + low.z + low.w + (((u64)high.x + high.y + high.z + high.w) << 32);
    uint32_t c = count.x + count.y + count.z + count.w;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        m += __shfl_xor_sync(0xffffffffu, m, o);
        c += __shfl_xor_sync(0xffffffffu, c, o);
    }
    if (t % 8 == 0) g.mass[t / 8] = m, g.count[t / 8] = c;
}
static_assert(kSampleThreads == 8 * kGroups, "eight threads a group");

template <typename V>
__device__ __forceinline__ V scanned(V v) {
    const int lane = (int)threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

// By a warp: the slice of the first histogram (C CTAs' together) that holds the answer to a limit into at[j], with what lies
// before it and what it holds; or, of slice b, the last two. Reads of other CTAs' memory are slow: groups first, then 64 slices.
__device__ __noinline__ void find(int j, int C, u64 limit, int b) {
    Shared& s = shared();
    const cg::cluster_group cluster = cg::this_cluster();
    const int lane = (int)threadIdx.x & 31;
    const u64 g0 = s.first_groups.mass[2 * lane], g1 = s.first_groups.mass[2 * lane + 1];
    const u64 g = scanned(g0 + g1);
    // which group: 2 lane or 2 lane + 1 of the lane that the limit lies in
    int group;
    if (b < 0) {
        const int in = min(__popc(__ballot_sync(0xffffffffu, g < limit)), 31);
        group = 2 * in + (__shfl_sync(0xffffffffu, g - g1, in) < limit);
    } else {
        group = b / 64;
    }
    const u64 to_odd = __shfl_sync(0xffffffffu, g - g1, group / 2), to_even = __shfl_sync(0xffffffffu, g - g1 - g0, group / 2);
    const u64 before = group & 1 ? to_odd : to_even;
    u64 m0 = 0, m1 = 0;
    const int at = 64 * group + 2 * lane;
#pragma unroll 4
    for (int i = 0; i < C; ++i) {
        const Slices* o = C > 1 ? cluster.map_shared_rank(&s.first, i) : &s.first;
        const uint2 low = *reinterpret_cast<const uint2*>(o->low + at), high = *reinterpret_cast<const uint2*>(o->high + at);
        m0 += (u64)low.x + ((u64)high.x << 32);
        m1 += (u64)low.y + ((u64)high.y << 32);
    }
    const u64 m = before + scanned(m0 + m1);
    bool odd;
    int in;
    if (b < 0) {
        in = min(__popc(__ballot_sync(0xffffffffu, m < limit)), 31);
        odd = m - m1 < limit;
    } else {
        in = b % 64 / 2;
        odd = b & 1;
    }
    if (lane == in) {
        s.at[j] = at + odd;
        s.at_mass[j] = odd ? m - m1 : m - m1 - m0;
        s.at_own[j] = odd ? m1 : m0;
    }
    __syncwarp();
}

// By a warp: the part of a slice's histogram (C CTAs' together) that holds the answer to a limit into at[0], with what lies before it and
// what it holds.
__device__ __noinline__ void find_part(int C, u64 mass_before, uint32_t count_before, bool by_count, u64 limit) {
    Shared& s = shared();
    const cg::cluster_group cluster = cg::this_cluster();
    const int lane = (int)threadIdx.x & 31;
    int b = 0;
    // groups 0 to 31 and 32 to 63, as far as the one with the answer; then its 32 parts
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {
        u64 m0 = 0;
        uint32_t c0 = 0;
        if (step < 2) {
            m0 = s.more_groups.mass[32 * step + lane];
            c0 = s.more_groups.count[32 * step + lane];
        } else {
#pragma unroll 1
            for (int i = 0; i < C; ++i) {
                const Parts* o = C > 1 ? cluster.map_shared_rank(&s.more, i) : &s.more;
                m0 += (u64)o->low[b + lane] + ((u64)o->high[b + lane] << 32);
                c0 += o->count[b + lane];
            }
        }
        const u64 m = scanned(m0);
        const uint32_t c = scanned(c0);
        const int at = __popc(__ballot_sync(0xffffffffu, (by_count ? (u64)count_before + c : mass_before + m) < limit));
        if (step == 0 && at == 32) {
            mass_before += __shfl_sync(0xffffffffu, m, 31);
            count_before += __shfl_sync(0xffffffffu, c, 31);
            continue;
        }
        const int in = min(at, 31);
        if (step < 2) {
            mass_before += __shfl_sync(0xffffffffu, m - m0, in);
            count_before += __shfl_sync(0xffffffffu, c - c0, in);
            b = 32 * (32 * step + in);
            step = 1;
        } else if (lane == in) {
            s.at[0] = b + in;
            s.at_mass[0] = mass_before + m - m0;
            s.at_own[0] = m0;
            s.at_count[0] = count_before + c - c0;
            s.at_members[0] = c0;
        }
    }
    __syncwarp();
}

// f(four values, the first one's token) for a CTA's tokens; values past the last one are -infinity. U 16-byte pieces a
// thread are on their way while as many are looked at.
template <typename E, int U = 2, typename F>
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
    int i = tid;
    if (i + (2 * U - 1) * kSampleThreads < vecs) {
        const uint4* q = v + tid;
        uint4 next[U];
#pragma unroll
        for (int k = 0; k < U; ++k) next[k] = q[k * kSampleThreads];
        do {
            uint4 now[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                now[k] = next[k];
                next[k] = q[(U + k) * kSampleThreads];
            }
#pragma unroll
            for (int k = 0; k < U; ++k) piece(now[k], i + k * kSampleThreads);
            q += U * kSampleThreads;
            i += U * kSampleThreads;
        } while (i + (2 * U - 1) * kSampleThreads < vecs);
#pragma unroll
        for (int k = 0; k < U; ++k) piece(next[k], i + k * kSampleThreads);
        i += U * kSampleThreads;
    }
#pragma unroll 1
    for (; i < vecs; i += kSampleThreads) piece(v[i], i);
#pragma unroll 1
    for (int i = vecs * V + 4 * tid; i < nv; i += 4 * kSampleThreads) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = i + e < nv ? to_f(in[i + e]) : -INFINITY;
        f(x, v0 + i);
    }
}

// Four weights (as Row::beside) into this CTA's histogram: a 64-bit sum as two of 32 bits. b: the slices, beside 2^23 as f32's bits
// (what lies above them leaves by overflow when they become addresses).
template <typename H>
__device__ __forceinline__ void add4(H& h, const uint32_t (&b)[4], const double (&w)[4]) {
    constexpr uint32_t kBeside = 0x4B000000u;
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(h.low) - (kBeside << 2);
    uint32_t was[4], high[4], any = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        asm volatile("atom.shared.add.u32 %0, [%1], %2;" : "=r"(was[e]) : "r"(to + (b[e] << 2)), "r"(__double2loint(w[e])) : "memory");
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t sum;
        asm("add.cc.u32 %0, %2, %3;\n\taddc.u32 %1, %4, 0xBCD00000;"  // (less the high word of 2^52)
            : "=r"(sum), "=r"(high[e])
            : "r"(was[e]), "r"(__double2loint(w[e])), "r"(__double2hiint(w[e])));
        any |= high[e];
    }
    if (any) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (high[e]) atomicAdd(&h.high[b[e] - kBeside], high[e]);
    }
}

template <typename E>
__device__ __noinline__ void numbers_pass(const E* in, int nv) {
    Shared& s = shared();
    const Row r = s.row;
    each<E>(in, 0, nv, [&](const float (&x)[4], int) {
#pragma unroll
        for (int e = 0; e < 4; ++e) atomicAdd(&s.first.low[r.bin(x[e])], 1u);
    });
}

// FULL: values down to the least of all numbers, and returns the sum of this thread's weights that min_p keeps.
template <typename E, bool FULL>
__device__ __noinline__ u64 sums_pass(const E* in, int nv) {
    Shared& s = shared();
    const Row r = s.row;
    u64 likely = 0;
    each<E>(in, 0, nv, [&](const float (&x)[4], int) {
        uint32_t b[4];
        double w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // (what is below the last slice's beginning, or no number, is there, and its weight is less than a half)
            const float y = FULL ? x[e] : fmaxf(x[e], r.floor), at = FULL ? r.place(y) : r.open_place(y);
            b[e] = __float_as_uint(at + 8388608.f);
            w[e] = r.beside(y, at, s.table);
            if (FULL) {
                if (at > (float)kLast - 0.5f) w[e] = kTwo52;
                const u64 n = Row::whole(w[e]);
                if (n >= r.least) likely += n;
            }
        }
        add4(s.first, b, w);
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
        uint32_t b[4];
        double w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t key = key_of(x[e]);
            const bool is = x[e] == x[e] && key >= lo && key <= hi;
            const float at = r.place(x[e]);
            const uint32_t to = is ? (hi - key) >> shift : 0u;
            b[e] = 0x4B000000u + to;
            w[e] = is && r.bin(x[e]) != kLast ? r.beside(x[e], at, s.table) : kTwo52;
            if (is) atomicAdd(&s.more.count[to], 1u);
        }
        add4(s.more, b, w);
    });
}

// The members into this CTA's memory (a histogram's place).
template <typename E, bool KEYS>
__device__ __noinline__ void gather_pass(const E* in, int v0, int nv) {
    Shared& s = shared();
    const Row r = s.row;
    const uint32_t lo = s.find.lo, hi = s.find.hi;
    const int b0 = s.find.b0, b1 = s.find.b1, b2 = s.find.b2;
    // values that the slices lie between, a slice more on either side
    const auto end_of = [&](int b, float off) { return r.step < INFINITY ? fmaf(-((float)b + off), r.step, r.m) : -off * INFINITY; };
    const float lo1 = end_of(b1, 1.5f), hi1 = end_of(b0, -1.5f), lo2 = end_of(b2, 1.5f), hi2 = end_of(b2, -1.5f);
    u64* const stage = reinterpret_cast<u64*>(s.more.low);
    each<E, 4 / (4 / (int)sizeof(E))>(in, v0, nv, [&](const float (&x)[4], int token) {
        uint32_t is = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (KEYS) {
                const uint32_t key = key_of(x[e]);
                if (x[e] == x[e] && key >= lo && key <= hi) is |= 1u << e;
            } else {
                if ((x[e] >= lo1 && x[e] <= hi1) || (x[e] >= lo2 && x[e] <= hi2)) is |= 1u << e;
            }
        }
        if (is) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (is >> e & 1u) {
                    const int b = r.bin(x[e]);
                    if (!KEYS && !((b >= b0 && b <= b1) || b == b2)) continue;
                    const uint32_t at = atomicAdd(&s.staged, 1u);
                    if (at < (uint32_t)kMembers) stage[at] = (u64)key_of(x[e]) << 32 | (uint32_t)~(token + e);
                }
        }
    });
}

// The largest of this thread's values.
template <typename E>
__device__ __noinline__ float most_pass(const E* in, int nv) {
    constexpr int PER = 4 / (int)sizeof(E), V = 4 * PER, U = 4;  // (from HBM: more on their way)
    const int tid = (int)threadIdx.x, vecs = ((uintptr_t)in & 15) == 0 ? nv / V : 0;
    float most = -INFINITY;
#pragma unroll 1
    for (int i = tid; i < vecs; i += U * kSampleThreads) {
        uint4 raw[U];
#pragma unroll
        for (int j = 0; j < U; ++j) raw[j] = reinterpret_cast<const uint4*>(in)[min(i + j * kSampleThreads, vecs - 1)];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
            for (int e = 0; e < V; ++e) most = fmaxf(most, value_in<E>(w[e / PER], e % PER));
        }
    }
#pragma unroll 1
    for (int i = vecs * V + tid; i < nv; i += kSampleThreads) most = fmaxf(most, to_f(in[i]));
    return most;
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
    cluster_barrier(C);
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

// What the CTAs' histograms hold, to all of them.
template <typename H>
__device__ __noinline__ void collect(const H& h, Groups& to, int C, int rank) {
    Shared& s = shared();
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = (int)threadIdx.x;
    __syncthreads();
    if (C == 1) {
        group(h, to);
        __syncthreads();
        return;
    }
    Groups& own = s.from[rank];
    group(h, own);
    __syncthreads();
    static_assert(kGroups * kSampleCluster == kSampleThreads, "a thread a group and CTA");
    const int g = tid % kGroups, c = tid / kGroups;
    if (c < C && c != rank) {
        Groups* const there = cluster.map_shared_rank(&own, c);
        there->mass[g] = own.mass[g];
        if (sizeof(H) == sizeof(Parts)) there->count[g] = own.count[g];
    }
    cluster_barrier(C);
    if (tid < kGroups) {
        u64 m = 0;
        uint32_t n = 0;
#pragma unroll 4
        for (int i = 0; i < C; ++i) m += s.from[i].mass[tid], n += s.from[i].count[tid];
        to.mass[tid] = m;
        to.count[tid] = n;
    }
    __syncthreads();
}

// No slice has more members than its sum has least weights of its (and half a unit each).
__device__ __forceinline__ float most_members(u64 sum, int slice) {
    return __fdividef((float)sum, fmaxf((float)shared().row.lift * exp2f(-(float)(slice + 1) / 64.f) * 0.97f - 1.f, 1e-9f));
}

// The slice of a histogram that holds the answer, and what to do with it. Every CTA works this out for itself, in its first warp.
__device__ __noinline__ void look(bool first, bool sums, int C) {
    Shared& s = shared();
    Search& f = s.find;
    const int lane = (int)threadIdx.x & 31, k = s.k;
    const int warp = (int)threadIdx.x >> 5;
    if (warp == 0) {
        if (s.fresh) {
            const u64 total = warp_sum(s.first_groups.mass[lane] + s.first_groups.mass[lane + 32]);
            if (lane == 0) {
                f.goal = kTopK;
                f.last = 0;
                s.fresh = 0;
                if (!sums) {
                    // (total: of the tokens' number, with those of the last slice that are never drawn)
                    f.limit = min((u64)k, total);
                } else {
                    u64 likely = 0;
                    for (int i = 0; i < C; ++i) likely += s.likely[i];
                    // (the first of the order is kept whatever min_p is)
                    f.likely = s.row.least ? max(likely, (u64)s.row.lift) : total;
                    if (f.k_slice < 0) next_goal(total);
                }
            }
            __syncwarp();
        }
        if (first)
            find(0, C, f.limit, sums && f.goal == kTopK ? f.k_slice : -1);
        else
            find_part(C, f.mass_before, f.count_before, f.goal == kTopK, f.limit);
    }
    __syncthreads();
    const int goal = f.goal, b = s.at[0];
    const bool by_key = f.last < 0;
    const u64 front = s.at_mass[0], own = s.at_own[0];
    const bool both = first && sums && !by_key && (goal == kTopP || (goal == kTopK && !(s.p < 1.f)));
    // (the end of what is kept lies in slice b: and the slices that can hold the token)
    if (both && warp < 2) find(1 + warp, C, drawn(s.u, min(warp ? front + own : front + 1, f.likely)), -1);
    __syncthreads();
    if (threadIdx.x == 0) {
        if (both) {
            f.op = kGather;
            f.b0 = s.at[1];
            f.b1 = s.at[2];
            f.b2 = b;
            f.by_count = goal == kTopK;
            f.goal = kBoth;
            f.mass_before = s.at_mass[1];
            f.more_before = front;
            f.count_before = f.k_before;
            const u64 middle = f.b1 < b ? s.at_mass[2] + s.at_own[2] - s.at_mass[1] : front - s.at_mass[1];
            f.last = most_members(middle, min(f.b1, b)) + (goal == kTopK ? (float)f.k_members : most_members(own, b)) <= (float)kMembers;
        } else {
            uint32_t lo = 0, hi = 0, members = first ? goal == kTopK && sums ? f.k_members : ~0u : s.at_members[0];
            bool into = false;
            if (!first) {
                hi = f.hi - ((uint32_t)b << f.shift);
                const uint32_t span = (1u << f.shift) - 1;
                lo = hi - f.lo > span ? hi - span : f.lo;
                f.count_before = s.at_count[0];
                into = true;
            } else if (!sums) {
                // front and own are numbers of tokens
                if (s.few && (b == kLast ? front : front + own) <= (u64)kMembers) {
                    // the kept ones and no more than kMembers in all (those of the last slice have no weight)
                    f.goal = kPrefix;
                    f.limit = b == kLast ? min(f.limit, front) : f.limit;
                    f.op = kGather;
                    f.b0 = 0;
                    f.b1 = f.b2 = b == kLast ? b - 1 : b;
                    f.last = 1;
                } else {
                    f.op = kSums;
                    f.k_slice = b == kLast ? -1 : b;
                    f.k_before = (uint32_t)front;
                    f.k_members = (uint32_t)own;
                }
            } else if (!by_key && (goal == kDraw || members <= (uint32_t)kMembers)) {
                f.mass_before = front;
                f.count_before = f.k_before;
                f.op = kGather;
                f.b0 = f.b1 = f.b2 = b;
                f.last = goal == kDraw && most_members(own, b) <= (float)kMembers;
            } else {
                lo = lowest_key(b);
                hi = b ? lowest_key(b - 1) - 1 : key_of(s.row.m);
                f.count_before = f.k_before;
                into = true;
            }
            if (into) {
                f.mass_before = front;
                f.lo = lo;
                f.hi = hi;
                f.last = 0;
                if (members <= (uint32_t)kMembers) {
                    f.op = kGatherKeys;
                } else if (lo < hi) {
                    f.op = kDivide;
                    f.shift = shift_of(hi - lo);
                } else {
                    // equal keys
                    const Row r = s.row;
                    const float x = value_of(lo);
                    const u64 w = r.weight(x, s.table);
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
    }
    __syncthreads();
}

// By the first CTA: of the members of slices [lo, hi], before which the row's sum and number are `before` and `number`, the first
// whose running sum, or number, reaches `limit`, into at_one; returns its running sum.
__device__ __noinline__ u64 reach(int lo, int hi, u64 before, uint32_t number, bool by_count, u64 limit) {
    Shared& s = shared();
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31, n = (int)s.members;
    const Row r = s.row;
    const u64* const weight = s.weight;
    uint32_t klo = 0, khi = ~0u;
    int part = -1;  // of the set, first divided into kSampleThreads parts by its place among the slices
    const float begin = (float)lo - 0.5f, scale = (float)kSampleThreads / (float)(hi - lo + 1);
    const auto part_of = [&](float x) {
        return (int)fminf(fmaxf((r.place(x) - begin) * scale, 0.f), (float)(kSampleThreads - 1));
    };
    // f(index, key) for this thread's members of the set; returns the set's size
    const auto members = [&](auto f) {
        int size = 0;
#pragma unroll 1
        for (int base = 0; base < n; base += kSampleThreads) {
            const int i = base + tid;
            const uint32_t key = i < n ? (uint32_t)(s.member[i] >> 32) : 0u;
            bool is = i < n && key >= klo && key <= khi;
            if (is) {
                const float x = value_of(key);
                const int b = r.bin(x);
                is = b >= lo && b <= hi && (part < 0 || part_of(x) == part);
            }
            if (is) f(i, key);
            size += __syncthreads_count(is);
        }
        return size;
    };
    const auto note = [&](int to, u64 w) {
        atomicAdd(&s.more.count[to], 1u);
        const uint32_t was = atomicAdd(&s.more.low[to], (uint32_t)w);
        atomicAdd(&s.more.high[to], (uint32_t)(w >> 32) + (was + (uint32_t)w < was));
    };
    int size = members([&](int i, uint32_t key) { note(part_of(value_of(key)), weight[i]); });
    {
        const u64 m0 = (u64)s.more.low[tid] + ((u64)s.more.high[tid] << 32);
        const uint32_t c0 = s.more.count[tid];
        const u64 m = scanned(m0);
        const uint32_t c = scanned(c0);
        if (lane == 31) s.warp_mass[warp] = m, s.warp_count[warp] = c;
        __syncthreads();
        u64 mass = before + m - m0;
        uint32_t count = number + c - c0;
#pragma unroll 4
        for (int i = 0; i < warp; ++i) mass += s.warp_mass[i], count += s.warp_count[i];
        const u64 had = by_count ? count : mass, has = by_count ? count + c0 : mass + m0;
        if (had < limit && limit <= has) {
            s.at[0] = tid;
            s.at_mass[0] = mass;
            s.at_count[0] = count;
            s.at_members[0] = c0;
        }
        s.more.low[tid] = s.more.high[tid] = s.more.count[tid] = 0;
        __syncthreads();
        part = s.at[0];
        before = s.at_mass[0];
        number = s.at_count[0];
        size = (int)s.at_members[0];
    }
#pragma unroll 1
    while (size > kFew) {
        // the set's keys from lowest to highest, divided
        uint32_t least = ~0u, most = 0;
        members([&](int, uint32_t key) {
            least = min(least, key);
            most = max(most, key);
        });
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) s.warp_lo[warp] = least, s.warp_hi[warp] = most;
        __syncthreads();
        klo = __reduce_min_sync(0xffffffffu, s.warp_lo[lane % kSampleWarps]);
        khi = __reduce_max_sync(0xffffffffu, s.warp_hi[lane % kSampleWarps]);
        if (klo == khi) break;
        const int shift = shift_of(khi - klo);
        members([&](int i, uint32_t key) { note((int)((khi - key) >> shift), weight[i]); });
        group(s.more, s.more_groups);
        __syncthreads();
        if (warp == 0) find_part(1, before, number, by_count, limit);
        __syncthreads();
        before = s.at_mass[0];
        number = s.at_count[0];
        size = (int)s.at_members[0];
        const uint32_t top = khi - ((uint32_t)s.at[0] << shift), span = (1u << shift) - 1;
        klo = top - klo > span ? top - span : klo;
        khi = top;
        clear(s.more);
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
#pragma unroll 1
        for (int i = tid; i < n; i += kSampleThreads) {
            const float x = value_of((uint32_t)(s.member[i] >> 32));
            const u64 w = r.weight(x, s.table);
            s.weight[i] = w;
            if (w >= r.least) likely += w;
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
    if (n <= kFew) {
        // a few members: four threads each find how many are before it and their sum, then a warp asks
        const int e = min(tid / 4, n - 1);
        const u64 mine = s.member[e], own = s.weight[e];
        u64 sum = 0;
        int place = 0;
#pragma unroll 4
        for (int i = tid % 4; i < n; i += 4)
            if (s.member[i] > mine) {
                ++place;
                sum += s.weight[i];
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            place += __shfl_xor_sync(0xffffffffu, place, o);
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (tid % 4 == 0 && tid / 4 < n) {
            s.set_member[place] = mine;
            s.set_weight[place] = sum + own;  // the running sum
            s.set_slice[place] = Row(s.row).bin(value_of((uint32_t)(mine >> 32)));
        }
        __syncthreads();
        if (warp != 0) return;
        // the first place in [from, n) whose running sum and `more` reach the limit
        const auto seek = [&](int from, u64 more, u64 limit) {
            int at = from;
#pragma unroll 1
            for (int i = lane; i - lane < n; i += 32) at += __popc(__ballot_sync(0xffffffffu, i >= from && i < n && s.set_weight[i] + more < limit));
            return min(at, n - 1);
        };
        int at = 0;
        if (goal == kPrefix) {
            kept = s.set_weight[s.find.limit - 1];
            if (p < 1.f) kept = s.set_weight[seek(0, 0, nucleus(p, kept))];
            kept = min(kept, likely);
            at = seek(0, 0, drawn(u, kept));
        } else if (goal == kBoth) {
            // (members of slices before b2, then those of b2, which others lie in front of)
            int ahead = 0;
            for (int i = lane; i - lane < n; i += 32) ahead += __popc(__ballot_sync(0xffffffffu, i < n && s.set_slice[i] < s.find.b2));
            const u64 more = s.find.more_before - (ahead ? s.set_weight[ahead - 1] : 0);
            at = s.find.by_count ? ahead + (int)(s.find.limit - s.find.count_before) - 1 : seek(ahead, more, s.find.limit);
            kept = min(s.set_weight[at] + more, s.find.likely);
            at = seek(0, s.find.mass_before, drawn(u, kept));
        } else if (goal == kTopK) {
            at = (int)(s.find.limit - s.find.count_before) - 1;
        } else {
            at = seek(0, s.find.mass_before, s.find.limit);
        }
        answer = s.find.mass_before + s.set_weight[at];
        if (lane == 0) s.at_one = s.set_member[at];
        __syncwarp();
    } else {
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
                hi = s.find.b1;
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
                    by_count = s.find.by_count;
                    number = s.find.count_before;
                } else {
                    lo = s.find.b0;
                    hi = s.find.b1;
                    kept = min(kept, s.find.likely);
                    limit = drawn(u, kept);
                }
            } else {
                if (s.find.op == kGather) lo = s.find.b0, hi = s.find.b1;
                by_count = goal == kTopK;
                number = s.find.count_before;
            }
            answer = reach(lo, hi, before, number, by_count, limit);
            if (q + 1 < questions) kept = answer;
        }
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
    cluster_begun(C);
    clear(s.first);
    clear(s.more);
    const double lift = __longlong_as_double((long long)(1023 + a.bits) << 52);
    if (tid < 32) s.table[tid] = exp2(-tid / 32.0) * lift;
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
        s.fresh = 1;
        s.row.per_t = 46.166241308446828 / (double)fmaxf(T0, 7.8886091e-31f);  // 2^-100: what follows stays within f32's range
        s.find.k_slice = -1;
        s.find.k_before = s.find.k_members = 0;
    }
    // ---- the largest
    {
        float e = most_pass<E>(in, nv);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) e = fmaxf(e, __shfl_xor_sync(0xffffffffu, e, o));
        if (lane == 0) s.warp_ends[warp] = e;
        __syncthreads();
        cluster_all_begun(C);
        if (warp == 0) {
            e = s.warp_ends[lane % kSampleWarps];
#pragma unroll
            for (int o = 1; o < kSampleWarps; o <<= 1) e = fmaxf(e, __shfl_xor_sync(0xffffffffu, e, o));
            if (lane < C) cluster.map_shared_rank(&s, lane)->ends[rank] = e;
        }
        cluster_barrier(C);
    }
    int op;
    {
        Row r;
        r.m = -INFINITY;
        for (int i = 0; i < C; ++i) r.m = fmaxf(r.m, s.ends[i]);
        if (r.m == -INFINITY) {
            if (rank == 0 && tid == 0) {
                a.token[row] = -1;
                if (a.logprob) a.logprob[row] = -INFINITY;
            }
            return;
        }
        // the first of the order; or, beside +infinity, only what is: tokens of equal weights
        op = !(T0 > 0.f) || k == 1 ? kTies : r.m == INFINITY ? kCrowd : k > 1 && k < a.vocab ? kNumbers : kSums;
        if (tid == 0) {
            r.half_m = 0.5f * r.m;
            r.per_t = s.row.per_t;
            r.lift = lift;
            r.least = min_p > 0.f ? min_p <= 1.f ? (u64)ceil((double)min_p * lift) : ~0ull : 0;
            r.scale = (float)(4.0 * r.per_t);  // (64 slices to 32 parts, for halves)
            const float step = 0.5f / (float)r.per_t;
            // (m a few million slices from 0 at most: sums and differences of slices' ends are off by a small part of one)
            const bool near = fabsf(r.m) < 4194304.f * step && step < 1e24f;
            r.step = near ? step : INFINITY;
            r.floor = near ? r.m - (float)kLast * step : -INFINITY;
            s.row = r;
            s.find.lo = key_of(r.m);
            s.find.nth = 1;
            s.find.logprob = 0.f;
        }
        __syncthreads();
    }
    // (a row takes two or three rounds, with equal keys by the thousand some more; none takes as many as this)
#pragma unroll 1
    for (int round = 0; round < 64; ++round) {
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
            const u64* const stage = reinterpret_cast<const u64*>(s.more.low);
#pragma unroll 1
            for (uint32_t i = tid; i < staged && base + i < (uint32_t)kMembers; i += kSampleThreads) head->member[base + i] = stage[i];
            __syncthreads();
            clear(s.more);
            cluster_barrier(C);
            if (last && rank != 0) return;
            if (rank == 0) {
                if (last && s.members > (uint32_t)kMembers) break;  // (cannot be; the other CTAs have gone)
                if (s.members > (uint32_t)kMembers) {
                    // (a slice whose tokens were not counted has more than that: by its keys)
                    if (tid == 0) {
                        if (s.find.goal == kBoth) s.find.goal = s.find.by_count ? kTopK : kTopP;
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
            cluster_barrier(C);
            if (rank != 0 && tid == 0) s.find = head->find;
            cluster_barrier(C);
            op = s.find.op;
            if (op == kDone) return;
        }
        if (op == kDivide) {
            cluster_barrier(C);  // what the histograms before held is read by all
            divide_pass<E>(in, nv);
        } else if (op == kNumbers) {
            numbers_pass<E>(in, nv);
        } else if (op == kSums) {
            if (k > 1 && k < a.vocab) {
                // (the numbers there are first: read by all, then cleared)
                cluster_barrier(C);
                clear(s.first);
                if (tid == 0) s.fresh = 1;
                __syncthreads();
            }
            if (s.row.least || s.row.floor == -INFINITY) {
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
        if (op == kDivide)
            collect(s.more, s.more_groups, C, rank);
        else if (op != kLook)
            collect(s.first, s.first_groups, C, rank);
        look(op != kDivide, op != kNumbers, C);
        if (op == kDivide) {
            cluster_barrier(C);  // read by all, then cleared
            clear(s.more);
            __syncthreads();
        }
        op = s.find.op;
    }
    if (rank == 0 && tid == 0) {
        a.token[row] = -1;
        if (a.logprob) a.logprob[row] = -INFINITY;
    }
    cluster_barrier(C);  // no CTA ends while another reads its memory
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
    while (vocab > 1ll << (62 - bits)) --bits;  // (at least 40)
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
