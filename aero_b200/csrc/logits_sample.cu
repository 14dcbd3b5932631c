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
constexpr int kBins = 4 * kSampleThreads;
constexpr int kMembers = 2048;
constexpr int kMostVocab = 1 << 22;
constexpr uint32_t kNone = 0x007FFFFFu;  // the key of -infinity

struct SampleArgs {
    const void* in;
    int64_t ld;
    int vocab, slice, bits;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int32_t* token;
    float* logprob;
};

// Keys in the values' order; -0 as 0, no number as -infinity.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? kNone : b >> 31 ? ~b : b | 0x80000000u;
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

// What all threads know of a row.
struct Row {
    float m;      // its largest logit
    float scale;  // of the first histogram: slice = (m - x) * scale
    double rate;  // log2(e) / T
    double least; // min_p
    double lift;  // 2^B
    __device__ int bin(uint32_t key) const {
        const float x = value_of(key), b = (x == m ? 0.f : m - x) * scale;
        return b < (float)(kBins - 1) ? (int)b : kBins - 1;
    }
    // w relative to the largest, in 64 bits
    __device__ double relative(uint32_t key) const {
        const float x = value_of(key);
        if (x == m) return 1.0;
        const double d = (double)m - (double)x;
        return d < 1e300 ? exp2(-d * rate) : 0.0;
    }
    // the nearest whole number of 2^-B (lift is at most 2^48)
    __device__ u64 whole(double relative) const {
        return (u64)(__double_as_longlong(fma(relative, lift, 4503599627370496.0)) - __double_as_longlong(4503599627370496.0));
    }
    __device__ u64 weight(uint32_t key) const { return whole(relative(key)); }
};

enum { kDone, kHistogram, kGather, kTies };   // what the cluster does next
// what the first CTA looks for: the end of what top_k keeps, of what top_p keeps, the token; or one of the first two
// among members that begin with the row's first, and then all the rest
enum { kTopK, kTopP, kDraw, kPrefixK, kPrefixP };

// The first CTA's orders to its cluster.
struct Plan {
    int op;
    uint32_t lo, hi;  // keys
    int shift;        // of a histogram: slice = (hi - key) >> shift; -1: Row::bin
    int masses;       // a histogram has sums too
    uint32_t nth;     // kTies: which of them, from 1
    float logprob;
};

// What the first CTA has found so far.
struct Search {
    int goal;
    u64 limit;               // the running sum, or number (kTopK), to be reached
    u64 mass_before, total;  // sums: before the slice in hand, of the row
    u64 kept;                // S
    u64 likely;              // of those that min_p keeps
    uint32_t count_before;
};

struct Shared {
    u64 own_mass[kBins];      // this CTA's histogram
    u64 first_mass[kBins];    // the row's first histogram (in the first CTA)
    u64 more_mass[kBins];     // the row's histogram of a slice (in the first CTA); then the members' running sums
    u64 member[kMembers];     // key, then all ones less the token's number (in the first CTA)
    uint32_t own_count[kBins], first_count[kBins], more_count[kBins];
    u64 warp_mass[kSampleWarps];
    uint32_t warp_count[kSampleWarps];
    u64 best, likely;         // this CTA's: largest key with its number; sum of those that min_p keeps
    uint32_t least;           // smallest key but -infinity's
    uint32_t ties;
    uint32_t members;
    Plan plan;
    Search find;
    int at;
    u64 at_mass, at_own;
    uint32_t at_count, at_members;
};

__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Exclusive sums over the CTA of a mass and a count a thread; every thread calls it.
__device__ void scan2(Shared& s, u64& mass, uint32_t& count) {
    const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
    const u64 m0 = mass;
    const uint32_t c0 = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 m = __shfl_up_sync(0xffffffffu, mass, o);
        const uint32_t c = __shfl_up_sync(0xffffffffu, count, o);
        if (lane >= o) mass += m, count += c;
    }
    __syncthreads();
    if (lane == 31) s.warp_mass[warp] = mass, s.warp_count[warp] = count;
    __syncthreads();
    for (int i = 0; i < warp; ++i) mass += s.warp_mass[i], count += s.warp_count[i];
    mass -= m0;
    count -= c0;
}

// The members' order: falling, by compare and exchange.
__device__ void sort_members(u64* a, int n) {
    int size = 1;
    while (size < n) size <<= 1;
    for (int i = n + (int)threadIdx.x; i < size; i += kSampleThreads) a[i] = 0;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int i = (int)threadIdx.x; i < size / 2; i += kSampleThreads) {
                const int x = 2 * i - (i & (j - 1)), y = x + j;
                const u64 p = a[x], q = a[y];
                if ((p < q) == ((x & k) == 0)) a[x] = q, a[y] = p;
            }
        }
    __syncthreads();
}

__device__ __forceinline__ float log_of(const Row& r, uint32_t key, u64 kept) {
    const float x = value_of(key);
    const double t = x == r.m ? 0.0 : ((double)r.m - (double)x) * r.rate;  // in powers of two
    return (float)((-t - log2((double)kept / r.lift)) * 0.6931471805599453);
}

// u S as the running sum to be reached: the first above it.
__device__ __forceinline__ u64 drawn(float u, u64 kept) {
    const double v = u > 0.f ? fmin((double)u, 1.0) * (double)kept : 0.0;
    return min((u64)v + 1, kept);
}
// p S, likewise: the kept ones end with the first that reaches it
__device__ __forceinline__ u64 nucleus(float p, u64 sum) {
    const double v = p > 0.f ? ceil((double)p * (double)sum) : 1.0;
    return min(max((u64)v, 1ull), sum);
}

// The next goal, once a prefix's sum is known.
__device__ void next_goal(Search& f, u64 kept, float p, float u) {
    if (f.goal == kTopK && p < 1.f) {
        f.goal = kTopP;
        f.limit = nucleus(p, kept);
    } else {
        f.goal = kDraw;
        f.kept = min(kept, f.likely);
        f.limit = drawn(u, f.kept);
    }
}

// The keys of the first histogram's slice b: `above` ones have a smaller slice. Row::bin does not rise with the key.
__device__ uint32_t lowest_key(const Row& r, int b) {  // the lowest key whose slice is at most b
    uint32_t lo = kNone + 1, hi = key_of(r.m);         // (the largest is of slice 0)
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (r.bin(mid) <= b)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

template <typename E>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    constexpr int V = 16 / (int)sizeof(E), U = 4;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = (int)blockIdx.x / C;
    const int v0 = min(a.vocab, rank * a.slice), nv = min(a.vocab - v0, a.slice);
    const E* in = static_cast<const E*>(a.in) + (int64_t)row * a.ld + v0;
    const bool vec = ((uintptr_t)in & 15) == 0;
    stream_turn();
    // f(key, token) for each of this CTA's tokens that is not -infinity
    const auto each = [&](auto f) {
        for (int base = 0; base < nv; base += kSampleThreads * V * U) {
            uint4 raw[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int i = base + (k * kSampleThreads + tid) * V;
                E* x = reinterpret_cast<E*>(raw + k);
                if (vec && i + V <= nv) {
                    raw[k] = *reinterpret_cast<const uint4*>(in + i);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (i + j < nv) x[j] = in[i + j];
                }
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int i = base + (k * kSampleThreads + tid) * V;
                const E* x = reinterpret_cast<const E*>(raw + k);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const uint32_t key = i + j < nv ? key_of(to_f(x[j])) : kNone;
                    if (key > kNone) f(key, v0 + i + j);
                }
            }
        }
    };
    // ---- the largest and the smallest
    u64 best = 0;
    uint32_t least = ~0u;
    each([&](uint32_t key, int token) {
        best = max(best, (u64)key << 32 | (uint32_t)~token);
        least = min(least, key);
    });
    best = warp_max(best);
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) s.warp_mass[warp] = best, s.warp_count[warp] = least;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kSampleWarps; ++i) {
            best = max(best, s.warp_mass[i]);
            least = min(least, s.warp_count[i]);
        }
        s.best = best;
        s.least = least;
        s.members = 0;
    }
    cluster.sync();
    best = 0, least = ~0u;
    for (int i = 0; i < C; ++i) {
        const Shared* o = cluster.map_shared_rank(&s, i);
        best = max(best, o->best);
        least = min(least, o->least);
    }
    const float T = a.temperature ? a.temperature[row] : 1.f;
    const int k = a.top_k ? a.top_k[row] : 0;
    if (best == 0 || !(T > 0.f) || k == 1) {
        if (rank == 0 && tid == 0) {
            a.token[row] = best == 0 ? -1 : (int)~(uint32_t)best;
            if (a.logprob) a.logprob[row] = best == 0 ? -INFINITY : 0.f;
        }
        cluster.sync();  // no CTA ends while another reads its memory
        return;
    }
    const float p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f, u = a.u[row];
    Row r;
    r.m = value_of((uint32_t)(best >> 32));
    r.rate = 1.4426950408889634 / (double)T;
    r.least = min_p > 0.f ? (double)min_p : 0.0;
    r.lift = __longlong_as_double((long long)(1023 + a.bits) << 52);
    {
        // the range that the first histogram divides: all values, or what matters of them
        const float all = r.m - value_of(least), matters = fmaxf(32.f * T, 24.f);
        const float range = all < matters ? all : matters;
        r.scale = range > 0.f ? fminf((float)(kBins - 1) / range, 1e30f) : 0.f;
    }
    const bool few = k > 1 && k <= kMembers;  // the first histogram needs no sums
    // ---- this CTA's histogram of the keys in [lo, hi], then the row's into the first CTA's arrays
    const auto histogram = [&](uint32_t lo, uint32_t hi, int shift, bool masses, bool first) {
        for (int i = tid; i < kBins; i += kSampleThreads) s.own_count[i] = 0, s.own_mass[i] = 0;
        __syncthreads();
        u64 likely = 0;
        each([&](uint32_t key, int) {
            if (key < lo || key > hi) return;
            const int b = shift < 0 ? r.bin(key) : (int)((hi - key) >> shift);
            atomicAdd(&s.own_count[b], 1u);
            if (masses) {
                const double w = r.relative(key);
                const u64 n = r.whole(w);
                if (n) atomicAdd(&s.own_mass[b], n);
                if (w >= r.least) likely += n;
            }
        });
        if (first) {
            likely = warp_sum(likely);
            if (lane == 0) s.warp_mass[warp] = likely;
            __syncthreads();
            if (tid == 0) {
                for (int i = 1; i < kSampleWarps; ++i) likely += s.warp_mass[i];
                s.likely = likely;
            }
        }
        cluster.sync();
        Shared* to = cluster.map_shared_rank(&s, 0);
        for (int b = rank * (kBins / C) + tid; b < (rank + 1) * (kBins / C); b += kSampleThreads) {
            uint32_t c = 0;
            u64 m = 0;
            for (int i = 0; i < C; ++i) {
                const Shared* o = cluster.map_shared_rank(&s, i);
                c += o->own_count[b];
                if (masses) m += o->own_mass[b];
            }
            (first ? to->first_count : to->more_count)[b] = c;
            (first ? to->first_mass : to->more_mass)[b] = m;
        }
        cluster.sync();
    };
    // ---- by the first CTA: the slice of a histogram that holds the answer, and what to do with it
    const auto look = [&](bool first, uint32_t hi, int shift) {
        const uint32_t* counts = first ? s.first_count : s.more_count;
        const u64* masses = first ? s.first_mass : s.more_mass;
        if (tid == 0 && first) s.find.mass_before = 0, s.find.count_before = 0;
        u64 m = 0;
        uint32_t c = 0;
        for (int i = 4 * tid; i < 4 * tid + 4; ++i) m += masses[i], c += counts[i];
        scan2(s, m, c);
        m += s.find.mass_before;
        c += s.find.count_before;
        const u64 limit = s.find.limit;
        const bool by_count = s.find.goal == kTopK;
        for (int i = 4 * tid; i < 4 * tid + 4; ++i) {
            const u64 had = by_count ? c : m, has = by_count ? c + counts[i] : m + masses[i];
            if (had < limit && limit <= has) {
                s.at = i;
                s.at_mass = m;
                s.at_count = c;
                s.at_members = counts[i];
            }
            m += masses[i];
            c += counts[i];
        }
        __syncthreads();
        if (tid != 0) return;
        Search& f = s.find;
        Plan& plan = s.plan;
        plan.masses = 1;
        f.mass_before = s.at_mass;
        f.count_before = s.at_count;
        uint32_t lo;
        if (shift < 0) {
            lo = lowest_key(r, s.at);
            hi = s.at ? lowest_key(r, s.at - 1) - 1 : key_of(r.m);
            if (f.goal != kDraw && s.at_count + s.at_members <= (uint32_t)kMembers) {
                // all that may be kept, at once
                f.goal = f.goal == kTopK ? kPrefixK : kPrefixP;
                plan.op = kGather;
                plan.lo = lo;
                plan.hi = ~0u;
                f.mass_before = 0;
                f.count_before = 0;
                return;
            }
        } else {
            hi -= (uint32_t)s.at << shift;
            const uint32_t span = (1u << shift) - 1;
            lo = hi - plan.lo > span ? hi - span : plan.lo;
        }
        plan.lo = lo;
        plan.hi = hi;
        if (s.at_members <= (uint32_t)kMembers) {
            plan.op = kGather;
        } else if (lo < hi) {
            plan.op = kHistogram;
            plan.shift = max(0, 21 - __clz((int)(hi - lo)));  // (hi - lo) >> shift < kBins = 2^11
        } else {
            // equal keys
            const u64 w = r.weight(lo);
            const u64 nth = f.goal == kTopK ? f.limit - f.count_before : (f.limit - f.mass_before + w - 1) / w;
            const u64 sum = f.mass_before + nth * w;
            if (f.goal == kDraw) {
                plan.op = kTies;
                plan.nth = (uint32_t)nth;
                plan.logprob = log_of(r, lo, f.kept);
            } else {
                next_goal(f, sum, p, u);
                plan.op = kHistogram;
                plan.shift = -2;  // the first histogram again, which is still there
            }
        }
    };
    // ---- by the first CTA: the members of a slice, sorted, and their running sums
    const auto settle = [&]() {
        const int n = (int)min(s.members, (uint32_t)kMembers);
        sort_members(s.member, n);
        constexpr int kRun = kMembers / kSampleThreads;
        u64* run = s.more_mass;
        static_assert(kMembers <= kBins, "the running sums' place");
        u64 w[kRun], m = 0;
        uint32_t likely = 0;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int at = kRun * tid + i;
            w[i] = 0;
            if (at < n) {
                const double x = r.relative((uint32_t)(s.member[at] >> 32));
                w[i] = r.whole(x);
                likely += x >= r.least;
            }
            m += w[i];
        }
        uint32_t before = likely;
        u64 sum = m;
        scan2(s, sum, before);
        sum += s.find.mass_before;
        u64 at_sum[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            sum += w[i];
            at_sum[i] = sum;
            if (kRun * tid + i < n) run[kRun * tid + i] = sum;
        }
        if (tid == kSampleThreads - 1) s.at_count = before + likely;  // of the members that min_p keeps
        __syncthreads();
        // the first running sum that reaches a limit
        const auto reaches = [&](u64 limit) {
            u64 had = at_sum[0] - w[0];
#pragma unroll
            for (int i = 0; i < kRun; ++i) {
                if (kRun * tid + i < n && had < limit && limit <= at_sum[i]) s.at = kRun * tid + i;
                had = at_sum[i];
            }
            __syncthreads();
            const int at = s.at;
            __syncthreads();
            return at;
        };
        const int goal = s.find.goal;
        int at;
        u64 kept = 0;
        if (goal >= kPrefixK) {
            kept = goal == kPrefixK ? run[(int)s.find.limit - 1] : run[reaches(s.find.limit)];
            if (goal == kPrefixK && p < 1.f) kept = run[reaches(nucleus(p, kept))];
            kept = min(kept, run[max(1u, s.at_count) - 1]);
            at = reaches(drawn(u, kept));
        } else if (goal == kTopK) {
            at = (int)(s.find.limit - s.find.count_before) - 1;
        } else {
            kept = s.find.kept;
            at = reaches(s.find.limit);
        }
        if (tid != 0) return;
        if (goal >= kDraw) {
            a.token[row] = (int)~(uint32_t)s.member[at];
            if (a.logprob) a.logprob[row] = log_of(r, (uint32_t)(s.member[at] >> 32), kept);
            s.plan.op = kDone;
        } else {
            next_goal(s.find, run[at], p, u);
            s.plan.op = kHistogram;
            s.plan.shift = -2;
        }
    };
    // ---- begin: the first histogram, and the first goal
    const auto begin = [&](bool masses) {
        histogram(kNone + 1, ~0u, -1, masses, true);
        if (rank != 0) return;
        u64 m = 0, likely = 0;
        uint32_t c = 0;
        for (int i = 4 * tid; i < 4 * tid + 4; ++i) m += s.first_mass[i], c += s.first_count[i];
        const u64 m0 = m;
        const uint32_t c0 = c;
        scan2(s, m, c);
        if (tid == kSampleThreads - 1) {
            Search& f = s.find;
            f.total = m + m0;
            const uint32_t count = c + c0;
            for (int i = 0; i < C; ++i) likely += cluster.map_shared_rank(&s, i)->likely;
            // (the first of the order stays whatever min_p is)
            f.likely = r.least > 0.0 ? max(likely, (u64)r.lift) : f.total;
            f.goal = kTopK;
            if (k > 1 && (uint32_t)k < count)
                f.limit = (u64)k;
            else if (few)
                f.limit = count;  // the members are all of them
            else
                next_goal(f, f.total, p, u);
        }
        __syncthreads();
        look(true, 0, -1);
        if (tid == 0 && !masses && s.find.goal != kPrefixK) s.plan.op = kHistogram, s.plan.shift = -1;  // with sums
    };
    begin(!few);
    for (;;) {
        cluster.sync();
        const Plan plan = cluster.map_shared_rank(&s, 0)->plan;
        if (plan.op == kDone) break;
        if (plan.op == kHistogram) {
            cluster.sync();  // the plan is read by all before it changes
            if (plan.shift == -1) {
                begin(true);
            } else if (plan.shift == -2) {
                if (rank == 0) {
                    look(true, 0, -1);
                }
            } else {
                histogram(plan.lo, plan.hi, plan.shift, true, false);
                if (rank == 0) look(false, plan.hi, plan.shift);
            }
        } else if (plan.op == kGather) {
            Shared* to = cluster.map_shared_rank(&s, 0);
            each([&](uint32_t key, int token) {
                if (key < plan.lo || key > plan.hi) return;
                const uint32_t at = atomicAdd(&to->members, 1u);
                if (at < (uint32_t)kMembers) to->member[at] = (u64)key << 32 | (uint32_t)~token;
            });
            cluster.sync();
            if (rank == 0) {
                settle();
                __syncthreads();
                if (tid == 0) s.members = 0;
            }
        } else {
            // the nth token with the key: each thread counts a run of tokens
            const int run = (nv + kSampleThreads - 1) / kSampleThreads;
            const int i0 = min(nv, tid * run), i1 = min(nv, i0 + run);
            uint32_t count = 0;
            for (int i = i0; i < i1; ++i) count += key_of(to_f(in[i])) == plan.lo;
            u64 none = 0;
            uint32_t before = count;
            scan2(s, none, before);
            if (tid == kSampleThreads - 1) s.ties = before + count;
            cluster.sync();
            for (int i = 0; i < rank; ++i) before += cluster.map_shared_rank(&s, i)->ties;
            if (before < plan.nth && plan.nth <= before + count) {
                for (int i = i0; i < i1; ++i)
                    if (key_of(to_f(in[i])) == plan.lo && ++before == plan.nth) a.token[row] = v0 + i;
                if (a.logprob) a.logprob[row] = plan.logprob;
            }
            break;
        }
    }
    cluster.sync();
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
