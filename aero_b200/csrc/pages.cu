// The paged key/value cache's handle, its books and its page moves
// (include/aero_cuda_pages.h).
//
// Books kernels (extend, fork, compact) are one CTA of 1024 threads: their work is a
// scan over the free pages and a few entries per sequence, a matter of latency. They
// check everything before they change anything, so a refused call leaves the books
// as they were. Every number they write follows from the call's list and the books
// alone (integer scans and sums), so a call's result does not depend on timing.
//
// Row and page moves are grids over 16-byte pieces, bound by HBM.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <string>

#include "gemm.h"
#include "internal.h"
#include "pages.h"

namespace aero {
namespace {

constexpr int kBooksThreads = 1024;

// One page move: rows [0, rows) of page src to page dst, in every layer and kv head.
struct PageJob {
    int32_t src, dst, rows;
};

// Scratch of the books kernels.
struct BooksWork {
    int32_t* list;    // (n_page) pages found by a scan
    int32_t* to;      // (n_page) where a moved page went
    int32_t* mark;    // (n_seq) which entry of the call's list names a sequence
    int32_t* first;   // (n_seq) entry -> its first place in list
    int32_t* len;     // (n_seq) entry -> its sequence's length when the call began
    PageJob* jobs;    // (max(n_page, n_seq))
    int32_t* n_jobs;
    int32_t* n_live;
    int32_t* lowest;  // every page below it is held: where a scan for free ones begins
};

// Exclusive sum of v over the CTA; *total the whole sum. Every thread calls it.
__device__ int block_scan(int v, int* total) {
    __shared__ int warp_sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        const int nw = (int)blockDim.x >> 5;
        const int w0 = lane < nw ? warp_sums[lane] : 0;
        int w = w0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        if (lane < nw) warp_sums[lane] = w;
    }
    __syncthreads();
    const int before = warp ? warp_sums[warp - 1] : 0;
    *total = warp_sums[((int)blockDim.x >> 5) - 1];
    __syncthreads();  // warp_sums may be written again
    return before + x - v;
}

// refs of pages [p0, p0 + 4), 1 past the last page (a 16-byte load: p0 a multiple of 4,
// the array is padded to one).
__device__ __forceinline__ int4 refs4(const PageView& c, int p0) {
    int4 r = make_int4(1, 1, 1, 1);
    if (p0 < c.n_page) {
        r = *reinterpret_cast<const int4*>(c.refs + p0);
        if (p0 + 1 >= c.n_page) r.y = 1;
        if (p0 + 2 >= c.n_page) r.z = 1;
        if (p0 + 3 >= c.n_page) r.w = 1;
    }
    return r;
}

// w.list[0 .. want) = the lowest free pages; false when there are fewer. The scan begins at w.lowest, 4096
// pages a step, so a decode step's extend finds its pages in the first steps where they lie just above
// it; where they do not, it walks the held pages between (a pool of 2^20 pages with one free: at its
// beginning 8 us, in its middle 124, at its end 238, once).
__device__ bool lowest_free(const PageView& c, const BooksWork& w, int want) {
    int32_t* list = w.list;
    int found = 0;
    for (int base = *w.lowest & ~3; base < c.n_page && found < want; base += 4 * (int)blockDim.x) {
        const int p0 = base + 4 * (int)threadIdx.x;
        const int4 r = refs4(c, p0);
        const int free4[4] = {r.x == 0, r.y == 0, r.z == 0, r.w == 0};
        int total;
        int at = found + block_scan(free4[0] + free4[1] + free4[2] + free4[3], &total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (free4[i]) {
                if (at < want) list[at] = p0 + i;
                ++at;
            }
        found += total;
    }
    __syncthreads();
    return found >= want;
}

__global__ void set_tables_kernel(PageView c, BooksWork w, const int32_t* table, const int32_t* length,
                                  const int32_t* refs) {
    stream_turn();
    if (blockIdx.x == 0 && threadIdx.x == 0) *w.lowest = 0;
    const int64_t nt = (int64_t)c.n_seq * c.max_pages, all = nt + c.n_seq + c.n_page;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        if (i < nt)
            c.table[i] = table[i];
        else if (i < nt + c.n_seq)
            c.length[i - nt] = length[i - nt];
        else
            c.refs[i - nt - c.n_seq] = refs[i - nt - c.n_seq];
    }
}

// Every sequence of the list inside [0, n_seq) and listed once? mark[s] ends as the
// number of one entry that names s; an entry that is not that one is a second.
__device__ bool distinct_seqs(const PageView& c, const int32_t* seqs, int n, int32_t* mark) {
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = seqs[i];
        if (s < 0 || s >= c.n_seq)
            bad = true;
        else
            mark[s] = i;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = seqs[i];
        if (s >= 0 && s < c.n_seq && mark[s] != i) bad = true;
    }
    return !__syncthreads_or(bad);
}

// Entry i's need of pages into first[i] as its place in the list of taken pages;
// returns the whole need, saturated at n_page + 1 (more than there are).
template <typename F>
__device__ int place_needs(int n, int n_page, int32_t* first, F need) {
    int total = 0;
    for (int base = 0; base < n; base += (int)blockDim.x) {
        const int i = base + (int)threadIdx.x;
        const int v = i < n ? need(i) : 0;
        int sum;
        const int at = total + block_scan(v, &sum);
        if (i < n) first[i] = at;
        total += sum;  // each need is at most max_pages; the host bounds n * max_pages by 2^30
    }
    __syncthreads();
    return min(total, n_page + 1);
}

__global__ void __launch_bounds__(kBooksThreads) extend_kernel(PageView c, BooksWork w, const int32_t* seqs,
                                                               const int32_t* counts, int n) {
    stream_turn();
    const int P = 1 << c.page_shift;
    if (!distinct_seqs(c, seqs, n, w.mark)) {
        if (threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_BAD_SEQ);
        return;
    }
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int len = pages_length(c, seqs[i]);
        w.len[i] = len;
        if (counts[i] < 0 || (int64_t)len + counts[i] > ((int64_t)c.max_pages << c.page_shift)) bad = true;
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_ROW_FULL);
        return;
    }
    const auto pages = [&](int len) { return (int)(((int64_t)len + P - 1) >> c.page_shift); };
    const int want = place_needs(n, c.n_page, w.first,
                                 [&](int i) { return pages(w.len[i] + counts[i]) - pages(w.len[i]); });
    if (!lowest_free(c, w, want)) {
        if (threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_NO_PAGES);
        return;
    }
    if (threadIdx.x == 0 && want > 0) *w.lowest = w.list[want - 1] + 1;
    for (int i = threadIdx.x; i < want; i += blockDim.x) c.refs[w.list[i]] = 1;
    // a warp per entry
    for (int i = (int)threadIdx.x >> 5; i < n; i += (int)blockDim.x >> 5) {
        const int s = seqs[i], len = w.len[i], have = pages(len), need = pages(len + counts[i]) - have;
        int32_t* row = c.table + (int64_t)s * c.max_pages + have;
        for (int j = threadIdx.x & 31; j < need; j += 32) row[j] = w.list[w.first[i] + j];
        if ((threadIdx.x & 31) == 0) c.length[s] = len + counts[i];
    }
}

// Also writes the copies of partly filled last pages as jobs for move_kernel.
__global__ void __launch_bounds__(kBooksThreads) fork_kernel(PageView c, BooksWork w,
                                                             const int32_t* parents,
                                                             const int32_t* children, int n) {
    stream_turn();
    const int P = 1 << c.page_shift;
    if (threadIdx.x == 0) *w.n_jobs = 0;
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) bad |= parents[i] < 0 || parents[i] >= c.n_seq;
    if (!distinct_seqs(c, children, n, w.mark) || __syncthreads_or(bad)) {
        if (threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_BAD_SEQ);
        return;
    }
    bad = false;
    bool torn = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int len = pages_length(c, parents[i]);
        w.len[i] = len;
        bad |= c.length[children[i]] != 0;
    }
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_NOT_EMPTY);
        return;
    }
    // the parents' pages, before anything is changed
    for (int i = (int)threadIdx.x >> 5; i < n; i += (int)blockDim.x >> 5) {
        const int held = (int)(((int64_t)w.len[i] + P - 1) >> c.page_shift);
        const int32_t* row = c.table + (int64_t)parents[i] * c.max_pages;
        for (int j = threadIdx.x & 31; j < held; j += 32) torn |= (uint32_t)row[j] >= (uint32_t)c.n_page;
    }
    if (__syncthreads_or(torn)) {
        if (threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_BAD_PAGE);
        return;
    }
    const int want = place_needs(n, c.n_page, w.first, [&](int i) { return (w.len[i] & (P - 1)) != 0; });
    if (!lowest_free(c, w, want)) {
        if (threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_NO_PAGES);
        return;
    }
    if (threadIdx.x == 0 && want > 0) *w.lowest = w.list[want - 1] + 1;
    if (threadIdx.x == 0) *w.n_jobs = want;
    for (int i = (int)threadIdx.x >> 5; i < n; i += (int)blockDim.x >> 5) {
        const int len = w.len[i], full = len >> c.page_shift, part = len & (P - 1), lane = (int)threadIdx.x & 31;
        const int32_t* from = c.table + (int64_t)parents[i] * c.max_pages;
        int32_t* row = c.table + (int64_t)children[i] * c.max_pages;
        for (int j = lane; j < full; j += 32) {
            const int p = from[j];
            row[j] = p;
            atomicAdd(c.refs + p, 1);  // a sum of ones: the same in any order
        }
        if (lane == 0) {
            c.length[children[i]] = len;
            if (part) {
                const int p = w.list[w.first[i]];
                row[full] = p;
                c.refs[p] = 1;
                w.jobs[w.first[i]] = PageJob{from[full], p, part};
            }
        }
    }
}

// The list of a free, for lists longer than a CTA of free_kernel can look over by itself.
__global__ void __launch_bounds__(kBooksThreads) free_check_kernel(PageView c, BooksWork w, const int32_t* seqs, int n) {
    stream_turn();
    const bool good = distinct_seqs(c, seqs, n, w.mark);
    if (threadIdx.x == 0) *w.n_jobs = good;
    if (!good && threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_BAD_SEQ);
}

constexpr int kFreeThreads = 256;  // and the longest list that free_kernel checks itself

// A CTA per listed sequence. Each looks over the whole list first (`checked`: free_check_kernel has), so
// that a list with a fault in it changes nothing.
__global__ void __launch_bounds__(kFreeThreads) free_kernel(PageView c, BooksWork w, const int32_t* seqs, int n, int checked) {
    stream_turn();
    __shared__ int held;
    __shared__ int list[kFreeThreads];
    const int P = 1 << c.page_shift;
    if (checked) {
        if (!*w.n_jobs) return;
    } else {
        const int i = (int)threadIdx.x, mine = i < n ? seqs[i] : 0;
        list[i] = mine;
        __syncthreads();
        bool bad = i < n && (mine < 0 || mine >= c.n_seq);
        for (int j = 0; j < n; ++j) bad |= j < i && i < n && list[j] == mine;
        if (__syncthreads_or(bad)) {
            if (blockIdx.x == 0 && threadIdx.x == 0) pages_flag(c, AERO_CUDA_PAGES_BAD_SEQ);
            return;
        }
    }
    const int s = seqs[blockIdx.x];
    if (threadIdx.x == 0) {
        const int64_t len = max(0, c.length[s]);
        c.length[s] = 0;
        held = (int)min((int64_t)c.max_pages, (len + P - 1) >> c.page_shift);
    }
    __syncthreads();
    int32_t* row = c.table + (int64_t)s * c.max_pages;
    for (int i = threadIdx.x; i < held; i += blockDim.x) {
        const int p = row[i];
        row[i] = -1;
        if (p < 0 || p >= c.n_page) {
            pages_flag(c, AERO_CUDA_PAGES_BAD_PAGE);
        } else {
            const int had = atomicSub(c.refs + p, 1);
            if (had <= 0) {  // the books did not hold it
                atomicAdd(c.refs + p, 1);
                pages_flag(c, AERO_CUDA_PAGES_BAD_PAGE);
            } else if (had == 1) {
                atomicMin(w.lowest, p);
            }
        }
    }
}

// Which live pages move into which free ones: with L live pages, the i-th free page
// below L takes the i-th live page at or above L (there are equally many). Sources lie
// at or above L and targets below, so the moves do not touch one another.
__global__ void __launch_bounds__(kBooksThreads) compact_kernel(PageView c, BooksWork w) {
    stream_turn();
    int live = 0;
    for (int base = 0; base < c.n_page; base += 4 * (int)blockDim.x) {
        const int p0 = base + 4 * (int)threadIdx.x;
        const int4 r = refs4(c, p0);
        live += p0 < c.n_page ? (r.x != 0) + (p0 + 1 < c.n_page && r.y != 0) + (p0 + 2 < c.n_page && r.z != 0) +
                                    (p0 + 3 < c.n_page && r.w != 0)
                              : 0;
    }
    int L;
    block_scan(live, &L);
    int holes = 0, movers = 0;
    for (int base = 0; base < c.n_page; base += 4 * (int)blockDim.x) {
        const int p0 = base + 4 * (int)threadIdx.x;
        const int4 r = refs4(c, p0);
        const int rr[4] = {r.x, r.y, r.z, r.w};
        // a page below L can only be a hole, one from L on only a mover
        int nh = 0, nm = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            nh += p0 + i < L && rr[i] == 0;
            nm += p0 + i >= L && p0 + i < c.n_page && rr[i] != 0;
        }
        // the low half of the sum counts holes, the high half movers: a step sees at most 4096 pages
        int sum;
        const int at = block_scan(nh + (nm << 16), &sum);
        int h = holes + (at & 0xFFFF), m = movers + (at >> 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = p0 + i;
            if (p < L && rr[i] == 0) w.jobs[h++].dst = p;
            if (p >= L && p < c.n_page && rr[i] != 0) w.list[m++] = p;
        }
        holes += sum & 0xFFFF;
        movers += sum >> 16;
    }
    __syncthreads();
    const int n = min(holes, movers);
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int from = w.list[i], to = w.jobs[i].dst;
        w.jobs[i].src = from;
        w.jobs[i].rows = 1 << c.page_shift;
        w.to[from] = to;
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    if (threadIdx.x == 0) {
        *w.n_jobs = n;
        *w.n_live = L;
        *w.lowest = L;
    }
}

__global__ void copy_jobs_kernel(PageView c, BooksWork w, const int32_t* src,
                                 const int32_t* dst, int n) {
    stream_turn();
    const int i = (int)(blockIdx.x * blockDim.x + threadIdx.x);
    if (i == 0) *w.n_jobs = n;
    if (i >= n) return;
    PageJob j{src[i], dst[i], 1 << c.page_shift};
    if ((uint32_t)j.src >= (uint32_t)c.n_page || (uint32_t)j.dst >= (uint32_t)c.n_page) {
        pages_flag(c, AERO_CUDA_PAGES_BAD_PAGE);
        j = PageJob{0, 0, 0};
    }
    w.jobs[i] = j;
}

constexpr int kMoveVec = 4;  // 16-byte pieces a thread moves per unit, all loaded before the first is stored
constexpr int kMoveUnit = 256 * kMoveVec;

// The jobs' rows, in every layer and kv head of K and V: a page of a layer is HK * P * D
// contiguous values; a unit is 16 KB of one. With `retable`, the table's entries
// from n_live on follow their pages.
__global__ void __launch_bounds__(256) move_kernel(PageView c, BooksWork w, uint4* k, uint4* v,
                                                   int retable) {
    stream_turn();
    const int P = 1 << c.page_shift, row_vec = c.D / 8;
    const int page_vec = c.HK * P * row_vec;
    const int pieces = (page_vec + kMoveUnit - 1) / kMoveUnit;
    if (retable) {
        const int L = *w.n_live;
        const int64_t nt = (int64_t)c.n_seq * c.max_pages;
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < nt; i += (int64_t)gridDim.x * blockDim.x) {
            const int p = c.table[i];
            // a live page from L on was moved; a number that is no page stays
            if (p >= L && p < c.n_page) c.table[i] = w.to[p];
        }
    }
    const int64_t per_job = (int64_t)c.n_layer * 2 * pieces;
    const int64_t units = (int64_t)*w.n_jobs * per_job;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const PageJob j = w.jobs[u / per_job];
        const int r = (int)(u % per_job);  // n_layer * 2 * pieces fits: the host checks
        const int layer = r / (2 * pieces), kv = (r / pieces) & 1, piece = r % pieces;
        uint4* pool = kv ? v : k;
        const uint4* s = pool + ((int64_t)layer * c.n_page + j.src) * page_vec;
        uint4* d = pool + ((int64_t)layer * c.n_page + j.dst) * page_vec;
        uint4 x[kMoveVec];
        bool on[kMoveVec];
#pragma unroll
        for (int i = 0; i < kMoveVec; ++i) {
            const int at = piece * kMoveUnit + i * 256 + (int)threadIdx.x;
            on[i] = at < page_vec && ((at / row_vec) & (P - 1)) < j.rows;
            if (on[i]) x[i] = __ldcs(s + at);
        }
#pragma unroll
        for (int i = 0; i < kMoveVec; ++i)
            if (on[i]) __stcs(d + piece * kMoveUnit + i * 256 + (int)threadIdx.x, x[i]);
    }
}

// K and V rows of T tokens. VEC: 16 bytes a thread, else one value (rows that do not
// start on 16 bytes).
template <typename E>
__global__ void __launch_bounds__(256) append_kernel(PageView c, int layer, const E* k, int64_t k_token,
                                                     int64_t k_head, const E* v, int64_t v_token,
                                                     int64_t v_head, const int32_t* seqs,
                                                     const int32_t* positions, int T, E* kp,
                                                     E* vp) {
    stream_turn();
    // E counts in pieces of the row: strides and D come in those
    constexpr int PER = sizeof(E) / 2;
    const int rowp = c.D / PER;
    const int64_t all = (int64_t)T * c.HK * rowp;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        const int d = (int)(i % rowp);
        const int64_t th = i / rowp;
        const int h = (int)(th % c.HK);
        const int64_t t = th / c.HK;
        // (the rows on their way while the page is looked for)
        const E x = __ldcs(k + t * k_token + h * k_head + d), y = __ldcs(v + t * v_token + h * v_head + d);
        const int s = seqs[t], p = positions[t];
        if (s < 0 || s >= c.n_seq) {
            pages_flag(c, AERO_CUDA_PAGES_BAD_SEQ);
            continue;
        }
        const int held = pages_length(c, s);
        const int page = p >= 0 && p >> c.page_shift < c.max_pages ? c.table[(int64_t)s * c.max_pages + (p >> c.page_shift)] : -1;
        if (p >= held || (uint32_t)page >= (uint32_t)c.n_page) {
            pages_flag(c, AERO_CUDA_PAGES_BAD_PAGE);
            continue;
        }
        if (c.refs[page] > 1) {  // another sequence reads it
            pages_flag(c, AERO_CUDA_PAGES_SHARED);
            continue;
        }
        const int64_t row = ((((int64_t)layer * c.n_page + page) * c.HK + h) << c.page_shift) + (p & ((1 << c.page_shift) - 1));
        kp[row * rowp + d] = x;
        vp[row * rowp + d] = y;
    }
}

// ------------------------------------------------------------------ host side
struct Pages {
    aero_cuda_pages_desc d{};
    cudaStream_t stream = nullptr, own_stream = nullptr;
    cudaEvent_t moved = nullptr;
    int n_sm = 148;
    PageView view{};
    BooksWork work{};
    void *k = nullptr, *v = nullptr, *books = nullptr;  // v: behind k, in one allocation
    size_t pool_bytes = 0, books_bytes = 0;
    float *decode_part = nullptr, *prompt_part = nullptr;
    uint32_t *decode_count = nullptr, *prompt_count = nullptr;
    CUtensorMap kmap{}, vmap{};
    std::string err;

    bool fail(const char* fmt, ...) {
        char buf[512];
        va_list ap;
        va_start(ap, fmt);
        std::vsnprintf(buf, sizeof(buf), fmt, ap);
        va_end(ap);
        err = buf;
        return false;
    }
    bool ok(cudaError_t e, const char* what) {
        if (e == cudaSuccess) return true;
        cudaGetLastError();
        return fail("%s: %s", what, cudaGetErrorString(e));
    }
    ~Pages() {
        if (stream) cudaStreamSynchronize(stream);
        if (k) guarded_free(k, pool_bytes, kKVCache);
        if (books) guarded_free(books, books_bytes, kScratch);
        if (moved) cudaEventDestroy(moved);
        if (own_stream) cudaStreamDestroy(own_stream);
    }
};

int log2_exact(int v) {
    int s = 0;
    while ((1 << s) < v) ++s;
    return (1 << s) == v ? s : -1;
}

const char* bad_desc(const aero_cuda_pages_desc& d) {
    if (d.n_layer <= 0 || d.n_page <= 0 || d.n_head_kv <= 0 || d.n_seq <= 0 || d.max_pages <= 0)
        return "n_layer, n_page, n_head_kv, n_seq and max_pages must be positive";
    if (d.page_size < 8 || d.page_size > 256 || log2_exact(d.page_size) < 0)
        return "page_size must be a power of two from 8 to 256";
    if (d.head_dim != 64 && d.head_dim != 128 && d.head_dim != 192 && d.head_dim != 256)
        return "head_dim must be 64, 128, 192 or 256";
    if (d.dtype != AERO_CUDA_TYPE_F16 && d.dtype != AERO_CUDA_TYPE_BF16)
        return "dtype must be AERO_CUDA_TYPE_F16 or AERO_CUDA_TYPE_BF16";
    if (d.n_head_kv > 1024 || d.n_layer > 4096) return "at most 1024 kv heads and 4096 layers";
    // rows of the pool are numbered in 31 bits (TMA coordinates); so are positions of a sequence
    if ((double)d.n_layer * d.n_page * d.n_head_kv * d.page_size >= 2147483648.0)
        return "the pool has 2^31 rows or more: n_layer * n_page * n_head_kv * page_size";
    if ((double)d.n_seq * d.max_pages > 1073741824.0 || (double)d.max_pages * d.page_size > 1073741824.0)
        return "n_seq * max_pages and max_pages * page_size must be at most 2^30";
    return nullptr;
}

struct Layout {
    size_t pool, books;                                                        // bytes of K (or V); of the books block
    size_t table, length, refs, status, list, to, mark, first, len, jobs, counts;  // offsets in the books block
    size_t dpart, dcount, ppart, pcount;
};

Layout layout(const aero_cuda_pages_desc& d, int n_sm) {
    Layout l{};
    l.pool = (size_t)d.n_layer * d.n_page * d.n_head_kv * d.page_size * d.head_dim * 2;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t o = at;
        at += (bytes + 255) & ~(size_t)255;
        return o;
    };
    l.table = take((size_t)d.n_seq * d.max_pages * 4);
    l.length = take((size_t)d.n_seq * 4);
    l.refs = take((size_t)d.n_page * 4);
    l.status = take(4);
    l.list = take((size_t)d.n_page * 4);
    l.to = take((size_t)d.n_page * 4);
    l.mark = take((size_t)d.n_seq * 4);
    l.first = take((size_t)d.n_seq * 4);
    l.len = take((size_t)d.n_seq * 4);
    l.jobs = take((size_t)std::max(d.n_page, d.n_seq) * sizeof(PageJob));
    l.counts = take(12);
    l.dpart = take(pages_decode_part_floats(d.head_dim, n_sm) * 4);
    l.dcount = take((size_t)pages_decode_max_grid(n_sm) * 4);
    l.ppart = take(pages_prompt_part_floats(d.head_dim, n_sm) * 4);
    l.pcount = take((size_t)pages_prompt_max_grid(n_sm) * 4);
    l.books = at;
    return l;
}

Pages* open_pages(const aero_cuda_pages_desc* desc, std::string* why) {
    if (!desc) return *why = "null description", nullptr;
    if (const char* b = bad_desc(*desc)) return *why = b, nullptr;
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count <= 0) {
        cudaGetLastError();
        return *why = "no CUDA device", nullptr;
    }
    if (desc->device < 0 || desc->device >= count) return *why = "no such CUDA device", nullptr;
    OnDevice on(desc->device);
    if (!on.good) return *why = "cudaSetDevice failed", nullptr;
    Pages* g = new (std::nothrow) Pages;
    if (!g) return *why = "out of host memory", nullptr;
    g->d = *desc;
    cudaDeviceGetAttribute(&g->n_sm, cudaDevAttrMultiProcessorCount, desc->device);
    const Layout l = layout(*desc, g->n_sm);
    const auto refuse = [&](const char* what) -> Pages* {
        cudaGetLastError();
        *why = what;
        delete g;
        return nullptr;
    };
    if (guarded_malloc(&g->k, 2 * l.pool, kKVCache) != cudaSuccess)
        return refuse("device allocation for the pages refused (memory guard budget or device memory)");
    g->pool_bytes = 2 * l.pool;
    g->v = static_cast<char*>(g->k) + l.pool;  // (l.pool is a multiple of a page's kv head, 1 KB or more)
    if (guarded_malloc(&g->books, l.books, kScratch) != cudaSuccess) return refuse("device allocation for the books refused (memory guard budget or device memory)");
    g->books_bytes = l.books;
    if (cudaStreamCreate(&g->own_stream) != cudaSuccess ||
        cudaEventCreateWithFlags(&g->moved, cudaEventDisableTiming) != cudaSuccess)
        return refuse("stream or event creation failed");
    g->stream = g->own_stream;
    char* b = static_cast<char*>(g->books);
    PageView& c = g->view;
    c.table = reinterpret_cast<int32_t*>(b + l.table);
    c.length = reinterpret_cast<int32_t*>(b + l.length);
    c.refs = reinterpret_cast<int32_t*>(b + l.refs);
    c.status = reinterpret_cast<int32_t*>(b + l.status);
    c.n_page = desc->n_page;
    c.page_shift = log2_exact(desc->page_size);
    c.HK = desc->n_head_kv;
    c.D = desc->head_dim;
    c.n_seq = desc->n_seq;
    c.max_pages = desc->max_pages;
    c.n_layer = desc->n_layer;
    BooksWork& w = g->work;
    w.list = reinterpret_cast<int32_t*>(b + l.list);
    w.to = reinterpret_cast<int32_t*>(b + l.to);
    w.mark = reinterpret_cast<int32_t*>(b + l.mark);
    w.first = reinterpret_cast<int32_t*>(b + l.first);
    w.len = reinterpret_cast<int32_t*>(b + l.len);
    w.jobs = reinterpret_cast<PageJob*>(b + l.jobs);
    w.n_jobs = reinterpret_cast<int32_t*>(b + l.counts);
    w.n_live = w.n_jobs + 1;
    w.lowest = w.n_jobs + 2;  // (zero at first: the books block is cleared)
    g->decode_part = reinterpret_cast<float*>(b + l.dpart);
    g->decode_count = reinterpret_cast<uint32_t*>(b + l.dcount);
    g->prompt_part = reinterpret_cast<float*>(b + l.ppart);
    g->prompt_count = reinterpret_cast<uint32_t*>(b + l.pcount);
    if (cudaMemsetAsync(g->k, 0, 2 * l.pool, g->stream) != cudaSuccess ||
        cudaMemsetAsync(g->books, 0, l.books, g->stream) != cudaSuccess ||
        cudaMemsetAsync(c.table, 0xFF, (size_t)desc->n_seq * desc->max_pages * 4, g->stream) != cudaSuccess ||
        cudaStreamSynchronize(g->stream) != cudaSuccess)
        return refuse("clearing the pool failed");
    const uint64_t rows = (uint64_t)desc->n_layer * desc->n_page * desc->n_head_kv * desc->page_size;
    const uint32_t box = (uint32_t)std::min(desc->page_size, 64);
    const CUtensorMapDataType dt =
        desc->dtype == AERO_CUDA_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (!encode_tmap_2d(&g->kmap, dt, 2, g->k, rows, (uint64_t)desc->head_dim, (uint64_t)desc->head_dim, box, 64,
                        CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_2d(&g->vmap, dt, 2, g->v, rows, (uint64_t)desc->head_dim, (uint64_t)desc->head_dim, box, 64,
                        CU_TENSOR_MAP_SWIZZLE_128B))
        return refuse("cuTensorMapEncodeTiled failed for the pool");
    return g;
}

// Runs f on the handle's device; C++ exceptions end here.
template <typename F>
int entry(void* cache, F f) {
    auto* g = static_cast<Pages*>(cache);
    if (!g) return -1;
    try {
        OnDevice on(g->d.device);
        if (!on.good) return g->fail("cudaSetDevice(%d) failed", g->d.device), -1;
        return f(*g) ? 0 : -1;
    } catch (...) {
        return -1;
    }
}

bool device_i32(Pages& g, const void* p, const char* what) {
    if (!is_device_ptr(p)) return g.fail("%s must be device memory", what);
    if ((uintptr_t)p & 3) return g.fail("%s is not aligned to 4 bytes", what);
    return true;
}

bool listed(Pages& g, const void* a, const char* an, const void* b, const char* bn, int n) {
    if (n < 0 || n > g.d.n_seq) return g.fail("n must be from 0 to n_seq = %d, got %d", g.d.n_seq, n);
    return n == 0 || (device_i32(g, a, an) && (!b || device_i32(g, b, bn)));
}

cudaError_t launch_move(Pages& g, int64_t max_jobs, int retable) {
    const PageView& c = g.view;
    const int64_t page_vec = (int64_t)c.HK * (c.D / 8) << c.page_shift;
    const int64_t units = max_jobs * c.n_layer * 2 * ((page_vec + kMoveUnit - 1) / kMoveUnit);
    const int64_t books = retable ? ((int64_t)c.n_seq * c.max_pages + 255) / 256 : 0;
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(std::max(units, books), (int64_t)g.n_sm * 8));
    return launch_in_turn(move_kernel, grid, 256, 0, g.stream, c, g.work, static_cast<uint4*>(g.k), static_cast<uint4*>(g.v),
                          retable);
}

bool layer_ok(Pages& g, int layer) {
    return (layer >= 0 && layer < g.d.n_layer) || g.fail("layer %d outside [0, %d)", layer, g.d.n_layer);
}

// A row of q, k, v or out may be read 16 bytes at a time.
bool vec16(const void* p, int64_t token, int64_t head) {
    return ((uintptr_t)p & 15) == 0 && token % 8 == 0 && head % 8 == 0;
}

}  // namespace
}  // namespace aero

using aero::Pages;

extern "C" {

void* aero_cuda_pages_open(const aero_cuda_pages_desc* desc, char* err, int errlen) {
    try {
        std::string why;
        Pages* g = aero::open_pages(desc, &why);
        if (!g && err && errlen > 0) std::snprintf(err, (size_t)errlen, "%s", why.c_str());
        return g;
    } catch (...) {
        if (err && errlen > 0) std::snprintf(err, (size_t)errlen, "out of host memory");
        return nullptr;
    }
}

int64_t aero_cuda_pages_plan_bytes(const aero_cuda_pages_desc* desc, int64_t* by_class) {
    if (!desc || aero::bad_desc(*desc)) return -1;
    int n_sm = 148;  // B200, where no device tells
    int count = 0;
    if (cudaGetDeviceCount(&count) == cudaSuccess && desc->device >= 0 && desc->device < count)
        cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, desc->device);
    else
        cudaGetLastError();
    const aero::Layout l = aero::layout(*desc, n_sm);
    if (by_class) {
        by_class[0] = (int64_t)(2 * l.pool);
        by_class[1] = (int64_t)l.books;
    }
    return (int64_t)(2 * l.pool + l.books);
}

void aero_cuda_pages_close(void* cache) {
    auto* g = static_cast<Pages*>(cache);
    if (!g) return;
    aero::OnDevice on(g->d.device);
    delete g;
}

int aero_cuda_pages_set_stream(void* cache, void* stream) {
    return aero::entry(cache, [&](Pages& g) {
        const cudaStream_t to = stream ? static_cast<cudaStream_t>(stream) : g.own_stream;
        if (to == g.stream) return true;
        // a captured stream cannot wait for work outside its graph, nor other work for it: who
        // captures has waited for what went before
        cudaStreamCaptureStatus was = cudaStreamCaptureStatusNone, is = cudaStreamCaptureStatusNone;
        const cudaError_t e0 = cudaStreamIsCapturing(g.stream, &was), e1 = cudaStreamIsCapturing(to, &is);
        if (e0 != cudaSuccess || e1 != cudaSuccess) cudaGetLastError();
        if ((e0 == cudaSuccess && was != cudaStreamCaptureStatusNone) || (e1 == cudaSuccess && is != cudaStreamCaptureStatusNone)) {
            g.stream = to;
            return true;
        }
        // (the legacy default stream cannot be asked while a blocking stream is captured: that is no
        // matter where the other of the two is the one, and an error where it is neither)
        if (!g.ok(e0, "set_stream") || !g.ok(e1, "set_stream")) return false;
        if (!g.ok(cudaEventRecord(g.moved, g.stream), "set_stream") ||
            !g.ok(cudaStreamWaitEvent(to, g.moved, 0), "set_stream"))
            return false;
        g.stream = to;
        return true;
    });
}

int aero_cuda_pages_buffers(void* cache, void** k, void** v, int32_t** table, int32_t** length, int32_t** refs) {
    auto* g = static_cast<Pages*>(cache);
    if (!g) return -1;
    if (k) *k = g->k;
    if (v) *v = g->v;
    if (table) *table = g->view.table;
    if (length) *length = g->view.length;
    if (refs) *refs = g->view.refs;
    return 0;
}

int aero_cuda_pages_status(void* cache) {
    int32_t code = -1;
    const int rc = aero::entry(cache, [&](Pages& g) {
        return g.ok(cudaMemcpyAsync(&code, g.view.status, 4, cudaMemcpyDeviceToHost, g.stream), "status") &&
               g.ok(cudaMemsetAsync(g.view.status, 0, 4, g.stream), "status") &&
               g.ok(cudaStreamSynchronize(g.stream), "status");
    });
    return rc == 0 ? code : -1;
}

const char* aero_cuda_pages_last_error(void* cache) {
    auto* g = static_cast<Pages*>(cache);
    return g ? g->err.c_str() : "null cache";
}

int aero_cuda_pages_set_tables(void* cache, const int32_t* table, const int32_t* length, const int32_t* refs) {
    return aero::entry(cache, [&](Pages& g) {
        if (!aero::device_i32(g, table, "table") || !aero::device_i32(g, length, "length") ||
            !aero::device_i32(g, refs, "refs"))
            return false;
        const int64_t all = (int64_t)g.d.n_seq * g.d.max_pages + g.d.n_seq + g.d.n_page;
        const unsigned grid = (unsigned)std::min<int64_t>((all + 255) / 256, (int64_t)g.n_sm * 8);
        return g.ok(aero::launch_in_turn(aero::set_tables_kernel, grid, 256, 0, g.stream, g.view, g.work, table, length, refs), "set_tables");
    });
}

int aero_cuda_pages_extend(void* cache, const int32_t* seqs, const int32_t* counts, int n) {
    return aero::entry(cache, [&](Pages& g) {
        if (!aero::listed(g, seqs, "seqs", counts, "counts", n)) return false;
        if (n > 0 && !counts) return g.fail("counts is required");
        if (n == 0) return true;
        return g.ok(aero::launch_in_turn(aero::extend_kernel, 1, aero::kBooksThreads, 0, g.stream, g.view, g.work, seqs, counts, n),
                    "extend");
    });
}

int aero_cuda_pages_append(void* cache, int layer, const void* k, int64_t k_token, int64_t k_head, const void* v,
                           int64_t v_token, int64_t v_head, const int32_t* seqs, const int32_t* positions, int T) {
    return aero::entry(cache, [&](Pages& g) {
        if (!aero::layer_ok(g, layer)) return false;
        if (T < 0) return g.fail("T must be >= 0, got %d", T);
        if (T == 0) return true;
        if (!aero::is_device_ptr(k) || !aero::is_device_ptr(v)) return g.fail("k and v must be device memory");
        if (((uintptr_t)k | (uintptr_t)v) & 1) return g.fail("k and v must be aligned to their type");
        if (!aero::device_i32(g, seqs, "seqs") || !aero::device_i32(g, positions, "positions")) return false;
        const bool vec = aero::vec16(k, k_token, k_head) && aero::vec16(v, v_token, v_head);
        const int per = vec ? 8 : 1;
        const int64_t all = (int64_t)T * g.d.n_head_kv * (g.d.head_dim / per);
        const unsigned grid = (unsigned)std::min<int64_t>((all + 255) / 256, (int64_t)g.n_sm * 16);
        const auto launch = [&](auto piece) {
            using E = decltype(piece);
            return aero::launch_in_turn(aero::append_kernel<E>, grid, 256, 0, g.stream, g.view, layer, static_cast<const E*>(k),
                                        k_token / per, k_head / per, static_cast<const E*>(v), v_token / per, v_head / per,
                                        seqs, positions, T, static_cast<E*>(g.k), static_cast<E*>(g.v));
        };
        return g.ok(vec ? launch(uint4{}) : launch(uint16_t{}), "append");
    });
}

int aero_cuda_pages_fork(void* cache, const int32_t* parents, const int32_t* children, int n) {
    return aero::entry(cache, [&](Pages& g) {
        if (!aero::listed(g, parents, "parents", children, "children", n)) return false;
        if (n > 0 && !children) return g.fail("children is required");
        if (n == 0) return true;
        return g.ok(aero::launch_in_turn(aero::fork_kernel, 1, aero::kBooksThreads, 0, g.stream, g.view, g.work, parents, children, n),
                    "fork") &&
               g.ok(aero::launch_move(g, n, 0), "fork");
    });
}

int aero_cuda_pages_free(void* cache, const int32_t* seqs, int n) {
    return aero::entry(cache, [&](Pages& g) {
        if (!aero::listed(g, seqs, "seqs", nullptr, "", n)) return false;
        if (n == 0) return true;
        const int checked = n > aero::kFreeThreads;
        return (!checked || g.ok(aero::launch_in_turn(aero::free_check_kernel, 1, aero::kBooksThreads, 0, g.stream, g.view, g.work, seqs, n), "free")) &&
               g.ok(aero::launch_in_turn(aero::free_kernel, (unsigned)n, aero::kFreeThreads, 0, g.stream, g.view, g.work, seqs, n, checked), "free");
    });
}

int aero_cuda_pages_copy(void* cache, const int32_t* src, const int32_t* dst, int n) {
    return aero::entry(cache, [&](Pages& g) {
        if (n < 0 || n > g.d.n_page) return g.fail("n must be from 0 to n_page = %d, got %d", g.d.n_page, n);
        if (n == 0) return true;
        if (!aero::device_i32(g, src, "src") || !aero::device_i32(g, dst, "dst")) return false;
        return g.ok(aero::launch_in_turn(aero::copy_jobs_kernel, (unsigned)(n + 255) / 256, 256, 0, g.stream, g.view, g.work, src, dst, n),
                    "copy") &&
               g.ok(aero::launch_move(g, n, 0), "copy");
    });
}

int aero_cuda_pages_compact(void* cache) {
    return aero::entry(cache, [&](Pages& g) {
        return g.ok(aero::launch_in_turn(aero::compact_kernel, 1, aero::kBooksThreads, 0, g.stream, g.view, g.work), "compact") &&
               g.ok(aero::launch_move(g, (g.d.n_page + 1) / 2, 1), "compact");
    });
}

int aero_cuda_pages_attend(void* cache, int layer, const void* q, int64_t q_token, int64_t q_head, int T, int n_head,
                           const int32_t* seqs, const int32_t* q_start, int n, float scale, int window, int sinks,
                           void* out, int64_t o_token, int64_t o_head) {
    return aero::entry(cache, [&](Pages& g) {
        if (!aero::layer_ok(g, layer)) return false;
        const int HK = g.d.n_head_kv;
        if (n_head <= 0 || n_head % HK || n_head / HK > 16)
            return g.fail("n_head must be a multiple of n_head_kv = %d, at most 16 times it; got %d", HK, n_head);
        if (T < 0 || n < 0 || T > (1 << 24) || n > (1 << 20)) return g.fail("T must be from 0 to 2^24, n from 0 to 2^20");
        if (!q_start && T != n) return g.fail("without q_start T must be n, one token per sequence (T %d, n %d)", T, n);
        if (q_start && T > 0 && n == 0) return g.fail("%d tokens of no sequence", T);
        if (window < 0 || sinks < 0) return g.fail("window and sinks must be >= 0");
        if (!(scale > 0.f) || !(scale < 1e30f)) return g.fail("scale must be positive and finite");
        if (T == 0) return true;
        if (!aero::is_device_ptr(q) || !aero::is_device_ptr(out)) return g.fail("q and out must be device memory");
        if (((uintptr_t)q | (uintptr_t)out) & 1) return g.fail("q and out must be aligned to their type");
        if (!aero::device_i32(g, seqs, "seqs") || (q_start && !aero::device_i32(g, q_start, "q_start"))) return false;
        aero::AttendArgs a{};
        a.c = g.view;
        a.q = q;
        a.q_token = q_token;
        a.q_head = q_head;
        a.out = out;
        a.o_token = o_token;
        a.o_head = o_head;
        a.seqs = seqs;
        a.q_start = q_start;
        a.layer = layer;
        a.T = T;
        a.n = n;
        a.H = n_head;
        a.window = window;
        a.sinks = window ? sinks : 0;
        a.scale_log2 = scale * 1.4426950408889634f;
        a.vec = aero::vec16(q, q_token, q_head) && aero::vec16(out, o_token, o_head);
        const bool bf16 = g.d.dtype == AERO_CUDA_TYPE_BF16;
        // Few tokens, or hardly more than one a sequence, go token by token: a tile of 128 rows
        // would be mostly empty, and its CTA costs some 12 us before it is done (B200, 4 x 8 heads of
        // 128, tokens against tiles: 8 tokens over 1000 positions 12 / 15 us, 16 over 4096 22 / 25, 32 of
        // 16 sequences over 2000 23 / 26, 64 of 64 over 2000 53 / 79; but 64 of one over 4096 48 / 38, 128
        // of 64 over 2000 91 / 80). The lengths, which the host does not know, would move the line: each
        // token reads its sequence again (8 of one over 32768 47 / 43, 32 of one 148 / 71, 32 of 8 over 8000
        // 51 / 44), and a batch of one prompt and many single tokens is not divided.
        const bool by_token = !q_start || T <= 32 || T < 2 * (int64_t)n;
        if (!by_token) {
            a.part = g.prompt_part;
            a.counters = g.prompt_count;
            return g.ok(aero::launch_pages_prompt(a, bf16, g.kmap, g.vmap, g.k, g.v, g.n_sm, g.stream), "attend");
        }
        a.part = g.decode_part;
        a.counters = g.decode_count;
        return g.ok(aero::launch_pages_decode(a, bf16, g.kmap, g.vmap, g.n_sm, g.stream), "attend");
    });
}

}  // extern "C"
