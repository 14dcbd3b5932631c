// The paged key/value cache (include/aero_cuda_pages.h): what its translation
// units share. pages.cu owns the handle and the books, pages_decode.cu the
// attention of single tokens, over all positions or over listed blocks, pages_prompt.cu that of
// several tokens a sequence, pages_select.cu the bounds of pages and the choice of blocks.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/aero_cuda_pages.h"

namespace aero {

// The caller's current device, put back on the way out.
struct OnDevice {
    int was = -1;
    bool good;
    explicit OnDevice(int device) {
        if (cudaGetDevice(&was) != cudaSuccess) was = -1;
        good = was == device || cudaSetDevice(device) == cudaSuccess;
        if (!good) cudaGetLastError();
        if (was == device) was = -1;
    }
    ~OnDevice() {
        if (was >= 0) cudaSetDevice(was);
    }
};

// Launches a kernel that begins while the one before it in the stream ends: such a kernel calls
// stream_turn() before it touches any memory that another kernel may have written or reads, and reads it
// by ordinary loads (or __ldcs and the like): those of the read-only path (__ldg, const __restrict__) are
// for memory that nothing writes while the kernel runs, and it runs before its turn.
template <typename... P, typename... A>
cudaError_t launch_in_turn(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A&&... args) {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = block;
    c.dynamicSmemBytes = smem;
    c.stream = s;
    c.attrs = &at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}

// The cache as kernels see it.
struct PageView {
    int32_t* table;   // (n_seq, max_pages)
    int32_t* length;  // (n_seq)
    int32_t* refs;    // (n_page)
    int32_t* status;  // first code recorded, 0: none
    int32_t n_page, page_shift, HK, D, n_seq, max_pages, n_layer;
    uint16_t* bounds;  // (n_layer, n_page, HK, 2, D) smallest and largest key values; null: not kept
};

#if defined(__CUDACC__)
// The next kernel of the stream may be brought up from here on; this one's turn comes when all
// before it have ended and what they wrote is visible.
__device__ __forceinline__ void stream_turn() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
// A barrier of a cluster of C CTAs; of one CTA an ordinary one, which costs a third.
__device__ __forceinline__ void cluster_barrier(int C) {
    if (C == 1) {
        __syncthreads();
        return;
    }
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// In two halves: a CTA's memory may be reached by the cluster's others once it has begun, so each says so at its
// beginning (cluster_begun), and nobody reaches for another's before all have (cluster_all_begun).
__device__ __forceinline__ void cluster_begun(int C) {
    if (C > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_all_begun(int C) {
    if (C > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void pages_flag(const PageView& c, int code) { atomicCAS(c.status, 0, code); }
// Length of sequence s as kernels may use it: 0 for a number outside the table,
// never past what its row of the table can hold.
__device__ __forceinline__ int pages_length(const PageView& c, int s) {
    if (s < 0 || s >= c.n_seq) return 0;
    const int64_t cap = (int64_t)c.max_pages << c.page_shift;
    const int n = c.length[s];
    return n < 0 ? 0 : (int64_t)n > cap ? (int)cap : n;
}
#endif

// One attention call. Strides are in elements; vec: q and out rows may be read and
// written 16 bytes at a time.
struct AttendArgs {
    PageView c;
    const void* q;
    int64_t q_token, q_head;
    void* out;
    int64_t o_token, o_head;
    const int32_t* seqs;
    const int32_t* q_start;  // null: one token per sequence
    int layer, T, n, H, window, sinks;
    float scale_log2;  // scale * log2(e): scores are in powers of two
    int vec;
    int over;           // places of pages_decode.cu's line that stand for a beginning and an end
    float* part;        // partial results of units that several CTAs share
    uint32_t* counters; // arrivals per shared unit; zero between launches
    const int32_t* blocks;  // (T, HK, width) blocks that a token's kv head attends to; null: all positions
    int width;
};

// One choice of blocks.
struct SelectArgs {
    PageView c;
    const void* q;
    int64_t q_token, q_head;
    const int32_t* seqs;
    const int32_t* q_start;
    int layer, T, n, H, first, recent, width;
    int vec;       // q's rows may be read 16 bytes at a time
    int32_t* out;  // (T, HK, width)
};

#if defined(__CUDACC__)
// By one CTA of a launch: q_start ascends from 0 to T.
template <typename A>
__device__ __forceinline__ void check_q_start(const A& a) {
    bool bad = false;
    for (int i = threadIdx.x; i < a.n; i += blockDim.x) bad |= a.q_start[i] > a.q_start[i + 1];
    if (threadIdx.x == 0) bad |= a.q_start[0] != 0 || a.q_start[a.n] != a.T;
    if (bad) pages_flag(a.c, AERO_CUDA_PAGES_BAD_ROWS);
}
// Which sequence token t is of, and how many of its positions the token sees at most
// (its own position + 1). q_start is searched within its n + 1 entries whatever they hold.
template <typename A>
__device__ __forceinline__ void token_rows(const A& a, int t, int& seq, int& n) {
    if (!a.q_start) {
        seq = a.seqs[t];
        n = pages_length(a.c, seq);
        return;
    }
    int lo = 0, hi = a.n;  // the last i < n with q_start[i] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    seq = a.seqs[lo];
    const int q0 = a.q_start[lo], q1 = a.q_start[lo + 1], len = pages_length(a.c, seq);
    n = len - (q1 - q0) + (t - q0) + 1;
    if (t < q0 || t >= q1 || q1 - q0 > len) {
        pages_flag(a.c, AERO_CUDA_PAGES_BAD_ROWS);
        n = 0;
    }
}
#endif

// Workspace the two kernels need for a cache of this shape.
size_t pages_decode_part_floats(int D, int n_sm);
size_t pages_prompt_part_floats(int D, int n_sm);
int pages_decode_max_grid(int n_sm);
int pages_prompt_max_grid(int n_sm);
// A box of rows of a visible position without a page starts here: wholly outside the pool, so the
// copy fills it with zeros.
constexpr int kNoPageRow = -64;
// kmap / vmap: (n_layer * n_page * HK * page rows, D) with boxes of min(page, 64)
// rows by 64 columns, 128-byte swizzle.
cudaError_t launch_pages_decode(const AttendArgs& a, bool bf16, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                int n_sm, cudaStream_t s);
// k, v: the pool itself.
cudaError_t launch_pages_prompt(const AttendArgs& a, bool bf16, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                const void* k, const void* v, int n_sm, cudaStream_t s);
// Bounds of the pages that n sequences hold, and of the pages that an append of T tokens wrote to.
cudaError_t launch_set_bounds(const PageView& c, bool bf16, int layer, const void* k, const int32_t* seqs, int n, int n_sm,
                              cudaStream_t s);
cudaError_t launch_append_bounds(const PageView& c, bool bf16, int layer, const void* k, const int32_t* seqs,
                                 const int32_t* positions, int T, int n_sm, cudaStream_t s);
// Pages a sequence may hold at most for launch_select.
constexpr int kSelectPages = 131072;
cudaError_t launch_select(const SelectArgs& a, bool bf16, int n_sm, cudaStream_t s);

}  // namespace aero
