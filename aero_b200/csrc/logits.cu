// Logits adjusted before sampling (include/aero_cuda_pages.h, aero_cuda_logits_adjust):
// penalties for the tokens of a row's history, biases of listed tokens, a grammar's
// mask.
//
// Bound by HBM: the logits are read and written once, in one launch. A CTA owns a slice
// of one row's vocabulary: it notes in shared memory what the row's history and biases
// say about the slice's tokens (counts are integer sums, so their order does not
// matter; biases of one token are added by one lane in the list's order), then streams
// the slice. Every CTA of a row reads the whole history (from L2 but for the first): a
// wider slice reads it fewer times, a narrower one fills the GPU at few rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <string>

#include "../../include/aero_cuda_pages.h"
#include "internal.h"
#include "pages.h"

namespace aero {
namespace {

constexpr int kLogitThreads = 512;
constexpr uint32_t kInPrompt = 0x80000000u;  // note of a token that the history holds, beside its count after the prompt

struct LogitArgs {
    const void* in;
    void* out;
    int64_t ld, ld_out;
    int vocab, slice;
    const int32_t* history;
    int64_t ld_history;
    const int32_t *n_history, *n_prompt;
    const float *repetition, *frequency, *presence;
    const int32_t *bias_start, *bias_token;
    const float* bias_value;
    const int32_t* mask;
    int64_t ld_mask;
};

template <typename E>
__device__ __forceinline__ float to_f(E v) {
    if constexpr (sizeof(E) == 4)
        return v;
    else if constexpr (std::is_same<E, __half>::value)
        return __half2float(v);
    else
        return __bfloat162float(v);
}
template <typename E>
__device__ __forceinline__ E from_f(float v) {
    if constexpr (sizeof(E) == 4)
        return v;
    else if constexpr (std::is_same<E, __half>::value)
        return __float2half_rn(v);
    else
        return __float2bfloat16_rn(v);
}

template <typename E>
__global__ void __launch_bounds__(kLogitThreads) adjust_kernel(const LogitArgs a) {
    extern __shared__ __align__(16) uint32_t notes[];                 // [slice], then [slice] biases
    float* bias = reinterpret_cast<float*>(notes + a.slice);
    const int r = (int)blockIdx.y, v0 = (int)blockIdx.x * a.slice, nv = min(a.slice, a.vocab - v0);
    const int tid = (int)threadIdx.x;
    const int nh = a.history ? max(0, a.n_history[r]) : 0;
    const int np = nh && a.n_prompt ? a.n_prompt[r] : 0;
    const int b0 = a.bias_start ? a.bias_start[r] : 0, b1 = a.bias_start ? a.bias_start[r + 1] : 0;
    if (nh > 0) {
        for (int i = tid; i < nv; i += kLogitThreads) notes[i] = 0;
        __syncthreads();
        const int32_t* h = a.history + (int64_t)r * a.ld_history;
        for (int i = tid; i < nh; i += kLogitThreads) {
            const uint32_t t = (uint32_t)(h[i] - v0);
            if (h[i] >= 0 && t < (uint32_t)nv) {
                if (i < np)
                    atomicOr(notes + t, kInPrompt);
                else
                    atomicAdd(notes + t, 1u);
            }
        }
    }
    if (b1 > b0) {
        for (int i = tid; i < nv; i += kLogitThreads) bias[i] = 0.f;
        __syncthreads();
        if (tid < 32) {
            for (int i = b0 + tid; i - tid < b1; i += 32) {
                const int t = i < b1 ? a.bias_token[i] : -1;
                const float x = i < b1 ? a.bias_value[i] : 0.f;
                const bool in = t >= v0 && t < v0 + nv;
                const uint32_t same = __match_any_sync(0xffffffffu, in ? t - v0 : -1);
                const bool leads = in && (same & ((1u << tid) - 1u)) == 0;
                float sum = leads ? bias[t - v0] : 0.f;
                // entries of one token, in the list's order
                uint32_t todo = same;
                while (__any_sync(0xffffffffu, leads && todo)) {
                    const int from = leads && todo ? __ffs((int)todo) - 1 : tid;
                    const float y = __shfl_sync(0xffffffffu, x, from);
                    if (leads && todo) {
                        sum += y;
                        todo &= todo - 1;
                    }
                }
                if (leads) bias[t - v0] = sum;
                __syncwarp();
            }
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[r] : 1.f;
    const float fr = a.frequency ? a.frequency[r] : 0.f, pr = a.presence ? a.presence[r] : 0.f;
    const uint32_t* bits = a.mask ? reinterpret_cast<const uint32_t*>(a.mask) + (int64_t)r * a.ld_mask : nullptr;
    const auto one = [&](float x, int i) {
        if (nh > 0) {
            const uint32_t note = notes[i];
            if (note) {
                x = x > 0.f ? x / rep : x * rep;
                const uint32_t c = note & ~kInPrompt;
                if (c) x = x - fr * (float)c - pr;
            }
        }
        if (b1 > b0) x += bias[i];
        return x;
    };
    const E* in = static_cast<const E*>(a.in) + (int64_t)r * a.ld + v0;
    E* out = static_cast<E*>(a.out) + (int64_t)r * a.ld_out + v0;
    constexpr int V = 16 / (int)sizeof(E);
    const bool vec = (((uintptr_t)in | (uintptr_t)out) & 15) == 0;
    const int whole = vec ? nv / V * V : 0;
    for (int i = tid * V; i < whole; i += kLogitThreads * V) {
        uint4 raw = __ldcs(reinterpret_cast<const uint4*>(in + i));
        // the bits of tokens v0 + i .. + V: one word, V divides 32 and the slice is a multiple of 32
        const uint32_t allow = bits ? bits[(v0 + i) >> 5] >> ((v0 + i) & 31) : 0xFFFFFFFFu;
        E* x = reinterpret_cast<E*>(&raw);
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = from_f<E>((allow >> j) & 1u ? one(to_f(x[j]), i + j) : -INFINITY);
        __stcs(reinterpret_cast<uint4*>(out + i), raw);
    }
    for (int i = whole + tid; i < nv; i += kLogitThreads) {
        const bool allow = !bits || (bits[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u;
        out[i] = from_f<E>(allow ? one(to_f(in[i]), i) : -INFINITY);
    }
}

bool refuse(const char* what) {
    set_free_error(what);
    return false;
}

bool device_or_null(const void* p) { return !p || (is_device_ptr(p) && ((uintptr_t)p & 3) == 0); }

}  // namespace
}  // namespace aero

extern "C" int aero_cuda_logits_adjust(const void* logits, int64_t ld, int dtype, int rows, int vocab,
                                       const int32_t* history, int64_t ld_history, const int32_t* n_history,
                                       const int32_t* n_prompt, const float* repetition, const float* frequency,
                                       const float* presence, const int32_t* bias_start, const int32_t* bias_token,
                                       const float* bias_value, const int32_t* mask, int64_t ld_mask, void* out,
                                       int64_t ld_out, void* stream) {
    using namespace aero;
    try {
        if (dtype != AERO_CUDA_TYPE_F32 && dtype != AERO_CUDA_TYPE_F16 && dtype != AERO_CUDA_TYPE_BF16)
            return refuse("logits are F32, F16 or BF16"), -1;
        if (rows < 0 || rows > 65535 || vocab <= 0) return refuse("rows must be from 0 to 65535 and vocab positive"), -1;
        if (rows == 0) return 0;
        if (ld < vocab || ld_out < vocab) return refuse("ld and ld_out must be at least vocab"), -1;
        const uintptr_t size = dtype == AERO_CUDA_TYPE_F32 ? 4 : 2;
        cudaPointerAttributes where{};
        if (cudaPointerGetAttributes(&where, logits) != cudaSuccess) {
            cudaGetLastError();
            where.type = cudaMemoryTypeUnregistered;
        }
        if ((where.type != cudaMemoryTypeDevice && where.type != cudaMemoryTypeManaged) || !is_device_ptr(out)) return refuse("logits and out must be device memory"), -1;
        if (((uintptr_t)logits | (uintptr_t)out) % size) return refuse("logits and out must be aligned to their type"), -1;
        if (history && !n_history) return refuse("a history needs n_history"), -1;
        if (bias_start && (!bias_token || !bias_value)) return refuse("bias_start needs bias_token and bias_value"), -1;
        if (mask && ld_mask < (vocab + 31) / 32) return refuse("ld_mask must be at least (vocab + 31) / 32"), -1;
        const void* arrays[] = {history, n_history, n_prompt, repetition, frequency, presence, bias_start, bias_token, bias_value, mask};
        for (const void* p : arrays)
            if (!device_or_null(p)) return refuse("histories, penalties, biases and masks must be device memory, aligned to 4 bytes"), -1;
        OnDevice on(where.device);
        if (!on.good) return refuse("cudaSetDevice failed"), -1;
        LogitArgs a{logits, out, ld, ld_out, vocab, 0, history, ld_history, n_history, n_prompt, repetition, frequency, presence, bias_start, bias_token, bias_value, mask, ld_mask};
        a.slice = 8192;
        const size_t smem = (size_t)a.slice * (bias_start ? 8 : 4);
        const dim3 grid((unsigned)((vocab + a.slice - 1) / a.slice), (unsigned)rows);
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        const auto launch = [&](auto kernel) {
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536);
            if (e != cudaSuccess) return e;
            kernel<<<grid, kLogitThreads, smem, s>>>(a);
            return cudaGetLastError();
        };
        const cudaError_t e = dtype == AERO_CUDA_TYPE_F32   ? launch(adjust_kernel<float>)
                              : dtype == AERO_CUDA_TYPE_F16 ? launch(adjust_kernel<__half>)
                                                            : launch(adjust_kernel<__nv_bfloat16>);
        if (e != cudaSuccess) {
            cudaGetLastError();
            set_free_error(std::string("logits_adjust: ") + cudaGetErrorString(e));
            return -1;
        }
        return 0;
    } catch (...) {
        return -1;
    }
}
