// Logits adjusted before sampling (include/aero_cuda_pages.h, aero_cuda_logits_adjust):
// penalties for the tokens of a row's history, biases of listed tokens, a grammar's
// mask.
//
// Bound by HBM: the logits are read and written once, in one launch. A CTA owns a slice
// of one row's vocabulary. It notes in shared memory what the row's history and biases say
// about the slice's tokens, while the slice's first logits are on their way, then streams the
// slice. Slices are as wide as shared memory allows and the number of rows asks for, so that all
// CTAs run at once and a history is read few times: with slices of 8192 tokens every CTA of the
// 19 of a row read it, and three waves of CTAs each waited for it (64 rows of 151936 with 8192
// tokens of history: 31 us; as it is 21 us, of which HBM's share is 12.6). Counts are integer sums, so their order does not matter; the
// biases of one token are added by its own thread in the list's order. A slice that more of them
// name (the list's place holds kBiasList) is streamed with the biased tokens left as they are, and those
// are adjusted after it: for 2 kBiasList tokens at a time a warp adds the row's list up in the list's
// place. (A bias for every one of 151936 tokens: 6.9 ms a row, 16 rows 7.5; with each biased token's
// thread walking the row's whole list 66 and 112.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <string>
#include <type_traits>

#include "../../include/aero_cuda_pages.h"
#include "internal.h"
#include "pages.h"

namespace aero {
namespace {

constexpr int kLogitThreads = 512;
constexpr int kLogitCtas = 2;     // of an SM
constexpr int kLogitBatch = 4;    // 16-byte pieces of the slice in flight a thread
constexpr int kBiasList = 512;    // biases of a slice kept in shared memory; with more, sums of as many tokens twice
constexpr int kNotesBytes = 81920;

struct LogitArgs {
    const void* in;
    void* out;
    int64_t ld, ld_out;
    int vocab, slice;
    const int32_t* history;
    int64_t ld_history;
    int history_width;  // entries of a row, however far apart the rows lie
    const int32_t *n_history, *n_prompt;
    const float *repetition, *frequency, *presence;
    const int32_t *bias_start, *bias_token;
    const float* bias_value;
    int n_bias;  // entries of bias_token and bias_value
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

// NB: bits of a token's note, its count after the prompt below a bit that says the prompt holds
// it: 16 for histories at most 32767 tokens wide, else 32.
template <typename E, int NB>
__global__ void __launch_bounds__(kLogitThreads, kLogitCtas) adjust_kernel(const LogitArgs a) {
    constexpr int V = 16 / (int)sizeof(E), U = kLogitBatch;
    constexpr uint32_t kInPrompt = 1u << (NB - 1);
    extern __shared__ __align__(16) uint32_t notes[];                    // slice * NB / 32
    const int S = a.slice;
    uint32_t* biased = notes + S / 32 * NB;                              // slice / 32: a bit for a token with biases
    int* listed = reinterpret_cast<int*>(biased + S / 32);               // number of the slice's biases, padded
    int* list_token = listed + 4;                                        // [kBiasList]
    float* list_value = reinterpret_cast<float*>(list_token + kBiasList);
    const int r = (int)blockIdx.y, v0 = (int)blockIdx.x * S, nv = min(S, a.vocab - v0);
    const int tid = (int)threadIdx.x;
    const E* in = static_cast<const E*>(a.in) + (int64_t)r * a.ld + v0;
    E* out = static_cast<E*>(a.out) + (int64_t)r * a.ld_out + v0;
    const bool vec = (((uintptr_t)in | (uintptr_t)out) & 15) == 0;
    const uint32_t* bits = a.mask ? reinterpret_cast<const uint32_t*>(a.mask) + (int64_t)r * a.ld_mask : nullptr;
    stream_turn();
    const int nh = a.history ? min(max(0, a.n_history[r]), a.history_width) : 0;
    const int np = nh && a.n_prompt ? a.n_prompt[r] : 0;
    // whatever bias_start holds, nothing outside the list is read
    const int b0 = a.bias_start ? min(max(a.bias_start[r], 0), a.n_bias) : 0;
    const int b1 = a.bias_start ? min(max(a.bias_start[r + 1], b0), a.n_bias) : 0;
    const float rep = a.repetition ? a.repetition[r] : 1.f;
    const float per = 1.f / rep;  // x * (1 / rep) for x / rep: one f32 rounding more
    const float fr = a.frequency ? a.frequency[r] : 0.f, pr = a.presence ? a.presence[r] : 0.f;
    uint4 raw[U];
    uint32_t allow[U];
    const auto load = [&](int base) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = base + (k * kLogitThreads + tid) * V;
            // the bits of tokens v0 + i .. + V: of one word, since V divides 32 and S is a multiple of 32
            allow[k] = bits && i < nv ? __ldca(bits + ((v0 + i) >> 5)) >> ((v0 + i) & 31) : 0xFFFFFFFFu;
            E* x = reinterpret_cast<E*>(raw + k);
            if (vec && i + V <= nv) {
                raw[k] = __ldcs(reinterpret_cast<const uint4*>(in + i));
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (i + j < nv) x[j] = in[i + j];
            }
        }
    };
    load(0);
    if (nh > 0 || b1 > b0) {
        const int clear = S / 32 * (NB + 1);  // (slices are multiples of 128)
        for (int i = tid; i < clear / 4; i += kLogitThreads) reinterpret_cast<uint4*>(notes)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        // warp 0: the slice's biases, in the list's order
        if (b1 > b0 && tid < 32) {
            int n = 0;
            for (int i = b0 + tid; i - tid < b1; i += 32) {
                const int t = i < b1 ? a.bias_token[i] - v0 : -1;
                const bool mine = t >= 0 && t < nv;
                const uint32_t who = __ballot_sync(0xffffffffu, mine);
                const int at = n + __popc(who & ((1u << tid) - 1u));
                if (mine) {
                    atomicOr(biased + (t >> 5), 1u << (t & 31));
                    if (at < kBiasList) {
                        list_token[at] = t;
                        list_value[at] = a.bias_value[i];
                    }
                }
                n += __popc(who);
            }
            if (tid == 0) *listed = n;
        }
        if (nh > 0) {
            const int32_t* h = a.history + (int64_t)r * a.ld_history;
            const auto note = [&](int token, int i) {
                const uint32_t t = (uint32_t)token - (uint32_t)v0;  // (past every slice for a negative token)
                if (t < (uint32_t)nv) {
                    const int shift = NB == 16 ? 16 * (int)(t & 1) : 0;
                    uint32_t* at = notes + (NB == 16 ? t >> 1 : t);
                    if (i < np)
                        atomicOr(at, kInPrompt << shift);
                    else
                        atomicAdd(at, 1u << shift);
                }
            };
            const int whole = ((uintptr_t)h & 15) == 0 ? nh & ~3 : 0;
            constexpr int kBatch = 4;  // 16-byte loads in flight a thread
            for (int i0 = 4 * tid; i0 < whole; i0 += 4 * kLogitThreads * kBatch) {
                int4 t[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int i = i0 + 4 * kLogitThreads * k;
                    t[k] = i < whole ? __ldcg(reinterpret_cast<const int4*>(h + i)) : make_int4(-1, -1, -1, -1);
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int i = i0 + 4 * kLogitThreads * k;
                    note(t[k].x, i);
                    note(t[k].y, i + 1);
                    note(t[k].z, i + 2);
                    note(t[k].w, i + 3);
                }
            }
            for (int i = whole + tid; i < nh; i += kLogitThreads) note(h[i], i);
        }
        __syncthreads();
    }
    // the sum of token v0 + t's biases, in the list's order
    const auto biases = [&](int t) {
        const int n = *listed;
        float sum = 0.f;
        for (int i = 0; i < n; ++i)
            if (list_token[i] == t) sum += list_value[i];
        return sum;
    };
    // what a token's note makes of its logit
    const auto penalised = [&](float y, uint32_t n) {
        const uint32_t c = n & (kInPrompt - 1u);
        // c as f32: below 2^23 in the last bits of 2^23
        const float cf = NB == 16 ? __uint_as_float(0x4B000000u | c) - 8388608.f : (float)c;
        const float f = n ? y > 0.f ? per : rep : 1.f;
        return y * f - (c ? fmaf(fr, cf, pr) : 0.f);
    };
    // later: biased tokens are left as they are
    const auto stream = [&](auto later) {
        for (int base = 0; base < nv; base += kLogitThreads * V * U) {
            if (base) load(base);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int i = base + (k * kLogitThreads + tid) * V;
                if (i >= nv) break;
                E* x = reinterpret_cast<E*>(raw + k);
                const uint32_t bb = b1 > b0 ? biased[i >> 5] >> (i & 31) : 0u;
#pragma unroll
                for (int j0 = 0; j0 < V; j0 += 4) {
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = to_f(x[j0 + j]);
                    uint32_t n[4] = {0u, 0u, 0u, 0u};
                    if (nh > 0) {
                        if constexpr (NB == 16) {
                            const uint2 w = *reinterpret_cast<const uint2*>(notes + (i + j0) / 2);
                            n[0] = w.x & 0xFFFFu, n[1] = w.x >> 16, n[2] = w.y & 0xFFFFu, n[3] = w.y >> 16;
                        } else {
                            const uint4 w = *reinterpret_cast<const uint4*>(notes + i + j0);
                            n[0] = w.x, n[1] = w.y, n[2] = w.z, n[3] = w.w;
                        }
                    }
                    if (n[0] | n[1] | n[2] | n[3] | (bb >> j0 & 15u)) {
                        // (without branches: one token in twenty has a note, so nearly every warp comes here)
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = penalised(y[j], n[j]);
                        if (!decltype(later)::value && bb >> j0 & 15u)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (bb >> (j0 + j) & 1u) y[j] += biases(i + j0 + j);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (!(decltype(later)::value && bb >> (j0 + j) & 1u)) x[j0 + j] = from_f<E>(allow[k] >> (j0 + j) & 1u ? y[j] : -INFINITY);
                }
                if (vec && i + V <= nv) {
                    __stcs(reinterpret_cast<uint4*>(out + i), raw[k]);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (i + j < nv) out[i + j] = x[j];
                }
            }
        }
    };
    if (b1 <= b0 || *listed <= kBiasList) {
        stream(std::false_type{});
        return;
    }
    stream(std::true_type{});
    float* sums = reinterpret_cast<float*>(list_token);  // [2 * kBiasList]
    for (int t0 = 0; t0 < nv; t0 += 2 * kBiasList) {
        __syncthreads();  // what the slice's threads stored; the sums before
        for (int t = tid; t < 2 * kBiasList; t += kLogitThreads) sums[t] = 0.f;
        __syncthreads();
        if (tid < 32) {
            constexpr int kBatch = 4;  // loads in flight a lane
            for (int i0 = b0; i0 < b1; i0 += 32 * kBatch) {
                int token[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int i = i0 + 32 * k + tid;
                    token[k] = i < b1 ? a.bias_token[i] : -1;
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int64_t t = (int64_t)token[k] - v0 - t0;
                    const bool mine = token[k] >= 0 && t >= 0 && t < min(2 * kBiasList, nv - t0);
                    const uint32_t who = __ballot_sync(0xffffffffu, mine);
                    if (!who) continue;
                    // lanes that name the same token, one after another
                    const uint32_t same = __match_any_sync(0xffffffffu, mine ? (int)t : -1 - tid);
                    const int turn = mine ? __popc(same & ((1u << tid) - 1u)) : 32;
                    const int turns = __reduce_max_sync(0xffffffffu, mine ? turn + 1 : 0);
                    const float value = mine ? a.bias_value[i0 + 32 * k + tid] : 0.f;
                    for (int n = 0; n < turns; ++n) {
                        if (turn == n) sums[t] += value;
                        __syncwarp();
                    }
                }
            }
        }
        __syncthreads();
        for (int t = t0 + tid; t < min(t0 + 2 * kBiasList, nv); t += kLogitThreads) {
            if (!(biased[t >> 5] >> (t & 31) & 1u)) continue;
            uint32_t n = 0;
            if (nh > 0) n = NB == 16 ? notes[t >> 1] >> 16 * (t & 1) & 0xFFFFu : notes[t];
            const float y = penalised(to_f(out[t]), n) + sums[t - t0];
            const int v = v0 + t;
            out[t] = from_f<E>(!bits || bits[v >> 5] >> (v & 31) & 1u ? y : -INFINITY);
        }
    }
}

template <typename E, int NB>
cudaError_t launch_adjust(const LogitArgs& a, int rows, int device, cudaStream_t s) {
    static thread_local int prepared = -1;  // the device whose attribute this thread has set
    if (prepared != device) {
        const cudaError_t e = cudaFuncSetAttribute(adjust_kernel<E, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, 98304);
        if (e != cudaSuccess) return e;
        prepared = device;
    }
    const size_t smem = (size_t)a.slice / 8 * (size_t)(NB + 1) + 16 + kBiasList * 8;
    const unsigned slices = (unsigned)(((int64_t)a.vocab + a.slice - 1) / a.slice);
    return launch_in_turn(adjust_kernel<E, NB>, dim3(slices, (unsigned)rows), kLogitThreads, smem, s, a);
}

bool refuse(const char* what) {
    set_free_error(what);
    return false;
}

bool device_or_null(const void* p) { return !p || (is_device_ptr(p) && ((uintptr_t)p & 3) == 0); }

bool adjust(const void* logits, int64_t ld, int dtype, int rows, int vocab, const int32_t* history, int64_t ld_history,
            int history_width, const int32_t* n_history, const int32_t* n_prompt, const float* repetition,
            const float* frequency, const float* presence, const int32_t* bias_start, const int32_t* bias_token,
            const float* bias_value, int n_bias, const int32_t* mask, int64_t ld_mask, void* out, int64_t ld_out,
            void* stream) {
    if (dtype != AERO_CUDA_TYPE_F32 && dtype != AERO_CUDA_TYPE_F16 && dtype != AERO_CUDA_TYPE_BF16)
        return refuse("logits are F32, F16 or BF16");
    if (rows < 0 || rows > 65535 || vocab <= 0) return refuse("rows must be from 0 to 65535 and vocab positive");
    if (rows == 0) return true;
    if (ld < vocab || ld_out < vocab) return refuse("ld and ld_out must be at least vocab");
    const uintptr_t size = dtype == AERO_CUDA_TYPE_F32 ? 4 : 2;
    cudaPointerAttributes where{};
    if (cudaPointerGetAttributes(&where, logits) != cudaSuccess) {
        cudaGetLastError();
        where.type = cudaMemoryTypeUnregistered;
    }
    if ((where.type != cudaMemoryTypeDevice && where.type != cudaMemoryTypeManaged) || !is_device_ptr(out)) return refuse("logits and out must be device memory");
    if (((uintptr_t)logits | (uintptr_t)out) % size) return refuse("logits and out must be aligned to their type");
    if (history && (ld_history < 0 || history_width < 1)) return refuse("ld_history must be >= 0 and the history's width positive");
    if (history && !n_history) return refuse("a history needs n_history");
    if (bias_start && (!bias_token || !bias_value)) return refuse("bias_start needs bias_token and bias_value");
    if (n_bias < 0) return refuse("n_bias must be >= 0");
    if (mask && ld_mask != 0 && ld_mask < (vocab + 31) / 32) return refuse("ld_mask must be 0 or at least (vocab + 31) / 32");
    const void* arrays[] = {history, n_history, n_prompt, repetition, frequency, presence, bias_start, bias_token, bias_value, mask};
    for (const void* p : arrays)
        if (!device_or_null(p)) return refuse("histories, penalties, biases and masks must be device memory, aligned to 4 bytes");
    OnDevice on(where.device);
    if (!on.good) return refuse("cudaSetDevice failed");
    LogitArgs a{logits, out, ld, ld_out, vocab, 0, history, ld_history, history ? history_width : 0, n_history, n_prompt, repetition, frequency, presence, bias_start, bias_token, bias_value, n_bias, mask, ld_mask};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int n_sm = 148;
    cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, where.device);
    // As many slices as leave two CTAs for each SM in one wave, none narrower than a CTA's first
    // batch of loads (f32; 16-bit logits: half of it), none wider than the notes' place.
    const int nb = a.history_width <= 32767 ? 16 : 32, widest = kNotesBytes / 4 * 32 / nb;
    const int64_t fill = std::max(1, kLogitCtas * n_sm / rows), least = ((int64_t)vocab + widest - 1) / widest;
    const int64_t most = std::max<int64_t>(least, vocab / (kLogitThreads * 4 * kLogitBatch) + 1);
    const int64_t slices = std::min(std::max(fill, least), most);
    a.slice = (int)std::min<int64_t>((((int64_t)vocab + slices - 1) / slices + 127) / 128 * 128, widest);
    const auto typed = [&](auto zero) {
        using E = decltype(zero);
        return nb == 16 ? launch_adjust<E, 16>(a, rows, where.device, s) : launch_adjust<E, 32>(a, rows, where.device, s);
    };
    const cudaError_t e = dtype == AERO_CUDA_TYPE_F32   ? typed(float{})
                          : dtype == AERO_CUDA_TYPE_F16 ? typed(__half{})
                                                        : typed(__nv_bfloat16{});
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_free_error(std::string("logits_adjust: ") + cudaGetErrorString(e));
        return false;
    }
    return true;
}

}  // namespace
}  // namespace aero

extern "C" {

int aero_cuda_logits_adjust_views(const void* logits, int64_t ld, int dtype, int rows, int vocab, const int32_t* history,
                                  int64_t ld_history, int history_width, const int32_t* n_history,
                                  const int32_t* n_prompt, const float* repetition, const float* frequency,
                                  const float* presence, const int32_t* bias_start, const int32_t* bias_token,
                                  const float* bias_value, int n_bias, const int32_t* mask, int64_t ld_mask,
                                  void* out, int64_t ld_out, void* stream) {
    try {
        return aero::adjust(logits, ld, dtype, rows, vocab, history, ld_history, history_width, n_history, n_prompt, repetition,
                            frequency, presence, bias_start, bias_token, bias_value, n_bias, mask, ld_mask, out, ld_out,
                            stream)
                   ? 0
                   : -1;
    } catch (...) {
        return -1;
    }
}

int aero_cuda_logits_adjust(const void* logits, int64_t ld, int dtype, int rows, int vocab, const int32_t* history,
                            int64_t ld_history, const int32_t* n_history, const int32_t* n_prompt,
                            const float* repetition, const float* frequency, const float* presence,
                            const int32_t* bias_start, const int32_t* bias_token, const float* bias_value,
                            const int32_t* mask, int64_t ld_mask, void* out, int64_t ld_out, void* stream) {
    const int width = (int)std::max<int64_t>(0, std::min<int64_t>(ld_history, INT32_MAX));
    return aero_cuda_logits_adjust_views(logits, ld, dtype, rows, vocab, history, ld_history, width, n_history, n_prompt,
                                         repetition, frequency, presence, bias_start, bias_token, bias_value,
                                         INT32_MAX, mask, ld_mask, out, ld_out, stream);
}

}  // extern "C"
