// 16-bit types of the paged cache and their warp-level matrix products.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "tc_common.cuh"

namespace aero {
namespace {

// Two f32 values rounded to nearest in the cache's type, packed (a in the low half).
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// A value of the cache's type in f32, and the low half of a pair of them.
template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t v) {
    if constexpr (BF16)
        return __uint_as_float((uint32_t)v << 16);
    else
        return __half2float(__ushort_as_half(v));
}
template <bool BF16>
__device__ __forceinline__ float low16(uint32_t pair) {
    return to_f32<BF16>((uint16_t)pair);
}

// Four 8x8 16-bit matrices from shared memory (lane i addresses row i % 8 of matrix i / 8).
template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
}

// An 8x8 16-bit matrix transposed across the warp (the fragment of one register a lane).
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t t;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
    return t;
}

// D (16x8 f32) += A (16x16) x B (16x8), operands in the cache's type.
template <bool BF16>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a row's weights are multiplied by, as a power of two, so that the largest of them is at most 2^15.
// f16 has no number below 2^-24 and full precision only from 2^-14 on: with a largest weight of 1 the
// many small ones of a long sequence would be lost to V's product while their sum l has them
// (65536 positions of weight 2^-25 beside one of 1: 0.2 %). bf16 reaches as far down as f32. The factor
// is in o and l alike, of all parts of a row, and leaves with their quotient.
template <bool BF16>
__device__ __forceinline__ float lifted(float m, float top) {
    return BF16 ? m : m - (15.f - top);  // top: how far above 2^0 a weight may lie beside a maximum of m
}

// Bounded wait of a whole warp for a phase of an mbarrier: true in every lane, or false in every
// lane after kWaitNs or when another warp has given up. Lanes may leave the polling at different
// tries; the vote brings them together again, as the .aligned instructions that follow need.
// The global timer is read now and then only (a read costs more than most of these waits last).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    bool ok = mbar_try(bar, parity);
    if (!ok) {
        uint64_t t0 = 0;
        for (int i = 1;; ++i) {
            ok = mbar_try(bar, parity);
            if (ok) break;
            if ((i & 63) == 0) {
                if (*abort_flag) break;
                const uint64_t now = gtimer();
                if (t0 == 0) t0 = now;
                if (now - t0 > kWaitNs) break;
            }
        }
    }
    return __all_sync(0xffffffffu, ok);
}

// 2^x, the hardware's approximation (relative error about 2^-22; 2^-inf = 0).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace
}  // namespace aero
