// Values in 4 bits, groups of them with a step and a lowest value each:  x = low + step * u,  u in 0..15.
//
// The codes go to the tensor core as they lie.  Among the low bits of a BF16 or FP16 the integer n (below 2^8, 2^11) is
// the number n * 2^-133, or n * 2^-24: below the smallest normal exactly so, and the first binade above continues it.  A mask
// makes two operands of a word: the nibbles 0 and 4 as they are, 1 and 5 times 16.  So a word of eight codes costs
// five instructions, no code is rounded, and the steps are applied to sums in FP32.  What meets them carries the
// power of two that brings the products back to the middle of FP32's range.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gemm_layer.cuh"
#include "sdpa_internal.h"
#include "tc05.cuh"

namespace bdattn {

// The eight codes of a word as four pairs (j, j + 4); those of 1 and 3 are sixteen times theirs.
__device__ __forceinline__ void codes8(uint32_t w, uint32_t (&r)[4]) {
    r[0] = w & 0x000f000fu;
    r[1] = w & 0x00f000f0u;
    r[2] = (w >> 8) & 0x000f000fu;
    r[3] = (w >> 8) & 0x00f000f0u;
}

// FP16 codes (in units of 2^-24, those of codes8's odd pairs, kSixteen: 2^-20) less eight: exact below the smallest normal too.
template <bool kSixteen>
__device__ __forceinline__ uint32_t less_eight(uint32_t u) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(kSixteen ? 0x00800080u : 0x00080008u));
    return r;
}

// D += A B, 16 x 8 x 16, FP32 sums.
template <bool kBf16>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (kBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with nothing to add to.
template <bool kBf16>
__device__ __forceinline__ void mma16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (kBf16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// D = A B, 16 x 8 x 8: FP32 values of which 11 bits count (all of a step or a low).
__device__ __forceinline__ void mma8_tf32_first(float (&d)[4], float a0, float a1, float a2, float a3, float b0, float b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)),
          "f"(0.0f));
}

// Loads of a kernel's operands: not of the read-only kind, since the kernel may be resident while the one that writes
// them still runs.  Codes are read once and leave what is kept in L1 where it is.
__device__ __forceinline__ uint4 load16_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load8_once(const void* p) {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load4_once(const void* p) {
    uint32_t v;
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// kWords words, 1, 2 or 4, aligned to their size.
template <int kWords>
__device__ __forceinline__ void load_words_once(const void* p, uint32_t (&w)[kWords]) {
    static_assert(kWords == 1 || kWords == 2 || kWords == 4, "a load's width");
    if constexpr (kWords == 4) {
        const uint4 v = load16_once(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (kWords == 2) {
        const uint2 v = load8_once(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = load4_once(p);
    }
}

}  // namespace bdattn
