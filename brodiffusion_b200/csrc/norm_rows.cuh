// Rows of 16-bit values for the norm kernels: reductions over a CTA, pieces of eight values from and to memory, the scale
// of a row's values in 8 bits.
#pragma once

#include <cuda_fp8.h>

#include <cfloat>
#include <mutex>
#include <vector>

#include "gemm_layer.cuh"
#include "sdpa_internal.h"
#include "tc05.cuh"

namespace bdattn {

constexpr float kE4m3Max = 448.0f;

// Sum and maximum over the CTA (at most 32 warps).
__device__ __forceinline__ void block_sum_max(float& s, float& m, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    const int warps = static_cast<int>(blockDim.x) >> 5;
    if (warps == 1) return;
    if ((threadIdx.x & 31) == 0) {
        red[threadIdx.x >> 5] = s;
        red[32 + (threadIdx.x >> 5)] = m;
    }
    __syncthreads();
    s = 0.0f;
    m = 0.0f;
    for (int w = 0; w < warps; ++w) {          // the same order in every thread
        s += red[w];
        m = fmaxf(m, red[32 + w]);
    }
}

// The scale of a row's values of 8 bits, and the factor that takes h g to them.
// The maximum of |h g| does not know of NaN, nor of an infinity under a gain of 0, but the sum of squares does.  (A maximum that
// keeps NaN costs the row an instruction a value: 16384 x 5120 105.3 us, this way 104.1.)  A row of zeros has scale 0 with
// an eps of 0 too, where the root is infinite.  448 / top is beyond FP32 for the tiniest rows: these go through `lift`
// times their values, which is uniform over a row and 1 for all others.
struct RowScale {
    float scale, factor, lift;
};
__device__ __forceinline__ RowScale row_scale(float ss, float top, float inv) {
    RowScale r;
    r.scale = !(ss <= FLT_MAX) ? __uint_as_float(0x7fffffffu) : top == 0.0f ? 0.0f : top * inv * (1.0f / kE4m3Max);
    r.factor = r.scale > 0.0f ? inv * (1.0f / r.scale) : inv;
    r.lift = 1.0f;
    if (top < 0x1p-100f) {
        r.lift = 0x1p100f;
        r.factor = top > 0.0f ? kE4m3Max / (top * 0x1p100f) : 0.0f;
    }
    return r;
}

__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}

// Eight values of a row from element c on, as many of them as exist.  With kShift a piece at the row's ends is
// not whole; all others lie on 16 bytes.
template <bool kShift>
__device__ __forceinline__ uint4 norm_load(const void* row, int c, int cols) {
    const uint16_t* const p = reinterpret_cast<const uint16_t*>(row) + c;
    if (!kShift || (c >= 0 && c + 8 <= cols)) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i >= 0 && c + i < cols) w[i >> 1] |= static_cast<uint32_t>(p[i]) << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool kBf16>
__device__ __forceinline__ void norm_wide(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = layer_pair<kBf16>(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
template <bool kBf16, bool kShift>
__device__ __forceinline__ void norm_store(void* row, int c, int cols, const float (&f)[8]) {
    uint16_t* const p = reinterpret_cast<uint16_t*>(row) + c;
    const uint32_t w[4] = {pack2<kBf16>(f[0], f[1]), pack2<kBf16>(f[2], f[3]), pack2<kBf16>(f[4], f[5]), pack2<kBf16>(f[6], f[7])};
    if (!kShift || (c >= 0 && c + 8 <= cols)) {
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i >= 0 && c + i < cols) p[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
    }
}
template <bool kShift>
__device__ __forceinline__ void norm_store_e4m3(void* row, int c, int cols, const float (&f)[8]) {
    uint8_t* const p = reinterpret_cast<uint8_t*>(row) + c;
    const uint32_t w[2] = {pack4_e4m3(f[0], f[1], f[2], f[3]), pack4_e4m3(f[4], f[5], f[6], f[7])};
    if (!kShift || (c >= 0 && c + 8 <= cols)) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i >= 0 && c + i < cols) p[i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
    }
}
// Eight gains from element c on (on 16 bytes without kShift).  Not through the read-only path: the kernel before this one may
// write them, and still run when this one is resident.
template <bool kBf16, bool kShift>
__device__ __forceinline__ void norm_gains(const void* gain, int is_f32, int c, int cols, float (&g)[8]) {
    if (gain == nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = 1.0f;
    } else if (is_f32 && kShift) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = c + i >= 0 && c + i < cols ? reinterpret_cast<const float*>(gain)[c + i] : 0.0f;
    } else if (is_f32) {
        // (two loads: eight of them, predicated off for gains of 16 bits, are instructions all the same)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(gain) + c + i);
            g[i] = v.x;
            g[i + 1] = v.y;
            g[i + 2] = v.z;
            g[i + 3] = v.w;
        }
    } else if (kShift) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = c + i >= 0 && c + i < cols ? layer_ld16<kBf16>(gain, c + i) : 0.0f;
    } else {
        norm_wide<kBf16>(*reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(gain) + c), g);
    }
}

// CTAs of a kernel that run at once, looked up once for each kernel, size and device.
inline int resident_ctas(const void* kern, int threads) {
    struct Seen { const void* kern; int threads, dev, ctas; };
    static std::mutex mu;
    static std::vector<Seen> seen;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return sm_count();
    std::lock_guard<std::mutex> lock(mu);
    for (const Seen& s : seen)
        if (s.kern == kern && s.threads == threads && s.dev == dev) return s.ctas;
    int per = 1;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, threads, 0) != cudaSuccess || per < 1) per = 1;
    seen.push_back({kern, threads, dev, per * sm_count()});
    return seen.back().ctas;
}

}  // namespace bdattn
