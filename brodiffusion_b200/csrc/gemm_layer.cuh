// What stands behind the accumulator of a layer's product (GemmLaunch::layer):
//   C = residual + gate * act(acc * x_scale * w_scale + bias)
// in FP32, rounded once.
#pragma once

#include "sdpa_internal.h"
#include "tc05.cuh"

namespace bdattn {

// x * sigmoid(k): GELU's tanh form is x sigmoid(2 u) with u = sqrt(2 / pi) (x + 0.044715 x^3), since
// (1 + tanh u) / 2 = sigmoid(2 u); SiLU is x sigmoid(x).  `t` is -k log2(e), at most 126: the
// approximate quotient is 0 for divisors beyond 2^126.
__device__ __forceinline__ float times_sigmoid(float x, float t) { return __fdividef(x, 1.0f + fast_exp2(t)); }
// The larger of both; NaN stays.  Below `least` an activation is within 2e-36 of 0, and x itself over 2^126 is not: -1e38
// would come out as -1.2.
__device__ __forceinline__ float at_least(float x, float least) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(least));
    return y;
}

template <int N>
__device__ __forceinline__ void activate(float (&f)[N], int act) {
    if (act == kActGelu) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = gelu_exact(f[i]);
    } else if (act == kActGeluTanh) {
        // -2 sqrt(2 / pi) log2(e) (x + 0.044715 x^3), 125.97 at -10
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = at_least(f[i], -10.0f);
            f[i] = times_sigmoid(x, x * fmaf(x * x, -0.10294324f, -2.3022082f));
        }
    } else if (act == kActSilu) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float x = at_least(f[i], -87.0f);
            f[i] = times_sigmoid(x, x * -1.44269504f);
        }
    }
}

template <bool kBf16>
__device__ __forceinline__ float layer_ld16(const void* base, long long i) {
    const uint16_t b = reinterpret_cast<const uint16_t*>(base)[i];
    return kBf16 ? __uint_as_float(static_cast<uint32_t>(b) << 16)
                 : __half2float(*reinterpret_cast<const __half*>(&b));
}
template <bool kBf16>
__device__ __forceinline__ float2 layer_pair(uint32_t w) {
    if constexpr (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// A scale.  Not through the read-only path: the kernel before this one may write it, and still run when this one is
// resident.
__device__ __forceinline__ float load_scale(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}

// Column values of a tile in shared memory, n to each of three arrays: bias, weight scale, gate.
template <bool kBf16>
__device__ __forceinline__ void layer_columns(const GemmProblem& p, float* cols, int n, int i, long long column, bool on) {
    cols[i] = on && p.bias != nullptr ? layer_ld16<kBf16>(p.bias, column) : 0.0f;
    cols[n + i] = on && p.w_scale != nullptr ? load_scale(p.w_scale + column) : 1.0f;
    cols[2 * n + i] = on && p.gate != nullptr ? layer_ld16<kBf16>(p.gate, column) : 1.0f;
}

// N columns of one row; cols: the arrays of layer_columns at the first of them; res: the row's residual, two
// values to a word.
template <bool kBf16, bool kFp8, int N>
__device__ __forceinline__ void layer_values(const GemmProblem& p, float (&f)[N], const float* cols, int n, float x_scale,
                                             const uint32_t (&res)[N / 2]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 b = *reinterpret_cast<const float4*>(cols + i);
        if constexpr (kFp8) {
            const float4 w = *reinterpret_cast<const float4*>(cols + n + i);
            f[i] = fmaf(f[i], x_scale * w.x, b.x);
            f[i + 1] = fmaf(f[i + 1], x_scale * w.y, b.y);
            f[i + 2] = fmaf(f[i + 2], x_scale * w.z, b.z);
            f[i + 3] = fmaf(f[i + 3], x_scale * w.w, b.w);
        } else {
            f[i] += b.x;
            f[i + 1] += b.y;
            f[i + 2] += b.z;
            f[i + 3] += b.w;
        }
    }
    activate(f, p.act);
    if (p.gate != nullptr) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 g = *reinterpret_cast<const float4*>(cols + 2 * n + i);
            f[i] *= g.x;
            f[i + 1] *= g.y;
            f[i + 2] *= g.z;
            f[i + 3] *= g.w;
        }
    }
    if (p.residual != nullptr) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 r = layer_pair<kBf16>(res[i]);
            f[2 * i] += r.x;
            f[2 * i + 1] += r.y;
        }
    }
}

// 32 x 32 residual values of a warp's tile, four lanes to a row as store_words32 writes them: lane -> (row lane / 4 of a
// group of eight, 16-byte piece lane % 4).
struct ResidualPiece {
    uint4 r[4];
    // base: element (first row, first column); rows / cols: how many of each exist
    __device__ __forceinline__ void load(const uint16_t* base, long long ld, int rows, int cols, int lane) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2), c = (lane & 3) * 8;
            r[i] = make_uint4(0u, 0u, 0u, 0u);
            // (not through the read-only path: the output may be the same matrix)
            if (row < rows && c < cols) r[i] = *reinterpret_cast<const uint4*>(base + row * ld + c);
        }
    }
    // This lane's own row, through 2 KB of shared memory.
    __device__ __forceinline__ void row_of_lane(uint8_t* stg, int lane, uint32_t (&w)[16]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2);
            *reinterpret_cast<uint4*>(stg + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4)) = r[i];
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(stg + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
            w[4 * c] = v.x;
            w[4 * c + 1] = v.y;
            w[4 * c + 2] = v.z;
            w[4 * c + 3] = v.w;
        }
        __syncwarp();
    }
};

}  // namespace bdattn
