// Residual addition and root-mean-square norm of rows, to 16 bits or to 8 bits (e4m3) with a
// scale per row:
//   h = x (+ r)          in FP32; r_out = h rounded to the storage type
//   y = h * rsqrt(mean(h^2) + eps) * g
//   out = y rounded, or  a = max|y| / 448,  out = e4m3(y / a),  out_scale = a
// The norm is taken of the unrounded sum, so y is rounded once.  A row lies in the registers of its
// threads between the one read and the one write.
#include <cuda_fp8.h>

#include "sdpa_internal.h"
#include "tc05.cuh"

namespace bdattn {
namespace {

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

template <bool kBf16>
__device__ __forceinline__ float norm_gain(const AddRmsNormArgs& a, int c) {
    if (a.gain == nullptr) return 1.0f;
    return a.gain_is_f32 ? __ldg(reinterpret_cast<const float*>(a.gain) + c) : load1<kBf16>(a.gain, c);
}

// One row to a CTA, an element at a time, any width and alignment; the row is read twice.
template <bool kBf16, bool kFp8>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const AddRmsNormArgs a) {
    __shared__ float red[64];
    wait_for_prior_grid();
    const long long row = blockIdx.x;
    const long long xo = row * a.ldx, ro = row * a.ldr;
    float ss = 0.0f, top = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        float h = load1<kBf16>(a.x, xo + c);
        if (a.residual != nullptr) h += load1<kBf16>(a.residual, ro + c);
        ss = fmaf(h, h, ss);
        top = fmaxf(top, fabsf(h * norm_gain<kBf16>(a, c)));
    }
    block_sum_max(ss, top, red);
    const float inv = rsqrtf(ss / static_cast<float>(a.cols) + a.eps);
    const float scale = top * inv * (1.0f / kE4m3Max);
    const float mul = scale > 0.0f ? 1.0f / scale : 1.0f;
    if (kFp8 && threadIdx.x == 0) a.out_scale[row] = scale;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        float h = load1<kBf16>(a.x, xo + c);
        if (a.residual != nullptr) h += load1<kBf16>(a.residual, ro + c);
        if (a.residual_out != nullptr) store1<kBf16>(a.residual_out, row * a.ldro + c, h);
        const float y = h * inv * norm_gain<kBf16>(a, c);
        if constexpr (kFp8)
            reinterpret_cast<uint8_t*>(a.out)[row * a.ldo + c] = __nv_cvt_float_to_fp8(y * mul, __NV_SATFINITE, __NV_E4M3);
        else
            store1<kBf16>(a.out, row * a.ldo + c, y);
    }
}

}  // namespace

cudaError_t launch_add_rmsnorm(const AddRmsNormArgs& a, bool bf16, bool fp8, cudaStream_t stream) {
    int threads = (a.cols + 31) / 32 * 32;
    threads = threads > 1024 ? 1024 : threads;
    const dim3 grid(static_cast<unsigned>(a.rows));
    auto go = [&](auto kern) { return launch_dependent(kern, grid, dim3(threads), 0, stream, a); };
    if (fp8) return bf16 ? go(add_rmsnorm_kernel<true, true>) : go(add_rmsnorm_kernel<false, true>);
    return bf16 ? go(add_rmsnorm_kernel<true, false>) : go(add_rmsnorm_kernel<false, false>);
}

}  // namespace bdattn
