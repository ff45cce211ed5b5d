// The norms behind one block and ahead of the next, with what stands between them:
//   b = x * rsqrt(mean(x^2) + eps) * post_gain             the block's output, normed
//   h = residual_scale * residual + gate[group of rows] * b    FP32;  residual_out = h rounded
//   y = h * rsqrt(mean(h^2) + eps) * gain
//   out = y rounded, or  a = max|y| / 448,  out = e4m3(y / a),  out_scale = a, or nothing
// x and residual are read once, both sums of squares are of unrounded values.  Bound by memory from a few hundred
// rows on (6 bytes an element for the stream and 1 or 2 for the output), by two meetings of a row's threads below: the second
// sum needs the first one's root.  16384 x 5120 to 8 bits 105 to 117 us by the GPU (5.0 to 5.6 TB/s), 4332 x 2240 in 16 bits 17.9 (4.3 TB/s), one row 2.4.
#include <type_traits>

#include "norm_rows.cuh"

namespace bdattn {
namespace {

// NaN where a row's sum of squares is not finite (its root would make zeros of finite values); a row of zeros stays one with an
// eps of 0 too.
__device__ __forceinline__ float sandwich_root(float ss, const SandwichNormArgs& a) {
    const float v = ss / static_cast<float>(a.cols) + a.eps;
    return !(ss <= FLT_MAX) ? __uint_as_float(0x7fffffffu) : v > 0.0f ? rsqrtf(v) : 0.0f;
}

// Two FP32 values to an instruction: the kernel is short of issue slots (16384 x 5120 131 us without).
__device__ __forceinline__ void mul2(float& a0, float& a1, float b0, float b1) {
    asm("{.reg .b64 x, y; mov.b64 x, {%0, %1}; mov.b64 y, {%2, %3}; mul.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x;}" : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}
// c += a * b
__device__ __forceinline__ void fma2(float& c0, float& c1, float a0, float a1, float b0, float b1) {
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%0, %1}; fma.rn.f32x2 z, x, y, z; mov.b64 {%0, %1}, z;}"
        : "+f"(c0), "+f"(c1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// Sum, and maximum where it is wanted, over the CTA (at most 32 warps); red: 64 floats, 16-byte aligned.
template <bool kMax>
__device__ __forceinline__ void sandwich_meet(float& s, float& m, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        if (kMax) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    const int warps = static_cast<int>(blockDim.x) >> 5;
    if (warps == 1) return;
    if ((threadIdx.x & 31) == 0) {
        red[threadIdx.x >> 5] = s;
        if (kMax) red[32 + (threadIdx.x >> 5)] = m;
    }
    __syncthreads();
    s = 0.0f;
    for (int w = 0; w < warps; w += 4) {          // the same order in every thread
        const float4 v = *reinterpret_cast<const float4*>(red + w);
        s += v.x;
        if (w + 1 < warps) s += v.y;
        if (w + 2 < warps) s += v.z;
        if (w + 3 < warps) s += v.w;
        if (kMax) {
            const float4 t = *reinterpret_cast<const float4*>(red + 32 + w);
            m = fmaxf(m, t.x);
            if (w + 1 < warps) m = fmaxf(m, t.y);
            if (w + 2 < warps) m = fmaxf(m, t.z);
            if (w + 3 < warps) m = fmaxf(m, t.w);
        }
    }
}

// As add_rmsnorm_kernel: a row to a team of kTeam lanes or, with kTeam = 0, to a CTA, kV pieces of eight values to a thread, in
// registers between the one read and the one write; the next row is on its way while this one is reduced.
template <bool kBf16, bool kFp8, int kV, int kTeam, bool kShift>
__global__ void __launch_bounds__(kTeam > 0 ? 128 : kV == 1 ? 1024 : 512, kTeam > 0 ? 1 : kV == 2 ? 2 : 1) sandwich_norm_kernel(const __grid_constant__ SandwichNormArgs a) {
    __shared__ __align__(16) float red[2][64];
    constexpr int kSide = kTeam > 0 ? 128 / (kTeam > 0 ? kTeam : 1) : 1;       // rows side by side
    const int team = kTeam > 0 ? kTeam : static_cast<int>(blockDim.x);
    const int me = kTeam > 0 ? static_cast<int>(threadIdx.x) & (kTeam - 1) : static_cast<int>(threadIdx.x);
    if (a.one_wave) dependents_may_launch();
    wait_for_prior_grid();
    // (rows and their step are below 2^31 and 2^24)
    const uint32_t rows = static_cast<uint32_t>(a.rows), step = gridDim.x * kSide;
    uint32_t row = blockIdx.x * kSide + (kTeam > 0 ? threadIdx.x / (kTeam > 0 ? kTeam : 1) : 0);
    auto shift_of = [&](uint32_t row) { return kShift ? static_cast<int>((a.shift + row * static_cast<uint32_t>(a.ldx)) & 7) : 0; };
    auto fetch = [&](const uint16_t* at, uint32_t row, uint4 (&v)[kV]) {
        const int s = shift_of(row);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const int c = (me + i * team) * 8 - s;
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row < rows && c < a.cols) v[i] = norm_load<kShift>(at, c, a.cols);
        }
    };
    auto reduce = [&](auto max, float& ss, float& top, float* const where) {
        constexpr bool kMax = decltype(max)::value;
        if constexpr (kTeam > 0) {
#pragma unroll
            for (int o = kTeam / 2; o > 0; o >>= 1) {
                ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (kMax) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            }
        } else {
            sandwich_meet<kMax>(ss, top, where);
        }
    };
    uint4 x[kV], r[kV];
    // rows by pointers that go on by the same number of bytes
    const uint16_t* xr = reinterpret_cast<const uint16_t*>(a.x) + row * a.ldx;
    const uint16_t* rr = reinterpret_cast<const uint16_t*>(a.residual) + row * a.ldr;
    uint16_t* ror = reinterpret_cast<uint16_t*>(a.residual_out) + row * a.ldro;
    uint8_t* outr = reinterpret_cast<uint8_t*>(a.out) + row * a.ldo * (kFp8 ? 1 : 2);
    fetch(xr, row, x);
    fetch(rr, row, r);
    // (all rows of a CTA's turn together: the teams of a warp meet in its shuffles)
    for (uint32_t base = blockIdx.x * kSide; base < rows; base += step) {
        const bool exists = kTeam == 0 || row < rows;
        const int s = shift_of(row);
        const uint16_t* const gate = a.gate == nullptr ? nullptr
            : reinterpret_cast<const uint16_t*>(a.gate) + min(row, rows - 1) / static_cast<uint32_t>(a.gate_rows) * a.ldg;
        float y[kV][8];
        float ss = 0.0f, ss1 = 0.0f, top = 0.0f;
        // x times what stands behind its norm, while its squares are added up
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int c = (me + v * team) * 8 - s;
            norm_wide<kBf16>(x[v], y[v]);
#pragma unroll
            for (int i = 0; i < 8; i += 2) fma2(ss, ss1, y[v][i], y[v][i + 1], y[v][i], y[v][i + 1]);
            if (exists && c < a.cols) {
                float t[8];
                if (a.post_gain != nullptr) {
                    norm_gains<kBf16, kShift>(a.post_gain, a.gain_is_f32, c, a.cols, t);
#pragma unroll
                    for (int i = 0; i < 8; i += 2) mul2(y[v][i], y[v][i + 1], t[i], t[i + 1]);
                }
                if (gate != nullptr) {
                    norm_gains<kBf16, kShift>(gate, 0, c, a.cols, t);
#pragma unroll
                    for (int i = 0; i < 8; i += 2) mul2(y[v][i], y[v][i + 1], t[i], t[i + 1]);
                }
            }
        }
        ss += ss1;
        xr += step * a.ldx;
        fetch(xr, row + step, x);
        reduce(std::false_type{}, ss, top, red[0]);
        const float inv_x = sandwich_root(ss, a);
        ss = ss1 = top = 0.0f;
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int c = (me + v * team) * 8 - s;
            if (exists && c < a.cols) {
                float t[8];
                norm_wide<kBf16>(r[v], t);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    mul2(t[i], t[i + 1], a.residual_scale, a.residual_scale);
                    fma2(t[i], t[i + 1], y[v][i], y[v][i + 1], inv_x, inv_x);
                    y[v][i] = t[i];
                    y[v][i + 1] = t[i + 1];
                    if (kShift) {
                        // (a piece's places off the row are not the row's, whatever the root is)
                        if (c + i < 0 || c + i >= a.cols) y[v][i] = 0.0f;
                        if (c + i + 1 < 0 || c + i + 1 >= a.cols) y[v][i + 1] = 0.0f;
                    }
                    fma2(ss, ss1, y[v][i], y[v][i + 1], y[v][i], y[v][i + 1]);
                }
                norm_store<kBf16, kShift>(ror, c, a.cols, y[v]);
            }
        }
        ss += ss1;
        const uint32_t now = row;
        row += step;
        rr += step * a.ldr;
        ror += step * a.ldro;
        uint8_t* const out = outr;
        outr += step * a.ldo * (kFp8 ? 1 : 2);
        fetch(rr, row, r);
        if (a.out == nullptr) {
            if (kTeam == 0) __syncthreads();       // (the next row's sums go where this one's were read)
            continue;
        }
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int c = (me + v * team) * 8 - s;
            if (exists && c < a.cols) {
                if (a.gain != nullptr) {
                    float g[8];
                    norm_gains<kBf16, kShift>(a.gain, a.gain_is_f32, c, a.cols, g);
#pragma unroll
                    for (int i = 0; i < 8; i += 2) mul2(y[v][i], y[v][i + 1], g[i], g[i + 1]);
                }
                if (kFp8) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(y[v][i]));
                }
            }
        }
        reduce(std::integral_constant<bool, kFp8>{}, ss, top, red[1]);
        float inv = sandwich_root(ss, a);
        if constexpr (kFp8) {
            const RowScale rs = row_scale(ss, top, inv);
            if (exists && me == 0) a.out_scale[now] = rs.scale;
            inv = rs.factor;
            if (rs.lift != 1.0f) {
#pragma unroll
                for (int v = 0; v < kV; ++v) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[v][i] *= rs.lift;
                }
            }
        }
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int c = (me + v * team) * 8 - s;
            if (exists && c < a.cols) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) mul2(y[v][i], y[v][i + 1], inv, inv);
                if constexpr (kFp8) norm_store_e4m3<kShift>(out, c, a.cols, y[v]);
                else norm_store<kBf16, kShift>(out, c, a.cols, y[v]);
            }
        }
    }
}

// Rows wider than the registers of a CTA, and tensors that are off 16 bytes by different numbers of elements: an element at a
// time, read three times (the second and third from the L2).  4096 x 20480 557 us, its bytes 102; 4096 x 5120 188, 31 by the kernel above.
template <bool kBf16>
__global__ void __launch_bounds__(1024) sandwich_norm_any_kernel(const __grid_constant__ SandwichNormArgs a) {
    __shared__ float red[2][64];
    wait_for_prior_grid();
    const long long row = blockIdx.x, xo = row * a.ldx, ro = row * a.ldr;
    const long long gate_at = a.gate != nullptr ? row / a.gate_rows * a.ldg : 0;
    auto vec = [&](const void* g, int is_f32, long long c) {
        return g == nullptr ? 1.0f : is_f32 ? reinterpret_cast<const float*>(g)[c] : layer_ld16<kBf16>(g, c);
    };
    auto put = [&](void* p, long long i, float v) { reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(pack2<kBf16>(v, 0.0f)); };
    float ss = 0.0f, top = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float v = layer_ld16<kBf16>(a.x, xo + c);
        ss = fmaf(v, v, ss);
    }
    block_sum_max(ss, top, red[0]);
    const float inv_x = sandwich_root(ss, a);
    auto sum = [&](int c) {
        const float b = layer_ld16<kBf16>(a.x, xo + c) * (inv_x * vec(a.post_gain, a.gain_is_f32, c));
        return fmaf(a.residual_scale, layer_ld16<kBf16>(a.residual, ro + c), a.gate != nullptr ? b * vec(a.gate, 0, gate_at + c) : b);
    };
    ss = top = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float h = sum(c);
        ss = fmaf(h, h, ss);
        top = fmaxf(top, fabsf(h * vec(a.gain, a.gain_is_f32, c)));
    }
    block_sum_max(ss, top, red[1]);
    const float inv = sandwich_root(ss, a);
    const RowScale rs = row_scale(ss, top, inv);
    if (a.out_scale != nullptr && threadIdx.x == 0) a.out_scale[row] = rs.scale;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float h = sum(c), g = vec(a.gain, a.gain_is_f32, c);
        put(a.residual_out, row * a.ldro + c, h);
        if (a.out_scale != nullptr)
            reinterpret_cast<uint8_t*>(a.out)[row * a.ldo + c] = __nv_cvt_float_to_fp8(h * g * rs.lift * rs.factor, __NV_SATFINITE, __NV_E4M3);
        else if (a.out != nullptr)
            put(a.out, row * a.ldo + c, h * inv * g);
    }
}

template <bool kBf16, bool kFp8>
cudaError_t launch_sandwich(SandwichNormArgs a, cudaStream_t stream) {
    // Elements that a tensor's rows lie off their vectors of eight: the same for all of them, as in launch_norm.
    auto off = [](const void* p, int bytes) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) / bytes % 8); };
    a.shift = off(a.x, 2);
    bool same = true;
    auto look = [&](const void* p, long long ld, int bytes) {
        if (p != nullptr) same = same && off(p, bytes) == a.shift && (ld - a.ldx) % 8 == 0;
    };
    look(a.residual, a.ldr, 2);
    look(a.residual_out, a.ldro, 2);
    look(a.out, a.ldo, a.out_scale != nullptr ? 1 : 2);
    const bool zero = a.cols % 8 == 0 && a.shift == 0 && a.ldx % 8 == 0 && off(a.post_gain, 2) == 0 && off(a.gain, 2) == 0 &&
                      off(a.gate, 2) == 0 && a.ldg % 8 == 0;
    auto go = [&](auto kern, int side, int threads) {
        const int most = resident_ctas(reinterpret_cast<const void*>(kern), threads);
        const long long ctas = (a.rows + side - 1) / side;
        a.one_wave = ctas <= sm_count();
        return launch_dependent(kern, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(threads), 0, stream, a);
    };
    auto pick = [&](auto shift) {
        constexpr bool kS = decltype(shift)::value;
        const int pieces = kS ? (a.cols + 14) / 8 : a.cols / 8;
        auto threads = [&](int v) { return ((pieces + v - 1) / v + 31) / 32 * 32; };
        if (pieces <= 8) return go(sandwich_norm_kernel<kBf16, kFp8, 1, 8, kS>, 16, 128);
        if (pieces <= 32) return go(sandwich_norm_kernel<kBf16, kFp8, 1, 32, kS>, 4, 128);
        // Few rows: a piece to a thread, the shortest chain.  More: two to a thread in 64 registers, which are twice as many warps as the
        // compiler would leave (16384 x 5120, 8-bit output, 157 us without the bound, 149 with it, 275 with one piece; 4332 x 2240 27.9, 21.5,
        // 24.5; all with single FP32 values to an instruction, with pairs of them 104.5 and 17.9).
        if (a.rows <= sm_count() && pieces <= 1024) return go(sandwich_norm_kernel<kBf16, kFp8, 1, 0, kS>, 1, threads(1));
        if (pieces <= 64) return go(sandwich_norm_kernel<kBf16, kFp8, 2, 32, kS>, 4, 128);
        if (pieces <= 128) return go(sandwich_norm_kernel<kBf16, kFp8, 4, 32, kS>, 4, 128);
        if (pieces <= 1024) return go(sandwich_norm_kernel<kBf16, kFp8, 2, 0, kS>, 1, threads(2));
        return go(sandwich_norm_kernel<kBf16, kFp8, 4, 0, kS>, 1, threads(4));
    };
    if (same && a.cols <= (zero ? 16384 : 16384 - 14)) return zero ? pick(std::false_type{}) : pick(std::true_type{});
    const int threads = a.cols < 1024 ? (a.cols + 31) / 32 * 32 : 1024;
    return launch_dependent(sandwich_norm_any_kernel<kBf16>, dim3(static_cast<unsigned>(a.rows)), dim3(threads), 0, stream, a);
}

}  // namespace

cudaError_t launch_sandwich_norm(const SandwichNormArgs& a, bool bf16, cudaStream_t stream) {
    if (a.out_scale != nullptr) return bf16 ? launch_sandwich<true, true>(a, stream) : launch_sandwich<false, true>(a, stream);
    return bf16 ? launch_sandwich<true, false>(a, stream) : launch_sandwich<false, false>(a, stream);
}

}  // namespace bdattn
