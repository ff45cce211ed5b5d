// Residual addition and root-mean-square norm of rows, to 16 bits or to 8 bits (e4m3) with a
// scale per row:
//   h = x (+ r)          in FP32; r_out = h rounded to the storage type
//   y = h * rsqrt(mean(h^2) + eps) * g
//   out = y rounded, or  a = max|y| / 448,  out = e4m3(y / a),  out_scale = a
// The norm is taken of the unrounded sum, so y is rounded once.  A row lies in the registers of its
// threads between the one read and the one write.
#include <type_traits>

#include "norm_rows.cuh"

namespace bdattn {
namespace {

// A row to a team of kTeam lanes (8, 16 or 32: 128 / kTeam rows side by side in a CTA) or, with kTeam = 0, to a
// CTA; kV pieces of eight values to a thread.  The CTAs stay and take further rows, whose values are on their way while
// a row is reduced and written.  The maximum of |h g| is found with the sum of squares, ahead of the
// root that scales it, so that a row is reduced once.
// kShift: rows that do not begin on 16 bytes, all of the call's tensors by the same number of elements: the
// pieces lie on 16 bytes all the same and the row's first and last are not whole.
template <bool kBf16, bool kFp8, int kV, int kTeam, bool kShift>
__global__ void __launch_bounds__(kTeam > 0 ? 128 : kV == 1 ? 1024 : 512) add_rmsnorm_kernel(const __grid_constant__ AddRmsNormArgs a) {
    __shared__ float red[2][64];
    constexpr int kSide = kTeam > 0 ? 128 / (kTeam > 0 ? kTeam : 1) : 1;       // rows side by side
    const int team = kTeam > 0 ? kTeam : static_cast<int>(blockDim.x);
    const int me = kTeam > 0 ? static_cast<int>(threadIdx.x) & (kTeam - 1) : static_cast<int>(threadIdx.x);
    if (a.one_wave) dependents_may_launch();
    wait_for_prior_grid();
    auto shift_of = [&](long long row) { return kShift ? static_cast<int>((a.shift + row * a.ldx) & 7) : 0; };
    uint4 x[kV], r[kV];
    auto fetch = [&](long long row) {
        const uint16_t* const xr = reinterpret_cast<const uint16_t*>(a.x) + row * a.ldx;
        const uint16_t* const rr = reinterpret_cast<const uint16_t*>(a.residual) + row * a.ldr;
        const int s = shift_of(row);
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int c = (me + v * team) * 8 - s;
            x[v] = r[v] = make_uint4(0u, 0u, 0u, 0u);
            if (row < a.rows && c < a.cols) {
                x[v] = norm_load<kShift>(xr, c, a.cols);
                if (a.residual != nullptr) r[v] = norm_load<kShift>(rr, c, a.cols);
            }
        }
    };
    const long long step = static_cast<long long>(gridDim.x) * kSide;
    long long row = static_cast<long long>(blockIdx.x) * kSide + (kTeam > 0 ? threadIdx.x / (kTeam > 0 ? kTeam : 1) : 0);
    fetch(row);
    int turn = 0;
    // (all rows of a CTA's turn together: the teams of a warp meet in its shuffles)
    for (long long base = static_cast<long long>(blockIdx.x) * kSide; base < a.rows; base += step, row += step, turn ^= 1) {
        const bool exists = kTeam == 0 || row < a.rows;
        const int s = shift_of(row);
        float y[kV][8];
        float ss = 0.0f, top = 0.0f;
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int c = (me + v * team) * 8 - s;
            float t[8];
            norm_wide<kBf16>(x[v], y[v]);
            norm_wide<kBf16>(r[v], t);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[v][i] += t[i];
                ss = fmaf(y[v][i], y[v][i], ss);
            }
        }
        const long long now = row;
        // the sum is written here, so that only its product with the gains is kept
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int c = (me + v * team) * 8 - s;
            if (exists && c < a.cols) {
                float g[8];
                norm_gains<kBf16, kShift>(a.gain, a.gain_is_f32, c, a.cols, g);
                if (a.residual_out != nullptr)
                    norm_store<kBf16, kShift>(reinterpret_cast<uint16_t*>(a.residual_out) + now * a.ldro, c, a.cols, y[v]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[v][i] *= g[i];
                    if (kFp8) top = fmaxf(top, fabsf(y[v][i]));
                }
            }
        }
        fetch(row + step);
        if constexpr (kTeam > 0) {
#pragma unroll
            for (int o = kTeam / 2; o > 0; o >>= 1) {
                ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (kFp8) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            }
        } else {
            block_sum_max(ss, top, red[turn]);
        }
        float inv = rsqrtf(ss / static_cast<float>(a.cols) + a.eps);
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
                for (int i = 0; i < 8; ++i) y[v][i] *= inv;
                if constexpr (kFp8) norm_store_e4m3<kShift>(reinterpret_cast<uint8_t*>(a.out) + now * a.ldo, c, a.cols, y[v]);
                else norm_store<kBf16, kShift>(reinterpret_cast<uint16_t*>(a.out) + now * a.ldo, c, a.cols, y[v]);
            }
        }
    }
}

// Rows of more than the registers of a CTA hold: read twice, the second time from the L2.
template <bool kBf16, bool kFp8, bool kShift>
__global__ void __launch_bounds__(1024) add_rmsnorm_wide_kernel(const __grid_constant__ AddRmsNormArgs a) {
    __shared__ float red[64];
    wait_for_prior_grid();
    const long long row = blockIdx.x;
    const uint16_t* const xr = reinterpret_cast<const uint16_t*>(a.x) + row * a.ldx;
    const uint16_t* const rr = reinterpret_cast<const uint16_t*>(a.residual) + row * a.ldr;
    const int s = kShift ? static_cast<int>((a.shift + row * a.ldx) & 7) : 0;
    auto sum = [&](int c, float (&h)[8], float (&g)[8]) {
        norm_wide<kBf16>(norm_load<kShift>(xr, c, a.cols), h);
        if (a.residual != nullptr) {
            norm_wide<kBf16>(norm_load<kShift>(rr, c, a.cols), g);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] += g[i];
        }
        norm_gains<kBf16, kShift>(a.gain, a.gain_is_f32, c, a.cols, g);
    };
    float ss = 0.0f, top = 0.0f;
    for (int c = static_cast<int>(threadIdx.x) * 8 - s; c < a.cols; c += 8192) {
        float h[8], g[8];
        sum(c, h, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            ss = fmaf(h[i], h[i], ss);
            if (kFp8) top = fmaxf(top, fabsf(h[i] * g[i]));
        }
    }
    block_sum_max(ss, top, red);
    float inv = rsqrtf(ss / static_cast<float>(a.cols) + a.eps), lift = 1.0f;
    if constexpr (kFp8) {
        const RowScale rs = row_scale(ss, top, inv);
        if (threadIdx.x == 0) a.out_scale[row] = rs.scale;
        inv = rs.factor;
        lift = rs.lift;
    }
    for (int c = static_cast<int>(threadIdx.x) * 8 - s; c < a.cols; c += 8192) {
        float h[8], g[8];
        sum(c, h, g);
        if (a.residual_out != nullptr) norm_store<kBf16, kShift>(reinterpret_cast<uint16_t*>(a.residual_out) + row * a.ldro, c, a.cols, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = kFp8 ? h[i] * g[i] * lift * inv : h[i] * (g[i] * inv);
        if constexpr (kFp8) norm_store_e4m3<kShift>(reinterpret_cast<uint8_t*>(a.out) + row * a.ldo, c, a.cols, h);
        else norm_store<kBf16, kShift>(reinterpret_cast<uint16_t*>(a.out) + row * a.ldo, c, a.cols, h);
    }
}

// Tensors that are off 16 bytes by different numbers of elements: an element at a time, read twice.
template <bool kBf16, bool kFp8>
__global__ void __launch_bounds__(1024) add_rmsnorm_any_kernel(const __grid_constant__ AddRmsNormArgs a) {
    __shared__ float red[64];
    wait_for_prior_grid();
    const long long row = blockIdx.x;
    const long long xo = row * a.ldx, ro = row * a.ldr;
    auto gain = [&](int c) {
        return a.gain == nullptr ? 1.0f : a.gain_is_f32 ? reinterpret_cast<const float*>(a.gain)[c] : layer_ld16<kBf16>(a.gain, c);
    };
    float ss = 0.0f, top = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        float h = layer_ld16<kBf16>(a.x, xo + c);
        if (a.residual != nullptr) h += layer_ld16<kBf16>(a.residual, ro + c);
        ss = fmaf(h, h, ss);
        top = fmaxf(top, fabsf(h * gain(c)));
    }
    block_sum_max(ss, top, red);
    const float inv = rsqrtf(ss / static_cast<float>(a.cols) + a.eps);
    const RowScale rs = row_scale(ss, top, inv);
    if (kFp8 && threadIdx.x == 0) a.out_scale[row] = rs.scale;
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
        float h = layer_ld16<kBf16>(a.x, xo + c);
        if (a.residual != nullptr) h += layer_ld16<kBf16>(a.residual, ro + c);
        if (a.residual_out != nullptr) store1<kBf16>(a.residual_out, row * a.ldro + c, h);
        if constexpr (kFp8)
            reinterpret_cast<uint8_t*>(a.out)[row * a.ldo + c] =
                __nv_cvt_float_to_fp8(h * gain(c) * rs.lift * rs.factor, __NV_SATFINITE, __NV_E4M3);
        else
            store1<kBf16>(a.out, row * a.ldo + c, h * inv * gain(c));
    }
}

template <bool kBf16, bool kFp8>
cudaError_t launch_norm(AddRmsNormArgs a, cudaStream_t stream) {
    // Elements that a tensor's first row lies off its vectors of eight: the same for all tensors, and in all
    // rows with the same ld mod 8, or the vectors of one would cross those of another.
    auto off = [](const void* p, int bytes) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) / bytes % 8); };
    a.shift = off(a.x, 2);
    bool same = true, zero = a.cols % 8 == 0 && a.shift == 0 && a.ldx % 8 == 0 && off(a.gain, 2) == 0;
    auto look = [&](const void* p, long long ld, int bytes) {
        if (p != nullptr) same = same && off(p, bytes) == a.shift && (ld - a.ldx) % 8 == 0;
    };
    look(a.residual, a.ldr, 2);
    look(a.residual_out, a.ldro, 2);
    look(a.out, a.ldo, kFp8 ? 1 : 2);
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
        if (pieces <= 8) return go(add_rmsnorm_kernel<kBf16, kFp8, 1, 8, kS>, 16, 128);
        if (pieces <= 16) return go(add_rmsnorm_kernel<kBf16, kFp8, 1, 16, kS>, 8, 128);
        if (pieces <= 32) return go(add_rmsnorm_kernel<kBf16, kFp8, 1, 32, kS>, 4, 128);
        // Few rows: a piece to a thread, the shortest chain (1 x 2560 2.0 us, a single row to a warp 2.6).  More rows than SMs: a
        // row to a warp up to 1024 columns (16384 x 640, 8-bit output, 15.4 us, to a CTA 17.6), then to a CTA with two pieces to a thread,
        // and beyond 4096 columns four, so that a CTA's two meetings stand against more bytes (16384 x 5120 101.6 us with
        // two, 99.0 with four, 134 with one; 8000 x 8192 89.7 and 75.5; 4096 x 2560 15.2 and 16.3; off 16 bytes two at all widths,
        // 9000 x 4101 72 and 84).
        if (a.rows <= sm_count() && pieces <= 1024) return go(add_rmsnorm_kernel<kBf16, kFp8, 1, 0, kS>, 1, threads(1));
        if (pieces <= 64) return go(add_rmsnorm_kernel<kBf16, kFp8, 2, 32, kS>, 4, 128);
        if (pieces <= 128) return go(add_rmsnorm_kernel<kBf16, kFp8, 4, 32, kS>, 4, 128);
        if (pieces <= (kS ? 1024 : 512)) return go(add_rmsnorm_kernel<kBf16, kFp8, 2, 0, kS>, 1, threads(2));
        if (pieces <= 2048) return go(add_rmsnorm_kernel<kBf16, kFp8, 4, 0, kS>, 1, threads(4));
        return launch_dependent(add_rmsnorm_wide_kernel<kBf16, kFp8, kS>, dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, stream, a);
    };
    if (zero && same) return pick(std::false_type{});
    if (same) return pick(std::true_type{});
    const int threads = a.cols < 1024 ? (a.cols + 31) / 32 * 32 : 1024;
    return launch_dependent(add_rmsnorm_any_kernel<kBf16, kFp8>, dim3(static_cast<unsigned>(a.rows)), dim3(threads), 0, stream, a);
}

}  // namespace

cudaError_t launch_add_rmsnorm(const AddRmsNormArgs& a, bool bf16, bool fp8, cudaStream_t stream) {
    if (fp8) return bf16 ? launch_norm<true, true>(a, stream) : launch_norm<false, true>(a, stream);
    return bf16 ? launch_norm<true, false>(a, stream) : launch_norm<false, false>(a, stream);
}

}  // namespace bdattn
