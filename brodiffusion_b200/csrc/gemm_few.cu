// A layer's product (gemm_layer.cuh) for few rows: single tokens and small batches of them.
//   C[m, n] = residual + gate * act(sum_k X[m, k] W[n, k] * scales + bias),  M <= 16
// What such a call costs is reading W once, so the weights go from memory straight to registers, many 16-byte
// loads in flight to a thread, and the products are mma.sync with sixteen rows of W as A and the (up to
// eight, or two eights of) rows of X as B: an instruction for 512 bytes of weights, no shared memory on the way.
// The order of K inside a product is free as long as both operands have the same: a lane's 16 bytes of
// a row are its words of two products (of 16 values of 16 bits, or 32 of 8 bits), so nothing is rearranged.
// The warps of a CTA share the K of sixteen rows in turns of 128 bytes, and where there are few rows of W a cluster of
// CTAs does; the sums meet in shared memory.
#include "gemm_layer.cuh"
#include "sdpa_internal.h"
#include "tc05.cuh"

namespace bdattn {
namespace {

constexpr int kFewN = 16;              // rows of W to a CTA
constexpr int kFewMaxParts = 8;

template <bool kBf16, bool kFp8>
__device__ __forceinline__ void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (kFp8) {
        asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        const uint32_t a[4] = {a0, a1, a2, a3};
        gen_mma<kBf16>(d, a, b0, b1);
    }
}
// Weights are read once: they leave what is kept in L1 where it is.  (Neither these loads nor those of X are of the
// read-only kind: this kernel may be resident while the one that writes its operands still runs.)
__device__ __forceinline__ uint4 load_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 load_kept(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

struct GemmFewArgs {
    GemmProblem p;          // K and the strides of X and W in 16-bit units
    const uint16_t* x;
    const uint16_t* w;
    long long ldx, ldw;
    int parts;              // CTAs of a cluster
};

// W: warps.  NR: rows of X in eights.  kDepth: turns of a warp in flight.  kCtas: CTAs of an SM; what hides the latency
// of memory are many warps with little in flight each (26 MB of weights, one row: 8 warps, two turns, three CTAs to an
// SM 6.3 us; 4 warps, three turns 8.6; a plain read of as many bytes takes 5.5).
template <bool kBf16, bool kFp8, int W, int NR, int kDepth, int kCtas>
__global__ void __launch_bounds__(W * 32, kCtas)
gemm_few_kernel(const __grid_constant__ GemmFewArgs a) {
    __shared__ float sums[W][kFewN * 8 * NR];
    __shared__ float parts_s[kFewMaxParts][kFewN * 8 * NR];
    const GemmProblem& p = a.p;
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int part = a.parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int n0 = static_cast<int>(blockIdx.y) * kFewN;
    const int g = lane >> 2, q = lane & 3;
    const int step = W * a.parts, first = part * W + warp;
    // Rows that do not exist are read as the last one that does: their sums go nowhere.
    const uint16_t* wp[2] = {a.w + static_cast<long long>(min(n0 + g, p.N - 1)) * a.ldw + first * 64 + q * 8,
                             a.w + static_cast<long long>(min(n0 + g + 8, p.N - 1)) * a.ldw + first * 64 + q * 8};
    const uint16_t* xp[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) xp[r] = a.x + min(r * 8 + g, p.M - 1) * a.ldx + first * 64 + q * 8;
    const int full = p.K / 64, n = first < full ? (full - first + step - 1) / step : 0;      // whole turns of this warp
    const long long advance = static_cast<long long>(step) * 64;
    if (a.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    dependents_may_launch();
    // While the kernel before this one ends, the first weights come into the L2.
    if (lane < 16 && n > 0) {
        const uint16_t* const at = a.w + static_cast<long long>(min(n0 + lane, p.N - 1)) * a.ldw + first * 64;
#pragma unroll
        for (int i = 0; i < kDepth; ++i)
            if (i < n) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + i * advance));
    }
    wait_for_prior_grid();

    uint4 wv[kDepth][2][2], xv[kDepth][2][NR];
    auto fetch = [&](uint4 (&w)[2][2], uint4 (&x)[2][NR]) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int h = 0; h < 2; ++h) w[s][h] = load_stream(wp[h] + s * 32);
#pragma unroll
            for (int r = 0; r < NR; ++r) x[s][r] = load_kept(xp[r] + s * 32);
        }
        wp[0] += advance;
        wp[1] += advance;
#pragma unroll
        for (int r = 0; r < NR; ++r) xp[r] += advance;
    };
    float acc[NR][4] = {};
    auto products = [&](const uint4 (&w)[2][2], const uint4 (&x)[2][NR]) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                few_mma<kBf16, kFp8>(acc[r], w[s][0].x, w[s][1].x, w[s][0].y, w[s][1].y, x[s][r].x, x[s][r].y);
                few_mma<kBf16, kFp8>(acc[r], w[s][0].z, w[s][1].z, w[s][0].w, w[s][1].w, x[s][r].z, x[s][r].w);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < kDepth; ++i)
        if (i < n) fetch(wv[i], xv[i]);
    for (int t = 0; t < n; t += kDepth) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
            if (t + i < n) {
                products(wv[i], xv[i]);
                if (t + i + kDepth < n) fetch(wv[i], xv[i]);
            }
        }
    }
    if (p.K % 64 != 0 && full % step == first) {
        // the last columns, fewer than a turn's
        uint4 w[2][2] = {}, x[2][NR] = {};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (full * 64 + s * 32 + q * 8 < p.K) {
#pragma unroll
                for (int h = 0; h < 2; ++h) w[s][h] = load_stream(wp[h] + s * 32);
#pragma unroll
                for (int r = 0; r < NR; ++r) x[s][r] = load_kept(xp[r] + s * 32);
            }
        }
        products(w, x);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[warp][(r * 8 + q * 2 + (e & 1)) * kFewN + g + 8 * (e >> 1)] = acc[r][e];
    }
    __syncthreads();
    if (a.parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int i = threadIdx.x; i < kFewN * 8 * NR; i += W * 32) {
        float f = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) f += sums[w][i];
        if (a.parts > 1)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa(smem_u32(&parts_s[part][i]), 0)), "f"(f) : "memory");
        else parts_s[0][i] = f;
    }
    // (the first CTA of a cluster finishes; without one a thread reads what it wrote itself)
    if (a.parts > 1) cluster_sync();
    if (part != 0) return;
    for (int i = threadIdx.x; i < kFewN * 8 * NR; i += W * 32) {
        const int m = i / kFewN, n = n0 + i % kFewN;
        if (m >= p.M || n >= p.N) continue;
        float f[1] = {0.0f};
        for (int k = 0; k < a.parts; ++k) f[0] += parts_s[k][i];
        if (kFp8) f[0] *= (p.x_scale != nullptr ? load_scale(p.x_scale + m) : 1.0f) * (p.w_scale != nullptr ? load_scale(p.w_scale + n) : 1.0f);
        if (p.bias != nullptr) f[0] += layer_ld16<kBf16>(p.bias, n);
        activate(f, p.act);
        if (p.gate != nullptr) f[0] *= layer_ld16<kBf16>(p.gate, n);
        if (p.residual != nullptr) f[0] += layer_ld16<kBf16>(p.residual, m * p.ldr + n);
        store1<kBf16>(p.C, m * p.ldc + n, f[0]);
    }
}

}  // namespace

cudaError_t launch_gemm_few(const GemmLaunch& L, const void* x, long long ldx, cudaStream_t stream) {
    GemmFewArgs a;
    a.p = L.args.p[0];
    a.x = reinterpret_cast<const uint16_t*>(x);
    a.w = reinterpret_cast<const uint16_t*>(L.W[0]);
    a.ldx = ldx;
    a.ldw = L.ldw[0];
    const int tiles = (a.p.N + kFewN - 1) / kFewN, turns = (a.p.K + 63) / 64;
    // K over a cluster while all CTAs run at once, three to an SM, and a warp has two turns (2560 x 2560 4.6 us over two,
    // 5.6 whole, 6.4 over four; 64 x 10240 3.4 over four, 6.8 whole; 1280 x 1280, 20 turns, 3.1 over two, 2.8 whole).
    int parts = 1;
    while (parts < kFewMaxParts && tiles * parts * 2 <= 3 * sm_count() && turns >= 32 * parts) parts *= 2;
    a.parts = parts;
    auto go = [&](auto kern, int warps) {
        return launch_dependent_cluster(kern, dim3(parts, tiles), dim3(warps * 32), 0, stream, dim3(parts), a);
    };
    // More CTAs than that: with a short K five of four warps to an SM (10240 x 1280 words 6.3 us, eight warps 7.9), else
    // four of eight warps with one turn in flight (8 rows x 10240 x 2560 9.4 us, 12.5 with two turns, 10.8 with four
    // warps; 20480 x 5120 31.9, 34.0 and 38.4).  Two eights of rows have no registers for more than one turn (16 x 5120 x 5120 in 8
    // bits 8.6 us, 16.3 with two; 16 x 20480 x 5120 38.5 with three CTAs, 44.1 with four).
    const bool many = tiles > 3 * sm_count(), brief = many && turns < 32;
    auto pick = [&](auto b, auto f) {
        constexpr bool kB = decltype(b)::value, kF = decltype(f)::value;
        if (a.p.M <= 8)
            return brief ? go(gemm_few_kernel<kB, kF, 4, 1, 2, 5>, 4) : many ? go(gemm_few_kernel<kB, kF, 8, 1, 1, 4>, 8)
                                                                             : go(gemm_few_kernel<kB, kF, 8, 1, 2, 3>, 8);
        return brief ? go(gemm_few_kernel<kB, kF, 4, 2, 1, 5>, 4) : go(gemm_few_kernel<kB, kF, 8, 2, 1, 3>, 8);
    };
    if (L.fp8) return L.bf16 ? pick(std::true_type{}, std::true_type{}) : pick(std::false_type{}, std::true_type{});
    return L.bf16 ? pick(std::true_type{}, std::false_type{}) : pick(std::false_type{}, std::false_type{});
}

}  // namespace bdattn
