// A layer's product with 4-bit weights:
//   C[m, n] = residual + gate * act(sum_k X[m, k] W[n, k] + bias),  W[n, k] = low[n, g] + step[n, g] u[n, k],  g = k / group
// as  sum_g step[n, g] (sum_{k in g} X u) + low[n, g] (sum_{k in g} X):  the codes u enter mma.sync as exact small integers
// (four_bit.cuh), the sums of X come from the same instruction with ones for weights, and step and low are applied to
// FP32 sums every 32 columns, so that nothing is rounded but X, W as they are given and the result.
//
// What a call of few rows costs is reading W once, 4 + 32 / group bits a value.  Packed weights (w4_pack_kernel) are tiles of 16 rows x 128
// columns in the order in which a warp's lanes want them: 16 bytes a lane for each eight of its rows, the steps and
// lows behind them, K tiles of a row tile one behind the other.
#include "four_bit.cuh"

namespace bdattn {
namespace {

constexpr int kW4MaxParts = 8;

__host__ __device__ constexpr int w4_tile_bytes(int group) { return 1024 + 16 * (128 / group) * 4; }

struct W4Args {
    GemmProblem p;          // M, N, K, C, bias, act, gate, residual
    const uint16_t* x;
    const uint8_t* w;
    long long ldx;
    int k_tiles, parts;     // tiles of 128 columns; CTAs of a cluster, which share them
};

// kGroups: groups of a tile's 128 columns.  W: warps, each with K tiles of its own.  T: row tiles of a CTA.  NR: rows of X in
// eights.
template <bool kBf16, int kGroups, int W, int T, int NR>
__global__ void __launch_bounds__(W * 32) w4_linear_kernel(const __grid_constant__ W4Args a) {
    extern __shared__ float w4_sums[];      // [W][16 T x 8 NR], then [parts][16 T x 8 NR]
    constexpr int kOut = 16 * T * 8 * NR, kTile = w4_tile_bytes(128 / kGroups);
    const GemmProblem& p = a.p;
    const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int part = a.parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int n_tiles = (p.N - 1) / 16 + 1, tile0 = static_cast<int>(blockIdx.x) / a.parts * T, m0 = static_cast<int>(blockIdx.y) * 8 * NR;
    const int first = part * W + warp, step = a.parts * W;
    const uint8_t* wp[T];
#pragma unroll
    for (int t = 0; t < T; ++t)      // (a row tile that does not exist is read as the last one: its sums go nowhere)
        wp[t] = a.w + static_cast<long long>(min(tile0 + t, n_tiles - 1)) * a.k_tiles * kTile;
    if (a.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    dependents_may_launch();
    wait_for_prior_grid();

    const uint16_t* xp[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) xp[r] = a.x + min(m0 + r * 8 + g, p.M - 1) * a.ldx + q * 8;

    uint4 wv[T][2];
    uint32_t sv[T][2][kGroups];
    auto fetch = [&](int kt) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const uint8_t* const at = wp[t] + static_cast<long long>(kt) * kTile;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                wv[t][h] = load16_once(at + h * 512 + lane * 16);
                load_words_once<kGroups>(at + 1024 + (g + 8 * h) * 4 * kGroups, sv[t][h]);
            }
        }
    };
    float y[T][NR][4] = {};
    if (first < a.k_tiles) fetch(first);
    for (int kt = first; kt < a.k_tiles; kt += step) {
        uint32_t w[T][2][4], sc[T][2][kGroups];
#pragma unroll
        for (int t = 0; t < T; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[t][h][0] = wv[t][h].x; w[t][h][1] = wv[t][h].y; w[t][h][2] = wv[t][h].z; w[t][h][3] = wv[t][h].w;
#pragma unroll
                for (int i = 0; i < kGroups; ++i) sc[t][h][i] = sv[t][h][i];
            }
        }
        if (kt + step < a.k_tiles) fetch(kt + step);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            // eight columns of X a lane, in the pairs of codes8
            const int c = kt * 128 + s * 32;
            uint32_t b[NR][4];
            float xs[NR][4];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (c + q * 8 < p.K) v = load16(xp[r] + c);
                b[r][0] = __byte_perm(v.x, v.z, 0x5410);
                b[r][1] = __byte_perm(v.x, v.z, 0x7632);
                b[r][2] = __byte_perm(v.y, v.w, 0x5410);
                b[r][3] = __byte_perm(v.y, v.w, 0x7632);
                if constexpr (kBf16) {
                    // 2^64, and 2^60 where the codes are sixteen times theirs: exact, beyond FP32 from |x| = 2^63 on
                    const __nv_bfloat162 up = __float2bfloat162_rn(0x1p64f), up16 = __float2bfloat162_rn(0x1p60f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        __nv_bfloat162& f = reinterpret_cast<__nv_bfloat162&>(b[r][i]);
                        f = __hmul2(f, (i & 1) ? up16 : up);
                    }
                }
                // sums of X over the 32 columns, in the places of their rows of C
                constexpr uint32_t kOne = kBf16 ? 0x3f803f80u : 0x3c003c00u, kOdd = kBf16 ? 0x41804180u : kOne;
                xs[r][0] = xs[r][1] = xs[r][2] = xs[r][3] = 0.0f;
                mma16<kBf16>(xs[r], kOne, kOne, kOne, kOne, b[r][0], b[r][2]);
                mma16<kBf16>(xs[r], kOdd, kOdd, kOdd, kOdd, b[r][1], b[r][3]);
                if constexpr (kBf16) {
                    xs[r][0] *= 0x1p-64f;
                    xs[r][1] *= 0x1p-64f;
                }
            }
#pragma unroll
            for (int t = 0; t < T; ++t) {
                uint32_t u[2][4];
                float2 sl[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    codes8<kBf16>(w[t][h][s], u[h]);
                    sl[h] = layer_pair<kBf16>(sc[t][h][s * kGroups / 4]);
                    sl[h].x *= kBf16 ? 0x1p69f : 0x1p24f;
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float d[4] = {};
                    mma16<kBf16>(d, u[0][0], u[1][0], u[0][2], u[1][2], b[r][0], b[r][2]);
                    mma16<kBf16>(d, u[0][1], u[1][1], u[0][3], u[1][3], b[r][1], b[r][3]);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        y[t][r][e] = fmaf(d[e], sl[e >> 1].x, fmaf(xs[r][e & 1], sl[e >> 1].y, y[t][r][e]));
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w4_sums[warp * kOut + (r * 8 + q * 2 + (e & 1)) * 16 * T + t * 16 + g + 8 * (e >> 1)] = y[t][r][e];
        }
    }
    float* const parts_s = w4_sums + W * kOut;
    __syncthreads();
    // (waited for ahead of the first store into a peer's shared memory: it has to run by then)
    if (a.parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int i = threadIdx.x; i < kOut; i += W * 32) {
        float f = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) f += w4_sums[w * kOut + i];
        if (a.parts > 1)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa(smem_u32(parts_s + part * kOut + i), 0)), "f"(f) : "memory");
        else parts_s[i] = f;
    }
    // (the first CTA of a cluster finishes; without one a thread reads what it wrote itself)
    if (a.parts > 1) cluster_sync();
    if (part != 0) return;
    for (int i = threadIdx.x; i < kOut; i += W * 32) {
        const int m = m0 + i / (16 * T);
        const long long n = tile0 * 16ll + i % (16 * T);
        if (m >= p.M || n >= p.N) continue;
        float f[1] = {0.0f};
        for (int k = 0; k < a.parts; ++k) f[0] += parts_s[k * kOut + i];
        if (p.bias != nullptr) f[0] += layer_ld16<kBf16>(p.bias, n);
        activate(f, p.act);
        if (p.gate != nullptr) f[0] *= layer_ld16<kBf16>(p.gate, n);
        if (p.residual != nullptr) f[0] += layer_ld16<kBf16>(p.residual, m * p.ldr + n);
        reinterpret_cast<uint16_t*>(p.C)[m * p.ldc + n] = static_cast<uint16_t>(pack2<kBf16>(f[0], 0.0f));
    }
}

// Row-major codes (two to a byte, the even column's in the low half) and pairs into the packed order; rows and columns that do
// not exist count for nothing (step and low 0).  A thread to a word of eight codes.
__global__ void __launch_bounds__(256) w4_pack_kernel(const W4PackArgs a) {
    wait_for_prior_grid();
    const int per = 256 + 16 * (128 / a.group);                   // words of a tile: codes, pairs
    const long long total = static_cast<long long>((a.N - 1) / 16 + 1) * a.k_tiles * per;
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += 256ll * gridDim.x) {
        const long long tile = i / per;
        const int at = static_cast<int>(i - tile * per), kt = static_cast<int>(tile % a.k_tiles);
        const long long row0 = tile / a.k_tiles * 16;
        uint32_t v = 0;
        if (at < 256) {
            const int lane = (at >> 2) & 31, s = at & 3;
            const long long row = row0 + (lane >> 2) + 8 * (at >> 7), col = kt * 128ll + s * 32 + (lane & 3) * 8;
            if (row < a.N && col < a.K)
                for (int b = 0; b < 4; ++b) v |= static_cast<uint32_t>(a.codes[row * a.codes_ld + col / 2 + b]) << (8 * b);
        } else {
            const int groups = 128 / a.group, j = at - 256;
            const long long row = row0 + j / groups, grp = static_cast<long long>(kt) * groups + j % groups;
            if (row < a.N && grp * a.group < a.K) {
                const uint16_t* const s = reinterpret_cast<const uint16_t*>(a.scales) + row * a.scales_ld + grp * 2;
                v = static_cast<uint32_t>(s[0]) | static_cast<uint32_t>(s[1]) << 16;
            }
        }
        reinterpret_cast<uint32_t*>(a.packed)[i] = v;
    }
}

template <bool kBf16, int kGroups, int W, int T, int NR>
cudaError_t go_w4(const W4Args& a, cudaStream_t stream) {
    const auto kern = w4_linear_kernel<kBf16, kGroups, W, T, NR>;
    const int smem = (W + a.parts) * 16 * T * 8 * NR * 4;
    const cudaError_t e = set_max_smem_once(kern, smem);
    if (e != cudaSuccess) return e;
    const int tiles = (a.p.N - 1) / 16 + 1;
    const dim3 grid(static_cast<unsigned>(a.parts * ((tiles + T - 1) / T)), static_cast<unsigned>((a.p.M + 8 * NR - 1) / (8 * NR)));
    return launch_dependent_cluster(kern, grid, dim3(W * 32), smem, stream, dim3(a.parts), a);
}

template <bool kBf16, int kGroups>
cudaError_t pick_w4(W4Args a, cudaStream_t stream) {
    const int tiles = (a.p.N - 1) / 16 + 1;
    auto parts = [&](int w, int t) {
        int n = 1;
        while (n < kW4MaxParts && (tiles + t - 1) / t * n * 2 <= 4 * sm_count() && a.k_tiles >= 2 * n * w) n *= 2;
        return n;
    };
    a.parts = parts(8, 2);
    if (a.p.M <= 8) return go_w4<kBf16, kGroups, 8, 2, 1>(a, stream);
    if (a.p.M <= 16) return go_w4<kBf16, kGroups, 8, 2, 2>(a, stream);
    if (a.p.M <= 32) return go_w4<kBf16, kGroups, 8, 2, 4>(a, stream);
    return go_w4<kBf16, kGroups, 8, 1, 8>(a, stream);
}

}  // namespace

cudaError_t launch_w4_linear(const GemmProblem& p, const void* x, long long ldx, const void* w, int group, bool bf16, cudaStream_t stream) {
    W4Args a;
    a.p = p;
    a.x = reinterpret_cast<const uint16_t*>(x);
    a.w = reinterpret_cast<const uint8_t*>(w);
    a.ldx = ldx;
    a.k_tiles = (p.K - 1) / 128 + 1;
    a.parts = 1;
    auto go = [&](auto b) {
        constexpr bool kB = decltype(b)::value;
        return group == 32 ? pick_w4<kB, 4>(a, stream) : group == 64 ? pick_w4<kB, 2>(a, stream) : pick_w4<kB, 1>(a, stream);
    };
    return bf16 ? go(std::true_type{}) : go(std::false_type{});
}

cudaError_t launch_w4_pack(const W4PackArgs& a, cudaStream_t stream) {
    const long long words = static_cast<long long>((a.N - 1) / 16 + 1) * a.k_tiles * (256 + 16 * (128 / a.group));
    const long long ctas = (words + 255) / 256, most = 16ll * sm_count();
    return launch_dependent(w4_pack_kernel, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(256), 0, stream, a);
}

}  // namespace bdattn
