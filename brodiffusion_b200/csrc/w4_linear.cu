// A layer's product with 4-bit weights:
//   C[m, n] = residual + gate * act(sum_k X[m, k] W[n, k] + bias),  W[n, k] = low[n, g] + step[n, g] u[n, k],  g = k / group
// as  sum_g step[n, g] (sum_{k in g} X u) + low[n, g] (sum_{k in g} X):  the codes u enter mma.sync as exact small integers
// (four_bit.cuh), the sums of X come from the same instruction with ones for weights, and step and low are applied to
// FP32 sums of a group, so that nothing is rounded but X, W as they are given and the result.
//
// What a call of few rows costs is reading W once, 4 + 32 / group bits a value.  Packed weights (w4_pack_kernel) are tiles of 16 rows x 128
// columns in the order in which a warp's lanes want them: 16 bytes a lane for each eight of its rows, the steps and
// lows behind them, K tiles of a row tile one behind the other.
#include "four_bit.cuh"

namespace bdattn {
namespace {

constexpr int kW4MaxParts = 8;

__host__ __device__ constexpr int w4_tile_bytes(int group) { return 1024 + 16 * (128 / group) * 4; }

// BF16 pairs times a power of two.
__device__ __forceinline__ uint32_t times_pow2(uint32_t v, uint32_t by) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(by));
    return r;
}

struct W4Args {
    GemmProblem p;          // M, N, K, C, bias, act, gate, residual
    const uint16_t* x;
    const uint8_t* w;
    long long ldx;
    int k_tiles, parts;     // tiles of 128 columns; CTAs of a cluster, which share them
};

// kGroups: groups of a tile's 128 columns.  W: warps, each with K tiles of its own.  T: row tiles of a CTA.  NR: rows of X in
// eights.  D: K tiles of a warp in flight, with the columns of X that go with them.  kCtas: CTAs of an SM.
template <bool kBf16, int kGroups, int W, int T, int NR, int D, int kCtas>
__global__ void __launch_bounds__(W * 32, kCtas) w4_few_kernel(const __grid_constant__ W4Args a) {
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
        wp[t] = a.w + (static_cast<long long>(min(tile0 + t, n_tiles - 1)) * a.k_tiles + first) * kTile;
    if (a.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    dependents_may_launch();
    // While the kernel before this one ends, the first weights come into the L2.
    if (lane * 128 < kTile) {
#pragma unroll
        for (int i = 0; i < D; ++i) {
#pragma unroll
            for (int t = 0; t < T; ++t)
                if (first + i * step < a.k_tiles) asm volatile("prefetch.global.L2 [%0];" ::"l"(wp[t] + static_cast<long long>(i) * step * kTile + lane * 128));
        }
    }
    wait_for_prior_grid();

    const uint16_t* xp[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) xp[r] = a.x + min(m0 + r * 8 + g, p.M - 1) * a.ldx + q * 8;

    uint4 wv[D][T][2], xv[D][4][NR];
    uint32_t sv[D][T][2][kGroups];
    int next = first;                // the K tile that is fetched next
    auto fetch = [&](int i) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                wv[i][t][h] = load16_once(wp[t] + h * 512 + lane * 16);
                load_words_once<kGroups>(wp[t] + 1024 + (g + 8 * h) * 4 * kGroups, sv[i][t][h]);
            }
            wp[t] += static_cast<long long>(step) * kTile;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int c = next * 128 + s * 32;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                xv[i][s][r] = make_uint4(0u, 0u, 0u, 0u);
                if (c + q * 8 < p.K) xv[i][s][r] = load16(xp[r] + c);
            }
        }
        next += step;
    };
    float y[T][NR][4] = {};
    auto products = [&](int i) {
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) {
            constexpr int kPer = 4 / kGroups;
            // sums of X over the group's columns, in the places of their rows of C: a product with ones, at 2^32 times their size, so
            // that no sum of values below 2^64 is beyond FP32
            float xs[NR][4];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                xs[r][0] = xs[r][1] = xs[r][2] = xs[r][3] = 0.0f;
#pragma unroll
                for (int s = gi * kPer; s < (gi + 1) * kPer; ++s) {
                    uint4& v = xv[i][s][r];
                    if constexpr (kBf16) {
                        // 2^64, and 2^60 where the codes are sixteen times theirs: exact, infinite from |x| = 2^64 on
                        v.x = times_pow2(v.x, 0x5f805f80u);
                        v.y = times_pow2(v.y, 0x5f805f80u);
                        v.z = times_pow2(v.z, 0x5d805d80u);
                        v.w = times_pow2(v.w, 0x5d805d80u);
                    }
                    constexpr uint32_t kOne = kBf16 ? 0x2f802f80u : 0x3c003c00u, kOdd = kBf16 ? 0x31803180u : kOne;
                    mma16<kBf16>(xs[r], kOne, kOne, kOne, kOne, v.x, v.y);
                    mma16<kBf16>(xs[r], kOdd, kOdd, kOdd, kOdd, v.z, v.w);
                }
                if constexpr (kBf16) {
                    xs[r][0] *= 0x1p-32f;
                    xs[r][1] *= 0x1p-32f;
                }
            }
#pragma unroll
            for (int t = 0; t < T; ++t) {
                // (two sums, half as long a chain of products each; FP16: X cannot carry the 1 / 16 of the odd pairs)
                float d[NR][4] = {}, e[NR][4] = {};
#pragma unroll
                for (int s = gi * kPer; s < (gi + 1) * kPer; ++s) {
                    uint32_t u[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4& w = wv[i][t][h];
                        codes8(s == 0 ? w.x : s == 1 ? w.y : s == 2 ? w.z : w.w, u[h]);
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const uint4& v = xv[i][s][r];
                        mma16<kBf16>(d[r], u[0][0], u[1][0], u[0][2], u[1][2], v.x, v.y);
                        mma16<kBf16>(e[r], u[0][1], u[1][1], u[0][3], u[1][3], v.z, v.w);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // (BF16: the codes' units go to the sums, since a step times them may be beyond FP32; that costs up to 3 %)
                    float2 sl = layer_pair<kBf16>(sv[i][t][h][gi]);
                    if (!kBf16) sl.x *= 0x1p24f;
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float f = kBf16 ? (d[r][2 * h + c] + e[r][2 * h + c]) * 0x1p69f : fmaf(e[r][2 * h + c], 0.0625f, d[r][2 * h + c]);
                            y[t][r][2 * h + c] = fmaf(f, sl.x, fmaf(xs[r][c], sl.y, y[t][r][2 * h + c]));
                        }
                    }
                }
            }
        }
    };
#pragma unroll
    for (int i = 0; i < D; ++i)
        if (next < a.k_tiles) fetch(i);
    for (int kt = first; kt < a.k_tiles; kt += D * step) {
#pragma unroll
        for (int i = 0; i < D; ++i) {
            if (kt + i * step < a.k_tiles) {
                products(i);
                if (next < a.k_tiles) fetch(i);
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
                for (int b = 0; b < 4; ++b) {
                    // columns 2 b and 2 b + 1 are the pair 0, 2, 1, 3 of codes8: those of a product lie side by side in X
                    const int pair = (b & 1) * 2 + (b >> 1);
                    const uint32_t two = a.codes[row * a.codes_ld + col / 2 + b];
                    v |= (two & 15u) << (4 * pair) | (two >> 4) << (16 + 4 * pair);
                }
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

// Packed tiles back to rows of 16 bits, a tile to a warp: a lane has the words of rows g and g + 8, so that the four lanes of a row write
// 64 bytes side by side.  low + step u in FP32, rounded once.  Bound by what it writes (10240 x 2560 12.6 us, 5.3 TB/s).
template <bool kBf16, int kGroups>
__global__ void __launch_bounds__(256) w4_unpack_kernel(const W4UnpackArgs a) {
    constexpr int kTile = w4_tile_bytes(128 / kGroups), kPer = 4 / kGroups;
    dependents_may_launch();
    wait_for_prior_grid();
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const long long tiles = static_cast<long long>((a.N - 1) / 16 + 1) * a.k_tiles;
    for (long long t = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); t < tiles; t += 8ll * gridDim.x) {
        const uint8_t* const from = a.packed + t * kTile;
        const int col0 = static_cast<int>(t % a.k_tiles) * 128 + q * 8;
        uint4 wv[2];
        uint32_t sv[2][kGroups];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wv[h] = load16_once(from + h * 512 + lane * 16);
            load_words_once<kGroups>(from + 1024 + (g + 8 * h) * 4 * kGroups, sv[h]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long row = t / a.k_tiles * 16 + g + 8 * h;
            if (row >= a.N) continue;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (col0 + s * 32 >= a.K) continue;
                const uint32_t w = s == 0 ? wv[h].x : s == 1 ? wv[h].y : s == 2 ? wv[h].z : wv[h].w;
                const float2 sl = layer_pair<kBf16>(sv[h][s / kPer]);
                // (NaN stays)
                constexpr float kMost = kBf16 ? 0x1.fep127f : 65504.0f;
                auto value = [&](int nibble) {
                    const float v = fmaf(sl.x, static_cast<float>((w >> (4 * nibble)) & 15u), sl.y);
                    return v > kMost ? kMost : v < -kMost ? -kMost : v;
                };
                // columns 2 b and 2 b + 1 are the nibbles p and p + 4, p = 0, 2, 1, 3
                *reinterpret_cast<uint4*>(a.w + row * a.ld + col0 + s * 32) =
                    make_uint4(pack2<kBf16>(value(0), value(4)), pack2<kBf16>(value(2), value(6)), pack2<kBf16>(value(1), value(5)), pack2<kBf16>(value(3), value(7)));
            }
        }
    }
}

template <bool kBf16, int kGroups, int W, int T, int NR, int D, int kCtas>
cudaError_t go_w4_few(const W4Args& a, cudaStream_t stream) {
    const auto kern = w4_few_kernel<kBf16, kGroups, W, T, NR, D, kCtas>;
    const int smem = (W + a.parts) * 16 * T * 8 * NR * 4;
    const cudaError_t e = set_max_smem_once(kern, smem);
    if (e != cudaSuccess) return e;
    const int tiles = (a.p.N - 1) / 16 + 1;
    const dim3 grid(static_cast<unsigned>(a.parts * ((tiles + T - 1) / T)), static_cast<unsigned>((a.p.M + 8 * NR - 1) / (8 * NR)));
    return launch_dependent_cluster(kern, grid, dim3(W * 32), smem, stream, dim3(a.parts), a);
}

// Which kernel: the one whose CTAs all run at once (n of them to an SM) with the fewest tiles to a warp behind one another, so
// that nearly all of W is on its way at the same time; K over a cluster where that takes it.  Few tiles: a row tile to a CTA, both of a
// warp's K tiles in registers (1368 x 1291, one row 2.3 us, two row tiles to a CTA 2.7; 2560 x 1280 2.5 and 2.7).  More:
// two row tiles to a CTA of eight warps, two or three CTAs to an SM (2560 x 2560 over three CTAs 2.9, over two 3.9, whole 4.1; 10240 x 2560
// whole 5.8, over two 8.3), and of four warps, five CTAs to an SM, for the rest (5120 x 5120 over four 6.0, over two CTAs of eight warps
// 6.8; 20480 x 5120 15.3, 15.6): that is where rows of W are longer than 24 K tiles and the second form finds room for clusters (10240 rows of 2560,
// 2944, 3328, 5120 columns 6.4, 7.0, 8.0, 10.4 us by the first, 6.9, 6.9, 8.0, 9.8 by the second; 13824 rows, which leave it none, 6.5, 7.0, 8.1, 10.7 and
// 8.9, 10.2, 11.4, 15.9).
template <bool kBf16, int kGroups>
cudaError_t pick_w4(W4Args a, cudaStream_t stream) {
    const int sms = sm_count(), tiles = (a.p.N - 1) / 16 + 1, pairs = (tiles + 1) / 2, kt = a.k_tiles;
    // the fewest CTAs to a cluster with which a warp has no more than `most` K tiles, if `ctas` such clusters fit `room` CTAs; or 0
    auto split = [&](long long ctas, long long room, int warps, int most) {
        for (int p = 1; p <= kW4MaxParts && p * ctas <= room; ++p)
            if ((kt - 1) / (warps * p) + 1 <= most) return p;
        return 0;
    };
    // as many as there is room for with two K tiles to a warp
    auto spread = [&](long long ctas, long long room, int warps) {
        int p = 1;
        while (p < kW4MaxParts && p * 2 * ctas <= room && kt >= warps * p * 4) p *= 2;
        return p;
    };
    if (a.p.M <= 8) {
        if ((a.parts = split(tiles, 2ll * sms, 8, 2)) != 0) return go_w4_few<kBf16, kGroups, 8, 1, 1, 2, 2>(a, stream);
        if ((a.parts = split(pairs, 2ll * sms, 8, 1)) != 0 || (a.parts = split(pairs, sms, 8, 2)) != 0)
            return go_w4_few<kBf16, kGroups, 8, 2, 1, 1, 2>(a, stream);
        a.parts = 1;
        if (pairs <= 3 * sms && (kt <= 24 || 2 * pairs > 5 * sms)) return go_w4_few<kBf16, kGroups, 8, 2, 1, 1, 3>(a, stream);
        a.parts = spread(pairs, 5ll * sms, 4);
        return go_w4_few<kBf16, kGroups, 4, 2, 1, 1, 5>(a, stream);
    }
    // More rows: sixteen a pass, which read W from the L2 after the first; the same rules, of all passes' CTAs.  Few tiles as above (13 x 1291 x 1368
    // 3.2 us, 40 rows 4.2, two row tiles to a CTA 5.1).  Else four warps, three CTAs to an SM (16 x 2560 x 10240 over four 9.9, eight warps over three
    // 10.8; 12 x 10240 x 2560 9.1, 11.8; 32 x 5120 x 5120 15.0, 17.5), but eight where several passes' CTAs of them all run at once (48 x 2560 x 10240
    // 19.3, 22.2) or those of four do not (48 x 5120 x 5120 20.8, 24.6).
    const long long passes = (a.p.M - 1) / 16 + 1;
    if ((a.parts = split(tiles * passes, sms, 8, 2)) != 0) return go_w4_few<kBf16, kGroups, 8, 1, 2, 2, 1>(a, stream);
    if ((a.parts = split(tiles * passes, 2ll * sms, 8, 3)) != 0) return go_w4_few<kBf16, kGroups, 8, 1, 2, 1, 2>(a, stream);
    if (passes > 1 && (pairs * passes <= 2ll * sms || pairs * passes > 3ll * sms)) {
        a.parts = spread(pairs * passes, 2ll * sms, 8);
        return go_w4_few<kBf16, kGroups, 8, 2, 2, 1, 2>(a, stream);
    }
    a.parts = spread(pairs * passes, 3ll * sms, 4);
    return go_w4_few<kBf16, kGroups, 4, 2, 2, 1, 3>(a, stream);
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

cudaError_t launch_w4_unpack(const W4UnpackArgs& a, bool bf16, cudaStream_t stream) {
    const long long ctas = (static_cast<long long>((a.N - 1) / 16 + 1) * a.k_tiles + 7) / 8, most = 16ll * sm_count();
    const dim3 grid(static_cast<unsigned>(ctas < most ? ctas : most));
    auto go = [&](auto b) {
        constexpr bool kB = decltype(b)::value;
        return a.group == 32   ? launch_dependent(w4_unpack_kernel<kB, 4>, grid, dim3(256), 0, stream, a)
               : a.group == 64 ? launch_dependent(w4_unpack_kernel<kB, 2>, grid, dim3(256), 0, stream, a)
                               : launch_dependent(w4_unpack_kernel<kB, 1>, grid, dim3(256), 0, stream, a);
    };
    return bf16 ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace bdattn
