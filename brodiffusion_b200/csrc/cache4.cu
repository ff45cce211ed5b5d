// New rows of K and V into a cache of 4-bit groups, and rows of it back to 16 bits.
//   group of a head's row:  low = min x,  step = (max x - min x) / 15 rounded to the storage type,
//                           u = round((x - low) / step) in 0..15 (0 where step is 0),  value low + step u
// A group with a value that is not finite has step and low NaN.  The quotients are rounded correctly, so that the same row has the
// same codes wherever it is worked out (values of 16 bits lie on the border between two codes every few hundred times).
//
// A head's row is HD / 2 bytes of codes and a (step, low) pair for each group.  Its codes lie in the order in which the attention
// kernel's lanes want them (S = HD / 32):
//   K: the word of columns 32 s + 8 q + 0..7 is word q S + s       (q < 4: lanes of a key, a load of S words each)
//   V: the half word of columns 32 s + 4 g + 0..3 is half g S + s  (g < 8: lanes of a column block)
// Both kernels move bytes.  A lane has eight columns, so that a warp has two rows of 128 columns (four of 64) of a head, and kCacheTurns
// such at once: reads of whole rows, writes that lie behind one another.
#include "four_bit.cuh"
#include "sdpa_window.cuh"

namespace bdattn {
namespace {

constexpr int kCacheTurns = 4;

// A lane's part of a call: columns 8 i .. 8 i + 7 of row `row` + turn * kRows of K or V of a head.
template <int HD, int kGroup>
struct CacheLane {
    static constexpr int kLanes = HD / 8, kRows = 32 / kLanes, S = HD / 32, kPairs = HD / kGroup;
    int i, row, place0;
    uint16_t* x;
    long long ld;
    uint8_t* codes;
    uint32_t* pairs;
    bool v;
    __device__ __forceinline__ explicit CacheLane(const Cache4RowsArgs& a) {
        const int lane = threadIdx.x & 31, head = blockIdx.y >> 1, b = blockIdx.z;
        v = (blockIdx.y & 1) != 0;
        i = lane % kLanes;
        row = (static_cast<int>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kRows * kCacheTurns + lane / kLanes;
        place0 = window_keys(a.kv_len, b, a.c.rows) - a.n_rows;
        ld = v ? a.v_ld : a.k_ld;
        x = reinterpret_cast<uint16_t*>(const_cast<void*>(v ? a.v : a.k)) + b * (v ? a.v_bs : a.k_bs) + static_cast<long long>(head) * HD + 8 * i;
        // (this lane's word of K, or its first half word of V, is at the same place in every row)
        codes = (v ? a.c.v_codes : a.c.k_codes) + b * a.c.codes_bs + head * a.c.codes_hs + (v ? (2 * (i & 3) * S + (i >> 2)) * 2 : ((i & 3) * S + (i >> 2)) * 4);
        pairs = reinterpret_cast<uint32_t*>((v ? a.c.v_scales : a.c.k_scales) + b * a.c.scales_bs + head * a.c.scales_hs) + 8 * i / kGroup;
    }
};

// The smaller, or larger, of two pairs of values; NaN stays.
template <bool kBf16, bool kMax>
__device__ __forceinline__ uint32_t extreme2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (kBf16 && kMax) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else if constexpr (kBf16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else if constexpr (kMax) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Two FP32 values to an instruction, of the kind that keeps what is below the normal range (the library is compiled to flush it).
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{.reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x;}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
// a * b + c
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 z, x, y, z; mov.b64 {%0, %1}, z;}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// a / b rounded to the nearest, by Markstein's correction of a * (1 / b); minus_b is -b, inv is 1 / b rounded to the nearest, the
// quotients neither huge nor tiny.  (What is left of a is below the normal range where b is below 2^-102.)
__device__ __forceinline__ float2 quotients(float2 a, float minus_b, float inv) {
    const float2 i = make_float2(inv, inv), q = fma2(a, i, make_float2(0.0f, 0.0f));
    return fma2(fma2(q, make_float2(minus_b, minus_b), a), i, q);
}

template <bool kBf16, int HD, int kGroup>
__global__ void __launch_bounds__(256) cache4_append_kernel(const Cache4RowsArgs a) {
    dependents_may_launch();
    wait_for_prior_grid();
    using Lane = CacheLane<HD, kGroup>;
    const Lane at(a);
    constexpr int kTeam = kGroup / 8;
    uint4 x[kCacheTurns];
#pragma unroll
    for (int n = 0; n < kCacheTurns; ++n) {
        const int row = at.row + n * Lane::kRows;
        x[n] = make_uint4(0u, 0u, 0u, 0u);
        if (row < a.n_rows) x[n] = load16_once(at.x + row * at.ld);
    }
#pragma unroll
    for (int n = 0; n < kCacheTurns; ++n) {
        if (at.row - static_cast<int>(threadIdx.x & 31) / Lane::kLanes + n * Lane::kRows >= a.n_rows) break;          // (of the whole warp)
        const int row = at.row + n * Lane::kRows, place = at.place0 + row;
        uint32_t lo2 = extreme2<kBf16, false>(extreme2<kBf16, false>(x[n].x, x[n].y), extreme2<kBf16, false>(x[n].z, x[n].w));
        uint32_t hi2 = extreme2<kBf16, true>(extreme2<kBf16, true>(x[n].x, x[n].y), extreme2<kBf16, true>(x[n].z, x[n].w));
#pragma unroll
        for (int o = 1; o < kTeam; o *= 2) {
            lo2 = extreme2<kBf16, false>(lo2, __shfl_xor_sync(0xffffffffu, lo2, o));
            hi2 = extreme2<kBf16, true>(hi2, __shfl_xor_sync(0xffffffffu, hi2, o));
        }
        const float low = layer_pair<kBf16>(extreme2<kBf16, false>(lo2, lo2 >> 16)).x, high = layer_pair<kBf16>(extreme2<kBf16, true>(hi2, hi2 >> 16)).x;
        const float2 minus = make_float2(-1.0f, -1.0f), low2 = make_float2(low, low);
        uint32_t pair = pack2<kBf16>(quotients(fma2(low2, minus, make_float2(high, high)), -15.0f, 1.0f / 15.0f).x, low);
        float step = layer_pair<kBf16>(pair).x;
        // (a value that is not finite has made one of both so)
        if (!(step <= FLT_MAX && fabsf(low) <= FLT_MAX)) {
            pair = kBf16 ? 0x7fc07fc0u : 0x7e007e00u;
            step = 0.0f;
        }
        // 1.5 * 2^23 more than a quotient is the nearest integer in the low bits; eight of them are added up shifted, and what the
        // rest of their bits comes to is taken off
        constexpr float kRound = 12582912.0f;
        constexpr uint32_t kRest = 0x4b400000u * 0x11111111u;
        uint32_t codes = 0;
        if (step > 0.0f) {
            const float inv = __frcp_rn(step);
            const uint32_t w[4] = {x[n].x, x[n].y, x[n].z, x[n].w};
#pragma unroll
            for (int e = 3; e >= 0; --e) {
                float2 u = quotients(fma2(low2, minus, layer_pair<kBf16>(w[e])), -step, inv);
                // (only steps below FP16's smallest normal are so much smaller than a fifteenth of the range that a code could be 16)
                if (!kBf16) u = make_float2(fminf(u.x, 15.0f), fminf(u.y, 15.0f));
                u = add2(u, make_float2(kRound, kRound));
                codes = codes * 16 + __float_as_uint(u.y);
                codes = codes * 16 + __float_as_uint(u.x);
            }
            codes -= kRest;
        }
        // (a place outside the cache is not written)
        if (row < a.n_rows && place >= 0 && place < a.c.rows) {
            uint8_t* const p = at.codes + static_cast<long long>(place) * (HD / 2);
            if (at.v) {
                *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(codes);
                *reinterpret_cast<uint16_t*>(p + 2 * Lane::S) = static_cast<uint16_t>(codes >> 16);
            } else {
                *reinterpret_cast<uint32_t*>(p) = codes;
            }
            if (at.i % kTeam == 0) at.pairs[static_cast<long long>(place) * Lane::kPairs] = pair;
        }
    }
}

template <bool kBf16, int HD, int kGroup>
__global__ void __launch_bounds__(256) cache4_read_kernel(const Cache4RowsArgs a) {
    dependents_may_launch();
    wait_for_prior_grid();
    using Lane = CacheLane<HD, kGroup>;
    const Lane at(a);
    uint32_t codes[kCacheTurns], pair[kCacheTurns];
#pragma unroll
    for (int n = 0; n < kCacheTurns; ++n) {
        const int row = at.row + n * Lane::kRows, place = at.place0 + row;
        codes[n] = pair[n] = 0;              // (zeros from outside the cache)
        if (row < a.n_rows && place >= 0 && place < a.c.rows) {
            const uint8_t* const p = at.codes + static_cast<long long>(place) * (HD / 2);
            if (at.v) {
                uint16_t c0, c1;
                asm volatile("ld.global.u16 %0, [%1];" : "=h"(c0) : "l"(p));
                asm volatile("ld.global.u16 %0, [%1];" : "=h"(c1) : "l"(p + 2 * Lane::S));
                codes[n] = static_cast<uint32_t>(c0) | static_cast<uint32_t>(c1) << 16;
            } else {
                asm volatile("ld.global.u32 %0, [%1];" : "=r"(codes[n]) : "l"(p));
            }
            asm volatile("ld.global.u32 %0, [%1];" : "=r"(pair[n]) : "l"(at.pairs + static_cast<long long>(place) * Lane::kPairs));
        }
    }
#pragma unroll
    for (int n = 0; n < kCacheTurns; ++n) {
        const int row = at.row + n * Lane::kRows;
        if (row >= a.n_rows) break;
        const float2 s = layer_pair<kBf16>(pair[n]);
        uint32_t r[4], out[4];
        // low + step u for the pairs (j, j + 4) of the word, rounded once by a fused multiplication and addition in 16 bits: a code behind
        // the bits of 128 (1024) is that much more than itself
        const uint32_t step2 = __byte_perm(pair[n], 0, 0x1010), low2 = __byte_perm(pair[n], 0, 0x3232);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t u = ((codes[n] >> (4 * e)) & 0x000f000fu) | (kBf16 ? 0x43004300u : 0x64006400u);
            if constexpr (kBf16) asm("{.reg .b32 t; sub.rn.bf16x2 t, %1, %2; fma.rn.bf16x2 %0, t, %3, %4;}" : "=r"(r[e]) : "r"(u), "r"(0x43004300u), "r"(step2), "r"(low2));
            else asm("{.reg .b32 t; sub.rn.f16x2 t, %1, %2; fma.rn.f16x2 %0, t, %3, %4;}" : "=r"(r[e]) : "r"(u), "r"(0x64006400u), "r"(step2), "r"(low2));
        }
        out[0] = __byte_perm(r[0], r[1], 0x5410);
        out[1] = __byte_perm(r[2], r[3], 0x5410);
        out[2] = __byte_perm(r[0], r[1], 0x7632);
        out[3] = __byte_perm(r[2], r[3], 0x7632);
        // (the rounded step may take the largest value past the type's range; NaN stays)
        const float most = kBf16 ? 0x1.fep127f : 65504.0f;
        if (fabsf(fmaf(s.x, 15.0f, s.y)) > most) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float f[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float v = fmaf(s.x, static_cast<float>((codes[n] >> (8 * e + 4 * h)) & 15u), s.y);
                    f[h] = v > most ? most : v < -most ? -most : v;
                }
                out[e] = pack2<kBf16>(f[0], f[1]);
            }
        }
        *reinterpret_cast<uint4*>(at.x + row * at.ld) = make_uint4(out[0], out[1], out[2], out[3]);
    }
}

template <class Kernel>
cudaError_t launch_rows(Kernel kern, const Cache4RowsArgs& a, cudaStream_t stream) {
    const int per = 256 / a.c.head_dim * kCacheTurns;          // rows of a warp
    const int warps = (a.n_rows - 1) / per + 1, w = warps < 8 ? warps : 8;
    return launch_dependent(kern, dim3(static_cast<unsigned>((warps - 1) / w + 1), static_cast<unsigned>(2 * a.c.kv_heads), static_cast<unsigned>(a.batch)),
                            dim3(32 * w), 0, stream, a);
}
template <bool kBf16, int HD, int kGroup>
cudaError_t append_or_read(const Cache4RowsArgs& a, bool append, cudaStream_t stream) {
    return append ? launch_rows(cache4_append_kernel<kBf16, HD, kGroup>, a, stream) : launch_rows(cache4_read_kernel<kBf16, HD, kGroup>, a, stream);
}
template <bool kBf16>
cudaError_t pick_rows(const Cache4RowsArgs& a, bool append, cudaStream_t stream) {
    const int g = a.c.group;
    if (a.c.head_dim == 64) return g == 32 ? append_or_read<kBf16, 64, 32>(a, append, stream) : append_or_read<kBf16, 64, 64>(a, append, stream);
    return g == 32 ? append_or_read<kBf16, 128, 32>(a, append, stream) : g == 64 ? append_or_read<kBf16, 128, 64>(a, append, stream)
                                                                                 : append_or_read<kBf16, 128, 128>(a, append, stream);
}

}  // namespace

cudaError_t launch_cache4_append(const Cache4RowsArgs& a, bool bf16, cudaStream_t stream) {
    return bf16 ? pick_rows<true>(a, true, stream) : pick_rows<false>(a, true, stream);
}
cudaError_t launch_cache4_read(const Cache4RowsArgs& a, bool bf16, cudaStream_t stream) {
    return bf16 ? pick_rows<true>(a, false, stream) : pick_rows<false>(a, false, stream);
}

}  // namespace bdattn
