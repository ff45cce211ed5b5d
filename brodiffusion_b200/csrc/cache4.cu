// New rows of K and V into a cache of 4-bit groups, and rows of it back to 16 bits.
//   group of a head's row:  low = min x,  step = (max x - min x) / 15 rounded to the storage type,
//                           u = round((x - low) / step) in 0..15 (0 where step is 0),  value low + step u
// A group with a value that is not finite has step and low NaN.  The quotients are IEEE ones, so that the same row has the same
// codes wherever it is worked out.
//
// A head's row is HD / 2 bytes of codes and a (step, low) pair for each group.  Its codes lie in the order in which the attention
// kernel's lanes want them (S = HD / 32):
//   K: the word of columns 32 s + 8 q + 0..7 is word q S + s       (q < 4: lanes of a key, a load of S words each)
//   V: the half word of columns 32 s + 4 g + 0..3 is half g S + s  (g < 8: lanes of a column block)
// Both kernels move bytes: a lane has four columns, so that a row of 128 columns is a warp's 256 bytes, and four
// rows of heads are on their way at once.
#include "four_bit.cuh"
#include "sdpa_window.cuh"

namespace bdattn {
namespace {

constexpr int kCacheItems = 4;      // rows of heads in flight to a lane

// One row of one head of K (0) or V (1): where it is in the cache and in the 16-bit tensor.
struct CacheItem {
    bool on;
    int kv, pos;
    const uint16_t* x;
    long long codes, scales;
};
__device__ __forceinline__ CacheItem cache_item(const Cache4RowsArgs& a, long long item) {
    CacheItem r;
    r.on = item < a.items;
    if (!r.on) item = 0;
    r.kv = static_cast<int>(item & 1);
    const long long row = (item >> 1) / a.c.kv_heads;
    const int head = static_cast<int>((item >> 1) - row * a.c.kv_heads), b = static_cast<int>(row / a.n_rows), i = static_cast<int>(row - static_cast<long long>(b) * a.n_rows);
    r.pos = window_keys(a.kv_len, b, a.c.rows) - a.n_rows + i;
    r.x = reinterpret_cast<const uint16_t*>(r.kv ? a.v : a.k) + b * (r.kv ? a.v_bs : a.k_bs) + i * (r.kv ? a.v_ld : a.k_ld) + head * static_cast<long long>(a.c.head_dim);
    r.codes = b * a.c.codes_bs + head * a.c.codes_hs + static_cast<long long>(r.pos) * (a.c.head_dim / 2);
    r.scales = b * a.c.scales_bs + head * a.c.scales_hs + static_cast<long long>(r.pos) * (2 * a.c.head_dim / a.c.group);
    return r;
}
// The half word of this lane's four columns 4 i .. 4 i + 3 in a row.
__device__ __forceinline__ int half_of(int i, int kv, int S) {
    const int s = i >> 3, g = i & 7;
    return kv ? g * S + s : ((g >> 1) * S + s) * 2 + (g & 1);
}

template <bool kBf16>
__global__ void __launch_bounds__(256) cache4_append_kernel(const Cache4RowsArgs a) {
    if (gridDim.x <= 148) dependents_may_launch();
    wait_for_prior_grid();
    const int lanes = a.c.head_dim / 4, i = threadIdx.x % lanes, per = 256 / lanes, team = a.c.group / 4;
    const int half_k = half_of(i, 0, a.c.head_dim / 32), half_v = half_of(i, 1, a.c.head_dim / 32);
    // (lanes that belong together are in one warp and take the same turns)
    for (long long base = static_cast<long long>(blockIdx.x) * per * kCacheItems; base < a.items; base += static_cast<long long>(gridDim.x) * per * kCacheItems) {
        uint2 x[kCacheItems];
        CacheItem it[kCacheItems];
#pragma unroll
        for (int n = 0; n < kCacheItems; ++n) {
            it[n] = cache_item(a, base + n * per + threadIdx.x / lanes);
            x[n] = load8_once(it[n].x + 4 * i);
        }
#pragma unroll
        for (int n = 0; n < kCacheItems; ++n) {
            const float2 f0 = layer_pair<kBf16>(x[n].x), f1 = layer_pair<kBf16>(x[n].y);
            const float f[4] = {f0.x, f0.y, f1.x, f1.y};
            float lo = fminf(fminf(f[0], f[1]), fminf(f[2], f[3])), hi = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
            // (minimum and maximum leave NaN out; the sum of |x| does not, nor an infinity)
            bool odd = !(fabsf(f[0]) + fabsf(f[1]) + fabsf(f[2]) + fabsf(f[3]) <= FLT_MAX);
            if (odd) odd = !(fabsf(f[0]) <= FLT_MAX && fabsf(f[1]) <= FLT_MAX && fabsf(f[2]) <= FLT_MAX && fabsf(f[3]) <= FLT_MAX);
            for (int o = 1; o < team; o *= 2) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            const uint32_t odds = __ballot_sync(0xffffffffu, odd);
            const uint32_t mine = (team == 32 ? 0xffffffffu : (1u << team) - 1u) << ((threadIdx.x & 31) & ~(team - 1));
            uint32_t pair = pack2<kBf16>(__fdiv_rn(hi - lo, 15.0f), lo);
            float step = layer_pair<kBf16>(pair).x;
            if ((odds & mine) != 0 || !(step <= FLT_MAX)) {
                pair = kBf16 ? 0x7fc07fc0u : 0x7e007e00u;
                step = 0.0f;
            }
            uint32_t codes = 0;
            if (step > 0.0f) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float u = fminf(rintf(__fdiv_rn(f[e] - lo, step)), 15.0f);
                    codes |= static_cast<uint32_t>(u) << (4 * e);
                }
            }
            // (a place outside the cache is not written)
            if (it[n].on && it[n].pos >= 0 && it[n].pos < a.c.rows) {
                reinterpret_cast<uint16_t*>((it[n].kv ? a.c.v_codes : a.c.k_codes) + it[n].codes)[it[n].kv ? half_v : half_k] = static_cast<uint16_t>(codes);
                if (i % team == 0)
                    reinterpret_cast<uint32_t*>((it[n].kv ? a.c.v_scales : a.c.k_scales) + it[n].scales)[i / team] = pair;
            }
        }
    }
}

template <bool kBf16>
__global__ void __launch_bounds__(256) cache4_read_kernel(const Cache4RowsArgs a) {
    if (gridDim.x <= 148) dependents_may_launch();
    wait_for_prior_grid();
    const int lanes = a.c.head_dim / 4, i = threadIdx.x % lanes, per = 256 / lanes, team = a.c.group / 4;
    const int half_k = half_of(i, 0, a.c.head_dim / 32), half_v = half_of(i, 1, a.c.head_dim / 32);
    for (long long base = static_cast<long long>(blockIdx.x) * per * kCacheItems; base < a.items; base += static_cast<long long>(gridDim.x) * per * kCacheItems) {
        uint32_t codes[kCacheItems], pair[kCacheItems];
        CacheItem it[kCacheItems];
#pragma unroll
        for (int n = 0; n < kCacheItems; ++n) {
            it[n] = cache_item(a, base + n * per + threadIdx.x / lanes);
            codes[n] = pair[n] = 0;              // (zeros from outside the cache)
            if (it[n].on && it[n].pos >= 0 && it[n].pos < a.c.rows) {
                uint16_t c;
                asm volatile("ld.global.u16 %0, [%1];" : "=h"(c) : "l"(reinterpret_cast<const uint16_t*>((it[n].kv ? a.c.v_codes : a.c.k_codes) + it[n].codes) + (it[n].kv ? half_v : half_k)));
                codes[n] = c;
                pair[n] = load4_once(reinterpret_cast<const uint32_t*>((it[n].kv ? a.c.v_scales : a.c.k_scales) + it[n].scales) + i / team);
            }
        }
#pragma unroll
        for (int n = 0; n < kCacheItems; ++n) {
            const float2 s = layer_pair<kBf16>(pair[n]);
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (the rounded step may take the largest value past the type's range; NaN stays)
                const float v = fmaf(s.x, static_cast<float>((codes[n] >> (4 * e)) & 15u), s.y), most = kBf16 ? 0x1.fep127f : 65504.0f;
                f[e] = v > most ? most : v < -most ? -most : v;
            }
            if (it[n].on) *reinterpret_cast<uint2*>(const_cast<uint16_t*>(it[n].x) + 4 * i) = make_uint2(pack2<kBf16>(f[0], f[1]), pack2<kBf16>(f[2], f[3]));
        }
    }
}

template <class Kernel>
cudaError_t launch_rows(Kernel kern, const Cache4RowsArgs& a, cudaStream_t stream) {
    const long long per = 256 / (a.c.head_dim / 4) * kCacheItems, ctas = (a.items + per - 1) / per, most = 8ll * sm_count();
    return launch_dependent(kern, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(256), 0, stream, a);
}

}  // namespace

cudaError_t launch_cache4_append(const Cache4RowsArgs& a, bool bf16, cudaStream_t stream) {
    return launch_rows(bf16 ? cache4_append_kernel<true> : cache4_append_kernel<false>, a, stream);
}
cudaError_t launch_cache4_read(const Cache4RowsArgs& a, bool bf16, cudaStream_t stream) {
    return launch_rows(bf16 ? cache4_read_kernel<true> : cache4_read_kernel<false>, a, stream);
}

}  // namespace bdattn
