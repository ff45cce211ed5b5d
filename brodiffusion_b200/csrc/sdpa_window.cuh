// Causal attention with a sliding window and visible first keys (sinks): the rule, and one
// query row of it in plain FP32 arithmetic.
//   batch item b has n = kv_len[b] keys (all Lk without kv_len); query i of Lq sits at position P = n - Lq + i;
//   key j is visible iff j <= P, (window == 0 or j > P - window or j < sinks) and key_mask[j] != 0.
// A row without a visible key gives zeros.
#pragma once

#include <cfloat>
#include <cuda_fp16.h>

#include "sdpa_internal.h"
#include "tc05.cuh"

namespace bdattn {

// Keys of batch item b.  The lengths lie in device memory, where the host cannot check them: one outside
// [0, Lk] counts as the nearer end.  (Neither they nor the key mask are read through the read-only path: the kernel before
// this one may write them.)
__device__ __forceinline__ int window_keys(const int* kv_len, int batch, int lk) {
    if (kv_len == nullptr) return lk;
    int n;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(n) : "l"(kv_len + batch));
    return max(0, min(lk, n));
}

// What queries at positions [first, last] see of n keys, but for the key mask: keys [0, sink_end) and
// [win_begin, win_end), which do not overlap (one range where they meet).
struct WindowSpan {
    int sink_end, win_begin, win_end;
};
__host__ __device__ __forceinline__ WindowSpan window_span(int first, int last, int window, int sinks) {
    WindowSpan s;
    s.win_end = last + 1 > 0 ? last + 1 : 0;
    s.win_begin = window > 0 && first >= window ? first - window + 1 : 0;
    s.sink_end = sinks < s.win_end ? sinks : s.win_end;
    if (s.win_begin <= s.sink_end) {
        s.win_begin = 0;
        s.sink_end = 0;
    }
    return s;
}

template <bool kBf16>
__device__ __forceinline__ float2 window_pair(const void* base, long long i) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(base) + i);
    if constexpr (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Output row i (of the concatenated query segments) of one head, by a whole warp; head_dim at most 256.
// The lanes have a key each for the scores of 32 keys and a few columns each for their share of the output.
// q_s: 1 KB of the warp's own shared memory.  Only visible keys are read, so that nothing a masked
// place holds, infinities and NaN included, reaches the row.
template <bool kBf16>
__device__ __noinline__ void window_row(const SdpaWindowArgs& a, int batch, int head, int i, float* q_s, int lane) {
    const int hd = a.head_dim, kv_head = head / a.kv_group;
    const int lk = a.kv_rows[0] + a.kv_rows[1], lq = a.q_rows[0] + a.q_rows[1];
    const int pos = window_keys(a.kv_len, batch, lk) - lq + i;
    const int qs = i >= a.q_rows[0] ? 1 : 0, qi = i - (qs ? a.q_rows[0] : 0);
    const WindowSpan span = window_span(pos, pos, a.window, a.sinks);
    const long long q_at = batch * a.q_bs[qs] + qi * a.q_ld[qs] + static_cast<long long>(head) * hd;
    __syncwarp();
    for (int c = 2 * lane; c < hd; c += 64) {
        const float2 q = window_pair<kBf16>(a.q[qs], q_at + c);
        q_s[c] = q.x;
        q_s[c + 1] = q.y;
    }
    __syncwarp();
    const float sl2 = a.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.0f;
    float acc[4][2] = {};
    for (int part = 0; part < 2; ++part) {
        const int begin = part ? span.win_begin : 0, end = part ? span.win_end : span.sink_end;
        for (int j0 = begin; j0 < end; j0 += 32) {
            const int j = j0 + lane;
            const bool on = j < end && (a.key_mask == nullptr || a.key_mask[j] != 0.0f);
            const uint32_t seen = __ballot_sync(0xffffffffu, on);
            if (seen == 0) continue;
            float s = -INFINITY;
            if (on) {
                const int ks = j >= a.kv_rows[0] ? 1 : 0, kj = j - (ks ? a.kv_rows[0] : 0);
                const long long at = batch * a.k_bs[ks] + kj * a.k_ld[ks] + static_cast<long long>(kv_head) * hd;
                float d0 = 0.0f, d1 = 0.0f;
                for (int c = 0; c < hd; c += 8) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float2 k = window_pair<kBf16>(a.k[ks], at + c + e);
                        d0 = fmaf(q_s[c + e], k.x, d0);
                        d1 = fmaf(q_s[c + e + 1], k.y, d1);
                    }
                }
                s = (d0 + d1) * sl2;
            }
            float top = s;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float m_new = fmaxf(m, top);
            const float ref = m_new == -INFINITY ? 0.0f : m_new;      // (all scores of minus infinity: weights of zero)
            const float alpha = m == -INFINITY ? 0.0f : exp2f(m - ref);
            const float p = on ? exp2f(s - ref) : 0.0f;
            m = m_new;
            l = l * alpha + p;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                acc[t][0] *= alpha;
                acc[t][1] *= alpha;
            }
            for (uint32_t left = seen; left != 0; left &= left - 1) {
                const int b = __ffs(left) - 1, jj = j0 + b;
                const float pj = __shfl_sync(0xffffffffu, p, b);
                const int vs = jj >= a.kv_rows[0] ? 1 : 0, vj = jj - (vs ? a.kv_rows[0] : 0);
                const long long at = batch * a.v_bs[vs] + vj * a.v_ld[vs] + static_cast<long long>(kv_head) * hd;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int c = 2 * lane + 64 * t;
                    if (c < hd) {
                        const float2 v = window_pair<kBf16>(a.v[vs], at + c);
                        acc[t][0] = fmaf(pj, v.x, acc[t][0]);
                        acc[t][1] = fmaf(pj, v.y, acc[t][1]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    // (a sum that is NaN stays: the row is NaN)
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const long long o_at = batch * a.o_bs[qs] + qi * a.o_ld[qs] + static_cast<long long>(head) * hd;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int c = 2 * lane + 64 * t;
        if (c < hd)
            *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.o[qs]) + o_at + c) =
                pack2<kBf16>(acc[t][0] * inv, acc[t][1] * inv);
    }
    __syncwarp();
}

}  // namespace bdattn
