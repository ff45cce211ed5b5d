// Causal attention over a cache in 4 bits (cache4.cu), with a sliding window and first keys that stay visible.
//   s_ij = scale * sum_g step_K[j, g] (sum_{c in g} q_ic u_jc) + low_K[j, g] (sum_{c in g} q_ic)
//   o_i  = (sum_j p_ij step_V[j, g] (u_j - 8) + sum_j p_ij (low_V[j, g] + 8 step_V[j, g])) / sum_j p_ij,   p_ij = exp(s_ij - max)
// (with u as it is, both sums would be some ten times the output of many keys, and the roundings of the first in proportion: fp16
// outputs of 8000 keys were off by 5.3e-4, with u - 8 by 2.8e-4, of which 2.1e-4 are the outputs' own).
// The codes enter mma.sync as exact FP16 integers (four_bit.cuh); steps and lows are applied to FP32 scores and to the
// FP32 weights ahead of their one rounding, to FP16.  The query heads that share a K/V head, and the new tokens, are the (eight or
// sixteen) columns of a product whose rows are sixteen keys, or sixteen columns of V.  A warp takes sixteen keys at a time through a
// ring in shared memory of its own (cp.async: straight to registers 285 us of 32 sequences of up to 32768 keys, the ring 257 at the same
// arithmetic) and has a running maximum, sum and accumulator of its own; these meet in shared memory, then in distributed
// shared memory, where every CTA of a head's cluster finishes its share of the rows.
// What a call has to do is read the visible rows once, 4 + 32 / group bits a value.  What bounds it is issue, some 450 instructions to sixteen
// keys of a warp: of 32 sequences of up to 32768 keys (237 us), reading alone took 136 us when the whole took 247, arithmetic alone 244.
#include "four_bit.cuh"
#include "sdpa_window.cuh"

#include <atomic>

namespace bdattn {
namespace {

constexpr int kC4MaxSplit = 16;
constexpr float kC4MostLift = 0x1p126f;

__device__ __forceinline__ uint32_t c4_transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void c4_store_cluster(uint32_t addr, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void c4_store_cluster(uint32_t addr, float2 v) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}
// 2^e for e in [-126, 127], and e of a normal number's power of two
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
__device__ __forceinline__ int exponent(float f) { return static_cast<int>(__float_as_uint(f) >> 23) - 127; }
// a / b, powers of two; 0 below FP32's normal range
__device__ __forceinline__ float pow2_ratio(float a, float b) {
    const int e = exponent(a) - exponent(b);
    return e < -126 ? 0.0f : pow2(min(e, 127));
}

template <int HD, int G, int W, int NR, int D>
struct Cache4Cfg {
    static constexpr int kRows = 8 * NR, kLd = HD + 4, kMergeRows = kRows + kC4MaxSplit - 1;
    static constexpr int kCodes = 16 * HD / 2, kScales = 16 * 4 * G, kStep = 2 * (kCodes + kScales);      // bytes of sixteen keys
    static constexpr int kRing = W * D * kStep, kSums = W * kRows * kLd * 4;                              // (the sums lie in the ring's place)
    static constexpr int kFirst = kRing > kSums ? kRing : kSums;
    static constexpr int kSmem = kFirst + (kMergeRows * (kLd + 2) + W * kRows * (2 + (G > 1 ? G : 0))) * 4;
};

// Global to shared memory, 4, 8 or 16 bytes.
template <int kBytes>
__device__ __forceinline__ void c4_copy(uint32_t dst, const void* src) {
    if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes) : "memory");
}
template <int kWords>
__device__ __forceinline__ void c4_lds(const uint8_t* p, uint32_t (&w)[kWords]) {
    if constexpr (kWords == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (kWords == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// HD: 64 or 128.  G: groups of a row.  W: warps.  NR: query rows in eights.  D: steps of a warp in shared memory.  kCtas: CTAs of an SM.
// kMask: with a key mask (without one, looking for it took 3 % of a call).
template <int HD, int G, bool kBf16, bool kMask, int W, int NR, int D, int kCtas>
__global__ void __launch_bounds__(W * 32, kCtas) sdpa_cache4_kernel(const __grid_constant__ SdpaCache4Args a) {
    using C = Cache4Cfg<HD, G, W, NR, D>;
    constexpr int S = HD / 32, kPer = S / G, kRows = C::kRows;
    extern __shared__ __align__(16) uint8_t c4_smem[];
    float* const o_warp = reinterpret_cast<float*>(c4_smem);                // [W][kRows][kLd], once the rings are done with
    float* const o_cta = reinterpret_cast<float*>(c4_smem + C::kFirst);     // [kMergeRows][kLd]
    float2* const ml_warp = reinterpret_cast<float2*>(o_cta + C::kMergeRows * C::kLd);     // [W][kRows]
    float2* const ml_cta = ml_warp + W * kRows;                             // [kMergeRows]
    float2* const lifts = ml_cta + C::kMergeRows;                           // [W][NR][G][4], pairs of rows (with more than one group)

    const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int split = a.split, part = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int unit = static_cast<int>(blockIdx.x) / split, kv_head = unit / a.row_tiles, row0 = unit % a.row_tiles * kRows;
    const int batch = blockIdx.y, rows = min(kRows, a.lq * a.kv_group - row0);
    // (waited for ahead of the first store into a peer's shared memory: it has to run by then)
    if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    dependents_may_launch();
    wait_for_prior_grid();

    const int n_keys = window_keys(a.kv_len, batch, a.c.rows), first_pos = n_keys - a.lq;      // of query 0
    const int pos_lo = first_pos + row0 / a.kv_group, pos_hi = first_pos + (row0 + rows - 1) / a.kv_group;
    const WindowSpan span = window_span(pos_lo, pos_hi, a.window, a.sinks);
    // steps of sixteen keys: those of the sinks, then those of the window, from the sixteen in which it begins
    const int sink_steps = (span.sink_end + 15) / 16, win0 = span.win_begin & ~15;
    const int steps = sink_steps + (span.win_end > span.win_begin ? (span.win_end - win0 + 15) / 16 : 0);

    // steps of which every query sees all sixteen keys, but for the key mask: of the sinks' those below whole_sinks, of the window's [whole_first, whole_end)
    const int whole_sinks = min(span.sink_end, pos_lo + 1) / 16;
    const int see_all = a.window == 0 || pos_hi < a.window ? 0 : pos_hi - a.window + 1;          // the first key that the last query's window has
    const int whole_first = sink_steps + (max(see_all, span.win_begin) - win0 + 15) / 16;
    const int whole_end = sink_steps + (min(span.win_end, pos_lo + 1) - win0) / 16;

    // The queries in FP16, a power of two from where the largest of a row is in [2^14, 2^15): what that rounds is 2^-35 of
    // the largest.  This lane has row g's columns 32 s + 8 q + 0..7 as the pairs of codes8, those of the odd pairs over 16.
    uint32_t qf[NR][S][4];
    float qs[NR][2], sl2[NR][2];          // row g's sum over group q in two parts of 11 bits; factor of the scores of columns 2 q and 2 q + 1
    int pos[NR][2];
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        const int r = row0 + min(nr * 8 + g, rows - 1), i = r / a.kv_group;
        const uint16_t* const qp = reinterpret_cast<const uint16_t*>(a.q) + batch * a.q_bs + i * a.q_ld +
                                   static_cast<long long>(kv_head * a.kv_group + r % a.kv_group) * HD + q * 8;
        float f[S][8], top = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const uint4 v = load16(qp + s * 32);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 p = layer_pair<kBf16>(w[e]);
                f[s][2 * e] = p.x;
                f[s][2 * e + 1] = p.y;
                top = fmaxf(top, fmaxf(fabsf(p.x), fabsf(p.y)));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // (zeros, and rows that are not finite, stay as they are)
        const int up = top > 0.0f && top <= FLT_MAX ? min(100, 141 - static_cast<int>(__float_as_uint(top) >> 23)) : 0;
        const float lift = pow2(up), lift16 = pow2(up - 4);
        float sum[G];
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
            sum[gi] = 0.0f;
#pragma unroll
            for (int s = gi * kPer; s < (gi + 1) * kPer; ++s) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[gi] += f[s][e] * lift;
            }
            sum[gi] += __shfl_xor_sync(0xffffffffu, sum[gi], 1);
            sum[gi] += __shfl_xor_sync(0xffffffffu, sum[gi], 2);
            // the codes count 2^-24 each
            sum[gi] *= 0x1p-24f;
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float l = (e & 1) ? lift16 : lift;
                qf[nr][s][e] = pack2<false>(f[s][e] * l, f[s][e + 4] * l);
            }
        }
        float mine = 0.0f;
#pragma unroll
        for (int gi = 0; gi < G; ++gi) mine = q == gi ? sum[gi] : mine;
        qs[nr][0] = __uint_as_float(__float_as_uint(mine) & 0xffffe000u);
        qs[nr][1] = mine - qs[nr][0];
        // (kept normal and finite: times the infinities and zeros that a difference of scores may be, it has to stay what it is)
        const float down = fminf(fmaxf(pow2(-up) * (0x1p24f * a.scale * 1.4426950408889634f), FLT_MIN), FLT_MAX);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int from = (2 * q + h) * 4;
            sl2[nr][h] = __shfl_sync(0xffffffffu, down, from);
            pos[nr][h] = first_pos + (row0 + min(nr * 8 + 2 * q + h, rows - 1)) / a.kv_group;
        }
    }

    // A step's keys come as they lie, sixteen bytes of codes and a key's pairs to a lane, into this warp's own part of shared
    // memory; the pieces of V's rows change places so that the four keys that a quarter of a warp reads at once lie in different banks.
    const uint8_t* const kc_base = a.c.k_codes + batch * a.c.codes_bs + kv_head * a.c.codes_hs;
    const uint8_t* const vc_base = a.c.v_codes + batch * a.c.codes_bs + kv_head * a.c.codes_hs;
    const uint16_t* const sc_base = (lane < 16 ? a.c.k_scales : a.c.v_scales) + batch * a.c.scales_bs + kv_head * a.c.scales_hs;
    uint8_t* const ring = c4_smem + warp * D * C::kStep;
    constexpr int kPieces = HD / 32;                // of a row
    auto fetch = [&](int step, int slot) {
        const int key0 = step < sink_steps ? step * 16 : win0 + (step - sink_steps) * 16;
        const uint32_t st = smem_u32(ring + slot * C::kStep);
        // (keys behind the last row are read as that one; nobody sees them)
#pragma unroll
        for (int i = 0; i < 16 * kPieces / 32; ++i) {
            const int row = (lane + 32 * i) / kPieces, c = lane % kPieces;
            const long long off = static_cast<long long>(min(key0 + row, a.c.rows - 1)) * (HD / 2) + c * 16;
            c4_copy<16>(st + row * (HD / 2) + c * 16, kc_base + off);
            c4_copy<16>(st + C::kCodes + row * (HD / 2) + (HD == 128 ? c ^ ((row >> 1) & 3) : c) * 16, vc_base + off);
        }
        c4_copy<4 * G>(st + 2 * C::kCodes + lane * 4 * G, sc_base + static_cast<long long>(min(key0 + (lane & 15), a.c.rows - 1)) * (2 * G));
    };
    const uint8_t* const k_at = ring + g * (HD / 2) + q * 4 * S;
    const uint8_t* const ks_at = ring + 2 * C::kCodes + g * 4 * G;
    const uint8_t* const low_at = ks_at + (q < G ? q : 0) * 4;
    // V: lanes of odd q take the second key of a pair first, and put the halves together the other way round
    const int odd_q = q & 1;
    const uint8_t* const v_at = ring + C::kCodes + 2 * q * (HD / 2) + (HD == 128 ? ((g >> 1) ^ q) * 16 + (g & 1) * 8 : g * 4);
    const uint32_t sel_low = odd_q ? 0x1054 : 0x5410, sel_high = odd_q ? 0x3276 : 0x7632;

    // Transposed accumulators: lane (g, q) has columns of V (rows of a product) in the tiles 2 s (columns 32 s + 4 g and + 2) and
    // 2 s + 1 (+ 1 and + 3, sixteen times them), for the query rows 2 q and 2 q + 1; lows, maxima and sums for its own keys.
    float m[NR][2], ref[NR][2], l[NR][2], o[NR][2 * S][4], lo[NR][G][2];          // (ref: the maximum, or 0 ahead of the first key that is seen)
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            m[nr][h] = -INFINITY;
            ref[nr][h] = l[nr][h] = 0.0f;
#pragma unroll
            for (int gi = 0; gi < G; ++gi) lo[nr][gi][h] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 2 * S; ++i) o[nr][i][0] = o[nr][i][1] = o[nr][i][2] = o[nr][i][3] = 0.0f;
    }
    // The weights times the steps of V, which FP16 has to hold, are lifted by powers of two to where the largest is some 2^11, for every query row by
    // what it sees, and by what counts of that, alone: a key that it does not see, or that has next to no weight, may have steps 2^100 times as large.
    // One lift serves all groups of a row while the largest of each is 2^2 or more by it; then (uneven) each has its own, in shared memory.
    // What FP16 loses below its normal range is 2^-19 of the largest a key then, at most.  (One lift for all rows, by the largest step that any of them might
    // see, took up to 6 % less: 32 sequences of up to 32768 keys 231 us, this way 237, of 8192 in groups of 128 83.2 and 83.8.)
    float lift[NR][2], fades[NR][2];      // (fades: scores from here on make 2^-8 and less of what a row has so far)
    float v_most = INFINITY;              // steps from here on might be too large
    bool uneven = false;
    uint32_t dead = 0;                    // groups that had nothing but steps of 0 when their lift was chosen
    float2* const own = lifts + warp * NR * G * 4 + q;
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        lift[nr][0] = lift[nr][1] = kC4MostLift;
        fades[nr][0] = fades[nr][1] = -INFINITY;
    }
    auto scale_o = [&](int nr, int gi, int c, float f) {
#pragma unroll
        for (int i = 2 * gi * kPer; i < 2 * (gi + 1) * kPer; ++i) {
            o[nr][i][c] *= f;
            o[nr][i][2 + c] *= f;
        }
    };
    const int stride = W * split;
    int step = part * W + warp, slot = 0;
#pragma unroll
    for (int i = 0; i < D - 1; ++i) {
        if (step + i * stride < steps) fetch(step + i * stride, i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // (two loops: what looks at the groups' own lifts is in the second alone, to which a warp goes for good when it has some; in one it cost 3 %)
    auto walk = [&](auto is_by_groups) {
    constexpr bool kByGroups = decltype(is_by_groups)::value;
    bool leave = false;
    for (; step < steps && !leave; step += stride) {
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
        __syncwarp();            // all lanes' copies are there, and all lanes have read the slot that is filled next
        if (step + (D - 1) * stride < steps) fetch(step + (D - 1) * stride, slot == 0 ? D - 1 : slot - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const int at = slot * C::kStep;
        slot = slot + 1 == D ? 0 : slot + 1;
        const int key0 = step < sink_steps ? step * 16 : win0 + (step - sink_steps) * 16;
        float mask = 1.0f;
        if (kMask) mask = load_scale(a.key_mask + min(key0 + (lane & 15), a.c.rows - 1));
        uint32_t kc[2][S], ks[2][G];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            c4_lds<S>(k_at + at + h * 8 * (HD / 2), kc[h]);
            c4_lds<G>(ks_at + at + h * 8 * 4 * G, ks[h]);
        }
        // scores: the lows' part by one product (this lane has those of group q), then the steps' of each group
        float s[NR][4];
        {
            float low[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t w = G == 1 ? ks[h][0] : *reinterpret_cast<const uint32_t*>(low_at + at + h * 8 * 4 * G);
                low[h] = G == 4 || q < G ? layer_pair<kBf16>(w).y : 0.0f;
            }
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                mma8_tf32_first(s[nr], low[0], low[1], low[0], low[1], qs[nr][0], qs[nr][1]);
            }
#pragma unroll
            for (int gi = 0; gi < G; ++gi) {
                float d[NR][4];
#pragma unroll
                for (int i = gi * kPer; i < (gi + 1) * kPer; ++i) {
                    uint32_t u[2][4];
                    codes8(kc[0][i], u[0]);
                    codes8(kc[1][i], u[1]);
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) {
                        if (i == gi * kPer) mma16_first<false>(d[nr], u[0][0], u[1][0], u[0][2], u[1][2], qf[nr][i][0], qf[nr][i][2]);
                        else mma16<false>(d[nr], u[0][0], u[1][0], u[0][2], u[1][2], qf[nr][i][0], qf[nr][i][2]);
                        mma16<false>(d[nr], u[0][1], u[1][1], u[0][3], u[1][3], qf[nr][i][1], qf[nr][i][3]);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float st = layer_pair<kBf16>(ks[h][gi]).x;
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) {
                        s[nr][2 * h] = fmaf(st, d[nr][2 * h], s[nr][2 * h]);
                        s[nr][2 * h + 1] = fmaf(st, d[nr][2 * h + 1], s[nr][2 * h + 1]);
                    }
                }
            }
        }
        uint32_t vp[2][G], vw[4][S / 2];
#pragma unroll
        for (int h = 0; h < 2; ++h) c4_lds<G>(ks_at + at + C::kScales + h * 8 * 4 * G, vp[h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) c4_lds<S / 2>(v_at + at + ((e >> 1) * 8 + ((e ^ odd_q) & 1)) * (HD / 2), vw[e]);

        // what is seen of the sixteen keys; all of it in most steps
        const uint32_t live = kMask ? __ballot_sync(0xffffffffu, mask != 0.0f) : 0xffffffffu;      // the sixteen twice
        const bool whole = (step < whole_sinks || (step >= whole_first && step < whole_end)) && live == 0xffffffffu;
        float careful = 0.0f;            // the largest step of V of this lane's keys
        bool odd = false;                // some of their pairs are not finite, and not all queries may see them
        uint32_t hidden = 0;             // of the scores, by bits
        if (!whole) {
            const int begin = step < sink_steps ? 0 : span.win_begin, end = step < sink_steps ? span.sink_end : span.win_end;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = key0 + g + 8 * h;
                const bool on = key >= begin && key < end && ((live >> (g + 8 * h)) & 1u) != 0;
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const bool seen = on && key <= pos[nr][c] && (a.window == 0 || pos[nr][c] - key < a.window || key < a.sinks);
                        if (!seen) {
                            s[nr][2 * h + c] = -INFINITY;
                            hidden |= 1u << (nr * 4 + 2 * h + c);
                        }
                    }
                }
                // what hidden rows hold counts for nothing (nor does a step that is not finite below, where some rows may not see it)
#pragma unroll
                for (int gi = 0; gi < G; ++gi) {
                    if (!on) vp[h][gi] = 0u;
                    const float2 v = layer_pair<kBf16>(vp[h][gi]);
                    careful = fmaxf(careful, v.x <= FLT_MAX ? v.x : 0.0f);
                    odd = odd || !(fabsf(v.x) <= FLT_MAX && fabsf(v.y) <= FLT_MAX);
                }
            }
            odd = __any_sync(0xffffffffu, odd);
        } else {
            // (in pairs of 16 bits, NaN left out; an infinity makes all rows NaN, since all see it)
            uint32_t top = vp[0][0];
#pragma unroll
            for (int i = 1; i < 2 * G; ++i) {
                if constexpr (kBf16) asm("max.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(vp[i / G][i % G]));
                else asm("max.f16x2 %0, %0, %1;" : "+r"(top) : "r"(vp[i / G][i % G]));
            }
            careful = fmaxf(0.0f, layer_pair<kBf16>(top).x);
        }
        // a step of V that might be too large, were its weight 1, is rare
        bool special = odd || (kByGroups && uneven) || __any_sync(0xffffffffu, careful >= v_most);
        if (kByGroups && dead != 0) {
            bool some = false;
#pragma unroll
            for (int i = 0; i < 2 * G; ++i) some = some || (((dead >> (i % G)) & 1u) != 0 && layer_pair<kBf16>(vp[i / G][i % G]).x != 0.0f);
            special = __any_sync(0xffffffffu, some) || special;
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            float top[2] = {fmaxf(s[nr][0], s[nr][2]), fmaxf(s[nr][1], s[nr][3])};
            // a new largest score is rare after the first steps
            if (__any_sync(0xffffffffu, top[0] > m[nr][0] || top[1] > m[nr][1])) {
                special = __any_sync(0xffffffffu, top[0] > fades[nr][0] || top[1] > fades[nr][1]) || special;
#pragma unroll
                for (int x = 4; x < 32; x *= 2) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], x));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], x));
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float now = fmaxf(m[nr][h], top[h]);
                    const float alpha = now == -INFINITY ? 1.0f : fast_exp2((m[nr][h] - now) * sl2[nr][h]);
                    m[nr][h] = now;
                    ref[nr][h] = now == -INFINITY ? 0.0f : now;
                    l[nr][h] *= alpha;
#pragma unroll
                    for (int gi = 0; gi < G; ++gi) {
                        lo[nr][gi][h] *= alpha;
                        scale_o(nr, gi, h, alpha);
                    }
                }
            }
        }
        // (code of its own where lifts are looked at, or pairs are not finite: as branches of one, its instructions are issued all the same)
        auto weigh = [&](auto is_special) {
            constexpr bool kSpecial = decltype(is_special)::value;
            float p[NR][4], by[NR][kSpecial ? G : 1][2];
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[nr][e] = fast_exp2((s[nr][e] - ref[nr][e & 1]) * sl2[nr][e & 1]);
                    l[nr][e & 1] += p[nr][e];
                }
                by[nr][0][0] = lift[nr][0];
                by[nr][0][1] = lift[nr][1];
            }
            if constexpr (kSpecial) {
                float highest = 0.0f;
                bool apart = false;
                dead = 0;
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        // (2^up: what the row has faded by)
                        const int up = static_cast<int>(fminf(fmaxf((m[nr][c] - fades[nr][c]) * sl2[nr][c] + 8.0f, 0.0f), 252.0f));
                        const float up0 = pow2(up / 2), up1 = pow2(up - up / 2);
                        float most[G], least = kC4MostLift, any = 0.0f;
#pragma unroll
                        for (int gi = 0; gi < G; ++gi) {
                            // what has faded comes up again, where there is something
                            bool nothing = fades[nr][c] == -INFINITY;
                            if constexpr (kByGroups) {
                                nothing = true;
#pragma unroll
                                for (int i = 2 * gi * kPer; i < 2 * (gi + 1) * kPer; ++i) nothing = nothing && o[nr][i][c] == 0.0f && o[nr][i][2 + c] == 0.0f;
                                nothing = (~__ballot_sync(0xffffffffu, nothing) & (0x11111111u << q)) == 0;
                            }
                            const float was = kByGroups && uneven ? reinterpret_cast<const float*>(own + (nr * G + gi) * 4)[c] : lift[nr][c];
                            float now = nothing ? kC4MostLift : fminf(was * up0 * up1, kC4MostLift);
                            // the largest of these sixteen keys goes to 2^11 where it is too large
                            float t = fmaxf(fmaxf(0.0f, p[nr][c] * layer_pair<kBf16>(vp[0][gi]).x), p[nr][2 + c] * layer_pair<kBf16>(vp[1][gi]).x);
#pragma unroll
                            for (int x = 4; x < 32; x *= 2) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
                            most[gi] = t = fminf(t, FLT_MAX);
                            if (t * now >= 0x1p15f) now = pow2(11 - exponent(t));
                            if (!nothing) scale_o(nr, gi, c, pow2_ratio(now, was));
                            by[nr][gi][c] = now;
                            any = fmaxf(any, t);
                            least = fminf(least, now);
                        }
                        fades[nr][c] = m[nr][c] == -INFINITY ? -INFINITY : m[nr][c] + 8.0f / sl2[nr][c];
                        lift[nr][c] = least;
                        if (m[nr][c] != -INFINITY) highest = fmaxf(highest, least);
#pragma unroll
                        for (int gi = 0; gi < G; ++gi) {
                            const float now = by[nr][gi][c];
                            const bool none = any > 0.0f && most[gi] == 0.0f;
                            if (none) dead |= 1u << gi;
                            apart = apart || !(now == least || (none ? now == kC4MostLift || now * 0x1p-64f <= least : most[gi] * least >= 4.0f));
                        }
                    }
                }
                if constexpr (G > 1) {
                    dead = __reduce_or_sync(0xffffffffu, dead);
                    __syncwarp();            // (all lanes have read their rows' lifts)
                    uneven = __any_sync(0xffffffffu, apart);
                    leave = !kByGroups && (uneven || dead != 0);
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
                        for (int gi = 0; gi < G; ++gi) {
                            if (uneven) {
                                if (g == 0) own[(nr * G + gi) * 4] = make_float2(by[nr][gi][0], by[nr][gi][1]);
                            } else {
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    scale_o(nr, gi, c, pow2_ratio(lift[nr][c], by[nr][gi][c]));
                                    by[nr][gi][c] = lift[nr][c];
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
                const uint32_t high = __reduce_max_sync(0xffffffffu, __float_as_uint(highest));
                v_most = high == 0 ? INFINITY : pow2(min(127, 15 - exponent(__uint_as_float(high))));
            }
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) {
                float lifted[4];
                if (!kSpecial) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) lifted[e] = p[nr][e] * lift[nr][e & 1];
                }
#pragma unroll
                for (int gi = 0; gi < G; ++gi) {
                    float w[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 v = layer_pair<kBf16>(vp[h][gi]);
                        const float mid = fmaf(8.0f, v.x, v.y);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int e = 2 * h + c;
                            w[e] = (kSpecial ? p[nr][e] * by[nr][kSpecial ? gi : 0][c] : lifted[e]) * v.x;
                            if (!kSpecial) lo[nr][gi][c] = fmaf(p[nr][e], mid, lo[nr][gi][c]);
                        }
                    }
                    if (kSpecial) {              // (what a query does not see is left out; zero times what it does see is NaN where that is not finite)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 v = layer_pair<kBf16>(vp[e >> 1][gi]);
                            if ((hidden >> (nr * 4 + e)) & 1u) w[e] = 0.0f;
                            else lo[nr][gi][e & 1] = fmaf(p[nr][e], fmaf(8.0f, v.x, v.y), lo[nr][gi][e & 1]);
                        }
                    }
                    const uint32_t b0 = c4_transpose8(pack2<false>(w[0], w[1])), b1 = c4_transpose8(pack2<false>(w[2], w[3]));
#pragma unroll
                    for (int i = gi * kPer; i < (gi + 1) * kPer; ++i) {
                        // four columns of two keys: the halves of a word of each
                        const uint32_t sel = (i & 1) ? sel_high : sel_low;
                        const uint32_t w0 = __byte_perm(vw[0][i / 2], vw[1][i / 2], sel), w1 = __byte_perm(vw[2][i / 2], vw[3][i / 2], sel);
                        uint32_t u0[4], u1[4];
                        codes8(w0, u0);
                        codes8(w1, u1);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            u0[e] = (e & 1) ? less_eight<true>(u0[e]) : less_eight<false>(u0[e]);
                            u1[e] = (e & 1) ? less_eight<true>(u1[e]) : less_eight<false>(u1[e]);
                        }
                        mma16<false>(o[nr][2 * i], u0[0], u0[2], u1[0], u1[2], b0, b1);
                        mma16<false>(o[nr][2 * i + 1], u0[1], u0[3], u1[1], u1[3], b0, b1);
                    }
                }
            }
        };
        if (__builtin_expect(special, 0)) weigh(std::true_type{});
        else weigh(std::false_type{});
    }
    };
    walk(std::false_type{});
    if constexpr (G > 1) walk(std::true_type{});
    // the warps' sums, whole: over the lanes' keys, the lows and the powers of two put in
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) {
                l[nr][h] += __shfl_xor_sync(0xffffffffu, l[nr][h], x);
#pragma unroll
                for (int gi = 0; gi < G; ++gi) lo[nr][gi][h] += __shfl_xor_sync(0xffffffffu, lo[nr][gi][h], x);
            }
        }
    }
    float* const mine = o_warp + warp * kRows * C::kLd;
    __syncthreads();
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = nr * 8 + 2 * q + h;
            // the maximum in units of log2, the same for all warps of the row
            if (g == 0) ml_warp[warp * kRows + r] = make_float2(m[nr][h] == -INFINITY ? -INFINITY : m[nr][h] * sl2[nr][h], l[nr][h]);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const float low = lo[nr][s / kPer][h];
                const float down = pow2(-exponent(uneven ? reinterpret_cast<const float*>(own + (nr * G + s / kPer) * 4)[h] : lift[nr][h]));
                *reinterpret_cast<float4*>(mine + r * C::kLd + 32 * s + 4 * g) =
                    make_float4(fmaf(o[nr][2 * s][h] * 0x1p24f, down, low), fmaf(o[nr][2 * s + 1][h] * 0x1p20f, down, low),
                                fmaf(o[nr][2 * s][2 + h] * 0x1p24f, down, low), fmaf(o[nr][2 * s + 1][2 + h] * 0x1p20f, down, low));
            }
        }
    }
    __syncthreads();
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    // The CTA's sums go to the CTAs that finish the rows: row r to CTA r % split, in whose place
    // part * ceil(kRows / split) + r / split it lies.
    constexpr int kUnits = HD / 4;
    const int per = (kRows + split - 1) / split;
    for (int u = threadIdx.x; u < rows * kUnits; u += W * 32) {
        const int r = u / kUnits, c = (u % kUnits) * 4;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, ml_warp[w * kRows + r].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 t = ml_warp[w * kRows + r];
            const float f = fast_exp2(t.x - ref);
            const float4 v = *reinterpret_cast<const float4*>(o_warp + (w * kRows + r) * C::kLd + c);
            acc.x = fmaf(f, v.x, acc.x);
            acc.y = fmaf(f, v.y, acc.y);
            acc.z = fmaf(f, v.z, acc.z);
            acc.w = fmaf(f, v.w, acc.w);
            sum = fmaf(f, t.y, sum);
        }
        const int place = part * per + r / split;
        if (split > 1) {
            c4_store_cluster(mapa(smem_u32(o_cta + place * C::kLd + c), r % split), acc);
            if (c == 0) c4_store_cluster(mapa(smem_u32(ml_cta + place), r % split), make_float2(top, sum));
        } else {
            *reinterpret_cast<float4*>(o_cta + place * C::kLd + c) = acc;
            if (c == 0) ml_cta[place] = make_float2(top, sum);
        }
    }
    if (split > 1) cluster_sync();
    else __syncthreads();
    for (int u = threadIdx.x; u < per * kUnits; u += W * 32) {
        const int x = u / kUnits, r = part + x * split, c = (u % kUnits) * 4;
        if (r >= rows) break;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float top = -INFINITY, sum = 0.0f;
        for (int k = 0; k < split; ++k) top = fmaxf(top, ml_cta[k * per + x].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        for (int k = 0; k < split; ++k) {
            const float2 t = ml_cta[k * per + x];
            const float4 v = *reinterpret_cast<const float4*>(o_cta + (k * per + x) * C::kLd + c);
            const float f = fast_exp2(t.x - ref);
            acc.x = fmaf(f, v.x, acc.x);
            acc.y = fmaf(f, v.y, acc.y);
            acc.z = fmaf(f, v.z, acc.z);
            acc.w = fmaf(f, v.w, acc.w);
            sum = fmaf(f, t.y, sum);
        }
        // (a sum that is NaN makes the row NaN)
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int i = (row0 + r) / a.kv_group, head = kv_head * a.kv_group + (row0 + r) % a.kv_group;
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.o) + batch * a.o_bs + i * a.o_ld + static_cast<long long>(head) * HD + c) =
            make_uint2(pack2<kBf16>(acc.x * inv, acc.y * inv), pack2<kBf16>(acc.z * inv, acc.w * inv));
    }
}

template <int HD, int G, bool kBf16, int W, int NR, int D, int kCtas>
cudaError_t go_cache4(SdpaCache4Args a, int split, cudaStream_t stream) {
    using C = Cache4Cfg<HD, G, W, NR, D>;
    const auto masked = sdpa_cache4_kernel<HD, G, kBf16, true, W, NR, D, kCtas>, plain = sdpa_cache4_kernel<HD, G, kBf16, false, W, NR, D, kCtas>;
    const auto kern = a.key_mask != nullptr ? masked : plain;
    cudaError_t e = set_max_smem_once(kern, C::kSmem);
    if (e == cudaSuccess && split > 8) {
        // clusters of more than eight CTAs are allowed once for each device, and again where that has no bit
        static std::atomic<unsigned long long> allowed{0};
        int dev = 0;
        e = cudaGetDevice(&dev);
        const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
        if (e == cudaSuccess && (allowed.load() & bit) == 0) {
            e = cudaFuncSetAttribute(masked, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(plain, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e == cudaSuccess) allowed.fetch_or(bit);
        }
    }
    if (e != cudaSuccess) return e;
    a.split = split;
    const dim3 grid(static_cast<unsigned>(split * a.c.kv_heads * a.row_tiles), static_cast<unsigned>(a.batch));
    return launch_dependent_cluster(kern, grid, dim3(W * 32), C::kSmem, stream, dim3(split), a);
}

template <int HD, int G, bool kBf16>
cudaError_t pick_cache4(SdpaCache4Args a, cudaStream_t stream) {
    const long long rows = static_cast<long long>(a.lq) * a.kv_group;
    const int nr = rows <= 8 ? 1 : 2, sms = sm_count();
    a.row_tiles = static_cast<int>((rows + 8 * nr - 1) / (8 * nr));
    const long long units = static_cast<long long>(a.batch) * a.c.kv_heads * a.row_tiles;
    // sixteens of keys that there are for the longest sequence
    const long long seen = a.window > 0 ? static_cast<long long>(a.window) + a.sinks + a.lq - 1 : a.c.rows;
    const long long steps = ((seen < a.c.rows ? seen : a.c.rows) + 15) / 16;
    auto least = [](long long x, long long y) { return static_cast<int>(x < y ? x : y); };
    // Few heads over long caches: eight warps to a CTA, two CTAs to an SM and the keys of a head over all CTAs there is room for, with two steps
    // to a warp (8 heads over 32768 keys: sixteen CTAs 27.4 us, eight 33.5, sixteen of four warps 34.2; 32 heads over 4000 keys: eight CTAs 9.6,
    // sixteen of four warps 11.3).
    if (nr == 1 && units * 8 <= 2 * sms && steps >= 128) {
        return go_cache4<HD, G, kBf16, 8, 1, 3, 2>(a, least(least(kC4MaxSplit, 2 * sms / units), steps / 16), stream);
    }
    // Else four warps.  SMs come in pairs, the CTAs of a cluster find their places within some of them: where there is more than one round, a
    // cluster is all the CTAs of a pair of SMs, or a part that divides them, so that no place stays empty (256 heads over up to 32768 keys,
    // three CTAs to an SM: over six 232 us, over five 240, seven 241, eight 238; keys all alike 303, 330, 336, 332), and the smallest such part with
    // two and a half rounds (512 heads over up to 8192 keys: over three 129, over six 137; 256 heads: over three 252).  Eight, where all run at
    // once, but one step to a warp at least (8 heads over 777 keys: over eight 4.1, over sixteen 4.4, over six 4.7).
    constexpr int kOne = HD == 64 || G == 1 ? 4 : 3, kTwo = HD == 64 ? (G == 1 ? 4 : 3) : 2;           // CTAs of an SM: what registers allow
    const int ctas = nr == 1 ? kOne : kTwo, slots = sms * ctas;
    int split = 8;
    if (units * 8 > slots) {
        split = 1;
        while (split < 2 * ctas && (2 * ctas % split != 0 || 2 * units * split < 5ll * slots)) ++split;
    }
    if (nr == 2 && units >= slots) split = 1;          // (509 x 2 rows, 16 heads of 64: whole 134, over two 144)
    split = least(split, (steps + 3) / 4);
    return nr == 1 ? go_cache4<HD, G, kBf16, 4, 1, 3, kOne>(a, split, stream) : go_cache4<HD, G, kBf16, 4, 2, 3, kTwo>(a, split, stream);
}

}  // namespace

cudaError_t launch_sdpa_cache4(const SdpaCache4Args& a, bool bf16, cudaStream_t stream) {
    auto go = [&](auto b) {
        constexpr bool kB = decltype(b)::value;
        const int groups = a.c.head_dim / a.c.group;
        if (a.c.head_dim == 64) return groups == 1 ? pick_cache4<64, 1, kB>(a, stream) : pick_cache4<64, 2, kB>(a, stream);
        return groups == 1 ? pick_cache4<128, 1, kB>(a, stream) : groups == 2 ? pick_cache4<128, 2, kB>(a, stream) : pick_cache4<128, 4, kB>(a, stream);
    };
    return bf16 ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace bdattn
