// Causal attention with a sliding window and visible first keys (sinks) for few query rows (single
// tokens, a few drafted ones), and a warp per row and head for any head_dim up to 256.
//
// Few rows: what a call costs is reading K and V once, so the query heads that share a K/V head, and the new
// tokens, are the (up to sixteen) rows of one mma.sync product, and the visible keys of a K/V head are shared by a
// cluster of CTAs: each walks its part in chunks of 64 keys through a ring of TMA copies, its four warps with 16 keys
// of a chunk, a running maximum, sum and accumulator each; these meet in shared memory, then in distributed
// shared memory, where every CTA finishes its share of the rows.  One launch, no workspace.
#include "sdpa_window.cuh"

namespace bdattn {
namespace {

constexpr int kWinWarps = 8;

template <bool kBf16>
__global__ void __launch_bounds__(kWinWarps * 32) sdpa_window_kernel(const __grid_constant__ SdpaWindowArgs a) {
    __shared__ float q_s[kWinWarps][256];
    wait_for_prior_grid();
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int i = static_cast<int>(blockIdx.x) * kWinWarps + warp;
    if (i < a.q_rows[0] + a.q_rows[1]) window_row<kBf16>(a, blockIdx.z, blockIdx.y, i, q_s[warp], lane);
}

constexpr int kFewKeys = 64;          // keys of a chunk
constexpr int kFewMaxSplit = 16;

// W: warps with the products; one more copies.  NR: query rows in eights.  KT: keys of a warp's step in sixteens,
// so that four or two warps share a chunk.
template <int HD, int W, int NR, int KT>
struct FewCfg {
    static constexpr int kThreads = (W + 1) * 32;
    static constexpr int kRows = 8 * NR;
    static constexpr int kTile = HD * 128;              // bytes of 64 rows: HD / 64 boxes of 64 x 128 bytes
    static constexpr int kStage = 2 * kTile;            // K and V
    static constexpr int kStages = (W == 4 ? 96 : 192) * 1024 / kStage;
    static constexpr int kGroups = W * KT / 4;          // warps that share a chunk take the chunks in turn
    static constexpr int kLd = HD + 4;                  // floats of a partial row
    // rows that a CTA gets from its cluster, split x ceil(kRows / split): up to 30 with sixteen rows, 16 where split is a power of two
    static constexpr int kMergeRows = NR == 1 || W == 4 ? 16 : 32;
    static constexpr int kBars = 2 * kStages * 8 + 16;
    static constexpr int kSmem = kStages * kStage + kBars + W * kRows * 8 + kMergeRows * (8 + kLd * 4) + 1024;
    static_assert(W * kRows * kLd * 4 <= kStages * kStage, "the warps' partial sums lie in the ring");
};

// The chunks of the visible keys: up to four ranges (sinks and window in each segment), 64 keys to a chunk.
struct FewChunks {
    int row[4], key[4], count[4], total;
    __device__ __forceinline__ void init(const SdpaWindowArgs& a, const WindowSpan& s) {
        const int k0 = a.kv_rows[0];
        const int begin[2] = {0, s.win_begin}, end[2] = {s.sink_end, s.win_end};
        total = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = (i & 1) ? max(begin[i >> 1], k0) : begin[i >> 1];
            const int e = (i & 1) ? end[i >> 1] : min(end[i >> 1], k0);
            key[i] = b;
            row[i] = (i & 1) ? b - k0 : b;
            count[i] = max(0, e - b);
            total += (count[i] + kFewKeys - 1) / kFewKeys;
        }
    }
    // segment, first row in it, first key and number of keys of chunk c
    __device__ __forceinline__ void at(int c, int& seg, int& r, int& k, int& n) const {
        seg = 0; r = 0; k = 0; n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int chunks = (count[i] + kFewKeys - 1) / kFewKeys;
            if (c >= 0 && c < chunks) {
                seg = i & 1;
                r = row[i] + c * kFewKeys;
                k = key[i] + c * kFewKeys;
                n = min(kFewKeys, count[i] - c * kFewKeys);
            }
            c -= chunks;
        }
    }
};

__device__ __forceinline__ void store_cluster(uint32_t addr, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, float2 v) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}

// The transpose of an 8 x 8 matrix of 16-bit values, two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int HD, bool kBf16, int W, int NR, int KT>
__global__ void __launch_bounds__(FewCfg<HD, W, NR, KT>::kThreads, W == 4 ? 2 : 1)
sdpa_few_kernel(const __grid_constant__ CUtensorMap tmK0, const __grid_constant__ CUtensorMap tmK1,
                const __grid_constant__ CUtensorMap tmV0, const __grid_constant__ CUtensorMap tmV1,
                const __grid_constant__ SdpaWindowArgs a, const int split, const int row_tiles) {
    using C = FewCfg<HD, W, NR, KT>;
    constexpr int kSteps = HD / 16, kGroups = C::kGroups, stages = C::kStages, kRows = C::kRows;
    extern __shared__ uint8_t few_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(few_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + stages * C::kStage);
    uint64_t* empty = full + stages;
    uint32_t* again_s = reinterpret_cast<uint32_t*>(empty + stages);
    float2* ml_warp = reinterpret_cast<float2*>(again_s + 4);                // [W][kRows] maximum and sum of a warp's keys
    float2* ml_cta = ml_warp + W * kRows;                                 // [split][x] of the cluster's CTAs, for the rows finished here
    float* o_cta = reinterpret_cast<float*>(ml_cta + C::kMergeRows);         // and their sums

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int part = split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int kv_head = static_cast<int>(blockIdx.y) / row_tiles, row0 = static_cast<int>(blockIdx.y) % row_tiles * kRows;
    const int batch = blockIdx.z;
    const int lq = a.q_rows[0], rows = min(kRows, lq * a.kv_group - row0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 4 / KT);
        }
        *again_s = 0;
        fence_mbar_init();
    }
    if (warp == W && lane == 0) {
        tma_prefetch_desc(&tmK0);
        tma_prefetch_desc(&tmV0);
    }
    __syncthreads();
    // (waited for ahead of the first store into a peer's shared memory: it has to run by then)
    if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    dependents_may_launch();
    wait_for_prior_grid();

    const int first_pos = window_keys(a.kv_len, batch, a.kv_rows[0] + a.kv_rows[1]) - lq;      // of query 0
    FewChunks chunks;
    chunks.init(a, window_span(first_pos + row0 / a.kv_group, first_pos + (row0 + rows - 1) / a.kv_group, a.window, a.sinks));
    const float sl2 = a.scale * 1.4426950408889634f;
    const int c_begin = static_cast<int>(static_cast<long long>(chunks.total) * part / split);
    const int c_end = static_cast<int>(static_cast<long long>(chunks.total) * (part + 1) / split);

    if (warp == W) {
        if (elect_one()) {
            int slot = 0, issued = 0;
            uint32_t phase = 1;
            bool ok = true;
            for (int c = c_begin; c < c_end; ++c) {
                ok = mbar_wait(&empty[slot], phase);
                if (!ok) break;
                int seg, r, k, n;
                chunks.at(c, seg, r, k, n);
                uint8_t* const st = ring + slot * C::kStage;
                mbar_arrive_expect_tx(&full[slot], C::kStage);
#pragma unroll
                for (int b = 0; b < HD / 64; ++b)
                    tma_load_4d(st + b * 8192, seg ? &tmK1 : &tmK0, &full[slot], b * 64, kv_head, r, batch);
#pragma unroll
                for (int b = 0; b < HD / 64; ++b)
                    tma_load_4d(st + C::kTile + b * 8192, seg ? &tmV1 : &tmV0, &full[slot], b * 64, kv_head, r, batch);
                ++issued;
                if (++slot == stages) { slot = 0; phase ^= 1; }
            }
            if (!ok)        // a wait ran out: the copies in flight land before the CTA ends
                for (int i = max(0, issued - stages); i < issued; ++i)
                    mbar_wait(&full[i % stages], static_cast<uint32_t>((i / stages) & 1));
        }
        __syncwarp();
    } else {
        // Scores and sums are transposed, S' = K Q' and O' = V' P': keys and columns are the sixteen rows of a
        // product and the query rows its eight columns, half the products that sixteen query rows take.
        // This thread has columns 2 (lane % 4) and the next of every eight query rows.
        uint32_t qf[NR][kSteps][2];
        int pos[NR][2];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const int rq = nr * 8 + (lane >> 2);
            const int i = (row0 + rq) / a.kv_group;
            const uint16_t* const q = reinterpret_cast<const uint16_t*>(a.q[0]) + batch * a.q_bs[0] + i * a.q_ld[0] +
                                      static_cast<long long>(kv_head * a.kv_group + (row0 + rq) % a.kv_group) * a.head_dim;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = k * 16 + e * 8 + (lane & 3) * 2;
                    qf[nr][k][e] = rq < rows && c < a.head_dim ? *reinterpret_cast<const uint32_t*>(q + c) : 0u;
                }
            }
            pos[nr][0] = first_pos + (row0 + min(nr * 8 + (lane & 3) * 2, rows - 1)) / a.kv_group;
            pos[nr][1] = first_pos + (row0 + min(nr * 8 + (lane & 3) * 2 + 1, rows - 1)) / a.kv_group;
        }
        float m[NR][2], l[NR][2], o[NR][kSteps][4];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            m[nr][0] = m[nr][1] = -INFINITY;
            l[nr][0] = l[nr][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) o[nr][i][0] = o[nr][i][1] = o[nr][i][2] = o[nr][i][3] = 0.0f;
        }
        constexpr int kSharing = 4 / KT;
        constexpr uint32_t kAll = KT == 2 ? 0xffffffffu : 0xffffu;
        const int key_w = warp % kSharing * 16 * KT;
        // ldmatrix rows of this lane: K keys (lane / 8 % 2) * 8 + lane % 8 with columns (lane / 16) * 8, V the other way round
        const int k_key = key_w + ((lane >> 3) & 1) * 8 + (lane & 7), k_piece = lane >> 4;
        const int v_key = key_w + (lane >> 4) * 8 + (lane & 7), v_piece = (lane >> 3) & 1;
        int slot = warp / kSharing;
        uint32_t phase = 0;
        for (int c = c_begin + warp / kSharing; c < c_end; c += kGroups) {
            while (slot >= stages) {
                slot -= stages;
                phase ^= 1;
            }
            int seg, r, key0, n;
            chunks.at(c, seg, r, key0, n);
            key0 += key_w;
            // which of the warp's keys exist and are let through by the key mask, one to a lane
            bool on = lane < 16 * KT && key_w + lane < n;
            if (a.key_mask != nullptr && on) on = a.key_mask[key0 + lane] != 0.0f;
            const uint32_t live = __ballot_sync(0xffffffffu, on);
            // A slot may pass from one group of warps to another.  That the slot's last user has released it says that its last
            // copy had landed: without this wait a group that is ahead could find the phase before that copy
            // and take it, by its parity, for the one behind.
            if (kGroups > 1 && !mbar_wait_warp(&empty[slot], phase ^ 1)) break;
            if (!mbar_wait_warp(&full[slot], phase)) break;
            uint8_t* const st = ring + slot * C::kStage;
            if (live != 0) {
                if (live != kAll) {
                    // values nobody sees may be anything: zeros, so that their weights of zero count for nothing
                    for (uint32_t dead = ~live & kAll; dead != 0; dead &= dead - 1) {
                        const int kr = key_w + __ffs(dead) - 1;
                        if (lane < HD / 8) *reinterpret_cast<uint4*>(st + C::kTile + (lane >> 3) * 8192 + kr * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    __syncwarp();
                }
                float s[KT][NR][4] = {};
                const uint32_t kb = smem_u32(st) + k_key * 128;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
#pragma unroll
                    for (int t = 0; t < KT; ++t) {
                        uint32_t f[4];
                        gen_ldsm4(f, kb + t * 2048 + (k >> 2) * 8192 + ((((k & 3) * 2 + k_piece) ^ (k_key & 7)) << 4));
#pragma unroll
                        for (int nr = 0; nr < NR; ++nr) gen_mma<kBf16>(s[t][nr], f, qf[nr][k][0], qf[nr][k][1]);
                    }
                }
                uint32_t p[KT][NR][2];
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float top[2] = {m[nr][0], m[nr][1]}, add[2];
#pragma unroll
                    for (int t = 0; t < KT; ++t) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int at = t * 16 + (e >> 1) * 8 + (lane >> 2), key = key0 + at, h = e & 1;
                            const bool seen = ((live >> at) & 1u) != 0 && key <= pos[nr][h] &&
                                              (a.window == 0 || pos[nr][h] - key < a.window || key < a.sinks);
                            s[t][nr][e] = seen ? s[t][nr][e] : -INFINITY;
                            top[h] = fmaxf(top[h], s[t][nr][e]);
                        }
                    }
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) {
                        top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], x));
                        top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], x));
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float ref = top[h] == -INFINITY ? 0.0f : top[h];
                        const float alpha = fast_exp2((m[nr][h] - ref) * sl2);
                        m[nr][h] = top[h];
                        l[nr][h] *= alpha;
                        add[h] = -ref * sl2;
#pragma unroll
                        for (int i = 0; i < kSteps; ++i) {
                            o[nr][i][h] *= alpha;
                            o[nr][i][2 + h] *= alpha;
                        }
                    }
#pragma unroll
                    for (int t = 0; t < KT; ++t) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            s[t][nr][e] = fast_exp2(fmaf(s[t][nr][e], sl2, add[e & 1]));
                            l[nr][e & 1] += s[t][nr][e];
                        }
                        // the weights to 16 bits for the second product (their sum is of the unrounded ones)
                        p[t][nr][0] = transpose8(pack2<kBf16>(s[t][nr][0], s[t][nr][1]));
                        p[t][nr][1] = transpose8(pack2<kBf16>(s[t][nr][2], s[t][nr][3]));
                    }
                }
                const uint32_t vb = smem_u32(st) + C::kTile + v_key * 128;
#pragma unroll
                for (int t = 0; t < KT; ++t) {
#pragma unroll
                    for (int d = 0; d < kSteps; ++d) {
                        uint32_t f[4];
                        gen_ldsm4_t(f, vb + t * 2048 + (d >> 2) * 8192 + ((((d & 3) * 2 + v_piece) ^ (v_key & 7)) << 4));
#pragma unroll
                        for (int nr = 0; nr < NR; ++nr) gen_mma<kBf16>(o[nr][d], f, p[t][nr][0], p[t][nr][1]);
                    }
                }
                if (live != kAll) fence_proxy_async_smem();      // the zeros, ahead of the next copy into their place
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[slot]);
            slot += kGroups;
        }
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) {
                l[nr][0] += __shfl_xor_sync(0xffffffffu, l[nr][0], x);
                l[nr][1] += __shfl_xor_sync(0xffffffffu, l[nr][1], x);
            }
        }
        // the warps' partial sums, in the ring once all of them are done with it
        asm volatile("bar.sync 1, %0;" ::"n"(W * 32) : "memory");
        float* const mine = reinterpret_cast<float*>(ring) + warp * kRows * C::kLd;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = nr * 8 + (lane & 3) * 2 + h;
                if (lane < 4) ml_warp[warp * kRows + r] = make_float2(m[nr][h], l[nr][h]);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    mine[r * C::kLd + i * 16 + (lane >> 2)] = o[nr][i][h];
                    mine[r * C::kLd + i * 16 + 8 + (lane >> 2)] = o[nr][i][2 + h];
                }
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(W * 32) : "memory");
    }
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    // The CTA's sums go to the CTAs that finish the rows: row r to CTA r % split, in whose place
    // part * ceil(kRows / split) + r / split it lies; a row is finished by HD / 4 threads of one CTA.
    constexpr int kUnits = HD / 4;
    const int per = (kRows + split - 1) / split;
    if (warp < W) {
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
                const float f = fast_exp2((t.x - ref) * sl2);
                const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(ring) + (w * kRows + r) * C::kLd + c);
                acc.x = fmaf(f, v.x, acc.x);
                acc.y = fmaf(f, v.y, acc.y);
                acc.z = fmaf(f, v.z, acc.z);
                acc.w = fmaf(f, v.w, acc.w);
                sum = fmaf(f, t.y, sum);
            }
            const int place = part * per + r / split;
            if (split > 1) {
                store_cluster(mapa(smem_u32(o_cta + place * C::kLd + c), r % split), acc);
                if (c == 0) store_cluster(mapa(smem_u32(ml_cta + place), r % split), make_float2(top, sum));
            } else {
                *reinterpret_cast<float4*>(o_cta + place * C::kLd + c) = acc;
                if (c == 0) ml_cta[place] = make_float2(top, sum);
            }
        }
    }
    if (split > 1) cluster_sync();
    else __syncthreads();

    if (warp < W) {
        for (int u = threadIdx.x; u < per * kUnits; u += W * 32) {
            const int x = u / kUnits, r = part + x * split, c = (u % kUnits) * 4;
            if (r >= rows) break;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float top = -INFINITY, sum = 0.0f;
#pragma unroll 4
            for (int k = 0; k < split; ++k) top = fmaxf(top, ml_cta[k * per + x].x);
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
            for (int k = 0; k < split; ++k) {
                const float2 t = ml_cta[k * per + x];
                const float4 v = *reinterpret_cast<const float4*>(o_cta + (k * per + x) * C::kLd + c);
                const float f = fast_exp2((t.x - ref) * sl2);
                acc.x = fmaf(f, v.x, acc.x);
                acc.y = fmaf(f, v.y, acc.y);
                acc.z = fmaf(f, v.z, acc.z);
                acc.w = fmaf(f, v.w, acc.w);
                sum = fmaf(f, t.y, sum);
            }
            // (a sum that is NaN makes the row NaN)
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            acc.x *= inv;
            acc.y *= inv;
            acc.z *= inv;
            acc.w *= inv;
            const int i = (row0 + r) / a.kv_group, head = kv_head * a.kv_group + (row0 + r) % a.kv_group;
            if (c < a.head_dim)
                *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.o[0]) + batch * a.o_bs[0] + i * a.o_ld[0] +
                                          static_cast<long long>(head) * a.head_dim + c) =
                    make_uint2(pack2<kBf16>(acc.x, acc.y), pack2<kBf16>(acc.z, acc.w));
            // a key that some rows see and others do not, with a value that is not finite
            const bool fine = fabsf(acc.x) <= FLT_MAX && fabsf(acc.y) <= FLT_MAX && fabsf(acc.z) <= FLT_MAX && fabsf(acc.w) <= FLT_MAX;
            if (!fine && fabsf(sum) <= FLT_MAX && lq > 1) atomicOr(again_s, 1u << r);
        }
    }
    __syncthreads();
    uint32_t again = *again_s;
    for (; again != 0; again &= again - 1) {
        const int r = row0 + __ffs(again) - 1;
        if (warp == 0) window_row<kBf16>(a, batch, kv_head * a.kv_group + r % a.kv_group, r / a.kv_group, reinterpret_cast<float*>(ring), lane);
    }
}

}  // namespace

// How a call's keys are shared: `most` clusters of `split` CTAs with eight warps (and a ring of 192 KB) run at once on
// this device, most[split] of them, looked up once.
template <int HD, bool kBf16, int W, int NR, int KT>
static cudaError_t few_clusters(const int** most) {
    static std::mutex mu;
    static int table[64][kFewMaxSplit + 1];
    static bool known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lock(mu);
    *most = table[dev];
    if (known[dev]) return cudaSuccess;
    using C = FewCfg<HD, W, NR, KT>;
    const auto kern = sdpa_few_kernel<HD, kBf16, W, NR, KT>;
    e = set_max_smem_once(kern, C::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    for (int s = 1; s <= kFewMaxSplit; ++s) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(s);
        cfg.blockDim = dim3(C::kThreads);
        cfg.dynamicSmemBytes = C::kSmem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = s;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&table[dev][s], kern, &cfg);
        if (e != cudaSuccess) return e;
    }
    known[dev] = true;
    return cudaSuccess;
}

template <int HD, bool kBf16, int W, int NR, int KT>
static cudaError_t launch_few(const SdpaFewLaunch& L, int row_tiles, int split, cudaStream_t stream) {
    using C = FewCfg<HD, W, NR, KT>;
    const int* most;
    cudaError_t e = few_clusters<HD, kBf16, W, NR, KT>(&most);       // (sets the kernel's attributes too)
    if (e != cudaSuccess) return e;
    const dim3 grid(static_cast<unsigned>(split), static_cast<unsigned>(L.num_kv_heads * row_tiles), static_cast<unsigned>(L.batch));
    return launch_dependent_cluster(sdpa_few_kernel<HD, kBf16, W, NR, KT>, grid, dim3(C::kThreads), C::kSmem, stream, dim3(split, 1, 1),
                                    L.tmK[0], L.tmK[1], L.tmV[0], L.tmV[1], L.args, split, row_tiles);
}

template <int HD, bool kBf16, int NR>
static cudaError_t plan_few(const SdpaFewLaunch& L, cudaStream_t stream) {
    const SdpaWindowArgs& a = L.args;
    const int row_tiles = (a.q_rows[0] * a.kv_group + 8 * NR - 1) / (8 * NR);
    // chunks of the longest sequence there can be
    const long long lk = static_cast<long long>(a.kv_rows[0]) + a.kv_rows[1];
    const long long seen = a.window > 0 ? static_cast<long long>(a.window) + a.sinks + a.q_rows[0] - 1 : lk;
    const long long units = static_cast<long long>(L.batch) * L.num_kv_heads * row_tiles;
    const long long chunks = ((seen < lk ? seen : lk) + kFewKeys - 1) / kFewKeys;
    // The keys of a K/V head go to as many CTAs as a cluster of this call's number can have with all of them running at
    // once, an SM to each; a cluster that has to wait for another's end costs more than any split gives (batch 1, 8 K/V
    // heads of 128, 32768 keys: over 8 CTAs 25.5 us, over 10 23.4, over 11, of which not all eight clusters run at once,
    // 35.8; 4 x 8 heads, 1028 keys: over 4 5.7, over 5 10.5).
    const int* most;
    cudaError_t e = few_clusters<HD, kBf16, 8, NR, 2>(&most);
    if (e != cudaSuccess) return e;
    int split = 1;
    for (int s = 2; s <= kFewMaxSplit && s <= chunks; ++s)
        if (most[s] >= units) split = s;
    // One or two chunks to a CTA: eight warps would find nothing to do (8 x 516 keys over 8 CTAs: 4.3 us with four
    // warps of 16 keys, 4.6 with eight, 5.4 with eight of 32).
    if (chunks <= 2 * split) {
        while (split & (split - 1)) --split;         // (the merge's room)
        return launch_few<HD, kBf16, 4, NR, 1>(L, row_tiles, split, stream);
    }
    if (split > 1 || units <= most[1]) return launch_few<HD, kBf16, 8, NR, 2>(L, row_tiles, split, stream);
    // More heads than SMs: two CTAs to an SM.
    return launch_few<HD, kBf16, 4, NR, 2>(L, row_tiles, 1, stream);
}

cudaError_t launch_sdpa_few(const SdpaFewLaunch& L, bool bf16, cudaStream_t stream) {
    const bool eight = L.args.q_rows[0] * L.args.kv_group <= 8;
    auto go = [&](auto b) {
        constexpr bool kB = decltype(b)::value;
        if (L.args.head_dim <= 64) return eight ? plan_few<64, kB, 1>(L, stream) : plan_few<64, kB, 2>(L, stream);
        return eight ? plan_few<128, kB, 1>(L, stream) : plan_few<128, kB, 2>(L, stream);
    };
    return bf16 ? go(std::true_type{}) : go(std::false_type{});
}

cudaError_t launch_sdpa_window(const SdpaWindowArgs& a, int num_heads, int batch, bool bf16, cudaStream_t stream) {
    const int lq = a.q_rows[0] + a.q_rows[1];
    const dim3 grid(static_cast<unsigned>((lq + kWinWarps - 1) / kWinWarps), static_cast<unsigned>(num_heads),
                    static_cast<unsigned>(batch));
    return launch_dependent(bf16 ? sdpa_window_kernel<true> : sdpa_window_kernel<false>, grid, dim3(kWinWarps * 32), 0, stream, a);
}

}  // namespace bdattn
