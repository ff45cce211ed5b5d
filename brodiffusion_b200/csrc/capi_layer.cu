// C-ABI layer of the operators of a causal pre-norm layer: argument validation and
// dispatch, with the helpers of capi.cu (one translation unit).
#include "../../include/bdattn.h"

#include "sdpa_internal.h"
#include "tc05.cuh"

namespace {

bool is_16bit(int dtype) { return dtype == BDATTN_BF16 || dtype == BDATTN_F16; }
bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Rows up to which a product goes to the kernel for few rows.
constexpr int kFewRowsMost = 16;
constexpr int kFewColsMost = 16 * 65535;      // its grid

// Whether a call with a window goes to the kernel for few query rows.  Up to 64 rows that share a K/V head it always
// does: the tensor-core kernel computes 128 rows of a single head whatever they are, and its CTAs walk the keys alone (8
// K/V heads of 128 with 24 query heads, 63 rows and 66, that is 21 tokens and 22: 300 keys 7.3 us and 8.4, 4000 keys 12.2 and 44.6; 8
// sequences of 4000 keys 49.9 and 89.7).  More rows go there as long as each sixteen of them have an SM, so that
// clusters can share their keys, and the modelled time is the lower one (few rows and tensor-core kernel: 8 query heads over 2 K/V
// heads of 128, 128 tokens over 16000 keys 47 and 159 us; 64 heads' tokens over 1000 keys 7.5 and 14.3; 64 tokens by themselves 5.7 and
// 5.6; with more CTAs than SMs 1000 tokens of 24 heads 68 and 18, 858 tokens of 2 x 3 heads 22 and 13).
bool few_rows(const bdattn::SdpaWindowArgs& g, int num_heads, int num_kv_heads, int batch) {
    const int sms = bdattn::sm_count(), lq = g.q_rows[0], lk = g.kv_rows[0] + g.kv_rows[1];
    const long long rows = static_cast<long long>(lq) * g.kv_group, tiles = num_kv_heads * ((rows + 15) / 16), units = batch * tiles;
    if (g.q_rows[1] > 0 || tiles > 65535) return false;
    if (rows <= 64) return true;
    if (units > sms) return false;
    // keys that sixteen rows see on average, and those that the 128 or 256 of the other kernel's CTA with the most see
    auto seen = [&](double keys, int more) { return g.window > 0 && 1.0 * g.window + g.sinks + more < keys ? 1.0 * g.window + g.sinks + more : keys; };
    const double few = 4.0 + 0.45 * (g.head_dim > 64 ? 1.0 : 0.7) * units * (seen(lk - 0.5 * lq, 16) / 64 + 0.5) / sms;
    const double pairs = 1.0 * batch * num_heads * ((lq + 255) / 256), singles = 1.0 * batch * num_heads * ((lq + 127) / 128);
    const bool lone = 2 * pairs <= sms;           // (its CTAs have one query tile each then: launch_t in sdpa_tc05.cu)
    const double steps = seen(lk, lone ? 128 : 256) / 128 + 1;
    return few < 4.0 + std::ceil((lone ? singles : pairs) / sms) * (2.0 + steps * (lone ? 1.2 : 1.45));
}

// The tensor-core attention kernel's arguments for a call with a window: head_dim <= 128.
int window_launch(const char* op, bdattn::SdpaLaunch& L, const bdattn::SdpaWindowArgs& g, int num_heads, int num_kv_heads, int batch,
                  bool bf16) {
    std::memset(&L, 0, sizeof(L));
    bdattn::SdpaDevArgs& a = L.args;
    for (int s = 0; s < 2; ++s) {
        // (a second segment that does not exist has the first one's maps and no rows)
        const int q = g.q_rows[s] > 0 ? s : 0, k = g.kv_rows[s] > 0 ? s : 0;
        if (make_map_heads(op, &L.tmQ[s], g.q[q], bf16, g.head_dim, num_heads, g.q_rows[q], batch, g.q_ld[q], g.q_bs[q], 128) ||
            make_map_heads(op, &L.tmK[s], g.k[k], bf16, g.head_dim, num_kv_heads, g.kv_rows[k], batch, g.k_ld[k], g.k_bs[k], 128) ||
            make_map_heads(op, &L.tmV[s], g.v[k], bf16, g.head_dim, num_kv_heads, g.kv_rows[k], batch, g.v_ld[k], g.v_bs[k], 128))
            return -1;
        a.q_rows[s] = g.q_rows[s];
        a.kv_rows[s] = g.kv_rows[s];
        a.o[s] = g.o[s];
        a.o_ld[s] = g.o_ld[s];
        a.o_bs[s] = g.o_bs[s];
    }
    a.q_ctas0 = (a.q_rows[0] + 255) / 256;
    a.kv_tiles0 = (a.kv_rows[0] + 127) / 128;
    a.kv_tiles = a.kv_tiles0 + (a.kv_rows[1] + 127) / 128;
    a.mask_mode = 1;
    a.q_offset = g.q_offset;
    a.lq_total = g.q_rows[0] + g.q_rows[1];
    a.hd_out = g.head_dim;
    a.kv_group = g.kv_group;
    a.key_mask = g.key_mask;
    a.scale_log2 = g.scale * 1.4426950408889634f;
    L.window = &g;
    L.q_ctas = a.q_ctas0 + (a.q_rows[1] + 255) / 256;
    L.num_heads = num_heads;
    L.batch = batch;
    L.head_dim = g.head_dim <= 64 ? 64 : 128;
    L.bf16 = bf16;
    return 0;
}

}  // namespace

extern "C" {

int bdattn_add_rmsnorm_fwd(const bdattn_add_rmsnorm_params* p, bdattn_stream_t stream) {
    const char* op = "bdattn_add_rmsnorm_fwd";
    if (p == nullptr) return fail("%s: params is null", op);
    if (require_sm100(op)) return -1;
    if (!is_16bit(p->dtype)) return fail("%s: dtype must be BF16 or F16 (got %d)", op, p->dtype);
    const bool fp8 = p->out_dtype == BDATTN_E4M3;
    if (!fp8 && p->out_dtype != p->dtype) return fail("%s: out_dtype must be dtype or E4M3 (got %d)", op, p->out_dtype);
    if (p->rows < 0 || p->cols < 1) return fail("%s: rows must be >= 0 and cols >= 1 (got %d and %d)", op, p->rows, p->cols);
    // (a thread's column goes on by 8192 past the last one)
    if (p->cols > INT32_MAX - 8192) return fail("%s: more than 2^31 - 8193 columns (got %d)", op, p->cols);
    if (p->rows == 0) return 0;
    if (p->x == nullptr || p->out == nullptr) return fail("%s: x/out is null", op);
    if (fp8 && p->out_scale == nullptr) return fail("%s: E4M3 output needs out_scale", op);
    if (!fp8 && p->out_scale != nullptr) return fail("%s: out_scale goes with E4M3 output only", op);
    if (p->gain != nullptr && p->gain_dtype != BDATTN_F32 && p->gain_dtype != p->dtype)
        return fail("%s: gain_dtype must be F32 or dtype (got %d)", op, p->gain_dtype);
    bdattn::AddRmsNormArgs a;
    std::memset(&a, 0, sizeof(a));
    a.rows = p->rows; a.cols = p->cols;
    a.ldx = p->x_ld != 0 ? p->x_ld : p->cols;
    a.ldr = p->residual_ld != 0 ? p->residual_ld : p->cols;
    a.ldro = p->residual_out_ld != 0 ? p->residual_out_ld : p->cols;
    a.ldo = p->out_ld != 0 ? p->out_ld : p->cols;
    if (a.ldx < p->cols || a.ldo < p->cols || (p->residual != nullptr && a.ldr < p->cols) ||
        (p->residual_out != nullptr && a.ldro < p->cols))
        return fail("%s: a row stride is smaller than the %d columns", op, p->cols);
    if (!aligned_to(p->x, 2) || !aligned_to(p->residual, 2) || !aligned_to(p->residual_out, 2) ||
        (!fp8 && !aligned_to(p->out, 2)) || !aligned_to(p->out_scale, 4) ||
        !aligned_to(p->gain, p->gain_dtype == BDATTN_F32 ? 4 : 2))
        return fail("%s: a tensor is not aligned to its element type", op);
    if (!(p->eps >= 0.0f)) return fail("%s: eps must be >= 0", op);
    a.x = p->x; a.residual = p->residual; a.residual_out = p->residual_out;
    a.gain = p->gain; a.gain_is_f32 = p->gain_dtype == BDATTN_F32 ? 1 : 0;
    a.out = p->out; a.out_scale = p->out_scale;
    a.eps = p->eps;
    cudaError_t e = bdattn::launch_add_rmsnorm(a, p->dtype == BDATTN_BF16, fp8, reinterpret_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(op, e);
    return 0;
}

int bdattn_linear_act_fwd(const bdattn_linear_act_params* p, bdattn_stream_t stream) {
    const char* op = "bdattn_linear_act_fwd";
    if (p == nullptr) return fail("%s: params is null", op);
    if (require_sm100(op)) return -1;
    if (!is_16bit(p->dtype)) return fail("%s: dtype must be BF16 or F16 (got %d)", op, p->dtype);
    const bool fp8 = p->in_dtype == BDATTN_E4M3;
    if (!fp8 && p->in_dtype != p->dtype) return fail("%s: in_dtype must be dtype or E4M3 (got %d)", op, p->in_dtype);
    if (!fp8 && (p->x_scale != nullptr || p->w_scale != nullptr)) return fail("%s: scales go with E4M3 operands only", op);
    if (p->act < BDATTN_ACT_NONE || p->act > BDATTN_ACT_SILU) return fail("%s: unknown activation %d", op, p->act);
    if (p->M < 0 || p->N < 1 || p->K < 1) return fail("%s: M must be >= 0, N and K >= 1 (got %d, %d, %d)", op, p->M, p->N, p->K);
    if (p->M == 0) return 0;
    const long long ldx = p->x_ld != 0 ? p->x_ld : p->K, ldw = p->w_ld != 0 ? p->w_ld : p->K;
    const long long ldr = p->residual_ld != 0 ? p->residual_ld : p->N, ldy = p->y_ld != 0 ? p->y_ld : p->N;
    if (fp8 && (p->K % 16 != 0 || ldx % 16 != 0 || ldw % 16 != 0))
        return fail("%s: inner size and row strides of E4M3 operands must be multiples of 16 (K=%d ldx=%lld ldw=%lld)", op, p->K, ldx, ldw);
    if (p->residual != nullptr && (ldr < p->N || ldr % 8 != 0 || !aligned16(p->residual)))
        return fail("%s: residual must be 16-byte aligned with a row stride of at least N and a multiple of 8 (got %lld)", op, ldr);
    if (!aligned_to(p->bias, 2) || !aligned_to(p->gate, 2) || !aligned_to(p->x_scale, 4) || !aligned_to(p->w_scale, 4))
        return fail("%s: bias, gate or scales are not aligned to their element type", op);
    bdattn::GemmLaunch L;
    std::memset(&L, 0, sizeof(L));
    L.bf16 = p->dtype == BDATTN_BF16;
    L.layer = true;
    L.fp8 = fp8;
    const int half = fp8 ? 2 : 1;        // e4m3 operands go through the 16-bit tensor maps in pairs
    if (add_gemm_problem(op, L, 0, p->x, ldx / half, p->w, ldw / half, p->bias, p->y, ldy, p->M, p->N, p->K / half, 0, 0)) return -1;
    bdattn::GemmProblem& g = L.args.p[0];
    g.act = p->act;
    g.gate = p->gate;
    g.residual = p->residual;
    g.ldr = ldr;
    g.x_scale = p->x_scale;
    g.w_scale = p->w_scale;
    if (p->M <= kFewRowsMost && p->N <= kFewColsMost) {
        const cudaError_t e = bdattn::launch_gemm_few(L, p->x, ldx / half, reinterpret_cast<cudaStream_t>(stream));
        return e != cudaSuccess ? cuda_fail(op, e) : 0;
    }
    return launch_gemm(op, L, 1, reinterpret_cast<cudaStream_t>(stream));
}

int bdattn_sdpa_window_fwd(const bdattn_sdpa_params* p, const bdattn_window_params* w, bdattn_stream_t stream) {
    const char* op = "flash_attention_windowed_forward";
    if (p == nullptr || w == nullptr) return fail("%s: params is null", op);
    if (require_sm100(op)) return -1;
    if (!is_16bit(p->dtype)) return fail("%s: dtype must be BF16 or F16 (got %d)", op, p->dtype);
    if (w->window < 0 || w->sinks < 0) return fail("%s: window and sinks must be >= 0 (got %d and %d)", op, w->window, w->sinks);
    if (p->mask_mode != BDATTN_MASK_CAUSAL) return fail("%s: mask_mode must be CAUSAL (got %d)", op, p->mask_mode);
    if (p->key_scale != nullptr || p->val_scale != nullptr) return fail("%s: per-key scales are not taken with a window", op);
    if (p->q_gain[0] != nullptr || p->q_gain[1] != nullptr || p->q_cos != nullptr || p->q_sin != nullptr)
        return fail("%s: query norm and RoPE are not taken with a window (bdattn_rmsnorm_rope ahead of it)", op);
    if (p->batch < 1 || p->num_heads < 1 || p->batch > 65535 || p->num_heads > 65535)
        return fail("%s: batch and num_heads must be in [1, 65535] (got %d and %d)", op, p->batch, p->num_heads);
    const int hd = p->head_dim;
    if (hd < 8 || hd > 256 || hd % 8 != 0) return fail("%s: head_dim must be a multiple of 8 in [8, 256] (got %d)", op, hd);
    const int nkv = p->num_kv_heads > 0 ? p->num_kv_heads : p->num_heads;
    if (p->num_kv_heads < 0 || p->num_heads % nkv != 0)
        return fail("%s: num_kv_heads must divide num_heads (got %d and %d)", op, p->num_kv_heads, p->num_heads);
    if (p->n_q_seg < 1 || p->n_q_seg > 2 || p->n_kv_seg < 1 || p->n_kv_seg > 2)
        return fail("%s: n_q_seg and n_kv_seg must be 1 or 2", op);
    if (!aligned_to(p->key_mask, 4) || !aligned_to(w->kv_len, 4)) return fail("%s: key_mask and kv_len must be 4-byte aligned", op);
    bdattn::SdpaWindowArgs g;
    std::memset(&g, 0, sizeof(g));
    const long long D = static_cast<long long>(p->num_heads) * hd, Dkv = static_cast<long long>(nkv) * hd;
    long long lq = 0, lk = 0;
    // one operand of a segment: its checks, and the stride between batch items that 0 stands for
    auto rows_of = [&](const char* what, int s, const void* ptr, int rows, long long ld, long long stride, long long cols,
                       long long* out) {
        if (ptr == nullptr) return fail("%s: %s segment %d is null", op, what, s);
        if (rows < 1) return fail("%s: %s segment %d has no rows", op, what, s);
        if (ld < cols) return fail("%s: the row stride of %s segment %d is smaller than its %lld columns", op, what, s, cols);
        if (ld % 8 != 0 || stride % 8 != 0 || !aligned16(ptr))
            return fail("%s: %s segment %d must be 16-byte aligned with strides that are multiples of 8 elements", op, what, s);
        *out = stride > 0 ? stride : rows * ld;
        return 0;
    };
    for (int s = 0; s < p->n_q_seg; ++s) {
        if (rows_of("q", s, p->q[s], p->q_rows[s], p->q_ld[s], p->q_batch_stride[s], D, &g.q_bs[s]) ||
            rows_of("o", s, p->o[s], p->q_rows[s], p->o_ld[s], p->o_batch_stride[s], D, &g.o_bs[s]))
            return -1;
        g.q[s] = p->q[s]; g.o[s] = p->o[s]; g.q_rows[s] = p->q_rows[s]; g.q_ld[s] = p->q_ld[s]; g.o_ld[s] = p->o_ld[s];
        lq += p->q_rows[s];
    }
    for (int s = 0; s < p->n_kv_seg; ++s) {
        if (rows_of("k", s, p->k[s], p->kv_rows[s], p->k_ld[s], p->k_batch_stride[s], Dkv, &g.k_bs[s]) ||
            rows_of("v", s, p->v[s], p->kv_rows[s], p->v_ld[s], p->v_batch_stride[s], Dkv, &g.v_bs[s]))
            return -1;
        g.k[s] = p->k[s]; g.v[s] = p->v[s]; g.kv_rows[s] = p->kv_rows[s]; g.k_ld[s] = p->k_ld[s]; g.v_ld[s] = p->v_ld[s];
        lk += p->kv_rows[s];
    }
    // positions and key numbers are 32-bit: n - Lq + i, P - window
    if (lq > (1 << 30) || lk > (1 << 30)) return fail("%s: more than 2^30 query or key rows", op);
    g.mask_mode = 1;
    g.q_offset = static_cast<int>(lk - lq);
    g.head_dim = hd;
    g.kv_group = p->num_heads / nkv;
    g.key_mask = p->key_mask;
    g.scale = p->softmax_scale > 0.0f ? p->softmax_scale : 1.0f / std::sqrt(static_cast<float>(hd));
    // a window, or sinks, of all keys is no window: from here on both are below 2^30
    g.window = w->window >= lk || w->sinks >= lk ? 0 : w->window;
    g.sinks = w->sinks < lk ? w->sinks : static_cast<int>(lk);
    g.kv_len = w->kv_len;
    const bool bf16 = p->dtype == BDATTN_BF16;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (hd <= 128 && few_rows(g, p->num_heads, nkv, p->batch)) {
        bdattn::SdpaFewLaunch L;
        for (int s = 0; s < 2; ++s) {
            const int k = s < p->n_kv_seg ? s : 0;
            if (make_map_heads(op, &L.tmK[s], g.k[k], bf16, hd, nkv, g.kv_rows[k], p->batch, g.k_ld[k], g.k_bs[k], 64) ||
                make_map_heads(op, &L.tmV[s], g.v[k], bf16, hd, nkv, g.kv_rows[k], p->batch, g.v_ld[k], g.v_bs[k], 64))
                return -1;
        }
        L.args = g;
        L.num_kv_heads = nkv;
        L.batch = p->batch;
        e = bdattn::launch_sdpa_few(L, bf16, st);
    } else if (hd <= 128) {
        bdattn::SdpaLaunch L;
        if (window_launch(op, L, g, p->num_heads, nkv, p->batch, bf16)) return -1;
        e = bdattn::launch_sdpa_tc05(L, st);
    } else {
        e = bdattn::launch_sdpa_window(g, p->num_heads, p->batch, bf16, st);
    }
    if (e != cudaSuccess) return cuda_fail(op, e);
    return 0;
}

}  // extern "C"
