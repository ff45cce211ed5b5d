// C-ABI layer of the operators of a layer in 4 bits: argument validation and dispatch, with the helpers of capi.cu
// and capi_layer.cu (one translation unit).
#include "../../include/bdattn.h"

#include "sdpa_internal.h"
#include "tc05.cuh"

namespace {

bool is_group(int group) { return group == 32 || group == 64 || group == 128; }

// The cache of a call: its checks and its strides.
int cache4_of(const char* op, const bdattn_cache4* c, bdattn::Cache4Dev* d) {
    if (c == nullptr) return fail("%s: cache is null", op);
    if (!is_16bit(c->dtype)) return fail("%s: dtype must be BF16 or F16 (got %d)", op, c->dtype);
    if (c->batch < 1 || c->batch > 65535 || c->num_kv_heads < 1 || c->num_kv_heads > 32767)
        return fail("%s: batch must be in [1, 65535], num_kv_heads in [1, 32767] (got %d and %d)", op, c->batch, c->num_kv_heads);
    if (c->head_dim != 64 && c->head_dim != 128) return fail("%s: head_dim must be 64 or 128 (got %d)", op, c->head_dim);
    if (!is_group(c->group) || c->group > c->head_dim)
        return fail("%s: group must be 32, 64 or 128 and no larger than head_dim (got %d)", op, c->group);
    if (c->rows < 1 || c->rows > (1 << 30)) return fail("%s: the cache must have between 1 and 2^30 rows (got %d)", op, c->rows);
    if (c->k_codes == nullptr || c->v_codes == nullptr || c->k_scales == nullptr || c->v_scales == nullptr)
        return fail("%s: a tensor of the cache is null", op);
    const long long code = c->head_dim / 2, scale = 2 * (c->head_dim / c->group);
    d->codes_hs = c->codes_head_stride != 0 ? c->codes_head_stride : c->rows * code;
    d->scales_hs = c->scales_head_stride != 0 ? c->scales_head_stride : c->rows * scale;
    d->codes_bs = c->codes_batch_stride != 0 ? c->codes_batch_stride : c->num_kv_heads * d->codes_hs;
    d->scales_bs = c->scales_batch_stride != 0 ? c->scales_batch_stride : c->num_kv_heads * d->scales_hs;
    // (what is behind the strides may lie either way round, but no two heads in the same memory)
    auto apart = [&](long long hs, long long bs, long long row) {
        const long long one = c->rows * row;
        if (c->num_kv_heads == 1 && c->batch == 1) return true;
        if (c->num_kv_heads == 1) return bs >= one;
        if (c->batch == 1) return hs >= one;
        return (hs >= one && bs / c->num_kv_heads >= hs) || (bs >= one && hs / c->batch >= bs);
    };
    if (!apart(d->codes_hs, d->codes_bs, code) || !apart(d->scales_hs, d->scales_bs, scale))
        return fail("%s: the cache's strides must be those of heads and batch items that do not overlap", op);
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || d->codes_hs % 16 != 0 || d->codes_bs % 16 != 0)
        return fail("%s: codes must be 16-byte aligned with strides that are multiples of 16", op);
    if (!aligned_to(c->k_scales, 2 * scale) || !aligned_to(c->v_scales, 2 * scale) || d->scales_hs % scale != 0 || d->scales_bs % scale != 0)
        return fail("%s: scales must be aligned to a row's pairs (%lld bytes), their strides too", op, 2 * scale);
    d->k_codes = static_cast<uint8_t*>(c->k_codes);
    d->v_codes = static_cast<uint8_t*>(c->v_codes);
    d->k_scales = static_cast<uint16_t*>(c->k_scales);
    d->v_scales = static_cast<uint16_t*>(c->v_scales);
    d->rows = c->rows;
    d->kv_heads = c->num_kv_heads;
    d->head_dim = c->head_dim;
    d->group = c->group;
    return 0;
}

// One 16-bit operand of a call on a cache: its checks, and what its strides of 0 stand for.
int cache4_operand(const char* op, const char* what, const void* p, int rows, int batch, long long cols, long long ld_in, long long bs_in,
                   long long* ld, long long* bs) {
    if (p == nullptr) return fail("%s: %s is null", op, what);
    *ld = ld_in != 0 ? ld_in : cols;
    *bs = bs_in != 0 ? bs_in : rows * *ld;
    if (*ld < cols) return fail("%s: the row stride of %s is smaller than its %lld columns", op, what, cols);
    if (*ld % 8 != 0 || *bs % 8 != 0 || !aligned16(p))
        return fail("%s: %s must be 16-byte aligned with strides that are multiples of 8 elements", op, what);
    if (batch > 1 && *bs < 0) return fail("%s: the batch stride of %s is negative", op, what);
    return 0;
}

int cache4_rows(const char* op, const bdattn_cache4* c, const bdattn_cache4_rows* r, bool append, bdattn_stream_t stream) {
    bdattn::Cache4RowsArgs a;
    std::memset(&a, 0, sizeof(a));
    if (require_sm100(op)) return -1;
    if (cache4_of(op, c, &a.c)) return -1;
    if (r == nullptr) return fail("%s: rows is null", op);
    if (r->rows < 0 || r->rows > (1 << 30)) return fail("%s: rows must be in [0, 2^30] (got %d)", op, r->rows);
    if (r->rows == 0) return 0;
    const long long cols = static_cast<long long>(c->num_kv_heads) * c->head_dim;
    if (cache4_operand(op, "k", r->k, r->rows, c->batch, cols, r->k_ld, r->k_batch_stride, &a.k_ld, &a.k_bs) ||
        cache4_operand(op, "v", r->v, r->rows, c->batch, cols, r->v_ld, r->v_batch_stride, &a.v_ld, &a.v_bs))
        return -1;
    if (!aligned_to(r->kv_len, 4)) return fail("%s: kv_len must be 4-byte aligned", op);
    a.k = r->k;
    a.v = r->v;
    a.n_rows = r->rows;
    a.kv_len = r->kv_len;
    a.batch = c->batch;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool bf16 = c->dtype == BDATTN_BF16;
    const cudaError_t e = append ? bdattn::launch_cache4_append(a, bf16, st) : bdattn::launch_cache4_read(a, bf16, st);
    return e != cudaSuccess ? cuda_fail(op, e) : 0;
}

}  // namespace

extern "C" {

int bdattn_sandwich_norm_fwd(const bdattn_sandwich_norm_params* p, bdattn_stream_t stream) {
    const char* op = "bdattn_sandwich_norm_fwd";
    if (p == nullptr) return fail("%s: params is null", op);
    if (require_sm100(op)) return -1;
    if (!is_16bit(p->dtype)) return fail("%s: dtype must be BF16 or F16 (got %d)", op, p->dtype);
    const bool fp8 = p->out != nullptr && p->out_dtype == BDATTN_E4M3;
    if (p->out != nullptr && !fp8 && p->out_dtype != p->dtype) return fail("%s: out_dtype must be dtype or E4M3 (got %d)", op, p->out_dtype);
    if (p->rows < 0 || p->cols < 1) return fail("%s: rows must be >= 0 and cols >= 1 (got %d and %d)", op, p->rows, p->cols);
    // (a thread's column goes on by 1024 past the last one)
    if (p->cols > INT32_MAX - 8192) return fail("%s: more than 2^31 - 8193 columns (got %d)", op, p->cols);
    if (p->rows == 0) return 0;
    if (p->x == nullptr || p->residual == nullptr || p->residual_out == nullptr) return fail("%s: x/residual/residual_out is null", op);
    if (fp8 && p->out_scale == nullptr) return fail("%s: E4M3 output needs out_scale", op);
    if (!fp8 && p->out_scale != nullptr) return fail("%s: out_scale goes with E4M3 output only", op);
    if (p->out == nullptr && p->gain != nullptr) return fail("%s: gain goes with out", op);
    if ((p->gain != nullptr || p->post_gain != nullptr) && p->gain_dtype != BDATTN_F32 && p->gain_dtype != p->dtype)
        return fail("%s: gain_dtype must be F32 or dtype (got %d)", op, p->gain_dtype);
    if (p->gate != nullptr && (p->gates < 1 || p->rows % p->gates != 0))
        return fail("%s: gates must divide the %d rows (got %d)", op, p->rows, p->gates);
    if (!(std::fabs(p->residual_scale) <= FLT_MAX)) return fail("%s: residual_scale must be finite", op);
    if (!(p->eps >= 0.0f)) return fail("%s: eps must be >= 0", op);
    bdattn::SandwichNormArgs a;
    std::memset(&a, 0, sizeof(a));
    a.rows = p->rows;
    a.cols = p->cols;
    a.ldx = p->x_ld != 0 ? p->x_ld : p->cols;
    a.ldr = p->residual_ld != 0 ? p->residual_ld : p->cols;
    a.ldro = p->residual_out_ld != 0 ? p->residual_out_ld : p->cols;
    a.ldo = p->out_ld != 0 ? p->out_ld : p->cols;
    a.ldg = p->gate_ld != 0 ? p->gate_ld : p->cols;
    if (a.ldx < p->cols || a.ldr < p->cols || a.ldro < p->cols || (p->out != nullptr && a.ldo < p->cols) ||
        (p->gate != nullptr && p->gates > 1 && a.ldg < p->cols))
        return fail("%s: a row stride is smaller than the %d columns", op, p->cols);
    const size_t gain_bytes = p->gain_dtype == BDATTN_F32 ? 4 : 2;
    if (!aligned_to(p->x, 2) || !aligned_to(p->residual, 2) || !aligned_to(p->residual_out, 2) || (!fp8 && !aligned_to(p->out, 2)) ||
        !aligned_to(p->out_scale, 4) || !aligned_to(p->gate, 2) || !aligned_to(p->gain, gain_bytes) || !aligned_to(p->post_gain, gain_bytes))
        return fail("%s: a tensor is not aligned to its element type", op);
    a.x = p->x;
    a.residual = p->residual;
    a.residual_out = p->residual_out;
    a.post_gain = p->post_gain;
    a.gain = p->gain;
    a.gain_is_f32 = p->gain_dtype == BDATTN_F32 ? 1 : 0;
    a.gate = p->gate;
    a.gate_rows = p->gate != nullptr ? p->rows / p->gates : 1;
    a.out = p->out;
    a.out_scale = p->out_scale;
    a.residual_scale = p->residual_scale;
    a.eps = p->eps;
    const cudaError_t e = bdattn::launch_sandwich_norm(a, p->dtype == BDATTN_BF16, reinterpret_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? cuda_fail(op, e) : 0;
}

size_t bdattn_w4_bytes(int N, int K, int group) {
    if (N < 1 || K < 1 || !is_group(group)) return 0;
    return static_cast<size_t>((N + 15ll) / 16) * ((K + 127ll) / 128) * (1024 + 16 * (128 / group) * 4);
}

int bdattn_w4_pack(const void* codes, long long codes_ld, const void* scales, long long scales_ld, void* packed, int N, int K,
                   int group, bdattn_stream_t stream) {
    const char* op = "bdattn_w4_pack";
    if (require_sm100(op)) return -1;
    if (!is_group(group)) return fail("%s: group must be 32, 64 or 128 (got %d)", op, group);
    if (N < 1 || K < 1 || K % 8 != 0 || K > (1 << 30)) return fail("%s: N must be >= 1 and K a multiple of 8 up to 2^30 (got %d and %d)", op, N, K);
    if (codes == nullptr || scales == nullptr || packed == nullptr) return fail("%s: codes/scales/packed is null", op);
    bdattn::W4PackArgs a;
    const long long groups = (static_cast<long long>(K) + group - 1) / group;
    a.codes_ld = codes_ld != 0 ? codes_ld : K / 2;
    a.scales_ld = scales_ld != 0 ? scales_ld : 2 * groups;
    if (a.codes_ld < K / 2 || a.scales_ld < 2 * groups) return fail("%s: a row stride is smaller than a row", op);
    if (!aligned16(packed) || !aligned_to(scales, 2)) return fail("%s: packed must be 16-byte aligned, scales 2-byte", op);
    a.codes = static_cast<const uint8_t*>(codes);
    a.scales = scales;
    a.packed = packed;
    a.N = N;
    a.K = K;
    a.group = group;
    a.k_tiles = static_cast<int>((K + 127ll) / 128);
    const cudaError_t e = bdattn::launch_w4_pack(a, reinterpret_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? cuda_fail(op, e) : 0;
}

int bdattn_w4_unpack(const void* packed, void* w, long long w_ld, int N, int K, int group, int dtype, bdattn_stream_t stream) {
    const char* op = "bdattn_w4_unpack";
    if (require_sm100(op)) return -1;
    if (!is_16bit(dtype)) return fail("%s: dtype must be BF16 or F16 (got %d)", op, dtype);
    if (!is_group(group)) return fail("%s: group must be 32, 64 or 128 (got %d)", op, group);
    if (N < 1 || K < 1 || K % 8 != 0 || K > (1 << 30)) return fail("%s: N must be >= 1 and K a multiple of 8 up to 2^30 (got %d and %d)", op, N, K);
    if (packed == nullptr || w == nullptr) return fail("%s: packed/w is null", op);
    bdattn::W4UnpackArgs a;
    a.ld = w_ld != 0 ? w_ld : K;
    if (a.ld < K) return fail("%s: a row stride is smaller than a row", op);
    if (a.ld % 8 != 0 || !aligned16(packed) || !aligned16(w))
        return fail("%s: packed and w must be 16-byte aligned, the row stride of w a multiple of 8 (got %lld)", op, a.ld);
    a.packed = static_cast<const uint8_t*>(packed);
    a.w = static_cast<uint16_t*>(w);
    a.N = N;
    a.K = K;
    a.group = group;
    a.k_tiles = (K - 1) / 128 + 1;
    const cudaError_t e = bdattn::launch_w4_unpack(a, dtype == BDATTN_BF16, reinterpret_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? cuda_fail(op, e) : 0;
}

int bdattn_linear_w4_fwd(const bdattn_linear_w4_params* p, bdattn_stream_t stream) {
    const char* op = "bdattn_linear_w4_fwd";
    if (p == nullptr) return fail("%s: params is null", op);
    if (require_sm100(op)) return -1;
    if (!is_16bit(p->dtype)) return fail("%s: dtype must be BF16 or F16 (got %d)", op, p->dtype);
    if (!is_group(p->group)) return fail("%s: group must be 32, 64 or 128 (got %d)", op, p->group);
    if (p->act < BDATTN_ACT_NONE || p->act > BDATTN_ACT_SILU) return fail("%s: unknown activation %d", op, p->act);
    if (p->M < 0 || p->N < 1 || p->K < 1 || p->K % 8 != 0)
        return fail("%s: M must be >= 0, N >= 1 and K a multiple of 8 (got %d, %d, %d)", op, p->M, p->N, p->K);
    // (a tile's columns go on past the last one; eight rows are a pass in the grid's second dimension)
    if (p->K > (1 << 30) || p->M > 8 * 65535) return fail("%s: more than 2^30 columns or 524280 rows (got %d and %d)", op, p->K, p->M);
    if (p->M == 0) return 0;
    if (p->x == nullptr || p->w == nullptr || p->y == nullptr) return fail("%s: x/w/y is null", op);
    bdattn::GemmProblem g;
    std::memset(&g, 0, sizeof(g));
    const long long ldx = p->x_ld != 0 ? p->x_ld : p->K;
    g.ldr = p->residual_ld != 0 ? p->residual_ld : p->N;
    g.ldc = p->y_ld != 0 ? p->y_ld : p->N;
    if (ldx < p->K || g.ldc < p->N || (p->residual != nullptr && g.ldr < p->N)) return fail("%s: a row stride is smaller than a row", op);
    if (ldx % 8 != 0 || !aligned16(p->x) || !aligned16(p->w))
        return fail("%s: x and w must be 16-byte aligned, the row stride of x a multiple of 8 (got %lld)", op, ldx);
    if (!aligned_to(p->y, 2) || !aligned_to(p->bias, 2) || !aligned_to(p->gate, 2) || !aligned_to(p->residual, 2))
        return fail("%s: a tensor is not aligned to its element type", op);
    g.M = p->M;
    g.N = p->N;
    g.K = p->K;
    g.C = p->y;
    g.bias = p->bias;
    g.gate = p->gate;
    g.residual = p->residual;
    g.act = p->act;
    const cudaError_t e = bdattn::launch_w4_linear(g, p->x, ldx, p->w, p->group, p->dtype == BDATTN_BF16, reinterpret_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? cuda_fail(op, e) : 0;
}

int bdattn_cache4_append(const bdattn_cache4* c, const bdattn_cache4_rows* r, bdattn_stream_t stream) {
    return cache4_rows("bdattn_cache4_append", c, r, true, stream);
}
int bdattn_cache4_read(const bdattn_cache4* c, const bdattn_cache4_rows* r, bdattn_stream_t stream) {
    return cache4_rows("bdattn_cache4_read", c, r, false, stream);
}

int bdattn_sdpa_cache4_fwd(const bdattn_cache4* c, const bdattn_sdpa_cache4_params* p, bdattn_stream_t stream) {
    const char* op = "bdattn_sdpa_cache4_fwd";
    bdattn::SdpaCache4Args a;
    std::memset(&a, 0, sizeof(a));
    if (require_sm100(op)) return -1;
    if (cache4_of(op, c, &a.c)) return -1;
    if (p == nullptr) return fail("%s: params is null", op);
    if (p->num_heads < 1 || p->num_heads > 65535 || p->num_heads % c->num_kv_heads != 0)
        return fail("%s: num_heads must be in [1, 65535] and a multiple of the cache's %d heads (got %d)", op, c->num_kv_heads, p->num_heads);
    if (p->window < 0 || p->sinks < 0) return fail("%s: window and sinks must be >= 0 (got %d and %d)", op, p->window, p->sinks);
    if (p->q_rows < 1) return fail("%s: q has no rows", op);
    const long long cols = static_cast<long long>(p->num_heads) * c->head_dim;
    if (cache4_operand(op, "q", p->q, p->q_rows, c->batch, cols, p->q_ld, p->q_batch_stride, &a.q_ld, &a.q_bs) ||
        cache4_operand(op, "o", p->o, p->q_rows, c->batch, cols, p->o_ld, p->o_batch_stride, &a.o_ld, &a.o_bs))
        return -1;
    if (!aligned_to(p->kv_len, 4) || !aligned_to(p->key_mask, 4)) return fail("%s: key_mask and kv_len must be 4-byte aligned", op);
    a.kv_group = p->num_heads / c->num_kv_heads;
    // positions, rows that share a head and tiles of them are 32-bit
    if (p->q_rows > (1 << 30) / p->num_heads) return fail("%s: more than 2^30 rows of heads", op);
    a.q = p->q;
    a.o = p->o;
    a.lq = p->q_rows;
    a.batch = c->batch;
    // a window, or sinks, of all keys is no window
    a.window = p->window >= c->rows || p->sinks >= c->rows ? 0 : p->window;
    a.sinks = p->sinks < c->rows ? p->sinks : c->rows;
    a.scale = p->softmax_scale > 0.0f ? p->softmax_scale : 1.0f / std::sqrt(static_cast<float>(c->head_dim));
    a.key_mask = p->key_mask;
    a.kv_len = p->kv_len;
    const cudaError_t e = bdattn::launch_sdpa_cache4(a, c->dtype == BDATTN_BF16, reinterpret_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? cuda_fail(op, e) : 0;
}

}  // extern "C"
