// C-ABI layer of the operators of a causal pre-norm layer: argument validation and
// dispatch, with the helpers of capi.cu (one translation unit).
#include "../../include/bdattn.h"

#include "sdpa_internal.h"
#include "tc05.cuh"

namespace {

bool is_16bit(int dtype) { return dtype == BDATTN_BF16 || dtype == BDATTN_F16; }
bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

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

}  // extern "C"
