// Causal attention with a sliding window and visible first keys (sinks), a warp per row and
// head: any head_dim up to 256.
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

}  // namespace

cudaError_t launch_sdpa_window(const SdpaWindowArgs& a, int num_heads, int batch, bool bf16, cudaStream_t stream) {
    const int lq = a.q_rows[0] + a.q_rows[1];
    const dim3 grid(static_cast<unsigned>((lq + kWinWarps - 1) / kWinWarps), static_cast<unsigned>(num_heads),
                    static_cast<unsigned>(batch));
    return launch_dependent(bf16 ? sdpa_window_kernel<true> : sdpa_window_kernel<false>, grid, dim3(kWinWarps * 32), 0, stream, a);
}

}  // namespace bdattn
