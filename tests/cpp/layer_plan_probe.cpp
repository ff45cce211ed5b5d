// The plan of a layer's product as a C function, for tests/test_layer_plan.py.
#include "../../brodiffusion_b200/csrc/gemm_plan.h"

extern "C" void probe_layer_plan(int M, int N, int K, int act, int sms, int* out) {
    const bdattn::GemmShape s = {M, N, K, false, false, N % 256 == 0};
    const bdattn::GemmPlan p = bdattn::plan_gemm(&s, 1, sms, act != 0 ? 2 : 1);
    out[0] = p.pair;
    out[1] = p.pair ? p.pair_cols : p.width;
    out[2] = p.split;
}
