// Second translation unit of libbdattn.so, compiled beside the first: the operators of a layer in 4 bits.  None of
// its kernels waits on a barrier of another agent, so none reports a status.
#define BDATTN_UNIT_WITHOUT_WAITS
#include "tc05.cuh"
#include "sandwich_norm.cu"
#include "w4_linear.cu"
#include "cache4.cu"
#include "sdpa_cache4.cu"
