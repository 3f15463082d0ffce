// Sampling from bfloat16 support.
#include "sbb_sample.cuh"

namespace sbb {
template cudaError_t launch_sample<__nv_bfloat16>(const __nv_bfloat16 *, const float *, long, long, long, Sampling, long long *, cudaStream_t);
}  // namespace sbb
