// Sampling from float32 support.
#include "sbb_sample.cuh"

namespace sbb {
template cudaError_t launch_sample<float>(const float *, const float *, long, long, long, Sampling, long long *, cudaStream_t);
}  // namespace sbb
