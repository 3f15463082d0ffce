// Sampling from float16 support.
#include "sbb_sample.cuh"

namespace sbb {
template cudaError_t launch_sample<__half>(const __half *, const float *, long, long, long, Sampling, long long *, cudaStream_t);
}  // namespace sbb
