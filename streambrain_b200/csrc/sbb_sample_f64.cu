// Sampling from float64 support.
#include "sbb_sample.cuh"

namespace sbb {
template cudaError_t launch_sample<double>(const double *, const float *, long, long, long, Sampling, long long *, cudaStream_t);
}  // namespace sbb
