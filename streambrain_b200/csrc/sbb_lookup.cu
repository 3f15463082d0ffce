// Support of coded samples and its gradient: sums of the weight rows that codes name, and sums of the gradient's rows by code.
#include "sbb_codes.cuh"
#include "sbb_launch.cuh"

namespace sbb {
namespace {

constexpr int kThreads = 256;

// A block has `lanes` threads across V columns each, and its other threads split the row's codes; the parts are added in order.
template <typename T, typename I, int V>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(const T *__restrict__ weights, const I *__restrict__ codes, long L, long N, long M, Wide<T> scale, T *__restrict__ out, int lanes) {
  after_previous();
  using W = Wide<T>;
  __shared__ W s_part[kThreads * V];
  const int parts = kThreads / lanes, part = threadIdx.x / lanes;
  const long r = blockIdx.x, col = ((long)blockIdx.y * lanes + threadIdx.x % lanes) * V;
  W acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = (W)0;
  if (col < M)
    for (long l = part; l < L; l += parts) {
      const long code = (long)codes[r * L + l];
      if (code < 0 || code >= N) continue;
      const Vec<T, V> w = *reinterpret_cast<const Vec<T, V> *>(weights + code * M + col);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += widen(w.v[v]);
    }
#pragma unroll
  for (int v = 0; v < V; ++v) s_part[threadIdx.x * V + v] = acc[v];
  __syncthreads();
  if (part != 0 || col >= M) return;
  for (int p = 1; p < parts; ++p)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] += s_part[(p * lanes + threadIdx.x) * V + v];
  Vec<T, V> o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.v[v] = narrow_to<T>(acc[v] * scale);
  *reinterpret_cast<Vec<T, V> *>(out + r * M + col) = o;
}

// A warp per weight row: it reads all codes in order and adds the gradient's row for each that names its own.
template <typename T, typename I>
__global__ void __launch_bounds__(kThreads)
    gradient_kernel(const T *__restrict__ grad, const I *__restrict__ codes, long entries, long L, long N, long M, Wide<T> scale, bool accumulate,
                    T *__restrict__ out) {
  after_previous();
  using W = Wide<T>;
  const int lane = threadIdx.x & 31;
  const long i = (long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), col = (long)blockIdx.y * 32 + lane;
  if (i >= N) return;
  W acc = (W)0;
  bool any = false;
  for (long e = 0; e < entries; e += 32) {
    const bool hit = e + lane < entries && (long)codes[e + lane] == i;
    for (unsigned m = __ballot_sync(0xffffffffu, hit); m != 0; m &= m - 1) {
      any = true;
      if (col < M) acc += widen(grad[(e + __ffs(m) - 1) / L * M + col]);
    }
  }
  if (col >= M || (accumulate && !any)) return;
  acc *= scale;
  if (accumulate) acc += widen(out[i * M + col]);
  out[i * M + col] = narrow_to<T>(acc);
}

}  // namespace

template <typename T, typename I>
cudaError_t launch_lookup(const T *weights, const I *codes, long rows, long L, long N, long M, double scale, T *out, cudaStream_t st) {
  const int vec = vector_width<T>(M, weights, out);
  const long across = (M + vec - 1) / vec;
  int lanes = 8;
  while (lanes < kThreads && lanes < across) lanes *= 2;
  const dim3 grid((unsigned)rows, (unsigned)((across + lanes - 1) / lanes));
  const Wide<T> s = (Wide<T>)scale;
  cudaError_t e;
  if (vec == 16 / (int)sizeof(T))
    e = launch_next(lookup_kernel<T, I, 16 / (int)sizeof(T)>, grid, kThreads, 0, st, weights, codes, L, N, M, s, out, lanes);
  else if (sizeof(T) == 2 && vec == 2)
    e = launch_next(lookup_kernel<T, I, 2>, grid, kThreads, 0, st, weights, codes, L, N, M, s, out, lanes);
  else
    e = launch_next(lookup_kernel<T, I, 1>, grid, kThreads, 0, st, weights, codes, L, N, M, s, out, lanes);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

size_t lookup_gradient_workspace(long, long, long, long, size_t) { return 0; }

template <typename T, typename I>
cudaError_t launch_lookup_gradient(const T *grad, const I *codes, long rows, long L, long N, long M, double scale, bool accumulate, T *out,
                                   void *, cudaStream_t st) {
  const dim3 grid((unsigned)((N + kThreads / 32 - 1) / (kThreads / 32)), (unsigned)((M + 31) / 32));
  const cudaError_t e = launch_next(gradient_kernel<T, I>, grid, kThreads, 0, st, grad, codes, rows * L, L, N, M, (Wide<T>)scale, accumulate, out);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

#define SBB_INSTANCE(T, I)                                                                                              \
  template cudaError_t launch_lookup<T, I>(const T *, const I *, long, long, long, long, double, T *, cudaStream_t);    \
  template cudaError_t launch_lookup_gradient<T, I>(const T *, const I *, long, long, long, long, double, bool, T *, void *, cudaStream_t);
#define SBB_INSTANCES(T) SBB_INSTANCE(T, int32_t) SBB_INSTANCE(T, int64_t)
SBB_INSTANCES(float)
SBB_INSTANCES(double)
SBB_INSTANCES(__half)
SBB_INSTANCES(__nv_bfloat16)

}  // namespace sbb
