// Distillation from a teacher of which only the best units of each group are kept.
//
// With p the softmax of the teacher's kept units, q the softmax of all of the student's group, both at temperature t, and w the
// row's weight: loss = w t^2 sum_k p_k (log p_k - log q_{u_k}), and d loss / d x_i = w t (q_i - sum over k with u_k = i of p_k).
#include "sbb_codes.cuh"
#include "sbb_launch.cuh"
#include "sbb_math.cuh"

namespace sbb {
namespace {

constexpr int kThreads = 256;

template <typename W>
__device__ __forceinline__ W block_sum(W v, W *s) {
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int i = 1; i < kThreads / 32; ++i) v += s[i];
  return v;
}
template <typename W>
__device__ __forceinline__ W block_max(W v, W *s) {
  for (int off = 16; off > 0; off >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, off));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int i = 1; i < kThreads / 32; ++i) v = fmax(v, s[i]);
  return v;
}

// A block per group.
template <typename T, typename I>
__global__ void __launch_bounds__(kThreads)
    distill_kernel(const T *__restrict__ support, const I *__restrict__ units, const T *__restrict__ teacher, const Wide<T> *__restrict__ weight,
                   long H, long Mc, long K, Wide<T> temperature, Wide<T> *__restrict__ loss, T *__restrict__ gradient) {
  after_previous();
  using W = Wide<T>;
  __shared__ W s_red[kThreads / 32];
  const long g = blockIdx.x;
  const T *x = support + g * Mc;
  const I *u = units + g * K;
  const T *t = teacher + g * K;
  const W inv = (W)1 / temperature, w = weight ? weight[g / H] : (W)1;
  W best = -INFINITY, total = 0, tbest = -INFINITY, ttotal = 0, sum = 0;
  if (w != (W)0) {
    for (long i = threadIdx.x; i < Mc; i += kThreads) best = fmax(best, widen(x[i]));
    best = block_max(best, s_red);
    for (long i = threadIdx.x; i < Mc; i += kThreads) total += sbb_exp((widen(x[i]) - best) * inv);
    total = block_sum(total, s_red);
    for (long k = threadIdx.x; k < K; k += kThreads)
      if ((long)u[k] >= 0 && (long)u[k] < Mc) tbest = fmax(tbest, widen(t[k]));
    tbest = block_max(tbest, s_red);
    for (long k = threadIdx.x; k < K; k += kThreads)
      if ((long)u[k] >= 0 && (long)u[k] < Mc) ttotal += sbb_exp((widen(t[k]) - tbest) * inv);
    ttotal = block_sum(ttotal, s_red);
  }
  if (w == (W)0 || best == -INFINITY || tbest == -INFINITY) {
    if (threadIdx.x == 0) loss[g] = 0;
    if (gradient)
      for (long i = threadIdx.x; i < Mc; i += kThreads) gradient[g * Mc + i] = narrow_to<T>((W)0);
    return;
  }
  const W shift = sbb_log(total) - sbb_log(ttotal);
  for (long k = threadIdx.x; k < K; k += kThreads) {
    if ((long)u[k] < 0 || (long)u[k] >= Mc) continue;
    const W z = (widen(t[k]) - tbest) * inv, p = sbb_exp(z) / ttotal;
    if (p > (W)0 || p != p) sum += p * (z - (widen(x[u[k]]) - best) * inv + shift);
  }
  sum = block_sum(sum, s_red);
  if (threadIdx.x == 0) loss[g] = w * temperature * temperature * sum;
  if (!gradient) return;
  const W wt = w * temperature;
  for (long i = threadIdx.x; i < Mc; i += kThreads)
    gradient[g * Mc + i] = narrow_to<T>(wt * (sbb_exp((widen(x[i]) - best) * inv) / total));
  __syncthreads();   // the kept units' elements are written again
  for (long k = threadIdx.x; k < K; k += kThreads) {
    const long i = (long)u[k];
    if (i < 0 || i >= Mc) continue;
    W p = 0;
    bool first = true;
    for (long j = 0; j < K; ++j)
      if ((long)u[j] == i) {
        first = first && j >= k;
        p += sbb_exp((widen(t[j]) - tbest) * inv) / ttotal;
      }
    if (first) gradient[g * Mc + i] = narrow_to<T>(wt * (sbb_exp((widen(x[i]) - best) * inv) / total - p));
  }
}

}  // namespace

template <typename T, typename I>
cudaError_t launch_distill(const T *support, const I *units, const T *teacher, const Wide<T> *weight, long rows, long H, long Mc, long K,
                           double temperature, Wide<T> *loss, T *gradient, cudaStream_t st) {
  const cudaError_t e = launch_next(distill_kernel<T, I>, dim3((unsigned)(rows * H)), kThreads, 0, st, support, units, teacher, weight, H, Mc, K,
                                    (Wide<T>)temperature, loss, gradient);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

#define SBB_INSTANCE(T, I) \
  template cudaError_t launch_distill<T, I>(const T *, const I *, const T *, const Wide<T> *, long, long, long, long, double, Wide<T> *, T *, cudaStream_t);
#define SBB_INSTANCES(T) SBB_INSTANCE(T, int32_t) SBB_INSTANCE(T, int64_t)
SBB_INSTANCES(float)
SBB_INSTANCES(double)
SBB_INSTANCES(__half)
SBB_INSTANCES(__nv_bfloat16)

}  // namespace sbb
