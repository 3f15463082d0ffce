// Launch interface of the operators on unit codes (device pointers, asynchronous on the given stream) and the types they
// share.  Every launcher returns cudaSuccess or the launch error and bumps the process-wide launch counter.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace sbb {

void count_launches(int n);   // sbb_kernels.cu
int sm_count();

// What sums are held in: 32 bits for everything narrower, 64 for double.
template <typename T>
struct WideOf {
  using type = float;
};
template <>
struct WideOf<double> {
  using type = double;
};
template <typename T>
using Wide = typename WideOf<T>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// The one rounding of a result, to nearest.
template <typename T>
__device__ __forceinline__ T narrow_to(Wide<T> v) {
  return v;
}
template <>
__device__ __forceinline__ __half narrow_to<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow_to<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// V neighbours, loaded and stored in one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// All of a vector's elements: 16-bit ones two at a time.
template <typename T, int V>
__device__ __forceinline__ void widen_all(const Vec<T, V> &a, Wide<T> (&f)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const unsigned two = reinterpret_cast<const unsigned *>(a.v)[i];
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[2 * i] = __uint_as_float(two << 16);
        f[2 * i + 1] = __uint_as_float(two & 0xffff0000u);
      } else {
        const float2 both = __half22float2(*reinterpret_cast<const __half2 *>(&two));
        f[2 * i] = both.x;
        f[2 * i + 1] = both.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = widen(a.v[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow_all(const Wide<T> (&f)[V]) {
  Vec<T, V> a;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        reinterpret_cast<unsigned *>(a.v)[i] = *reinterpret_cast<const unsigned *>(&two);
      } else {
        const __half2 two = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        reinterpret_cast<unsigned *>(a.v)[i] = *reinterpret_cast<const unsigned *>(&two);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) a.v[i] = narrow_to<T>(f[i]);
  }
  return a;
}
// The largest element; a NaN is passed over.
template <typename T, int V>
__device__ __forceinline__ Wide<T> max_all(const Vec<T, V> &a) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 m = *reinterpret_cast<const T2 *>(a.v);
#pragma unroll
    for (int i = 1; i < V / 2; ++i) m = __hmax2(m, *reinterpret_cast<const T2 *>(a.v + 2 * i));
    return fmaxf(widen(m.x), widen(m.y));
  } else {
    Wide<T> m = widen(a.v[0]);
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmax(m, widen(a.v[i]));
    return m;
  }
}

// How many elements one access may hold: 16 bytes where all rows start on such a boundary, two 16-bit elements where they start
// on one of four bytes (a warp's request is then a whole line), else one.
template <typename T>
inline int vector_width(long row_elems, const void *a, const void *b) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | (uintptr_t)(row_elems * (long)sizeof(T));
  if ((bits & 15u) == 0) return 16 / (int)sizeof(T);
  if (sizeof(T) == 2 && (bits & 3u) == 0) return 2;
  return 1;
}

// out[r, :] = scale * sum_l weights[codes[r, l], :]   (weights is [N, M]; codes outside [0, N) name nothing)
template <typename T, typename I>
cudaError_t launch_lookup(const T *weights, const I *codes, long rows, long L, long N, long M, double scale, T *out, cudaStream_t st);

// out[i, :] = scale * sum over (r, l) with codes[r, l] == i of grad[r, :], added to what is there with `accumulate`.
// `workspace`: lookup_gradient_workspace() bytes, 16-byte aligned, free again when the call's work has ended.
size_t lookup_gradient_workspace(long rows, long L, long N, long M, size_t wide);
template <typename T, typename I>
cudaError_t launch_lookup_gradient(const T *grad, const I *codes, long rows, long L, long N, long M, double scale, bool accumulate, T *out,
                                   void *workspace, cudaStream_t st);

// One unit per (row, group of Mc) drawn from the softmax of support[rows, H * Mc]; codes[rows, H] = h * Mc + unit, or -1.
struct Sampling {
  double temperature, top_p, min_p;
  double inv_t;   // of `temperature`, filled in by launch_sample
  long top_k;
  const float *temperature_rows, *top_p_rows, *min_p_rows;   // not null: a value per row in place of the scalar
  const int *top_k_rows;
};
template <typename T>
cudaError_t launch_sample(const T *support, const float *random, long rows, long H, long Mc, Sampling s, long long *codes, cudaStream_t st);

// loss[rows, H] and (gradient != null) gradient[rows, H * Mc] of the divergence from a teacher's K kept units per group.
template <typename T, typename I>
cudaError_t launch_distill(const T *support, const I *units, const T *teacher, const Wide<T> *weight, long rows, long H, long Mc, long K,
                           double temperature, Wide<T> *loss, T *gradient, cudaStream_t st);

}  // namespace sbb
