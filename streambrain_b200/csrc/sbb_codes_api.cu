// C entries of the operators on unit codes: checks of arguments, choice of types.  See include/sbb200.h.
#include "../../include/sbb200.h"
#include "sbb_codes.cuh"

#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace sbb {
void set_last_error(const char *message);   // sbb_api.cu
}

namespace {

int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  sbb::set_last_error(buf);
  return code;
}

#define ARG(cond, ...) \
  do {                 \
    if (!(cond)) return fail(SBB_ERR_INVALID, __VA_ARGS__); \
  } while (0)
// Counts that kernels hold in 32 bits; elements are addressed in 64.
#define FITS(n, ...) \
  do {               \
    if ((n) > 0x7fffffffll) return fail(SBB_ERR_UNSUPPORTED, __VA_ARGS__); \
  } while (0)

int need_device() {
  static std::atomic<bool> found{false};   // (a device that is there stays)
  if (found) return SBB_OK;
  int n = 0;
  if (cudaGetDeviceCount(&n) != cudaSuccess) {
    (void)cudaGetLastError();
    n = 0;
  }
  if (n <= 0) return fail(SBB_ERR_NO_DEVICE, "no CUDA device is available; this library has no CPU path");
  found = true;
  return SBB_OK;
}

int done(cudaError_t e, const char *what) {
  if (e == cudaSuccess) return SBB_OK;
  (void)cudaGetLastError();   // reported here: the launch that asks next may not find it and fail for it
  return fail(SBB_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

size_t element(int dtype) { return dtype == SBB_F64 ? 8 : dtype == SBB_F32 ? 4 : dtype == SBB_F16 || dtype == SBB_BF16 ? 2 : 0; }

bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// a * b, at most 2^62; for factors that are not negative
long long product(long long a, long long b) { return a > 0 && b > (1ll << 62) / a ? 1ll << 62 : a * b; }

// Calls f(element, index) with values of the two types.
template <typename I, typename F>
cudaError_t with_element(int dtype, F f) {
  switch (dtype) {
    case SBB_F32: return f(float(), I());
    case SBB_F64: return f(double(), I());
    case SBB_F16: return f(__half(), I());
    default: return f(__nv_bfloat16(), I());
  }
}
template <typename F>
cudaError_t with_types(int dtype, int index_bytes, F f) {
  return index_bytes == 4 ? with_element<int32_t>(dtype, f) : with_element<int64_t>(dtype, f);
}

int check_lookup(const char *what, int dtype, const void *a, const void *codes, int code_bytes, long rows, long L, long N, long M, const void *out) {
  const size_t e = element(dtype);
  ARG(e != 0, "%s: invalid dtype %d", what, dtype);
  ARG(code_bytes == 4 || code_bytes == 8, "%s: codes are of 4 or 8 bytes, not %d", what, code_bytes);
  ARG(rows >= 0 && L >= 0 && N > 0 && M > 0, "%s: bad shape rows=%ld codes=%ld N=%ld M=%ld", what, rows, L, N, M);
  FITS(product(rows, L), "%s: %ld x %ld codes are more than 2^31 - 1", what, rows, L);
  FITS(rows, "%s: more than 2^31 - 1 rows", what);
  FITS(N, "%s: more than 2^31 - 1 weight rows", what);
  FITS(product(M, 32), "%s: rows of more than 2^26 - 1 units", what);
  ARG(aligned(a, e) && aligned(out, e) && aligned(codes, (size_t)code_bytes), "%s: misaligned pointer", what);
  return SBB_OK;
}

}  // namespace

extern "C" {

int sbb_lookup(int dtype, const void *weights_dev, const void *codes_dev, int code_bytes, long rows, long codes_per_row, long N, long M,
               double scale, void *out_dev, void *stream) {
  if (const int rc = check_lookup("lookup", dtype, weights_dev, codes_dev, code_bytes, rows, codes_per_row, N, M, out_dev)) return rc;
  ARG(weights_dev && ((out_dev && (codes_dev || codes_per_row == 0)) || rows == 0), "lookup: null pointer");
  if (const int rc = need_device()) return rc;
  if (rows == 0) return SBB_OK;
  return done(with_types(dtype, code_bytes,
                         [&](auto t, auto i) {
                           return sbb::launch_lookup((const decltype(t) *)weights_dev, (const decltype(i) *)codes_dev, rows, codes_per_row, N, M,
                                                     scale, (decltype(t) *)out_dev, (cudaStream_t)stream);
                         }),
              "lookup");
}

size_t sbb_lookup_gradient_workspace(int dtype, long rows, long codes_per_row, long N, long M) {
  if (element(dtype) == 0 || rows <= 0 || codes_per_row <= 0 || N <= 0 || M <= 0 || product(rows, codes_per_row) > 0x7fffffffll) return 0;
  return sbb::lookup_gradient_workspace(rows, codes_per_row, N, M, dtype == SBB_F64 ? 8 : 4);
}

int sbb_lookup_gradient(int dtype, const void *grad_dev, const void *codes_dev, int code_bytes, long rows, long codes_per_row, long N, long M,
                        double scale, int accumulate, void *out_dev, void *workspace_dev, size_t workspace_bytes, void *stream) {
  if (const int rc = check_lookup("lookup_gradient", dtype, grad_dev, codes_dev, code_bytes, rows, codes_per_row, N, M, out_dev)) return rc;
  const bool any = rows > 0 && codes_per_row > 0;
  ARG(out_dev && ((grad_dev && codes_dev) || !any), "lookup_gradient: null pointer");
  const size_t need = sbb_lookup_gradient_workspace(dtype, rows, codes_per_row, N, M);
  ARG(need == 0 || (workspace_dev && aligned(workspace_dev, 16) && workspace_bytes >= need),
      "lookup_gradient: needs a workspace of %zu bytes on a boundary of 16, got %zu", need, workspace_bytes);
  if (const int rc = need_device()) return rc;
  if (!any) {
    if (accumulate) return SBB_OK;
    return done(cudaMemsetAsync(out_dev, 0, (size_t)N * (size_t)M * element(dtype), (cudaStream_t)stream), "lookup_gradient");
  }
  return done(with_types(dtype, code_bytes,
                         [&](auto t, auto i) {
                           return sbb::launch_lookup_gradient((const decltype(t) *)grad_dev, (const decltype(i) *)codes_dev, rows, codes_per_row, N,
                                                              M, scale, accumulate != 0, (decltype(t) *)out_dev, workspace_dev, (cudaStream_t)stream);
                         }),
              "lookup_gradient");
}

int sbb_sample_minicolumns(int dtype, const void *support_dev, const float *random_dev, long rows, long H, long Mc, const sbb_sampling *how,
                           long long *codes_dev, void *stream) {
  const size_t e = element(dtype);
  ARG(e != 0, "sample_minicolumns: invalid dtype %d", dtype);
  ARG(rows >= 0 && H > 0 && Mc > 0, "sample_minicolumns: bad shape rows=%ld H=%ld Mc=%ld", rows, H, Mc);
  ARG(how != nullptr, "sample_minicolumns: null pointer");
  ARG(std::isfinite(how->temperature) && how->temperature >= 0 && how->top_p >= 0 && how->min_p >= 0 && how->min_p <= 1,
      "sample_minicolumns: temperature %g, top_p %g, min_p %g: a finite temperature and top_p of 0 or more, min_p from 0 to 1 are wanted",
      how->temperature, how->top_p, how->min_p);
  FITS(product(rows, H), "sample_minicolumns: %ld x %ld hypercolumns are more than 2^31 - 1", rows, H);
  FITS(Mc, "sample_minicolumns: more than 2^31 - 1 units in a hypercolumn");
  ARG((support_dev && random_dev && codes_dev) || rows == 0, "sample_minicolumns: null pointer");
  ARG(aligned(support_dev, e) && aligned(random_dev, 4) && aligned(codes_dev, 8) && aligned(how->temperature_rows, 4) &&
          aligned(how->top_p_rows, 4) && aligned(how->min_p_rows, 4) && aligned(how->top_k_rows, 4),
      "sample_minicolumns: misaligned pointer");
  if (const int rc = need_device()) return rc;
  if (rows == 0) return SBB_OK;
  // (rounded to float, so that a number gives what a value for every row gives)
  const sbb::Sampling s = {(float)how->temperature, (float)how->top_p, (float)how->min_p, 0, how->top_k,
                           how->temperature_rows, how->top_p_rows, how->min_p_rows, how->top_k_rows};
  return done(with_element<int>(dtype,
                                [&](auto t, int) {
                                  return sbb::launch_sample((const decltype(t) *)support_dev, random_dev, rows, H, Mc, s, codes_dev,
                                                            (cudaStream_t)stream);
                                }),
              "sample_minicolumns");
}

int sbb_distill(int dtype, const void *support_dev, const void *teacher_units_dev, int unit_bytes, const void *teacher_dev,
                const void *weight_dev, long rows, long H, long Mc, long K, double temperature, void *loss_dev, void *gradient_dev, void *stream) {
  const size_t e = element(dtype), wide = dtype == SBB_F64 ? 8 : 4;
  ARG(e != 0, "distill: invalid dtype %d", dtype);
  ARG(unit_bytes == 4 || unit_bytes == 8, "distill: units are of 4 or 8 bytes, not %d", unit_bytes);
  ARG(rows >= 0 && H > 0 && Mc > 0 && K >= 0, "distill: bad shape rows=%ld H=%ld Mc=%ld K=%ld", rows, H, Mc, K);
  ARG(temperature >= 1e-15 && temperature <= 1e15, "distill: temperature %g is not from 1e-15 to 1e15", temperature);
  FITS(product(rows, H), "distill: %ld x %ld hypercolumns are more than 2^31 - 1", rows, H);
  FITS(Mc, "distill: more than 2^31 - 1 units in a hypercolumn");
  FITS(K, "distill: more than 2^31 - 1 kept units");
  ARG((support_dev && loss_dev && ((teacher_units_dev && teacher_dev) || K == 0)) || rows == 0, "distill: null pointer");
  ARG(aligned(support_dev, e) && aligned(teacher_dev, e) && aligned(gradient_dev, e) && aligned(teacher_units_dev, (size_t)unit_bytes) &&
          aligned(weight_dev, wide) && aligned(loss_dev, wide),
      "distill: misaligned pointer");
  if (const int rc = need_device()) return rc;
  if (rows == 0) return SBB_OK;
  return done(with_types(dtype, unit_bytes,
                         [&](auto t, auto i) {
                           using T = decltype(t);
                           return sbb::launch_distill((const T *)support_dev, (const decltype(i) *)teacher_units_dev, (const T *)teacher_dev,
                                                      (const sbb::Wide<T> *)weight_dev, rows, H, Mc, K, temperature, (sbb::Wide<T> *)loss_dev,
                                                      (T *)gradient_dev, (cudaStream_t)stream);
                         }),
              "distill");
}

}  // extern "C"
