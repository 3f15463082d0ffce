// Drawing a unit of every group from the softmax of its support, with temperature, top-k, top-p and min-p, from given numbers.
//
// With w_i = exp((x_i - max) / t) and the units in order of falling w (equal ones: lowest index first), top-k, top-p and min-p
// each keep a beginning of that order, so what is kept is all units not behind one (value, index).  Finding that unit takes no
// sort: a histogram of counts and masses over the values' bits says which bin it lies in, and the bin is cut again until few
// units are left, which are compared with one another.
// A random number may lie next to the border of two units, and of a million draws some do within 32 bits' accuracy.  So weights
// are formed in 64 bits and summed as integers, multiples of 2^-q: the sums are the same in any order and their errors below
// n 2^-q of the largest weight.
#include "sbb_codes.cuh"
#include "sbb_launch.cuh"

namespace sbb {
namespace {

typedef unsigned long long u64;

// Bits in the order of the values; -0 counts as +0, a NaN as -infinity (it is never drawn).
template <typename W>
struct Keys;
template <>
struct Keys<float> {
  using type = unsigned;
  static __device__ __forceinline__ unsigned of(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
};
template <>
struct Keys<double> {
  using type = u64;
  static __device__ __forceinline__ u64 of(double v) {
    const u64 b = (u64)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
  }
};
template <typename W>
__device__ __forceinline__ W no_nan(W v) {
  return v == v ? v : (W)-INFINITY;
}

struct Settings {
  double inv_t, top_p, min_p;
  long top_k;   // n: all
};
__device__ __forceinline__ Settings settings_of(const Sampling &s, long row, long n) {
  const double t = s.temperature_rows ? (double)s.temperature_rows[row] : s.temperature;
  Settings r;
  r.top_k = s.top_k_rows ? (long)s.top_k_rows[row] : s.top_k;
  r.top_p = s.top_p_rows ? (double)s.top_p_rows[row] : s.top_p;
  r.min_p = s.min_p_rows ? (double)s.min_p_rows[row] : s.min_p;
  if (r.top_k <= 0 || r.top_k > n) r.top_k = n;
  if (!(t > 0)) r.top_k = 1;
  r.inv_t = t > 0 ? 1 / t : 1;
  return r;
}

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2048, kBinsEach = kBins / kThreads, kFew = 256;

struct Shared {
  u64 mass[kBins];
  unsigned count[kBins];
  u64 few_key[kFew], few_mass[kFew];
  long few_index[kFew];
  u64 sum[kWarps];
  u64 result[4];
  long index[2];
  int bin;
  unsigned few;
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ u64 block_sum(u64 v, u64 *s) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < kWarps; ++i) v += s[i];
  return v;
}
// The sum over the threads in front, in order.
__device__ __forceinline__ u64 block_before(u64 v, u64 *s) {
  u64 in = v;
  const int lane = threadIdx.x & 31;
  for (int off = 1; off < 32; off *= 2) {
    const u64 o = __shfl_up_sync(0xffffffffu, in, off);
    if (lane >= off) in += o;
  }
  __syncthreads();
  if (lane == 31) s[threadIdx.x >> 5] = in;
  __syncthreads();
  u64 base = 0;
  for (int i = 0; i < (int)(threadIdx.x >> 5); ++i) base += s[i];
  return base + in - v;
}

template <typename T>
struct Group {
  using W = Wide<T>;
  using Key = typename Keys<W>::type;
  const T *x;
  long n;
  W best;
  double inv_t, one;   // one: 2^q, the mass of the largest weight

  __device__ __forceinline__ W value(long i) const { return no_nan(widen(x[i])); }
  __device__ __forceinline__ double weight(W v) const {
    return v == best ? 1.0 : v == (W)-INFINITY ? 0.0 : exp(((double)v - (double)best) * inv_t);
  }
  __device__ __forceinline__ u64 mass(double w) const { return __double2ull_rn(w * one); }
  __device__ __forceinline__ u64 mass_of(W v) const { return mass(weight(v)); }
};

// The last unit of a beginning of the order: `count` units where it is a count, else those with less than `limit` in front.
template <typename Key>
struct Cut {
  Key key;
  long index;
  u64 mass;   // of the units up to it
};
template <typename Key>
__device__ __forceinline__ bool kept(Key key, long i, const Cut<Key> &c) {
  return key > c.key || (key == c.key && i <= c.index);
}

// The first unit in index order at which the running sum of weigh(i) passes `target`; the last one with a weight where none does
// (rounding of the target).  -1 where nothing has a weight.
template <typename F>
__device__ long locate(long n, F weigh, u64 target, Shared &s) {
  const long each = (n + kWarps - 1) / kWarps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long lo = min(n, warp * each), hi = min(n, lo + each);
  u64 mine = 0;
  for (long i = lo + lane; i < hi; i += 32) mine += weigh(i);
  mine = warp_sum(mine);
  __syncthreads();
  if (lane == 0) s.sum[warp] = mine;
  if (threadIdx.x == 0) s.index[0] = -1;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += s.sum[i];
    all += s.sum[i];
  }
  if (all > 0 && target >= all) target = all - 1;
  if (mine > 0 && before <= target && target < before + mine) {
    for (long i0 = lo; i0 < hi; i0 += 32) {
      u64 in = i0 + lane < hi ? weigh(i0 + lane) : 0;
      for (int off = 1; off < 32; off *= 2) {
        const u64 o = __shfl_up_sync(0xffffffffu, in, off);
        if (lane >= off) in += o;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + in > target);
      if (past) {
        if (lane == 0) s.index[0] = i0 + __ffs(past) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, in, 31);
    }
  }
  __syncthreads();
  return s.index[0];
}

template <typename T>
__device__ Cut<typename Keys<Wide<T>>::type> select(const Group<T> &g, bool by_count, u64 count, double limit, Shared &s) {
  using W = Wide<T>;
  using Key = typename Keys<W>::type;
  Key lo = Keys<W>::of((W)-INFINITY), hi = Keys<W>::of(g.best);
  u64 above_count = 0, above_mass = 0;   // of the units above hi
  for (;;) {
    int shift = 0;
    while (((hi - lo) >> shift) >= (Key)kBins) ++shift;
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.count[b] = 0, s.mass[b] = 0;
    __syncthreads();
    for (long i = threadIdx.x; i < g.n; i += kThreads) {
      const W v = g.value(i);
      const Key key = Keys<W>::of(v);
      if (key < lo || key > hi) continue;
      const int b = (int)((hi - key) >> shift);   // bin 0 holds the largest
      atomicAdd(&s.count[b], 1u);
      const u64 m = g.mass_of(v);
      if (m) atomicAdd(&s.mass[b], m);
    }
    __syncthreads();
    u64 c = 0, m = 0;
    for (int j = 0; j < kBinsEach; ++j) {
      c += s.count[threadIdx.x * kBinsEach + j];
      m += s.mass[threadIdx.x * kBinsEach + j];
    }
    u64 cb = above_count + block_before(c, s.sum), mb = above_mass + block_before(m, s.sum);
    if (threadIdx.x == 0) s.bin = -1;
    __syncthreads();
    // the last bin that begins inside
    for (int j = 0; j < kBinsEach; ++j) {
      const int b = threadIdx.x * kBinsEach + j;
      if (s.count[b] && (by_count ? cb < count : (double)mb < limit || cb == 0)) atomicMax(&s.bin, b);
      cb += s.count[b];
      mb += s.mass[b];
    }
    __syncthreads();
    const int bin = s.bin;
    if (bin / kBinsEach == (int)threadIdx.x) {
      for (int j = kBinsEach - 1; j >= bin % kBinsEach; --j) {
        cb -= s.count[threadIdx.x * kBinsEach + j];
        mb -= s.mass[threadIdx.x * kBinsEach + j];
      }
      s.result[0] = cb;
      s.result[1] = mb;
      s.few = 0;
    }
    __syncthreads();
    above_count = s.result[0];
    above_mass = s.result[1];
    const unsigned in_bin = s.count[bin];
    const Key width = (Key)1 << shift, top = hi - (Key)bin * width;
    if (top - lo >= width) lo = top - (width - 1);
    hi = top;
    if (in_bin <= kFew) break;
    if (lo == hi) {   // equal values: so many of the lowest indices
      Cut<Key> r;
      r.key = hi;
      u64 take = in_bin;
      W v = g.best;
      const long first = locate(g.n, [&](long i) { return (u64)(Keys<W>::of(g.value(i)) == hi); }, 0, s);
      v = g.value(first);
      const u64 m = g.mass_of(v);
      if (by_count) {
        take = min(take, count - above_count);
      } else if (m > 0) {
        const double q = (limit - (double)above_mass) / (double)m;
        u64 t = q > 1 ? (q < (double)in_bin ? (u64)q : in_bin) : 1;
        while (t > 1 && !((double)(above_mass + (t - 1) * m) < limit)) --t;
        while (t < in_bin && (double)(above_mass + t * m) < limit) ++t;
        take = t;
      }
      r.index = locate(g.n, [&](long i) { return (u64)(Keys<W>::of(g.value(i)) == hi); }, take - 1, s);
      r.mass = above_mass + take * m;
      return r;
    }
    __syncthreads();   // the histogram has been read
  }
  for (long i = threadIdx.x; i < g.n; i += kThreads) {
    const W v = g.value(i);
    const Key key = Keys<W>::of(v);
    if (key < lo || key > hi) continue;
    const unsigned at = atomicAdd(&s.few, 1u);
    s.few_key[at] = key;
    s.few_index[at] = i;
    s.few_mass[at] = g.mass_of(v);
  }
  __syncthreads();
  const int few = (int)s.few;
  bool keep = false;
  u64 cb = above_count, mb = above_mass;
  if ((int)threadIdx.x < few) {
    const u64 key = s.few_key[threadIdx.x];
    const long index = s.few_index[threadIdx.x];
    for (int j = 0; j < few; ++j)
      if (s.few_key[j] > key || (s.few_key[j] == key && s.few_index[j] < index)) {
        cb += 1;
        mb += s.few_mass[j];
      }
    keep = by_count ? cb < count : (double)mb < limit || cb == 0;
  }
  const u64 n_kept = block_sum(keep, s.sum);
  if (keep && cb + 1 == above_count + n_kept) {
    s.result[2] = s.few_key[threadIdx.x];
    s.result[3] = mb + s.few_mass[threadIdx.x];
    s.index[1] = s.few_index[threadIdx.x];
  }
  __syncthreads();
  return Cut<Key>{(Key)s.result[2], s.index[1], s.result[3]};
}

// A block per group.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    sample_kernel(const T *__restrict__ support, const float *__restrict__ random, long H, long Mc, Sampling how, double one, long long *__restrict__ codes) {
  after_previous();
  using W = Wide<T>;
  using Key = typename Keys<W>::type;
  __shared__ Shared s;
  const long g = blockIdx.x;
  const Settings set = settings_of(how, g / H, Mc);
  Group<T> group{support + g * Mc, Mc, (W)-INFINITY, set.inv_t, one};
  Key top = 0;
  for (long i = threadIdx.x; i < Mc; i += kThreads) {
    const W v = group.value(i);
    const Key k = Keys<W>::of(v);
    if (k > top) top = k, group.best = v;
  }
  for (int off = 16; off > 0; off >>= 1) group.best = fmax(group.best, __shfl_xor_sync(0xffffffffu, group.best, off));
  if ((threadIdx.x & 31) == 0) reinterpret_cast<W *>(s.sum)[threadIdx.x >> 5] = group.best;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) group.best = fmax(group.best, reinterpret_cast<W *>(s.sum)[i]);
  __syncthreads();
  if (group.best == (W)-INFINITY) {
    if (threadIdx.x == 0) codes[g] = -1;
    return;
  }
  Cut<Key> cut{0, Mc, 0};
  if (set.top_k < Mc) cut = select(group, true, (u64)set.top_k, 0.0, s);
  if (set.top_p < 1) {
    u64 total = cut.mass;
    if (set.top_k >= Mc) {
      total = 0;
      for (long i = threadIdx.x; i < Mc; i += kThreads) total += group.mass_of(group.value(i));
      total = block_sum(total, s.sum);
    }
    cut = select(group, false, 0, set.top_p * (double)total, s);
  }
  auto weigh = [&](long i) -> u64 {
    const W v = group.value(i);
    if (!kept(Keys<W>::of(v), i, cut)) return 0;
    const double w = group.weight(v);
    return w >= set.min_p || v == group.best ? group.mass(w) : 0;
  };
  u64 total = 0;
  for (long i = threadIdx.x; i < Mc; i += kThreads) total += weigh(i);
  total = block_sum(total, s.sum);
  const double at = (double)random[g] * (double)total;
  const long unit = locate(Mc, weigh, at > 0 ? (u64)at : 0, s);
  if (threadIdx.x == 0) codes[g] = unit < 0 ? -1 : g % H * Mc + unit;
}

}  // namespace

template <typename T>
cudaError_t launch_sample(const T *support, const float *random, long rows, long H, long Mc, Sampling s, long long *codes, cudaStream_t st) {
  int q = 50;
  while (q > 20 && ((double)Mc * (double)(1ull << q)) >= 4.6e18) --q;   // no sum passes 2^62
  const cudaError_t e = launch_next(sample_kernel<T>, dim3((unsigned)(rows * H)), kThreads, 0, st, support, random, H, Mc, s, (double)(1ull << q), codes);
  if (e == cudaSuccess) count_launches(1);
  return e;
}
template cudaError_t launch_sample<float>(const float *, const float *, long, long, long, Sampling, long long *, cudaStream_t);
template cudaError_t launch_sample<double>(const double *, const float *, long, long, long, Sampling, long long *, cudaStream_t);
template cudaError_t launch_sample<__half>(const __half *, const float *, long, long, long, Sampling, long long *, cudaStream_t);
template cudaError_t launch_sample<__nv_bfloat16>(const __nv_bfloat16 *, const float *, long, long, long, Sampling, long long *, cudaStream_t);

}  // namespace sbb
