// Distillation from a teacher of which only the best units of each group are kept.
//
// With p the softmax of the teacher's kept units, q the softmax of all of the student's group, both at temperature t, and w the
// row's weight: loss = w t^2 sum_k p_k (log p_k - log q_{u_k}), and d loss / d x_i = w t (q_i - sum over k with u_k = i of p_k).
// What bounds it is memory: the student's support is read once and its gradient written once.  Groups of up to 512 units are a
// warp's, in its registers; wider ones a cluster's of blocks, which keep their parts in shared memory for the gradient while they
// form the running maximum and sum.
#include "sbb_codes.cuh"
#include "sbb_launch.cuh"
#include "sbb_math.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace sbb {
namespace {

template <typename T>
struct Distill {
  using W = Wide<T>;
  const T *support;
  const void *units;   // of 8 bytes where wide_units, else of 4
  bool wide_units;
  const T *teacher;
  const W *weight;
  unsigned groups, H, n, K;
  W temperature, c;    // expo(d, c) = exp(d / temperature)
  W *loss;
  T *gradient;

  // The unit of an entry of group g; n or more: absent
  __device__ __forceinline__ unsigned unit(long g, unsigned k) const {
    const long at = g * K + k;
    if (wide_units) {
      const long long u = static_cast<const long long *>(units)[at];
      return u >= 0 && u < (long long)n ? (unsigned)u : n;
    }
    return (unsigned)static_cast<const int *>(units)[at];   // (a negative one is above 2^31)
  }
};

// exp(d / t): for float 2^(d log2(e) / t) by ex2.approx, off by 2^-22 of it and by 3 x 2^-24 for every unit of its exponent
__device__ __forceinline__ float expo(float d, float c) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * c));
  return r;
}
__device__ __forceinline__ double expo(double d, double c) { return exp(d * c); }

template <typename W>
__device__ __forceinline__ W warp_sum(W v) {
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ double warp_max(double v) {
  for (int off = 16; off > 0; off >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

// ---- a warp per group ------------------------------------------------------

constexpr int kWarpThreads = 256, kWarps = kWarpThreads / 32;

// Lane l holds vectors l, l + 32, ... of V units each, NV of them.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(kWarpThreads) distill_warp_kernel(const Distill<T> p) {
  after_previous();
  using W = Wide<T>;
  __shared__ Vec<W, V> s_kept[kWarps][NV * 32];   // what the teacher gives each unit
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, step = gridDim.x * kWarps, rows = step / p.H, rest = step % p.H;
  W *const kept = s_kept[warp][0].v;
  unsigned g = blockIdx.x * kWarps + warp, row = g / p.H, h = g % p.H;
  for (; g < p.groups; g += step, row += rows, h += rest) {
    if (h >= p.H) h -= p.H, row += 1;
    const T *const x = p.support + (long)g * p.n;
    T *const out = p.gradient + (long)g * p.n;
    const W w = p.weight ? p.weight[row] : (W)1;
    Vec<T, V> raw[NV];
    W e[NV][V], best = -INFINITY, total = 0, tbest = -INFINITY, ttotal = 0, sum = 0;
    unsigned u0 = p.n;
    W t0 = -INFINITY, x0 = 0;
    if (w != (W)0) {
#pragma unroll
      for (int r = 0; r < NV; ++r)
        if ((r * 32 + lane) * V < p.n) raw[r] = *reinterpret_cast<const Vec<T, V> *>(x + (r * 32 + lane) * V);
      if (lane < p.K) {
        u0 = p.unit(g, lane);
        if (u0 < p.n) {
          t0 = widen(p.teacher[(long)g * p.K + lane]);
          x0 = widen(x[u0]);
        }
      }
#pragma unroll
      for (int r = 0; r < NV; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          e[r][v] = (r * 32 + lane) * V < p.n ? widen(raw[r].v[v]) : (W)-INFINITY;
          best = fmax(best, e[r][v]);
        }
      best = warp_max(best);
      if (u0 < p.n) tbest = t0;
      for (unsigned k = lane + 32; k < p.K; k += 32)
        if (p.unit(g, k) < p.n) tbest = fmax(tbest, widen(p.teacher[(long)g * p.K + k]));
      tbest = warp_max(tbest);
    }
    bool nothing = w == (W)0 || best == -INFINITY || tbest == -INFINITY;
    if (nothing && w != (W)0) {   // (the maxima pass over NaN, which is not nothing)
      bool nan = u0 < p.n && t0 != t0;
#pragma unroll
      for (int r = 0; r < NV; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) nan = nan || e[r][v] != e[r][v];
      for (unsigned k = lane + 32; k < p.K; k += 32) nan = nan || (p.unit(g, k) < p.n && isnan(widen(p.teacher[(long)g * p.K + k])));
      nothing = !__any_sync(0xffffffffu, nan);
    }
    if (nothing) {
      if (lane == 0) p.loss[g] = 0;
      if (p.gradient) {
        Vec<T, V> zero;
#pragma unroll
        for (int v = 0; v < V; ++v) zero.v[v] = narrow_to<T>((W)0);
#pragma unroll
        for (int r = 0; r < NV; ++r)
          if ((r * 32 + lane) * V < p.n) *reinterpret_cast<Vec<T, V> *>(out + (r * 32 + lane) * V) = zero;
      }
      continue;
    }
    if (p.gradient) {
      Vec<W, V> zero;
#pragma unroll
      for (int v = 0; v < V; ++v) zero.v[v] = 0;
#pragma unroll
      for (int r = 0; r < NV; ++r) s_kept[warp][r * 32 + lane] = zero;
      __syncwarp();
    }
#pragma unroll
    for (int r = 0; r < NV; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        e[r][v] = expo(e[r][v] - best, p.c);
        total += e[r][v];
      }
    total = warp_sum(total);
    const W p0 = u0 < p.n ? expo(t0 - tbest, p.c) : (W)0;
    ttotal = p0;
    for (unsigned k = lane + 32; k < p.K; k += 32)
      if (p.unit(g, k) < p.n) ttotal += expo(widen(p.teacher[(long)g * p.K + k]) - tbest, p.c);
    ttotal = warp_sum(ttotal);
    const W inv = (W)1 / p.temperature, shift = sbb_log(total) - sbb_log(ttotal), share = (W)1 / ttotal;
    for (unsigned k0 = 0; k0 < p.K; k0 += 32) {
      const unsigned k = k0 + lane;
      unsigned u = u0;
      W t = t0, xu = x0, pk = p0;
      if (k0 > 0) {
        u = k < p.K ? p.unit(g, k) : p.n;
        pk = 0;
        if (u < p.n) {
          t = widen(p.teacher[(long)g * p.K + k]);
          xu = widen(x[u]);
          pk = expo(t - tbest, p.c);
        }
      }
      const bool there = u < p.n;
      pk *= share;
      if (there && !(pk == (W)0)) sum += pk * (((t - tbest) - (xu - best)) * inv + shift);
      if (p.gradient) {
        // a unit named twice has both parts, added in the order of the entries
        const unsigned same = __match_any_sync(0xffffffffu, there ? u : ~lane);
        W part = pk;
        if (__any_sync(0xffffffffu, (same & (same - 1)) != 0)) {
          part = 0;
          for (int j = 0; j < 32; ++j) {
            const W o = __shfl_sync(0xffffffffu, pk, j);
            if (same >> j & 1) part += o;
          }
        }
        if (there && __ffs(same) - 1 == (int)lane) kept[u] += part;
        __syncwarp();
      }
    }
    sum = warp_sum(sum);
    if (lane == 0) p.loss[g] = w * p.temperature * p.temperature * sum;
    if (!p.gradient) continue;
    const W wt = w * p.temperature, scale = wt / total;
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if ((r * 32 + lane) * V < p.n) {
        const Vec<W, V> k = s_kept[warp][r * 32 + lane];
        Vec<T, V> o;
#pragma unroll
        for (int v = 0; v < V; ++v) o.v[v] = narrow_to<T>(e[r][v] * scale - wt * k.v[v]);
        *reinterpret_cast<Vec<T, V> *>(out + (r * 32 + lane) * V) = o;
      }
    __syncwarp();
  }
}

// ---- a cluster per group ---------------------------------------------------

constexpr int kThreads = 512, kBlockWarps = kThreads / 32, kMostBlocks = 8;
constexpr int kStage = 100 * 1024;   // bytes of a group that a block keeps in shared memory
constexpr int kEntries = 512;        // kept units that wait in shared memory; those of longer lists are read again

// A running maximum and the sum of exp((x - maximum) / t).
template <typename W>
struct Running {
  W best, sum;
  __device__ __forceinline__ void add(const Running &o, W c) {
    const W b = fmax(best, o.best);
    if (b == -INFINITY) {
      sum += o.sum;   // (0, or a NaN)
      return;
    }
    sum = (best == b ? sum : sum * expo(best - b, c)) + (o.best == b ? o.sum : o.sum * expo(o.best - b, c));
    best = b;
  }
};
template <typename W>
__device__ __forceinline__ Running<W> warp_add(Running<W> r, W c) {
  for (int off = 16; off > 0; off >>= 1) r.add(Running<W>{__shfl_xor_sync(0xffffffffu, r.best, off), __shfl_xor_sync(0xffffffffu, r.sum, off)}, c);
  return r;
}

template <typename W>
struct Block {
  Running<W> part[kBlockWarps], own;
  W sum[kBlockWarps];
  W kept[kEntries];
  unsigned unit[kEntries];
};

template <typename W>
__device__ __forceinline__ W block_sum(W v, W *s) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int i = 1; i < kBlockWarps; ++i) v += s[i];
  return v;
}
// The same for a running maximum and sum; every warp's and every lane's order is the same, so all threads have the same bits.
template <typename W>
__device__ __forceinline__ Running<W> block_add(Running<W> r, W c, Running<W> *s) {
  r = warp_add(r, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = r;
  __syncthreads();
  r = s[0];
#pragma unroll
  for (int i = 1; i < kBlockWarps; ++i) r.add(s[i], c);
  return r;
}

// STAGED: the part waits in shared memory between the sum and the gradient; else (no gradient, or groups beyond what a cluster
// holds) it is read again.  V: units of an access.
template <typename T, int V, bool STAGED>
__global__ void __launch_bounds__(kThreads) distill_block_kernel(const Distill<T> p, unsigned part) {
  after_previous();
  using W = Wide<T>;
  extern __shared__ uint4 s_values[];
  __shared__ Block<W> s;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned blocks = cluster.num_blocks(), g = blockIdx.x / blocks, rank = cluster.block_rank();
  const unsigned begin = min(p.n, rank * part), size = min(part, p.n - begin), vectors = size / V;   // (V divides both)
  const T *const x = p.support + (long)g * p.n + begin;
  T *const out = p.gradient + (long)g * p.n + begin;
  Vec<T, V> *const stage = reinterpret_cast<Vec<T, V> *>(s_values);
  const W w = p.weight ? p.weight[g / p.H] : (W)1;
  Running<W> r{-INFINITY, 0}, t{-INFINITY, 0};
  if (w != (W)0) {
    constexpr int U = 4;
    for (unsigned i = threadIdx.x; i < vectors; i += U * kThreads) {
      Vec<T, V> a[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < vectors) a[u] = reinterpret_cast<const Vec<T, V> *>(x)[i + u * kThreads];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < vectors) {
          if constexpr (STAGED) stage[i + u * kThreads] = a[u];
          W m = widen(a[u].v[0]);
#pragma unroll
          for (int v = 1; v < V; ++v) m = fmax(m, widen(a[u].v[v]));
          if (m > r.best) {
            r.sum *= expo(r.best - m, p.c);   // (of -infinity: the sum is 0, or a NaN)
            r.best = m;
          }
          const W from = r.best == -INFINITY ? (W)0 : r.best;
#pragma unroll
          for (int v = 0; v < V; ++v) r.sum += expo(widen(a[u].v[v]) - from, p.c);
        }
    }
    r = block_add(r, p.c, s.part);
    for (unsigned k = threadIdx.x; k < p.K; k += kThreads)
      if (p.unit(g, k) < p.n) {
        const W v = widen(p.teacher[(long)g * p.K + k]);
        t.add(Running<W>{v, v == -INFINITY ? (W)0 : v == v ? (W)1 : v}, p.c);
      }
    t = block_add(t, p.c, s.part);
    if (blocks > 1) {
      if (threadIdx.x == 0) s.own = r;
      cluster.sync();
      r = cluster.map_shared_rank(&s, 0)->own;
      for (unsigned b = 1; b < blocks; ++b) r.add(cluster.map_shared_rank(&s, b)->own, p.c);
      cluster.sync();   // (a block may go on to its end, which the others read from)
    }
  }
  if (w == (W)0 || (r.best == -INFINITY && r.sum == (W)0) || (t.best == -INFINITY && t.sum == (W)0)) {
    if (rank == 0 && threadIdx.x == 0) p.loss[g] = 0;
    if (p.gradient) {
      Vec<T, V> zero;
#pragma unroll
      for (int v = 0; v < V; ++v) zero.v[v] = narrow_to<T>((W)0);
      for (unsigned i = threadIdx.x; i < vectors; i += kThreads) reinterpret_cast<Vec<T, V> *>(out)[i] = zero;
    }
    return;
  }
  const W inv = (W)1 / p.temperature, shift = sbb_log(r.sum) - sbb_log(t.sum), wt = w * p.temperature, scale = wt / r.sum, share = (W)1 / t.sum;
  auto kept = [&](unsigned k) { return expo(widen(p.teacher[(long)g * p.K + k]) - t.best, p.c) * share; };
  if (rank == 0) {
    W sum = 0;
    for (unsigned k = threadIdx.x; k < p.K; k += kThreads) {
      const unsigned u = p.unit(g, k);
      if (u >= p.n) continue;
      const W z = widen(p.teacher[(long)g * p.K + k]) - t.best, pk = expo(z, p.c) * share;
      if (!(pk == (W)0)) sum += pk * ((z - (widen(p.support[(long)g * p.n + u]) - r.best)) * inv + shift);
    }
    sum = block_sum(sum, s.sum);
    if (threadIdx.x == 0) p.loss[g] = w * p.temperature * p.temperature * sum;
  }
  if (!p.gradient) return;
  const bool listed = p.K <= kEntries;
  if (listed)
    for (unsigned k = threadIdx.x; k < p.K; k += kThreads) {
      const unsigned u = p.unit(g, k);
      s.unit[k] = u;
      s.kept[k] = u < p.n ? kept(k) : (W)0;
    }
  for (unsigned i = threadIdx.x; i < vectors; i += kThreads) {
    const Vec<T, V> a = STAGED ? stage[i] : reinterpret_cast<const Vec<T, V> *>(x)[i];
    Vec<T, V> o;
#pragma unroll
    for (int v = 0; v < V; ++v) o.v[v] = narrow_to<T>(expo(widen(a.v[v]) - r.best, p.c) * scale);
    reinterpret_cast<Vec<T, V> *>(out)[i] = o;
  }
  __syncthreads();   // the kept units' elements are written again, each by the first entry that names it
  for (unsigned k = threadIdx.x; k < p.K; k += kThreads) {
    const unsigned u = listed ? s.unit[k] : p.unit(g, k);
    if (u < begin || u >= begin + size) continue;
    W sum = 0;
    bool first = true;
    for (unsigned j = 0; j < p.K; ++j)
      if ((listed ? s.unit[j] : p.unit(g, j)) == u) {
        first = first && j >= k;
        sum += listed ? s.kept[j] : kept(j);
      }
    if (first) out[u - begin] = narrow_to<T>(expo(widen(p.support[(long)g * p.n + u]) - r.best, p.c) * scale - wt * sum);
  }
}

template <typename T, int V, int NV>
cudaError_t launch_warps(const Distill<T> &p, cudaStream_t st) {
  const unsigned most = 16 * (unsigned)sm_count(), blocks = (p.groups + kWarps - 1) / kWarps;
  return launch_next(distill_warp_kernel<T, V, NV>, dim3(blocks < most ? blocks : most), kWarpThreads, 0, st, p);
}

template <typename T, int V, bool STAGED>
cudaError_t launch_blocks(const Distill<T> &p, unsigned part, unsigned cluster, cudaStream_t st) {
  const size_t smem = STAGED ? (size_t)part * sizeof(T) : 0;
  if (smem > 0) {   // (holds for the current device)
    const cudaError_t e = cudaFuncSetAttribute(distill_block_kernel<T, V, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStage);
    if (e != cudaSuccess) return e;
  }
  return launch_clusters(distill_block_kernel<T, V, STAGED>, dim3(p.groups * cluster), dim3(cluster), kThreads, smem, st, p, part);
}

template <typename T>
cudaError_t launch_wide(const Distill<T> &p, int vec, cudaStream_t st) {
  const size_t bytes = (size_t)p.n * sizeof(T);
  unsigned cluster = 1;
  // the smallest cluster whose blocks hold their parts; a larger one where groups are too few for the SMs and parts long
  if (p.gradient)
    while (cluster < kMostBlocks && bytes > (size_t)cluster * kStage) cluster *= 2;
  while (cluster < kMostBlocks && (size_t)p.groups * cluster * 2 <= (size_t)sm_count() && p.n / cluster > 4096) cluster *= 2;
  const unsigned part = ((p.n + cluster - 1) / cluster + 15) / 16 * 16;
  if ((size_t)p.groups * cluster > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const bool staged = p.gradient && (size_t)part * sizeof(T) <= kStage;
  constexpr int V = 16 / (int)sizeof(T);
  if (vec == V) return staged ? launch_blocks<T, V, true>(p, part, cluster, st) : launch_blocks<T, V, false>(p, part, cluster, st);
  return staged ? launch_blocks<T, 1, true>(p, part, cluster, st) : launch_blocks<T, 1, false>(p, part, cluster, st);
}

}  // namespace

template <typename T, typename I>
cudaError_t launch_distill(const T *support, const I *units, const T *teacher, const Wide<T> *weight, long rows, long H, long Mc, long K,
                           double temperature, Wide<T> *loss, T *gradient, cudaStream_t st) {
  using W = Wide<T>;
  const Distill<T> p = {support, units, sizeof(I) == 8, teacher, weight, (unsigned)(rows * H), (unsigned)H, (unsigned)Mc, (unsigned)K,
                        (W)temperature, sizeof(W) == 4 ? (W)(1.4426950408889634 / temperature) : (W)(1 / temperature), loss, gradient};
  constexpr int V = 16 / (int)sizeof(T);
  const int vec = vector_width<T>(Mc, support, gradient);
  cudaError_t e;
  if (Mc > 512) {
    e = launch_wide(p, vec, st);
  } else if (vec == V) {
    const long vectors = (Mc + 32 * V - 1) / (32 * V);
    if constexpr (V == 8) {
      e = vectors <= 1 ? launch_warps<T, V, 1>(p, st) : launch_warps<T, V, 2>(p, st);
    } else if constexpr (V == 4) {
      e = vectors <= 1 ? launch_warps<T, V, 1>(p, st) : vectors <= 2 ? launch_warps<T, V, 2>(p, st) : vectors <= 3 ? launch_warps<T, V, 3>(p, st) : launch_warps<T, V, 4>(p, st);
    } else {
      e = vectors <= 1 ? launch_warps<T, V, 1>(p, st) : vectors <= 2 ? launch_warps<T, V, 2>(p, st) : vectors <= 4 ? launch_warps<T, V, 4>(p, st) : launch_warps<T, V, 8>(p, st);
    }
  } else {
    e = Mc <= 32 ? launch_warps<T, 1, 1>(p, st) : Mc <= 64 ? launch_warps<T, 1, 2>(p, st) : Mc <= 128 ? launch_warps<T, 1, 4>(p, st)
        : Mc <= 256 ? launch_warps<T, 1, 8>(p, st) : launch_warps<T, 1, 16>(p, st);
  }
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
