// Distillation from a teacher of which only the best units of each group are kept.
//
// With p the softmax of the teacher's kept units, q the softmax of all of the student's group, both at temperature t, and w the
// row's weight: loss = w t^2 sum_k p_k (log p_k - log q_{u_k}), and d loss / d x_i = w t (q_i - sum over k with u_k = i of p_k).
// What bounds it is memory: the student's support is read once and its gradient written once.  Groups of up to 512 units are 8
// to 32 lanes', in their registers; wider ones a cluster's of blocks, which keep their parts in shared memory for the gradient while they
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

// The same for all of f: exp((f - best) / t), their sum, and a product with one factor; floats two at a time where there are two (the
// exponentials' own pipe is busy half of the time, the rest is the issue of what stands around them).
struct Two {
  unsigned long long v;
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void add(const Two &o) { asm("add.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(o.v)); }
  __device__ __forceinline__ void mul(const Two &o) { asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(o.v)); }
  __device__ __forceinline__ void get(float &a, float &b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
template <typename W, int V>
__device__ __forceinline__ void expo_all(W (&f)[V], W best, W c) {
  if constexpr (sizeof(W) == 4 && V % 2 == 0) {
    const Two minus(-best, -best), factor(c, c);
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      Two d(f[v], f[v + 1]);
      d.add(minus);
      d.mul(factor);
      d.get(f[v], f[v + 1]);
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f[v]));
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f[v + 1]));
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = expo(f[v] - best, c);
  }
}
template <typename W, int V>
__device__ __forceinline__ W sum_all(const W (&f)[V]) {
  if constexpr (sizeof(W) == 4 && V % 2 == 0) {
    Two s(f[0], f[1]);
#pragma unroll
    for (int v = 2; v < V; v += 2) s.add(Two(f[v], f[v + 1]));
    float a, b;
    s.get(a, b);
    return a + b;
  } else {
    W s = f[0];
#pragma unroll
    for (int v = 1; v < V; ++v) s += f[v];
    return s;
  }
}
template <typename W, int V>
__device__ __forceinline__ void scale_all(W (&f)[V], W by) {
  if constexpr (sizeof(W) == 4 && V % 2 == 0) {
    const Two factor(by, by);
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      Two p(f[v], f[v + 1]);
      p.mul(factor);
      p.get(f[v], f[v + 1]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] *= by;
  }
}

template <typename W>
__device__ __forceinline__ W warp_sum(W v) {
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ double warp_max(double v) {
  for (int off = 16; off > 0; off >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}

// ---- lanes of a warp per group ----------------------------------------------

constexpr int kWarpThreads = 256;

// LANES lanes take a group, 8, 16 or 32: as few as hold it in their registers, so that a warp's reductions serve several groups.  Lane l
// holds vectors l, l + LANES, ... of V units each, NV of them.  Instructions and the latency of the reductions bound it: 102400 groups of
// 300 float32 units, 8 kept, 49 us (a warp each 61), 0.79 of a plain copy's bandwidth; 224000 of 100, 5 kept, 53 us (137).
template <typename T, int V, int NV, int LANES>
__global__ void __launch_bounds__(kWarpThreads, sizeof(T) * V * NV <= 80 ? 3 : 2) distill_warp_kernel(const Distill<T> p) {
  after_previous();
  using W = Wide<T>;
  constexpr unsigned kGroups = kWarpThreads / LANES;   // of a block at a time
  __shared__ Vec<W, V> s_kept[kGroups][NV * LANES];   // what the teacher gives each unit
  const unsigned lane = threadIdx.x % LANES, group = threadIdx.x / LANES, step = gridDim.x * kGroups, rows = step / p.H, rest = step % p.H;
  const unsigned first_lane = (threadIdx.x & 31) - lane, mask = (0xffffffffu >> (32 - LANES)) << first_lane;   // the group's lanes
  auto group_max = [&](W v) {
    if constexpr (LANES == 32) return warp_max(v);
    for (int off = LANES / 2; off > 0; off >>= 1) v = fmax(v, __shfl_xor_sync(mask, v, off));
    return v;
  };
  W *const kept = s_kept[group][0].v;
  unsigned g = blockIdx.x * kGroups + group, row = g / p.H, h = g % p.H;
  // the next group's units and teacher, under way while one is worked on
  struct Ahead {
    Vec<T, V> raw[NV];
    unsigned u;
    T t;
  } next;
  auto fetch = [&](unsigned i) {
    const T *const x = p.support + (long)i * p.n;
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if ((r * LANES + lane) * V < p.n) next.raw[r] = *reinterpret_cast<const Vec<T, V> *>(x + (r * LANES + lane) * V);
    if (lane < p.K) {
      next.u = p.unit(i, lane);
      next.t = p.teacher[(long)i * p.K + lane];
    }
  };
  if (g < p.groups) fetch(g);
  for (; g < p.groups; g += step, row += rows, h += rest) {
    if (h >= p.H) h -= p.H, row += 1;
    const T *const x = p.support + (long)g * p.n;
    T *const out = p.gradient + (long)g * p.n;
    const W w = p.weight ? p.weight[row] : (W)1;
    W e[NV][V], best = -INFINITY, total = 0, tbest = -INFINITY, ttotal = 0, sum = 0;
#pragma unroll
    for (int r = 0; r < NV; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) e[r][v] = (r * LANES + lane) * V < p.n ? widen(next.raw[r].v[v]) : (W)-INFINITY;
    const unsigned u0 = lane < p.K ? next.u : p.n;
    const W t0 = u0 < p.n ? widen(next.t) : (W)-INFINITY, x0 = u0 < p.n ? widen(x[u0]) : (W)0;
    if (g + step < p.groups) fetch(g + step);
    if (w != (W)0) {
#pragma unroll
      for (int r = 0; r < NV; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) best = fmax(best, e[r][v]);
      best = group_max(best);
      tbest = t0;
      for (unsigned k = lane + LANES; k < p.K; k += LANES)
        if (p.unit(g, k) < p.n) tbest = fmax(tbest, widen(p.teacher[(long)g * p.K + k]));
      tbest = group_max(tbest);
    }
    bool nothing = w == (W)0 || best == -INFINITY || tbest == -INFINITY;
    if (nothing && w != (W)0) {   // (the maxima pass over NaN, which is not nothing)
      bool nan = false, teacher_nan = u0 < p.n && t0 != t0;
#pragma unroll
      for (int r = 0; r < NV; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) nan = nan || e[r][v] != e[r][v];
      for (unsigned k = lane + LANES; k < p.K; k += LANES)
        teacher_nan = teacher_nan || (p.unit(g, k) < p.n && isnan(widen(p.teacher[(long)g * p.K + k])));
      const bool student = best != -INFINITY || __any_sync(mask, nan), teacher = tbest != -INFINITY || __any_sync(mask, teacher_nan);
      nothing = !student || !teacher;
    }
    if (nothing) {
      if (lane == 0) p.loss[g] = 0;
      if (p.gradient) {
        Vec<T, V> zero;
#pragma unroll
        for (int v = 0; v < V; ++v) zero.v[v] = narrow_to<T>((W)0);
#pragma unroll
        for (int r = 0; r < NV; ++r)
          if ((r * LANES + lane) * V < p.n) *reinterpret_cast<Vec<T, V> *>(out + (r * LANES + lane) * V) = zero;
      }
      continue;
    }
    if (p.gradient) {
      Vec<W, V> zero;
#pragma unroll
      for (int v = 0; v < V; ++v) zero.v[v] = 0;
#pragma unroll
      for (int r = 0; r < NV; ++r) s_kept[group][r * LANES + lane] = zero;
      __syncwarp(mask);
    }
#pragma unroll
    for (int r = 0; r < NV; ++r) {
      expo_all(e[r], best, p.c);
      total += sum_all(e[r]);
    }
    const W inv = (W)1 / p.temperature;
    // the teacher's side without its divisor, so that three sums run side by side
    auto entry = [&](bool there, W t, W xu) {
      const W pk = there ? expo(t - tbest, p.c) : (W)0;
      ttotal += pk;
      if (!(pk == (W)0)) sum += pk * (((t - tbest) - (xu - best)) * inv);
      return pk;
    };
    const W p0 = entry(u0 < p.n, t0, x0);
    for (unsigned k = lane + LANES; k < p.K; k += LANES) {
      const unsigned u = p.unit(g, k);
      if (u < p.n) entry(true, widen(p.teacher[(long)g * p.K + k]), widen(x[u]));
    }
    for (int off = LANES / 2; off > 0; off >>= 1) {
      total += __shfl_xor_sync(mask, total, off);
      ttotal += __shfl_xor_sync(mask, ttotal, off);
      sum += __shfl_xor_sync(mask, sum, off);
    }
    const W share = (W)1 / ttotal;
    sum = sum * share + (sbb_log(total) - sbb_log(ttotal));
    if (p.gradient)
      for (unsigned k0 = 0; k0 < p.K; k0 += LANES) {
        unsigned u = u0;
        W pk = p0;
        if (k0 > 0) {
          u = k0 + lane < p.K ? p.unit(g, k0 + lane) : p.n;
          pk = u < p.n ? expo(widen(p.teacher[(long)g * p.K + k0 + lane]) - tbest, p.c) : (W)0;
        }
        pk *= share;
        // A unit named twice has both parts, added in the order of the entries: whoever reads another's mark than its own has one.
        const bool there = u < p.n;
        W before = 0;
        if (there && k0 > 0) before = kept[u];
        __syncwarp(mask);
        if (there) kept[u] = (W)lane;
        __syncwarp(mask);
        if (__any_sync(mask, there && kept[u] != (W)lane)) {
          const unsigned same = __match_any_sync(mask, there ? u : ~lane) >> first_lane;
          W part = 0;
          for (int j = 0; j < LANES; ++j) {
            const W o = __shfl_sync(mask, pk, j, LANES);
            if (same >> j & 1) part += o;
          }
          pk = part;
        }
        __syncwarp(mask);
        if (there) kept[u] = before + pk;   // (those that name the same unit write the same)
        __syncwarp(mask);
      }
    if (lane == 0) p.loss[g] = w * p.temperature * p.temperature * sum;
    if (!p.gradient) continue;
    const W wt = w * p.temperature, scale = wt / total;
#pragma unroll
    for (int r = 0; r < NV; ++r)
      if ((r * LANES + lane) * V < p.n) {
        const Vec<W, V> k = s_kept[group][r * LANES + lane];
        scale_all(e[r], scale);
#pragma unroll
        for (int v = 0; v < V; ++v) e[r][v] -= wt * k.v[v];
        *reinterpret_cast<Vec<T, V> *>(out + (r * LANES + lane) * V) = narrow_all<T, V>(e[r]);
      }
    __syncwarp(mask);
  }
}

// ---- a cluster per group ---------------------------------------------------

constexpr int kMostBlocks = 8;
constexpr int kStage = 100 * 1024;   // bytes of a group that a block keeps in shared memory
// Threads of a block: as many kept units wait in shared memory; longer lists are read again, as many at a time.  Groups of up to 8192 units go to
// small blocks: 16000 groups of 520 float32 units take 55 us, and took 151 in large ones; 4000 of 6000 units 47 and 57.
constexpr int kLarge = 512, kSmall = 128;
constexpr unsigned kSmallMost = 8192;

// A running maximum and the sum of exp((x - maximum) / t).
template <typename W>
struct Running {
  W best, sum;
  __device__ __forceinline__ void move_to(W b, W c) {   // b: no less than best
    if (best != b) sum *= expo(best - b, c), best = b;
  }
  __device__ __forceinline__ void add(W v, W c) {
    if (v > best) move_to(v, c);
    sum += v == -INFINITY ? (W)0 : v == best && v < (W)INFINITY ? (W)1 : expo(v - (best == -INFINITY ? (W)0 : best), c);   // (+infinity: NaN)
  }
};

template <typename W, int THREADS>
struct Block {
  W best[2][THREADS / 32], sum[2][THREADS / 32], loss[THREADS / 32];
  Running<W> own;
  Vec<W, 2> kept[THREADS];   // unit (as bits), p
};

// Two of them over all threads; all have the same bits.  (Joining maxima and sums one by one took as long as a row of 32000 units
// itself.)
template <typename W, int THREADS>
__device__ __forceinline__ void block_join(Running<W> &r, Running<W> &t, W c, Block<W, THREADS> &s) {
  constexpr unsigned kBlockWarps = THREADS / 32;
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const W r_warp = warp_max(r.best), t_warp = warp_max(t.best);
  if (lane == 0) s.best[0][warp] = r_warp, s.best[1][warp] = t_warp;
  __syncthreads();
  r.move_to(warp_max(lane < kBlockWarps ? s.best[0][lane] : (W)-INFINITY), c);
  t.move_to(warp_max(lane < kBlockWarps ? s.best[1][lane] : (W)-INFINITY), c);
  const W r_sum = warp_sum(r.sum), t_sum = warp_sum(t.sum);
  if (lane == 0) s.sum[0][warp] = r_sum, s.sum[1][warp] = t_sum;
  __syncthreads();
  r.sum = warp_sum(lane < kBlockWarps ? s.sum[0][lane] : (W)0);
  t.sum = warp_sum(lane < kBlockWarps ? s.sum[1][lane] : (W)0);
}

// STAGED: the part waits in shared memory between the sum and the gradient; else (no gradient, or groups beyond what a cluster
// holds) it is read again.  LONG: there is a gradient and a list of more entries than threads; `room` units' parts of it fit the shared
// memory.  (Within the kernel for short lists, 512 x 50001 float16 took 34.5 us and not 33, without a gradient 20 and not 18.5.)
// VECTOR: 16-byte accesses from the first boundary on, the elements in front of it and behind the last one by single threads; else
// (support and gradient lie differently to the boundaries) element by element.
// Instructions, and phases that do not overlap within a block, bound it: 4096 x 32000 bf16 units, 64 kept, 114 us, 62 % of the issue slots
// busy, 0.70 of a plain copy's bandwidth.
template <typename T, bool VECTOR, bool STAGED, int THREADS, bool LONG>
__global__ void __launch_bounds__(THREADS, 1536 / THREADS) distill_block_kernel(const Distill<T> p, unsigned part, unsigned room) {
  after_previous();
  using W = Wide<T>;
  constexpr unsigned kThreads = THREADS, kBlockWarps = THREADS / 32;
  constexpr int V = VECTOR ? 16 / (int)sizeof(T) : 1;
  extern __shared__ uint4 s_values[];
  __shared__ Block<W, THREADS> s;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned blocks = cluster.num_blocks(), g = blockIdx.x / blocks, rank = cluster.block_rank(), lane = threadIdx.x & 31;
  const unsigned begin = min(p.n, rank * part), size = min(part, p.n - begin);
  const T *const x = p.support + (long)g * p.n + begin;
  T *const out = p.gradient ? p.gradient + (long)g * p.n + begin : nullptr;
  const unsigned lead = VECTOR ? min(size, (unsigned)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (unsigned)sizeof(T)) : 0;
  const unsigned vectors = (size - lead) / V, tail = size - lead - vectors * V;
  unsigned single = size;   // the thread's element outside the vectors
  if constexpr (VECTOR) {
    if (threadIdx.x < lead) single = threadIdx.x;
    if (threadIdx.x - 32 < tail) single = lead + vectors * V + threadIdx.x - 32;   // (a warp of its own)
  }
  Vec<T, V> *const stage = reinterpret_cast<Vec<T, V> *>(s_values);
  const Vec<T, V> *const from = reinterpret_cast<const Vec<T, V> *>(x + lead);
  const W w = p.weight ? p.weight[g / p.H] : (W)1;
  Running<W> r{-INFINITY, 0}, t{-INFINITY, 0};
  // the thread's first kept unit, under way while the row is read
  unsigned u0 = p.n;
  W t0 = 0, x0 = 0, own = 0;
  if (w != (W)0) {
    if (threadIdx.x < p.K) {
      u0 = p.unit(g, threadIdx.x);
      t0 = widen(p.teacher[(long)g * p.K + threadIdx.x]);
    }
    if (single < size) own = widen(x[single]);
    constexpr int U = 4;
    for (unsigned i = threadIdx.x; i < vectors; i += U * kThreads) {
      Vec<T, V> a[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < vectors) a[u] = from[i + u * kThreads];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * kThreads >= vectors) break;
        if constexpr (STAGED) stage[i + u * kThreads] = a[u];
        const W m = max_all(a[u]);
        if (m > r.best) r.move_to(m, p.c);
        const W b = r.best == -INFINITY ? (W)0 : r.best;
        W f[V];
        widen_all(a[u], f);
        expo_all(f, b, p.c);
        r.sum += sum_all(f);
      }
    }
    if (single < size) r.add(own, p.c);
    if (u0 < p.n) {
      x0 = widen(p.support[(long)g * p.n + u0]);
      t.add(t0, p.c);
    }
    for (unsigned k = threadIdx.x + kThreads; k < p.K; k += kThreads)
      if (p.unit(g, k) < p.n) t.add(widen(p.teacher[(long)g * p.K + k]), p.c);
    block_join(r, t, p.c, s);
    if (blocks > 1) {
      if (threadIdx.x == 0) s.own = r;
      cluster.sync();
      W best = r.best;
      for (unsigned b = 0; b < blocks; ++b) best = fmax(best, cluster.map_shared_rank(&s, b)->own.best);
      W sum = 0;
      for (unsigned b = 0; b < blocks; ++b) {
        Running<W> o = cluster.map_shared_rank(&s, b)->own;
        o.move_to(best, p.c);
        sum += o.sum;
      }
      r = Running<W>{best, sum};
      cluster.sync();   // (a block may go on to its end, which the others read from)
    }
  }
  if (w == (W)0 || (r.best == -INFINITY && r.sum == (W)0) || (t.best == -INFINITY && t.sum == (W)0)) {
    if (rank == 0 && threadIdx.x == 0) p.loss[g] = 0;
    if (out) {
      Vec<T, V> zero;
#pragma unroll
      for (int v = 0; v < V; ++v) zero.v[v] = narrow_to<T>((W)0);
      for (unsigned i = threadIdx.x; i < vectors; i += kThreads) reinterpret_cast<Vec<T, V> *>(out + lead)[i] = zero;
      if (single < size) out[single] = narrow_to<T>((W)0);
    }
    return;
  }
  const W inv = (W)1 / p.temperature, shift = sbb_log(r.sum) - sbb_log(t.sum), wt = w * p.temperature, scale = wt / r.sum, share = (W)1 / t.sum;
  auto p_of = [&](W v) { return expo(v - t.best, p.c) * share; };
  const bool listed = !LONG && p.K <= kThreads;
  {
    W sum = 0;
    for (unsigned k = threadIdx.x; k < p.K; k += kThreads) {
      unsigned u = u0;
      W v = t0, xu = x0;
      if (k >= kThreads) {
        u = p.unit(g, k);
        if (u < p.n) v = widen(p.teacher[(long)g * p.K + k]), xu = widen(p.support[(long)g * p.n + u]);
      }
      const W pk = u < p.n ? p_of(v) : (W)0;
      if (!(pk == (W)0)) sum += pk * (((v - t.best) - (xu - r.best)) * inv + shift);
      if (listed) {
        s.kept[k].v[1] = pk;
        *reinterpret_cast<unsigned *>(&s.kept[k].v[0]) = u;
      }
    }
    sum = warp_sum(sum);
    if (lane == 0) s.loss[threadIdx.x >> 5] = sum;
  }
  __syncthreads();
  if (rank == 0 && threadIdx.x < 32) {
    const W sum = warp_sum(lane < kBlockWarps ? s.loss[lane] : (W)0);
    if (lane == 0) p.loss[g] = w * p.temperature * p.temperature * sum;
  }
  if (!out) return;
  // What the teacher gives the unit of this thread's entry, if the entry is the first that names it; the parts in order.
  auto given = [&](unsigned k, unsigned u, W &sum) {
    bool first = true;
    sum = 0;
    for (unsigned j = 0; j < p.K; ++j) {
      const Vec<W, 2> e = s.kept[j];
      const unsigned o = *reinterpret_cast<const unsigned *>(&e.v[0]);
      if (o == u) {
        first = first && j >= k;
        sum += e.v[1];
      }
    }
    return first;
  };
  W sum0 = 0;
  const bool mine = !LONG && u0 >= begin && u0 < begin + size && given(threadIdx.x, u0, sum0);
  for (unsigned i = threadIdx.x; i < vectors; i += kThreads) {
    W f[V];
    widen_all(STAGED ? stage[i] : from[i], f);
    expo_all(f, r.best, p.c);
    scale_all(f, scale);
    reinterpret_cast<Vec<T, V> *>(out + lead)[i] = narrow_all<T, V>(f);
  }
  if (single < size) out[single] = narrow_to<T>(expo(own - r.best, p.c) * scale);
  __syncthreads();   // the kept units' elements are written again
  if (mine) out[u0 - begin] = narrow_to<T>(expo(x0 - r.best, p.c) * scale - wt * sum0);
  if constexpr (!LONG) return;
  // A long list: what the teacher gives `room` units at a time is added up in shared memory, kThreads entries at a time.  (Comparing every
  // entry with all others took the square of their number.)
  W *const parts = reinterpret_cast<W *>(s_values);
  for (unsigned lo = 0; lo < size; lo += room) {
    const unsigned here = min(room, size - lo);
    for (unsigned i = threadIdx.x; i < here; i += kThreads) parts[i] = 0;
    __syncthreads();
    for (unsigned k0 = 0; k0 < p.K; k0 += kThreads) {
      const unsigned k = k0 + threadIdx.x, u = k < p.K ? p.unit(g, k) : p.n, at = u - begin - lo;   // (wraps for units in front)
      const bool there = u < p.n && at < here;
      W sum = there ? p_of(widen(p.teacher[(long)g * p.K + k])) : (W)0;
      s.kept[threadIdx.x].v[1] = sum;
      *reinterpret_cast<unsigned *>(&s.kept[threadIdx.x].v[0]) = there ? at : ~0u;
      const W before = there ? parts[at] : (W)0;
      __syncthreads();
      // Whoever reads another's mark than its own shares its unit: the parts in the order of the entries then.
      if (there) parts[at] = (W)threadIdx.x;
      __syncthreads();
      const bool shared = there && parts[at] != (W)threadIdx.x;
      if (__syncthreads_or(shared) && there) {
        sum = 0;
        for (unsigned j = 0; j < kThreads; ++j) {
          const Vec<W, 2> e = s.kept[j];
          if (*reinterpret_cast<const unsigned *>(&e.v[0]) == at) sum += e.v[1];
        }
      }
      if (there) parts[at] = before + sum;   // (those that name the same unit write the same)
      __syncthreads();
    }
    for (unsigned i = threadIdx.x; i < here; i += kThreads) {
      const W given = parts[i];
      if (given != (W)0) out[lo + i] = narrow_to<T>(expo(widen(x[lo + i]) - r.best, p.c) * scale - wt * given);
    }
    __syncthreads();
  }
}

template <typename T, int V, int NV, int LANES>
cudaError_t launch_warps(const Distill<T> &p, cudaStream_t st) {
  constexpr unsigned groups = kWarpThreads / LANES;
  const unsigned most = 16 * (unsigned)sm_count(), blocks = (p.groups + groups - 1) / groups;
  return launch_next(distill_warp_kernel<T, V, NV, LANES>, dim3(blocks < most ? blocks : most), kWarpThreads, 0, st, p);
}

template <typename T, bool VECTOR, bool STAGED, int THREADS, bool LONG = false>
cudaError_t launch_blocks(const Distill<T> &p, unsigned part, unsigned cluster, cudaStream_t st) {
  size_t smem = STAGED ? (size_t)part * sizeof(T) : 0;
  unsigned room = 0;
  if constexpr (LONG) {
    constexpr unsigned most = kStage / sizeof(Wide<T>);
    room = part < most ? part : most;
    if (smem < room * sizeof(Wide<T>)) smem = room * sizeof(Wide<T>);
  }
  auto kernel = distill_block_kernel<T, VECTOR, STAGED, THREADS, LONG>;
  if (smem > 0) {   // (holds for the current device)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kStage);
    if (e != cudaSuccess) return e;
  }
  return launch_clusters(kernel, dim3(p.groups * cluster), dim3(cluster), THREADS, smem, st, p, part, room);
}

template <typename T>
cudaError_t launch_wide(const Distill<T> &p, cudaStream_t st) {
  const size_t bytes = (size_t)p.n * sizeof(T);
  unsigned cluster = 1;
  // the smallest cluster whose blocks hold their parts; a larger one where groups are too few for the SMs and parts long
  if (p.gradient)
    while (cluster < kMostBlocks && bytes > (size_t)cluster * kStage) cluster *= 2;
  while (cluster < kMostBlocks && (size_t)p.groups * cluster * 2 <= (size_t)sm_count() && p.n / cluster > 4096) cluster *= 2;
  const unsigned part = ((p.n + cluster - 1) / cluster + 15) / 16 * 16;
  if ((size_t)p.groups * cluster > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const bool staged = p.gradient && (size_t)part * sizeof(T) <= kStage;
  const bool vector = !p.gradient || ((reinterpret_cast<uintptr_t>(p.support) ^ reinterpret_cast<uintptr_t>(p.gradient)) & 15) == 0;
  if (p.gradient && p.K > (p.n <= kSmallMost && cluster == 1 ? kSmall : kLarge)) {   // (groups for small blocks are staged)
    if (!vector) return launch_blocks<T, false, false, kLarge, true>(p, part, cluster, st);
    if (p.n <= kSmallMost && cluster == 1) return launch_blocks<T, true, true, kSmall, true>(p, part, 1, st);
    return staged ? launch_blocks<T, true, true, kLarge, true>(p, part, cluster, st) : launch_blocks<T, true, false, kLarge, true>(p, part, cluster, st);
  }
  if (p.n <= kSmallMost && cluster == 1) {
    if (vector) return staged ? launch_blocks<T, true, true, kSmall>(p, part, 1, st) : launch_blocks<T, true, false, kSmall>(p, part, 1, st);
    return staged ? launch_blocks<T, false, true, kSmall>(p, part, 1, st) : launch_blocks<T, false, false, kSmall>(p, part, 1, st);
  }
  if (vector) return staged ? launch_blocks<T, true, true, kLarge>(p, part, cluster, st) : launch_blocks<T, true, false, kLarge>(p, part, cluster, st);
  return staged ? launch_blocks<T, false, true, kLarge>(p, part, cluster, st) : launch_blocks<T, false, false, kLarge>(p, part, cluster, st);
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
    e = launch_wide(p, st);
  } else if (Mc <= 64) {   // eight lanes a group.  227000 float64 groups of 16, 16 kept, without a gradient: 63 us, with a warp each 173
    if (vec != V) {
      e = Mc <= 8 ? launch_warps<T, 1, 1, 8>(p, st) : Mc <= 16 ? launch_warps<T, 1, 2, 8>(p, st) : Mc <= 32 ? launch_warps<T, 1, 4, 8>(p, st)
          : launch_warps<T, 1, 8, 8>(p, st);
    } else if constexpr (V == 8) {
      e = launch_warps<T, V, 1, 8>(p, st);
    } else if constexpr (V == 4) {
      e = Mc <= 32 ? launch_warps<T, V, 1, 8>(p, st) : launch_warps<T, V, 2, 8>(p, st);
    } else {
      e = Mc <= 16 ? launch_warps<T, V, 1, 8>(p, st) : Mc <= 32 ? launch_warps<T, V, 2, 8>(p, st) : launch_warps<T, V, 4, 8>(p, st);
    }
  } else if (Mc <= 128) {
    e = vec == V ? launch_warps<T, V, 16 / V, 8>(p, st) : launch_warps<T, 1, 16, 8>(p, st);
  } else if (vec == V) {   // (20 float32 units a lane leave registers for three blocks on an SM: with two, groups of 300 take 62 us, not 49)
    if constexpr (V == 8) {
      e = Mc <= 256 ? launch_warps<T, V, 4, 8>(p, st) : launch_warps<T, V, 4, 16>(p, st);
    } else if constexpr (V == 4) {
      e = Mc <= 256 ? launch_warps<T, V, 4, 16>(p, st) : Mc <= 320 ? launch_warps<T, V, 5, 16>(p, st) : Mc <= 384 ? launch_warps<T, V, 3, 32>(p, st)
          : launch_warps<T, V, 4, 32>(p, st);
    } else {
      e = Mc <= 256 ? launch_warps<T, V, 8, 16>(p, st) : launch_warps<T, V, 8, 32>(p, st);
    }
  } else {
    e = Mc <= 256 ? launch_warps<T, 1, 16, 16>(p, st) : launch_warps<T, 1, 16, 32>(p, st);
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
