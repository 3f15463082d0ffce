// Drawing a unit of every group from the softmax of its support, with temperature, top-k, top-p and min-p, from given numbers.
//
// With w_i = exp((x_i - max) / t) and the units in order of falling w (equal ones: lowest index first), top-k, top-p and min-p
// each keep a beginning of that order, so what is kept is all units not behind one (value, index): a cut.  Finding it takes no
// sort of the group: counts and masses over parts of the values' range say in which part it lies, and the few units of that part
// are compared with one another.
// A random number may lie next to the border of two units, and of a million draws some do within 32 bits' accuracy.  So weights
// are formed in 64 bits and summed as integers, multiples of 2^-q: the sums are the same in any order and their errors below
// n 2^-q of the largest weight; where the random number is small, of what is looked for (Lift).
// Groups of up to 512 units (1024 of the types summed in 32 bits) are a warp's, in its registers; wider ones a cluster's of blocks, each
// with a part of the group in shared memory, so that the support is read from memory once.
// (A source for each type, compiled side by side, includes this.)
#pragma once
#include "sbb_codes.cuh"
#include "sbb_launch.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

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
  static __device__ __forceinline__ float value(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
};
template <>
struct Keys<double> {
  using type = u64;
  static __device__ __forceinline__ u64 of(double v) {
    const u64 b = (u64)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
  }
  static __device__ __forceinline__ double value(u64 k) { return __longlong_as_double((long long)(k >> 63 ? k ^ (1ull << 63) : ~k)); }
};
template <typename W>
__device__ __forceinline__ W no_nan(W v) {
  return v == v ? v : (W)-INFINITY;
}

struct Settings {
  double inv_t, top_p, min_p;
  unsigned top_k;   // n: all
};
__host__ __device__ __forceinline__ double inverse(double t) { return t > 1e-300 ? 1 / t : t > 0 ? 1e300 : 1; }
__device__ __forceinline__ double min_p_of(const Sampling &s, long row) { return s.min_p_rows ? (double)s.min_p_rows[row] : s.min_p; }
__device__ __forceinline__ Settings settings_of(const Sampling &s, long row, unsigned n) {
  const bool own = s.temperature_rows != nullptr;
  const float t = own ? s.temperature_rows[row] : s.temperature > 0 ? 1 : 0;
  const long k = s.top_k_rows ? (long)s.top_k_rows[row] : s.top_k;
  Settings r;
  r.top_k = k <= 0 || k > (long)n ? n : (unsigned)k;
  r.top_p = s.top_p_rows ? (double)s.top_p_rows[row] : s.top_p;
  r.min_p = min_p_of(s, row);
  if (!(t > 0)) r.top_k = 1;
  r.inv_t = own ? inverse((double)t) : s.inv_t;
  return r;
}

// round(exp(d / t) 2^q) for d <= 0, by Tang's method (ACM TOMS 15, 1989): 2^(n/64) from a table, exp of the rest (below
// ln 2 / 128) by its series to the fifth power (3e-17).  A dozen operations on the FP64 pipe.
constexpr int kTable = 64;
struct Weights {
  const double *table;   // 2^(j/64), in shared memory
  double c;              // 64 / (t ln 2)
  int q;

  static __device__ __forceinline__ void fill(double *table) {
    if (threadIdx.x < kTable) table[threadIdx.x] = exp2(threadIdx.x * (1.0 / kTable));
  }
  __device__ __forceinline__ Weights(const double *tab, double inv_t, int q_) : table(tab), c(inv_t * 92.332482616893656877), q(q_) {}
  __device__ __forceinline__ u64 one() const { return 1ull << q; }
  // 2^lift times the mass of a weight of 2^(x/64)
  __device__ __forceinline__ u64 power(double x, int lift) const {
    constexpr double kRound = 6755399441055744.0;            // 1.5 * 2^52: what is added to it is rounded to an integer
    constexpr double a = 0.010830424696249145252;            // ln 2 / 64
    constexpr double a2 = a * a / 2, a3 = a2 * a / 3, a4 = a3 * a / 4, a5 = a4 * a / 5;
    if (!(x > -(double)kTable * (q + lift + 2))) return 0;
    const double big = x + kRound, r = x - (big - kRound);
    const int n = __double2loint(big);
    const double p = fma(fma(fma(fma(fma(a5, r, a4), r, a3), r, a2), r, a), r, 1.0);
    const double v = table[n & (kTable - 1)] * p;
    const double scaled = __hiloint2double(__double2hiint(v) + (((n >> 6) + q + lift) << 20), __double2loint(v));
    return (u64)__double_as_longlong(scaled + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
  template <typename W>
  __device__ __forceinline__ u64 of(W v, W best) const {   // v is no NaN
    return v == best ? one() : power(((double)v - (double)best) * c, 0);
  }
  // 2^lift times the weight where that is less than the largest, else as much as the largest
  template <typename W>
  __device__ __forceinline__ u64 lifted(W v, W best, int lift) const {
    const double x = ((double)v - (double)best) * c;
    return v == best || x >= -(double)kTable * lift ? one() : power(x, lift);
  }
  // Whether a weight reaches min_p, however small: compared where min_p lies from 1/2 to 1
  template <typename W>
  __device__ __forceinline__ bool reaches(W v, W best, double min_p) const {
    if (!(min_p > 0)) return true;
    const int lift = max(0, 1022 - (__double2hiint(min_p) >> 20));
    return lifted(v, best, lift) >= (u64)__double2ll_rn(fmin(ldexp(min_p, lift), 1.0) * (double)one());
  }
};

// A small random number may fall to units whose weights are nothing, or a few multiples of 2^-q, beside the largest.  The draw is then
// made by weights multiplied by 2^lift and cut off at 2^q, where what is looked for, the random number times the sum of the kept
// weights, lies from 2^(q-1) to 2^q: sums up to it are exact to n 2^-q of it, and a weight that is cut off passes it by itself.
// For 0 (and what is below, and NaN) it is the first unit whose weight is above 0 in 64 bits.
// Small is below 2^-20: other numbers pass what weights below 2^-q may add up to, and so few draws are small that the microseconds
// they take longer are hardly met (with 2^-12, 40960 groups of 256 float32 units took 55 us and not 53).  What draws them is kept short,
// so that it takes few registers from the others: a call to a function of its own at the end of a block's draw cost 4000 groups of 8192
// float32 units with a top-p 316 us and not 309, and 256 x 128000 bf16 with settings of each row 2 %.
__device__ __forceinline__ bool is_small(float random) { return !(random >= 1.f / (1 << 20)); }
struct Lift {
  int lift;
  u64 target;   // what is looked for
  __device__ __forceinline__ Lift(float random, u64 total, int q) {
    const double at = (double)random * (double)total;
    lift = at > 0 ? max(0, q - 1 - ((__double2hiint(at) >> 20) - 1023)) : 1074 - q;   // (0: of very many weights; less than their sum)
    target = at > 0 ? (u64)ldexp(at, lift) : 0;
  }
};

// A cut, and the mass of what is not behind it.
template <typename Key>
struct Cut {
  Key key;
  unsigned index;
  u64 mass;
};
template <typename Key>
__device__ __forceinline__ bool kept(Key key, unsigned i, const Cut<Key> &c) {
  return key > c.key || (key == c.key && i <= c.index);
}
// Whether a unit with this much in front of it is kept: by count where a count is asked for, else by mass; the first always.
struct Want {
  bool by_count;
  unsigned count;
  u64 limit;
  __device__ __forceinline__ bool inside(unsigned c, u64 m) const { return by_count ? c < count : c == 0 || m < limit; }
};
__device__ __forceinline__ Want want_count(unsigned count) { return Want{true, count, 0}; }
// less than top_p of the mass in front: integers below the product are those below the next integer
__device__ __forceinline__ Want want_mass(double top_p, u64 mass) { return Want{false, 0, top_p > 0 ? __double2ull_ru(top_p * (double)mass) : 0}; }
// How many of `in` equal units of mass m are kept, the first of which is.
__device__ __forceinline__ unsigned equal_ones(const Want &w, unsigned in, u64 m, unsigned above_count, u64 above_mass) {
  if (w.by_count) return min(in, w.count - above_count);
  if (m == 0) return in;
  if (w.limit <= above_mass) return 1;
  return (unsigned)min((u64)in, (w.limit - above_mass + m - 1) / m);
}
__device__ __forceinline__ u64 target_of(float random, u64 total) {
  const double at = (double)random * (double)total;
  const u64 t = at > 0 ? at < 9e18 ? (u64)at : total : 0;
  return t < total ? t : total - 1;   // (a random number of 1, or the product's rounding)
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
// The same for values below 2^54, in two sums of 27 bits.
__device__ __forceinline__ u64 warp_sum_54(u64 v) {
  const unsigned lo = __reduce_add_sync(0xffffffffu, (unsigned)v & 0x7ffffffu), hi = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 27));
  return ((u64)hi << 27) + lo;
}
template <typename V>
__device__ __forceinline__ V warp_up_to(V v) {   // the sum over the lanes in front and one's own
  const int lane = threadIdx.x & 31;
  for (int off = 1; off < 32; off *= 2) {
    const V o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  return v;
}
__device__ __forceinline__ unsigned warp_max(unsigned v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ u64 warp_max(u64 v) {
  for (int off = 16; off > 0; off >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
__device__ __forceinline__ unsigned warp_min(unsigned v) { return __reduce_min_sync(0xffffffffu, v); }
__device__ __forceinline__ u64 warp_min(u64 v) { return ~warp_max(~v); }

// ---- a warp per group ------------------------------------------------------

// Blocks on an SM, as registers allow; the launch has twice as many, since some draws take longer.  Lanes of 32 units leave no registers
// for the next group's.
template <int EACH>
constexpr int kWarpBlocks = EACH <= 4 ? 4 : EACH <= 8 ? 3 : 2;

constexpr int kWarpThreads = 256, kWarps = kWarpThreads / 32;
constexpr int kWarpBits = 48;   // q: the sum of a lane's 32 masses stays below 2^54

template <typename Key>
struct alignas(16) Few {   // the units a cut lies among
  Key key[32];
  u64 mass[32];
  unsigned index[32];
};

// A group in a warp: lane l holds units l * EACH to l * EACH + EACH - 1, those behind the group's end at -infinity.
template <typename W, int EACH>
struct WarpGroup {
  using Key = typename Keys<W>::type;
  Key key[EACH];
  u64 mass[EACH];

  __device__ __forceinline__ unsigned first() const { return (threadIdx.x & 31) * EACH; }

  // `behind`: units of at most this mass are behind the cut.
  __device__ __forceinline__ Cut<Key> cut(const Want &want, u64 behind, Key best, Few<Key> &few) const {
    const unsigned lane = threadIdx.x & 31;
    // units in [lo, hi], units above; those at -infinity, which are never drawn, are out of it
    const Key none = Keys<W>::of((W)-INFINITY);
    Key lo = ~(Key)0, hi = best;
    unsigned to_lo = 0, above_count = 0;   // units from lo up, from above hi up
#pragma unroll
    for (int r = 0; r < EACH; ++r)
      if (key[r] > none && (want.by_count || mass[r] > behind)) lo = min(lo, key[r]);
    lo = warp_min(lo);
#pragma unroll
    for (int r = 0; r < EACH; ++r) to_lo += key[r] >= lo;
    to_lo = __reduce_add_sync(0xffffffffu, to_lo);
    u64 above_mass = 0;
    for (int round = 0; to_lo - above_count > 32 && lo < hi; ++round) {
      const W mid = Keys<W>::value(lo) * (W)0.5 + Keys<W>::value(hi) * (W)0.5;
      Key pivot = round < 8 && mid == mid ? Keys<W>::of(mid) : lo + (hi - lo) / 2 + 1;   // half the values, later half the bits
      pivot = pivot <= lo ? lo + 1 : pivot > hi ? hi : pivot;
      unsigned c = 0;
      u64 m = 0;
#pragma unroll
      for (int r = 0; r < EACH; ++r)
        if (key[r] >= pivot) c += 1, m += mass[r];
      c = __reduce_add_sync(0xffffffffu, c);
      if (!want.by_count) m = warp_sum_54(m);
      if (c < to_lo && want.inside(c, m)) {
        above_count = c;
        above_mass = m;
        hi = pivot - 1;
      } else {
        to_lo = c;
        lo = pivot;
      }
    }
    const unsigned in = to_lo - above_count;
    Cut<Key> r;
    unsigned c = 0;
#pragma unroll
    for (int q = 0; q < EACH; ++q) c += key[q] >= lo && key[q] <= hi;
    unsigned at = warp_up_to(c) - c;
    if (in > 32) {   // equal ones
      u64 m = 0;
#pragma unroll
      for (int q = 0; q < EACH; ++q)
        if (key[q] == lo) m = mass[q];
      m = warp_max(m);
      const unsigned take = equal_ones(want, in, m, above_count, above_mass);
      unsigned index = 0;
#pragma unroll
      for (int q = 0; q < EACH; ++q)
        if (key[q] == lo && ++at == take) index = first() + q + 1;
      r.key = lo;
      r.index = __reduce_max_sync(0xffffffffu, index) - 1;
      r.mass = above_mass + take * m;
    } else {
      // In index order, a lane each; in the order of the values once more, for the masses in front.
#pragma unroll
      for (int q = 0; q < EACH; ++q)
        if (key[q] >= lo && key[q] <= hi) {
          few.key[at] = key[q];
          few.mass[at] = mass[q];
          few.index[at] = first() + q;
          ++at;
        }
      if (lane >= in) few.key[lane] = 0;   // (no unit's key)
      __syncwarp();
      const Key k = few.key[lane];
      const u64 m = lane < in ? few.mass[lane] : 0;
      unsigned rank = __popc(__match_any_sync(0xffffffffu, k) & ((1u << lane) - 1));
      constexpr int V = 16 / (int)sizeof(Key);
#pragma unroll
      for (int j = 0; j < 32; j += V) {
        const Vec<Key, V> o = *reinterpret_cast<const Vec<Key, V> *>(&few.key[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) rank += o.v[i] > k;
      }
      __syncwarp();
      if (lane < in) few.mass[rank] = m;
      __syncwarp();
      const u64 by_rank = lane < in ? few.mass[lane] : 0, before = above_mass + warp_up_to(by_rank) - by_rank;
      // (the last lane inside: every rank in front of it is inside too)
      const unsigned last = __popc(__ballot_sync(0xffffffffu, lane < in && want.inside(above_count + lane, before))) - 1;
      const unsigned who = __ffs(__ballot_sync(0xffffffffu, lane < in && rank == last)) - 1;
      r.key = __shfl_sync(0xffffffffu, k, who);
      r.index = few.index[who];
      r.mass = __shfl_sync(0xffffffffu, before + by_rank, last);
      __syncwarp();
    }
    if (want.by_count) {   // the masses in front have not been summed in the rounds
      u64 all = 0;
#pragma unroll
      for (int q = 0; q < EACH; ++q)
        if (kept(key[q], first() + q, r)) all += mass[q];
      r.mass = warp_sum_54(all);
    }
    return r;
  }
};

// A lane's units as they are in memory; what is done to them waits until they are used.
template <typename T, int EACH>
__device__ __forceinline__ void load_units(const T *x, unsigned n, bool whole, T (&v)[EACH]) {
  const unsigned first = (threadIdx.x & 31) * EACH;
  const T none = narrow_to<T>((Wide<T>)-INFINITY);
  if (whole) {   // rows and lanes' parts start on boundaries, and a lane's part is the group's or not
    constexpr int V = EACH * (int)sizeof(T) <= 16 ? EACH : 16 / (int)sizeof(T);
#pragma unroll
    for (int r = 0; r < EACH; r += V) {
      Vec<T, V> a;
#pragma unroll
      for (int i = 0; i < V; ++i) a.v[i] = none;
      if (first < n) a = *reinterpret_cast<const Vec<T, V> *>(x + first + r);
#pragma unroll
      for (int i = 0; i < V; ++i) v[r + i] = a.v[i];
    }
  } else {
#pragma unroll
    for (int r = 0; r < EACH; ++r) v[r] = first + r < n ? x[first + r] : none;
  }
}

// The unit drawn of those that are kept, for a small random number.
template <typename T, int EACH>
__device__ __noinline__ int draw_small(const T *x, unsigned n, bool whole, double inv_t, double min_p, float random, const double *table,
                                       typename Keys<Wide<T>>::type top, typename Keys<Wide<T>>::type cut_key, unsigned cut_index) {
  using W = Wide<T>;
  using Key = typename Keys<W>::type;
  const unsigned lane = threadIdx.x & 31;
  const Weights weights(table, inv_t, kWarpBits);
  const W best = Keys<W>::value(top);
  const Cut<Key> cut{cut_key, cut_index, 0};
  T raw[EACH];
  load_units<T, EACH>(x, n, whole, raw);
  u64 total = 0, mass[EACH];
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    const W v = no_nan(widen(raw[r]));
    const bool in = kept(Keys<W>::of(v), lane * EACH + r, cut) && weights.reaches(v, best, min_p);
    if (!in) raw[r] = narrow_to<T>((W)-INFINITY);
    total += in ? weights.lifted(v, best, 0) : 0;
  }
  const Lift small(random, warp_sum_54(total), kWarpBits);
  total = 0;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    mass[r] = weights.lifted(no_nan(widen(raw[r])), best, small.lift);   // (0 at -infinity)
    total += mass[r];
  }
  const u64 up_to = warp_up_to(total);
  const unsigned who = __ffs(__ballot_sync(0xffffffffu, up_to > small.target)) - 1;
  u64 run = up_to - total;
  unsigned index = lane * EACH;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    run += mass[r];
    index += run <= small.target;
  }
  return (int)__shfl_sync(0xffffffffu, index, who);
}

// The unit drawn from one group, or -1; the same for all lanes.
template <typename T, int EACH>
__device__ __noinline__ int draw_exactly(const T *x, unsigned n, bool whole, const Settings &set, float random, const double *table,
                                         Few<typename Keys<Wide<T>>::type> &few) {
  using W = Wide<T>;
  using Key = typename Keys<W>::type;
  const unsigned lane = threadIdx.x & 31;
  T raw[EACH];
  W v[EACH];
  load_units<T, EACH>(x, n, whole, raw);
  WarpGroup<W, EACH> group;
  Key top = 0;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    v[r] = no_nan(widen(raw[r]));
    group.key[r] = Keys<W>::of(v[r]);
    top = max(top, group.key[r]);
  }
  top = warp_max(top);
  const W best = Keys<W>::value(top);
  if (!(best > (W)-INFINITY)) return -1;
  if (set.top_k == 1) {
    unsigned index = n;
#pragma unroll
    for (int r = EACH - 1; r >= 0; --r)
      if (group.key[r] == top) index = lane * EACH + r;
    return (int)warp_min(index);
  }
  const Weights weights(table, set.inv_t, kWarpBits);
#pragma unroll
  for (int r = 0; r < EACH; ++r) group.mass[r] = weights.of(v[r], best);
  Cut<Key> cut{0, n, 0};
  if (set.top_k < n) cut = group.cut(want_count(set.top_k), 0, top, few);
  if (set.top_p < 1) {
    if (set.top_k >= n) {
#pragma unroll
      for (int r = 0; r < EACH; ++r) cut.mass += group.mass[r];
      cut.mass = warp_sum_54(cut.mass);
    }
    // Units of at most 1/n of what may be left out are, all of them together, no more than that.
    const Want want = want_mass(set.top_p, cut.mass);
    cut = group.cut(want, want.limit > 0 && want.limit < cut.mass ? (cut.mass - want.limit) / n : 0, top, few);
  }
  if (is_small(random)) return draw_small<T, EACH>(x, n, whole, set.inv_t, set.min_p, random, table, top, cut.key, cut.index);
  if (set.min_p > 0) {
    const u64 least = (u64)__double2ll_rn(fmin(set.min_p, 1.0) * (double)weights.one());
#pragma unroll
    for (int r = 0; r < EACH; ++r)
      if (group.mass[r] < least) group.mass[r] = 0;
  }
  u64 total = 0;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    if (!kept(group.key[r], lane * EACH + r, cut)) group.mass[r] = 0;
    total += group.mass[r];
  }
  const u64 up_to = warp_up_to(total);
  const u64 target = target_of(random, __shfl_sync(0xffffffffu, up_to, 31));
  const unsigned who = __ffs(__ballot_sync(0xffffffffu, up_to > target)) - 1;
  u64 run = up_to - total;
  unsigned index = lane * EACH;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    run += group.mass[r];
    index += run <= target;
  }
  return (int)__shfl_sync(0xffffffffu, index, who);
}

// The same in 32 bits, with a bound on what that can be off: where a decision lies within the bound the draw is in doubt, and is
// made again in 64 bits.  With 100 units that is one draw in some thousands; the others cost a third of the instructions.
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ float warp_min(float v) { return -warp_max(-v); }
__device__ __forceinline__ float warp_sum(float v) {
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
struct FewFloats {
  float key[32], mass[32];
  unsigned index[32];
};

template <int EACH>
struct QuickGroup {
  float v[EACH], w[EACH];   // w = exp((v - best) / t), the largest 1
  float error;              // bound on a sum's
  bool doubt;

  __device__ __forceinline__ unsigned first() const { return (threadIdx.x & 31) * EACH; }
  __device__ __forceinline__ bool kept(int r, float value, unsigned index) const { return v[r] > value || (v[r] == value && first() + r <= index); }
  // value, index: the last unit kept; returns the mass up to it.  `limit`: by mass, else the first `count`.
  __device__ __forceinline__ float cut(bool by_count, unsigned count, float limit, float behind, float best, FewFloats &few, float &value, unsigned &index) {
    const unsigned lane = threadIdx.x & 31;
    auto inside = [&](unsigned c, float m) {
      if (by_count) return c < count;
      doubt = doubt || fabsf(m - limit) <= error;
      return m < limit;
    };
    float lo = INFINITY, hi = best, above = 0;
    unsigned to_lo = 0, above_count = 0;
#pragma unroll
    for (int r = 0; r < EACH; ++r)
      if (v[r] > -INFINITY && (by_count || w[r] > behind)) lo = fminf(lo, v[r]);
    lo = warp_min(lo);
#pragma unroll
    for (int r = 0; r < EACH; ++r) to_lo += v[r] >= lo;
    to_lo = __reduce_add_sync(0xffffffffu, to_lo);
    for (int round = 0; to_lo - above_count > 32 && !doubt; ++round) {
      const float pivot = 0.5f * lo + 0.5f * hi;
      unsigned c = 0;
      float m = 0;
#pragma unroll
      for (int r = 0; r < EACH; ++r)
        if (v[r] >= pivot) c += 1, m += w[r];
      c = __reduce_add_sync(0xffffffffu, c);
      if (!by_count) m = warp_sum(m);
      // (equal values, or values far from evenly spread, are left to the exact form)
      doubt = doubt || !(pivot > lo && pivot < hi) || round > 8;
      if (c < to_lo && inside(c, m)) {
        above_count = c;
        above = m;
        hi = pivot;   // units at the pivot itself have been counted
        hi = __uint_as_float(pivot > 0 ? __float_as_uint(pivot) - 1 : pivot < 0 ? __float_as_uint(pivot) + 1 : 0x80000001u);
      } else {
        to_lo = c;
        lo = pivot;
      }
    }
    if (doubt) return 0;
    const unsigned in = to_lo - above_count;
    unsigned c = 0;
#pragma unroll
    for (int q = 0; q < EACH; ++q) c += v[q] >= lo && v[q] <= hi;
    unsigned at = warp_up_to(c) - c;
#pragma unroll
    for (int q = 0; q < EACH; ++q)
      if (v[q] >= lo && v[q] <= hi) {
        few.key[at] = v[q];
        few.mass[at] = w[q];
        few.index[at] = first() + q;
        ++at;
      }
    if (lane >= in) few.key[lane] = -INFINITY;
    __syncwarp();
    const float k = few.key[lane], m = lane < in ? few.mass[lane] : 0;
    unsigned rank = __popc(__match_any_sync(0xffffffffu, k) & ((1u << lane) - 1));
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 o = *reinterpret_cast<const float4 *>(&few.key[j]);
      rank += o.x > k;
      rank += o.y > k;
      rank += o.z > k;
      rank += o.w > k;
    }
    __syncwarp();
    if (lane < in) few.mass[rank] = m;
    __syncwarp();
    const float by_rank = lane < in ? few.mass[lane] : 0, up_to = above + warp_up_to(by_rank), before = up_to - by_rank;
    // (the very first is kept by definition)
    const bool in_it = lane < in && (above_count + lane == 0 || inside(above_count + lane, before));
    const unsigned last = __popc(__ballot_sync(0xffffffffu, in_it)) - 1;
    const unsigned who = __ffs(__ballot_sync(0xffffffffu, lane < in && rank == last)) - 1;
    value = __shfl_sync(0xffffffffu, k, who);
    index = few.index[who & 31];
    const float mass = __shfl_sync(0xffffffffu, up_to, last & 31);
    doubt = __any_sync(0xffffffffu, doubt);
    __syncwarp();
    if (!by_count) return mass;
    float all = 0;
#pragma unroll
    for (int q = 0; q < EACH; ++q) all += kept(q, value, index) ? w[q] : 0;
    return warp_sum(all);
  }
};

// The unit, or -1; -2 in doubt.
template <int EACH>
__device__ __forceinline__ int draw_quickly(QuickGroup<EACH> &g, unsigned n, const Settings &set, float random, FewFloats &few) {
  const unsigned lane = threadIdx.x & 31;
  float best = -INFINITY;
#pragma unroll
  for (int r = 0; r < EACH; ++r) best = fmaxf(best, g.v[r]);
  best = warp_max(best);
  if (best == -INFINITY) return -1;
  if (set.top_k == 1) {
    unsigned index = n;
#pragma unroll
    for (int r = EACH - 1; r >= 0; --r)
      if (g.v[r] == best) index = lane * EACH + r;
    return (int)__reduce_min_sync(0xffffffffu, index);
  }
  const float c = (float)(set.inv_t * 1.4426950408889634);
  if (best == INFINITY || !(c > 1e-30f && c < 1e30f)) return -2;
  float total = 0;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(g.w[r]) : "f"((g.v[r] - best) * c));
    total += g.w[r];
  }
  // A weight is off by 2^-22 of it (ex2.approx) and by 3 x 2^-24 = 1.8e-7 for every unit x of its exponent: x exp(-x) is below 0.37, so
  // by less than 3.1e-7 of the largest weight, 1, and, where it counts at all (x < 40), by 7.5e-6 of itself.  Two sums of them are
  // compared.  Of their roundings, each 2^-24 of the sum of all at most:
  //   a border of the last step, the sum in front of the lane and its units one by one: EACH - 1 in every lane, 5 over the lanes, 1 for
  //   taking the lane's own out, EACH; against the random number's part of a sum: EACH - 1, 5, and 1 for the product;
  //   a mass at a cut: EACH - 1 and 5 up to a round's bound, 5 in the list, 1 for adding the two, 1 for taking out its own; against the
  //   limit: EACH - 1, 5, and 1 for the product.
  constexpr int kBorder = (EACH - 1) + 5 + 1 + EACH + (EACH - 1) + 5 + 1, kCut = (EACH - 1) + 5 + 5 + 1 + 1 + (EACH - 1) + 5 + 1;
  constexpr int kRoundings = kBorder > kCut ? kBorder : kCut;
  total = warp_sum(total);
  g.error = 2 * fminf(3.1e-7f * n, 7.5e-6f * total) + (kRoundings + 1) * 6e-8f * total;   // (one more for the bound's own; 2^-24 is 5.97e-8)
  g.doubt = false;
  float value = -INFINITY, mass = total;
  unsigned index = n;
  if (set.top_k < n) mass = g.cut(true, set.top_k, 0, 0, best, few, value, index);
  if (set.top_p < 1 && !g.doubt) {
    const float limit = (float)set.top_p * mass;
    // units of at most 1/n of what may be left out are, all of them together, no more than that
    const float behind = fmaxf(0.f, (mass - limit - 4 * g.error) / n);
    mass = g.cut(false, 0, limit, set.top_k < n ? 0 : behind, best, few, value, index);
  }
  if (g.doubt) return -2;
  if (set.min_p > 0) {
    const float least = fminf((float)set.min_p, 1.f);
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
      g.doubt = g.doubt || (fabsf(g.w[r] - least) <= 1e-5f * least && g.v[r] != best);
      if (g.w[r] < least && g.v[r] != best) g.w[r] = 0;
    }
  }
  float own = 0;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    if (!g.kept(r, value, index)) g.w[r] = 0;
    own += g.w[r];
  }
  const float up_to = warp_up_to(own), all = __shfl_sync(0xffffffffu, up_to, 31), target = random * all, error = g.error;
  // the borders of this lane's units, the one in front of them among these
  float run = up_to - own;
  bool doubt = g.doubt || !(random >= 0 && random < 1) || fabsf(run - target) <= error;
  unsigned unit = lane * EACH;
#pragma unroll
  for (int r = 0; r < EACH; ++r) {
    run += g.w[r];
    doubt = doubt || fabsf(run - target) <= error;
    unit += run <= target;
  }
  if (__any_sync(0xffffffffu, doubt)) return -2;
  const unsigned who = __ffs(__ballot_sync(0xffffffffu, up_to > target)) - 1;
  return (int)__shfl_sync(0xffffffffu, unit, who & 31);
}

// Instructions bound it: 122880 groups of 100 float32 units with a top-p of 0.9 87 us, 600 instructions a group, 80 % of the issue slots busy
// (no top-p 41 us, greedy 24).  All in registers, a warp needs no barrier; a block for a group of 520 took twice as long.
template <typename T, int EACH>
__global__ void __launch_bounds__(kWarpThreads, kWarpBlocks<EACH>)
    sample_warp_kernel(const T *__restrict__ support, const float *__restrict__ random, unsigned groups, unsigned H, unsigned n, bool whole,
                       const Sampling how, long long *__restrict__ codes) {
  after_previous();
  using W = Wide<T>;
  using Key = typename Keys<W>::type;
  constexpr bool QUICK = sizeof(W) == 4, AHEAD = QUICK && EACH <= 16;
  __shared__ double s_table[kTable];
  __shared__ Few<Key> s_few[kWarps];
  static_assert(sizeof(Few<Key>) >= sizeof(FewFloats), "one place for both");
  Weights::fill(s_table);
  __syncthreads();
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, step = gridDim.x * kWarps, rows = step / H, rest = step % H;
  const bool own = how.temperature_rows || how.top_k_rows || how.top_p_rows || how.min_p_rows;
  Settings set;
  if (!own) set = settings_of(how, 0, n);
  unsigned g = blockIdx.x * kWarps + warp, row = g / H, h = g % H;
  if (g >= groups) return;
  T next[EACH];   // the next group's units, under way
  if constexpr (AHEAD) load_units<T, EACH>(support + (long)g * n, n, whole, next);
  for (; g < groups; g += step, row += rows, h += rest) {
    if (h >= H) h -= H, row += 1;
    const T *const x = support + (long)g * n;
    if (own) set = settings_of(how, row, n);
    const float u = random[g];
    int unit = -2;
    if constexpr (QUICK) {
      QuickGroup<EACH> group;
      if constexpr (!AHEAD) load_units<T, EACH>(x, n, whole, next);
#pragma unroll
      for (int r = 0; r < EACH; ++r) group.v[r] = no_nan(widen(next[r])) + 0.f;   // (no -0)
      if (AHEAD && g + step < groups) load_units<T, EACH>(x + (long)step * n, n, whole, next);
      unit = draw_quickly(group, n, set, u, reinterpret_cast<FewFloats &>(s_few[warp]));
    }
    if (unit == -2) unit = draw_exactly<T, EACH>(x, n, whole, set, u, s_table, s_few[warp]);
    if (lane == 0) codes[g] = unit < 0 ? -1ll : (long long)h * n + unit;
    __syncwarp();
  }
}

// ---- a cluster per group ---------------------------------------------------

constexpr int kMostBlocks = 8;       // of a cluster
constexpr int kStage = 64 * 1024;    // bytes of a group that a block keeps in shared memory
// Threads of a block.  Where there are four groups for every SM, or they are short, small blocks with fewer and wider bins and a shorter
// list take groups of up to 8192 units.  A top-p over float32, large and small blocks, us a call: 16000 groups of 520, 947 and 239; of
// 8192, 4000 groups 345 and 306, 600 groups 66 and 64, but 160 groups 31 and 49.
constexpr int kLarge = 512, kSmall = 128;
constexpr unsigned kSmallMost = 8192;
template <int THREADS>
struct Shape {
  static constexpr int kThreads = THREADS, kBlockWarps = THREADS / 32;
  static constexpr int kPer = THREADS == kLarge ? 128 : 32;              // bins to one of the weights' exponent, 16 of these
  static constexpr int kBins = 16 * kPer, kBinsEach = kBins / THREADS;
  static constexpr int kList = THREADS;                                  // units that are ranked, a thread each
  static constexpr unsigned kQuickCount = THREADS / 2;                   // a top-k of up to this many goes by the threads' maxima
};

template <int THREADS>
struct Block : Shape<THREADS> {
  using Shape<THREADS>::kBins;
  using Shape<THREADS>::kList;
  using Shape<THREADS>::kBlockWarps;
  unsigned bin_count[kBins], bin_low[kBins], bin_high[kBins];   // masses in halves
  u64 list_key[kList];
  unsigned list_index[kList];
  u64 sorted_mass[kList];
  double table[kTable];
  u64 sum[kBlockWarps];
  u64 swap[2][2];     // what a block tells the others, in turn
  u64 unit;           // what one block finds for all
  u64 found[4];       // what the first block finds: a bin, the count and mass in front of it, the units in it; or a cut
  unsigned list;      // units in the list
  int bin;

  __device__ __forceinline__ u64 mass(int b) const { return ((u64)bin_high[b] << 32) + bin_low[b]; }
};

template <int THREADS>
__device__ __forceinline__ u64 block_sum(u64 v, u64 *s) {
  constexpr int kBlockWarps = THREADS / 32;
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kBlockWarps; ++i) v += s[i];
  return v;
}
template <int THREADS, typename Key>
__device__ __forceinline__ Key block_max(Key v, u64 *s) {
  constexpr int kBlockWarps = THREADS / 32;
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 m = 0;
#pragma unroll
  for (int i = 0; i < kBlockWarps; ++i) m = max(m, s[i]);
  return (Key)m;
}
// The sum over the threads in front, in order.
template <int THREADS>
__device__ __forceinline__ u64 block_before(u64 v, u64 *s) {
  constexpr int kBlockWarps = THREADS / 32;
  const u64 in = warp_up_to(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 31) s[threadIdx.x >> 5] = in;
  __syncthreads();
  u64 base = 0;
#pragma unroll
  for (int i = 0; i < kBlockWarps; ++i) base += i < (int)(threadIdx.x >> 5) ? s[i] : 0;
  return base + in - v;
}

// The part of a group that a block works on: units [begin, begin + size), as elements [lead, lead + size) of `vectors` vectors.
// Elements around them are -infinity: in shared memory, STAGED, they are there; else the first and the last vector are put
// together from the elements that exist.
template <typename T, bool STAGED, int THREADS>
struct Part : Shape<THREADS> {
  using Shape<THREADS>::kThreads;
  using Shape<THREADS>::kBlockWarps;
  using Shape<THREADS>::kPer;
  using Shape<THREADS>::kBins;
  using Shape<THREADS>::kBinsEach;
  using Shape<THREADS>::kList;
  using W = Wide<T>;
  using Key = typename Keys<W>::type;
  static constexpr int V = 16 / (int)sizeof(T);
  const Vec<T, V> *x;
  unsigned begin, size, lead, vectors;
  W best;
  Block<THREADS> &s;
  cg::cluster_group cluster;
  int turn;

  __device__ __forceinline__ Part(const Vec<T, V> *x_, unsigned begin_, unsigned size_, unsigned lead_, unsigned vectors_, Block<THREADS> &s_,
                                  cg::cluster_group cluster_)
      : x(x_), begin(begin_), size(size_), lead(lead_), vectors(vectors_), best(0), s(s_), cluster(cluster_), turn(0) {}
  __device__ __forceinline__ u64 block_sum(u64 v, u64 *sum) const { return sbb::block_sum<THREADS>(v, sum); }
  __device__ __forceinline__ u64 block_before(u64 v, u64 *sum) const { return sbb::block_before<THREADS>(v, sum); }

  // whole vectors: [first_whole(), end_whole())
  __device__ __forceinline__ unsigned first_whole() const { return STAGED || lead == 0 ? 0 : 1; }
  __device__ __forceinline__ unsigned end_whole() const { return STAGED ? vectors : (lead + size) / V; }
  __device__ __forceinline__ Vec<T, V> load(unsigned i) const {
    if (i >= first_whole() && i < end_whole()) return x[i];
    Vec<T, V> a;
    const T *const element = reinterpret_cast<const T *>(x);
#pragma unroll
    for (int v = 0; v < V; ++v) a.v[v] = i * V + v >= lead && i * V + v < lead + size ? element[i * V + v] : narrow_to<T>((W)-INFINITY);
    return a;
  }
  // f(vector, its number) for vectors lo, lo + step, ... below hi, in rising order; U in flight, their loads without conditions among
  // them.  A first and a last vector that are not whole are put together by themselves.
  template <int U, typename F>
  __device__ __forceinline__ void range(unsigned lo, unsigned hi, unsigned step, F f) const {
    unsigned i = lo;
    if (!STAGED && i < first_whole() && i < hi) {
      f(load(i), i);
      i += step;
    }
    const unsigned end = min(hi, end_whole());
    for (; i < end; i += U * step) {
      Vec<T, V> a[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * step < end) a[u] = x[i + u * step];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * step < end) f(a[u], i + u * step);
    }
    if constexpr (!STAGED) {
      const unsigned last = end_whole();
      if (last < hi && last >= first_whole() && last >= lo && (last - lo) % step == 0) f(load(last), last);
    }
  }
  // f(value, unit) for the units above -infinity (no NaN is) of a vector
  template <typename F>
  __device__ __forceinline__ void units(const Vec<T, V> &a, unsigned i, F f) const {
    W w[V];
    widen_all(a, w);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (w[v] > (W)-INFINITY) f(w[v], begin + i * V + v - lead);
  }
  // ... of all vectors
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    range<1>(threadIdx.x, vectors, kThreads, [&](const Vec<T, V> &a, unsigned i) { units(a, i, f); });
  }
  // The same for units of at least `low`, which most vectors have none of: marked in a word first, so that there is one copy of f's
  // code (32 of them, for the vectors in flight, did not stay in the instruction cache: 39 us a pass over 128000 units, 12 so).
  template <typename F>
  __device__ __forceinline__ void range_from(W low, unsigned lo, unsigned hi, unsigned step, F f) const {
    constexpr int U = 32 / V < 4 ? 32 / V : 4;
    const T *const element = reinterpret_cast<const T *>(x);
    auto marks = [&](const Vec<T, V> &a) {
      unsigned m = 0;
      if (max_all(a) >= low)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const W w = widen(a.v[v]);
          m |= (w >= low && w > (W)-INFINITY ? 1u : 0u) << v;
        }
      return m;
    };
    auto run = [&](unsigned m, unsigned i) {
      for (; m != 0; m &= m - 1) {
        const unsigned bit = __ffs(m) - 1, at = (i + bit / V * step) * V + bit % V;
        f((W)widen(element[at]), begin + at - lead);
      }
    };
    const unsigned first = first_whole(), end = min(hi, end_whole()), last = end_whole();
    unsigned i = lo, edge = 0, at = 0;
    if (!STAGED && i < first && i < hi) {
      edge = marks(load(i)), at = i;
      i += step;
    } else if (!STAGED && last < hi && last >= first && last >= lo && (last - lo) % step == 0) {
      edge = marks(load(last)), at = last;
    }
    if constexpr (!STAGED) run(edge, at);
    if (!STAGED && lo < first && lo < hi && last < hi && last >= first && (last - lo) % step == 0) run(marks(load(last)), last);   // (both ends)
    for (; i < end; i += U * step) {
      Vec<T, V> a[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * step < end) a[u] = x[i + u * step];
      unsigned m = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * step < end) m |= marks(a[u]) << (u * V);
      run(m, i);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each_from(W low, F f) const {
    range_from(low, threadIdx.x, vectors, kThreads, f);
  }

  // f(a, b) of every block's two values, in the blocks' order.
  // (Two places in turn: one is written again only behind another exchange's barrier.)
  template <typename F>
  __device__ __forceinline__ void exchange(u64 a, u64 b, F f) {
    if (cluster.num_blocks() == 1) {
      f(a, b);
      return;
    }
    if (threadIdx.x == 0) s.swap[turn][0] = a, s.swap[turn][1] = b;
    cluster.sync();
    for (unsigned o = 0; o < cluster.num_blocks(); ++o) {
      const Block<THREADS> *const other = cluster.map_shared_rank(&s, o);
      f(other->swap[turn][0], other->swap[turn][1]);
    }
    turn ^= 1;
  }
  __device__ __forceinline__ u64 cluster_sum(u64 v) {   // of a value of each block
    u64 all = 0;
    exchange(v, 0, [&](u64 a, u64) { all += a; });
    return all;
  }

  // The first unit at which the running sum of weigh(value, unit) passes target(sum of all), which is below that sum; known to every
  // block when all have passed a barrier of the cluster.
  // Units below `low` weigh nothing.
  template <typename F, typename G>
  __device__ void locate(W low, F weigh, G target) {
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned lo = 0, hi = vectors;
    auto by_warp = [&](u64 &all) {   // sums of the warps' shares of vectors [lo, hi)
      const unsigned share = (hi - lo + kBlockWarps - 1) / kBlockWarps, from = min(hi, lo + warp * share);
      u64 mine = 0;
      if (low > (W)-INFINITY)
        range_from(low, from + lane, min(hi, from + share), 32, [&](W v, unsigned i) { mine += weigh(v, i); });
      else
        range<1>(from + lane, min(hi, from + share), 32, [&](const Vec<T, V> &a, unsigned i) { units(a, i, [&](W v, unsigned j) { mine += weigh(v, j); }); });
      mine = warp_sum(mine);
      __syncthreads();
      if (lane == 0) s.sum[warp] = mine;
      __syncthreads();
      all = 0;
#pragma unroll
      for (int w = 0; w < kBlockWarps; ++w) all += s.sum[w];
      return share;
    };
    u64 all;
    unsigned share = by_warp(all);
    u64 total = 0, before = 0;
    unsigned o = 0;
    exchange(all, 0, [&](u64 a, u64) {
      if (o++ < cluster.block_rank()) before += a;
      total += a;
    });
    const u64 at = target(total);
    if (at < before || at >= before + all) return;
    for (;;) {   // the share that it lies in
      unsigned w = 0;
      while (before + s.sum[w] <= at) before += s.sum[w++];
      lo = min(hi, lo + w * share);
      hi = min(hi, lo + share);
      if (hi - lo <= kThreads) break;
      share = by_warp(all);
    }
    u64 mine = 0;
    const unsigned i = lo + threadIdx.x;
    if (i < hi) units(load(i), i, [&](W v, unsigned j) { mine += weigh(v, j); });
    u64 run = before + block_before(mine, s.sum);
    if (run <= at && at < run + mine) {
      bool found = false;
      units(load(i), i, [&](W v, unsigned j) {
        run += weigh(v, j);
        if (!found && run > at) {
          found = true;
          for (unsigned b = 0; b < cluster.num_blocks(); ++b) cluster.map_shared_rank(&s, b)->unit = j;
        }
      });
    }
  }

  // Fills the bins: bin_of(value) in [0, kBins) or -1, masses where `masses` is set; the first block gets the sums of all.  Returns
  // this thread's sum of the masses of all units, `total` asked for.
  // Masses are added in halves with a carry: an addition of 64 bits to shared memory is a loop, and where values are equal
  // (16-bit types) a long one: 256 rows of 128000 bf16 units, a few of them without a top-k, 1030 us (560 so).
  template <typename F>
  __device__ u64 histogram(F bin_of, bool masses, bool total, const Weights &weights) {
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.bin_count[b] = 0, s.bin_low[b] = 0, s.bin_high[b] = 0;
    __syncthreads();
    u64 all = 0;
    each([&](W v, unsigned) {
      const int b = bin_of(v);
      u64 m = 0;
      if (total || (masses && b >= 0)) m = weights.of(v, best);
      all += m;
      if (b < 0) return;
      atomicAdd(&s.bin_count[b], 1u);
      if (!masses || m == 0) return;
      const unsigned low = (unsigned)m, old = atomicAdd(&s.bin_low[b], low), high = (unsigned)(m >> 32) + (old + low < low);
      if (high) atomicAdd(&s.bin_high[b], high);
    });
    cluster.sync();
    if (cluster.block_rank() == 0 && cluster.num_blocks() > 1)
      for (int b = threadIdx.x; b < kBins; b += kThreads) {
        unsigned c = s.bin_count[b];
        u64 m = s.mass(b);
        for (unsigned o = 1; o < cluster.num_blocks(); ++o) {
          const Block<THREADS> *const other = cluster.map_shared_rank(&s, o);
          c += other->bin_count[b];
          if (masses) m += other->mass(b);
        }
        s.bin_count[b] = c;
        s.bin_low[b] = (unsigned)m;
        s.bin_high[b] = (unsigned)(m >> 32);
      }
    __syncthreads();
    return all;
  }
  struct Found {
    int bin;
    unsigned in_bin, above_count;
    u64 above_mass;
  };
  // The last bin that begins inside, from the first block's sums; known to every block.
  __device__ Found find(const Want &want, unsigned above_count, u64 above_mass) {
    if (cluster.block_rank() == 0) {
      if (threadIdx.x == 0) s.bin = 0;
      u64 c = 0, m = 0;
#pragma unroll
      for (int j = 0; j < kBinsEach; ++j) {
        c += s.bin_count[threadIdx.x * kBinsEach + j];
        m += s.mass(threadIdx.x * kBinsEach + j);
      }
      const u64 c0 = above_count + block_before(c, s.sum), m0 = above_mass + block_before(m, s.sum);
      u64 cb = c0, mb = m0;
#pragma unroll
      for (int j = 0; j < kBinsEach; ++j) {
        const int b = threadIdx.x * kBinsEach + j;
        if (s.bin_count[b] && want.inside((unsigned)cb, mb)) atomicMax(&s.bin, b);
        cb += s.bin_count[b];
        mb += s.mass(b);
      }
      __syncthreads();
      const int bin = s.bin;
      if (bin / kBinsEach == (int)threadIdx.x) {
        cb = c0, mb = m0;
        for (int b = threadIdx.x * kBinsEach; b < bin; ++b) cb += s.bin_count[b], mb += s.mass(b);
        const u64 in = s.bin_count[bin];
        for (unsigned o = 0; o < cluster.num_blocks(); ++o) {
          u64 *const to = cluster.map_shared_rank(&s, o)->found;
          to[0] = bin;
          to[1] = cb;
          to[2] = mb;
          to[3] = in;
        }
      }
    }
    cluster.sync();
    const Found f{(int)s.found[0], (unsigned)s.found[3], (unsigned)s.found[1], s.found[2]};
    return f;
  }
  // Puts a unit into the first block's list while there is room; s.list there counts all.  (It is 0 at first; the first block sets it
  // back to 0 ahead of a barrier of the cluster.)
  __device__ __forceinline__ void put(W v, unsigned unit) {
    Block<THREADS> *const first = cluster.num_blocks() == 1 ? &s : cluster.map_shared_rank(&s, 0);
    const unsigned at = atomicAdd(&first->list, 1u);
    if (at >= kList) return;
    // (of 32-bit keys, one number in the order of the units)
    first->list_key[at] = sizeof(Key) == 4 ? (u64)Keys<W>::of(v) << 32 | ~unit : (u64)Keys<W>::of(v);
    first->list_index[at] = unit;
  }
  // How many of the first `count` numbers of a list are above (below) one's own: four a step.
  template <bool ABOVE, typename N>
  __device__ __forceinline__ unsigned count_of(const N *list, unsigned count, N own, unsigned &equal) const {
    constexpr int E = 16 / (int)sizeof(N);
    unsigned c = 0, e = 0;
#pragma unroll 4
    for (unsigned j = 0; j < count; j += E) {
      const Vec<N, E> o = reinterpret_cast<const Vec<N, E> *>(list)[j / E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (j + i < count) {
          c += ABOVE ? o.v[i] > own : o.v[i] < own;
          e += o.v[i] == own;
        }
      }
    }
    equal = e;
    return c;
  }
  // The first block's list: a thread's entry, its rank in the order and what lies in front of it.
  struct Ranked {
    Key key;
    unsigned index, rank;
    u64 mass, before;
  };
  __device__ Ranked rank(unsigned count, const Weights &weights) {
    Ranked r{};
    r.rank = kList;
    if (threadIdx.x < count) {
      const u64 own = s.list_key[threadIdx.x];
      r.key = (Key)(sizeof(Key) == 4 ? own >> 32 : own);
      r.index = s.list_index[threadIdx.x];
      r.mass = weights.of(Keys<W>::value(r.key), best);
      unsigned equal;
      r.rank = count_of<true>(s.list_key, count, own, equal);
      if (equal > 1)   // (of 64-bit keys alone)
        for (unsigned j = 0; j < count; ++j) r.rank += s.list_key[j] == own && s.list_index[j] < r.index;
      s.sorted_mass[r.rank] = r.mass;
    }
    r.before = sum_in_front(count, r.rank);
    return r;
  }
  // Of s.sorted_mass[0 .. count), the sum in front of entry `at`.
  __device__ __forceinline__ u64 sum_in_front(unsigned count, unsigned at) {
    __syncthreads();
    const u64 before = block_before(threadIdx.x < count ? s.sorted_mass[threadIdx.x] : 0, s.sum);
    __syncthreads();
    if (threadIdx.x < count) s.sorted_mass[threadIdx.x] = before;
    __syncthreads();
    return threadIdx.x < count ? s.sorted_mass[at] : 0;
  }
  // The unit drawn from the first block's list, which holds all that may be kept; by that block alone.  `total`: the mass of all
  // units, where there is no top-k.
  __device__ void draw(unsigned count, const Settings &set, unsigned n, u64 total, u64 least, const Weights &weights, float random, long long base,
                       long long *code) {
    const Ranked r = rank(count, weights);
    bool keep = threadIdx.x < count;
    if (set.top_k < n) {
      keep = keep && r.rank < set.top_k;
      if (set.top_p < 1) total = block_sum(keep ? r.mass : 0, s.sum);
    }
    if (set.top_p < 1) keep = keep && want_mass(set.top_p, total).inside(r.rank, r.before);
    keep = keep && r.mass >= least;   // (the largest have 2^q, which is no less)
    u64 mass = keep ? r.mass : 0, target = block_sum(mass, s.sum);
    if (is_small(random)) {
      const W v = Keys<W>::value(r.key);
      keep = keep && weights.reaches(v, best, set.min_p);
      const Lift small(random, block_sum(keep ? r.mass : 0, s.sum), weights.q);
      mass = keep ? weights.lifted(v, best, small.lift) : 0;
      target = small.target;
    } else {
      target = target_of(random, target);
    }
    unsigned equal, at = 0;
    if (threadIdx.x < count) {
      at = count_of<false>(s.list_index, count, r.index, equal);
      s.sorted_mass[at] = mass;
    }
    const u64 before = sum_in_front(count, at);
    if (mass > 0 && before <= target && target < before + mass) *code = base + r.index;
  }

  // The cut of a top-p by sums in 32 bits with a bound on what they can be off, or false: exact sums have to decide.  Only the units
  // above the cut have their weights formed in 64 bits; in the exact form, which adds masses to bins, all have.
  // A weight e^-x is off by 2^-22 of it and 3 x 2^-24 for every unit of x; over n weights of sum S the mean of x, by weight, is at
  // most ln n (where all are equal); a sum of eight is off by 7 x 2^-24 more.  So S is off by S (1.8e-7 ln n + 7e-7) at most.
  template <typename F>
  __device__ bool cut_quickly(F bin_of, const Settings &set, unsigned n, const Weights &weights, Cut<Key> &cut) {
    constexpr double kOne = 1099511627776.0;   // 2^40: 32-bit weights are summed in fixed point, up to 2^22 of them
    const float c = (float)(set.inv_t * 1.4426950408889634);
    if (best == INFINITY || !(c > 1e-30f && c < 1e30f) || !(set.top_p > 0) || n > 1u << 22) return false;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.bin_count[b] = 0;
    __syncthreads();
    double sum = 0;
    range<STAGED ? 1 : 4>(threadIdx.x, vectors, kThreads, [&](const Vec<T, V> &a, unsigned) {
      float w[V], eight = 0;
      widen_all(a, w);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        w[v] = fmaxf(w[v], -3.4e38f);   // (-infinity or a NaN: weighs nothing)
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((w[v] - (float)best) * c));
        eight += e;
      }
      sum += eight;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int b = bin_of(w[v]);
        if (b < kBins - 1) atomicAdd(&s.bin_count[b], 1u);
      }
    });
    const u64 total = cluster_sum(block_sum(__double2ull_rn(sum * kOne), s.sum));   // (with the barriers that the bins need)
    const double error = (double)total * (1.9e-7 * log((double)n) + 8e-7) * (1 + set.top_p) + 1024;
    const double limit = set.top_p * (double)total;
    if (cluster.block_rank() == 0) {
      if (threadIdx.x == 0) s.found[0] = kBins, s.found[1] = kBins;
      unsigned count[kBinsEach];
      double low = 0, high = 0;   // bounds on the bins' masses: a unit of bin b weighs e^-(b +- 1/2)/kPer
      constexpr double kUp = kPer == 128 ? 1.0041 : 1.0161, kDown = kPer == 128 ? 0.9959 : 0.9842;   // (e^1/256 is 1.0039, e^1/64 1.0158)
#pragma unroll
      for (int j = 0; j < kBinsEach; ++j) {
        const int b = threadIdx.x * kBinsEach + j;
        count[j] = s.bin_count[b];
        for (unsigned o = 1; o < cluster.num_blocks(); ++o) count[j] += cluster.map_shared_rank(&s, o)->bin_count[b];
        s.bin_count[b] = count[j];
        const double w = kOne * count[j] * (double)__expf(-b * (1.f / kPer));
        high += w * kUp;
        low += w * kDown;
      }
      double high_up_to = (double)block_before((u64)high, s.sum), low_up_to = (double)block_before((u64)low, s.sum);
      __syncthreads();   // s.found is there
#pragma unroll
      for (int j = 0; j < kBinsEach; ++j) {
        const int b = threadIdx.x * kBinsEach + j;
        const double w = kOne * count[j] * (double)__expf(-b * (1.f / kPer));
        high_up_to += w * kUp + 1;
        low_up_to += w * kDown;
        if (high_up_to + kThreads >= limit - error) atomicMin(&s.found[0], (u64)b);
        if (low_up_to >= limit + error) atomicMin(&s.found[1], (u64)b);
      }
      __syncthreads();
      const int first = (int)s.found[0], last = (int)s.found[1];
      unsigned in = 0, above = 0;
#pragma unroll
      for (int j = 0; j < kBinsEach; ++j) {
        const int b = threadIdx.x * kBinsEach + j;
        if (b < first) above += count[j];
        if (b >= first && b <= last) in += count[j];
      }
      const u64 both = block_sum((u64)above << 32 | in, s.sum);
      if (threadIdx.x == 0)
        for (unsigned o = 0; o < cluster.num_blocks(); ++o) {
          u64 *const to = cluster.map_shared_rank(&s, o)->found;
          to[0] = first;
          to[1] = last >= kBins - 1 ? kList + 1 : (unsigned)both;
          to[2] = last;
          to[3] = both >> 32;
        }
    }
    cluster.sync();
    const int first = (int)s.found[0], last = (int)s.found[2];
    const unsigned in = (unsigned)s.found[1], above_count = (unsigned)s.found[3];
    if (in > kList) return false;
    u64 above = 0;
    const W low = best - (W)((last + 2) / (kPer * set.inv_t));   // no unit of the bins lies below
    each_from(low, [&](W v, unsigned i) {
      const int b = bin_of(v);
      if (b > last) return;
      if (b < first)
        above += weights.of(v, best);
      else
        put(v, i);
    });
    above = cluster_sum(block_sum(above, s.sum));   // (one block: its barriers are between the list's entries and their reader)
    Ranked r{};
    if (cluster.block_rank() == 0) {
      r = rank(in, weights);
      if (threadIdx.x == 0) s.list = 0;
    }
    // Decided by the sum in 32 bits, and again by the exact one where a unit lies within the bound of the limit (a few rows of a
    // hundred).
    const double scale = (double)weights.one() / kOne;   // the masses' unit
    Want want{false, 0, (u64)(limit * scale)};
    double off = error * scale;
    for (;;) {
      if (cluster.block_rank() == 0) {
        const u64 before = above + r.before;
        const bool here = threadIdx.x < in, keep = here && want.inside(above_count + r.rank, before);
        const bool doubt = here && above_count + r.rank > 0 && fabs((double)before - (double)want.limit) <= off;
        const u64 n_kept = block_sum(keep, s.sum);
        const bool again = __syncthreads_or(doubt) || n_kept == 0;
        if (again ? threadIdx.x == 0 : keep && r.rank + 1 == n_kept)
          for (unsigned o = 0; o < cluster.num_blocks(); ++o) {
            u64 *const to = cluster.map_shared_rank(&s, o)->found;
            to[0] = again ? 0 : (u64)r.key;
            to[1] = r.index;
          }
      }
      cluster.sync();
      if (s.found[0] != 0) break;   // (no unit's key)
      if (off < 0) return false;
      u64 exact = 0;
      each([&](W v, unsigned) { exact += weights.of(v, best); });
      want = want_mass(set.top_p, cluster_sum(block_sum(exact, s.sum)));
      off = -1;
    }
    cut = Cut<Key>{(Key)s.found[0], (unsigned)s.found[1], 0};
    return true;
  }

  // The cut that `want` asks for among all units: bins of equal width in the value's distance from the largest first (`found`, by
  // linear_bin), then, while a bin holds too many for the list, bins of its values' bits.
  template <typename F>
  __device__ Cut<Key> cut(const Want &want, Found found, F linear_bin, const Weights &weights) {
    Key lo = 0, hi = ~(Key)0;
    unsigned above_count = found.above_count, in = found.in_bin;
    u64 above_mass = found.above_mass;
    const int bin = found.bin;
    auto among = [&](W v) {
      const Key k = Keys<W>::of(v);
      return linear_bin(v) == bin && k >= lo && k <= hi;
    };
    while (in > kList && lo < hi) {
      Key low = ~(Key)0, high = 0;
      each([&](W v, unsigned) {
        if (among(v)) {
          const Key k = Keys<W>::of(v);
          low = min(low, k);
          high = max(high, k);
        }
      });
      const Key high_here = block_max<THREADS>(high, s.sum), low_here = block_max<THREADS>((Key)~low, s.sum);
      high = 0, low = 0;
      exchange(high_here, low_here, [&](u64 a, u64 b) { high = max(high, (Key)a), low = max(low, (Key)b); });
      lo = (Key)~low, hi = high;
      if (lo == hi) break;
      int shift = 0;
      while (((hi - lo) >> shift) >= (Key)kBins) ++shift;
      histogram([&](W v) { return among(v) ? (int)((hi - Keys<W>::of(v)) >> shift) : -1; }, !want.by_count, false, weights);
      const Found f = find(want, above_count, above_mass);
      above_count = f.above_count;
      above_mass = f.above_mass;
      in = f.in_bin;
      const Key width = (Key)1 << shift, top = hi - (Key)f.bin * width;
      if (top - lo >= width) lo = top - (width - 1);
      hi = top;
    }
    if (in > kList) {   // equal values
      const u64 m = weights.of(Keys<W>::value(hi), best);
      const unsigned take = equal_ones(want, in, m, above_count, above_mass);
      const Key key = hi;
      locate(Keys<W>::value(key), [&](W v, unsigned) { return (u64)(Keys<W>::of(v) == key); }, [&](u64) { return (u64)(take - 1); });
      cluster.sync();
      return Cut<Key>{key, (unsigned)s.unit, above_mass + take * m};
    }
    cluster.sync();   // (the list is empty)
    each([&](W v, unsigned i) {
      if (among(v)) put(v, i);
    });
    cluster.sync();
    if (cluster.block_rank() == 0) {
      const unsigned count = s.list;
      const Ranked r = rank(count, weights);
      const bool keep = threadIdx.x < count && want.inside(above_count + r.rank, above_mass + r.before);
      const u64 n_kept = block_sum(keep, s.sum);
      if (threadIdx.x == 0) s.list = 0;
      if (keep && r.rank + 1 == n_kept)
        for (unsigned o = 0; o < cluster.num_blocks(); ++o) {
          u64 *const to = cluster.map_shared_rank(&s, o)->found;
          to[0] = r.key;
          to[1] = r.index;
          to[2] = above_mass + r.before + r.mass;
        }
    }
    cluster.sync();
    return Cut<Key>{(Key)s.found[0], (unsigned)s.found[1], s.found[2]};
  }
};

// Few groups are bound by latency, the barriers of a block and its cluster: one of 32000 float16 units, top-k 50 and top-p 0.9, 12 us.
// Many by instructions on every unit: 256 x 128000 bf16 with a top-k of 100 33 us (greedy 14, the support at the copy bandwidth 10), with
// settings of each row, some without a top-k, 113.
template <typename T, bool STAGED, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
    sample_block_kernel(const T *__restrict__ support, const float *__restrict__ random, unsigned H, unsigned n, unsigned part, const Sampling how,
                        int q, long long *__restrict__ codes) {
  after_previous();
  using W = Wide<T>;
  using Key = typename Keys<W>::type;
  using P = Part<T, STAGED, THREADS>;
  constexpr int V = P::V, kThreads = THREADS, kBins = P::kBins, kList = P::kList;
  extern __shared__ uint4 s_values[];
  __shared__ Block<THREADS> s;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned blocks = cluster.num_blocks(), g = blockIdx.x / blocks, rank = cluster.block_rank();
  const unsigned begin = min(n, rank * part), size = min(part, n - begin);
  const T *const from = support + (long)g * n + begin;
  const Settings set = settings_of(how, g / H, n);
  Weights::fill(s.table);
  if (threadIdx.x == 0) s.list = 0;
  // vectors begin on 16-byte boundaries of memory, in shared memory too
  const unsigned lead = (unsigned)(reinterpret_cast<uintptr_t>(from) & 15) / (unsigned)sizeof(T), vectors = size ? (lead + size + V - 1) / V : 0;
  const Vec<T, V> *const memory = reinterpret_cast<const Vec<T, V> *>(from - lead);
  W mine = -INFINITY;   // the largest of the values that pass through this thread, and the first vector that has it
  unsigned where = 0;
  Part<T, false, THREADS>(memory, begin, size, lead, vectors, s, cluster).template range<STAGED ? 4 : 8>(threadIdx.x, vectors, kThreads, [&](const Vec<T, V> &a, unsigned i) {
    if constexpr (STAGED) reinterpret_cast<Vec<T, V> *>(s_values)[i] = a;
    const W m = max_all(a);
    if (m > mine) mine = m, where = i;
  });
  P p(STAGED ? reinterpret_cast<const Vec<T, V> *>(s_values) : memory, begin, size, lead, vectors, s, cluster);
  const Key own = Keys<W>::of(mine);
  Key top = block_max<THREADS>(own, s.sum), low = 0;
  const bool by_count = set.top_k < n, quick = by_count && set.top_k > 1 && set.top_k <= P::kQuickCount;
  if (quick) {
    // A value that at least this block's share of the k units reach: the share's largest of the threads' maxima, in its first bits.
    const unsigned share = (set.top_k + blocks - 1) / blocks;
    constexpr int kLow = (int)sizeof(Key) * 8 - 32;
    const unsigned bits = (unsigned)(own >> kLow);
    unsigned reached = 0;
    constexpr int kBits = sizeof(T) == 2 ? 16 : 20;   // (those of a 16-bit element)
    for (int b = 31; b > 31 - kBits; --b)
      if (__syncthreads_count(bits >= (reached | 1u << b)) >= (int)share) reached |= 1u << b;
    low = (Key)reached << kLow;
  }
  {
    Key best = 0, lowest = ~(Key)0;
    p.exchange(top, low, [&](u64 a, u64 b) { best = max(best, (Key)a), lowest = min(lowest, (Key)b); });
    top = best, low = lowest;
  }
  const W best = p.best = Keys<W>::value(top);
  if (!(best > (W)-INFINITY)) {
    if (rank == 0 && threadIdx.x == 0) codes[g] = -1;
    cluster.sync();   // (a block's place is there while others read it)
    return;
  }
  const long long base = (long long)(g % H) * n;
  const Weights weights(s.table, set.inv_t, q);
  const u64 least = set.min_p > 0 ? (u64)__double2ll_rn(fmin(set.min_p, 1.0) * (double)weights.one()) : 0;
  if (quick) {
    const W from_here = low > Keys<W>::of((W)-INFINITY) ? Keys<W>::value(low) : (W)-INFINITY;
    p.each_from(from_here, [&](W v, unsigned i) { p.put(v, i); });
    cluster.sync();
    const unsigned count = cluster.map_shared_rank(&s, 0)->list;
    cluster.sync();
    if (count <= kList) {
      if (rank == 0) p.draw(count, set, n, 0, least, weights, random[g], base, codes + g);
      return;
    }
    if (rank == 0 && threadIdx.x == 0) s.list = 0;   // (values that lie unevenly over the threads, or many equal ones)
  }
  if (set.top_k == 1) {   // the first of the largest; vectors that lie behind one another in a thread lie so in the group
    u64 last = 0;
    if (mine == best) {
      unsigned unit = ~0u;
      p.units(p.load(where), where, [&](W v, unsigned i) {
        if (v == best) unit = min(unit, i);
      });
      last = ~unit;
    }
    last = block_max<THREADS>(last, s.sum);
    u64 of_all = 0;
    p.exchange(last, 0, [&](u64 a, u64) { of_all = max(of_all, a); });
    if (rank == 0 && threadIdx.x == 0) codes[g] = base + (long long)(unsigned)~of_all;
    cluster.sync();
    return;
  }
  Cut<Key> cut{0, n, 0};
  {
    if (by_count || set.top_p < 1) {
      // bins of 1/128 (1/32) in the weights' exponents, to the nearest; all units whose weight is below e^-16 share the last one
      const W scale = (W)(P::kPer * set.inv_t);
      auto bin = [&](W v) -> int {
        const W d = v == best ? (W)0 : fmin((best - v) * scale, (W)(kBins - 1));
        return sizeof(W) == 4 ? (int)(__float_as_uint((float)d + 8388608.f) & (kBins - 1)) : (int)rint(d);   // (2^23: rounds to an integer)
      };
      bool quick_p = false;
      if constexpr (sizeof(W) == 4) quick_p = !by_count && p.cut_quickly(bin, set, n, weights, cut);
      if (!quick_p) {
        u64 total = p.histogram(bin, !by_count, !by_count, weights);
        if (!by_count) total = p.cluster_sum(p.block_sum(total, s.sum));
        Want want = by_count ? want_count(set.top_k) : want_mass(set.top_p, total);
        const auto found = p.find(want, 0, 0);
        if (!by_count && found.above_count + found.in_bin <= kList) {
          // all that may be kept fits the list: the first block goes on by itself
          p.each([&](W v, unsigned i) {
            if (bin(v) <= found.bin) p.put(v, i);
          });
          cluster.sync();
          if (rank == 0) p.draw(s.list, set, n, total, least, weights, random[g], base, codes + g);
          return;
        }
        cut = p.cut(want, found, bin, weights);
        if (by_count && set.top_p < 1) {
          u64 sum = 0;
          p.each([&](W v, unsigned i) {
            if (kept(Keys<W>::of(v), i, cut)) sum += weights.of(v, best);
          });
          want = want_mass(set.top_p, p.cluster_sum(p.block_sum(sum, s.sum)));
          p.histogram(bin, true, false, weights);
          cut = p.cut(want, p.find(want, 0, 0), bin, weights);
        }
      }
    }
    const W value = cut.key ? Keys<W>::value(cut.key) : (W)-INFINITY;
    p.locate(
        value,
        [&](W v, unsigned i) -> u64 {
          if (!(v > value || (v == value && i <= cut.index))) return 0;
          const u64 m = weights.of(v, best);
          return m >= least ? m : 0;
        },
        [&](u64 total) {
          if (!is_small(random[g])) return target_of(random[g], total);
          s.sorted_mass[0] = total;   // (the same from every thread)
          return ~0ull;
        });
    // A small random number's: from the front, by the first block alone.  (Most are found in the first units.)
    if (rank == 0 && is_small(random[g])) {
      __syncthreads();
      const Lift small(random[g], s.sorted_mass[0], q);
      const T *const group = support + (long)g * n;
      u64 before = 0;
#pragma unroll 1
      for (unsigned i0 = 0; i0 < n; i0 += kThreads) {   // (the largest passes what is looked for)
        const unsigned i = i0 + threadIdx.x;
        const W v = i < n ? no_nan(widen(group[i])) : (W)-INFINITY;
        const bool in = (v > value || (v == value && i <= cut.index)) && weights.reaches(v, best, min_p_of(how, g / H));
        const u64 m = in ? weights.lifted(v, best, small.lift) : 0, run = before + p.block_before(m, s.sum);
        if (run <= small.target && small.target < run + m) s.unit = i;
        for (int w = 0; w < P::kBlockWarps; ++w) before += s.sum[w];   // (the warps' sums, from block_before)
        if (before > small.target) break;
      }
    }
  }
  cluster.sync();
  if (rank == 0 && threadIdx.x == 0) codes[g] = base + (long long)s.unit;
}

// 2^q: no sum of n masses passes 2^62.
int mass_bits(long n) {
  int q = 50;
  while (q > 20 && (double)n * (double)(1ull << q) >= 4.6e18) --q;
  return q;
}

template <typename T, int EACH>
cudaError_t launch_warps(const T *support, const float *random, unsigned groups, unsigned H, unsigned n, const Sampling &s, long long *codes,
                         cudaStream_t st) {
  constexpr size_t piece = EACH * sizeof(T) < 16 ? EACH * sizeof(T) : 16;
  const bool whole = n % EACH == 0 && (reinterpret_cast<uintptr_t>(support) | n * sizeof(T)) % piece == 0;
  const unsigned most = 2 * kWarpBlocks<EACH> * (unsigned)sm_count(), blocks = (groups + kWarps - 1) / kWarps;
  return launch_next(sample_warp_kernel<T, EACH>, dim3(blocks < most ? blocks : most), kWarpThreads, 0, st, support, random, groups, H, n, whole, s,
                     codes);
}

template <typename T, bool STAGED, int THREADS>
cudaError_t launch_blocks(const T *support, const float *random, unsigned groups, unsigned H, unsigned n, unsigned part, unsigned cluster,
                          const Sampling &s, long long *codes, cudaStream_t st) {
  const size_t smem = STAGED ? (size_t)part * sizeof(T) + 16 : 0;   // (a vector more where the part begins inside one)
  if (smem > 0) {   // (holds for the current device)
    const cudaError_t e = cudaFuncSetAttribute(sample_block_kernel<T, STAGED, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStage + 16);
    if (e != cudaSuccess) return e;
  }
  return launch_clusters(sample_block_kernel<T, STAGED, THREADS>, dim3(groups * cluster), dim3(cluster), THREADS, smem, st, support, random, H, n, part, s,
                         mass_bits(n), codes);
}

}  // namespace

template <typename T>
cudaError_t launch_sample(const T *support, const float *random, long rows, long H, long Mc, Sampling s, long long *codes, cudaStream_t st) {
  const unsigned groups = (unsigned)(rows * H), n = (unsigned)Mc, h = (unsigned)H;
  s.inv_t = inverse(s.temperature);
  cudaError_t e;
  if (n <= 32) {
    e = launch_warps<T, 1>(support, random, groups, h, n, s, codes, st);
  } else if (n <= 64) {
    e = launch_warps<T, 2>(support, random, groups, h, n, s, codes, st);
  } else if (n <= 128) {
    e = launch_warps<T, 4>(support, random, groups, h, n, s, codes, st);
  } else if (n <= 256) {
    e = launch_warps<T, 8>(support, random, groups, h, n, s, codes, st);
  } else if (n <= 512) {
    e = launch_warps<T, 16>(support, random, groups, h, n, s, codes, st);
  } else if (n <= 1024 && sizeof(Wide<T>) == 4) {
    // (16000 groups of 520 float32 units: a top-p 98 us here and 239 in small blocks, a top-k of 20 90 and 107; of float64, 193 and 193,
    // 202 and 115)
    if constexpr (sizeof(Wide<T>) == 4) e = launch_warps<T, 32>(support, random, groups, h, n, s, codes, st);
  } else {
    // With a group for every SM, a block each, which reads its group again where it has to (it is in L2 by then).  Fewer: the smallest
    // cluster whose blocks hold their parts in shared memory, and a larger one while there are SMs and parts are long.
    const size_t bytes = (size_t)n * sizeof(T);
    unsigned cluster = 1;
    const bool alone = groups >= (unsigned)sm_count();
    // Where every row has its own top-k, some may have none and take several times as long: two blocks share a row if all fit side by
    // side.  256 x 128000 bf16, us a call: 157 with one, 112 with two; with one top-k of 100 for all 33 and 46.
    if (alone && n > kSmallMost && s.top_k_rows && groups < 2 * (unsigned)sm_count()) cluster = 2;
    if (!alone) {
      while (cluster < kMostBlocks && bytes > (size_t)cluster * kStage) cluster *= 2;
      while (cluster < kMostBlocks && (size_t)groups * cluster * 2 <= (size_t)sm_count() && n / cluster > 2048) cluster *= 2;
    }
    constexpr unsigned V = 16 / (unsigned)sizeof(T);
    const unsigned part = ((n + cluster - 1) / cluster + V - 1) / V * V;
    if ((size_t)groups * cluster > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const bool staged = !alone && (size_t)part * sizeof(T) <= kStage;
    if (alone && n <= kSmallMost && (n <= 2048 || groups >= 4 * (unsigned)sm_count())) {
      e = launch_blocks<T, false, kSmall>(support, random, groups, h, n, part, cluster, s, codes, st);
    } else {
      e = staged ? launch_blocks<T, true, kLarge>(support, random, groups, h, n, part, cluster, s, codes, st)
                 : launch_blocks<T, false, kLarge>(support, random, groups, h, n, part, cluster, s, codes, st);
    }
  }
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace sbb
