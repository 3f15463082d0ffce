// Support of coded samples and its gradient: sums of the weight rows that codes name, and sums of the gradient's rows by code.
#include "sbb_codes.cuh"
#include "sbb_launch.cuh"

namespace sbb {
namespace {

constexpr int kThreads = 256;

// `lanes` threads take V columns each of a row's tile; `parts` such groups of a block split the row's codes and the parts are added in
// order; the block's other groups take other rows or tiles.  Codes are read eight at a time, so that as many weight rows are in
// flight, and the next eight while these are.
template <typename T, typename I, int V>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(const T *__restrict__ weights, const I *__restrict__ codes, long rows, long L, long N, long M, Wide<T> scale, T *__restrict__ out,
                  int lanes, int parts, unsigned tiles) {
  after_previous();
  using W = Wide<T>;
  extern __shared__ unsigned char s_raw[];
  W *const s_part = reinterpret_cast<W *>(s_raw);   // [threads][V], where parts > 1
  const int group = threadIdx.x / lanes, part = group % parts;
  const long item = (long)blockIdx.x * (kThreads / (lanes * parts)) + group / parts, r = item / tiles;
  const long col = (item % tiles * lanes + threadIdx.x % lanes) * V;
  const bool here = r < rows && col < M;
  W acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = (W)0;
  if (here) {
    constexpr int U = 8;
    const I *const code = codes + r * L;
    const T *const from = weights + col;
    I c[U];
    auto read = [&](long l) {
#pragma unroll
      for (int u = 0; u < U; ++u) c[u] = l + u * parts < L ? code[l + u * parts] : (I)-1;
    };
    read(part);
    for (long l = part; l < L; l += U * parts) {
      Vec<T, V> x[U];
      bool named[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        named[u] = c[u] >= 0 && (long)c[u] < N;
        if (named[u]) x[u] = *reinterpret_cast<const Vec<T, V> *>(from + (long)c[u] * M);
      }
      if (l + U * parts < L) read(l + U * parts);
      // the eight among themselves first: a chain of L additions loses digits that one of L / 8 keeps
      W eight[V];
#pragma unroll
      for (int v = 0; v < V; ++v) eight[v] = (W)0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (named[u]) {
          W f[V];
          widen_all(x[u], f);
#pragma unroll
          for (int v = 0; v < V; ++v) eight[v] += f[v];
        }
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += eight[v];
    }
  }
  if (parts > 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) s_part[threadIdx.x * V + v] = acc[v];
    __syncthreads();
    if (part != 0) return;
    for (int p = 1; p < parts; ++p)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += s_part[(p * lanes + threadIdx.x) * V + v];
  }
  if (!here) return;
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] *= scale;
  *reinterpret_cast<Vec<T, V> *>(out + r * M + col) = narrow_all<T, V>(acc);
}

// One code a row: copies of weight rows, U under way per thread.  A block takes whole pieces of kThreads * U vectors of the result.
template <typename T, typename I, int V, int U>
__global__ void __launch_bounds__(kThreads)
    lookup_one_kernel(const T *__restrict__ weights, const I *__restrict__ codes, long rows, long N, long M, Wide<T> scale, T *__restrict__ out,
                      unsigned across) {
  after_previous();
  using W = Wide<T>;
  const long first = (long)blockIdx.x * (kThreads * U), row0 = first / across;
  const unsigned at0 = (unsigned)(first - row0 * across) + threadIdx.x;   // (the one division of 64 bits)
  Vec<T, V> x[U];
  unsigned r[U], col[U];
  I c[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned at = at0 + u * kThreads;
    r[u] = at / across;
    col[u] = (at - r[u] * across) * V;
    c[u] = row0 + r[u] < rows ? codes[row0 + r[u]] : (I)-1;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (c[u] >= 0 && (long)c[u] < N) {
      x[u] = *reinterpret_cast<const Vec<T, V> *>(weights + (long)c[u] * M + col[u]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) x[u].v[v] = narrow_to<T>((W)0);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row0 + r[u] >= rows) continue;
    W f[V];
    widen_all(x[u], f);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] *= scale;
    *reinterpret_cast<Vec<T, V> *>(out + (row0 + r[u]) * M + col[u]) = narrow_all<T, V>(f);
  }
}

template <typename T, typename I, int V>
cudaError_t launch_lookup_as(const T *weights, const I *codes, long rows, long L, long N, long M, double scale, T *out, cudaStream_t st) {
  const long across = M / V;
  if (L == 1) {
    constexpr int U = V == 1 ? 8 : 4;
    const long blocks = (rows * across + kThreads * U - 1) / (kThreads * U);
    if (blocks > 0x7fffffffl) return cudaErrorInvalidConfiguration;
    return launch_next(lookup_one_kernel<T, I, V, U>, dim3((unsigned)blocks), kThreads, 0, st, weights, codes, rows, N, M, (Wide<T>)scale, out,
                       (unsigned)across);
  }
  // Few rows of many codes: narrow tiles (of a line of 128 bytes and more) and the codes split until the SMs have work, four codes or
  // more a part.
  const long want = 1024l * sm_count();
  int lanes = 1;
  while (lanes < 32 && lanes < across) lanes *= 2;
  while (lanes > 8 && rows * across * (L / 16) < want && rows * ((across + lanes - 1) / lanes) < 2 * sm_count()) lanes /= 2;
  int parts = 1;
  while (parts * lanes < kThreads && parts * 8 <= L && rows * across * parts < want) parts *= 2;
  const long tiles = (across + lanes - 1) / lanes, each = kThreads / (lanes * parts), blocks = (rows * tiles + each - 1) / each;
  if (blocks > 0x7fffffffl) return cudaErrorInvalidConfiguration;
  const size_t smem = parts > 1 ? kThreads * V * sizeof(Wide<T>) : 0;
  return launch_next(lookup_kernel<T, I, V>, dim3((unsigned)blocks), kThreads, smem, st, weights, codes, rows, L, N, M, (Wide<T>)scale, out, lanes, parts,
                     (unsigned)tiles);
}

// ---- gradient --------------------------------------------------------------
//
// The codes are sorted (stably, so that the sums of a weight row run in the order of the samples whatever the schedule), and
// then every weight row is the sum of a run of the gradient's rows.  Runs may be of any length, so the sorted entries are cut
// into equal chunks: a chunk writes the runs that lie in it and leaves the part of a run that crosses its border in the
// workspace, from where join_kernel adds the parts in order.

constexpr unsigned kRankMost = 8192;   // entries that are ranked by comparing all with all

__device__ __forceinline__ unsigned key_of(long code, long N) { return code >= 0 && code < N ? (unsigned)code : (unsigned)N; }

// a < b for numbers of up to 2^31 (the difference's sign: an instruction less than a comparison and a choice)
__device__ __forceinline__ unsigned below(unsigned a, unsigned b) { return (a - b) >> 31; }

// Sorted position of an entry = the entries with a smaller key + those with the same key in front.  A warp takes four entries;
// one launch where a radix sort is four.
template <typename I>
__global__ void __launch_bounds__(kThreads)
    rank_kernel(const I *__restrict__ codes, unsigned entries, unsigned L, long N, unsigned *__restrict__ key, unsigned *__restrict__ row,
                unsigned *__restrict__ some) {
  after_previous();
  __shared__ uint4 s_key[kRankMost / 4];
  unsigned *const s = reinterpret_cast<unsigned *>(s_key);
  const unsigned padded = (entries + 3) & ~3u;
  for (unsigned i0 = threadIdx.x; i0 < padded; i0 += 8 * kThreads) {   // (eight loads in flight: one by one the 30 KB took 8 us)
    long c[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) c[u] = i0 + u * kThreads < entries ? (long)codes[i0 + u * kThreads] : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u * kThreads < padded) s[i0 + u * kThreads] = i0 + u * kThreads < entries ? key_of(c[u], N) : 0x7fffffffu;
  }
  __syncthreads();
  const unsigned lane = threadIdx.x & 31, e0 = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * 4;
  if (e0 >= entries) return;
  const uint4 own = s_key[e0 / 4];
  const unsigned k[4] = {own.x, own.y, own.z, own.w};
  unsigned n[4] = {0, 0, 0, 0};
  for (unsigned j = lane; j < e0 / 4; j += 32) {
    const uint4 o = s_key[j];
#pragma unroll
    for (int q = 0; q < 4; ++q) n[q] += below(o.x, k[q] + 1) + below(o.y, k[q] + 1) + below(o.z, k[q] + 1) + below(o.w, k[q] + 1);
  }
  for (unsigned j = e0 / 4 + 1 + lane; j < padded / 4; j += 32) {
    const uint4 o = s_key[j];
#pragma unroll
    for (int q = 0; q < 4; ++q) n[q] += below(o.x, k[q]) + below(o.y, k[q]) + below(o.z, k[q]) + below(o.w, k[q]);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    unsigned r = __reduce_add_sync(0xffffffffu, n[q]);
#pragma unroll
    for (int o = 0; o < 4; ++o) r += o < q ? k[o] <= k[q] : k[o] < k[q];
    if (lane == 0 && e0 + q < entries) {
      key[r] = k[q];
      row[r] = (e0 + q) / L;
      if (some != nullptr && k[q] < (unsigned)N) some[k[q]] = r;
    }
  }
}

// A pass of a radix sort, least significant digit first: counts of the digits of every tile of entries ...
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kDigitBits = 9, kDigits = 1 << kDigitBits;

template <typename I, bool FIRST>
__device__ __forceinline__ unsigned sort_key(const I *codes, const unsigned *key, unsigned i, long N) {
  return FIRST ? key_of((long)codes[i], N) : key[i];
}

template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
    digits_kernel(const I *__restrict__ codes, const unsigned *__restrict__ key, unsigned entries, long N, int shift, unsigned tile,
                  unsigned *__restrict__ counts) {
  after_previous();
  __shared__ unsigned s_count[kDigits];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) s_count[d] = 0;
  __syncthreads();
  const unsigned lo = blockIdx.x * tile, hi = min(entries, lo + tile);
  for (unsigned i = lo + threadIdx.x; i < hi; i += kSortThreads)
    atomicAdd(&s_count[(sort_key<I, FIRST>(codes, key, i, N) >> shift) & (kDigits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) counts[blockIdx.x * kDigits + d] = s_count[d];
}

// ... and the move: an entry goes behind all smaller digits, the same digit in tiles in front, in the tile's warps in front, and
// in its own warp in front.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
    move_kernel(const I *__restrict__ codes, const unsigned *__restrict__ key, const unsigned *__restrict__ row, unsigned entries, unsigned L, long N,
                int shift, unsigned tile, const unsigned *__restrict__ counts, unsigned *__restrict__ key_to, unsigned *__restrict__ row_to,
                unsigned *__restrict__ some) {
  after_previous();
  static_assert(kDigits == kSortThreads, "a thread per digit");
  __shared__ unsigned s_at[kSortWarps][kDigits];
  __shared__ unsigned s_warp[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&s_at[0][0])[i] = 0;
  __syncthreads();
  const unsigned each = tile / kSortWarps, lo = blockIdx.x * tile + warp * each, hi = min(entries, lo + each);   // (tile: a multiple of 512)
  for (unsigned i = lo + lane; i < hi; i += 32) atomicAdd(&s_at[warp][(sort_key<I, FIRST>(codes, key, i, N) >> shift) & (kDigits - 1)], 1u);
  unsigned all = 0, before = 0;
#pragma unroll 16
  for (unsigned b = 0; b < gridDim.x; ++b) {
    const unsigned c = counts[b * kDigits + threadIdx.x];
    all += c;
    before += b < blockIdx.x ? c : 0;
  }
  unsigned in = all;
  for (int off = 1; off < 32; off *= 2) {
    const unsigned o = __shfl_up_sync(0xffffffffu, in, off);
    if (lane >= off) in += o;
  }
  if (lane == 31) s_warp[warp] = in;
  __syncthreads();
  unsigned at = before + in - all;
  for (int w = 0; w < warp; ++w) at += s_warp[w];
  for (int w = 0; w < kSortWarps; ++w) {
    const unsigned c = s_at[w][threadIdx.x];
    s_at[w][threadIdx.x] = at;
    at += c;
  }
  __syncthreads();
  for (unsigned i0 = lo; i0 < hi; i0 += 32) {
    const bool there = i0 + lane < hi;
    const unsigned kk = there ? sort_key<I, FIRST>(codes, key, i0 + lane, N) : 0;
    const unsigned digit = there ? (kk >> shift) & (kDigits - 1) : kDigits;
    const unsigned same = __match_any_sync(0xffffffffu, digit);
    if (there) {
      const unsigned to = s_at[warp][digit] + __popc(same & ((1u << lane) - 1));
      key_to[to] = kk;
      row_to[to] = FIRST ? (i0 + lane) / L : row[i0 + lane];
      if (some != nullptr && kk < (unsigned)N) some[kk] = to;
    }
    __syncwarp();
    if (there && (same >> lane) == 1u) s_at[warp][digit] += __popc(same);   // the last of its kind
    __syncwarp();
  }
}

template <typename T, int V>
struct Sums {
  const T *grad;
  const unsigned *key, *row;   // sorted
  const unsigned *some;        // per weight row: the position of a code that names it, or anything where none does
  unsigned entries, chunk;
  long N, M;
  Wide<T> scale;
  bool accumulate;
  T *out;
  Wide<T> *partial;   // [chunk][run from the chunk before, run into the next][M]
  int lanes;
  unsigned tiles;     // of `lanes` vectors
  int zero_rows;      // of a block

  using W = Wide<T>;
  __device__ __forceinline__ void write(unsigned i, long col, const W (&acc)[V]) const {
    T *const to = out + (long)i * M + col;
    Vec<T, V> o;
    if (accumulate) o = *reinterpret_cast<const Vec<T, V> *>(to);
#pragma unroll
    for (int v = 0; v < V; ++v) o.v[v] = narrow_to<T>(accumulate ? acc[v] * scale + widen(o.v[v]) : acc[v] * scale);
    *reinterpret_cast<Vec<T, V> *>(to) = o;
  }
  __device__ __forceinline__ W *part(unsigned c, int which, long col) const { return partial + (2l * c + which) * M + col; }
};

constexpr int kZeroRows = 128;   // most rows of a block that sets rows to zero

// `lanes` threads take a chunk and a tile of columns.  Among the `sum_blocks` blocks that do so lie `zero_blocks` that set rows
// without a code to zero, evenly, so that memory is read and written at the same time.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 4) sums_kernel(const Sums<T, V> p, unsigned sum_blocks, unsigned zero_blocks) {
  after_previous();
  using W = Wide<T>;
  const unsigned zero_before = (unsigned)((unsigned long long)blockIdx.x * zero_blocks / gridDim.x);
  if ((unsigned)((unsigned long long)(blockIdx.x + 1) * zero_blocks / gridDim.x) != zero_before) {
    __shared__ bool s_absent[kZeroRows];
    const long n0 = (long)zero_before * p.zero_rows;
    const int rows = (int)min((long)p.zero_rows, p.N - n0);
    if ((int)threadIdx.x < rows) {
      const unsigned n = (unsigned)n0 + threadIdx.x, at = p.some[n];   // (nothing has written it where no code names the row)
      s_absent[threadIdx.x] = at >= p.entries || p.key[at] != n;
    }
    __syncthreads();
    Vec<T, V> zero;
#pragma unroll
    for (int v = 0; v < V; ++v) zero.v[v] = narrow_to<T>((W)0);
    const unsigned across = (unsigned)(p.M / V);
    unsigned r = threadIdx.x / across, c = threadIdx.x % across;
    const unsigned dr = kThreads / across, dc = kThreads % across;
    while ((int)r < rows) {
      if (s_absent[r]) *reinterpret_cast<Vec<T, V> *>(p.out + (n0 + r) * p.M + (long)c * V) = zero;
      r += dr;
      c += dc;
      if (c >= across) c -= across, ++r;
    }
    return;
  }
  // the block's sorted entries, with one more at either end
  extern __shared__ unsigned s_entry[];
  const unsigned groups = kThreads / p.lanes, g0 = (blockIdx.x - zero_before) * groups, g = g0 + threadIdx.x / p.lanes, c = g / p.tiles;
  const unsigned first = g0 / p.tiles * p.chunk, end = min(p.entries, ((g0 + groups - 1) / p.tiles + 1) * p.chunk), size = end > first ? end - first : 0;
  unsigned *const s_key = s_entry + 1, *const s_row = s_entry + size + 2;
  for (unsigned i = threadIdx.x; i < size + 2; i += kThreads) {
    const unsigned at = first + i - 1;   // (wraps below zero)
    s_entry[i] = at < p.entries ? p.key[at] : ~0u;
  }
  for (unsigned i = threadIdx.x; i < size; i += kThreads) s_row[i] = p.row[first + i];
  __syncthreads();
  const long col = ((long)(g % p.tiles) * p.lanes + threadIdx.x % p.lanes) * V;
  const unsigned b = c * p.chunk, e = min(p.entries, b + p.chunk);
  if (b >= p.entries || col >= p.M) return;
  W acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = (W)0;
  const unsigned *key = s_key + (b - first), *row = s_row + (b - first);
  unsigned n = e - b;
  while (n > 0 && key[n - 1] >= (unsigned)p.N) --n;   // codes that name nothing are the last ones
  if (n == 0) return;
  unsigned cur = key[0];
  bool head = s_entry[b - first] == cur;
  auto flush = [&](int which) {   // 2: the run lies in the chunk
    if (which == 2) {
      p.write(cur, col, acc);
    } else {
      W *const to = p.part(c, which, col);
#pragma unroll
      for (int v = 0; v < V; ++v) to[v] = acc[v];
    }
  };
  // Four loads without conditions in flight, four blocks on an SM.  65536 rows of 1024 bf16 elements, us a call: with conditions
  // between the loads 117, eight loads and three blocks 78, two pairs of four in turn 79 to 90 (registers), this 79.
  constexpr int U = 4;
  const T *const from = p.grad + col;
  for (unsigned i = 0; i < n; i += U) {
    Vec<T, V> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const Vec<T, V> *>(from + (long)row[min(i + u, n - 1)] * p.M);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= n) break;
      const unsigned k = key[i + u];
      if (k != cur) {
        flush(head ? 0 : 2);
        cur = k;
        head = false;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = (W)0;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += widen(x[u].v[v]);
    }
  }
  flush(head ? 0 : key[n] == cur ? 1 : 2);
}

// Adds the parts of the runs that cross the end of a chunk and begin in it: a group of `lanes` threads for each chunk and tile
// of columns, all groups of the block together for runs of many parts (of which a block, with chunks that follow one another,
// has few).
constexpr unsigned kLongRun = 32;
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) join_kernel(const Sums<T, V> p) {
  after_previous();
  using W = Wide<T>;
  __shared__ unsigned s_last[kThreads / 4];   // of each group's run, 0: none or short
  __shared__ W s_sum[kThreads * V];
  const unsigned groups = kThreads / p.lanes, own = threadIdx.x / p.lanes, lane = threadIdx.x % p.lanes;
  const unsigned chunks = (p.entries + p.chunk - 1) / p.chunk;
  auto sum = [&](W(&acc)[V], unsigned from, unsigned to, unsigned step, long col) {   // parts [from, to], four in flight
    for (; from <= to; from += 4 * step) {
      Vec<W, V> x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (from + u * step <= to) x[u] = *reinterpret_cast<const Vec<W, V> *>(p.part(from + u * step, 0, col));
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (from + u * step <= to)
#pragma unroll
          for (int v = 0; v < V; ++v) acc[v] += x[u].v[v];
    }
  };
  const unsigned blocks = (chunks + groups - 1) / groups, c0 = blockIdx.x % blocks * groups, c = c0 + own;
  const long col = ((long)(blockIdx.x / blocks) * p.lanes + lane) * V;
  unsigned cur = 0, last = 0;
  if (c + 1 < chunks) {
    const unsigned b = c * p.chunk, e = b + p.chunk;
    cur = p.key[e - 1];
    if (p.key[e] == cur && cur < (unsigned)p.N && !(b > 0 && p.key[b] == cur && p.key[b - 1] == cur)) {
      // the last chunk that begins inside the run: the group's threads try that many places at a time
      last = c + 1;
      unsigned end = chunks;
      const unsigned mask = (p.lanes == 32 ? ~0u : (1u << p.lanes) - 1) << (threadIdx.x & 31 & ~(p.lanes - 1));
      for (unsigned step = 1; last + 1 < end; step = (end - last - 1 + p.lanes - 1) / p.lanes) {   // first the chunks that follow
        const unsigned at = last + (lane + 1) * step;
        const int in = __popc(__ballot_sync(mask, at < end && p.key[at * p.chunk] == cur));
        last += in * step;
        if (in < p.lanes) end = min(end, last + step);
      }
    }
  }
  if (lane == 0) s_last[own] = last > c + kLongRun ? last : 0;
  W acc[V];
  if (last > 0 && col < p.M) {
    const W *const from = p.part(c, 1, col);
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = from[v];
    if (last <= c + kLongRun) {
      sum(acc, c + 1, last, 1, col);
      p.write(cur, col, acc);
    }
  }
  __syncthreads();
  for (unsigned q = 0; q < groups; ++q) {
    const unsigned to = s_last[q];
    if (to == 0) continue;
    W part[V];
#pragma unroll
    for (int v = 0; v < V; ++v) part[v] = (W)0;
    if (col < p.M) sum(part, c0 + q + 1 + own, to, groups, col);
#pragma unroll
    for (int v = 0; v < V; ++v) s_sum[threadIdx.x * V + v] = part[v];
    __syncthreads();
    if (own == q && col < p.M) {
      for (unsigned o = 0; o < groups; ++o)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += s_sum[(o * p.lanes + lane) * V + v];
      p.write(cur, col, acc);
    }
    __syncthreads();
  }
}

// Sizes of a gradient call.
struct GradientPlan {
  unsigned entries, chunk, chunks;
  bool rank;
  unsigned tile, blocks;   // of the sort's passes
  int passes;
  size_t padded, counts, some, partial;   // elements: a key or row array, the digits' counts, a position per row, the parts of runs
};
GradientPlan gradient_plan(long rows, long L, long N, long M) {
  GradientPlan p = {};
  p.entries = (unsigned)(rows * L);
  p.rank = p.entries <= kRankMost;
  // as many chunks as keep all threads busy with a vector of 16 bytes each, of 8 to 64 entries
  const long want = 2048l * sm_count() * 4;
  long chunk = (long)p.entries * M / want / 8 * 8;
  chunk = chunk < 8 ? 8 : chunk > 64 ? 64 : chunk;
  p.chunk = (unsigned)chunk;
  p.chunks = (p.entries + p.chunk - 1) / p.chunk;
  p.padded = ((size_t)p.entries + 7) / 8 * 8;
  p.some = ((size_t)N + 7) / 8 * 8;
  p.partial = p.chunks > 1 ? 2 * (size_t)p.chunks * (size_t)M : 0;
  if (!p.rank) {
    int bits = 1;
    while (bits < 32 && (N >> bits) != 0) ++bits;   // N stands for codes that name nothing
    p.passes = (bits + kDigitBits - 1) / kDigitBits;
    // up to 128 tiles: every block of a pass reads the counts of all
    p.tile = ((p.entries + 127) / 128 + kSortThreads - 1) / kSortThreads * kSortThreads;
    if (p.tile < 1024) p.tile = 1024;
    p.blocks = (p.entries + p.tile - 1) / p.tile;
    p.counts = (size_t)p.blocks * kDigits;
  }
  return p;
}

template <typename T, int V>
cudaError_t launch_sums(Sums<T, V> p, unsigned chunks, cudaStream_t st) {
  const long across = p.M / V;
  p.lanes = 4;
  while (p.lanes < 32 && p.lanes < across) p.lanes *= 2;
  p.tiles = (unsigned)((across + p.lanes - 1) / p.lanes);
  const unsigned per = kThreads / p.lanes;
  const long zero_rows = 32768 / (p.M * (long)sizeof(T));   // 32 KB a block
  p.zero_rows = (int)(zero_rows < 1 ? 1 : zero_rows > kZeroRows ? kZeroRows : zero_rows);
  const size_t blocks = ((size_t)chunks * p.tiles + per - 1) / per, zero = p.accumulate ? 0 : ((size_t)p.N + p.zero_rows - 1) / p.zero_rows;
  if (blocks + zero > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const size_t smem = (2 * ((per + p.tiles - 1) / p.tiles + 1) * (size_t)p.chunk + 2) * sizeof(unsigned);
  cudaError_t e = launch_next(sums_kernel<T, V>, dim3((unsigned)(blocks + zero)), kThreads, smem, st, p, (unsigned)blocks, (unsigned)zero);
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (chunks == 1) return e;
  const size_t join = (((size_t)chunks + per - 1) / per) * p.tiles;
  e = launch_next(join_kernel<T, V>, dim3((unsigned)join), kThreads, 0, st, p);
  if (e == cudaSuccess) count_launches(1);
  return e;
}

}  // namespace

template <typename T, typename I>
cudaError_t launch_lookup(const T *weights, const I *codes, long rows, long L, long N, long M, double scale, T *out, cudaStream_t st) {
  const int vec = vector_width<T>(M, weights, out);
  cudaError_t e;
  if (vec == 16 / (int)sizeof(T)) {
    e = launch_lookup_as<T, I, 16 / (int)sizeof(T)>(weights, codes, rows, L, N, M, scale, out, st);
  } else {
    if constexpr (sizeof(T) == 2)
      e = vec == 2 ? launch_lookup_as<T, I, 2>(weights, codes, rows, L, N, M, scale, out, st)
                   : launch_lookup_as<T, I, 1>(weights, codes, rows, L, N, M, scale, out, st);
    else
      e = launch_lookup_as<T, I, 1>(weights, codes, rows, L, N, M, scale, out, st);
  }
  if (e == cudaSuccess) count_launches(1);
  return e;
}

size_t lookup_gradient_workspace(long rows, long L, long N, long M, size_t wide) {
  const GradientPlan p = gradient_plan(rows, L, N, M);
  return ((p.rank ? 2 : 4) * p.padded + p.counts + p.some) * sizeof(unsigned) + 64 + p.partial * wide;
}

template <typename T, typename I>
cudaError_t launch_lookup_gradient(const T *grad, const I *codes, long rows, long L, long N, long M, double scale, bool accumulate, T *out,
                                   void *workspace, cudaStream_t st) {
  const GradientPlan p = gradient_plan(rows, L, N, M);
  unsigned *key = static_cast<unsigned *>(workspace), *row = key + p.padded, *const some = accumulate ? nullptr : row + p.padded, *end = row + p.padded + p.some;
  cudaError_t e;
  if (p.rank) {
    e = launch_next(rank_kernel<I>, dim3((p.entries + kThreads / 8 - 1) / (kThreads / 8)), kThreads, 0, st, codes, p.entries, (unsigned)L, N, key, row, some);
    if (e != cudaSuccess) return e;
    count_launches(1);
  } else {
    unsigned *key2 = end, *row2 = key2 + p.padded, *counts = row2 + p.padded;
    end = counts + p.counts;
    for (int pass = 0; pass < p.passes; ++pass) {
      const int shift = pass * kDigitBits;
      const bool first = pass == 0;
      unsigned *const last = pass + 1 == p.passes ? some : nullptr;
      e = first ? launch_next(digits_kernel<I, true>, dim3(p.blocks), kSortThreads, 0, st, codes, key, p.entries, N, shift, p.tile, counts)
                : launch_next(digits_kernel<I, false>, dim3(p.blocks), kSortThreads, 0, st, codes, key, p.entries, N, shift, p.tile, counts);
      if (e != cudaSuccess) return e;
      e = first ? launch_next(move_kernel<I, true>, dim3(p.blocks), kSortThreads, 0, st, codes, key, row, p.entries, (unsigned)L, N, shift, p.tile,
                              counts, key2, row2, last)
                : launch_next(move_kernel<I, false>, dim3(p.blocks), kSortThreads, 0, st, codes, key, row, p.entries, (unsigned)L, N, shift, p.tile,
                              counts, key2, row2, last);
      if (e != cudaSuccess) return e;
      count_launches(2);
      unsigned *const k = key, *const r = row;
      key = key2, row = row2, key2 = k, row2 = r;
    }
  }
  Wide<T> *const partial = reinterpret_cast<Wide<T> *>((reinterpret_cast<uintptr_t>(end) + 63) / 64 * 64);   // (read 32 bytes at a time)
  const int vec = vector_width<T>(M, grad, out);
  const Wide<T> s = (Wide<T>)scale;
  constexpr int V = 16 / (int)sizeof(T);
  if (vec == V) return launch_sums(Sums<T, V>{grad, key, row, some, p.entries, p.chunk, N, M, s, accumulate, out, partial, 0, 0}, p.chunks, st);
  if constexpr (sizeof(T) == 2)
    if (vec == 2) return launch_sums(Sums<T, 2>{grad, key, row, some, p.entries, p.chunk, N, M, s, accumulate, out, partial, 0, 0}, p.chunks, st);
  return launch_sums(Sums<T, 1>{grad, key, row, some, p.entries, p.chunk, N, M, s, accumulate, out, partial, 0, 0}, p.chunks, st);
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
