// Support of coded samples and its gradient: sums of the weight rows that codes name, and sums of the gradient's rows by code.
#include "sbb_codes.cuh"
#include "sbb_launch.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace sbb {
namespace {

constexpr int kThreads = 256;

// `lanes` threads take V columns each of a row's tile; `parts` such groups of a block split the row's codes and the parts are added in
// order; the block's other groups take other rows or tiles.  Codes are read eight at a time, so that as many weight rows are in
// flight, and the next eight while these are.  Bytes of the weight rows bound it: 4096 x 30 codes of 3000 x 1000 float32 51 us, 9.6 TB/s
// (mostly out of L2); 784 codes of one row of 3000 float32 4.6 us, two trips to memory behind one another and the join of the parts.
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
// Memory bounds it: 16384 codes of 50000 x 1024 bf16 8.2 us, 0.86 of a plain copy's bandwidth.
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
// into equal chunks and these joined to spans: a block writes the runs that lie in its span and leaves the part of a run that
// crosses the span's border in the workspace, from where join_kernel adds the parts in order.

// Entries that are ranked by comparing all with all, and that a cluster sorts.  Codes of 30000 x 64 float32, us a call: 4000 12.0 and
// (cluster) 15.0, 5000 14.4 and 15.4, 8000 22.9 and 15.5; 64000 (cluster) 27 and (launches for every pass) 37, 130000 46 and 61.
constexpr unsigned kRankMost = 5120, kClusterMost = 131072;

__device__ __forceinline__ unsigned key_of(long code, long N) { return code >= 0 && code < N ? (unsigned)code : (unsigned)N; }

// Bytes [begin, begin + bytes) of the result that a launch of the sort sets to zero beside its own work, which leaves most SMs and
// all of the memory's bandwidth idle.  Rows that codes name are written again later; knowing them and leaving them out, in the
// launch that sums, took 78 us for 65536 codes of 50000 x 1024 bf16.
struct Zero {
  unsigned char *begin;
  size_t bytes;
};
constexpr size_t kZeroBlock = 64 * 1024;   // bytes of a block
__host__ __device__ __forceinline__ unsigned zero_blocks(const Zero &z) { return (unsigned)((z.bytes + kZeroBlock - 1) / kZeroBlock); }
__device__ __forceinline__ void set_zero(const Zero &z, unsigned block) {
  unsigned char *const from = z.begin + block * kZeroBlock;
  const size_t bytes = min(kZeroBlock, z.bytes - block * kZeroBlock);
  const size_t head = min(bytes, (size_t)((16 - (reinterpret_cast<uintptr_t>(from) & 15)) & 15)), body = (bytes - head) / 16;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (size_t i = threadIdx.x; i < body; i += blockDim.x) reinterpret_cast<uint4 *>(from + head)[i] = zero;
  const size_t rest = bytes - body * 16;   // bytes at either end, an even number of them
  for (size_t i = threadIdx.x * 2; i < rest; i += blockDim.x * 2)
    *reinterpret_cast<unsigned short *>(from + (i < head ? i : body * 16 + i)) = 0;
}

// a < b for numbers of up to 2^31 (the difference's sign: an instruction less than a comparison and a choice)
__device__ __forceinline__ unsigned below(unsigned a, unsigned b) { return (a - b) >> 31; }

// Sorted position of an entry = the entries with a smaller key + those with the same key in front.  A warp takes four entries;
// one launch where a radix sort is four.  Comparisons bound it, the entries squared: 3840 codes with their sums 9.6 us.
template <typename I>
__global__ void __launch_bounds__(kThreads)
    rank_kernel(const I *__restrict__ codes, unsigned entries, unsigned L, long N, uint2 *__restrict__ to, unsigned blocks, const Zero zero) {
  after_previous();
  if (blockIdx.x >= blocks) return set_zero(zero, blockIdx.x - blocks);
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
      to[r] = make_uint2(k[q], (e0 + q) / L);
    }
  }
}

// A pass of a radix sort, least significant digit first: counts of the digits of every tile of entries ...
constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kDigitBits = 9, kDigits = 1 << kDigitBits;

template <typename I, bool FIRST>
__device__ __forceinline__ unsigned sort_key(const I *codes, const uint2 *from, unsigned i, long N) {
  return FIRST ? key_of((long)codes[i], N) : from[i].x;
}

template <typename I, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
    digits_kernel(const I *__restrict__ codes, const uint2 *__restrict__ key, unsigned entries, long N, int shift, unsigned tile,
                  unsigned *__restrict__ counts, unsigned blocks, const Zero zero) {
  after_previous();
  if (blockIdx.x >= blocks) return set_zero(zero, blockIdx.x - blocks);
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
    move_kernel(const I *__restrict__ codes, const uint2 *__restrict__ key, unsigned entries, unsigned L, long N, int shift, unsigned tile,
                const unsigned *__restrict__ counts, uint2 *__restrict__ to_entry, unsigned blocks, const Zero zero) {
  after_previous();
  if (blockIdx.x >= blocks) return set_zero(zero, blockIdx.x - blocks);
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
  for (unsigned b = 0; b < blocks; ++b) {
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
    const uint2 own = !there ? make_uint2(0, 0) : FIRST ? make_uint2(key_of((long)codes[i0 + lane], N), (i0 + lane) / L) : key[i0 + lane];
    const unsigned kk = own.x;
    const unsigned digit = there ? (kk >> shift) & (kDigits - 1) : kDigits;
    const unsigned same = __match_any_sync(0xffffffffu, digit);
    if (there) {
      const unsigned to = s_at[warp][digit] + __popc(same & ((1u << lane) - 1));
      to_entry[to] = own;
    }
    __syncwarp();
    if (there && (same >> lane) == 1u) s_at[warp][digit] += __popc(same);   // the last of its kind
    __syncwarp();
  }
}

// The same sort by one cluster in one launch, for as many entries as its threads hold: an entry's place is found in registers and
// shared memory, and the entries move between the blocks' shared memories.  They are put in order within the block first, so that
// neighbours go to neighbouring places (one by one, each store was 32 requests, and 65536 entries took 24 us).  The steps of a pass and the
// cluster's barriers between them bound it: 7505 entries of two passes 8 us, 65536 with 100 MB of zeros beside them 29 us.
constexpr int kClusterThreads = 1024, kClusterWarps = kClusterThreads / 32, kClusterBlocks = 16;

struct SortSpace {
  unsigned short at[kClusterWarps][kDigits];
  unsigned all[kDigits];               // the block's entries of each digit
  unsigned own[kDigits], base[kDigits];  // where a digit begins in the block, and where its entries go
  unsigned warp[2][kClusterWarps];
};

// EACH entries a thread.  `space`: two entries' room for each of the block's.
template <typename I, int EACH>
__device__ void cluster_sort(cg::cluster_group cluster, SortSpace &s, uint2 *space, const I *codes, unsigned entries, unsigned L, long N, int passes,
                             int digit_bits, uint2 *result) {
  constexpr unsigned kHere = kClusterThreads * EACH;
  uint2 *const hold = space, *const order = space + kHere;
  const unsigned rank = cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1u << digit_bits;
  const unsigned slot0 = warp * (32 * EACH) + lane, first = rank * kHere + slot0;   // a warp's entries lie together
  const unsigned here = entries > rank * kHere ? min(kHere, entries - rank * kHere) : 0;
  uint2 entry[EACH];
#pragma unroll
  for (int r = 0; r < EACH; ++r) entry[r].x = first + r * 32 < entries ? key_of((long)codes[first + r * 32], N) : ~0u;
#pragma unroll
  for (int r = 0; r < EACH; ++r) entry[r].y = (first + r * 32) / L;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    for (unsigned i = threadIdx.x; i < kClusterWarps * kDigits / 2; i += kClusterThreads) reinterpret_cast<unsigned *>(s.at)[i] = 0;
    __syncthreads();
    unsigned short place[EACH];   // among the warp's entries of the same digit
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
      const bool there = first + r * 32 < entries;
      const unsigned digit = there ? (entry[r].x >> shift) & (digits - 1) : kDigits + 1;
      const unsigned same = __match_any_sync(0xffffffffu, digit), front = __popc(same & ((1u << lane) - 1));
      if (there) place[r] = (unsigned short)(s.at[warp][digit] + front);
      __syncwarp();
      if (there && (same >> lane) == 1u) s.at[warp][digit] = (unsigned short)(place[r] + 1);   // the last of its kind
      __syncwarp();
    }
    __syncthreads();
    unsigned run = 0;
    if (threadIdx.x < digits) {
#pragma unroll 8
      for (int w = 0; w < kClusterWarps; ++w) {
        const unsigned c = s.at[w][threadIdx.x];
        s.at[w][threadIdx.x] = (unsigned short)run;
        run += c;
      }
      s.all[threadIdx.x] = run;
    }
    cluster.sync();   // (and every block has read what it holds)
    unsigned all = 0, before = 0;
    if (threadIdx.x < digits)
#pragma unroll
      for (unsigned o = 0; o < kClusterBlocks; ++o) {
        const unsigned c = cluster.map_shared_rank(&s, o)->all[threadIdx.x];
        all += c;
        before += o < rank ? c : 0;
      }
    unsigned in = all, in_own = run;
    for (int off = 1; off < 32; off *= 2) {
      const unsigned o = __shfl_up_sync(0xffffffffu, in, off), p = __shfl_up_sync(0xffffffffu, in_own, off);
      if (lane >= off) in += o, in_own += p;
    }
    if (lane == 31) s.warp[0][warp] = in, s.warp[1][warp] = in_own;
    __syncthreads();
    if (threadIdx.x < digits) {
      unsigned base = before + in - all, own = in_own - run;
      for (unsigned w = 0; w < warp; ++w) base += s.warp[0][w], own += s.warp[1][w];
      s.base[threadIdx.x] = base;
      s.own[threadIdx.x] = own;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < EACH; ++r)
      if (first + r * 32 < entries) {
        const unsigned digit = (entry[r].x >> shift) & (digits - 1);
        order[s.own[digit] + s.at[warp][digit] + place[r]] = entry[r];
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
      const unsigned i = threadIdx.x + r * kClusterThreads;
      if (i >= here) continue;
      const uint2 e = order[i];
      const unsigned digit = (e.x >> shift) & (digits - 1), to = s.base[digit] + i - s.own[digit];
      if (pass + 1 == passes)
        result[to] = e;
      else
        cluster.map_shared_rank(hold, to / kHere)[to % kHere] = e;
    }
    cluster.sync();
    if (pass + 1 < passes) {
#pragma unroll
      for (int r = 0; r < EACH; ++r) entry[r] = hold[slot0 + r * 32];
    }
  }
}

template <typename I, int EACH>
__global__ void __launch_bounds__(kClusterThreads, 1)
    sort_kernel(const I *__restrict__ codes, unsigned entries, unsigned L, long N, int passes, int digit_bits, uint2 *__restrict__ result,
                const Zero zero) {
  after_previous();
  if (blockIdx.x >= kClusterBlocks) {   // (whole clusters; those behind the last piece have none)
    if (blockIdx.x - kClusterBlocks < zero_blocks(zero)) set_zero(zero, blockIdx.x - kClusterBlocks);
    return;
  }
  extern __shared__ uint2 s_space[];
  __shared__ SortSpace s;
  cluster_sort<I, EACH>(cg::this_cluster(), s, s_space, codes, entries, L, N, passes, digit_bits, result);
}

// Entries of a span, whose keys and rows (and a key at either end) lie in shared memory beside two parts for every thread: 48 KB in
// all, which a block has without asking.
constexpr size_t kPartMost = 32;   // bytes of a part
constexpr unsigned kSpanMost = ((48 * 1024 - 2 * kThreads * kPartMost) / sizeof(unsigned) - 2) / 2;

template <typename T, int V>
struct Sums {
  const T *grad;
  const uint2 *entry;   // sorted: code, row of the gradient
  unsigned entries, chunk, span;   // of a group of threads, of a block
  long N, M;
  Wide<T> scale;
  bool accumulate;
  T *out;
  Wide<T> *partial;   // [span][run from the span before, run into the next][M]
  int lanes;
  unsigned tiles;     // of `lanes` vectors

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

// `lanes` threads take a chunk and a tile of columns, a block the chunks of a span.  A run inside a chunk is written; the others'
// parts wait in shared memory and the group in which a run begins (the first one, for a run from the span before) adds them up.
// Memory bounds it: 65536 rows of 1024 bf16 elements in the order of their codes 33 us, 0.55 of the DRAM peak.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 4) sums_kernel(const Sums<T, V> p) {
  after_previous();
  using W = Wide<T>;
  static_assert(sizeof(Vec<W, V>) <= kPartMost, "kSpanMost");
  __shared__ Vec<W, V> s_head[kThreads], s_tail[kThreads];
  // the block's sorted entries, with one more at either end
  extern __shared__ unsigned s_entry[];
  const unsigned span = blockIdx.x / p.tiles, first = span * p.span, size = min(p.span, p.entries - first);
  unsigned *const s_key = s_entry + 1, *const s_row = s_entry + size + 2;
  for (unsigned i = threadIdx.x; i < size + 2; i += kThreads) {
    const unsigned at = first + i - 1;   // (wraps below zero)
    const uint2 own = at < p.entries ? p.entry[at] : make_uint2(~0u, 0);
    s_entry[i] = own.x;
    if (i > 0 && i <= size) s_row[i - 1] = own.y;
  }
  __syncthreads();
  const unsigned group = threadIdx.x / p.lanes, b = group * p.chunk, e = min(size, b + p.chunk);
  const long col = ((long)(blockIdx.x % p.tiles) * p.lanes + threadIdx.x % p.lanes) * V;
  const bool here = b < size && col < p.M && s_key[b] < (unsigned)p.N;   // (codes that name nothing are the last ones)
  W acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = (W)0;
  bool begins = false;   // a run begins in this chunk and goes on behind it
  if (here) {
    const unsigned *const key = s_key + b, *const row = s_row + b;
    unsigned n = e - b;
    while (key[n - 1] >= (unsigned)p.N) --n;
    unsigned cur = key[0];
    bool head = s_entry[b] == cur;   // the key in front
    auto keep = [&](Vec<W, V> &to) {
#pragma unroll
      for (int v = 0; v < V; ++v) to.v[v] = acc[v];
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
          if (head)
            keep(s_head[threadIdx.x]);
          else
            p.write(cur, col, acc);
          cur = k;
          head = false;
#pragma unroll
          for (int v = 0; v < V; ++v) acc[v] = (W)0;
        }
        W f[V];
        widen_all(x[u], f);
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += f[v];
      }
    }
    if (head) {
      keep(s_head[threadIdx.x]);
    } else if (key[n] == cur) {
      keep(s_tail[threadIdx.x]);
      begins = true;
    } else {
      p.write(cur, col, acc);
    }
  }
  __syncthreads();
  if (!here) return;
  auto collect = [&](unsigned cur, unsigned from, int which) {   // the groups' parts from `from` on, while the run goes on
    unsigned end = from * p.chunk;
    while (end < size && s_key[end] == cur) {
      const Vec<W, V> more = s_head[threadIdx.x % p.lanes + from * p.lanes];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += more.v[v];
      end = min(size, end + p.chunk);
      ++from;
      if (s_key[end - 1] != cur) break;
    }
    if (which == 0 || (end == size && s_key[size - 1] == cur && s_key[size] == cur)) {
      W *const to = p.part(span, which, col);
#pragma unroll
      for (int v = 0; v < V; ++v) to[v] = acc[v];
    } else {
      p.write(cur, col, acc);
    }
  };
  if (begins) {
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = s_tail[threadIdx.x].v[v];
    collect(s_key[e - 1], group + 1, 1);
  }
  if (group == 0 && s_entry[0] == s_key[0]) {
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = (W)0;
    collect(s_key[0], 0, 0);
  }
}

// Adds the parts of the runs that cross the end of a span and begin in it: a group of `lanes` threads for each span and tile
// of columns, all groups of the block together for runs of many parts (of which a block, with spans that follow one another,
// has few).  Latency bounds it: 3 to 6 us.
constexpr unsigned kLongRun = 32;
template <typename T, int V, int THREADS>
struct JoinSpace {
  unsigned last[THREADS / 4];   // of each group's run, 0: none or short
  Wide<T> sum[THREADS * V];
};
template <typename T, int V, int THREADS>
__device__ __forceinline__ void join_runs(const Sums<T, V> &p, unsigned block, JoinSpace<T, V, THREADS> &s) {
  using W = Wide<T>;
  unsigned *const s_last = s.last;
  W *const s_sum = s.sum;
  const unsigned groups = THREADS / p.lanes, own = threadIdx.x / p.lanes, lane = threadIdx.x % p.lanes;
  const unsigned spans = (p.entries + p.span - 1) / p.span;
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
  const unsigned blocks = (spans + groups - 1) / groups, c0 = block % blocks * groups, c = c0 + own;
  const long col = ((long)(block / blocks) * p.lanes + lane) * V;
  unsigned cur = 0, last = 0;
  if (c + 1 < spans) {
    const unsigned b = c * p.span, e = b + p.span;
    cur = p.entry[e - 1].x;
    if (p.entry[e].x == cur && cur < (unsigned)p.N && !(b > 0 && p.entry[b].x == cur && p.entry[b - 1].x == cur)) {
      // the last span that begins inside the run: the group's threads try that many places at a time
      last = c + 1;
      unsigned end = spans;
      const unsigned mask = (p.lanes == 32 ? ~0u : (1u << p.lanes) - 1) << (threadIdx.x & 31 & ~(p.lanes - 1));
      for (unsigned step = 1; last + 1 < end; step = (end - last - 1 + p.lanes - 1) / p.lanes) {   // first those that follow
        const unsigned at = last + (lane + 1) * step;
        const int in = __popc(__ballot_sync(mask, at < end && p.entry[at * p.span].x == cur));
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

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) join_kernel(const Sums<T, V> p) {
  after_previous();
  __shared__ JoinSpace<T, V, kThreads> s;
  join_runs(p, blockIdx.x, s);
}

// Whether the device takes a cluster of sixteen blocks (eight are what every device takes).
template <typename I, int EACH>
cudaError_t sort_config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute (&attr)[2], cudaStream_t st) {
  const size_t smem = 2 * sizeof(uint2) * kClusterThreads * EACH;
  cudaError_t e = cudaFuncSetAttribute(sort_kernel<I, EACH>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(sort_kernel<I, EACH>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kClusterBlocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg = {};
  cfg.gridDim = dim3(kClusterBlocks);
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return e;
}
bool cluster_fits() {
  static const bool fits = [] {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    int clusters = 0;
    cudaError_t e = sort_config<int64_t, 8>(cfg, attr, nullptr);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, sort_kernel<int64_t, 8>, &cfg);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess && clusters > 0;
  }();
  return fits;
}
// Sizes of a gradient call.
struct GradientPlan {
  unsigned entries, chunk, span, spans;
  int lanes;
  unsigned tiles;
  bool rank, cluster;      // how the codes are sorted; else by launches for every pass
  unsigned tile, blocks;   // of these passes
  int passes, digit_bits;
  size_t counts, partial;   // elements: the digits' counts, the parts of runs
};
// `vec`: units of an access
GradientPlan gradient_plan(long rows, long L, long N, long M, int vec) {
  GradientPlan p = {};
  p.entries = (unsigned)(rows * L);
  p.rank = p.entries <= kRankMost;
  p.cluster = !p.rank && p.entries <= kClusterMost && cluster_fits();
  const long across = M / vec;
  p.lanes = 4;
  while (p.lanes < 32 && p.lanes < across) p.lanes *= 2;
  p.tiles = (unsigned)((across + p.lanes - 1) / p.lanes);
  // as many chunks as keep all threads busy, of 8 to 64 entries (56 where a block has 64 groups: kSpanMost)
  const long want = 2048l * sm_count() / p.lanes, fits = kSpanMost / (kThreads / p.lanes) / 8 * 8, most = fits < 64 ? fits : 64;
  long chunk = (long)p.entries * p.tiles / want / 8 * 8;
  chunk = chunk < 8 ? 8 : chunk > most ? most : chunk;
  p.chunk = (unsigned)chunk;
  p.span = p.chunk * (kThreads / p.lanes);
  p.spans = (p.entries + p.span - 1) / p.span;
  p.partial = p.spans > 1 ? 2 * (size_t)p.spans * (size_t)M : 0;
  int bits = 1;
  while (bits < 32 && (N >> bits) != 0) ++bits;   // N stands for codes that name nothing
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  if (!p.rank && !p.cluster) {
    // up to 128 tiles: every block of a pass reads the counts of all
    p.tile = ((p.entries + 127) / 128 + kSortThreads - 1) / kSortThreads * kSortThreads;
    if (p.tile < 1024) p.tile = 1024;
    p.blocks = (p.entries + p.tile - 1) / p.tile;
    p.counts = (size_t)p.blocks * kDigits;
  }
  return p;
}

template <typename I, int EACH>
cudaError_t launch_sort(const I *codes, const GradientPlan &p, long L, long N, uint2 *entry, const Zero &zero, cudaStream_t st) {
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  const cudaError_t e = sort_config<I, EACH>(cfg, attr, st);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(kClusterBlocks * (1 + (zero_blocks(zero) + kClusterBlocks - 1) / kClusterBlocks));
  return cudaLaunchKernelEx(&cfg, sort_kernel<I, EACH>, codes, p.entries, (unsigned)L, N, p.passes, p.digit_bits, entry, zero);
}

template <typename T, int V>
cudaError_t launch_sums(const Sums<T, V> &p, unsigned spans, cudaStream_t st) {
  const size_t blocks = (size_t)spans * p.tiles;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const size_t smem = (2 * (size_t)p.span + 2) * sizeof(unsigned);
  cudaError_t e = launch_next(sums_kernel<T, V>, dim3((unsigned)blocks), kThreads, smem, st, p);
  if (e != cudaSuccess) return e;
  count_launches(1);
  if (spans == 1) return e;
  const unsigned per = kThreads / p.lanes;
  e = launch_next(join_kernel<T, V>, dim3((spans + per - 1) / per * p.tiles), kThreads, 0, st, p);
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
  GradientPlan p = gradient_plan(rows, L, N, M, 1);
  for (int vec = 2; vec <= 8 && M % vec == 0; vec *= 2) {   // the width of the accesses depends on addresses
    const size_t partial = gradient_plan(rows, L, N, M, vec).partial;
    if (partial > p.partial) p.partial = partial;
  }
  return (p.rank || p.cluster ? 1 : 2) * (size_t)p.entries * sizeof(uint2) + p.counts * sizeof(unsigned) + 64 + p.partial * wide;
}

template <typename T, typename I>
cudaError_t launch_lookup_gradient(const T *grad, const I *codes, long rows, long L, long N, long M, double scale, bool accumulate, T *out,
                                   void *workspace, cudaStream_t st) {
  const int vec = vector_width<T>(M, grad, out);
  const GradientPlan p = gradient_plan(rows, L, N, M, vec);
  uint2 *entry = static_cast<uint2 *>(workspace);
  void *end = entry + p.entries;
  // the result's bytes over the sort's launches
  const size_t bytes = accumulate ? 0 : (size_t)N * (size_t)M * sizeof(T);
  auto zero = [&](int launch, int launches) {
    const size_t from = bytes / launches / 256 * 256 * launch, to = launch + 1 == launches ? bytes : bytes / launches / 256 * 256 * (launch + 1);
    return Zero{reinterpret_cast<unsigned char *>(out) + from, to - from};
  };
  if (bytes / kZeroBlock > 0x40000000) return cudaErrorInvalidConfiguration;
  cudaError_t e;
  if (p.rank) {
    const Zero z = zero(0, 1);
    const unsigned blocks = (p.entries + kThreads / 8 - 1) / (kThreads / 8);
    e = launch_next(rank_kernel<I>, dim3(blocks + zero_blocks(z)), kThreads, 0, st, codes, p.entries, (unsigned)L, N, entry, blocks, z);
    if (e != cudaSuccess) return e;
    count_launches(1);
  } else if (p.cluster) {
    const unsigned each = (p.entries + kClusterThreads * kClusterBlocks - 1) / (kClusterThreads * kClusterBlocks);
    const Zero z = zero(0, 1);
    e = each <= 1   ? launch_sort<I, 1>(codes, p, L, N, entry, z, st)
        : each <= 2 ? launch_sort<I, 2>(codes, p, L, N, entry, z, st)
        : each <= 4 ? launch_sort<I, 4>(codes, p, L, N, entry, z, st)
                    : launch_sort<I, 8>(codes, p, L, N, entry, z, st);
    if (e != cudaSuccess) return e;
    count_launches(1);
  } else {
    uint2 *other = entry + p.entries;
    unsigned *const counts = reinterpret_cast<unsigned *>(other + p.entries);
    end = counts + p.counts;
    for (int pass = 0; pass < p.passes; ++pass) {
      const int shift = pass * kDigitBits;
      const Zero z = zero(2 * pass, 2 * p.passes), z2 = zero(2 * pass + 1, 2 * p.passes);
      auto digits = pass == 0 ? digits_kernel<I, true> : digits_kernel<I, false>;
      auto move = pass == 0 ? move_kernel<I, true> : move_kernel<I, false>;
      e = launch_next(digits, dim3(p.blocks + zero_blocks(z)), kSortThreads, 0, st, codes, entry, p.entries, N, shift, p.tile, counts, p.blocks, z);
      if (e != cudaSuccess) return e;
      e = launch_next(move, dim3(p.blocks + zero_blocks(z2)), kSortThreads, 0, st, codes, entry, p.entries, (unsigned)L, N, shift, p.tile, counts, other,
                      p.blocks, z2);
      if (e != cudaSuccess) return e;
      count_launches(2);
      uint2 *const moved = other;
      other = entry, entry = moved;
    }
  }
  Wide<T> *const partial = reinterpret_cast<Wide<T> *>((reinterpret_cast<uintptr_t>(end) + 63) / 64 * 64);   // (read 32 bytes at a time)
  const Wide<T> s = (Wide<T>)scale;
#define SBB_SUMS(V) launch_sums(Sums<T, V>{grad, entry, p.entries, p.chunk, p.span, N, M, s, accumulate, out, partial, p.lanes, p.tiles}, p.spans, st)
  if constexpr (sizeof(T) == 2)
    if (vec == 2) return SBB_SUMS(2);
  return vec == 1 ? SBB_SUMS(1) : SBB_SUMS(16 / (int)sizeof(T));
#undef SBB_SUMS
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
