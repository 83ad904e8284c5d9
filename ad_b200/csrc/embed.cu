// Embedding rows of given tokens and the table's gradient: ad_embed, ad_embed_grad.
//
//   y[r] = scale T[t_r];   dT[v] = scale sum of dy[r] over the r with t_r = v
//
// Bound by memory.  Forward: a warp a row and a slice of its columns, four 16-byte
// loads a lane under way.
//
// Gradient: the rows of dy that belong to one token are summed in the order of
// their positions, so that nothing depends on scheduling.  Positions are sorted by
// token (a stable radix sort of at most 10 bits a pass: counts of each 2048 keys, their
// running sums, the move; up to 16384 keys all in one launch); sorted positions are cut into chunks of 32, and a warp walks
// a chunk over a slice of columns, with a running sum in 32 bits.  A token whose rows
// lie in one chunk is written there and then; a sum that goes on in the next chunk
// is left in memory, and a last kernel joins such partial sums, a block a token and
// slice, found through a list.  A token that comes up thousands of times so costs
// no more than others.  Rows of tokens that do not come up are cleared by further
// blocks of the sort's launches, once the first two have noted which these are (in one
// launch: all rows).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops_common.cuh"

namespace {

using namespace adops;

struct EmbedArgs {
  const void* table;
  long long ldt, vocab;
  const void* tokens;
  int tok64;
  long long rows;
  int width;
  float scale;
  void* y;
  long long ldy;
};

template <typename T, int V>
__global__ void __launch_bounds__(256) embed_kernel(const __grid_constant__ EmbedArgs a) {
  after_previous();
  constexpr int U = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = a.width / V;                      // vectors of a row
  const int slices = (per + 32 * U - 1) / (32 * U);  // a warp's share
  const long long items = a.rows * slices;
  for (long long i = blockIdx.x * 8ll + warp; i < items; i += gridDim.x * 8ll) {
    const long long r = slices == 1 ? i : i / slices;
    const int first = static_cast<int>(i - r * slices) * (32 * U) + lane;
    const long long t = token_at(a.tokens, a.tok64, r);
    const T* from = static_cast<const T*>(a.table) + t * a.ldt;
    T* to = static_cast<T*>(a.y) + r * a.ldy;
    const bool known = t >= 0 && t < a.vocab;
    const float fill = t < 0 ? 0.0f : __int_as_float(0x7fffffff);
    Vec<T, V> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = first + 32 * u;
      if (known && c < per) x[u] = load_vec<T, V>(from + c * V);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = first + 32 * u;
      if (c >= per) continue;
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = known ? to_float(x[u].v[j]) * a.scale : fill;
      round_to<T, V>(v, x[u]);
      store_vec<T, V>(to + c * V, x[u]);
    }
  }
}

// ------------------------------------------------------------------ sort

constexpr int TILE = 2048, SORT_THREADS = 256, SORT_WARPS = 8, KEYS = TILE / SORT_THREADS;
constexpr int MAX_BITS = 10, MAX_DIGITS = 1 << MAX_BITS;

// Rows of the table's gradient to clear: `units` of `unit` bytes each, by `lanes` lanes,
// `rows` of them (a power of two up to 8) by a warp.
struct Clear {
  unsigned char* p;
  long long row_stride, from, to;
  const unsigned char* seen;  // eight rows a byte; NULL: all are cleared
  int unit, units, lanes, rows;
};

// Keys and the positions that they came from; the first pass takes them from the
// tokens themselves, the others from the previous pass.  Tokens outside of the
// vocabulary have its size as their key and end up last.
struct SortArgs {
  const void* tokens;
  int tok64;
  long long vocab;
  const int *keys, *at;
  int *keys_out, *at_out;
  int n, tiles, shift, digits;
  int* counts;  // [digits][tiles], then their running sums
  int* totals;  // [digits]
  int* joins;   // the numbers of short and of long joins, cleared ahead of the sums
  unsigned* seen;  // a bit for each token that comes up: cleared by the first launch, set by the second
  int seen_words, noting;  // blocks of the second launch that set them
  Clear clear;     // this launch's share of the rows to clear
};
// Blocks from `first` on clear; whether this is one of them.  A warp takes one to eight
// rows (whose bits lie in a byte), a group of its lanes a row at a time.
__device__ __forceinline__ bool clears(const Clear& c, unsigned first) {
  if (blockIdx.x < first) return false;
  const long long warps = static_cast<long long>(gridDim.x - first) * (blockDim.x >> 5);
  const int lane = threadIdx.x & 31, at_once = 32 / c.lanes < c.rows ? 32 / c.lanes : c.rows, l = lane & (c.lanes - 1);
  if (lane / c.lanes >= at_once) return true;
  for (long long r0 = c.from + ((blockIdx.x - first) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * static_cast<long long>(c.rows); r0 < c.to;
       r0 += warps * c.rows) {
    const unsigned seen = c.seen ? c.seen[r0 >> 3] >> (r0 & 7) : 0u;
    for (int j = lane / c.lanes; j < c.rows && r0 + j < c.to; j += at_once) {
      if (seen >> j & 1) continue;
      unsigned char* p = c.p + (r0 + j) * c.row_stride;
      if (c.unit == 16)
        for (int i = l; i < c.units; i += c.lanes) reinterpret_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
      else if (c.unit == 4)
        for (int i = l; i < c.units; i += c.lanes) reinterpret_cast<unsigned*>(p)[i] = 0;
      else
        for (int i = l; i < c.units; i += c.lanes) reinterpret_cast<unsigned short*>(p)[i] = 0;
    }
  }
  return true;
}
__device__ __forceinline__ int key_of(const SortArgs& a, int i) {
  if (a.keys) return a.keys[i];
  const long long t = token_at(a.tokens, a.tok64, i);
  return static_cast<int>(t < 0 || t >= a.vocab ? a.vocab : t);
}

__global__ void __launch_bounds__(SORT_THREADS) count_kernel(const __grid_constant__ SortArgs a) {
  after_previous();
  __shared__ int hist[MAX_DIGITS];
  if (clears(a.clear, a.tiles)) return;
  if (blockIdx.x == 0 && threadIdx.x < 2) a.joins[threadIdx.x] = 0;
  for (int d = threadIdx.x; d < a.digits; d += SORT_THREADS) hist[d] = 0;
  if (a.seen)
    for (int i = blockIdx.x * SORT_THREADS + threadIdx.x; i < a.seen_words; i += a.tiles * SORT_THREADS) a.seen[i] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    const int i = blockIdx.x * TILE + j * SORT_THREADS + threadIdx.x;
    if (i >= a.n) continue;
    atomicAdd(&hist[(key_of(a, i) >> a.shift) & (a.digits - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.digits; d += SORT_THREADS) a.counts[static_cast<long long>(d) * a.tiles + blockIdx.x] = hist[d];
}

// A digit's counts to running sums over the tiles, a warp a digit.
__global__ void __launch_bounds__(256) scan_kernel(const __grid_constant__ SortArgs a) {
  after_previous();
  const unsigned scanning = (a.digits + 7) / 8;
  if (clears(a.clear, scanning + a.noting)) return;
  if (blockIdx.x >= scanning) {  // which tokens come up
    for (int i = (blockIdx.x - scanning) * 256 + threadIdx.x; i < a.n; i += a.noting * 256) {
      const int key = key_of(a, i);
      const unsigned bit = 1u << (key & 31);
      if (key < a.vocab && !(a.seen[key >> 5] & bit)) atomicOr(&a.seen[key >> 5], bit);
    }
    return;
  }
  const int d = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (d >= a.digits) return;
  int* c = a.counts + static_cast<long long>(d) * a.tiles;
  int before = 0;
  for (int i0 = 0; i0 < a.tiles; i0 += 32) {
    const int i = i0 + lane, mine = i < a.tiles ? c[i] : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (i < a.tiles) c[i] = before + sum - mine;
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) a.totals[d] = before;
}

// Running sums over `digits` values of shared memory, in place, by the whole block.
__device__ __forceinline__ void scan_digits(int* v, int digits, int* warp_sums) {
  constexpr int PER = MAX_DIGITS / SORT_THREADS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x[PER], sum = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int d = threadIdx.x * PER + j;
    x[j] = d < digits ? v[d] : 0;
    sum += x[j];
  }
  int all = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += y;
  }
  if (lane == 31) warp_sums[warp] = all;
  __syncthreads();
  int before = all - sum;
  for (int w = 0; w < warp; ++w) before += warp_sums[w];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int d = threadIdx.x * PER + j;
    if (d < digits) v[d] = before;
    before += x[j];
  }
  __syncthreads();
}

// The lanes with this lane's digit (-1: none), bit by bit: __match_any_sync takes longer the more
// digits differ (8192 tokens sorted by a block: 45 us, 40).
__device__ __forceinline__ unsigned same_digit(int digit) {
  unsigned same = __ballot_sync(0xffffffffu, digit >= 0);
#pragma unroll
  for (int b = 0; b < MAX_BITS; ++b) {
    const unsigned set = __ballot_sync(0xffffffffu, digit >> b & 1);
    same &= digit >> b & 1 ? set : ~set;
  }
  return same;
}

// Where each key of a tile goes: its place among the tile's keys of its digit,
// from the warps' counts.  `base`: where the tile's first key of each digit goes.
struct TileSort {
  int hist[SORT_WARPS][MAX_DIGITS];
  int base[MAX_DIGITS];
  int warp_sums[SORT_WARPS];
};
__device__ __forceinline__ void rank_tile(TileSort& s, const int (&digit)[KEYS], int (&place)[KEYS], int digits) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    // lanes behind the last key have a digit of -1
    const unsigned same = same_digit(digit[j]);
    const int before = __popc(same & ((1u << lane) - 1));
    int seen = 0;
    if (digit[j] >= 0) seen = s.hist[warp][digit[j]];
    __syncwarp();
    if (digit[j] >= 0 && before == 0) s.hist[warp][digit[j]] = seen + __popc(same);
    __syncwarp();
    place[j] = seen + before;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += SORT_THREADS) {
    int run = s.base[d];
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) {
      const int x = s.hist[w][d];
      s.hist[w][d] = run;
      run += x;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < KEYS; ++j)
    if (digit[j] >= 0) place[j] += s.hist[warp][digit[j]];
}

__global__ void __launch_bounds__(SORT_THREADS) move_kernel(const __grid_constant__ SortArgs a) {
  after_previous();
  __shared__ TileSort s;
  if (clears(a.clear, a.tiles)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < a.digits; d += SORT_THREADS) {
    s.base[d] = a.totals[d];
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) s.hist[w][d] = 0;
  }
  __syncthreads();
  scan_digits(s.base, a.digits, s.warp_sums);
  for (int d = threadIdx.x; d < a.digits; d += SORT_THREADS)
    s.base[d] += a.counts[static_cast<long long>(d) * a.tiles + blockIdx.x];
  int key[KEYS], digit[KEYS], place[KEYS];
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    const int i = blockIdx.x * TILE + warp * (KEYS * 32) + j * 32 + lane;
    key[j] = i < a.n ? key_of(a, i) : 0;
    digit[j] = i < a.n ? (key[j] >> a.shift) & (a.digits - 1) : -1;
  }
  __syncthreads();
  rank_tile(s, digit, place, a.digits);
#pragma unroll
  for (int j = 0; j < KEYS; ++j) {
    const int i = blockIdx.x * TILE + warp * (KEYS * 32) + j * 32 + lane;
    if (i < a.n) {
      a.keys_out[place[j]] = key[j];
      a.at_out[place[j]] = a.at ? a.at[i] : i;
    }
  }
}

// All passes over at most ONE keys, by one block, PER keys a thread; others clear.  (Gradients of
// 2049 tokens of 1000, rows of 512 bytes: 16.5 us, in three launches 23.3.  Of 500 of them: 14.1,
// 17.0 with eight keys a thread.)
constexpr int ONE = 4096, ONE_THREADS = 1024, ONE_WARPS = ONE_THREADS / 32;
struct OneSort {
  union {
    unsigned short hist[ONE_WARPS][MAX_DIGITS];  // of the warps, then where their keys go
    struct {
      int keys[ONE];
      short at[ONE];
    };
  };
  int warp_sums[ONE_WARPS];
};
template <int PER>
__global__ void __launch_bounds__(ONE_THREADS) sort_kernel(const __grid_constant__ SortArgs a, int bits, int passes) {
  after_previous();
  extern __shared__ __align__(16) unsigned char raw[];
  OneSort& s = *reinterpret_cast<OneSort*>(raw);
  if (clears(a.clear, 1)) return;
  if (threadIdx.x < 2) a.joins[threadIdx.x] = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << bits, d = threadIdx.x;
  int key[PER], from[PER], digit[PER], place[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    from[j] = warp * (PER * 32) + j * 32 + lane;
    key[j] = from[j] < a.n ? key_of(a, from[j]) : 0;
  }
  for (int p = 0; p < passes; ++p) {
    if (d < digits)
      for (int w = 0; w < ONE_WARPS; ++w) s.hist[w][d] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {  // places among the warp's keys of a digit
      digit[j] = -1;
      if (warp * (PER * 32) + j * 32 >= a.n) continue;
      const bool there = warp * (PER * 32) + j * 32 + lane < a.n;
      digit[j] = there ? (key[j] >> (p * bits)) & (digits - 1) : -1;
      const unsigned same = same_digit(digit[j]);
      const int before = __popc(same & ((1u << lane) - 1));
      const int seen = there ? s.hist[warp][digit[j]] : 0;
      __syncwarp();
      if (there && before == 0) s.hist[warp][digit[j]] = static_cast<unsigned short>(seen + __popc(same));
      __syncwarp();
      place[j] = seen + before;
    }
    __syncthreads();
    // running sums over the digits, of all warps' counts, a digit a thread
    int mine = 0;
    if (d < digits)
      for (int w = 0; w < ONE_WARPS; ++w) mine += s.hist[w][d];
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) s.warp_sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      int x = s.warp_sums[lane];
      const int own = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      s.warp_sums[lane] = x - own;
    }
    __syncthreads();
    if (d < digits) {
      int run = s.warp_sums[warp] + sum - mine;
      for (int w = 0; w < ONE_WARPS; ++w) {
        const int x = s.hist[w][d];
        s.hist[w][d] = static_cast<unsigned short>(run);
        run += x;
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (digit[j] >= 0) place[j] += s.hist[warp][digit[j]];
    __syncthreads();  // the counts have served: keys and positions go in their place
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (digit[j] >= 0) s.keys[place[j]] = key[j], s.at[place[j]] = static_cast<short>(from[j]);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = warp * (PER * 32) + j * 32 + lane;
      if (i < a.n) key[j] = s.keys[i], from[j] = s.at[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = warp * (PER * 32) + j * 32 + lane;
    if (i < a.n) a.keys_out[i] = key[j], a.at_out[i] = from[j];
  }
}

// All passes over at most MANY keys, by the blocks of one cluster, PER keys a thread; other
// clusters clear.  The blocks tell one another how often each digit comes up through their
// shared memory; keys go from pass to pass through L2.
// (5670 tokens of 30000, rows of 1 KB: 25.8 us; one block 29.7, six launches 41.0.  16288 of 50001,
// rows of 2 KB: 40 and 61.  With eight keys a thread 16385 of 30000 take 50, in six launches 40: a
// key's place is anywhere, and a multiprocessor stores 32 bytes a clock.)
constexpr int CLUSTER = 8, MANY = 2 * ONE_THREADS * CLUSTER;
struct ManySort {
  unsigned short hist[ONE_WARPS][MAX_DIGITS];  // of the warps, then where their keys go: less than MANY
  int total[MAX_DIGITS];                       // of the block
  int warp_sums[ONE_WARPS];
};
static_assert(MANY <= 0x10000, "16 bits hold where a key goes");
struct Passes {
  int *keys[2], *at[2];  // pass p writes p & 1
  int bits, count;
};
__device__ __forceinline__ int read_of(const int* mine, int rank) {
  int v;
  asm volatile(
      "{\n\t.reg .u32 there;\n\t"
      "mapa.shared::cluster.u32 there, %1, %2;\n\t"
      "ld.shared::cluster.s32 %0, [there];\n\t}"
      : "=r"(v)
      : "r"(static_cast<unsigned>(__cvta_generic_to_shared(mine))), "r"(rank)
      : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int PER>
__global__ void __launch_bounds__(ONE_THREADS) cluster_sort_kernel(const __grid_constant__ SortArgs a, const __grid_constant__ Passes b) {
  after_previous();
  extern __shared__ __align__(16) unsigned char raw[];
  ManySort& s = *reinterpret_cast<ManySort*>(raw);
  if (clears(a.clear, CLUSTER)) return;  // whole clusters
  const int rank = blockIdx.x;           // of the first one
  if (rank == 0 && threadIdx.x < 2) a.joins[threadIdx.x] = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << b.bits, d = threadIdx.x;
  const int first = rank * (PER * ONE_THREADS) + warp * (PER * 32) + lane;
  int key[PER], from[PER], digit[PER], place[PER];
  for (int p = 0; p < b.count; ++p) {
    const int in = p & 1 ? 0 : 1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = first + j * 32;
      key[j] = i >= a.n ? 0 : p ? __ldcg(b.keys[in] + i) : key_of(a, i);
      from[j] = i >= a.n ? 0 : p ? __ldcg(b.at[in] + i) : i;
    }
    if (d < digits)
      for (int w = 0; w < ONE_WARPS; ++w) s.hist[w][d] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {  // places among the warp's keys of a digit
      const bool there = first + j * 32 < a.n;
      digit[j] = there ? (key[j] >> (p * b.bits)) & (digits - 1) : -1;
      const unsigned same = same_digit(digit[j]);
      const int before = __popc(same & ((1u << lane) - 1));
      const int seen = there ? s.hist[warp][digit[j]] : 0;
      __syncwarp();
      if (there && before == 0) s.hist[warp][digit[j]] = static_cast<unsigned short>(seen + __popc(same));
      __syncwarp();
      place[j] = seen + before;
    }
    __syncthreads();
    int mine = 0;
    if (d < digits) {
      for (int w = 0; w < ONE_WARPS; ++w) mine += s.hist[w][d];
      s.total[d] = mine;
    }
    cluster_sync();
    int all = 0, ahead = 0;  // of the cluster's blocks, and of those before this one
    if (d < digits) {
#pragma unroll
      for (int q = 0; q < CLUSTER; ++q) {
        const int x = read_of(&s.total[d], q);
        all += x;
        if (q < rank) ahead += x;
      }
    }
    int sum = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) s.warp_sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      int x = s.warp_sums[lane];
      const int own = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      s.warp_sums[lane] = x - own;
    }
    __syncthreads();
    if (d < digits) {
      int run = s.warp_sums[warp] + sum - all + ahead;
      for (int w = 0; w < ONE_WARPS; ++w) {
        const int x = s.hist[w][d];
        s.hist[w][d] = static_cast<unsigned short>(run);
        run += x;
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (digit[j] < 0) continue;
      const int to = place[j] + s.hist[warp][digit[j]];
      __stcg(b.keys[in ^ 1] + to, key[j]);
      __stcg(b.at[in ^ 1] + to, from[j]);
    }
    cluster_sync();  // what was written is there for all; and no block leaves, or counts again, ahead of the others' reads
  }
}

// ------------------------------------------------------------------ sums

constexpr int SPAN = 32;   // sorted positions a chunk
constexpr int SHORT = 16;  // chunks that a token goes on in and one warp joins

struct SumArgs {
  const void* dy;
  long long lddy;
  const int *keys, *at;  // sorted
  int n, chunks, width, vocab;
  float scale;
  void* out;
  int out_type;
  long long ldo;
  int accumulate;
  float* part;  // [chunks][2][ldp]: a sum that began earlier, one that goes on
  long long ldp;
  int *joins, *list;  // the numbers of tokens whose sums are to be joined, and where they begin: short and long ones
  int vec_out;  // the result takes the vectors that dy does
};

// V columns of a row of the result.
template <int V>
__device__ __forceinline__ void write_sum(const SumArgs& a, int key, int col, float (&v)[V]) {
  const long long at = key * a.ldo + col;
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] *= a.scale;
  if (V > 1 && a.vec_out && !a.accumulate) {
    if (a.out_type == AD_F32) {
      float* p = static_cast<float*>(a.out) + at;
      if constexpr (V % 4 == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 4) store_vec<float, 4>(p + j, {{v[j], v[j + 1], v[j + 2], v[j + 3]}});
        return;
      }
    } else if constexpr (V % 2 == 0) {
      if (a.out_type == AD_BF16) {
        Vec<__nv_bfloat16, V> w;
        round_to<__nv_bfloat16, V>(v, w);
        store_vec<__nv_bfloat16, V>(static_cast<__nv_bfloat16*>(a.out) + at, w);
      } else {
        Vec<__half, V> w;
        round_to<__half, V>(v, w);
        store_vec<__half, V>(static_cast<__half*>(a.out) + at, w);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    store_any(a.out, a.out_type, at + j, a.accumulate ? load_any(a.out, a.out_type, at + j) + v[j] : v[j]);
}

template <typename T, int V>
__global__ void __launch_bounds__(128) sum_kernel(const __grid_constant__ SumArgs a) {
  after_previous();
  constexpr int U = 8;  // rows under way
  const int lane = threadIdx.x & 31;
  const int per = a.width / V, slices = (per + 31) / 32;
  const long long items = static_cast<long long>(a.chunks) * slices;
  for (long long item = blockIdx.x * 4ll + (threadIdx.x >> 5); item < items; item += gridDim.x * 4ll) {
    const int chunk = static_cast<int>(item / slices), slice = static_cast<int>(item - static_cast<long long>(chunk) * slices);
    const int first = chunk * SPAN, count = min(SPAN, a.n - first);
    const int vec = slice * 32 + lane;
    const bool in = vec < per;
    const int col = vec * V;
    const int my_key = lane < count ? a.keys[first + lane] : a.vocab;
    const int my_at = lane < count ? a.at[first + lane] : 0;
    const int earlier = first ? a.keys[first - 1] : -1;
    const int later = first + SPAN < a.n ? a.keys[first + SPAN] : a.vocab;
    // keys past the vocabulary are last
    const int used = __popc(__ballot_sync(0xffffffffu, my_key < a.vocab));
    if (!used) continue;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    bool began = __shfl_sync(0xffffffffu, my_key, 0) != earlier;
    for (int i0 = 0; i0 < used; i0 += U) {
      Vec<T, V> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = __shfl_sync(0xffffffffu, my_at, (i0 + u) & 31);
        if (i0 + u < used && in) x[u] = load_vec<T, V>(static_cast<const T*>(a.dy) + at * a.lddy + col);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u;
        const int key = __shfl_sync(0xffffffffu, my_key, i & 31), next_here = __shfl_sync(0xffffffffu, my_key, (i + 1) & 31);
        if (i < used) {
          if (in) {
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += to_float(x[u].v[j]);
          }
          const bool last = i + 1 == SPAN;  // of the chunk: the token may go on in the next one
          const int next = last ? later : next_here;
          if (next != key || last) {
            const bool ends = next != key;
            if (began && ends) {
              if (in) write_sum<V>(a, key, col, sum);
            } else {
              if (in) {
                float* p = a.part + (2ll * chunk + (began ? 1 : 0)) * a.ldp + col;
                if constexpr (V % 4 == 0) {
#pragma unroll
                  for (int j = 0; j < V; j += 4) store_vec<float, 4>(p + j, {{sum[j], sum[j + 1], sum[j + 2], sum[j + 3]}});
                } else {
#pragma unroll
                  for (int j = 0; j < V; ++j) p[j] = sum[j];
                }
              }
              if (began && slice == 0 && lane == 0) {
                const int beyond = chunk + SHORT + 1;
                const int kind = beyond < a.chunks && a.keys[beyond * SPAN] == key;
                a.list[kind * a.chunks + atomicAdd(&a.joins[kind], 1)] = chunk;
              }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] = 0.0f;
            began = true;
          }
        }
      }
    }
  }
}

// Four columns of a row of the result.
__device__ __forceinline__ void write_four(const SumArgs& a, int key, int col, float4 x) {
  float v[4] = {x.x, x.y, x.z, x.w};
  if (a.vec_out && col + 4 <= a.width) {
    write_sum<4>(a, key, col, v);
  } else {
    for (int j = 0; j < 4 && col + j < a.width; ++j) {
      float one[1] = {v[j]};
      write_sum<1>(a, key, col + j, one);
    }
  }
}

// The partial sums of a token: the chunk where it began, then those that it goes
// on in.  128 columns at a time: by a warp where there are few, in their order, else by
// eight warps by turns, whose sums are joined in the warps' order.  (All of them by
// blocks, a search of the token's end ahead of each 128 columns: 47 us for 131072 rows
// of 2048 instead of 22.)
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ SumArgs a) {
  after_previous();
  __shared__ float4 buf[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slices = (a.width + 127) / 128;
  auto add = [&](float4& x, int c, int chunk, int col) {
    const float4 y = *reinterpret_cast<const float4*>(a.part + (2ll * c + (c == chunk ? 1 : 0)) * a.ldp + col);
    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
  };
  // the token, and how many of the next 32 chunks begin with it
  auto look = [&](int chunk, int& key) {
    key = a.keys[chunk * SPAN + SPAN - 1];
    const int c = chunk + 1 + lane;
    return __popc(__ballot_sync(0xffffffffu, c < a.chunks && a.keys[c * SPAN] == key));
  };
  const long long longs = static_cast<long long>(a.joins[1]) * slices;
  for (long long item = blockIdx.x; item < longs; item += gridDim.x) {
    const int chunk = a.list[a.chunks + item / slices], col = static_cast<int>(item % slices) * 128 + lane * 4;
    int key, last = chunk + look(chunk, key);
    if (last == chunk + 32) {  // by halving
      int past = a.chunks;
      while (past - last > 1) {
        const int mid = last + (past - last) / 2;
        if (a.keys[mid * SPAN] == key)
          last = mid;
        else
          past = mid;
      }
    }
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (col < a.width) {
#pragma unroll 4
      for (int c = chunk + warp; c <= last; c += 8) add(x, c, chunk, col);
    }
    buf[warp][lane] = x;
    __syncthreads();
    if (warp == 0 && col < a.width) {
      for (int w = 1; w < 8; ++w) {
        const float4 y = buf[w][lane];
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
      }
      write_four(a, key, col, x);
    }
    __syncthreads();
  }
  const long long shorts = static_cast<long long>(a.joins[0]) * slices;
  for (long long item = blockIdx.x * 8ll + warp; item < shorts; item += gridDim.x * 8ll) {
    const int chunk = a.list[item / slices], col = static_cast<int>(item % slices) * 128 + lane * 4;
    int key;
    const int last = chunk + look(chunk, key);
    if (col >= a.width) continue;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int c = chunk; c <= last; ++c) add(x, c, chunk, col);
    write_four(a, key, col, x);
  }
}

// ------------------------------------------------------------------ host

struct Layout {
  bool one, many;  // sorted by one block, by a cluster
  int bits, passes, tiles, chunks;
  long long ldp;
  size_t keys[2], at[2], counts, totals, seen, joins, list, part, total;
};
Layout plan(long long rows, long long vocab, long long width) {
  Layout l;
  int bits = 1;
  while (vocab >> bits) ++bits;
  l.passes = (bits + MAX_BITS - 1) / MAX_BITS;
  l.bits = (bits + l.passes - 1) / l.passes;
  l.one = rows <= ONE, l.many = !l.one && rows <= MANY;
  l.tiles = static_cast<int>((rows + TILE - 1) / TILE);
  l.chunks = static_cast<int>((rows + SPAN - 1) / SPAN);
  l.ldp = (width + 3) / 4 * 4;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int k = 0; k < 2; ++k) l.keys[k] = take(4ull * rows), l.at[k] = take(4ull * rows);
  l.counts = take(4ull * l.tiles << l.bits);
  l.totals = take(4ull << l.bits);
  l.seen = take((vocab + 31) / 32 * 4);
  l.joins = take(8);
  l.list = take(8ull * l.chunks);
  l.part = take(8ull * l.chunks * l.ldp);
  l.total = at;
  return l;
}

template <typename T, int V>
cudaError_t embed(const EmbedArgs& a, int sms, cudaStream_t st) {
  const long long per = a.width / V, items = a.rows * ((per + 127) / 128);
  const long long blocks = std::min<long long>((items + 7) / 8, 16ll * sms);
  return launch_early<embed_kernel<T, V>>(dim3(static_cast<unsigned>(blocks)), 256, 0, st, a);
}
template <typename T, int V>
cudaError_t sums(const SumArgs& a, int sms, cudaStream_t st) {
  const long long items = static_cast<long long>(a.chunks) * ((a.width / V + 31) / 32);
  const long long blocks = std::min<long long>((items + 3) / 4, 32ll * sms);
  return launch_early<sum_kernel<T, V>>(dim3(static_cast<unsigned>(blocks)), 128, 0, st, a);
}

int check(const char* who, int dtype, int64_t rows, int64_t vocab, int64_t width) {
  if (dtype < AD_F32 || dtype > AD_F16) return fail("%s: unknown element type %d", who, dtype);
  if (rows < 0 || vocab < 1 || width < 0) return fail("%s: %lld rows of %lld, %lld tokens", who, (long long)rows, (long long)width, (long long)vocab);
  if (rows > (1 << 30) || vocab > (1 << 30) || width > (1 << 24))
    return fail("%s: at most 2^30 rows and tokens, of 2^24 elements", who);
  return 0;
}

}  // namespace

extern "C" int ad_embed(int device, int dtype, const void* tokens, int tok64, int64_t rows, const void* table, int64_t ldt,
                        int64_t vocab, int64_t width, float scale, void* y, int64_t ldy, void* stream) {
  const char* who = "ad_embed";
  if (check(who, dtype, rows, vocab, width)) return 1;
  if (!std::isfinite(scale)) return fail("%s: scale %g", who, scale);
  if (!rows || !width) return 0;
  if (rows > 1 && ldy < width) return fail("%s: rows overlap", who);
  if (!tokens || !table || !y) return fail("%s: null operand", who);
  const int es = elem_size(dtype);
  if (!aligned(tokens, tok64 ? 8 : 4) || !aligned({table, y}, es)) return fail("%s: an operand is not aligned to its elements", who);
  if (overlap({{y, rows, width * es, ldy * es, true}, {table, vocab, width * es, ldt * es, false}, {tokens, 1, rows * (tok64 ? 8 : 4), 0, false}}))
    return fail("%s: results overlap operands or one another", who);
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
  const int sms = sm_count(guard.device());
  if (!sms) return fail("%s: no device properties", who);
  const EmbedArgs a = {table, ldt, vocab, tokens, tok64, rows, static_cast<int>(width), scale, y, ldy};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // 16 bytes at a time where every row of both allows it, else 4, else an element
  auto fits = [&](int bytes) {
    const int v = bytes / es;
    return width % v == 0 && (vocab == 1 || ldt % v == 0) && (rows == 1 || ldy % v == 0) && aligned(table, bytes) && aligned(y, bytes);
  };
  const bool wide = fits(16), pair = es == 2 && fits(4);
  const cudaError_t e = dtype == AD_F32    ? (wide ? embed<float, 4>(a, sms, st) : embed<float, 1>(a, sms, st))
                        : dtype == AD_BF16 ? (wide   ? embed<__nv_bfloat16, 8>(a, sms, st)
                                              : pair ? embed<__nv_bfloat16, 2>(a, sms, st)
                                                     : embed<__nv_bfloat16, 1>(a, sms, st))
                                           : (wide   ? embed<__half, 8>(a, sms, st)
                                              : pair ? embed<__half, 2>(a, sms, st)
                                                     : embed<__half, 1>(a, sms, st));
  return e == cudaSuccess ? 0 : fail_cuda(who, e);
}

extern "C" int ad_embed_grad_workspace(int64_t rows, int64_t vocab, int64_t width, size_t* bytes) {
  const char* who = "ad_embed_grad_workspace";
  if (!bytes) return fail("%s: null operand", who);
  if (check(who, AD_F32, rows, vocab, width)) return 1;
  *bytes = rows && width ? plan(rows, vocab, width).total : 0;
  return 0;
}

extern "C" int ad_embed_grad(int device, int dtype, const void* dy, int64_t lddy, const void* tokens, int tok64,
                             int64_t rows, int64_t vocab, int64_t width, float scale, int out_type, void* out, int64_t ldo,
                             int accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "ad_embed_grad";
  if (check(who, dtype, rows, vocab, width)) return 1;
  if (out_type != dtype && out_type != AD_F32) return fail("%s: unknown type %d of the result", who, out_type);
  if (!std::isfinite(scale)) return fail("%s: scale %g", who, scale);
  if (!width) return 0;
  if (vocab > 1 && ldo < width) return fail("%s: rows overlap", who);
  const int es = elem_size(dtype), os = elem_size(out_type);
  if (!out || !aligned(out, os)) return fail("%s: an operand is null or not aligned to its elements", who);
  if (!rows) return accumulate ? 0 : ad_clear_rows(device, out, ldo * os, width * os, vocab, stream);
  if (!dy || !tokens) return fail("%s: null operand", who);
  if (!aligned(tokens, tok64 ? 8 : 4) || !aligned(dy, es)) return fail("%s: an operand is not aligned to its elements", who);
  const Layout l = plan(rows, vocab, width);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.total)
    return fail("%s: needs %zu bytes of workspace, 256-byte aligned", who, l.total);
  if (overlap({{out, vocab, width * os, ldo * os, true}, {workspace, 1, static_cast<long long>(l.total), 0, true},
               {dy, rows, width * es, lddy * es, false}, {tokens, 1, rows * (tok64 ? 8 : 4), 0, false}}))
    return fail("%s: results overlap operands or one another", who);
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
  const int sms = sm_count(guard.device());
  if (!sms) return fail("%s: no device properties", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  auto ints = [&](size_t at) { return reinterpret_cast<int*>(ws + at); };

  SortArgs s = {};
  s.tokens = tokens, s.tok64 = tok64, s.vocab = vocab, s.n = static_cast<int>(rows), s.tiles = l.tiles;
  s.counts = ints(l.counts), s.totals = ints(l.totals), s.joins = ints(l.joins);
  // One launch sorts few tokens, and clears all rows beside.  With more,
  // the launches of the sort wait for memory most of the time.  The first two note which
  // tokens come up; each of the others clears a share of the rows beside its work, and leaves those
  // to the sums (131072 tokens of as many, rows of 8 KB: 454 us, 509 with all rows cleared).
  const bool single = l.one || l.many, note = !single && !accumulate;
  Clear clear = {};
  clear.p = static_cast<unsigned char*>(out), clear.row_stride = ldo * os;
  const long long bytes = width * os;
  auto whole = [&](int unit) { return bytes % unit == 0 && (vocab == 1 || clear.row_stride % unit == 0) && aligned(out, unit); };
  clear.unit = whole(16) ? 16 : whole(4) ? 4 : 2;
  clear.units = static_cast<int>(bytes / clear.unit);
  for (clear.lanes = 1; clear.lanes < 32 && clear.lanes < clear.units;) clear.lanes *= 2;
  for (clear.rows = 8; clear.rows > 1 && clear.rows * bytes > 4096;) clear.rows /= 2;  // 4 KB a warp (8: 98 us instead of 94)
  const int early = note ? 2 : 0, launches = (single ? 1 : 3 * l.passes) - early;
  const long long share = (vocab + 8 * launches - 1) / (8 * launches) * 8;
  auto clearing = [&](int launch) {  // blocks that clear in one of the launches
    if (accumulate || launch < early) return 0u;
    s.clear = clear;
    s.clear.from = std::min<long long>(vocab, (launch - early) * share), s.clear.to = std::min<long long>(vocab, s.clear.from + share);
    const int per = (single ? ONE_WARPS : SORT_WARPS) * clear.rows;  // rows a block
    return static_cast<unsigned>(std::min<long long>((s.clear.to - s.clear.from + per - 1) / per, (single ? 8ll : 32ll) * sms));
  };
  cudaError_t e;
  int to = 0;
  if (l.one) {
    s.keys_out = ints(l.keys[0]), s.at_out = ints(l.at[0]);
    const unsigned more = clearing(0);
    int most = 0;
    auto go = [&](auto v) {
      constexpr int PER = decltype(v)::value;
      const cudaError_t f = shared_room<sort_kernel<PER>>(&most);
      if (f != cudaSuccess) return f;
      if (most < static_cast<int>(sizeof(OneSort))) return cudaErrorInvalidConfiguration;
      return launch_early<sort_kernel<PER>>(dim3(1 + more), ONE_THREADS, sizeof(OneSort), st, s, l.bits, l.passes);
    };
    e = rows <= ONE_THREADS       ? go(std::integral_constant<int, 1>())
        : rows <= 2 * ONE_THREADS ? go(std::integral_constant<int, 2>())
                                  : go(std::integral_constant<int, 4>());
    if (e != cudaSuccess) return fail_cuda(who, e);
  } else if (l.many) {
    to = (l.passes - 1) & 1;
    const Passes b = {{ints(l.keys[0]), ints(l.keys[1])}, {ints(l.at[0]), ints(l.at[1])}, l.bits, l.passes};
    const unsigned more = (clearing(0) + CLUSTER - 1) / CLUSTER * CLUSTER;
    int most = 0;
    auto go = [&](auto v) {
      constexpr int PER = decltype(v)::value;
      const cudaError_t f = shared_room<cluster_sort_kernel<PER>>(&most);
      if (f != cudaSuccess) return f;
      if (most < static_cast<int>(sizeof(ManySort))) return cudaErrorInvalidConfiguration;
      return launch_early_cluster<cluster_sort_kernel<PER>>(CLUSTER, dim3(CLUSTER + more), ONE_THREADS, sizeof(ManySort), st, s, b);
    };
    e = rows <= ONE_THREADS * CLUSTER ? go(std::integral_constant<int, 1>()) : go(std::integral_constant<int, 2>());
    if (e != cudaSuccess) return fail_cuda(who, e);
  } else {
    if (note) {
      s.seen = reinterpret_cast<unsigned*>(ws + l.seen), s.seen_words = static_cast<int>((vocab + 31) / 32);
      clear.seen = ws + l.seen;
    }
    s.digits = 1 << l.bits;
    for (int p = 0; p < l.passes; ++p) {
      to = p & 1;
      s.shift = p * l.bits;
      s.keys = p ? ints(l.keys[to ^ 1]) : nullptr, s.at = p ? ints(l.at[to ^ 1]) : nullptr;
      s.keys_out = ints(l.keys[to]), s.at_out = ints(l.at[to]);
      unsigned more = clearing(3 * p);
      e = launch_early<count_kernel>(dim3(l.tiles + more), SORT_THREADS, 0, st, s);
      more = clearing(3 * p + 1);
      s.noting = p || !note ? 0 : std::min((s.n + 1023) / 1024, 8 * sms);
      if (e == cudaSuccess) e = launch_early<scan_kernel>(dim3((s.digits + 7) / 8 + s.noting + more), 256, 0, st, s);
      s.seen = nullptr;
      more = clearing(3 * p + 2);
      if (e == cudaSuccess) e = launch_early<move_kernel>(dim3(l.tiles + more), SORT_THREADS, 0, st, s);
      if (e != cudaSuccess) return fail_cuda(who, e);
    }
  }

  SumArgs a = {};
  a.dy = dy, a.lddy = lddy;
  a.keys = ints(l.keys[to]), a.at = ints(l.at[to]);
  a.n = s.n, a.chunks = l.chunks, a.width = static_cast<int>(width), a.vocab = static_cast<int>(vocab);
  a.scale = scale, a.out = out, a.out_type = out_type, a.ldo = ldo, a.accumulate = accumulate;
  a.part = reinterpret_cast<float*>(ws + l.part), a.ldp = l.ldp;
  a.joins = s.joins, a.list = ints(l.list);
  auto fits = [&](int bytes) {
    const int v = bytes / es;
    return width % v == 0 && (rows == 1 || lddy % v == 0) && aligned(dy, bytes);
  };
  // rows of 64 bytes and more a slice: 16 bytes a lane where the rows are long enough for a warp
  const bool wide = fits(16) && (es == 4 || width >= 128), pair = es == 2 && fits(4);
  a.vec_out = width % (16 / os) == 0 && (vocab == 1 || ldo % (16 / os) == 0) && aligned(out, 16);
  e = dtype == AD_F32    ? (wide ? sums<float, 4>(a, sms, st) : sums<float, 1>(a, sms, st))
      : dtype == AD_BF16 ? (wide   ? sums<__nv_bfloat16, 8>(a, sms, st)
                            : pair ? sums<__nv_bfloat16, 2>(a, sms, st)
                                   : sums<__nv_bfloat16, 1>(a, sms, st))
                         : (wide   ? sums<__half, 8>(a, sms, st)
                            : pair ? sums<__half, 2>(a, sms, st)
                                   : sums<__half, 1>(a, sms, st));
  if (e != cudaSuccess) return fail_cuda(who, e);
  const long long joins = static_cast<long long>(l.chunks) * ((width + 127) / 128);
  e = launch_early<join_kernel>(dim3(static_cast<unsigned>(std::min<long long>(joins, 8ll * sms))), 256, 0, st, a);
  return e == cudaSuccess ? 0 : fail_cuda(who, e);
}
