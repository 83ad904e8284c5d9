// Log probabilities of given tokens with entropy and best alternatives:
// ad_token_logprobs and its gradient ad_token_logprobs_grad.
//
// With x a row of logits, k the factor on them (the reciprocal temperature),
// m = max x, s = sum exp(k (x - m)), p = exp(k (x - m)) / s:
//
//   logp    = k (x[token] - m) - ln s
//   entropy = ln s - sum p k (x - m)       (both terms are positive: no cancellation)
//   d loss / d x_j = k (g (1[j = token] - p_j) - e p_j (ln p_j + entropy))
//
// for the gradients g of logp and e of the entropy.
//
// Bound by memory: the row is read once, every thread keeping a running
// maximum, sum and weighted sum that are rescaled together when the maximum
// grows (once for some vectors, not once a value).  Few rows over a large
// vocabulary are split over a cluster of blocks that join through distributed
// shared memory.  The best alternatives come from the same pass: a warp keeps
// its 32 best in registers, one a lane, sorted; values above the worst of the
// wanted ones so far are queued in shared memory and merged 32 at a time.  The
// order is that of (logit, then lower index), a total one, so that the result
// does not depend on scheduling.
//
// Measured: 8191 x 65537 bf16 224 us (4.8 TB/s; instructions: about 13 a value)
// and its gradient 334 us (6.4 TB/s); 2048 x 50001 fp32 with four alternatives 97
// + 125 us; 4 x 131072 bf16 4.8 us, with 20 alternatives 9.8.
//
// Exponentials are those of the multifunction unit (2^x to 2 units in the last
// place) and the factor k times log2 e is rounded once: log probabilities are
// within 3e-7 of themselves where exact steps in 32 bits leave 6e-8.  Both are one
// instruction a value, and instructions are what bounds the forward pass.
//
// A NaN among the logits makes logp, entropy and gradient NaN; it is no alternative.
// Values masked with -inf or a large negative number have p = 0 beside larger
// ones; a row with nothing but -inf has logp = -inf, entropy 0 and no gradient.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>

#include "ops_common.cuh"

namespace {

using namespace adops;
namespace cg = cooperative_groups;

constexpr int MAX_TOP = 32;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float GONE = -200.0f;  // 2^GONE is 0 in 32 bits

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// An offset m k beyond this (a mask of -1e10 or of a type's lowest value, where
// nothing larger is left) is not used: its rounding, of 2^-24 its size, would be a
// factor on the sum that grows out of range.  Differences from m are taken before
// they are multiplied instead, an instruction more for each value.
constexpr float MOST_OFFSET = 1048576.0f;

// Running softmax statistics: largest value m, sum and sum weighted with the
// exponent to base 2, both relative to the offset o = m k (rounded; all that
// follows goes by the rounded one), or to m k itself where the offset is huge.
// -FLT_MAX rather than -inf at the start: -inf values then lie infinitely below
// it and count for nothing.
struct Soft {
  // The factor to base 2.  It stays a number for the largest factors: infinite, it
  // would make a NaN of a value's distance of 0 from itself.
  __device__ __forceinline__ static float factor(float scale) { return fminf(scale * LOG2E, FLT_MAX); }
  float m = -FLT_MAX, o, s = 0.0f, w = 0.0f;
  __device__ __forceinline__ explicit Soft(float k) : o(offset(m, k)) {}
  __device__ __forceinline__ static bool huge(float o) { return !(fabsf(o) <= MOST_OFFSET); }
  __device__ __forceinline__ bool huge() const { return huge(o); }
  // rounded for good: contracted into a later difference it would not be the offset
  __device__ __forceinline__ static float offset(float m, float k) { return __fmul_rn(m, k); }
  // The distance of what sums are relative to, from (m, o) to (to, to_o).  ANY:
  // offsets may be huge; they are not where there is a sum, else.
  template <bool ANY>
  __device__ __forceinline__ static float below(float m, float o, float to, float to_o, float k) {
    if (!ANY) return fmaxf(o - to_o, GONE);
    const float d = huge(o) ? (huge(to_o) ? (m - to) * k : fmaf(m, k, -to_o)) : huge(to_o) ? -fmaf(to, k, -o) : o - to_o;
    return fmaxf(d, GONE);
  }
  template <bool ANY = true>
  __device__ __forceinline__ void raise(float to, float k) {
    const float to_o = offset(to, k), d = below<ANY>(m, o, to, to_o, k), f = exp2_approx(d);
    w = f * fmaf(d, s, w);
    s *= f;
    m = to;
    o = to_o;
  }
  __device__ __forceinline__ static void plus(float x, float k, float o, float& s, float& w) {
    const float d = fmaf(x, k, -o), e = exp2_approx(d);
    s += e;
    w = fmaf(e, fmaxf(d, GONE), w);
  }
  template <bool HUGE>
  __device__ __forceinline__ void add(float x, float k) {
    const float d = HUGE ? (x - m) * k : fmaf(x, k, -o), e = exp2_approx(d);
    s += e;  // a NaN stays here
    w = fmaf(e, fmaxf(d, GONE), w);
  }
  template <bool ANY>
  __device__ __forceinline__ void join(float om, float os, float ow, float k) {
    const float to = fmaxf(m, om);
    raise<ANY>(to, k);
    Soft other(k);
    other.m = om, other.o = offset(om, k), other.s = os, other.w = ow;
    other.raise<ANY>(to, k);
    s += other.s;
    w += other.w;
  }
  template <bool ANY>
  __device__ __forceinline__ void join_all(float k) {
#pragma unroll
    for (int i = 16; i; i >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, i), os = __shfl_xor_sync(0xffffffffu, s, i),
                  ow = __shfl_xor_sync(0xffffffffu, w, i);
      join<ANY>(om, os, ow, k);
    }
  }
  // Lanes without a sum do not count, wherever their offset lies: one look for the
  // five joins (4 x 131072 bf16 4.8 us; looked for in each 5.6).
  __device__ __forceinline__ void join_lanes(float k) {
    if (__any_sync(0xffffffffu, huge() && s != 0.0f))
      join_all<true>(k);
    else
      join_all<false>(k);
  }
  // Natural logarithm of a value's share, given that of the sum.  A value far
  // below the maximum (masked with the type's lowest value) may leave the range of
  // 32 bits when it is multiplied by k, where its distance times the factor does
  // not; and the distance may, where the products with the factor do not.
  __device__ __forceinline__ float log_share(float x, float k, float scale, float ln_s) const {
    const float d = fmaf(x, k, -o);
    if (!huge() && !isinf(d)) return LN2 * d - ln_s;
    const float far = x - m;
    return (isinf(far) ? fmaf(x, scale, -(m * scale)) : far * scale) - ln_s;
  }
};

// The largest of a thread's values, -FLT_MAX at least; NaNs do not count.
template <typename T, int U>
__device__ __forceinline__ float largest(const uint4 (&r)[U]) {
  if constexpr (sizeof(T) == 2) {  // two by one instruction
    typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
    T2 big[U * 4];
#pragma unroll
    for (int q = 0; q < U; ++q) memcpy(big + q * 4, &r[q], sizeof(r[q]));
#pragma unroll
    for (int n = U * 2; n; n /= 2)
#pragma unroll
      for (int i = 0; i < n; ++i) big[i] = __hmax2(big[i], big[i + n]);
    return fmaxf(fmaxf(to_float(big[0].x), to_float(big[0].y)), -FLT_MAX);
  } else {
    float big = -FLT_MAX;
#pragma unroll
    for (int q = 0; q < U; ++q) {
      float e[4];
      unpack<T>(r[q], e);
#pragma unroll
      for (int j = 0; j < 4; ++j) big = fmaxf(big, e[j]);
    }
    return big;
  }
}
// 16 bytes of -inf
template <typename T>
__device__ __forceinline__ uint4 nothing() {
  const unsigned w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

// Alternatives order by this: larger logit first, then lower index.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);  // -0 counts as +0
  return u ^ (static_cast<unsigned>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
typedef unsigned long long u64;
__device__ __forceinline__ u64 entry_of(float x, unsigned index) {
  return static_cast<u64>(order_of(x)) << 32 | (0xffffffffu - index);
}

template <typename U>
__device__ __forceinline__ U exchange(U v, int o, bool keep_larger) {
  const U other = __shfl_xor_sync(0xffffffffu, v, o);
  return (v > other) == keep_larger ? v : other;
}
// Largest first over the lanes of a warp.
template <typename U>
__device__ __forceinline__ U sort_warp(U v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1) v = exchange(v, o, ((lane & o) == 0) == ((lane & size) == 0 || size == 32));
  return v;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ u64 merge_warp(u64 a, u64 b) {
  const int lane = threadIdx.x & 31;
  const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
  u64 v = a > r ? a : r;
#pragma unroll
  for (int o = 16; o; o >>= 1) v = exchange(v, o, (lane & o) == 0);
  return v;
}

struct LogprobArgs {
  const void* logits;
  long long ld;
  long long rows;
  int vocab, top, tok64;
  const void* tokens;
  float scale;
  float *logp, *entropy, *stats, *top_logp;
  long long* top_index;
};

constexpr int QUEUE = 64;  // entries of a warp's queue: under 32 left over and 32 new

// A warp's best so far.
struct Best {
  u64 list = 0;  // lane i: the i-th best
  u64 bar = 0;   // a value has to pass this to be among the wanted ones
  int queued = 0;

  __device__ __forceinline__ void flush(u64* queue, u64* shared_bar, int top) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    const int n = queued < 32 ? queued : 32;
    const u64 v = lane < n ? queue[lane] : 0;
    const u64 rest = lane + 32 < queued ? queue[lane + 32] : 0;
    __syncwarp();
    if (lane + 32 < queued) queue[lane] = rest;
    queued -= n;
    list = merge_warp(list, sort_warp(v));
    const u64 mine = __shfl_sync(0xffffffffu, list, top - 1);
    if (lane == 0 && mine > *reinterpret_cast<volatile u64*>(shared_bar)) atomicMax(shared_bar, mine);
    __syncwarp();
    const u64 all = *reinterpret_cast<volatile u64*>(shared_bar);
    bar = mine > all ? mine : all;
    bar = __shfl_sync(0xffffffffu, bar, 0);
  }
  // All lanes call; `x` counts where `valid`.
  __device__ __forceinline__ void offer(float x, unsigned index, bool valid, u64* queue, u64* shared_bar, int top) {
    const u64 e = entry_of(x, index);
    const bool in = valid && x == x && e > bar;
    const unsigned who = __ballot_sync(0xffffffffu, in);
    if (!who) return;
    if (in) queue[queued + __popc(who & ((1u << (threadIdx.x & 31)) - 1))] = e;
    queued += __popc(who);
    if (queued >= 32) flush(queue, shared_bar, top);
  }
};

constexpr int MAX_WARPS = 16;
constexpr int VECS = 4, AHEAD = 2;  // vectors of a round, rounds under way

struct Shared {
  float m[MAX_WARPS], s[MAX_WARPS], w[MAX_WARPS];
  u64 bar;
  u64 queue[MAX_WARPS][QUEUE];
  u64 list[MAX_WARPS][32];
  // this block's result, read by the first block of the cluster
  float bm, bs, bw;
  u64 blist[32];
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(512) logprob_kernel(const __grid_constant__ LogprobArgs a) {
  constexpr int V = 16 / sizeof(T), U = VECS;
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned parts_u = cluster.num_blocks();
  const int parts = parts_u, part = cluster.block_rank();
  const long long row = blockIdx.x / parts_u;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const float k = Soft::factor(a.scale);
  if (TOP) {
    if (threadIdx.x == 0) sh.bar = 0;
    __syncthreads();
  }
  // The row as unaligned head, vectors, tail.
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(a.vocab, off ? V - off : 0);
  const int vecs = (a.vocab - head) / V, tail0 = head + vecs * V;
  const int share = (vecs + parts - 1) / parts;
  const int v0 = min(vecs, part * share), v1 = min(vecs, v0 + share);
  Soft soft(k);
  Best best;
  u64* queue = sh.queue[warp];

  // The lanes of a warp stay together for the votes.  Vectors to come are copied
  // into the thread's own places in shared memory, AHEAD rounds before they are
  // worked on: there is nothing to wait for but its own copies.
  typedef uint4 Set[U];
  extern __shared__ __align__(16) unsigned char ring[];
  const unsigned places = static_cast<unsigned>(__cvta_generic_to_shared(ring)) + threadIdx.x * 16;
  const int step = blockDim.x * U;
  int base = v0 + warp * 32;
  auto fetch = [&](int stage, int base) {
    const T* p = x + head + static_cast<long long>(base + lane) * V;
#pragma unroll
    for (int q = 0; q < U; ++q)
      if (base + q * static_cast<int>(blockDim.x) + lane < v1)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(places + (stage * U + q) * blockDim.x * 16),
                     "l"(p + static_cast<long long>(q * blockDim.x) * V));
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto take = [&](Set& r, int stage, int base) {
    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
#pragma unroll
    for (int q = 0; q < U; ++q) {
      r[q] = nothing<T>();
      if (base + q * static_cast<int>(blockDim.x) + lane < v1)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[q].x), "=r"(r[q].y), "=r"(r[q].z), "=r"(r[q].w)
                     : "r"(places + (stage * U + q) * blockDim.x * 16)
                     : "memory");
    }
  };
  auto work = [&](const Set& r, int base, bool start) {
    const float big = largest<T, U>(r);
    if (big > soft.m) soft.raise(big, k);
    if (soft.huge()) {
#pragma unroll
      for (int q = 0; q < U; ++q) {
        float e[V];
        unpack<T>(r[q], e);
#pragma unroll
        for (int j = 0; j < V; ++j) soft.add<true>(e[j], k);
      }
    } else {
      float s2 = 0.0f, w2 = 0.0f;  // two chains of sums
#pragma unroll
      for (int q = 0; q < U; ++q) {
        float e[V];
        unpack<T>(r[q], e);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          soft.add<false>(e[j], k);
          Soft::plus(e[j + 1], k, soft.o, s2, w2);
        }
      }
      soft.s += s2;
      soft.w += w2;
    }
    if (TOP) {
      // The first values: the wanted number of a warp's lanes' maxima reach
      // `seed`, so no alternative lies below it, nor below the largest seed.
      if (start) {
        const unsigned seed = __shfl_sync(0xffffffffu, sort_warp(order_of(big)), a.top - 1);
        if (lane == 0 && seed > order_of(-FLT_MAX)) atomicMax(&sh.bar, static_cast<u64>(seed) << 32);
        __syncthreads();
        best.bar = *reinterpret_cast<volatile u64*>(&sh.bar);
      }
      const float bar = best.bar ? value_of(static_cast<unsigned>(best.bar >> 32)) : -INFINITY;
      if (__any_sync(0xffffffffu, big >= bar || best.bar == 0)) {
        unsigned pass = 0;
#pragma unroll
        for (int q = 0; q < U; ++q) {
          float e[V];
          unpack<T>(r[q], e);
          if (base + q * static_cast<int>(blockDim.x) + lane < v1) {
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (e[j] >= bar) pass |= 1u << (q * V + j);
          }
        }
        // one a lane at a time, read again: registers cannot be indexed
        while (__any_sync(0xffffffffu, pass != 0)) {
          const int bit = __ffs(pass) - 1;
          pass &= pass - 1;
          const int i = head + (base + (bit / V) * static_cast<int>(blockDim.x) + lane) * V + bit % V;
          best.offer(bit >= 0 ? to_float(x[i]) : 0.0f, i, bit >= 0, queue, &sh.bar, a.top);
        }
      }
    }
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(i, base + i * step);
  int stage = 0;
  for (bool start = true; start || base < v1; start = false) {
    Set r;
    take(r, stage, base);
    fetch(stage, base + AHEAD * step);
    stage = stage + 1 == AHEAD ? 0 : stage + 1;
    work(r, base, start);
    base += step;
  }
  // Head and tail: fewer than a vector each, by the first block's first warp.
  if (part == 0 && warp == 0) {
    const int rest = head + (a.vocab - tail0);
    const bool has = lane < rest;
    const int i = lane < head ? lane : tail0 + (lane - head);
    const float xi = has ? to_float(x[i]) : -INFINITY;
    if (has) {
      if (xi > soft.m) soft.raise(xi, k);
      if (soft.huge())
        soft.add<true>(xi, k);
      else
        soft.add<false>(xi, k);
    }
    if (TOP) best.offer(xi, i, has, queue, &sh.bar, a.top);
  }
  // Lanes, warps, blocks; lists by pairs.
  soft.join_lanes(k);
  if (lane == 0) sh.m[warp] = soft.m, sh.s[warp] = soft.s, sh.w[warp] = soft.w;
  if (TOP) {
    while (best.queued) best.flush(queue, &sh.bar, a.top);
    sh.list[warp][lane] = best.list;
  }
  __syncthreads();
  if (TOP)
    for (int n = 1; n < warps; n *= 2) {
      if (warp % (2 * n) == 0 && warp + n < warps) sh.list[warp][lane] = merge_warp(sh.list[warp][lane], sh.list[warp + n][lane]);
      __syncthreads();
    }
  if (warp == 0) {
    soft = Soft(k);
    if (lane < warps) soft.m = sh.m[lane], soft.o = Soft::offset(soft.m, k), soft.s = sh.s[lane], soft.w = sh.w[lane];
    soft.join_lanes(k);
    if (TOP) best.list = sh.list[0][lane];
    if (parts > 1) {
      if (lane == 0) sh.bm = soft.m, sh.bs = soft.s, sh.bw = soft.w;
      if (TOP) sh.blist[lane] = best.list;
    }
  }
  if (parts > 1) {
    cluster.sync();
    if (part == 0) {
      if (TOP) {
        if (warp < parts) sh.list[warp][lane] = cluster.map_shared_rank(&sh, warp)->blist[lane];
        for (int i = warps + warp; i < parts; i += warps) sh.list[i][lane] = cluster.map_shared_rank(&sh, i)->blist[lane];
        __syncthreads();
        for (int n = 1; n < parts; n *= 2) {
          for (int i = 2 * n * warp; i + n < parts; i += 2 * n * warps)
            sh.list[i][lane] = merge_warp(sh.list[i][lane], sh.list[i + n][lane]);
          __syncthreads();
        }
      }
      if (warp == 0) {
        soft = Soft(k);
        if (lane < parts) {
          const Shared* other = cluster.map_shared_rank(&sh, lane);
          soft.m = other->bm, soft.o = Soft::offset(soft.m, k), soft.s = other->bs, soft.w = other->bw;
        }
        soft.join_lanes(k);
        if (TOP) best.list = sh.list[0][lane];
      }
    }
    cluster.sync();  // no block ends while its shared memory is read
  }
  if (part == 0 && warp == 0) {
    const bool empty = soft.s == 0.0f;
    const float ln_s = empty ? 0.0f : logf(soft.s);
    if (lane == 0) {
      const long long t =
          a.tok64 ? static_cast<const long long*>(a.tokens)[row] : static_cast<const int*>(a.tokens)[row];
      float lp = 0.0f;
      if (t >= a.vocab)
        lp = __int_as_float(0x7fffffff);
      else if (t >= 0)
        lp = empty ? -INFINITY : soft.log_share(to_float(x[t]), k, a.scale, ln_s);
      const float h = empty ? 0.0f : ln_s - LN2 * (soft.w / soft.s);
      a.logp[row] = lp;
      a.entropy[row] = h;
      reinterpret_cast<float4*>(a.stats)[row] =
          make_float4(soft.m, soft.s, h, empty ? -INFINITY : (soft.huge() ? soft.m * a.scale : LN2 * soft.o) + ln_s);
    }
    if (TOP && lane < a.top) {
      const float v = value_of(static_cast<unsigned>(best.list >> 32));
      a.top_logp[row * a.top + lane] = empty ? -INFINITY : soft.log_share(v, k, a.scale, ln_s);
      a.top_index[row * a.top + lane] =
          best.list ? static_cast<long long>(0xffffffffu - static_cast<unsigned>(best.list)) : -1ll;
    }
  }
}

struct LogprobGradArgs {
  const void* logits;
  void* out;
  long long ld, ldo;
  long long rows;
  int vocab, segments, tok64;
  const void* tokens;
  float scale;
  const float *stats, *g_logp, *g_entropy;
};

constexpr int GRAD_THREADS = 256, GRAD_VECS = 4;  // a block's share of a row: so many vectors a thread

// V = 1 where rows of the result are not aligned as those of the logits are.
template <typename T, int V>
__global__ void __launch_bounds__(GRAD_THREADS) logprob_grad_kernel(const __grid_constant__ LogprobGradArgs a) {
  const unsigned row_u = blockIdx.x / static_cast<unsigned>(a.segments);
  const long long row = row_u;
  const int seg = blockIdx.x - row_u * a.segments;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  T* y = static_cast<T*>(a.out) + row * a.ldo;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = V == 1 ? 0 : min(a.vocab, off ? V - off : 0);
  const int vecs = (a.vocab - head) / V, tail0 = head + vecs * V;
  Vec<T, V> r[GRAD_VECS];
  const int first = seg * (GRAD_THREADS * GRAD_VECS) + threadIdx.x;
#pragma unroll
  for (int q = 0; q < GRAD_VECS; ++q) {
    const int v = first + q * GRAD_THREADS;
    if (v < vecs) r[q] = load_vec<T, V>(x + head + static_cast<long long>(v) * V);
  }
  const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
  const long long t = a.tok64 ? static_cast<const long long*>(a.tokens)[row] : static_cast<const int*>(a.tokens)[row];
  const bool empty = st.y == 0.0f;  // the log of the sum may be past 32 bits for another reason
  float g = t >= 0 && a.g_logp ? a.g_logp[row] : 0.0f;
  const float e = a.g_entropy ? a.g_entropy[row] : 0.0f;
  if (t >= a.vocab) g *= __int_as_float(0x7fffffff);
  const float hot = empty ? 0.0f : g * a.scale;
  // with l = k (x - m): -k p (g + e (l - ln s + H)) = q exp(l) (g' + e l)
  const float k = Soft::factor(a.scale), el = e * LN2;
  const float c = empty ? 0.0f : -a.scale / st.y, b = empty ? 0.0f : g + e * (st.z - logf(st.y));
  const float o = Soft::offset(st.x, k);
  const bool huge = Soft::huge(o);
  auto grad = [&](float d) { return c * exp2_approx(d) * fmaf(el, fmaxf(d, GONE), b); };
#pragma unroll
  for (int q = 0; q < GRAD_VECS; ++q) {
    const int v = first + q * GRAD_THREADS;
    if (v >= vecs) continue;
    const int i = head + v * V;
    float z[V];
    if constexpr (V == 1) {
      z[0] = to_float(r[q].v[0]);
    } else {
      uint4 w;
      memcpy(&w, &r[q], sizeof(w));
      unpack<T>(w, z);
    }
    if (huge) {
#pragma unroll
      for (int j = 0; j < V; ++j) z[j] = grad((z[j] - st.x) * k);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) z[j] = grad(fmaf(z[j], k, -o));
    }
    if (t >= i && t < i + V) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (t == i + j) z[j] += hot;
    }
    Vec<T, V> w;
    round_to<T, V>(z, w);
    store_vec<T, V>(y + i, w);
  }
  const int rest = head + (a.vocab - tail0);
  if (seg == 0 && static_cast<int>(threadIdx.x) < rest) {
    const int i = static_cast<int>(threadIdx.x) < head ? threadIdx.x : tail0 + (threadIdx.x - head);
    const float xi = to_float(x[i]);
    y[i] = from_float<T>(grad(huge ? (xi - st.x) * k : fmaf(xi, k, -o)) + (t == i ? hot : 0.0f));
  }
}

template <typename T>
cudaError_t forward(const LogprobArgs& a, int sms, cudaStream_t s) {
  const int vecs = a.vocab / (16 / static_cast<int>(sizeof(T)));
  // Threads for four vectors each; where there are rows enough for all
  // multiprocessors not so many that joining them costs more than it saves.
  // Blocks of a cluster while the rows leave multiprocessors without work and a
  // block keeps a vector a thread.
  const int most = a.rows >= 8ll * sms ? 128 : a.rows >= 4ll * sms ? 256 : 512;
  int threads = 64;
  while (threads < most && threads * 4 < vecs) threads *= 2;
  int parts = 1;
  while (parts < 8 && a.rows * parts * 2 <= sms && parts * 2 * threads <= vecs) parts *= 2;
  const int share = (vecs + parts - 1) / parts, rounds = (share + threads * VECS - 1) / (threads * VECS);
  const int bytes = threads * VECS * 16 * std::min(std::max(rounds, 1), AHEAD);
  const void* kernel = a.top ? reinterpret_cast<const void*>(logprob_kernel<T, true>)
                             : reinterpret_cast<const void*>(logprob_kernel<T, false>);
  if (bytes + static_cast<int>(sizeof(Shared)) + 1024 > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(static_cast<unsigned>(a.rows * parts));
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = bytes;
  c.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  return a.top ? cudaLaunchKernelEx(&c, logprob_kernel<T, true>, a) : cudaLaunchKernelEx(&c, logprob_kernel<T, false>, a);
}

template <typename T>
cudaError_t backward(LogprobGradArgs a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool same = ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 &&
                    ((a.ld - a.ldo) * static_cast<long long>(sizeof(T))) % 16 == 0;
  const long long per = static_cast<long long>(GRAD_THREADS) * GRAD_VECS * (same ? V : 1);
  a.segments = static_cast<int>((a.vocab + per - 1) / per);
  const long long blocks = a.rows * a.segments;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  return same ? launch<logprob_grad_kernel<T, V>>(static_cast<unsigned>(blocks), GRAD_THREADS, 0, s, a)
              : launch<logprob_grad_kernel<T, 1>>(static_cast<unsigned>(blocks), GRAD_THREADS, 0, s, a);
}

int check(const char* who, int dtype, const void* logits, int64_t ld, int64_t rows, int64_t vocab, const void* tokens,
          int tok64, float scale) {
  if (dtype < AD_F32 || dtype > AD_F16) return fail("%s: unknown element type %d", who, dtype);
  if (rows < 0 || vocab < 1 || vocab > 0x7fff0000ll) return fail("%s: %lld rows of %lld logits", who, (long long)rows, (long long)vocab);
  if (rows > 0x0fffffffll) return fail("%s: %lld rows in one call", who, (long long)rows);
  if (!(scale > 0.0f) || scale > FLT_MAX) return fail("%s: the factor %g is not a positive number", who, scale);
  if (rows && (!logits || !tokens)) return fail("%s: null operand", who);
  if (rows > 1 && ld < vocab) return fail("%s: rows overlap", who);
  if (!aligned(logits, elem_size(dtype))) return fail("%s: unaligned logits", who);
  if (!aligned(tokens, tok64 ? 8 : 4)) return fail("%s: unaligned tokens", who);
  return 0;
}

}  // namespace

extern "C" int ad_token_logprobs(int device, int dtype, const void* logits, int64_t ld, int64_t rows, int64_t vocab,
                                 const void* tokens, int tok64, float scale, int top, float* logp, float* entropy,
                                 float* stats, float* top_logp, int64_t* top_index, void* stream) {
  if (check("ad_token_logprobs", dtype, logits, ld, rows, vocab, tokens, tok64, scale)) return 1;
  if (top < 0 || top > MAX_TOP || top > vocab)
    return fail("ad_token_logprobs: %d alternatives (at most %d, and no more than logits)", top, MAX_TOP);
  if (rows == 0) return 0;
  if (!logp || !entropy || !stats || !aligned(stats, 16) || !aligned({logp, entropy}, 4) ||
      (top && (!top_logp || !top_index || !aligned(top_logp, 4) || !aligned(top_index, 8))))
    return fail("ad_token_logprobs: null or unaligned result");
  DeviceGuard g(device);
  if (g.error() != cudaSuccess) return fail_cuda("ad_token_logprobs", g.error());
  const int sms = sm_count(g.device());
  if (!sms) return fail("ad_token_logprobs: no device properties");
  LogprobArgs a = {};
  a.logits = logits, a.ld = ld, a.rows = rows, a.vocab = static_cast<int>(vocab), a.top = top;
  a.tokens = tokens, a.tok64 = tok64, a.scale = scale;
  a.logp = logp, a.entropy = entropy, a.stats = stats, a.top_logp = top_logp;
  a.top_index = reinterpret_cast<long long*>(top_index);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == AD_F32    ? forward<float>(a, sms, s)
                        : dtype == AD_BF16 ? forward<__nv_bfloat16>(a, sms, s)
                                           : forward<__half>(a, sms, s);
  if (e != cudaSuccess) return fail_cuda("ad_token_logprobs", e);
  return 0;
}

extern "C" int ad_token_logprobs_grad(int device, int dtype, const void* logits, int64_t ld, int64_t rows,
                                      int64_t vocab, const void* tokens, int tok64, float scale, const float* stats,
                                      const float* g_logp, const float* g_entropy, void* grad, int64_t ld_grad,
                                      void* stream) {
  if (check("ad_token_logprobs_grad", dtype, logits, ld, rows, vocab, tokens, tok64, scale)) return 1;
  if (rows == 0) return 0;
  if (!stats || !aligned(stats, 16) || !grad || !aligned(grad, elem_size(dtype)) || !aligned({g_logp, g_entropy}, 4))
    return fail("ad_token_logprobs_grad: null or unaligned operand");
  if (rows > 1 && ld_grad < vocab) return fail("ad_token_logprobs_grad: rows of the gradient overlap");
  DeviceGuard g(device);
  if (g.error() != cudaSuccess) return fail_cuda("ad_token_logprobs_grad", g.error());
  LogprobGradArgs a = {};
  a.logits = logits, a.out = grad, a.ld = ld, a.ldo = ld_grad, a.rows = rows, a.vocab = static_cast<int>(vocab);
  a.tokens = tokens, a.tok64 = tok64, a.scale = scale;
  a.stats = stats, a.g_logp = g_logp, a.g_entropy = g_entropy;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == AD_F32    ? backward<float>(a, s)
                        : dtype == AD_BF16 ? backward<__nv_bfloat16>(a, s)
                                           : backward<__half>(a, s);
  if (e != cudaSuccess) return fail_cuda("ad_token_logprobs_grad", e);
  return 0;
}
