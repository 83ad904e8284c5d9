#ifndef AD_B200_BLOCK_NORM_CUH
#define AD_B200_BLOCK_NORM_CUH
// The glue between two blocks of a transformer in one pass: ad_block_norm and
// its gradient ad_block_norm_grad.
//
//   u = norm(z) wa + ba        the norm after a block (u = z without wa)
//   h = scale x + act(gate) u  the gated, scaled residual sum
//   y = norm(h) wb + bb        the norm before the next block (no y without wb)
//
// norm(v) = (v - m) / sqrt(mean (v - m)^2 + eps), m = mean v for a LayerNorm
// and 0 for an RMS norm; act is the identity or the sigmoid; the gate has one
// row for every `rows_per_gate` rows.  With nz, nh the normalised rows, rz, rh
// the reciprocal deviations and d = dy wb,
//
//   t  = dh + rh (d - nh mean(d nh) [- mean d])      the whole gradient of h
//   dx = scale t,  du = t act(gate),  dgate = t u act'(gate)
//   dz = rz (e - nz mean(e nz) [- mean e]),  e = du wa
//   dwa = sum du nz,  dba = sum du,  dwb = sum dy nh,  dbb = sum dy
//
// Bound by memory: one block keeps its row in registers and loops over rows,
// so every tensor crosses the bus once.  The gradient computes h again from x,
// z and the gate, which costs the bytes that reading h would and keeps h's
// rounding out of it.  Statistics and sums are held in 32 bits.  Column sums
// (weights, and a gate shared by rows) are kept in registers over a block's
// consecutive rows, written out once a block (a gate's as soon as its rows end
// where a block has whole runs of them), and added in the blocks' order by a
// second kernel, so that results do not depend on scheduling.
//
// Measured, forward and gradient: 16384 x 1024 fp32 LayerNorm with a shared gate
// 58 + 102 us (4.2 TB/s over both), 65535 x 2048 bf16 RMS with a sigmoid gate
// 224 + 459 us (5.1 TB/s), gradient 500 with one gate row for all; 65536 x 1023 bf16, whose
// rows allow single elements only, 689 us (2.0 TB/s).
//
// Wide rows: the gradient's sums and row do not fit the registers.  Spilled stores
// a thread: 224 to 752 bytes with 16 elements a thread (6145 to 8192 wide, single
// elements from 4097), 3 to 5.5 KB with 32 (beyond), up to 272 with 768 threads
// (4097 to 6144; none for 16-bit RMS rows without a shared gate).  RMS in bf16:
// 16384 x 4096 95 + 232 us (4.3 TB/s over both), 8192 x 8192 107 + 332 (3.1), 4096
// x 16384 193 + 1280 (0.9), 2048 x 32768 220 + 1650 (0.7).  fp32 RMS rows of 7172 to
// 8192 read their weights again for each row: 8192 x 7168 170 us forward, 8192 x
// 8192 195 (5.5 TB/s both).
#include <algorithm>

#include "ops_common.cuh"

namespace adops {

struct NormArgs {
  const void *x, *z, *gate, *dh, *dy;
  long long ldx, ldz, ldg, lddh, lddy;
  const void *wa, *ba, *wb, *bb;
  int wtype;
  void *h, *y, *dx, *dz, *dgate;
  long long ldh, ldy, lddx, lddz, lddg;
  float* stats;  // [rows][4]: mean and reciprocal deviation of z, then of h
  float* part;   // [blocks][sums][width]
  long long rows, rows_per_gate;
  // gradient: rows of a run (those of a shared gate, else all), blocks that share
  // a run (0: a block has whole runs), rows of a block
  long long run, blocks_per_run, rows_per_block;
  int width, sigmoid, layer;
  int staged;  // bytes of weights and biases kept in shared memory
  float scale, eps;
};

// rows fit 32 bits: a short division
__device__ __forceinline__ long long gate_row(const NormArgs& a, long long row) {
  return a.rows_per_gate == 1 ? row : static_cast<unsigned>(row) / static_cast<unsigned>(a.rows_per_gate);
}

// Offset of a row: both factors fit 32 bits, one instruction.
__device__ __forceinline__ unsigned long long at(long long row, long long ld) {
  return static_cast<unsigned long long>(static_cast<unsigned>(row)) * static_cast<unsigned>(ld);
}

// 32-bit elements: to 2 units in the last place.  16-bit ones: to 2 + 1.2 |x|, at
// most 107 where the result is neither 0 nor infinite, which is 2^-17 of it and
// far below their own rounding.
template <typename T>
__device__ __forceinline__ float exponential(float x) {
  return sizeof(T) == 4 ? expf(x) : __expf(x);
}
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
  return __fdividef(1.0f, 1.0f + exponential<T>(-g));
}
// With its slope: shares 1 / (1 + e) and e / (1 + e), without a difference that
// could cancel; the sigmoid is one of them by g's sign, its slope their product.
template <typename T>
__device__ __forceinline__ float sigmoid(float g, float& slope) {
  const float e = exponential<T>(-fabsf(g)), large = __fdividef(1.0f, 1.0f + e), small = e * large;
  slope = large * small;
  return g >= 0.0f ? large : small;
}

// Sums over the block of N values a thread; every thread gets them.  `buf`
// alternates between two areas so that one barrier a call is enough.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* smem, int& flip) {
  static_assert(N == 1 || N == 2, "");
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  float s;
  if (N == 1) {
    s = warp_sum(v[0]);
  } else {  // each half of the warp adds up one of the two
    const bool up = lane & 16;
    s = (up ? v[N - 1] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[N - 1], 16);
#pragma unroll
    for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  float* buf = smem + flip * (2 * 32);
  flip ^= 1;
  if ((lane & (N == 1 ? 31 : 15)) == 0) buf[lane * 2 + (threadIdx.x >> 5)] = s;  // the second value from 32 on
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = 0.0f;
  for (int w = 0; w < warps; w += 4) {  // areas past the warps hold zeros
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float4 q = *reinterpret_cast<const float4*>(buf + k * 32 + w);
      v[k] += (q.x + q.y) + (q.z + q.w);
    }
  }
}

// A thread's share of a row; zeros past the width.
template <typename T, int V, int NV>
struct Raw {
  Vec<T, V> q[NV];
  __device__ __forceinline__ void load(const T* p, int width) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (n * blockDim.x + threadIdx.x) * V;
      if (c < width) {
        q[n] = load_vec<T, V>(p + c);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) q[n].v[j] = from_float<T>(0.0f);
      }
    }
  }
  __device__ __forceinline__ void floats(float (&o)[NV * V]) const {
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int j = 0; j < V; ++j) o[n * V + j] = to_float(q[n].v[j]);
  }
};
template <typename T, int V, int NV>
__device__ __forceinline__ void store_row(T* p, int width, const float (&o)[NV * V]) {
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * blockDim.x + threadIdx.x) * V;
    if (c < width) {
      Vec<T, V> r;
      round_to<T, V>(o + n * V, r);
      store_vec<T, V>(p + c, r);
    }
  }
}
template <int V, int NV>
__device__ __forceinline__ void store_sums(float* p, int width, const float (&o)[NV * V]) {
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * blockDim.x + threadIdx.x) * V;
    if (c < width) {
      constexpr int W = V < 4 ? V : 4;
#pragma unroll
      for (int k = 0; k < V; k += W) {
        Vec<float, W> r;
#pragma unroll
        for (int j = 0; j < W; ++j) r.v[j] = o[n * V + k + j];
        store_vec<float, W>(p + c + k, r);
      }
    }
  }
}
// A weight or bias vector in 32 bits, whichever of its two types it is held in.
template <typename T, int V, int NV>
__device__ __forceinline__ void load_weights(const void* p, int wtype, int width, float (&o)[NV * V]) {
  if (wtype == AD_F32) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int c = (n * blockDim.x + threadIdx.x) * V;
      constexpr int W = V < 4 ? V : 4;
#pragma unroll
      for (int k = 0; k < V; k += W) {
        Vec<float, W> r = {};
        if (c < width) r = load_vec<float, W>(static_cast<const float*>(p) + c + k);
#pragma unroll
        for (int j = 0; j < W; ++j) o[n * V + k + j] = r.v[j];
      }
    }
  } else {
    Raw<T, V, NV> r;
    r.load(static_cast<const T*>(p), width);
    r.floats(o);
  }
}

// The four vectors in shared memory for the block's life: loads of them between
// the rows' would queue behind those for a microsecond each.  Quads of a vector's
// elements lie in planes, so that neighbouring threads read neighbouring words.
enum { W_WA = 0, W_WB = 1, W_BA = 2, W_BB = 3 };
template <int V>
__host__ __device__ constexpr int quad() {
  return V < 4 ? V : 4;
}
template <typename T, int V, int NV, int N>
struct Weights {  // the first N of them
  const NormArgs& a;
  float* sm;
  int vecs;
  __device__ __forceinline__ Weights(const NormArgs& args, float* shared) : a(args), sm(shared) {
    vecs = (a.width + V - 1) / V;
    if (!a.staged) return;
    const void* from[4] = {a.wa, a.wb, a.ba, a.bb};
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (!from[k]) continue;
      float o[NV * V];
      load_weights<T, V, NV>(from[k], a.wtype, a.width, o);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int v = n * blockDim.x + threadIdx.x;
        if (v < vecs) {
#pragma unroll
          for (int j = 0; j < V; ++j) sm[((k * (V / quad<V>()) + j / 4) * vecs + v) * quad<V>() + j % 4] = o[n * V + j];
        }
      }
    }
    // a thread reads what it wrote: no barrier
  }
  __device__ __forceinline__ void get(int k, float (&o)[NV * V]) const {
    if (!a.staged) {
      load_weights<T, V, NV>(k == W_WA ? a.wa : k == W_WB ? a.wb : k == W_BA ? a.ba : a.bb, a.wtype, a.width, o);
      return;
    }
    constexpr int Q = quad<V>();
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int v = n * blockDim.x + threadIdx.x;
#pragma unroll
      for (int p = 0; p < V / Q; ++p) {
        Vec<float, Q> r = {};
        if (v < vecs) r = load_vec<float, Q>(sm + ((k * (V / Q) + p) * vecs + v) * Q);
#pragma unroll
        for (int j = 0; j < Q; ++j) o[n * V + p * Q + j] = r.v[j];
      }
    }
  }
};

// Mean and reciprocal deviation of a row held by the block; elements past the
// width are zero on entry.
template <int V, int NV>
__device__ __forceinline__ void moments(const float (&v)[NV * V], bool layer, int width, float eps, float* smem, int& flip,
                                        float& mean, float& r) {
  float s[1] = {0.0f};
  mean = 0.0f;
  if (layer) {
#pragma unroll
    for (int i = 0; i < NV * V; ++i) s[0] += v[i];
    block_sum<1>(s, smem, flip);
    mean = s[0] / width;
    s[0] = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if ((n * blockDim.x + threadIdx.x) * V < width) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = v[n * V + j] - mean;
          s[0] = fmaf(d, d, s[0]);
        }
      }
  } else {
#pragma unroll
    for (int i = 0; i < NV * V; ++i) s[0] = fmaf(v[i], v[i], s[0]);
  }
  block_sum<1>(s, smem, flip);
  r = 1.0f / sqrtf(s[0] / width + eps);
}

// The S rows to come of K operands, brought into shared memory while earlier ones
// are worked on.  A thread copies and reads its own vectors only, so there is
// nothing to wait for but its own copies.  (Kept in registers instead, the next
// row was waited for all the same: 888 us for 65535 x 2048 bf16 gradients.)
// Single elements (V = 1) are too small for such copies and rows of over 8192
// elements too large: they are read when due.
template <typename T, int V, int NV, int K, int S>
struct Ahead {
  static constexpr bool DIRECT = V == 1 || V * NV > 16;
  unsigned base;
  int width;
  __device__ __forceinline__ Ahead(void* shared, int w)
      : base(static_cast<unsigned>(__cvta_generic_to_shared(shared))), width(w) {}
  __device__ __forceinline__ unsigned slot(int stage, int k, int n) const {
    return base + (((stage * K + k) * NV + n) * blockDim.x + threadIdx.x) * 16;
  }
  __device__ __forceinline__ void copy(int stage, int k, const T* row) const {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = (n * blockDim.x + threadIdx.x) * V;
        if (c < width) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot(stage, k, n)), "l"(row + c));
      }
    }
  }
  __device__ __forceinline__ void commit() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // The oldest row's copies are done.
  __device__ __forceinline__ void wait() const { asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory"); }
  __device__ __forceinline__ void read(int stage, int k, const T* row, float (&o)[NV * V]) const {
    if constexpr (DIRECT) {
      Raw<T, V, NV> r;
      r.load(row, width);
      r.floats(o);
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if ((n * blockDim.x + threadIdx.x) * V < width)
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                       : "r"(slot(stage, k, n))
                       : "memory");
        unpack<T>(q, o + n * V);
      }
    }
  }
  static int bytes(int threads) { return DIRECT ? 0 : S * K * NV * threads * 16; }
};

constexpr int FORWARD_ROWS = 2;
// Whether the gradient's registers are held down so that 768 threads fit a
// multiprocessor rather than 512: without means and biases, for 16-bit elements,
// vectors then spill nothing (65535 x 2048 bf16: 723 -> 671 us both directions), or
// 88 bytes with a shared gate and up to 104 where elements are single; else the sums
// spill more (16384 x 1024 fp32 LayerNorm: 163 -> 211 us).
template <typename T, bool GEN>
__host__ __device__ constexpr bool slim() {
  return sizeof(T) == 2 && !GEN;
}
// Rows that the gradient copies ahead: what the threads' shares of five operands
// leave room for.
template <typename T, int V, int NV, int MAXT, bool GEN>
__host__ __device__ constexpr int grad_rows() {
  return sizeof(T) == 4 ? (MAXT == 768 || V * NV > 8 ? 1 : 2) : (MAXT == 768 || V * NV > 8 || slim<T, GEN>() ? 2 : 4);
}

// GEN: with a LayerNorm's means or with biases; without it both are known to be
// absent.  MAXT: threads a block may have; with 256 of them several blocks share
// a multiprocessor.
template <typename T, int V, int NV, int MAXT, bool GEN>
__global__ void __launch_bounds__(MAXT, MAXT == 256 ? (V * NV <= 8 ? 4 : 2) : 1)
    norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ __align__(16) float smem[2 * 2 * 32];
  for (int i = threadIdx.x; i < 2 * 2 * 32; i += blockDim.x) smem[i] = 0.0f;
  __syncthreads();
  extern __shared__ __align__(16) float staged[];
  int flip = 0;
  constexpr int E = NV * V;
  const Ahead<T, V, NV, 3, FORWARD_ROWS> ahead(staged + a.staged / 4, a.width);
  auto pz = [&](long long row) { return static_cast<const T*>(a.z) + at(row, a.ldz); };
  auto px = [&](long long row) { return static_cast<const T*>(a.x) + at(row, a.ldx); };
  auto pg = [&](long long row) { return static_cast<const T*>(a.gate) + at(gate_row(a, row), a.ldg); };
  auto fetch = [&](int stage, long long row) {
    if (row < a.rows) {
      ahead.copy(stage, 0, pz(row));
      ahead.copy(stage, 1, px(row));
      if (a.gate) ahead.copy(stage, 2, pg(row));
    }
    ahead.commit();
  };
  for (int k = 0; k < FORWARD_ROWS; ++k) fetch(k, blockIdx.x + static_cast<long long>(k) * gridDim.x);
  const Weights<T, V, NV, GEN ? 4 : 2> weights(a, staged);
  int stage = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float x[E], u[E], act[E], w[E];
    ahead.wait();
    ahead.read(stage, 0, pz(row), u);
    ahead.read(stage, 1, px(row), x);
    if (a.gate) ahead.read(stage, 2, pg(row), act);
    fetch(stage, row + static_cast<long long>(FORWARD_ROWS) * gridDim.x);
    stage = stage + 1 == FORWARD_ROWS ? 0 : stage + 1;
    float mz = 0.0f, rz = 1.0f, mh = 0.0f, rh = 1.0f;
    if (a.wa) {
      moments<V, NV>(u, GEN && a.layer, a.width, a.eps, smem, flip, mz, rz);
      weights.get(W_WA, w);
#pragma unroll
      for (int i = 0; i < E; ++i) u[i] = (GEN ? u[i] - mz : u[i]) * rz * w[i];
      if (GEN && a.ba) {
        weights.get(W_BA, w);
#pragma unroll
        for (int i = 0; i < E; ++i) u[i] += w[i];
      }
    }
    if (a.gate) {
      if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < E; ++i) act[i] = sigmoid<T>(act[i]);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) u[i] *= act[i];
    }
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = fmaf(a.scale, x[i], u[i]);
    store_row<T, V, NV>(static_cast<T*>(a.h) + at(row, a.ldh), a.width, x);
    if (a.wb) {
      moments<V, NV>(x, GEN && a.layer, a.width, a.eps, smem, flip, mh, rh);
      weights.get(W_WB, w);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = (GEN ? x[i] - mh : x[i]) * rh * w[i];
      if (GEN && a.bb) {
        weights.get(W_BB, w);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] += w[i];
      }
      store_row<T, V, NV>(static_cast<T*>(a.y) + at(row, a.ldy), a.width, x);
    }
    if (threadIdx.x == 0)
      reinterpret_cast<float4*>(a.stats)[row] = make_float4(mz, rz, mh, rh);
  }
}

// Sums of one block's rows, in this order; the finishing kernel reads them so.
enum { SUM_WA = 0, SUM_WB = 1, SUM_BA = 2, SUM_BB = 3, SUM_GATE = 4, SUMS = 5 };

// SHARED: the gate's rows are shared, its gradient is a sum over rows.
template <typename T, int V, int NV, int MAXT, bool GEN, bool SHARED>
__global__ void __launch_bounds__(MAXT, MAXT != 256 || V * NV > 8 ? 1 : slim<T, GEN>() ? 3 : 2) norm_grad_kernel(const __grid_constant__ NormArgs a) {
  __shared__ __align__(16) float smem[2 * 2 * 32];
  for (int i = threadIdx.x; i < 2 * 2 * 32; i += blockDim.x) smem[i] = 0.0f;
  __syncthreads();
  extern __shared__ __align__(16) float staged[];
  int flip = 0;
  constexpr int E = NV * V;
  float swa[E], swb[E], sba[E], sbb[E], sg[E];
#pragma unroll
  for (int i = 0; i < E; ++i) swa[i] = swb[i] = sba[i] = sbb[i] = sg[i] = 0.0f;
  long long r0 = blockIdx.x * a.rows_per_block, r1 = min(a.rows, r0 + a.rows_per_block);
  const bool whole = a.blocks_per_run == 0;
  if (!whole) {
    const long long run = blockIdx.x / a.blocks_per_run;
    r0 = run * a.run + (blockIdx.x - run * a.blocks_per_run) * a.rows_per_block;
    r1 = min((run + 1) * a.run, r0 + a.rows_per_block);
  }
  long long left = a.run;  // rows of the run to come
  const bool layer = GEN && a.layer;
  const float inv = 1.0f / a.width;
  constexpr int S = grad_rows<T, V, NV, MAXT, GEN>();
  const Ahead<T, V, NV, 5, S> ahead(staged + a.staged / 4, a.width);
  auto pz = [&](long long row) { return static_cast<const T*>(a.z) + at(row, a.ldz); };
  auto px = [&](long long row) { return static_cast<const T*>(a.x) + at(row, a.ldx); };
  auto pg = [&](long long row) { return static_cast<const T*>(a.gate) + at(gate_row(a, row), a.ldg); };
  auto pdh = [&](long long row) { return static_cast<const T*>(a.dh) + at(row, a.lddh); };
  auto pdy = [&](long long row) { return static_cast<const T*>(a.dy) + at(row, a.lddy); };
  auto fetch = [&](int stage, long long row) {
    if (row < r1) {
      ahead.copy(stage, 0, pz(row));
      if (a.gate) ahead.copy(stage, 1, pg(row));
      if (a.wb) {
        ahead.copy(stage, 2, px(row));
        ahead.copy(stage, 3, pdy(row));
      }
      ahead.copy(stage, 4, pdh(row));
    }
    ahead.commit();
  };
  auto slopes = [&](long long row) {  // of the row's gate, onto its sums
    if (!a.sigmoid) return;
    Raw<T, V, NV> g;
    g.load(pg(row), a.width);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float slope;
      sigmoid<T>(to_float(g.q[i / V].v[i % V]), slope);
      sg[i] *= slope;
    }
  };
  for (int k = 0; k < S; ++k) fetch(k, r0 + k);
  const Weights<T, V, NV, GEN ? 3 : 2> weights(a, staged);
  int stage = 0;
  float4 rst = r0 < r1 ? reinterpret_cast<const float4*>(a.stats)[r0] : make_float4(0, 0, 0, 0);
  for (long long row = r0; row < r1; ++row) {
    const float4 st = rst;
    const float mz = st.x, rz = st.y, mh = st.z, rh = st.w;
    float nz[E], u[E], act[E], t[E], w[E], nh[E], d[E];
    ahead.wait();
    ahead.read(stage, 0, pz(row), nz);
    ahead.read(stage, 4, pdh(row), t);
    if (a.wb) {
      ahead.read(stage, 2, px(row), nh);
      ahead.read(stage, 3, pdy(row), d);
    }
    if (a.gate) {
      ahead.read(stage, 1, pg(row), act);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) act[i] = 1.0f;
    }
    fetch(stage, row + S);
    stage = stage + 1 == S ? 0 : stage + 1;
    if (row + 1 < r1) rst = reinterpret_cast<const float4*>(a.stats)[row + 1];
#pragma unroll
    for (int i = 0; i < E; ++i) u[i] = nz[i];
    if (a.wa) {
      weights.get(W_WA, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        nz[i] = (GEN ? nz[i] - mz : nz[i]) * rz;
        u[i] = nz[i] * w[i];
      }
      if (GEN && a.ba) {
        weights.get(W_BA, w);
#pragma unroll
        for (int i = 0; i < E; ++i) u[i] += w[i];
      }
    }
    // h in nh; from here on u is the gate's part of its own gradient (but for the
    // slope of a shared gate, which its sum is multiplied with)
    if (a.sigmoid && a.gate) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        float slope = 1.0f;
        act[i] = SHARED ? sigmoid<T>(act[i]) : sigmoid<T>(act[i], slope);
        nh[i] = a.wb ? fmaf(a.scale, nh[i], act[i] * u[i]) : 0.0f;
        u[i] *= slope;
      }
    } else if (a.wb) {
#pragma unroll
      for (int i = 0; i < E; ++i) nh[i] = fmaf(a.scale, nh[i], act[i] * u[i]);
    }
    if (a.wb) {
      float q[2] = {0.0f, 0.0f};
      weights.get(W_WB, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        nh[i] = (GEN ? nh[i] - mh : nh[i]) * rh;
        swb[i] = fmaf(d[i], nh[i], swb[i]);
        if (GEN) sbb[i] += d[i];
        d[i] *= w[i];
        q[0] = fmaf(d[i], nh[i], q[0]);
        if (layer) q[1] += d[i];
      }
      if (GEN)
        block_sum<2>(q, smem, flip);
      else
        block_sum<1>(reinterpret_cast<float(&)[1]>(q), smem, flip);
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] += rh * (d[i] - nh[i] * (q[0] * inv) - (layer ? q[1] * inv : 0.0f));
    }
    float o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = a.scale * t[i];
    store_row<T, V, NV>(static_cast<T*>(a.dx) + at(row, a.lddx), a.width, o);
    if (a.gate) {
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = t[i] * u[i];
      if (SHARED) {
#pragma unroll
        for (int i = 0; i < E; ++i) sg[i] += o[i];
      }
      if (!SHARED) store_row<T, V, NV>(static_cast<T*>(a.dgate) + at(row, a.lddg), a.width, o);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) t[i] *= act[i];
    if (a.wa) {
      float q[2] = {0.0f, 0.0f};
      weights.get(W_WA, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        swa[i] = fmaf(t[i], nz[i], swa[i]);
        if (GEN) sba[i] += t[i];
        t[i] *= w[i];
        q[0] = fmaf(t[i], nz[i], q[0]);
        if (layer) q[1] += t[i];
      }
      if (GEN)
        block_sum<2>(q, smem, flip);
      else
        block_sum<1>(reinterpret_cast<float(&)[1]>(q), smem, flip);
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] = rz * (t[i] - nz[i] * (q[0] * inv) - (layer ? q[1] * inv : 0.0f));
    }
    store_row<T, V, NV>(static_cast<T*>(a.dz) + at(row, a.lddz), a.width, t);
    if (SHARED && whole && --left == 0) {
      slopes(row);
      store_row<T, V, NV>(static_cast<T*>(a.dgate) + row / a.run * a.lddg, a.width, sg);
#pragma unroll
      for (int i = 0; i < E; ++i) sg[i] = 0.0f;
      left = a.run;
    }
  }
  if (SHARED && !whole) slopes(r0);
  float* part = a.part + static_cast<long long>(blockIdx.x) * SUMS * a.width;
  store_sums<V, NV>(part + SUM_WA * a.width, a.width, swa);
  store_sums<V, NV>(part + SUM_WB * a.width, a.width, swb);
  if (GEN) {
    store_sums<V, NV>(part + SUM_BA * a.width, a.width, sba);
    store_sums<V, NV>(part + SUM_BB * a.width, a.width, sbb);
  }
  if (SHARED && !whole) store_sums<V, NV>(part + SUM_GATE * a.width, a.width, sg);
}

// `ahead`: bytes of the rows to come; `blocks` 0: as many as are resident at a
// time, each with every so-many-th row.
template <auto KERNEL>
cudaError_t run_norm(NormArgs a, int vectors, int v, int ahead, unsigned blocks, int sms, int threads, cudaStream_t s) {
  a.staged = (vectors * 4 * ((a.width + v - 1) / v * v) + 15) / 16 * 16;
  int room = 0;
  cudaError_t e = shared_room<KERNEL>(&room);
  if (e != cudaSuccess) return e;
  // rows to come go before weights, which are read again for each row where both do not fit
  if (a.staged > 64 * 1024 || a.staged + ahead > room) a.staged = 0;
  const int bytes = a.staged + ahead;
  if (!blocks && a.rows <= sms) {
    blocks = static_cast<unsigned>(a.rows);
  } else if (!blocks) {
    int per = 1;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, KERNEL, threads, bytes);
    if (e != cudaSuccess) return e;
    blocks = static_cast<unsigned>(std::min(a.rows, 1ll * std::max(per, 1) * sms));
  }
  return launch<KERNEL>(blocks, threads, bytes, s, a);
}

// GRAD: which of the two directions; each is built for the sizes below that take it.
template <bool GRAD, typename T, int V, int NV, int MAXT>
cudaError_t start_norm(const NormArgs& a, bool gen, unsigned blocks, int sms, int threads, cudaStream_t s) {
  if constexpr (!GRAD) {
    const int f = Ahead<T, V, NV, 3, FORWARD_ROWS>::bytes(threads);
    return gen ? run_norm<norm_kernel<T, V, NV, MAXT, true>>(a, 4, V, f, 0, sms, threads, s)
               : run_norm<norm_kernel<T, V, NV, MAXT, false>>(a, 2, V, f, 0, sms, threads, s);
  } else {
    const bool shared = a.gate && a.rows_per_gate > 1;
    const int g = gen ? Ahead<T, V, NV, 5, grad_rows<T, V, NV, MAXT, true>()>::bytes(threads)
                      : Ahead<T, V, NV, 5, grad_rows<T, V, NV, MAXT, false>()>::bytes(threads);
    if (gen)
      return shared ? run_norm<norm_grad_kernel<T, V, NV, MAXT, true, true>>(a, 3, V, g, blocks, sms, threads, s)
                    : run_norm<norm_grad_kernel<T, V, NV, MAXT, true, false>>(a, 3, V, g, blocks, sms, threads, s);
    return shared ? run_norm<norm_grad_kernel<T, V, NV, MAXT, false, true>>(a, 2, V, g, blocks, sms, threads, s)
                  : run_norm<norm_grad_kernel<T, V, NV, MAXT, false, false>>(a, 2, V, g, blocks, sms, threads, s);
  }
}

// Eight elements of a row to a thread while 512 threads are enough for it (768
// in the gradient, whose sums for 16 do not fit a thread's registers), 16 while
// 512 are, else 32 to each of up to 1024; 16 in the forward pass of rows
// wide enough for two warps, because what a row costs each warp besides its
// elements (two sums over the block, addresses) is as much as eight elements do.  `vec`: all addresses and sizes
// allow 16-byte vectors; single elements else.
template <typename T>
cudaError_t start_norm_typed(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, int sms, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  auto threads_for = [&](int per) { return ((a.width + per - 1) / per + 31) / 32 * 32; };
  const int t8 = threads_for(8), t16 = threads_for(16), t32 = threads_for(32);
  if (!grad) {
    if (vec) {
      if (t16 < 64) return start_norm<false, T, V, 8 / V, 256>(a, gen, blocks, sms, t8, s);
      if (t16 <= 256) return start_norm<false, T, V, 16 / V, 256>(a, gen, blocks, sms, t16, s);
      if (t16 <= 512) return start_norm<false, T, V, 16 / V, 512>(a, gen, blocks, sms, t16, s);
      return start_norm<false, T, V, 32 / V, 1024>(a, gen, blocks, sms, t32, s);
    }
    if (t8 <= 256) return start_norm<false, T, 1, 8, 256>(a, gen, blocks, sms, t8, s);
    if (t8 <= 512) return start_norm<false, T, 1, 8, 512>(a, gen, blocks, sms, t8, s);
    if (t16 <= 512) return start_norm<false, T, 1, 16, 512>(a, gen, blocks, sms, t16, s);
    return start_norm<false, T, 1, 32, 1024>(a, gen, blocks, sms, t32, s);
  }
  if (vec) {
    if (t8 <= 256) return start_norm<true, T, V, 8 / V, 256>(a, gen, blocks, sms, t8, s);
    if (t8 <= 512) return start_norm<true, T, V, 8 / V, 512>(a, gen, blocks, sms, t8, s);
    if (t8 <= 768) return start_norm<true, T, V, 8 / V, 768>(a, gen, blocks, sms, t8, s);
    if (t16 <= 512) return start_norm<true, T, V, 16 / V, 512>(a, gen, blocks, sms, t16, s);
    return start_norm<true, T, V, 32 / V, 1024>(a, gen, blocks, sms, t32, s);
  }
  if (t8 <= 256) return start_norm<true, T, 1, 8, 256>(a, gen, blocks, sms, t8, s);
  if (t8 <= 512) return start_norm<true, T, 1, 8, 512>(a, gen, blocks, sms, t8, s);
  if (t16 <= 512) return start_norm<true, T, 1, 16, 512>(a, gen, blocks, sms, t16, s);
  return start_norm<true, T, 1, 32, 1024>(a, gen, blocks, sms, t32, s);
}

cudaError_t start_norm_f32(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, int sms, cudaStream_t s);
cudaError_t start_norm_bf16(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, int sms, cudaStream_t s);
cudaError_t start_norm_f16(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, int sms, cudaStream_t s);

}  // namespace adops

#endif
