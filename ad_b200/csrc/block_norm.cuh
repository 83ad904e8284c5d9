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
  float scale, eps;
};

__device__ __forceinline__ float act_of(float g, int sigmoid) {
  return sigmoid ? 1.0f / (1.0f + __expf(-g)) : g;
}

// Sums over the block of N values a thread; every thread gets them.  `buf`
// alternates between two areas so that one barrier a call is enough.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* smem, int& flip) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = warp_sum(v[k]);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return;
  float* buf = smem + flip * (2 * 32);
  flip ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) buf[k * 32 + (threadIdx.x >> 5)] = v[k];
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = warp_sum(lane < warps ? buf[k * 32 + lane] : 0.0f);
}

template <typename T, int V, int NV>
__device__ __forceinline__ void load_row(const T* p, int width, float (&o)[NV * V]) {
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * blockDim.x + threadIdx.x) * V;
    if (c < width) {
      const Vec<T, V> r = load_vec<T, V>(p + c);
#pragma unroll
      for (int j = 0; j < V; ++j) o[n * V + j] = to_float(r.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) o[n * V + j] = 0.0f;
    }
  }
}
template <typename T, int V, int NV>
__device__ __forceinline__ void store_row(T* p, int width, const float (&o)[NV * V]) {
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * blockDim.x + threadIdx.x) * V;
    if (c < width) {
      Vec<T, V> r;
#pragma unroll
      for (int j = 0; j < V; ++j) r.v[j] = from_float<T>(o[n * V + j]);
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
    load_row<T, V, NV>(static_cast<const T*>(p), width, o);
  }
}

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

// GEN: with a LayerNorm's means or with biases; without it both are known to be
// absent.  MAXT: threads a block may have; with 256 of them several blocks share
// a multiprocessor.
template <typename T, int V, int NV, int MAXT, bool GEN>
__global__ void __launch_bounds__(MAXT, MAXT == 256 ? 4 : 1) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float smem[2 * 2 * 32];
  int flip = 0;
  constexpr int E = NV * V;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float x[E], u[E], w[E];
    load_row<T, V, NV>(static_cast<const T*>(a.x) + row * a.ldx, a.width, x);
    load_row<T, V, NV>(static_cast<const T*>(a.z) + row * a.ldz, a.width, u);
    float mz = 0.0f, rz = 1.0f, mh = 0.0f, rh = 1.0f;
    if (a.wa) {
      moments<V, NV>(u, GEN && a.layer, a.width, a.eps, smem, flip, mz, rz);
      load_weights<T, V, NV>(a.wa, a.wtype, a.width, w);
#pragma unroll
      for (int i = 0; i < E; ++i) u[i] = (u[i] - mz) * rz * w[i];
      if (GEN && a.ba) {
        load_weights<T, V, NV>(a.ba, a.wtype, a.width, w);
#pragma unroll
        for (int i = 0; i < E; ++i) u[i] += w[i];
      }
    }
    if (a.gate) {
      load_row<T, V, NV>(static_cast<const T*>(a.gate) + row / a.rows_per_gate * a.ldg, a.width, w);
#pragma unroll
      for (int i = 0; i < E; ++i) u[i] *= act_of(w[i], a.sigmoid);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = fmaf(a.scale, x[i], u[i]);
    store_row<T, V, NV>(static_cast<T*>(a.h) + row * a.ldh, a.width, x);
    if (a.wb) {
      moments<V, NV>(x, GEN && a.layer, a.width, a.eps, smem, flip, mh, rh);
      load_weights<T, V, NV>(a.wb, a.wtype, a.width, w);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = (x[i] - mh) * rh * w[i];
      if (GEN && a.bb) {
        load_weights<T, V, NV>(a.bb, a.wtype, a.width, w);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] += w[i];
      }
      store_row<T, V, NV>(static_cast<T*>(a.y) + row * a.ldy, a.width, x);
    }
    if (threadIdx.x == 0)
      reinterpret_cast<float4*>(a.stats)[row] = make_float4(mz, rz, mh, rh);
  }
}

// Sums of one block's rows, in this order; the finishing kernel reads them so.
enum { SUM_WA = 0, SUM_WB = 1, SUM_BA = 2, SUM_BB = 3, SUM_GATE = 4, SUMS = 5 };

// SHARED: the gate's rows are shared, its gradient is a sum over rows.
template <typename T, int V, int NV, int MAXT, bool GEN, bool SHARED>
__global__ void __launch_bounds__(MAXT, MAXT == 256 ? 2 : 1) norm_grad_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float smem[2 * 2 * 32];
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
  for (long long row = r0; row < r1; ++row) {
    const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
    const float mz = st.x, rz = st.y, mh = st.z, rh = st.w;
    float nz[E], u[E], act[E], slope[E], t[E], w[E];
    load_row<T, V, NV>(static_cast<const T*>(a.z) + row * a.ldz, a.width, nz);
    if (a.gate) {
      load_row<T, V, NV>(static_cast<const T*>(a.gate) + row / a.rows_per_gate * a.ldg, a.width, act);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        act[i] = act_of(act[i], a.sigmoid);
        slope[i] = a.sigmoid ? act[i] * (1.0f - act[i]) : 1.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) act[i] = slope[i] = 1.0f;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) u[i] = nz[i];
    if (a.wa) {
      load_weights<T, V, NV>(a.wa, a.wtype, a.width, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        nz[i] = (nz[i] - mz) * rz;
        u[i] = nz[i] * w[i];
      }
      if (GEN && a.ba) {
        load_weights<T, V, NV>(a.ba, a.wtype, a.width, w);
#pragma unroll
        for (int i = 0; i < E; ++i) u[i] += w[i];
      }
    }
    load_row<T, V, NV>(static_cast<const T*>(a.dh) + row * a.lddh, a.width, t);
    if (a.wb) {
      float nh[E], d[E], q[2] = {0.0f, 0.0f};
      load_row<T, V, NV>(static_cast<const T*>(a.x) + row * a.ldx, a.width, nh);
      load_row<T, V, NV>(static_cast<const T*>(a.dy) + row * a.lddy, a.width, d);
      load_weights<T, V, NV>(a.wb, a.wtype, a.width, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        nh[i] = (fmaf(a.scale, nh[i], act[i] * u[i]) - mh) * rh;
        swb[i] = fmaf(d[i], nh[i], swb[i]);
        if (GEN) sbb[i] += d[i];
        d[i] *= w[i];
        q[0] = fmaf(d[i], nh[i], q[0]);
        if (layer) q[1] += d[i];
      }
      block_sum<2>(q, smem, flip);
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] += rh * (d[i] - nh[i] * (q[0] * inv) - (layer ? q[1] * inv : 0.0f));
    }
    float o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = a.scale * t[i];
    store_row<T, V, NV>(static_cast<T*>(a.dx) + row * a.lddx, a.width, o);
    if (a.gate) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        o[i] = t[i] * u[i] * slope[i];
        if (SHARED) sg[i] += o[i];
      }
      if (!SHARED) store_row<T, V, NV>(static_cast<T*>(a.dgate) + row * a.lddg, a.width, o);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) t[i] *= act[i];
    if (a.wa) {
      float q[2] = {0.0f, 0.0f};
      load_weights<T, V, NV>(a.wa, a.wtype, a.width, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        swa[i] = fmaf(t[i], nz[i], swa[i]);
        if (GEN) sba[i] += t[i];
        t[i] *= w[i];
        q[0] = fmaf(t[i], nz[i], q[0]);
        if (layer) q[1] += t[i];
      }
      block_sum<2>(q, smem, flip);
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] = rz * (t[i] - nz[i] * (q[0] * inv) - (layer ? q[1] * inv : 0.0f));
    }
    store_row<T, V, NV>(static_cast<T*>(a.dz) + row * a.lddz, a.width, t);
    if (SHARED && whole && --left == 0) {
      store_row<T, V, NV>(static_cast<T*>(a.dgate) + row / a.run * a.lddg, a.width, sg);
#pragma unroll
      for (int i = 0; i < E; ++i) sg[i] = 0.0f;
      left = a.run;
    }
  }
  float* part = a.part + static_cast<long long>(blockIdx.x) * SUMS * a.width;
  store_sums<V, NV>(part + SUM_WA * a.width, a.width, swa);
  store_sums<V, NV>(part + SUM_WB * a.width, a.width, swb);
  if (GEN) {
    store_sums<V, NV>(part + SUM_BA * a.width, a.width, sba);
    store_sums<V, NV>(part + SUM_BB * a.width, a.width, sbb);
  }
  if (SHARED && !whole) store_sums<V, NV>(part + SUM_GATE * a.width, a.width, sg);
}

template <typename T, int V, int NV, int MAXT>
cudaError_t start_norm(const NormArgs& a, bool grad, bool gen, unsigned blocks, int threads, cudaStream_t s) {
  const bool shared = a.gate && a.rows_per_gate > 1;
  if (!grad) {
    if (gen)
      norm_kernel<T, V, NV, MAXT, true><<<blocks, threads, 0, s>>>(a);
    else
      norm_kernel<T, V, NV, MAXT, false><<<blocks, threads, 0, s>>>(a);
  } else if (gen) {
    if (shared)
      norm_grad_kernel<T, V, NV, MAXT, true, true><<<blocks, threads, 0, s>>>(a);
    else
      norm_grad_kernel<T, V, NV, MAXT, true, false><<<blocks, threads, 0, s>>>(a);
  } else {
    if (shared)
      norm_grad_kernel<T, V, NV, MAXT, false, true><<<blocks, threads, 0, s>>>(a);
    else
      norm_grad_kernel<T, V, NV, MAXT, false, false><<<blocks, threads, 0, s>>>(a);
  }
  return cudaGetLastError();
}

// Eight elements a thread while the row fits 1024 threads so, else 32.  `vec`:
// all addresses and sizes allow 16-byte vectors.
template <typename T>
cudaError_t start_norm_typed(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  const int per = a.width <= 8192 ? 8 : 32;
  const int threads = ((a.width + per - 1) / per + 31) / 32 * 32;
  if (per == 8) {
    if (threads <= 256)
      return vec ? start_norm<T, V, 8 / V, 256>(a, grad, gen, blocks, threads, s)
                 : start_norm<T, 1, 8, 256>(a, grad, gen, blocks, threads, s);
    if (threads <= 512)
      return vec ? start_norm<T, V, 8 / V, 512>(a, grad, gen, blocks, threads, s)
                 : start_norm<T, 1, 8, 512>(a, grad, gen, blocks, threads, s);
    return vec ? start_norm<T, V, 8 / V, 1024>(a, grad, gen, blocks, threads, s)
               : start_norm<T, 1, 8, 1024>(a, grad, gen, blocks, threads, s);
  }
  return vec ? start_norm<T, V, 32 / V, 1024>(a, grad, gen, blocks, threads, s)
             : start_norm<T, 1, 32, 1024>(a, grad, gen, blocks, threads, s);
}

cudaError_t start_norm_f32(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, cudaStream_t s);
cudaError_t start_norm_bf16(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, cudaStream_t s);
cudaError_t start_norm_f16(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, cudaStream_t s);

}  // namespace adops

#endif
