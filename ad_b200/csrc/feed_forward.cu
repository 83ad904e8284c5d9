// A gated feed-forward block and its gradient: ad_feed_forward, ad_feed_forward_grad.
//
//   g = x Wg^T;  u = x Wu^T;  h = act(g) u;  y = h Wd^T
//   dh = dy Wd;  du = dh act(g);  dg = dh u act'(g)
//   dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dWd = dy^T h
//
// Bound by the tensor cores (gemm16.cuh) where there are many rows.  One kernel
// makes g, u and h: a tile's operands are rows of both matrices, half its columns
// each, so that x comes once and the activation and the product are its epilogue's;
// g and u go to memory only when the gradient will want them.  Backward, dh never
// leaves the tile: its epilogue reads g and u and writes dg, du and h, made again
// from g and u.  dx is one product over both K's; it and the weights' three gradients are one launch.
//
// What enters a product (h, dg, du) is rounded to the operands' type, once: g and
// u are kept in 32 bits.  Kept in 16, all gradients but x's went through three roundings
// instead of two: 3.0e-3 to 3.5e-3 off (norm-wise, bf16) instead of 2.4e-3, of which
// the result's own rounding is 1.7e-3.
#include <cmath>

#include "gemm16.cuh"

namespace {

using namespace adgemm;

enum Act { SILU = 0, GELU = 1, GELU_TANH = 2, RELU = 3, ACTS = 4 };

// Two values that one instruction works on.
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 apart(Two x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ unsigned rounded(Two x, int half) {
  const float2 v = apart(x);
  return pack2(v.x, v.y, half);
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, float b, float c) { return fma2(a, two(b, b), two(c, c)); }
__device__ __forceinline__ Two mul2(Two a, float b) { return mul2(a, two(b, b)); }
__device__ __forceinline__ Two exp2_2(Two x) {
  float2 v = apart(x);
  asm("ex2.approx.f32 %0, %0;" : "+f"(v.x));
  asm("ex2.approx.f32 %0, %0;" : "+f"(v.y));
  return two(v.x, v.y);
}
__device__ __forceinline__ Two reciprocal2(Two x) {
  float2 v = apart(x);
  asm("rcp.approx.f32 %0, %0;" : "+f"(v.x));
  asm("rcp.approx.f32 %0, %0;" : "+f"(v.y));
  return two(v.x, v.y);
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float DENSITY = 0.39894228040143268f;    // 1 / sqrt(2 pi)
constexpr float TANH_SCALE = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float TANH_CUBE = 0.044715f;

// What act(z) = z p is z times, and with SLOPE the derivative, of two values; where
// these say nothing else, errors are a few of 32 bits.
template <int ACT, bool SLOPE>
__device__ __forceinline__ Two share(Two z, Two& slope) {
  const float2 v = apart(z);
  if (ACT == RELU) {
    const Two p = two(v.x > 0.0f ? 1.0f : v.x == v.x ? 0.0f : v.x, v.y > 0.0f ? 1.0f : v.y == v.y ? 0.0f : v.y);
    slope = p;
    return p;
  }
  if (ACT == GELU) {
    // What the normal distribution has beyond |z| is exp(-z^2 / 2) R(|z|), and R, which falls from 1/2 like
    // 1 / |z|, a polynomial in t = 1 / (1 + 0.3 |z|) without a constant, in the manner of Hastings: these
    // coefficients have the least largest error relative to R (1.2e-7 up to |z| = 13.2, where the exponential
    // leaves the normal numbers), fitted in 64 bits.  In 32 bits the whole is within (0.75 z^2 + 9) 2^-24 of
    // itself on the negative side, where it is what z is multiplied by, and 4 2^-24 on the other.  (With
    // erfcf 43 us instead of 40 for 4095 x 512 x 2048.)
    const Two e = exp2_2(mul2(mul2(z, z), -0.5f * LOG2E));
    const Two t = reciprocal2(fma2(two(fabsf(v.x), fabsf(v.y)), 0.3f, 1.0f));
    Two poly = fma2(t, 0.0360888243f, -0.158933669f);
    constexpr float C[6] = {0.209346309f, -0.0564500354f, 0.130032599f, 0.0994650722f, 0.120826311f, 0.11962454f};
#pragma unroll
    for (int i = 0; i < 6; ++i) poly = fma2(poly, t, two(C[i], C[i]));
    const Two tail = mul2(mul2(poly, t), e);
    const float2 below = apart(tail), above = apart(fma2(tail, -1.0f, 1.0f));
    const Two p = two(v.x < 0.0f ? below.x : above.x, v.y < 0.0f ? below.y : above.y);
    if (SLOPE) slope = fma2(mul2(z, DENSITY), e, p);
    return p;
  }
  // The logistic function of z, or of 2 y where tanh(y) is asked for: 1 + tanh(y) is
  // twice that.  From 30 on it is 0 or 1 in 32 bits and the cube is kept from overflowing.
  Two w = z, q = z;  // its argument, and z times the argument's derivative
  if (ACT == GELU_TANH) {
    const Two c = two(v.x > 30.0f ? 30.0f : v.x < -30.0f ? -30.0f : v.x, v.y > 30.0f ? 30.0f : v.y < -30.0f ? -30.0f : v.y);
    const Two square = mul2(c, c), scaled = mul2(c, TANH_SCALE);
    w = mul2(scaled, fma2(square, TANH_CUBE, 1.0f));
    q = mul2(scaled, fma2(square, 3.0f * TANH_CUBE, 1.0f));
  }
  const Two p = reciprocal2(fma2(exp2_2(mul2(w, -LOG2E)), 1.0f, 1.0f));
  if (SLOPE) slope = fma2(mul2(q, p), fma2(p, -1.0f, 1.0f), p);
  return p;
}
// act(z).
template <int ACT>
__device__ __forceinline__ Two activated(Two z) {
  Two slope;
  const Two p = share<ACT, false>(z, slope);
  return ACT == RELU ? two(apart(z).x > 0.0f ? apart(z).x : apart(p).x, apart(z).y > 0.0f ? apart(z).y : apart(p).y) : mul2(z, p);
}

// h of 32 columns from accumulators of both products.
struct Gated {
  static constexpr bool DUAL = true;
  static constexpr int WARPS = 16, SIDE = 4096, PART = 0;
  static constexpr double US[3] = {6.0, 4.5, 3.0};
  using Units = ByNumber;
  struct Params {
    unsigned short* h;
    float *gate, *up;  // NULL when not kept
    long long ldh, ldg, ldu;
    int vec_h, vec_g, vec_u, act;
  };
  struct State {
    __device__ State(const Params&, const Shape&, const Spot&) {}
    __device__ void end(const Params&, const Shape&, const Spot&) {}
    template <int ACT, int HALF>
    __device__ static void gated(const float (&g)[32], const float (&u)[32], unsigned (&w)[16]) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        w[j] = rounded(mul2(activated<ACT>(two(g[2 * j], g[2 * j + 1])), two(u[2 * j], u[2 * j + 1])), HALF);
    }
    template <int ACT>
    __device__ static void gated(const float (&g)[32], const float (&u)[32], unsigned (&w)[16], int half) {
      if (half)
        gated<ACT, 1>(g, u, w);
      else
        gated<ACT, 0>(g, u, w);
    }
    __device__ void chunk(const Params& p, const Shape& a, const Spot& s, int col0, unsigned acc, int cols) {
      unsigned q[32], t[32], w[16];
      float g[32], u[32];
      tmem_issue32(acc, q);
      tmem_issue32(acc + cols, t);
      tmem_wait32(q);
      tmem_wait32(t);
      if (s.last) accumulator_read(s);
#pragma unroll
      for (int j = 0; j < 32; ++j) g[j] = __uint_as_float(q[j]), u[j] = __uint_as_float(t[j]);
      if (s.dead) {
#pragma unroll
        for (int j = 0; j < 32; ++j) g[j] = u[j] = __int_as_float(0x7fffffff);
      }
      // All warps come here at once: half of them store first and the others compute
      // first, so that the two overlap (4095 x 512 x 2048, gelu: 36 us instead of 40)
      const bool late = s.part & 1;
      auto keep = [&] {
        put32(s, g, p.gate, p.ldg, s.m, s.n, col0, p.vec_g);
        put32(s, u, p.up, p.ldu, s.m, s.n, col0, p.vec_u);
      };
      if (p.gate && !late) keep();
      switch (p.act) {
        case SILU: gated<SILU>(g, u, w, a.half); break;
        case GELU: gated<GELU>(g, u, w, a.half); break;
        case GELU_TANH: gated<GELU_TANH>(g, u, w, a.half); break;
        default: gated<RELU>(g, u, w, a.half);
      }
      put16(s, w, p.h, p.ldh, s.m, s.n, col0, p.vec_h);
      if (p.gate && late) keep();
    }
  };
};

// dg, du and h from an accumulator of dh, eight columns of a row a lane.
struct GatedGrad {
  static constexpr bool DUAL = false;
  static constexpr int WARPS = 16, SIDE = 4096, PART = 0;
  static constexpr double US[3] = {11.0, 5.5, 3.2};
  using Units = ByNumber;
  struct Params {
    const float *gate, *up;
    long long ldg, ldu;
    int vec;  // of g and u
    unsigned short *dg, *du, *h;
    long long ld;  // of these, whose rows are aligned
    int act;
  };
  // Eight columns of g and u in a row of a chunk.
  struct Kept {
    float4 g[2], u[2];
  };
  struct State {
    Kept kept[2];  // what comes next, under way
    // the warp's first chunk, ahead of the wait for the accumulator
    __device__ State(const Params& p, const Shape&, const Spot& s) {
      const int col0 = s.unit.col * s.width + s.part * CHUNK;
      if (fast(p, s, col0)) fetch(p, s, col0, 0, kept[0]), fetch(p, s, col0, 1, kept[1]);
    }
    __device__ static bool fast(const Params& p, const Spot& s, int col0) { return p.vec && col0 + CHUNK <= s.n; }
    __device__ void end(const Params&, const Shape&, const Spot&) {}
    template <int ACT>
    __device__ __forceinline__ static void both(Two dh, Two g, Two u, Two& dg, Two& du, Two& h) {
      Two slope;
      const Two p = share<ACT, true>(g, slope);
      const Two act = ACT == RELU ? activated<ACT>(g) : mul2(g, p);
      dg = mul2(mul2(dh, u), slope), du = mul2(dh, act), h = mul2(act, u);
    }
    __device__ static void fetch(const Params& p, const Spot& s, int col0, int i, Kept& k) {
      const long long row = s.row0 + i * 8 + (s.lane >> 2);
      const int col = col0 + (s.lane & 3) * 8;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        k.g[j] = k.u[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (row < s.m) {
          k.g[j] = reinterpret_cast<const float4*>(p.gate + row * p.ldg + col)[j];
          k.u[j] = reinterpret_cast<const float4*>(p.up + row * p.ldu + col)[j];
        }
      }
    }
    template <int ACT, int HALF>
    __device__ __forceinline__ void part(const Params& p, const Spot& s, int col0) {
      const int next = col0 + s.stride;
      const bool more = !s.last && fast(p, s, next);
      const int q = s.lane & 3;
      long long at = (s.row0 + (s.lane >> 2)) * p.ld + col0 + q * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (s.lane >> 2);
        const Kept c = kept[i & 1];
        if (i + 2 < 4)
          fetch(p, s, col0, i + 2, kept[i & 1]);
        else if (more)
          fetch(p, s, next, i - 2, kept[i & 1]);
        unsigned dg[4], du[4], h[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 d = staged(s, r, 2 * q + j);
          Two x, y, z;
          both<ACT>(two(d.x, d.y), two(c.g[j].x, c.g[j].y), two(c.u[j].x, c.u[j].y), x, y, z);
          dg[2 * j] = rounded(x, HALF), du[2 * j] = rounded(y, HALF), h[2 * j] = rounded(z, HALF);
          both<ACT>(two(d.z, d.w), two(c.g[j].z, c.g[j].w), two(c.u[j].z, c.u[j].w), x, y, z);
          dg[2 * j + 1] = rounded(x, HALF), du[2 * j + 1] = rounded(y, HALF), h[2 * j + 1] = rounded(z, HALF);
        }
        if (s.row0 + r < s.m) {
          *reinterpret_cast<uint4*>(p.dg + at) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
          *reinterpret_cast<uint4*>(p.du + at) = make_uint4(du[0], du[1], du[2], du[3]);
          *reinterpret_cast<uint4*>(p.h + at) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        at += 8 * p.ld;
      }
    }
    template <int ACT>
    __device__ __forceinline__ void part(const Params& p, const Shape& a, const Spot& s, int col0) {
      if (a.half)
        part<ACT, 1>(p, s, col0);
      else
        part<ACT, 0>(p, s, col0);
    }
    template <int ACT>
    __device__ static void columns(const Params& p, const Shape& a, const Spot& s, int col0) {
      const int col = col0 + s.lane;
      if (col >= s.n) return;
      for (int r = 0; r < 32 && s.row0 + r < s.m; ++r) {
        const float dh = staged1(s, r);
        const int type = a.half ? AD_F16 : AD_BF16;
        const long long row = s.row0 + r;
        Two x, y, z;
        both<ACT>(two(dh, dh), two(p.gate[row * p.ldg + col], 0.0f), two(p.up[row * p.ldu + col], 0.0f), x, y, z);
        const float dg = apart(x).x, du = apart(y).x, h = apart(z).x;
        store_any(p.dg, type, row * p.ld + col, dg);
        store_any(p.du, type, row * p.ld + col, du);
        store_any(p.h, type, row * p.ld + col, h);
      }
    }
    __device__ void chunk(const Params& p, const Shape& a, const Spot& s, int col0, unsigned acc, int) {
      float v[32];
      take32(s, acc, v);
      stage32(s, v);
      if (fast(p, s, col0)) {
        switch (p.act) {
          case SILU: part<SILU>(p, a, s, col0); break;
          case GELU: part<GELU>(p, a, s, col0); break;
          case GELU_TANH: part<GELU_TANH>(p, a, s, col0); break;
          default: part<RELU>(p, a, s, col0);
        }
      } else {
        switch (p.act) {
          case SILU: columns<SILU>(p, a, s, col0); break;
          case GELU: columns<GELU>(p, a, s, col0); break;
          case GELU_TANH: columns<GELU_TANH>(p, a, s, col0); break;
          default: columns<RELU>(p, a, s, col0);
        }
      }
    }
  };
};

// ------------------------------------------------------------------ a few rows

// Up to FEW rows take the CUDA cores, and the weights are read once: a warp takes
// a row of them (of both matrices for h), 16 bytes a lane at a time, against all
// rows of x; `shared_by` warps of a block share a row of the weights where
// it is long and there are few.  One row is bound by the weights.  With more, x is unpacked anew for each row
// of the weights, and the CUDA cores bound it: 1, 2, 4 and 8 rows of 1024 with 4096 hidden, bf16, take 6.4, 8.0, 13.3 and
// 24 us (the tensor cores 17.5 for any number up to 16), of 4096 with 14336 hidden (352 MB, 54 us at full rate) 73, 100,
// 187 and 350 (76).
struct RowsArgs {
  const unsigned short *x, *w0, *w1;
  long long ldx, ld0, ld1;
  int rows, n, k, act;
  unsigned short* out;
  long long ldo;
  float *gate, *up;
  long long ldg, ldu;
};

// V elements as they are loaded, and their values.
template <int V>
using Raw = typename Word<2 * V>::type;
template <int V>
__device__ __forceinline__ Raw<V> raw_row(const unsigned short* p) {
  return *reinterpret_cast<const Raw<V>*>(p);
}
template <int V>
__device__ __forceinline__ void open_row(const Raw<V>& r, int half, float (&v)[V]) {
  if constexpr (V == 8) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack2(w[j], half);
      v[2 * j] = f.x, v[2 * j + 1] = f.y;
    }
  } else if constexpr (V == 2) {
    const float2 f = unpack2(r, half);
    v[0] = f.x, v[1] = f.y;
  } else {
    v[0] = unpack2(r, half).x;
  }
}

// 64 registers a thread at most, or the blocks of 4096 rows would not all be resident.
template <int T, int V, int HALF, bool DUAL>
__global__ void __launch_bounds__(256, 4) rows_kernel(const __grid_constant__ RowsArgs a, int shared_by) {
  constexpr int U = DUAL ? 2 : 4;  // loads of weights under way, in each matrix
  __shared__ float buf[8][2 * T];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * (8 / shared_by) + warp / shared_by, share = warp % shared_by;
  const int first = (share * 32 + lane) * V, step = 32 * V * shared_by;
  const bool in = row < a.n;
  const unsigned short *w0 = a.w0 + row * a.ld0, *w1 = DUAL ? a.w1 + row * a.ld1 : nullptr;
  Raw<V> p[U], q[U];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (in && k0 + u * step < a.k) {
        p[u] = raw_row<V>(w0 + k0 + u * step);
        if (DUAL) q[u] = raw_row<V>(w1 + k0 + u * step);
      }
  };
  // The second product's weights are under way before the first has ended, which
  // does not write them; it began when all before it had ended.
  if (!DUAL) fetch(first);
  after_previous();
  if (DUAL) fetch(first);
  float s[2][T];
#pragma unroll
  for (int t = 0; t < T; ++t) s[0][t] = s[1][t] = 0.0f;
  for (int k0 = first; in && k0 < a.k;) {
    Raw<V> pc[U], qc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) pc[u] = p[u], qc[u] = q[u];
    const int now = k0;
    k0 += U * step;
    fetch(k0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = now + u * step;
      if (k >= a.k) break;
      float pv[V], qv[V], x[V];
      open_row<V>(pc[u], HALF, pv);
      if (DUAL) open_row<V>(qc[u], HALF, qv);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        if (t >= a.rows) break;
        open_row<V>(raw_row<V>(a.x + t * a.ldx + k), HALF, x);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s[0][t] = fmaf(pv[j], x[j], s[0][t]);
          if (DUAL) s[1][t] = fmaf(qv[j], x[j], s[1][t]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < T; ++t) {
    s[0][t] = warp_sum(s[0][t]);
    if (DUAL) s[1][t] = warp_sum(s[1][t]);
  }
  if (lane == 0) {
#pragma unroll
    for (int t = 0; t < T; ++t) buf[warp][2 * t] = s[0][t], buf[warp][2 * t + 1] = s[1][t];
  }
  __syncthreads();
  if (row >= a.n || share || lane >= a.rows) return;
  float g = buf[warp][2 * lane], u = buf[warp][2 * lane + 1];
  for (int i = 1; i < shared_by; ++i) g += buf[warp + i][2 * lane], u += buf[warp + i][2 * lane + 1];
  if (DUAL) {
    if (a.gate) {
      a.gate[lane * a.ldg + row] = g;
      a.up[lane * a.ldu + row] = u;
    }
    switch (a.act) {
      case SILU: g = apart(activated<SILU>(two(g, g))).x; break;
      case GELU: g = apart(activated<GELU>(two(g, g))).x; break;
      case GELU_TANH: g = apart(activated<GELU_TANH>(two(g, g))).x; break;
      default: g = apart(activated<RELU>(two(g, g))).x;
    }
    g *= u;
  }
  const unsigned w = pack2(g, 0.0f, HALF);
  a.out[lane * a.ldo + row] = static_cast<unsigned short>(w);
}

constexpr int FEW = 8;

template <int T, bool DUAL>
cudaError_t start_rows(const RowsArgs& a, int half, int sms, cudaStream_t st) {
  // 16 bytes at a time where rows allow it, else 4, else an element
  auto fits = [&](int v) {
    auto whole = [&](const void* p, long long ld, long long rows) { return aligned(p, 2 * v) && (rows <= 1 || ld % v == 0); };
    return a.k % v == 0 && whole(a.x, a.ldx, a.rows) && whole(a.w0, a.ld0, a.n) && (!DUAL || whole(a.w1, a.ld1, a.n));
  };
  // warps for all of the device, as long as each has 512 elements of a row
  int shared_by = 1;
  while (shared_by < 8 && a.n * shared_by < 16 * sms && a.k / (2 * shared_by) >= 512) shared_by *= 2;
  const dim3 grid((a.n + 8 / shared_by - 1) / (8 / shared_by));
  auto go = [&](auto v) {
    constexpr int V = decltype(v)::value;
    return half ? launch_early<rows_kernel<T, V, 1, DUAL>>(grid, 256, 0, st, a, shared_by)
                : launch_early<rows_kernel<T, V, 0, DUAL>>(grid, 256, 0, st, a, shared_by);
  };
  return fits(8)   ? go(std::integral_constant<int, 8>())
         : fits(2) ? go(std::integral_constant<int, 2>())
                   : go(std::integral_constant<int, 1>());
}
template <bool DUAL>
cudaError_t few_rows(const RowsArgs& a, int half, int sms, cudaStream_t st) {
  return a.rows == 1   ? start_rows<1, DUAL>(a, half, sms, st)
         : a.rows == 2 ? start_rows<2, DUAL>(a, half, sms, st)
         : a.rows <= 4 ? start_rows<4, DUAL>(a, half, sms, st)
                       : start_rows<FEW, DUAL>(a, half, sms, st);
}

// ------------------------------------------------------------------ host

struct Operand {
  const void* p;
  long long ld, rows, cols;
};

struct Layout {
  size_t pack[5], h, dg, du, partial, total;
  long long ld;  // of h, dg, du
  int tiling;    // of the product with an epilogue of its own
};

// ops: x, Wg, Wu, Wd and, for the gradient, dy.
Layout plan(const Device& d, const Operand* ops, int count, long long rows, long long width, long long hidden) {
  Layout l = {};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += room(bytes);
    return here;
  };
  if (count == 4 && rows <= FEW) {  // h alone
    l.ld = round_up(hidden, 64);
    l.h = take(2ull * rows * l.ld);
    l.total = at;
    return l;
  }
  for (int i = 0; i < count; ++i)
    if (!tma_ready(ops[i].p, ops[i].ld, ops[i].rows)) l.pack[i] = take(2ull * ops[i].rows * round_up(ops[i].cols, 64));
  l.ld = round_up(hidden, 64);
  l.h = take(2ull * rows * l.ld);
  if (count == 5) {
    l.dg = take(2ull * rows * l.ld);
    l.du = take(2ull * rows * l.ld);
  }
  const long long kblocks = (width + BK - 1) / BK;
  l.tiling = count == 4 ? tiling_for<Gated, true>(rows, hidden, kblocks, d.sms) : tiling_for<GatedGrad>(rows, hidden, kblocks, d.sms);
  l.partial = take(partial_bytes(d));
  l.total = at;
  return l;
}

int check(const char* who, int dtype, int64_t rows, int64_t width, int64_t hidden, int act, const Operand* ops, int count) {
  if (dtype != AD_BF16 && dtype != AD_F16) return fail("%s: unknown element type %d (AD_BF16 or AD_F16)", who, dtype);
  if (rows < 0 || width < 1 || hidden < 1) return fail("%s: %lld rows of %lld, %lld hidden", who, (long long)rows, (long long)width, (long long)hidden);
  if (rows > (1 << 24) || width > (1 << 20) || hidden > (1 << 20)) return fail("%s: at most 2^24 rows of 2^20 elements", who);
  if (act < 0 || act >= ACTS) return fail("%s: unknown activation %d", who, act);
  for (int i = 0; i < count; ++i) {
    if (ops[i].rows > 1 && ops[i].ld < ops[i].cols) return fail("%s: rows overlap", who);
    if (!aligned(ops[i].p, 2)) return fail("%s: an operand is not aligned to its elements", who);
  }
  return 0;
}

// Operands as TMA reads them: themselves, or their copies.
int ready(const char* who, const Device& d, const Operand* ops, int count, const size_t* copies, unsigned char* ws, Mat* m,
          cudaStream_t st) {
  Pack packs[MAX_PACKS];
  int n = 0;
  for (int i = 0; i < count; ++i) {
    m[i] = Mat{ops[i].p, ops[i].ld};
    if (tma_ready(ops[i].p, ops[i].ld, ops[i].rows)) continue;
    m[i] = Mat{ws + copies[i], round_up(ops[i].cols, 64)};
    packs[n++] = {ops[i].p, ws + copies[i], ops[i].rows, ops[i].cols, ops[i].ld, m[i].ld};
  }
  return pack_rows(who, d, packs, n, st);
}

bool vec32(const void* p, long long ld, long long rows) { return aligned(p, 16) && (rows <= 1 || ld % 4 == 0); }

}  // namespace

extern "C" int ad_feed_forward_workspace(int device, int dtype, const void* x, int64_t ldx, const void* w_gate,
                                         int64_t ld_gate, const void* w_up, int64_t ld_up, const void* w_down,
                                         int64_t ld_down, const void* dy, int64_t lddy, int64_t rows, int64_t width,
                                         int64_t hidden, int grad, size_t* bytes) {
  const char* who = "ad_feed_forward_workspace";
  if (!bytes) return fail("%s: null operand", who);
  const Operand ops[5] = {{x, ldx, rows, width}, {w_gate, ld_gate, hidden, width}, {w_up, ld_up, hidden, width},
                          {w_down, ld_down, width, hidden}, {dy, lddy, rows, width}};
  const int count = grad ? 5 : 4;
  if (check(who, dtype, rows, width, hidden, 0, ops, count)) return 1;
  *bytes = 0;
  if (!rows) return 0;
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
  const Device d = {guard.device(), sm_count(guard.device())};
  if (!d.sms) return fail("%s: no device properties", who);
  *bytes = plan(d, ops, count, rows, width, hidden).total;
  return 0;
}

extern "C" int ad_feed_forward(int device, int dtype, int act, const void* x, int64_t ldx, const void* w_gate,
                               int64_t ld_gate, const void* w_up, int64_t ld_up, const void* w_down, int64_t ld_down,
                               int64_t rows, int64_t width, int64_t hidden, void* y, int64_t ldy, float* gate, int64_t ldg,
                               float* up, int64_t ldu, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "ad_feed_forward";
  const Operand ops[4] = {{x, ldx, rows, width}, {w_gate, ld_gate, hidden, width}, {w_up, ld_up, hidden, width},
                          {w_down, ld_down, width, hidden}};
  if (check(who, dtype, rows, width, hidden, act, ops, 4)) return 1;
  if ((gate == nullptr) != (up == nullptr) && rows) return fail("%s: gate and up are kept together", who);
  if (rows > 1 && (ldy < width || (gate && (ldg < hidden || ldu < hidden)))) return fail("%s: rows overlap", who);
  if (!rows) return 0;
  if (!x || !w_gate || !w_up || !w_down || !y) return fail("%s: null operand", who);
  if (!aligned(y, 2) || !aligned({gate, up}, 4)) return fail("%s: an operand is not aligned to its elements", who);
  if (overlap({{y, rows, width * 2, ldy * 2, true}, {gate, rows, hidden * 4, ldg * 4, true}, {up, rows, hidden * 4, ldu * 4, true},
               {workspace, 1, static_cast<long long>(workspace_bytes), 0, true}, {x, rows, width * 2, ldx * 2, false},
               {w_gate, hidden, width * 2, ld_gate * 2, false}, {w_up, hidden, width * 2, ld_up * 2, false},
               {w_down, width, hidden * 2, ld_down * 2, false}}))
    return fail("%s: results overlap operands or one another", who);
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
  const Device d = {guard.device(), sm_count(guard.device())};
  if (!d.sms) return fail("%s: no device properties", who);
  const int half = dtype == AD_F16;
  const Layout l = plan(d, ops, 4, rows, width, hidden);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.total)
    return fail("%s: needs %zu bytes of workspace, 256-byte aligned", who, l.total);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  if (rows <= FEW) {
    auto half_ptr = [](const void* q) { return static_cast<const unsigned short*>(q); };
    unsigned short* h = reinterpret_cast<unsigned short*>(ws + l.h);
    RowsArgs r = {half_ptr(x), half_ptr(w_gate), half_ptr(w_up), ldx, ld_gate, ld_up, static_cast<int>(rows),
                  static_cast<int>(hidden), static_cast<int>(width), act, h, l.ld, gate, up, ldg, ldu};
    cudaError_t e = few_rows<true>(r, half, d.sms, st);
    r = {h, half_ptr(w_down), nullptr, l.ld, ld_down, 0, static_cast<int>(rows), static_cast<int>(width),
         static_cast<int>(hidden), act, static_cast<unsigned short*>(y), ldy, nullptr, nullptr, 0, 0};
    if (e == cudaSuccess) e = few_rows<false>(r, half, d.sms, st);
    return e == cudaSuccess ? 0 : fail_cuda(who, e);
  }
  Mat m[4];
  if (ready(who, d, ops, 4, l.pack, ws, m, st)) return 1;
  const Problem p = {rows, hidden, width, width, false, false, {m[0], {}}, {m[1], m[2]}};
  Gated::Params q = {};
  q.h = reinterpret_cast<unsigned short*>(ws + l.h), q.ldh = l.ld, q.vec_h = 1;
  q.gate = gate, q.up = up;
  q.ldg = ldg, q.ldu = ldu, q.vec_g = vec32(gate, ldg, rows), q.vec_u = vec32(up, ldu, rows);
  q.act = act;
  if (start<Gated>(who, d, p, half, l.tiling, q, st)) return 1;
  const Problem product = {rows, width, hidden, hidden, false, false, {{ws + l.h, l.ld}, {}}, {m[3], {}}};
  const Result result = {y, ldy, dtype, false, nullptr, 0, nullptr};
  return store_products(who, d, half, &product, &result, 1, reinterpret_cast<float*>(ws + l.partial), st);
}

extern "C" int ad_feed_forward_grad(int device, int dtype, int act, const void* dy, int64_t lddy, const void* x,
                                    int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up,
                                    const void* w_down, int64_t ld_down, const float* gate, int64_t ldg, const float* up,
                                    int64_t ldu, int64_t rows, int64_t width, int64_t hidden, void* dx, int64_t lddx,
                                    int dw_type, void* dw_gate, int64_t lddw_gate, void* dw_up, int64_t lddw_up,
                                    void* dw_down, int64_t lddw_down, int accumulate, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* who = "ad_feed_forward_grad";
  const Operand ops[5] = {{x, ldx, rows, width}, {w_gate, ld_gate, hidden, width}, {w_up, ld_up, hidden, width},
                          {w_down, ld_down, width, hidden}, {dy, lddy, rows, width}};
  if (check(who, dtype, rows, width, hidden, act, ops, 5)) return 1;
  if (dw_type != dtype && dw_type != AD_F32) return fail("%s: unknown type %d of the weights' gradients", who, dw_type);
  const size_t es = elem_size(dw_type);
  if (!dw_gate || !dw_up || !dw_down || !aligned({dw_gate, dw_up, dw_down}, es))
    return fail("%s: an operand is null or not aligned to its elements", who);
  if ((rows > 1 && (lddx < width || ldg < hidden || ldu < hidden)) ||
      (hidden > 1 && (lddw_gate < width || lddw_up < width)) || (width > 1 && lddw_down < hidden))
    return fail("%s: rows overlap", who);
  if (!rows) {
    if (accumulate) return 0;
    return ad_clear_rows(device, dw_gate, lddw_gate * es, width * es, hidden, stream) ||
           ad_clear_rows(device, dw_up, lddw_up * es, width * es, hidden, stream) ||
           ad_clear_rows(device, dw_down, lddw_down * es, hidden * es, width, stream);
  }
  if (!dy || !x || !w_gate || !w_up || !w_down || !gate || !up || !dx) return fail("%s: null operand", who);
  if (!aligned(dx, 2) || !aligned({gate, up}, 4)) return fail("%s: an operand is not aligned to its elements", who);
  const long long wide = width * es, tall = hidden * es, e = es;
  if (overlap({{dx, rows, width * 2, lddx * 2, true}, {dw_gate, hidden, wide, lddw_gate * e, true}, {dw_up, hidden, wide, lddw_up * e, true},
               {dw_down, width, tall, lddw_down * e, true}, {workspace, 1, static_cast<long long>(workspace_bytes), 0, true},
               {dy, rows, width * 2, lddy * 2, false}, {x, rows, width * 2, ldx * 2, false},
               {w_gate, hidden, width * 2, ld_gate * 2, false}, {w_up, hidden, width * 2, ld_up * 2, false},
               {w_down, width, hidden * 2, ld_down * 2, false}, {gate, rows, hidden * 4, ldg * 4, false}, {up, rows, hidden * 4, ldu * 4, false}}))
    return fail("%s: results overlap operands or one another", who);
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
  const Device d = {guard.device(), sm_count(guard.device())};
  if (!d.sms) return fail("%s: no device properties", who);
  const int half = dtype == AD_F16;
  const Layout l = plan(d, ops, 5, rows, width, hidden);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.total)
    return fail("%s: needs %zu bytes of workspace, 256-byte aligned", who, l.total);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  Mat m[5];
  if (ready(who, d, ops, 5, l.pack, ws, m, st)) return 1;
  const Mat h = {ws + l.h, l.ld}, dg = {ws + l.dg, l.ld}, du = {ws + l.du, l.ld};

  const Problem p = {rows, hidden, width, width, false, true, {m[4], {}}, {m[3], {}}};
  GatedGrad::Params q = {};
  q.gate = gate, q.up = up;
  q.ldg = ldg, q.ldu = ldu, q.vec = vec32(gate, ldg, rows) && vec32(up, ldu, rows);
  q.dg = reinterpret_cast<unsigned short*>(ws + l.dg), q.du = reinterpret_cast<unsigned short*>(ws + l.du);
  q.h = reinterpret_cast<unsigned short*>(ws + l.h), q.ld = l.ld;
  q.act = act;
  if (start<GatedGrad>(who, d, p, half, l.tiling, q, st)) return 1;

  const bool more = accumulate != 0;
  const Problem products[4] = {{rows, width, 2 * hidden, hidden, false, true, {dg, du}, {m[1], m[2]}},
                               {hidden, width, rows, rows, true, true, {dg, {}}, {m[0], {}}},
                               {hidden, width, rows, rows, true, true, {du, {}}, {m[0], {}}},
                               {width, hidden, rows, rows, true, true, {m[4], {}}, {h, {}}}};
  const Result results[4] = {{dx, lddx, dtype, false, nullptr, 0, nullptr},
                             {dw_gate, lddw_gate, dw_type, more, nullptr, 0, nullptr},
                             {dw_up, lddw_up, dw_type, more, nullptr, 0, nullptr},
                             {dw_down, lddw_down, dw_type, more, nullptr, 0, nullptr}};
  return store_products(who, d, half, products, results, 4, reinterpret_cast<float*>(ws + l.partial), st);
}
