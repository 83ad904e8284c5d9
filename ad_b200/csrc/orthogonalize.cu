// Newton-Schulz orthogonalisation of matrix updates: ad_orthogonalize.
//
// For a matrix G with m <= n (a taller one is taken as its transpose):
//
//   X = G / (|G|_F + eps);  a few times:  A = X X^T,  B = b A + c A A,  X = a X + B X
//
// which maps every singular value s to a s + b s^3 + c s^5 and leaves the
// singular vectors alone.
//
// Bound by the tensor cores: products of 16-bit operands (f16, whose 11 bits
// serve better here than bf16's 8: all values lie in a range known beforehand
// and are held times a power of two) on tcgen05, accumulated in 32 bits.  The
// places where fewer bits would hurt are kept out of the operands: X itself is
// held in 32 bits and only its copies as operands are rounded, because early
// steps multiply the error of a X by a in directions where G has next to
// nothing; and the diagonals of A and B, which are large beside the rest once
// the singular values come near 1, are held in 32 bits and added in the
// epilogues.  The result is then within about 1e-3 (norm-wise) of the exact
// iteration, rank-one matrices included.
//
// Operands are K-major tiles brought by TMA: rows of X for X X^T, rows of the
// symmetric A for A A, rows of B and of X^T for B X.  The last product's
// epilogue writes X both ways; with a row of the accumulator to each lane the
// transposed store is the coalesced one.
#include <cuda.h>

#include <cmath>
#include <initializer_list>

#include "ops_common.cuh"

namespace {

using namespace adops;

constexpr int BM = 128, BK = 64;  // tile rows; elements of K a stage (128 bytes, the swizzle's width)
constexpr int STAGES = 4;
constexpr int MAX_STEPS = 32;
constexpr int NORM_BLOCKS = 64;  // blocks that share a matrix's norm

enum Mode { GRAM = 0, POLY = 1, UPDATE = 2 };

struct Step {  // one product's epilogue
  int m, n;        // of X
  int ldx, ldt, lda;  // rows of X, of X^T, of A and B (elements)
  float scale;     // GRAM: of the accumulator; POLY, UPDATE: see the epilogue
  float p, q;
  __half *a, *b, *xh, *xt_next;  // X^T is an operand of the product that replaces it: two of them
  float *xf, *da, *db;
  void* out;       // UPDATE: the result, when this is the last step
  int out_type;
  long long out_batch, out_row, out_col;
  float out_scale;
  int* err;
};

__device__ __forceinline__ unsigned smem_u32(const void* p) {
  return static_cast<unsigned>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ bool bar_try(unsigned long long* b, unsigned phase) {
  unsigned ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(phase)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Bounded wait (2 s): false when the phase never completed.
__device__ __noinline__ bool bar_wait(unsigned long long* b, unsigned phase) {
  if (bar_try(b, phase)) return true;
  const unsigned long long t0 = now();
  while (true) {
    for (int i = 0; i < 256; ++i)
      if (bar_try(b, phase)) return true;
    if (now() - t0 > 2000000000ull) return false;
  }
}
// K-major tile with 128-byte rows, 128-byte swizzle.
__device__ __forceinline__ unsigned long long tile_desc(const void* p) {
  const unsigned long long a = (smem_u32(p) >> 4) & 0x3FFFull;
  return a | (1ull << 16) | ((1024ull >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void tmem_ld32(unsigned taddr, unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// 32 values of a row: 16 bytes at a time where all are inside.
__device__ __forceinline__ void store_half32(__half* p, const float (&v)[32], int inside) {
  if (inside >= 32) {
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
      Vec<__half, 8> w;
#pragma unroll
      for (int j = 0; j < 8; ++j) w.v[j] = __float2half_rn(v[k + j]);
      store_vec<__half, 8>(p + k, w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < inside) p[j] = __float2half_rn(v[j]);
  }
}

template <int MODE>
__device__ __forceinline__ void epilogue32(const Step& s, long long mat, int row, int col0, const unsigned (&acc)[32]) {
  const int width = MODE == UPDATE ? s.n : s.m;
  const int inside = row < s.m ? width - col0 : 0;
  float v[32];
  if (MODE == GRAM) {
    if (inside <= 0) return;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = __uint_as_float(acc[j]) * s.scale;
      if (col0 + j == row) {
        s.da[mat * s.m + row] = v[j];
        v[j] = 0.0f;
      }
    }
    store_half32(s.a + (mat * s.m + row) * s.lda + col0, v, inside);
  } else if (MODE == POLY) {
    // B = p A + q (A_o A_o + (d_row + d_col) A_o), A_o without its diagonal d
    if (inside <= 0) return;
    const __half* a = s.a + (mat * s.m + row) * s.lda + col0;
    const float* d = s.da + mat * s.m;
    const float dr = d[row];
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
      if (k >= inside) break;
      const Vec<__half, 8> w = load_vec<__half, 8>(a + k);  // the row's padding is readable
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = col0 + k + j;
        const float ao = to_float(w.v[j]), dc = k + j < inside ? d[c] : 0.0f;
        v[k + j] = s.p * ao + s.q * (__uint_as_float(acc[k + j]) + (dr + dc) * ao);
        if (c == row) {
          s.db[mat * s.m + row] = s.p * dr + s.q * (__uint_as_float(acc[k + j]) + dr * dr);
          v[k + j] = 0.0f;
        }
      }
    }
    store_half32(s.b + (mat * s.m + row) * s.lda + col0, v, inside);
  } else {
    // X = p X + q (B_o X_h + d X_h)
    const long long at = (mat * s.m + row) * s.ldx + col0;
    const float d = inside > 0 ? s.db[mat * s.m + row] : 0.0f;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; k += 4) {
      if (k >= inside) break;
      const Vec<float, 4> w = load_vec<float, 4>(s.xf + at + k);  // the row's padding is readable
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[k + j] = s.p * w.v[j] + s.q * (__uint_as_float(acc[k + j]) + d * __half2float(__float2half_rn(w.v[j])));
    }
    if (s.out) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < inside)
          store_any(s.out, s.out_type, mat * s.out_batch + row * s.out_row + (col0 + j) * s.out_col, v[j] * s.out_scale);
      return;
    }
    if (inside > 0) {
#pragma unroll
      for (int k = 0; k < 32; k += 4) {
        if (k + 4 <= inside) {
          Vec<float, 4> w;
#pragma unroll
          for (int j = 0; j < 4; ++j) w.v[j] = v[k + j];
          store_vec<float, 4>(s.xf + at + k, w);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (k + j < inside) s.xf[at + k + j] = v[k + j];
        }
      }
      store_half32(s.xh + at, v, inside);
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < inside) s.xt_next[(mat * s.n + col0 + j) * s.ldt + row] = __float2half_rn(v[j]);
    }
  }
}

template <int BN>
constexpr int gemm_smem() {
  return STAGES * (BM + BN) * BK * 2 + 1024 + 256;
}

// C = P Q^T over one tile: P [m rows][k], Q [n rows][k], both K-major.
// tp, tq: maps over all matrices' rows; prow, qrow: rows of one matrix.
template <int MODE, int BN>
__global__ void __launch_bounds__(128, 1)
    ns_gemm(const __grid_constant__ CUtensorMap tp, const __grid_constant__ CUtensorMap tq, int prow, int qrow,
            int kblocks, const __grid_constant__ Step s) {
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  constexpr unsigned P_BYTES = BM * BK * 2, Q_BYTES = BN * BK * 2, STAGE = P_BYTES + Q_BYTES;
  unsigned long long* full = reinterpret_cast<unsigned long long*>(smem + STAGES * STAGE);
  unsigned long long* empty = full + STAGES;
  unsigned long long* accb = empty + STAGES;
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(accb + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* consumed = abort_flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
  const long long mat = blockIdx.z;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&empty[i])));
    }
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(accb)));
    *abort_flag = 0;
    *consumed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(BN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = *tmem_slot;

  if (warp == 0 && lane == 0) {
    int issued = 0;
    for (int kb = 0; kb < kblocks; ++kb) {
      const int i = kb % STAGES;
      if (kb >= STAGES && !bar_wait(&empty[i], ((kb / STAGES) - 1) & 1)) {
        *abort_flag = 1;
        atomicExch(s.err, 1);
        break;
      }
      if (*abort_flag) break;
      unsigned char* st = smem + i * STAGE;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&full[i])), "r"(STAGE)
                   : "memory");
      asm volatile(
          "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
              smem_u32(st)),
          "l"(reinterpret_cast<unsigned long long>(&tp)), "r"(smem_u32(&full[i])), "r"(kb * BK),
          "r"(static_cast<int>(mat * prow) + m0)
          : "memory");
      asm volatile(
          "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
              smem_u32(st + P_BYTES)),
          "l"(reinterpret_cast<unsigned long long>(&tq)), "r"(smem_u32(&full[i])), "r"(kb * BK),
          "r"(static_cast<int>(mat * qrow) + n0)
          : "memory");
      issued = kb + 1;
    }
    if (*abort_flag)
      for (int kb = *consumed; kb < issued; ++kb) bar_wait(&full[kb % STAGES], (kb / STAGES) & 1);
  } else if (warp == 1 && lane == 0) {
    // D f32, A and B f16, both K-major
    constexpr unsigned IDESC = (1u << 4) | (static_cast<unsigned>(BN >> 3) << 17) | ((128u >> 4) << 24);
    for (int kb = 0; kb < kblocks; ++kb) {
      const int i = kb % STAGES;
      if (!bar_wait(&full[i], (kb / STAGES) & 1)) {
        *abort_flag = 1;
        atomicExch(s.err, 2);
        break;
      }
      if (*abort_flag) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      unsigned char* st = smem + i * STAGE;
      const unsigned long long pd = tile_desc(st), qd = tile_desc(st + P_BYTES);
#pragma unroll
      for (int k = 0; k < BK / 16; ++k) {
        const unsigned long long adv = static_cast<unsigned long long>(k * 32) >> 4;
        const unsigned more = (kb > 0 || k > 0) ? 1u : 0u;
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(tmem),
            "l"(pd + adv), "l"(qd + adv), "r"(IDESC), "r"(more)
            : "memory");
      }
      asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                       smem_u32(&empty[i]))
                   : "memory");
      *consumed = kb + 1;
    }
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(accb))
                 : "memory");
  }
  __syncwarp();

  const bool ok = bar_wait(accb, 0);
  if (!ok) atomicExch(s.err, 3);
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  __syncthreads();
  const bool good = ok && !*abort_flag && *reinterpret_cast<volatile int*>(s.err) == 0;
  const int row = m0 + warp * 32 + lane;
  for (int c = 0; c < BN / 32; ++c) {
    unsigned r[32];
    tmem_ld32(tmem + (static_cast<unsigned>(warp * 32) << 16) + static_cast<unsigned>(c * 32), r);
    if (!good) {  // a wait ran out: the result shows it
#pragma unroll
      for (int j = 0; j < 32; ++j) r[j] = 0x7fffffffu;
    }
    epilogue32<MODE>(s, mat, row, n0 + c * 32, r);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(BN) : "memory");
}

struct LoadArgs {
  const void* g;
  int type;
  long long batch, row, col;  // strides of G seen as m x n
  int m, n, ldx, ldt;
  float eps, scale;
  double* part;
  __half *xh, *xt;
  float* xf;
};

// A share of a matrix's sum of squares, in 64 bits: no scale of the update overflows.
__global__ void __launch_bounds__(256) ns_norm(const __grid_constant__ LoadArgs a) {
  __shared__ double buf[8];
  const long long mat = blockIdx.y;
  const bool by_row = a.col == 1 || a.row != 1;  // along the axis of adjacent elements
  const int outer = by_row ? a.m : a.n, inner = by_row ? a.n : a.m;
  const long long so = by_row ? a.row : a.col, si = by_row ? a.col : a.row;
  double s = 0.0;
  for (int o = blockIdx.x; o < outer; o += gridDim.x)
    for (int i = threadIdx.x; i < inner; i += blockDim.x) {
      const double x = load_any(a.g, a.type, mat * a.batch + o * so + i * si);
      s += x * x;
    }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) s += buf[w];
    a.part[mat * NORM_BLOCKS + blockIdx.x] = s;
  }
}

// X = G scale / (|G| + eps), in 32 bits, as operand, and transposed as operand.
__global__ void __launch_bounds__(256) ns_load(const __grid_constant__ LoadArgs a) {
  __shared__ float t[32][33];
  const long long mat = blockIdx.z;
  const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x, ty = threadIdx.y;
  double sum = 0.0;
  for (int k = 0; k < NORM_BLOCKS; ++k) sum += a.part[mat * NORM_BLOCKS + k];
  const float f = static_cast<float>(a.scale / (sqrt(sum) + a.eps));
  const bool by_row = a.col == 1 || a.row != 1;
  for (int k = ty; k < 32; k += 8) {
    const int r = by_row ? r0 + k : r0 + tx, c = by_row ? c0 + tx : c0 + k;
    const float x = r < a.m && c < a.n ? load_any(a.g, a.type, mat * a.batch + r * a.row + c * a.col) * f : 0.0f;
    t[r - r0][c - c0] = x;
  }
  __syncthreads();
  for (int k = ty; k < 32; k += 8) {
    if (r0 + k < a.m && c0 + tx < a.n) {
      const long long at = (mat * a.m + r0 + k) * a.ldx + c0 + tx;
      a.xf[at] = t[k][tx];
      a.xh[at] = __float2half_rn(t[k][tx]);
    }
    if (c0 + k < a.n && r0 + tx < a.m) a.xt[(mat * a.n + c0 + k) * a.ldt + r0 + tx] = __float2half_rn(t[tx][k]);
  }
}

// No steps: the normalised matrix itself.
__global__ void ns_copy(const __grid_constant__ Step s) {
  const long long mat = blockIdx.y;
  const long long n = static_cast<long long>(s.m) * s.n;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int r = static_cast<int>(i / s.n), c = static_cast<int>(i - static_cast<long long>(r) * s.n);
    store_any(s.out, s.out_type, mat * s.out_batch + r * s.out_row + c * s.out_col,
              s.xf[(mat * s.m + r) * s.ldx + c] * s.out_scale);
  }
}

struct Layout {
  long long m, n, ldx, ldt, lda;
  size_t part, xf, xh, xt[2], a, b, da, db, total;
};
Layout plan(long long count, long long rows, long long cols) {
  Layout l;
  l.m = rows < cols ? rows : cols;
  l.n = rows < cols ? cols : rows;
  l.ldx = (l.n + 7) / 8 * 8;
  l.ldt = l.lda = (l.m + 7) / 8 * 8;
  size_t at = 256;  // the error word
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.part = take(sizeof(double) * NORM_BLOCKS * count);
  l.xf = take(4ull * count * l.m * l.ldx);
  l.xh = take(2ull * count * l.m * l.ldx);
  for (size_t& t : l.xt) t = take(2ull * count * l.n * l.ldt);
  l.a = take(2ull * count * l.m * l.lda);
  l.b = take(2ull * count * l.m * l.lda);
  l.da = take(4ull * count * l.m);
  l.db = take(4ull * count * l.m);
  l.total = at;
  return l;
}

// Powers of two that keep what a step holds in 16 bits below 2^15, from the
// largest singular value that can arise: the maxima of a x + b x^3 + c x^5 and
// b l + c l^2 over [0, largest so far] lie at an end or at a root of their
// derivatives.
struct Scales {
  double x[MAX_STEPS + 1], a[MAX_STEPS], b[MAX_STEPS];
  bool ok = true;
};
double below(double largest) {  // with a twentieth to spare for rounding
  return std::ldexp(1.0, 14 - std::ilogb(std::fmax(1.05 * largest, 1e-20)));
}
Scales scales_for(int steps, const float* coef) {
  Scales s;
  double top = 1.0;
  for (int k = 0; k <= steps; ++k) {
    if (!(top <= 1024.0)) {
      s.ok = false;
      return s;
    }
    s.x[k] = below(top);
    if (k == steps) break;
    const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2], end = top * top;
    auto inner = [&](double l) { return std::fabs(b * l + c * l * l); };
    auto f = [&](double l) { return std::fabs(std::sqrt(l) * (a + b * l + c * l * l)); };
    auto with = [&](double best, double l, auto fn) { return l > 0.0 && l < end ? std::fmax(best, fn(l)) : best; };
    s.a[k] = below(end);
    s.b[k] = below(c != 0.0 ? with(inner(end), -b / (2.0 * c), inner) : inner(end));
    double next = f(end);
    if (c != 0.0) {
      const double q = 9.0 * b * b - 20.0 * a * c;
      if (q >= 0.0)
        for (double sign : {-1.0, 1.0}) next = with(next, (-3.0 * b + sign * std::sqrt(q)) / (10.0 * c), f);
    } else if (b != 0.0) {
      next = with(next, -a / (3.0 * b), f);
    }
    top = next;
  }
  return s;
}

template <int MODE, int BN>
cudaError_t gemm(const CUtensorMap& tp, const CUtensorMap& tq, int prow, int qrow, int m, int n, int k, int count,
                 const Step& s, cudaStream_t st) {
  static bool ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(ns_gemm<MODE, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, gemm_smem<BN>());
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  ns_gemm<MODE, BN><<<dim3((n + BN - 1) / BN, (m + BM - 1) / BM, count), 128, gemm_smem<BN>(), st>>>(
      tp, tq, prow, qrow, (k + BK - 1) / BK, s);
  return cudaGetLastError();
}

}  // namespace

extern "C" int ad_orthogonalize_workspace(int64_t count, int64_t rows, int64_t cols, size_t* bytes) {
  if (!bytes || count < 0 || rows < 0 || cols < 0) return fail("ad_orthogonalize_workspace: bad argument");
  *bytes = count && rows && cols ? plan(count, rows, cols).total : 0;
  return 0;
}

extern "C" int ad_orthogonalize(int device, int dtype, const void* g, int64_t count, int64_t rows, int64_t cols,
                                int64_t batch_stride, int64_t row_stride, int64_t col_stride, int steps,
                                const float* coefficients, float eps, int out_dtype, void* out,
                                int64_t out_batch_stride, int64_t out_row_stride, int64_t out_col_stride,
                                void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype < AD_F32 || dtype > AD_F16 || out_dtype < AD_F32 || out_dtype > AD_F16)
    return fail("ad_orthogonalize: unknown element type %d or %d", dtype, out_dtype);
  if (count < 0 || rows < 0 || cols < 0) return fail("ad_orthogonalize: negative size");
  if (steps < 0 || steps > MAX_STEPS || (steps && !coefficients))
    return fail("ad_orthogonalize: %d steps (0 to %d, three coefficients each)", steps, MAX_STEPS);
  if (!(eps >= 0.0f)) return fail("ad_orthogonalize: eps %g", eps);
  if (count == 0 || rows == 0 || cols == 0) return 0;
  if (count > 65535 || rows > 65536 || cols > 65536)
    return fail("ad_orthogonalize: %lld matrices of %lld x %lld (at most 65535 of 65536 x 65536)", (long long)count,
                (long long)rows, (long long)cols);
  const Layout l = plan(count, rows, cols);
  if (count * l.n > 0x7fffffffll) return fail("ad_orthogonalize: too many rows in one call");
  if (!g || !out) return fail("ad_orthogonalize: null operand");
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.total)
    return fail("ad_orthogonalize: needs %zu bytes of workspace, 256-byte aligned", l.total);
  for (int i = 0; i < 3 * steps; ++i)
    if (!std::isfinite(coefficients[i])) return fail("ad_orthogonalize: a coefficient is not a number");
  const Scales sc = scales_for(steps, coefficients);
  if (!sc.ok) return fail("ad_orthogonalize: these coefficients let singular values grow past 1024");
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail("ad_orthogonalize: %s", cudaGetErrorString(guard.error()));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* w = static_cast<unsigned char*>(workspace);
  const bool tall = rows > cols;
  const int m = static_cast<int>(l.m), n = static_cast<int>(l.n), num = static_cast<int>(count);

  LoadArgs la = {};
  la.g = g, la.type = dtype;
  la.batch = batch_stride, la.row = tall ? col_stride : row_stride, la.col = tall ? row_stride : col_stride;
  la.m = m, la.n = n, la.ldx = static_cast<int>(l.ldx), la.ldt = static_cast<int>(l.ldt);
  la.eps = eps, la.scale = static_cast<float>(sc.x[0]);
  la.part = reinterpret_cast<double*>(w + l.part);
  la.xf = reinterpret_cast<float*>(w + l.xf);
  la.xh = reinterpret_cast<__half*>(w + l.xh);
  la.xt = reinterpret_cast<__half*>(w + l.xt[0]);
  cudaError_t e = cudaMemsetAsync(w, 0, 256, st);
  if (e != cudaSuccess) return fail("ad_orthogonalize: %s", cudaGetErrorString(e));
  ns_norm<<<dim3(NORM_BLOCKS, num), 256, 0, st>>>(la);
  ns_load<<<dim3((n + 31) / 32, (m + 31) / 32, num), dim3(32, 8), 0, st>>>(la);
  e = cudaGetLastError();
  if (e != cudaSuccess) return fail("ad_orthogonalize: %s", cudaGetErrorString(e));

  Step s = {};
  s.m = m, s.n = n, s.ldx = la.ldx, s.ldt = la.ldt, s.lda = static_cast<int>(l.lda);
  s.a = reinterpret_cast<__half*>(w + l.a);
  s.b = reinterpret_cast<__half*>(w + l.b);
  s.xf = la.xf, s.xh = la.xh;
  s.da = reinterpret_cast<float*>(w + l.da);
  s.db = reinterpret_cast<float*>(w + l.db);
  s.err = reinterpret_cast<int*>(w);
  s.out_type = out_dtype;
  s.out_batch = out_batch_stride;
  s.out_row = tall ? out_col_stride : out_row_stride, s.out_col = tall ? out_row_stride : out_col_stride;
  if (steps == 0) {
    s.out = out;
    s.out_scale = static_cast<float>(1.0 / sc.x[0]);
    ns_copy<<<dim3(256, num), 256, 0, st>>>(s);
    e = cudaGetLastError();
    if (e != cudaSuccess) return fail("ad_orthogonalize: %s", cudaGetErrorString(e));
    return 0;
  }
  constexpr int BN = 128;
  // maps of X, A, B as left operands (128 rows a box), X, A and X^T as right ones
  alignas(64) CUtensorMap tx, ta, tb, txq, taq, tt[2];
  struct {
    CUtensorMap* map;
    const void* base;
    long long rows, cols, ld;
    int box;
  } const maps[7] = {{&tx, s.xh, count * m, n, l.ldx, BM},  {&ta, s.a, count * m, m, l.lda, BM},
                     {&tb, s.b, count * m, m, l.lda, BM},   {&txq, s.xh, count * m, n, l.ldx, BN},
                     {&taq, s.a, count * m, m, l.lda, BN},  {&tt[0], w + l.xt[0], count * n, m, l.ldt, BN},
                     {&tt[1], w + l.xt[1], count * n, m, l.ldt, BN}};
  for (const auto& t : maps)
    if (ad_tmap_2d(reinterpret_cast<uint64_t>(t.base), t.rows, t.cols, 2ull * t.ld, t.box, BK, 2, 128, t.map)) return 1;
  for (int k = 0; k < steps; ++k) {
    const double a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
    const double sx = sc.x[k], sa = sc.a[k], sb = sc.b[k];
    s.scale = static_cast<float>(sa / (sx * sx));
    e = gemm<GRAM, BN>(tx, txq, m, m, m, m, n, num, s, st);
    if (e == cudaSuccess) {
      s.p = static_cast<float>(b * sb / sa);
      s.q = static_cast<float>(c * sb / (sa * sa));
      e = gemm<POLY, BN>(ta, taq, m, m, m, m, m, num, s, st);
    }
    if (e == cudaSuccess) {
      const double up = sc.x[k + 1] / sx;
      s.p = static_cast<float>(a * up);
      s.q = static_cast<float>(up / sb);
      if (k + 1 == steps) s.out = out, s.out_scale = static_cast<float>(1.0 / sc.x[steps]);
      s.xt_next = reinterpret_cast<__half*>(w + l.xt[(k + 1) & 1]);
      e = gemm<UPDATE, BN>(tb, tt[k & 1], m, n, m, n, m, num, s, st);
    }
    if (e != cudaSuccess) return fail("ad_orthogonalize: %s", cudaGetErrorString(e));
  }
  return 0;
}
