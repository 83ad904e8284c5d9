// Products of 16-bit matrices on tcgen05 with an epilogue of the caller's: the
// core of the feed-forward block and of the log probabilities of a linear layer.
//
//   C[m][n] = sum_k A(m, k) B(n, k)
//
// accumulated in 32 bits in tensor memory.  An operand lies in memory with its
// rows along K (K-major) or across it (A as [K][M], B as [K][N]): no transposed
// copies are made, the matrix instruction takes either.
//
// Bound by the tensor cores, and before them by what a multiprocessor can bring
// from L2 (60 to 80 GB/s): a pair of blocks (cta_group::2) works on a tile of 256
// x 256, so that 32 KB a block serve 4.2 MFLOP; single blocks on 128 x 128 or 128 x
// 64 are for products with too few large tiles.  Blocks stay resident and take
// every so-many-th tile; in a block one warp brings operands by TMA, one issues
// the products into one of two accumulators, sixteen work on the other, so that a
// tile's epilogue is hidden behind the next tile's products.  Tiles are walked in
// bands of rows, so that the tiles under way at a time share operands in L2.
// Few tiles with a long K are split over K: partial sums go to memory in 32 bits
// and are joined in order.  Nothing depends on scheduling.
#ifndef AD_B200_GEMM16_CUH
#define AD_B200_GEMM16_CUH

#include <cuda.h>

#include <algorithm>

#include "ops_common.cuh"

namespace ad_b200_internal {
// runtime.cu: TMA descriptor of a row-major matrix of 16-bit elements, swizzled
// over 128 bytes; what lies outside reads as zero.  0, or 1 with an error set.
int tmap_2d_16(const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, uint32_t box_cols,
               void* out128);
}

namespace adgemm {

using namespace adops;

constexpr int BK = 64;            // elements of K a stage: 128 bytes, the swizzle's width
constexpr int BOX = 64 * BK * 2;  // bytes of a box of 64 x 64
constexpr int EPI_WARPS = 16, PARTS = EPI_WARPS / 4;  // warps that share 32 rows, each with every fourth chunk
constexpr int THREADS = 32 * (2 + EPI_WARPS);
constexpr int CHUNK = 32;                  // columns that an epilogue takes at a time
constexpr int SIDE = 32 * CHUNK * 4;       // bytes of shared memory of an epilogue warp: 32 rows of them
constexpr int MAX_GROUPS = 3;

// Tiles: CTAS blocks work on one of 128 CTAS rows and BN columns.
template <int CTAS_, int BN_>
struct Tile {
  static constexpr int CTAS = CTAS_, BN = BN_, M = 128 * CTAS;
  static constexpr int QN = BN / CTAS;  // columns whose operand a block holds
  static constexpr int P_BYTES = 128 * BK * 2, Q_BYTES = QN * BK * 2, STAGE = P_BYTES + Q_BYTES;
  static constexpr int STAGES = (225 * 1024 - EPI_WARPS * SIDE) / STAGE < 8 ? (225 * 1024 - EPI_WARPS * SIDE) / STAGE : 8;
  static constexpr int SMEM = STAGES * STAGE + EPI_WARPS * SIDE + 1024 + 256;
  static constexpr int TMEM = 2 * BN;
};

struct Shape {
  int m, n;                        // of each group
  int kblocks, kblocks0;           // all, and those of the first operands (the others' follow)
  int row_tiles, col_tiles, groups, splits, per_split;
  int band;                        // row tiles that share a walk over the columns
  int units;
  int a_turned, b_turned;          // operands lie across K
  int half;                        // f16, else bf16
};
struct Maps {
  CUtensorMap a[MAX_GROUPS], b[MAX_GROUPS];
};

struct Unit {
  int row, col, group, split;
};
__device__ __forceinline__ Unit unit_of(const Shape& s, int u) {
  Unit t;
  const int tiles = s.row_tiles * s.col_tiles;
  const int gs = u / tiles;
  u -= gs * tiles;
  t.split = gs / s.groups;
  t.group = gs - t.split * s.groups;
  const int per = s.band * s.col_tiles, band = u / per;
  u -= band * per;
  const int rows = min(s.band, s.row_tiles - band * s.band);
  t.col = u / rows;
  t.row = band * s.band + u - t.col * rows;
  return t;
}

__device__ __forceinline__ unsigned smem_u32(const void* p) {
  return static_cast<unsigned>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ unsigned in_block(unsigned addr, unsigned rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ bool bar_try(unsigned long long* b, unsigned phase) {
  unsigned ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
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
constexpr unsigned long long PATIENCE = 2000000000ull;  // every wait ends after 2 s

// False when the phase never completed, or at once when another role gave up.
static __device__ __noinline__ bool bar_wait_slow(unsigned long long* b, unsigned phase, volatile int* gave_up) {
  const unsigned long long t0 = now();
  while (true) {
    for (int i = 0; i < 64; ++i)
      if (bar_try(b, phase)) return true;
    if (*gave_up || now() - t0 > PATIENCE) return false;
  }
}
__device__ __forceinline__ bool bar_wait(unsigned long long* b, unsigned phase, volatile int* gave_up) {
  return bar_try(b, phase) || bar_wait_slow(b, phase, gave_up);
}

// Shared-memory descriptors, 128-byte swizzle.  K-major: 8 rows of 128 bytes
// make a group.  Across K: 64 columns to a row of 128 bytes, a row for each k;
// the next 64 columns lie a box further.
__device__ __forceinline__ unsigned long long desc_k(unsigned at) {
  return ((at >> 4) & 0x3FFFull) | (1ull << 16) | ((1024ull >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ unsigned long long desc_turned(unsigned at) {
  return ((at >> 4) & 0x3FFFull) | ((static_cast<unsigned long long>(BOX) >> 4) << 16) | ((1024ull >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// 32 columns of the thread's row of an accumulator: the load, and the wait for it,
// which takes the registers along so that nothing reads them before.
__device__ __forceinline__ void tmem_issue32(unsigned taddr, unsigned (&q)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];"
      : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]), "=r"(q[8]),
        "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15]), "=r"(q[16]),
        "=r"(q[17]), "=r"(q[18]), "=r"(q[19]), "=r"(q[20]), "=r"(q[21]), "=r"(q[22]), "=r"(q[23]), "=r"(q[24]),
        "=r"(q[25]), "=r"(q[26]), "=r"(q[27]), "=r"(q[28]), "=r"(q[29]), "=r"(q[30]), "=r"(q[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait32(unsigned (&q)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(q[0]), "+r"(q[1]), "+r"(q[2]), "+r"(q[3]), "+r"(q[4]), "+r"(q[5]), "+r"(q[6]), "+r"(q[7]),
                 "+r"(q[8]), "+r"(q[9]), "+r"(q[10]), "+r"(q[11]), "+r"(q[12]), "+r"(q[13]), "+r"(q[14]),
                 "+r"(q[15]), "+r"(q[16]), "+r"(q[17]), "+r"(q[18]), "+r"(q[19]), "+r"(q[20]), "+r"(q[21]),
                 "+r"(q[22]), "+r"(q[23]), "+r"(q[24]), "+r"(q[25]), "+r"(q[26]), "+r"(q[27]), "+r"(q[28]),
                 "+r"(q[29]), "+r"(q[30]), "+r"(q[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld32(unsigned taddr, float (&v)[32]) {
  unsigned q[32];
  tmem_issue32(taddr, q);
  tmem_wait32(q);
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(q[j]);
}

__device__ __forceinline__ uint4 lds128(unsigned addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(unsigned addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Two values rounded to a word of 16-bit elements; the two elements of one.
__device__ __forceinline__ unsigned pack2(float a, float b, int half) {
  if (half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float2 unpack2(unsigned w, int half) {
  if (half) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// What a warp's epilogue knows of its tile: 32 rows from row0 on, of which the
// thread's accumulator row is row0 + lane, and where it may keep 4 KB.
struct Spot {
  int lane, quad, part, row0, unit_col, group, split;
  int odd;        // every other tile of the block
  unsigned side;
  bool dead;  // a wait ran out: results are NaNs
};

// A warp's 32 x 32 values as 16-bit elements: each thread's row into shared
// memory (64 bytes a row, 16-byte pieces exchanged so that neither direction meets
// a bank twice) and from there to memory, eight rows an instruction.
__device__ __forceinline__ void put16(const Spot& s, const unsigned (&w)[16], unsigned short* out, long long ld, int m,
                                      int n, int col0, int vec) {
  const unsigned mine = s.side + s.lane * 64, turn = (s.lane >> 1) & 3;
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 4; ++p) sts128(mine + ((p ^ turn) << 4), make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]));
  __syncwarp();
  if (vec && col0 + CHUNK <= n) {
    const int p = s.lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (s.lane >> 2);
      const uint4 x = lds128(s.side + r * 64 + ((p ^ ((r >> 1) & 3)) << 4));
      if (s.row0 + r < m) *reinterpret_cast<uint4*>(out + (s.row0 + r) * ld + col0 + p * 8) = x;
    }
  } else {  // a column a lane
    const int col = col0 + s.lane, p = s.lane >> 3;
    if (col < n) {
      for (int r = 0; r < 32 && s.row0 + r < m; ++r) {
        unsigned short x;
        asm volatile("ld.shared.u16 %0, [%1];"
                     : "=h"(x)
                     : "r"(s.side + r * 64 + ((p ^ ((r >> 1) & 3)) << 4) + (s.lane & 7) * 2)
                     : "memory");
        out[(s.row0 + r) * ld + col] = x;
      }
    }
  }
}

// The same in 32 bits (128 bytes a row), left in shared memory for reads by row.
__device__ __forceinline__ void stage32(const Spot& s, const float (&v)[32]) {
  const unsigned mine = s.side + s.lane * 128, turn = s.lane & 7;
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 8; ++p)
    sts128(mine + ((p ^ turn) << 4), make_uint4(__float_as_uint(v[4 * p]), __float_as_uint(v[4 * p + 1]),
                                                __float_as_uint(v[4 * p + 2]), __float_as_uint(v[4 * p + 3])));
  __syncwarp();
}
// Four columns (4 p ...) of row r of them.
__device__ __forceinline__ float4 staged(const Spot& s, int r, int p) {
  const uint4 x = lds128(s.side + r * 128 + ((p ^ (r & 7)) << 4));
  return make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w));
}

// The lane's column of row r of them.
__device__ __forceinline__ float staged1(const Spot& s, int r) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];"
               : "=f"(x)
               : "r"(s.side + r * 128 + (((s.lane >> 2) ^ (r & 7)) << 4) + (s.lane & 3) * 4)
               : "memory");
  return x;
}

// A warp's 32 x 32 values in 32 bits to memory.
__device__ __forceinline__ void put32(const Spot& s, const float (&v)[32], float* out, long long ld, int m, int n, int col0,
                                      int vec) {
  stage32(s, v);
  if (vec && col0 + CHUNK <= n) {
    const int q = s.lane & 7;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + (s.lane >> 3);
      const float4 x = staged(s, r, q);
      if (s.row0 + r < m) *reinterpret_cast<float4*>(out + (s.row0 + r) * ld + col0 + q * 4) = x;
    }
  } else {  // a column a lane
    const int col = col0 + s.lane;
    if (col < n)
      for (int r = 0; r < 32 && s.row0 + r < m; ++r) out[(s.row0 + r) * ld + col] = staged1(s, r);
  }
}

// ------------------------------------------------------------------ the kernel

// EPI: static constexpr bool DUAL (B's tiles hold half their columns of each of
// two operands); Params; a State that is constructed for a tile (loads that need
// no accumulator), whose chunk() takes 32 columns, and whose end() all warps call.
template <typename TILE, typename EPI>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Shape a,
                const __grid_constant__ typename EPI::Params params) {
  constexpr int CTAS = TILE::CTAS, BN = TILE::BN, STAGES = TILE::STAGES;
  constexpr int COLS = EPI::DUAL ? BN / 2 : BN;  // columns of the result
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char* side = smem + STAGES * TILE::STAGE;
  unsigned long long* full = reinterpret_cast<unsigned long long*>(side + EPI_WARPS * SIDE);
  unsigned long long* empty = full + STAGES;
  unsigned long long* acc_full = empty + STAGES;
  unsigned long long* acc_empty = acc_full + 2;
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(acc_empty + 2);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 1 ? 0 : blockIdx.x & 1;
  const int first = blockIdx.x / CTAS, stride = gridDim.x / CTAS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&empty[i])));
    }
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&acc_full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&acc_empty[i])), "r"(CTAS * EPI_WARPS));
    }
    *gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if (CTAS == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(TILE::TMEM)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(TILE::TMEM)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (CTAS == 2) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {  // operands
      // what earlier kernels wrote is read through the async proxy
      asm volatile("fence.proxy.async.global;" ::: "memory");
      int n = 0;  // stages used so far
      bool stop = false;
      for (int u = first; u < a.units && !stop; u += stride) {
        const Unit t = unit_of(a, u);
        const int kb0 = t.split * a.per_split, kb1 = min(a.kblocks, kb0 + a.per_split);
        const int p0 = t.row * TILE::M + rank * 128;
        const int q0 = EPI::DUAL ? t.col * COLS : t.col * BN + rank * TILE::QN;
        for (int kb = kb0; kb < kb1; ++kb, ++n) {
          const int i = n % STAGES;
          if (n >= STAGES && !bar_wait(&empty[i], (n / STAGES - 1) & 1, gave_up)) {
            *gave_up = 1;
            stop = true;
            break;
          }
          const unsigned st = smem_u32(smem) + i * TILE::STAGE;
          unsigned bar = smem_u32(&full[i]);
          if (rank == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(CTAS * TILE::STAGE)
                         : "memory");
          if (CTAS == 2) bar = in_block(bar, 0);
          auto load = [&](const CUtensorMap* map, unsigned to, int x0, int y0) {
            if (CTAS == 1)
              asm volatile(
                  "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
                  "[%2];" ::"r"(to),
                  "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(x0), "r"(y0)
                  : "memory");
            else
              asm volatile(
                  "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                  "[%1, {%3, %4}], [%2];" ::"r"(to),
                  "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(x0), "r"(y0)
                  : "memory");
          };
          const int second = kb >= a.kblocks0;
          const int k0 = (second ? kb - a.kblocks0 : kb) * BK, which = t.group + second;
          const CUtensorMap *pa = &maps.a[which], *pb = &maps.b[which];
          if (a.a_turned) {
#pragma unroll
            for (int h = 0; h < 2; ++h) load(pa, st + h * BOX, p0 + h * 64, k0);
          } else {
            load(pa, st, k0, p0);
          }
          const unsigned sq = st + TILE::P_BYTES;
          if (EPI::DUAL) {
            if (CTAS == 2) {
              load(&maps.b[rank], sq, k0, q0);
            } else {
              load(&maps.b[0], sq, k0, q0);
              load(&maps.b[1], sq + TILE::Q_BYTES / 2, k0, q0);
            }
          } else if (a.b_turned) {
#pragma unroll
            for (int h = 0; h < TILE::QN / 64; ++h) load(pb, sq + h * BOX, q0 + h * 64, k0);
          } else {
            load(pb, sq, k0, q0);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {  // products
      // D in 32 bits; operand types (bf16: 1) in bits 7 and 10; across K: bits 15 and 16
      const unsigned idesc = (1u << 4) | (a.half ? 0u : (1u << 7) | (1u << 10)) | (a.a_turned ? 1u << 15 : 0u) |
                             (a.b_turned ? 1u << 16 : 0u) | (static_cast<unsigned>(BN >> 3) << 17) |
                             (static_cast<unsigned>(TILE::M >> 4) << 24);
      const unsigned long long p_step = a.a_turned ? (16 * 128) >> 4 : 32 >> 4;
      const unsigned long long q_step = a.b_turned ? (16 * 128) >> 4 : 32 >> 4;
      int n = 0, c = 0;  // stages, accumulators used so far
      bool stop = false;
      for (int u = first; u < a.units && !stop; u += stride, ++c) {
        const Unit t = unit_of(a, u);
        const int kb0 = t.split * a.per_split, kb1 = min(a.kblocks, kb0 + a.per_split);
        if (c >= 2 && !bar_wait(&acc_empty[c & 1], (c / 2 - 1) & 1, gave_up)) {
          *gave_up = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned acc = tmem + (c & 1) * BN;
        for (int kb = kb0; kb < kb1; ++kb, ++n) {
          const int i = n % STAGES;
          if (!bar_wait(&full[i], (n / STAGES) & 1, gave_up)) {
            *gave_up = 1;
            stop = true;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const unsigned st = smem_u32(smem) + i * TILE::STAGE;
          const unsigned long long pd = a.a_turned ? desc_turned(st) : desc_k(st);
          const unsigned long long qd = a.b_turned ? desc_turned(st + TILE::P_BYTES) : desc_k(st + TILE::P_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const unsigned more = (kb > kb0 || k > 0) ? 1u : 0u;
            if (CTAS == 1)
              asm volatile(
                  "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                  " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(acc),
                  "l"(pd + k * p_step), "l"(qd + k * q_step), "r"(idesc), "r"(more)
                  : "memory");
            else
              asm volatile(
                  "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                  " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(acc),
                  "l"(pd + k * p_step), "l"(qd + k * q_step), "r"(idesc), "r"(more)
                  : "memory");
          }
          auto commit = [&](unsigned long long* bar) {
            if (CTAS == 1)
              asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                               smem_u32(bar))
                           : "memory");
            else
              asm volatile(
                  "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], "
                  "%1;" ::"r"(smem_u32(bar)),
                  "h"(static_cast<unsigned short>(3))
                  : "memory");
          };
          commit(&empty[i]);
          if (kb + 1 == kb1) commit(&acc_full[c & 1]);
        }
      }
    }
  } else {  // epilogues
    const int quad = warp & 3, part = (warp - 2) >> 2;  // 32 rows; which of their chunks
    Spot s;
    s.lane = lane, s.quad = quad, s.part = part;
    s.side = smem_u32(side) + (warp - 2) * SIDE;
    s.dead = false;
    int c = 0;
    for (int u = first; u < a.units; u += stride, ++c) {
      const Unit t = unit_of(a, u);
      s.row0 = t.row * TILE::M + rank * 128 + quad * 32;
      s.unit_col = t.col, s.group = t.group, s.split = t.split;
      const int chunks = (min(COLS, a.n - t.col * COLS) + CHUNK - 1) / CHUNK;
      typename EPI::State e(params, a, s);
      if (!s.dead && !bar_wait(&acc_full[c & 1], (c / 2) & 1, gave_up)) {
        s.dead = true;
        *gave_up = 1;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned acc = tmem + (static_cast<unsigned>(quad * 32) << 16) + (c & 1) * BN;
      // a warp without a row of the result still has to say that it is done
      if (s.row0 < a.m)
        for (int ch = part; ch < chunks; ch += PARTS) e.chunk(params, a, s, t.col * COLS + ch * CHUNK, acc + ch * CHUNK, COLS);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0 && !s.dead) {  // the accumulator is free
        const unsigned bar = CTAS == 1 ? smem_u32(&acc_empty[c & 1]) : in_block(smem_u32(&acc_empty[c & 1]), 0);
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
      }
      s.odd = c & 1;
      e.end(params, a, s);
    }
  }
  __syncwarp();
  // A role that gave up leaves copies and products in flight: let them land
  // before shared and tensor memory are given back.
  __syncthreads();
  if (*gave_up) {
    const unsigned long long t0 = now();
    while (now() - t0 < 5000000ull) {
    }
  }
  if (CTAS == 2) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1) {
    if (CTAS == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TILE::TMEM) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TILE::TMEM) : "memory");
  }
}

// ------------------------------------------------------------------ host

// A 16-bit matrix that TMA can read: 16-byte aligned rows.
struct Mat {
  const void* p;
  long long ld;
};
inline bool tma_ready(const void* p, long long ld, long long rows) {
  return aligned(p, 16) && (rows <= 1 || ld % 8 == 0);
}
inline long long round_up(long long x, long long to) { return (x + to - 1) / to * to; }
inline size_t room(size_t bytes) { return (bytes + 255) / 256 * 256; }

struct Problem {
  int device, half;
  long long m, n, k, k0;  // k0: K of the first operands when there are two in a row (else k)
  int groups;             // products of one shape in one launch
  bool a_turned, b_turned;
  Mat a[MAX_GROUPS], b[MAX_GROUPS];
};

// How a problem is laid out over the device: the tile with the smallest estimated
// time, from measured costs of 64 elements of K (a pair of blocks on 256 x 256: 0.45
// us, single blocks on 128 x 128: 0.47 and 128 x 64: 0.40, all of them L2's rate) and
// 4 us for a product's start and its last epilogue; each tile is a wave's part.  A
// split costs its partial sums' way to memory and back at 4 TB/s, and a launch of 4 us.
struct Plan {
  int tile;  // 0: 2 x 256, 1: 128, 2: 64
  int splits;
  double us;
};
inline Plan plan_for(long long m, long long n, long long kblocks, int groups, bool dual, bool may_split, int sms) {
  struct { int m, n, workers; double us; } const tiles[3] = {{256, 256, sms / 2, 0.45}, {128, 128, sms, 0.47}, {128, 64, sms, 0.40}};
  Plan best = {0, 1, 1e30};
  for (int i = 0; i < 3; ++i) {
    const int cols = dual ? tiles[i].n / 2 : tiles[i].n;
    const long long count = groups * ((m + tiles[i].m - 1) / tiles[i].m) * ((n + cols - 1) / cols);
    for (int s = 1; s <= (may_split ? 16 : 1); ++s) {
      const long long per = (kblocks + s - 1) / s;
      if (s > 1 && (per < 8 || (kblocks + per - 1) / per != s)) continue;
      const double rounds = static_cast<double>((count * s + tiles[i].workers - 1) / tiles[i].workers);
      double us = rounds * per * tiles[i].us + 4.0;
      if (s > 1) us += 4.0 + 8e-6 * s * groups * static_cast<double>(m) * n / 4.0;
      if (us < best.us * 0.97) best = {i, s, us};
    }
  }
  return best;
}

template <typename TILE, typename EPI>
cudaError_t start_tile(const Problem& p, Shape s, const typename EPI::Params& params, int sms, cudaStream_t st, int* bad) {
  Maps maps = {};
  const int cols = EPI::DUAL ? TILE::BN / 2 : TILE::BN;
  s.row_tiles = static_cast<int>((p.m + TILE::M - 1) / TILE::M);
  s.col_tiles = static_cast<int>((p.n + cols - 1) / cols);
  // about as many rows as columns under way at a time
  s.band = TILE::M == 256 ? 8 : 16;
  const long long units = static_cast<long long>(s.row_tiles) * s.col_tiles * s.groups * s.splits;
  *bad = units > 0x3fffffffll ? fail("too many tiles in one product") : 0;
  s.units = static_cast<int>(units);
  const int operands = EPI::DUAL ? 2 : std::max(s.groups, s.kblocks0 < s.kblocks ? 2 : 1);
  for (int i = 0; i < operands && !*bad; ++i) {
    const long long k = s.kblocks0 == s.kblocks ? p.k : i ? p.k - p.k0 : p.k0;
    if (!EPI::DUAL || i == 0)
      *bad |= p.a_turned ? ad_b200_internal::tmap_2d_16(p.a[i].p, k, p.m, p.a[i].ld, 64, 64, &maps.a[i])
                         : ad_b200_internal::tmap_2d_16(p.a[i].p, p.m, k, p.a[i].ld, 128, 64, &maps.a[i]);
    const int rows = EPI::DUAL && TILE::CTAS == 1 ? TILE::QN / 2 : TILE::QN;
    *bad |= p.b_turned ? ad_b200_internal::tmap_2d_16(p.b[i].p, k, p.n, p.b[i].ld, 64, 64, &maps.b[i])
                       : ad_b200_internal::tmap_2d_16(p.b[i].p, p.n, k, p.b[i].ld, rows, 64, &maps.b[i]);
  }
  if (*bad) return cudaSuccess;
  int room = 0;
  cudaError_t e = shared_room<gemm_kernel<TILE, EPI>>(&room);
  if (e != cudaSuccess) return e;
  if (room < TILE::SMEM) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t c = {};
  c.blockDim = dim3(THREADS);
  c.dynamicSmemBytes = TILE::SMEM;
  c.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = TILE::CTAS;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  // blocks or pairs of them at a time: more would start when others have ended, with a whole share of the units each
  static std::atomic<int> resident[64];
  int workers = p.device < 64 ? resident[p.device].load() : 0;
  if (!workers) {
    c.gridDim = dim3(sms / TILE::CTAS * TILE::CTAS);
    e = cudaOccupancyMaxActiveClusters(&workers, gemm_kernel<TILE, EPI>, &c);
    if (e != cudaSuccess) return e;
    workers = std::max(1, std::min(workers, sms / TILE::CTAS));
    if (p.device < 64) resident[p.device] = workers;
  }
  c.gridDim = dim3(std::min(s.units, workers) * TILE::CTAS);
  return cudaLaunchKernelEx(&c, gemm_kernel<TILE, EPI>, maps, s, params);
}

// Launches a problem under a plan.  0, or 1 with an error set.
template <typename EPI>
int start(const char* who, const Problem& p, const Plan& plan, const typename EPI::Params& params, int sms, cudaStream_t st) {
  Shape s = {};
  s.m = static_cast<int>(p.m), s.n = static_cast<int>(p.n);
  s.kblocks0 = static_cast<int>((p.k0 + BK - 1) / BK);
  s.kblocks = s.kblocks0 + static_cast<int>((p.k - p.k0 + BK - 1) / BK);
  s.groups = p.groups;
  s.per_split = (s.kblocks + plan.splits - 1) / plan.splits;
  s.splits = (s.kblocks + s.per_split - 1) / s.per_split;  // none without a share: nothing would end its wait
  s.a_turned = p.a_turned, s.b_turned = p.b_turned, s.half = p.half;
  int bad = 0;
  cudaError_t e = plan.tile == 0   ? start_tile<Tile<2, 256>, EPI>(p, s, params, sms, st, &bad)
                  : plan.tile == 1 ? start_tile<Tile<1, 128>, EPI>(p, s, params, sms, st, &bad)
                                   : start_tile<Tile<1, 64>, EPI>(p, s, params, sms, st, &bad);
  if (bad) return 1;
  if (e != cudaSuccess) return fail_cuda(who, e);
  return 0;
}

// ------------------------------------------------------------------ products to memory (gemm16.cu)

// A result: m x n of a type (AD_F32 or the operands'), added to what it holds
// when `accumulate`.
struct Out {
  void* p;
  long long ld;
};
// The products of a problem, times *alpha (device memory; NULL: 1), to out[group].
// `partial`: at least partial_bytes() of memory, 16-byte aligned.  With `sums`, a
// first or later part of a sum over products (one group): the partial sums stay in
// `partial` and only the `last` part's call writes the result.
struct Sums {
  bool first, last;
};
Plan store_plan(const Problem& p, int sms);
size_t partial_bytes(const Problem& p, const Plan& plan, bool sums);
int store_product(const char* who, const Problem& p, const Plan& plan, int type, const Out* out, bool accumulate,
                  const float* alpha, float* partial, const Sums* sums, int sms, cudaStream_t st);
// A copy of a 16-bit matrix whose rows TMA can read.
int pack_rows(const char* who, const void* p, long long ld, long long rows, long long cols, void* to, long long ld_to,
              cudaStream_t st);

}  // namespace adgemm

#endif
