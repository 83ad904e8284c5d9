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
// One kernel makes all products.  Its blocks (or pairs of blocks, whose tensor
// cores share a tile of 256 x 256) stay resident and take every so-many-th tile
// of one list: the steps in order, in a step the three products, in a product
// the matrices.  A tile waits only for the previous product of its own matrix, by
// a counter in memory, so that a batch leaves no gaps between products.  Within
// a block one warp brings operands by TMA, one issues the products into one of
// two accumulators, eight work on the other: 32 columns at a time they join
// the accumulator with what the epilogue needs of X or A, which a further warp
// has brought into shared memory ahead of them, and leave the result in its
// place, from where the last warp sends it off by TMA (lanes hold rows, so that
// direct loads and stores would touch 32 lines each).  A and B are symmetric:
// tiles on one side of the diagonal are computed and written twice.
//
// Operands: rows of X for X X^T and of the symmetric A for A A, K-major; for
// B X the rows of B, K-major, and X itself as it lies, N-major.  X is held as
// the sum of two f16 numbers, the larger of which is the operand: X crosses the
// bus as 2 + 2 bytes in each direction.
//
// Measured, five steps: 12 x 4096 x 1024 1290 us (649 TFLOP/s of the halves that
// symmetry leaves), 4096 x 4096 1400 to 1600 us (860 to 980), 512 x 512 119 us,
// where every product is a wait of 7.4 us.  A block's operands come from L2 at 60 to
// 80 GB/s, which accounts for half of the large case: its 6.5 GB of operands take
// 595 us at that rate, the epilogues' 2.4 GB 217, norm and load 103.  The rest, some
// 370 us, is not accounted for; the epilogues' reads of tensor memory, 8 columns
// at a time, and items of unequal cost dealt out in turn have not been measured apart.
#include <cuda.h>

#include <cmath>
#include <initializer_list>

#include "ops_common.cuh"

namespace {

using namespace adops;

constexpr int BK = 64;  // elements of K a stage: 128 bytes, the swizzle's width
constexpr int BOX = 64 * BK * 2;  // bytes of a TMA box: 64 rows
constexpr int EPI_WARPS = 8;
constexpr int LOADER = 2 + EPI_WARPS, STORER = LOADER + 1;  // warps that serve the epilogues
constexpr int THREADS = 32 * (STORER + 1);
constexpr int CHUNK_COLS = 32, CHUNK = 128 * CHUNK_COLS * 2;  // what an epilogue takes at a time: 128 rows of 16 bits
constexpr int MAX_STEPS = 32;
constexpr int NORM_BLOCKS = 64;  // blocks that share a matrix's norm

enum Phase { GRAM = 0, POLY = 1, UPDATE = 2 };

// Tiles: CTAS blocks work on one of 128 CTAS rows and BN columns.
template <int CTAS, int BN>
struct Tile {
  static constexpr int M = 128 * CTAS, N = BN;
  static constexpr int QN = BN / CTAS;  // columns whose operand a block holds
  static constexpr int P_BYTES = 128 * BK * 2, Q_BYTES = QN * BK * 2, STAGE = P_BYTES + Q_BYTES;
  // buffers of two chunks for the epilogues, by turns for each half of their warps
  // (six of them and a stage less: the same within 2%)
  static constexpr int SIDES = 4;
  static constexpr int STAGES = (224 * 1024 - SIDES * 2 * CHUNK) / STAGE;
  static constexpr int SMEM = STAGES * STAGE + SIDES * 2 * CHUNK + 1024 + 512;
  static constexpr int RATIO = M / N;  // column tiles beside a row tile on the diagonal
};

struct StepScale {
  float gram, poly_p, poly_q, up_p, up_q;
};

struct NsArgs {
  int count, m, n, steps;
  int ldx;            // a row of X (elements)
  int sym, up;        // tiles of a matrix in GRAM and POLY, in UPDATE
  int row_tiles, sym_cols;
  __half *hi[2], *lo;
  float *da, *db;
  void* out;
  int out_type, out_vec;
  long long out_batch, out_row, out_col;
  float out_scale;
  int* err;
  unsigned* ready;  // a matrix's finished tiles (counted once a block)
  StepScale step[MAX_STEPS];
};

// TMA maps.  Operands, swizzled over 128 bytes: boxes of 64 elements of K by 128
// rows, and by 64 (also 64 rows of K by 64 columns).  Chunks for the epilogues:
// boxes of 32 columns by 128 rows, swizzled over 64 bytes; transposed ones: 64
// columns by 32 rows.  X's larger part is there twice: a step reads one, writes the other.
enum {
  WIDE_X = 0, WIDE_A = 2, WIDE_B = 3, NARROW_X = 4, NARROW_A = 6,
  CHUNK_X = 7, CHUNK_LO = 9, CHUNK_A = 10, CHUNK_B = 11, TURNED_A = 12, TURNED_B = 13, MAPS = 14
};
struct Maps {
  CUtensorMap m[MAPS];
};

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
__device__ __noinline__ bool bar_wait_slow(unsigned long long* b, unsigned phase, volatile int* gave_up) {
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
__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __noinline__ bool count_wait(const unsigned* p, unsigned need, volatile int* gave_up) {
  if (load_acquire(p) >= need) return true;
  const unsigned long long t0 = now();
  while (true) {
    for (int i = 0; i < 32; ++i)
      if (load_acquire(p) >= need) return true;
    if (*gave_up || now() - t0 > PATIENCE) return false;
  }
}

// Shared-memory descriptors, 128-byte swizzle.  K-major: 8 rows of 128 bytes
// make a group.  N-major: 64 columns to a row of 128 bytes, a row for each k;
// the next 64 columns lie a box further.
__device__ __forceinline__ unsigned long long desc_k(const void* p) {
  return ((smem_u32(p) >> 4) & 0x3FFFull) | (1ull << 16) | ((1024ull >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ unsigned long long desc_n(const void* p) {
  return ((smem_u32(p) >> 4) & 0x3FFFull) | ((static_cast<unsigned long long>(BOX) >> 4) << 16) |
         ((1024ull >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void tmem_ld8(unsigned taddr, float (&r)[8]) {
  unsigned q[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = __uint_as_float(q[j]);
}

__device__ __forceinline__ uint4 lds128(unsigned addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts128(unsigned addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void sts16(unsigned addr, float v) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"(__half_as_ushort(__float2half_rn(v))) : "memory");
}
__device__ __forceinline__ float2 halves(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ unsigned packed(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}

// A box of 64 rows and 64 columns from or to a matrix.
__device__ __forceinline__ void box_load(const CUtensorMap* map, unsigned to, unsigned bar, int col, int row, int mat) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          to),
      "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(col), "r"(row), "r"(mat)
      : "memory");
}
__device__ __forceinline__ void box_store(const CUtensorMap* map, unsigned from, int col, int row, int mat) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<unsigned long long>(map)),
               "r"(from), "r"(col), "r"(row), "r"(mat)
               : "memory");
}
__device__ __forceinline__ void bar_expect(unsigned long long* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Eight elements of a row of the result.
__device__ __forceinline__ void store_result(const NsArgs& a, long long mat, int row, int col0, float (&v)[8], int inside) {
  const long long at = mat * a.out_batch + row * a.out_row + col0 * a.out_col;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= a.out_scale;
  if (a.out_vec && inside >= 8) {
    if (a.out_type == AD_F32) {
      float* p = static_cast<float*>(a.out) + at;
      store_vec<float, 4>(p, {{v[0], v[1], v[2], v[3]}});
      store_vec<float, 4>(p + 4, {{v[4], v[5], v[6], v[7]}});
    } else if (a.out_type == AD_BF16) {
      Vec<__nv_bfloat16, 8> w;
#pragma unroll
      for (int j = 0; j < 8; ++j) w.v[j] = from_float<__nv_bfloat16>(v[j]);
      store_vec<__nv_bfloat16, 8>(static_cast<__nv_bfloat16*>(a.out) + at, w);
    } else {
      Vec<__half, 8> w;
#pragma unroll
      for (int j = 0; j < 8; ++j) w.v[j] = from_float<__half>(v[j]);
      store_vec<__half, 8>(static_cast<__half*>(a.out) + at, w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < inside) store_any(a.out, a.out_type, at + j * a.out_col, v[j]);
  }
}

// One item of the list.
struct Item {
  int step, phase, mat, row, col;  // row, col: of tiles
};
template <typename TILE>
__device__ __forceinline__ Item item_of(const NsArgs& a, int t) {
  Item i;
  const int sym_all = a.count * a.sym, per_step = 2 * sym_all + a.count * a.up;
  i.step = t / per_step;
  int r = t - i.step * per_step;
  if (r < 2 * sym_all) {
    i.phase = r >= sym_all ? POLY : GRAM;
    r -= i.phase * sym_all;
    i.mat = r / a.sym;
    r -= i.mat * a.sym;
    for (i.row = 0;; ++i.row) {
      const int n = min((i.row + 1) * TILE::RATIO, a.sym_cols);
      if (r < n) break;
      r -= n;
    }
    i.col = r;
  } else {
    i.phase = UPDATE;
    r -= 2 * sym_all;
    i.mat = r / a.up;
    r -= i.mat * a.up;
    i.col = r / a.row_tiles;
    i.row = r - i.col * a.row_tiles;
  }
  return i;
}

// Chunks of an item's tile that are not wholly past the matrix.
template <typename TILE>
__device__ __forceinline__ int chunks_of(const NsArgs& a, const Item& i) {
  const int width = (i.phase == UPDATE ? a.n : a.m) - i.col * TILE::N;
  return min(TILE::N, width + CHUNK_COLS - 1) / CHUNK_COLS;
}
// Whether the right operand is (part of) the left one: tiles on the diagonal of
// A A^T.  What a block brings from L2 bounds these products, so it comes once.
template <typename TILE>
__device__ __forceinline__ bool on_diagonal(const Item& i) {
  return i.phase != UPDATE && i.col / TILE::RATIO == i.row;
}
// Tiles of its matrix that have to be finished before an item's operands are there.
__device__ __forceinline__ unsigned needed(const NsArgs& a, const Item& i, int ctas) {
  return static_cast<unsigned>(ctas) * (i.step * (2 * a.sym + a.up) + i.phase * a.sym);
}

template <int CTAS, int BN>
__global__ void __launch_bounds__(THREADS, 1)
    ns_kernel(const __grid_constant__ Maps maps, const __grid_constant__ NsArgs a) {
  using TILE = Tile<CTAS, BN>;
  constexpr int STAGES = TILE::STAGES, SIDES = TILE::SIDES;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  // the epilogues' buffers behind the operands' stages
  unsigned char* side = smem + STAGES * TILE::STAGE;
  unsigned long long* full = reinterpret_cast<unsigned long long*>(side + SIDES * 2 * CHUNK);
  unsigned long long* empty = full + STAGES;
  unsigned long long* acc_full = empty + STAGES;
  unsigned long long* acc_empty = acc_full + 2;
  unsigned long long* side_full = acc_empty + 2;   // a buffer holds what the epilogue needs
  unsigned long long* side_done = side_full + SIDES;   // ... and then its results
  unsigned long long* side_empty = side_done + SIDES;  // ... which are under way
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(side_empty + SIDES);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 1 ? 0 : blockIdx.x & 1;
  const int first = blockIdx.x / CTAS, stride = gridDim.x / CTAS;
  const int items = a.steps * a.count * (2 * a.sym + a.up);

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&empty[i])));
    }
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&acc_full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&acc_empty[i])), "r"(CTAS * EPI_WARPS));
    }
    for (int i = 0; i < SIDES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&side_full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&side_done[i])), "r"(EPI_WARPS / 2));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&side_empty[i])));
    }
    *gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if (CTAS == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(2 * BN)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(2 * BN)
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
      int n = 0;      // stages used so far
      for (int t = first; t < items; t += stride) {
        const Item it = item_of<TILE>(a, t);
        if (!count_wait(a.ready + it.mat, needed(a, it, CTAS), gave_up)) {
          *gave_up = 1;
          atomicExch(a.err, 1);
          break;
        }
        // what others wrote through the generic proxy is read through the async one
        asm volatile("fence.proxy.async.global;" ::: "memory");
        const int x = it.step & 1;
        const CUtensorMap* p = &maps.m[it.phase == GRAM ? WIDE_X + x : it.phase == POLY ? WIDE_A : WIDE_B];
        const CUtensorMap* q = it.phase == UPDATE ? &maps.m[NARROW_X + x]
                               : TILE::QN == 128  ? p
                                                  : &maps.m[it.phase == GRAM ? NARROW_X + x : NARROW_A];
        const int kblocks = ((it.phase == GRAM ? a.n : a.m) + BK - 1) / BK;
        const int p0 = it.row * TILE::M + rank * 128;
        const int q0 = it.col * BN + rank * TILE::QN;
        const bool once = on_diagonal<TILE>(it);
        bool stop = false;
        for (int kb = 0; kb < kblocks; ++kb, ++n) {
          const int i = n % STAGES;
          if (n >= STAGES && !bar_wait(&empty[i], (n / STAGES - 1) & 1, gave_up)) {
            *gave_up = 1;
            atomicExch(a.err, 2);
            stop = true;
            break;
          }
          unsigned char* st = smem + i * TILE::STAGE;
          unsigned bar = smem_u32(&full[i]);
          if (rank == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                         "r"(CTAS * (once ? TILE::P_BYTES : TILE::STAGE))
                         : "memory");
          if (CTAS == 2) bar = in_block(bar, 0);
          auto load = [&](const CUtensorMap* map, unsigned char* to, int x0, int y0) {
            if (CTAS == 1)
              asm volatile(
                  "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
                  "[%2];" ::"r"(smem_u32(to)),
                  "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(x0), "r"(y0), "r"(it.mat)
                  : "memory");
            else
              asm volatile(
                  "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
                  "[%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(to)),
                  "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(x0), "r"(y0), "r"(it.mat)
                  : "memory");
          };
          load(p, st, kb * BK, p0);
          unsigned char* sq = st + TILE::P_BYTES;
          if (it.phase == UPDATE) {
#pragma unroll
            for (int h = 0; h < TILE::QN / 64; ++h) load(q, sq + h * BOX, q0 + h * 64, kb * BK);
          } else if (!once) {
            load(q, sq, kb * BK, q0);
          }
        }
        if (stop) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {  // products
      // D f32, operands f16; bit 16: the right operand is N-major
      constexpr unsigned IDESC =
          (1u << 4) | (static_cast<unsigned>(BN >> 3) << 17) | (static_cast<unsigned>(TILE::M >> 4) << 24);
      int n = 0, c = 0;  // stages, accumulators used so far
      for (int t = first; t < items; t += stride, ++c) {
        const Item it = item_of<TILE>(a, t);
        const int kblocks = ((it.phase == GRAM ? a.n : a.m) + BK - 1) / BK;
        if (c >= 2 && !bar_wait(&acc_empty[c & 1], (c / 2 - 1) & 1, gave_up)) {
          *gave_up = 1;
          atomicExch(a.err, 3);
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned acc = tmem + (c & 1) * BN;
        const unsigned idesc = IDESC | (it.phase == UPDATE ? 1u << 16 : 0u);
        const int q_at = on_diagonal<TILE>(it) ? it.col % TILE::RATIO * (TILE::QN * BK * 2) : TILE::P_BYTES;
        const unsigned long long q_step = it.phase == UPDATE ? (16 * 128) >> 4 : 32 >> 4;
        bool stop = false;
        for (int kb = 0; kb < kblocks; ++kb, ++n) {
          const int i = n % STAGES;
          if (!bar_wait(&full[i], (n / STAGES) & 1, gave_up)) {
            *gave_up = 1;
            atomicExch(a.err, 4);
            stop = true;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          unsigned char* st = smem + i * TILE::STAGE;
          const unsigned long long pd = desc_k(st);
          const unsigned long long qd = it.phase == UPDATE ? desc_n(st + q_at) : desc_k(st + q_at);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const unsigned more = (kb > 0 || k > 0) ? 1u : 0u;
            if (CTAS == 1)
              asm volatile(
                  "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                  " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(acc),
                  "l"(pd + k * (32 >> 4)), "l"(qd + k * q_step), "r"(idesc), "r"(more)
                  : "memory");
            else
              asm volatile(
                  "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                  " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(acc),
                  "l"(pd + k * (32 >> 4)), "l"(qd + k * q_step), "r"(idesc), "r"(more)
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
          if (kb + 1 == kblocks) commit(&acc_full[c & 1]);
        }
        if (stop) break;
      }
    }
  } else if (warp < LOADER) {  // epilogues
    const int quad = warp & 3, part = (warp - 2) >> 2;  // 32 rows; every other chunk
    const int r = quad * 32 + lane;
    const unsigned swizzle = ((r >> 1) & 3) << 4;
    int c = 0, e = 0;   // accumulators, chunks used so far
    bool dead = false;  // a wait ran out: the rest of the list is walked without work, the result shows it
    for (int t = first; t < items; t += stride, ++c) {
      const Item it = item_of<TILE>(a, t);
      const int chunks = chunks_of<TILE>(a, it);
      const int row = it.row * TILE::M + rank * 128 + r;
      const bool row_in = row < a.m;
      const long long row_all = static_cast<long long>(it.mat) * a.m + row;
      const bool last = it.phase == UPDATE && it.step + 1 == a.steps;
      const bool mirror = it.phase != UPDATE && !on_diagonal<TILE>(it);
      // X = p X + q (acc + d X_hi);  B = p A + q (acc + (d_row + d_col) A);  A = q acc
      const StepScale& sc = a.step[it.step];
      const float p = it.phase == UPDATE ? sc.up_p : sc.poly_p;
      const float q = it.phase == UPDATE ? sc.up_q : it.phase == POLY ? sc.poly_q : sc.gram;
      bool waited = false;  // for the accumulator: after the loads below are under way
      auto wait_acc = [&] {
        if (!dead && !bar_wait(&acc_full[c & 1], (c / 2) & 1, gave_up)) dead = true;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        waited = true;
      };
      const unsigned acc = tmem + (static_cast<unsigned>(quad * 32) << 16) + (c & 1) * BN;
      for (int ch = (e ^ part) & 1; ch < chunks; ch += 2) {
        const int b = (e + ch) % SIDES;
        if (!dead && !bar_wait(&side_full[b], ((e + ch) / SIDES) & 1, gave_up)) dead = true;
        const int col0 = it.col * BN + ch * CHUNK_COLS;
        const unsigned s0 = smem_u32(side) + b * (2 * CHUNK), s1 = s0 + CHUNK;
        float d = 0.0f, mine = 0.0f;  // the row's diagonal element; lane j: column j's
        if (it.phase != GRAM) {
          if (row_in) d = __ldcg((it.phase == POLY ? a.da : a.db) + row_all);
          if (it.phase == POLY && col0 + lane < a.m) mine = __ldcg(a.da + static_cast<long long>(it.mat) * a.m + col0 + lane);
        }
        if (!waited) wait_acc();
        if (dead) {
          *gave_up = 1;
          atomicExch(a.err, 5);
        }
#pragma unroll 1
        for (int g = 0; g < CHUNK_COLS / 8; ++g) {
          float v[8];
          tmem_ld8(acc + ch * CHUNK_COLS + g * 8, v);
          const unsigned at = r * (2 * CHUNK_COLS) + ((g * 16) ^ swizzle);
          uint4 x = make_uint4(0, 0, 0, 0), y = x;
          if (it.phase != GRAM) x = lds128(s0 + at);
          if (it.phase == UPDATE) y = lds128(s1 + at);
          const unsigned xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
          const int diagonal = it.phase == UPDATE ? -1 : row - col0 - g * 8;  // which of the 8, if one
          float on_diagonal = 0.0f;
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            const float2 xh = halves(xs[k / 2]), xl = halves(ys[k / 2]);
            if (k == diagonal) on_diagonal = v[k];
            if (k + 1 == diagonal) on_diagonal = v[k + 1];
            const float d0 = it.phase == POLY ? d + __shfl_sync(0xffffffffu, mine, g * 8 + k) : d;
            const float d1 = it.phase == POLY ? d + __shfl_sync(0xffffffffu, mine, g * 8 + k + 1) : d;
            v[k] = fmaf(p, xh.x + xl.x, q * fmaf(d0, xh.x, v[k]));
            v[k + 1] = fmaf(p, xh.y + xl.y, q * fmaf(d1, xh.y, v[k + 1]));
            if (k == diagonal) v[k] = 0.0f;
            if (k + 1 == diagonal) v[k + 1] = 0.0f;
          }
          if (diagonal >= 0 && diagonal < 8 && row_in) {
            if (it.phase == GRAM)
              a.da[row_all] = q * on_diagonal;
            else
              a.db[row_all] = fmaf(p, d, q * fmaf(d, d, on_diagonal));
          }
          if (last) {
            if (dead) {
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = __int_as_float(0x7fffffff);
            }
            const int inside = row_in ? a.n - col0 - g * 8 : 0;
            if (inside > 0) store_result(a, it.mat, row, col0 + g * 8, v, inside);
            continue;
          }
          unsigned w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = packed(v[2 * k], v[2 * k + 1]);
          sts128(s0 + at, make_uint4(w[0], w[1], w[2], w[3]));
          if (it.phase == UPDATE) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 h = halves(w[k]);
              w[k] = packed(v[2 * k] - h.x, v[2 * k + 1] - h.y);
            }
            sts128(s1 + at, make_uint4(w[0], w[1], w[2], w[3]));
          } else if (mirror) {  // rows and columns exchanged: 32 rows of 64 columns for each 64 rows here
#pragma unroll
            for (int j = 0; j < 8; ++j)
              sts16(s1 + (r >> 6) * (CHUNK / 2) + (g * 8 + j) * 128 + (((r & 63) * 2) ^ (j << 4)), v[j]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(&side_done[b]);
      }
      e += chunks;
      if (!waited) wait_acc();
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0 && !dead) {  // the accumulator is free
        const unsigned bar = CTAS == 1 ? smem_u32(&acc_empty[c & 1]) : in_block(smem_u32(&acc_empty[c & 1]), 0);
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
      }
    }
  } else if (warp == LOADER) {
    if (lane == 0) {  // what the epilogues need of X or A
      int e = 0;
      bool stop = false;
      for (int t = first; t < items && !stop; t += stride) {
        const Item it = item_of<TILE>(a, t);
        const int chunks = chunks_of<TILE>(a, it);
        if (!count_wait(a.ready + it.mat, needed(a, it, CTAS), gave_up)) {
          *gave_up = 1;
          atomicExch(a.err, 6);
          break;
        }
        asm volatile("fence.proxy.async.global;" ::: "memory");
        const int row = it.row * TILE::M + rank * 128;
        for (int ch = 0; ch < chunks; ++ch, ++e) {
          const int b = e % SIDES;
          if (e >= SIDES && !bar_wait(&side_empty[b], (e / SIDES - 1) & 1, gave_up)) {
            *gave_up = 1;
            atomicExch(a.err, 7);
            stop = true;
            break;
          }
          const unsigned s0 = smem_u32(side) + b * (2 * CHUNK), bar = smem_u32(&side_full[b]);
          const int col = it.col * BN + ch * CHUNK_COLS;
          if (it.phase == GRAM) {
            bar_arrive(&side_full[b]);
          } else if (it.phase == POLY) {
            bar_expect(&side_full[b], CHUNK);
            box_load(&maps.m[CHUNK_A], s0, bar, col, row, it.mat);
          } else {
            bar_expect(&side_full[b], 2 * CHUNK);
            box_load(&maps.m[CHUNK_X + (it.step & 1)], s0, bar, col, row, it.mat);
            box_load(&maps.m[CHUNK_LO], s0 + CHUNK, bar, col, row, it.mat);
          }
        }
      }
    }
  } else {
    if (lane == 0) {  // their results
      int e = 0, under_way = -1;  // chunks used so far; the buffer of a store not yet waited for
      bool stop = false;
      for (int t = first; t < items && !stop; t += stride) {
        const Item it = item_of<TILE>(a, t);
        const int chunks = chunks_of<TILE>(a, it);
        const bool last = it.phase == UPDATE && it.step + 1 == a.steps;
        const bool mirror = it.phase != UPDATE && !on_diagonal<TILE>(it);
        const int row = it.row * TILE::M + rank * 128;
        const CUtensorMap* to =
            &maps.m[it.phase == GRAM ? CHUNK_A : it.phase == POLY ? CHUNK_B : CHUNK_X + ((it.step + 1) & 1)];
        const CUtensorMap* turned = &maps.m[it.phase == GRAM ? TURNED_A : TURNED_B];
        for (int ch = 0; ch < chunks; ++ch, ++e) {
          const int b = e % SIDES;
          if (!bar_wait(&side_done[b], (e / SIDES) & 1, gave_up)) {
            *gave_up = 1;
            atomicExch(a.err, 8);
            stop = true;
            break;
          }
          if (*gave_up) {
            stop = true;
            break;
          }
          if (!last) {
            const unsigned s0 = smem_u32(side) + b * (2 * CHUNK), s1 = s0 + CHUNK;
            const int col = it.col * BN + ch * CHUNK_COLS;
            if (row < a.m) {
              box_store(to, s0, col, row, it.mat);
              if (it.phase == UPDATE) box_store(&maps.m[CHUNK_LO], s1, col, row, it.mat);
            }
            for (int h = 0; h < 2; ++h)
              if (mirror && row + 64 * h < a.m) box_store(turned, s1 + h * (CHUNK / 2), row + 64 * h, col, it.mat);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            if (under_way >= 0) {  // the one before has been read
              asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
              bar_arrive(&side_empty[under_way]);
            }
            under_way = b;
          } else {
            bar_arrive(&side_empty[b]);
          }
        }
        if (!stop && !last) {
          // written, and there for other blocks' copies
          asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
          asm volatile("fence.proxy.async.global;" ::: "memory");
          asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(a.ready + it.mat) : "memory");
          bar_arrive(&side_empty[under_way]);
          under_way = -1;
        }
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
  }
}

struct LoadArgs {
  const void* g;
  long long batch, outer_stride, inner_stride;  // G as `outer` runs of `inner` elements, adjacent ones where there are any
  int outer, inner;
  int turned;  // runs are columns of X, not rows
  int m, n, ldx;
  float eps, scale;
  double* part;
  __half *hi, *lo;
  int* err;
  unsigned* ready;
};

// V adjacent elements of a run.
template <typename T, int V>
__device__ __forceinline__ void load_run(const LoadArgs& a, const T* p, float (&x)[V]) {
  if (V == 1) {
    x[0] = to_float(*p);
  } else {
    const Vec<T, V> w = load_vec<T, V>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = to_float(w.v[j]);
  }
}

// A share of a matrix's sum of squares, in 64 bits: no scale of the update
// overflows.  Clears the counters of the products on the way.
template <typename T, int V>
__global__ void __launch_bounds__(256) ns_norm(const __grid_constant__ LoadArgs a) {
  constexpr int U = 4;  // loads in flight
  __shared__ double buf[8];
  const long long mat = blockIdx.y;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.ready[mat] = 0;
    if (mat == 0) *a.err = 0;
  }
  const T* g = static_cast<const T*>(a.g) + mat * a.batch;
  const unsigned per = a.inner / V;
  const long long total = static_cast<long long>(a.outer) * per, step = static_cast<long long>(gridDim.x) * 256;
  double s = 0.0;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += U * step) {
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long k = i + u * step;
      if (k < total) {
        const long long o = k / per;
        load_run<T, V>(a, g + o * a.outer_stride + (k - o * per) * V * a.inner_stride, x[u]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[u][j] = 0.0f;
      }
    }
    // squares of a few in 32 bits where that can neither overflow nor vanish
    // (conversions to 64 bits would take longer than the loads: 88 us for 200 MB)
    float q = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) q = fmaf(x[u][j], x[u][j], q);
    if (q > 1e-25f && q < 1e37f) {
      s += q;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double y = x[u][j];
          s = fma(y, y, s);
        }
    }
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

// X = G scale / (|G| + eps) as the sum of two f16 numbers, 64 x 64 elements a
// block.  The last matrices first: the norm's pass has left them in L2.
template <typename T, int V>
__global__ void __launch_bounds__(256) ns_load(const __grid_constant__ LoadArgs a) {
  __shared__ float t[64][65];
  __shared__ double factor;
  const long long mat = gridDim.z - 1 - blockIdx.z;
  const T* g = static_cast<const T*>(a.g) + mat * a.batch;
  const int i0 = blockIdx.x * 64, o0 = blockIdx.y * 64;  // along a run, of runs
  constexpr int PER = 64 / V;                            // vectors of a run here
  constexpr int N = 64 * PER / 256;
  float x[N][V];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = k * 256 + threadIdx.x, o = o0 + at / PER, i = i0 + at % PER * V;
    if (o < a.outer && i < a.inner) {
      load_run<T, V>(a, g + o * a.outer_stride + i * a.inner_stride, x[k]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k][j] = 0.0f;
    }
  }
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int k = threadIdx.x; k < NORM_BLOCKS; k += 32) s += a.part[mat * NORM_BLOCKS + k];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) factor = s == 0.0 ? 0.0 : a.scale / (sqrt(s) + a.eps);  // zeros stay zeros, whatever eps is
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = k * 256 + threadIdx.x, o = at / PER, i = at % PER * V;
#pragma unroll
    for (int j = 0; j < V; ++j) t[a.turned ? i + j : o][a.turned ? o : i + j] = x[k][j];
  }
  __syncthreads();
  // Norms under 5e-35 have a factor past the range of 32 bits, though not its
  // products: these are taken in 64 then.
  const float f = static_cast<float>(factor);
  const bool wide = factor > 1e37;
  const int r0 = a.turned ? i0 : o0, c0 = a.turned ? o0 : i0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // 8 adjacent elements of a row of X
    const int at = k * 256 + threadIdx.x, r = at / 8, c = at % 8 * 8;
    if (r0 + r >= a.m || c0 + c >= a.n) continue;
    Vec<__half, 8> h, l;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = wide ? static_cast<float>(t[r][c + j] * factor) : t[r][c + j] * f;
      h.v[j] = __float2half_rn(y);
      l.v[j] = __float2half_rn(y - __half2float(h.v[j]));
    }
    const long long to = (mat * a.m + r0 + r) * a.ldx + c0 + c;  // the row's padding takes zeros
    store_vec<__half, 8>(a.hi + to, h);
    store_vec<__half, 8>(a.lo + to, l);
  }
}

template <typename T, int V>
cudaError_t load(const LoadArgs& a, int count, cudaStream_t st) {
  const cudaError_t e = launch<ns_norm<T, V>>(dim3(NORM_BLOCKS, count), 256, 0, st, a);
  if (e != cudaSuccess) return e;
  return launch<ns_load<T, V>>(dim3((a.inner + 63) / 64, (a.outer + 63) / 64, count), 256, 0, st, a);
}

// No steps: the normalised matrix itself.
__global__ void ns_copy(const __grid_constant__ NsArgs s) {
  const long long mat = blockIdx.y;
  const long long n = static_cast<long long>(s.m) * s.n;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int r = static_cast<int>(i / s.n), c = static_cast<int>(i - static_cast<long long>(r) * s.n);
    const long long at = (mat * s.m + r) * s.ldx + c;
    store_any(s.out, s.out_type, mat * s.out_batch + r * s.out_row + c * s.out_col,
              (__half2float(s.hi[0][at]) + __half2float(s.lo[at])) * s.out_scale);
  }
}

struct Layout {
  long long m, n, ldx, lda;
  size_t head, part, hi[2], lo, a, b, da, db, total;
};
Layout plan(long long count, long long rows, long long cols) {
  Layout l;
  l.m = rows < cols ? rows : cols;
  l.n = rows < cols ? cols : rows;
  // rows start on 128-byte lines, or a box's rows would touch two each
  l.ldx = (l.n + 63) / 64 * 64;
  l.lda = (l.m + 63) / 64 * 64;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.head = take(256 + 4ull * count);  // the error word, then the counters
  l.part = take(sizeof(double) * NORM_BLOCKS * count);
  for (size_t& t : l.hi) t = take(2ull * count * l.m * l.ldx);
  l.lo = take(2ull * count * l.m * l.ldx);
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

// The list's tiles for one tile size, and a step's time in us as estimated from
// measured costs of a tile's 64 elements of K and of a product's start and end
// (4.6 us, and 1.4 for each 64 columns of the last tile's epilogue):
// each product in as many rounds as its tiles make for the blocks.  What a block
// can bring from L2 (70 to 80 GB/s) bounds the first, so that a large tile costs
// hardly more than a small one: small ones are for matrices that leave most
// blocks without a large one.
struct Tiling {
  long long sym, up;
  int row_tiles, sym_cols;
  double us;
};
template <typename TILE>
Tiling tiling(long long count, long long m, long long n, int workers, double per_kblock) {
  Tiling t;
  t.row_tiles = static_cast<int>((m + TILE::M - 1) / TILE::M);
  t.sym_cols = static_cast<int>((m + TILE::N - 1) / TILE::N);
  t.sym = 0;
  for (int i = 0; i < t.row_tiles; ++i) t.sym += std::min(static_cast<long long>(i + 1) * TILE::RATIO, static_cast<long long>(t.sym_cols));
  t.up = t.row_tiles * ((n + TILE::N - 1) / TILE::N);
  const double kn = static_cast<double>((n + BK - 1) / BK), km = static_cast<double>((m + BK - 1) / BK);
  auto rounds = [&](long long tiles) { return static_cast<double>((count * tiles + workers - 1) / workers); };
  t.us = per_kblock * (rounds(t.sym) * (kn + km) + rounds(t.up) * km) + 3 * (4.6 + 1.4 * TILE::N / 64);
  return t;
}

template <int CTAS, int BN>
cudaError_t start(const Maps& maps, NsArgs& a, const Tiling& t, int sms, int device, cudaStream_t st) {
  using TILE = Tile<CTAS, BN>;
  cudaLaunchConfig_t c = {};
  c.blockDim = dim3(THREADS);
  c.dynamicSmemBytes = TILE::SMEM;
  c.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CTAS;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeCooperative;  // blocks wait for one another: all of them have to be resident
  at[1].val.cooperative = 1;
  c.attrs = at;
  static std::atomic<int> resident[64];  // blocks or pairs of them at a time, asked for once
  int most_workers = device < 64 ? resident[device].load() : 0;
  if (!most_workers) {
    cudaError_t e = cudaFuncSetAttribute(ns_kernel<CTAS, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, TILE::SMEM);
    if (e != cudaSuccess) return e;
    c.gridDim = dim3(sms / CTAS * CTAS);
    c.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&most_workers, ns_kernel<CTAS, BN>, &c);
    if (e != cudaSuccess) return e;
    most_workers = std::min(most_workers, sms / CTAS);
    if (most_workers < 1) return cudaErrorCooperativeLaunchTooLarge;
    if (device < 64) resident[device] = most_workers;
  }
  a.sym = static_cast<int>(t.sym), a.up = static_cast<int>(t.up);
  a.row_tiles = t.row_tiles, a.sym_cols = t.sym_cols;
  const long long most = a.count * std::max(t.sym, t.up);  // tiles of one product
  c.gridDim = dim3(static_cast<unsigned>(std::min<long long>(most_workers, most)) * CTAS);
  c.numAttrs = 2;
  return cudaLaunchKernelEx(&c, ns_kernel<CTAS, BN>, maps, a);
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
  if (!aligned(g, elem_size(dtype)) || !aligned(out, elem_size(out_dtype)))
    return fail("ad_orthogonalize: an operand is not aligned to its elements");
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.total)
    return fail("ad_orthogonalize: needs %zu bytes of workspace, 256-byte aligned", l.total);
  for (int i = 0; i < 3 * steps; ++i)
    if (!std::isfinite(coefficients[i])) return fail("ad_orthogonalize: a coefficient is not a number");
  const Scales sc = scales_for(steps, coefficients);
  if (!sc.ok) return fail("ad_orthogonalize: these coefficients let singular values grow past 1024");
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda("ad_orthogonalize", guard.error());
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* w = static_cast<unsigned char*>(workspace);
  const bool tall = rows > cols;
  const int m = static_cast<int>(l.m), n = static_cast<int>(l.n), num = static_cast<int>(count);

  LoadArgs la = {};
  la.g = g, la.batch = batch_stride;
  const bool by_row = col_stride == 1 || row_stride != 1;
  la.outer = static_cast<int>(by_row ? rows : cols), la.inner = static_cast<int>(by_row ? cols : rows);
  la.outer_stride = by_row ? row_stride : col_stride, la.inner_stride = by_row ? col_stride : row_stride;
  la.turned = by_row == tall;
  la.m = m, la.n = n, la.ldx = static_cast<int>(l.ldx);
  la.eps = eps, la.scale = static_cast<float>(sc.x[0]);
  la.part = reinterpret_cast<double*>(w + l.part);
  la.hi = reinterpret_cast<__half*>(w + l.hi[0]);
  la.lo = reinterpret_cast<__half*>(w + l.lo);
  const bool vec = la.inner_stride == 1 && la.inner % 4 == 0 && la.outer_stride % 4 == 0 && batch_stride % 4 == 0 &&
                   aligned(g, 4 * elem_size(dtype));
  la.err = reinterpret_cast<int*>(w);
  la.ready = reinterpret_cast<unsigned*>(w + 256);
  cudaError_t e = dtype == AD_F32    ? (vec ? load<float, 4>(la, num, st) : load<float, 1>(la, num, st))
                  : dtype == AD_BF16 ? (vec ? load<__nv_bfloat16, 4>(la, num, st) : load<__nv_bfloat16, 1>(la, num, st))
                                     : (vec ? load<__half, 4>(la, num, st) : load<__half, 1>(la, num, st));
  if (e != cudaSuccess) return fail_cuda("ad_orthogonalize", e);

  NsArgs s = {};
  s.count = num, s.m = m, s.n = n, s.steps = steps;
  s.ldx = la.ldx;
  for (int k = 0; k < 2; ++k) s.hi[k] = reinterpret_cast<__half*>(w + l.hi[k]);
  s.lo = la.lo;
  s.da = reinterpret_cast<float*>(w + l.da);
  s.db = reinterpret_cast<float*>(w + l.db);
  s.err = la.err, s.ready = la.ready;
  s.out = out, s.out_type = out_dtype;
  s.out_batch = out_batch_stride;
  s.out_row = tall ? out_col_stride : out_row_stride, s.out_col = tall ? out_row_stride : out_col_stride;
  s.out_scale = static_cast<float>(1.0 / sc.x[steps]);
  const int per16 = 16 / elem_size(out_dtype);
  s.out_vec = s.out_col == 1 && s.out_row % per16 == 0 && s.out_batch % per16 == 0 && aligned(out, 16);
  if (steps == 0) {
    e = launch<ns_copy>(dim3(256, num), 256, 0, st, s);
    if (e != cudaSuccess) return fail_cuda("ad_orthogonalize", e);
    return 0;
  }
  for (int k = 0; k < steps; ++k) {
    const double a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
    const double sx = sc.x[k], sa = sc.a[k], sb = sc.b[k], up = sc.x[k + 1] / sx;
    s.step[k] = {static_cast<float>(sa / (sx * sx)), static_cast<float>(b * sb / sa), static_cast<float>(c * sb / (sa * sa)),
                 static_cast<float>(a * up), static_cast<float>(up / sb)};
  }
  Maps maps;
  void* const xh[2] = {w + l.hi[0], w + l.hi[1]};
  void* const ab[2] = {w + l.a, w + l.b};
  int bad = 0;
  auto map = [&](int k, const void* base, bool of_x, int box_rows, int box_cols, int swizzle) {
    bad |= ad_b200_internal::tmap_3d_16(base, count, m, of_x ? n : m, of_x ? l.ldx : l.lda, box_rows, box_cols, swizzle,
                                        &maps.m[k]);
  };
  for (int k = 0; k < 2; ++k) {
    map(WIDE_X + k, xh[k], true, 128, BK, 128);
    map(WIDE_A + k, ab[k], false, 128, BK, 128);
    map(NARROW_X + k, xh[k], true, 64, BK, 128);
    map(CHUNK_X + k, xh[k], true, 128, CHUNK_COLS, 2 * CHUNK_COLS);
    map(CHUNK_A + k, ab[k], false, 128, CHUNK_COLS, 2 * CHUNK_COLS);
    map(TURNED_A + k, ab[k], false, CHUNK_COLS, 64, 128);
  }
  map(NARROW_A, ab[0], false, 64, BK, 128);
  map(CHUNK_LO, s.lo, true, 128, CHUNK_COLS, 2 * CHUNK_COLS);
  if (bad) return 1;

  const int sms = sm_count(guard.device());
  if (!sms) return fail("ad_orthogonalize: no device properties");
  const Tiling big = tiling<Tile<2, 256>>(count, m, n, sms / 2, 0.45);
  const Tiling mid = tiling<Tile<1, 128>>(count, m, n, sms, 0.47);
  const Tiling small = tiling<Tile<1, 64>>(count, m, n, sms, 0.40);
  const Tiling& best = big.us <= mid.us && big.us <= small.us ? big : mid.us <= small.us ? mid : small;
  if (steps * count * (2 * best.sym + best.up) > 0x3fffffffll) return fail("ad_orthogonalize: too many tiles in one call");
  e = &best == &big   ? start<2, 256>(maps, s, best, sms, guard.device(), st)
      : &best == &mid ? start<1, 128>(maps, s, best, sms, guard.device(), st)
                      : start<1, 64>(maps, s, best, sms, guard.device(), st);
  if (e != cudaSuccess) return fail_cuda("ad_orthogonalize", e);
  return 0;
}
