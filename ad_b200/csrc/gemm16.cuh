// Products of 16-bit matrices on tcgen05 with an epilogue of the caller's: the
// core of the feed-forward block and of the log probabilities of a linear layer.
//
//   C[m][n] = sum_k A(m, k) B(n, k)
//
// accumulated in 32 bits in tensor memory.  An operand lies in memory with its
// rows along K (K-major) or across it (A as [K][M], B as [K][N]): no transposed
// copies are made, the matrix instruction takes either.
//
// Bound by the tensor cores, in long runs by the power they may draw.  A pair of
// blocks (cta_group::2) works on a tile of 256 x 256, so that 32 KB a block serve 4.2
// MFLOP: 64 elements of K take the tensor cores 512 clocks, in which a multiprocessor can
// just be sent those 32 KB (64 bytes a clock).  Counted in a copy, they take 590 to 615, both
// threads waiting for loads that are 2 us under way; at the 1.3 to 1.4 GHz that large products
// leave the tensor cores are busy 93 to 96% of the time.  Single blocks on 128 x 128 or
// 128 x 64 are for products with too few large tiles.
// Blocks stay resident and take their share of the tiles; in a block one thread brings
// operands by TMA, one issues the products into one of two accumulators, eight or sixteen
// warps work on the other, so that a tile's epilogue is hidden behind the next tile's
// products.  Tiles are walked in bands of rows, so that the tiles under way at a time
// share operands in L2.  The two issuing threads are the narrowest place: with what they
// do for 64 elements of K computed as it comes (which stage, which operands, descriptors
// of 64 bits) 16384 x 2048 over 8192 took 400 to 430 us, with loops that only count
// 334 (1.65 PFLOP/s; cuBLAS 359), although loads left out altogether had changed little.
// Products to memory (gemm16.cu) are dealt out as whole tiles and, where the last round
// would leave blocks without one, as parts of a tile's K, whose sums are joined in
// order.  Nothing depends on scheduling.
#ifndef AD_B200_GEMM16_CUH
#define AD_B200_GEMM16_CUH

#include <cuda.h>

#include <algorithm>

#include "ops_common.cuh"
#include "schedule.h"

namespace ad_b200_internal {
// runtime.cu: TMA descriptor of a row-major matrix of 16-bit elements, swizzled
// over 128 bytes; what lies outside reads as zero.  0, or 1 with an error set.
int tmap_2d_16(const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, uint32_t box_cols,
               void* out128);
}

namespace adgemm {

using namespace adops;

constexpr int BOX = 64 * BK * 2;  // bytes of a box of 64 x 64
constexpr int CHUNK = 32;         // columns that an epilogue takes at a time
constexpr int MAX_MAPS = 6;

// Tiles: CTAS blocks work on one of 128 CTAS rows and BN columns.  An epilogue has
// WARPS warps, and SIDE bytes of shared memory for each of them.
template <int CTAS_, int BN_, typename EPI>
struct Tile {
  static constexpr int CTAS = CTAS_, BN = BN_, M = 128 * CTAS;
  static constexpr int QN = BN / CTAS;  // columns whose operand a block holds
  static constexpr int P_BYTES = 128 * BK * 2, Q_BYTES = QN * BK * 2, STAGE = P_BYTES + Q_BYTES;
  static constexpr int SIDES = EPI::WARPS * EPI::SIDE, MOST = (225 * 1024 - SIDES) / STAGE;
  static constexpr int STAGES = MOST < 8 ? MOST : 8;
  static constexpr int SMEM = STAGES * STAGE + SIDES + 1024 + 256;
  static constexpr int THREADS = 32 * (2 + EPI::WARPS);
  static constexpr int TMEM = 2 * BN;
};

// One of the products of a launch.
struct Group {
  int m, n;
  int kblocks0;            // of the first operands (the second ones' follow)
  int a_turned, b_turned;  // operands lie across K
  int map;                 // its first operands' maps
};
struct Shape {
  Group group[MAX_GROUPS];
  int half;  // f16, else bf16
  // the only group's, where units go by number
  int kblocks, row_tiles, col_tiles, units;
  int band;  // row tiles that share a walk over the columns
};
struct Maps {
  CUtensorMap a[MAX_MAPS], b[MAX_MAPS];
};

// A tile, or a part of its K.
struct Unit {
  int group, row, col, kb0, kb1;
  int slot;  // where partial sums go, or -1
};
// Whole tiles by number: for epilogues that need whole sums.
struct ByNumber {
  template <typename P>
  __device__ static void range(const P&, const Shape& s, int worker, int workers, int& first, int& end, int& step) {
    first = worker, end = s.units, step = workers;
  }
  template <typename P>
  __device__ static Unit unit(const P&, const Shape& s, int u) {
    const int per = s.band * s.col_tiles, band = u / per;
    u -= band * per;
    const int rows = min(s.band, s.row_tiles - band * s.band);
    Unit t;
    t.group = 0, t.slot = -1;
    t.col = u / rows;
    t.row = band * s.band + u - t.col * rows;
    t.kb0 = 0, t.kb1 = s.kblocks;
    return t;
  }
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
// the next 64 columns lie a box further.  The upper word is the same for both; the lower
// one has the address, and how far 16 elements of K are.
constexpr unsigned DESC_UPPER = (1024u >> 4) | (1u << 14) | (2u << 29);
template <bool TURNED>
__device__ __forceinline__ unsigned desc_lower(unsigned at) {
  return (at >> 4) | (TURNED ? static_cast<unsigned>(BOX >> 4) << 16 : 1u << 16);
}
template <bool TURNED>
constexpr unsigned DESC_STEP = TURNED ? (16 * 128) >> 4 : 32 >> 4;

template <int CTAS>
__device__ __forceinline__ void mma(unsigned acc, unsigned p, unsigned q, unsigned idesc, unsigned more) {
  if (CTAS == 1)
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.u32 p, %5, 0;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}" ::"r"(acc),
        "r"(p), "r"(q), "n"(DESC_UPPER), "r"(idesc), "r"(more)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.u32 p, %5, 0;\n mov.b64 a, {%1, %3};\n mov.b64 b, {%2, %3};\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n}" ::"r"(acc),
        "r"(p), "r"(q), "n"(DESC_UPPER), "r"(idesc), "r"(more)
        : "memory");
}
template <int CTAS>
__device__ __forceinline__ void commit(unsigned bar) {
  if (CTAS == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(static_cast<unsigned short>(3))
        : "memory");
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

// 16 columns, added to sums that are there.
__device__ __forceinline__ void tmem_add16(unsigned taddr, float* v) {
  unsigned q[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]), "=r"(q[8]),
        "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]), "=r"(q[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(q[0]), "+r"(q[1]), "+r"(q[2]), "+r"(q[3]), "+r"(q[4]), "+r"(q[5]), "+r"(q[6]), "+r"(q[7]),
                 "+r"(q[8]), "+r"(q[9]), "+r"(q[10]), "+r"(q[11]), "+r"(q[12]), "+r"(q[13]), "+r"(q[14]), "+r"(q[15])
               :
               : "memory");
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] += __uint_as_float(q[j]);
}

__device__ __forceinline__ unsigned lds32(unsigned addr) {
  unsigned v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
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
  int lane, quad, part, row0;
  Unit unit;
  int m, n;       // of the result
  int width, stride;  // of a tile; columns from a chunk of the warp's to its next
  int odd;        // every other tile of the block
  unsigned side;
  unsigned free_bar;  // to arrive at once the accumulator has been read
  bool last;          // the warp's last chunk of the tile
  bool dead;          // a wait ran out: results are NaNs
};

// The warp has read its part of the accumulator.  Relaxed: what is ordered is the
// reads of tensor memory, by the fence; a release would wait for the warp's stores too.
__device__ __forceinline__ void accumulator_read(const Spot& s) {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  if (s.lane == 0 && !s.dead)
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(s.free_bar) : "memory");
}
// 32 columns of the warp's rows; the accumulator is given back with the last ones.
__device__ __forceinline__ void take32(const Spot& s, unsigned acc, float (&v)[32]) {
  tmem_ld32(acc, v);
  if (s.last) accumulator_read(s);
  if (s.dead) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __int_as_float(0x7fffffff);
  }
}

// The same, added to v.
__device__ __forceinline__ void add32(const Spot& s, unsigned acc, float (&v)[32]) {
  tmem_add16(acc, v);
  tmem_add16(acc + 16, v + 16);
  if (s.last) accumulator_read(s);
  if (s.dead) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __int_as_float(0x7fffffff);
  }
}

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
    unsigned short* to = out + (s.row0 + (s.lane >> 2)) * ld + col0 + p * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (s.lane >> 2);
      const uint4 x = lds128(s.side + r * 64 + ((p ^ ((r >> 1) & 3)) << 4));
      if (s.row0 + r < m) *reinterpret_cast<uint4*>(to) = x;
      to += 8 * ld;
    }
  } else {
    // two rows at a time, half a warp each, a word a lane; where the row starts in the
    // upper half of one, words from the second column on, and the first and last one
    // apart by the last lane.  Read ahead of the stores, eight at a time (dW of 62044 x
    // 3802 over 4: 296 us, 491 one at a time; 142 where rows are aligned).
    const int h = s.lane >> 4, l = s.lane & 15, left = n - col0;
    unsigned short* row = out + (s.row0 + h) * ld + col0;
    const int shift = (reinterpret_cast<uintptr_t>(row) >> 1) & 1;  // of every second row too
    const int c0 = 2 * l + shift, c1 = (c0 + 1) & 31;
#pragma unroll 1
    for (int r0 = h; r0 < 32; r0 += 16) {
      unsigned x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r0 + 2 * i;
        x[i] = lds32(s.side + r * 64 + (((l >> 2) ^ ((r >> 1) & 3)) << 4) + (l & 3) * 4);
        const unsigned next = __shfl_sync(0xffffffffu, x[i], (l + 1) & 15, 16);
        if (shift) x[i] = x[i] >> 16 | next << 16;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (s.row0 + r0 + 2 * i < m) {
          if (c1 && c1 < left) {
            *reinterpret_cast<unsigned*>(row + c0) = x[i];
          } else {
            if (c0 < left) row[c0] = static_cast<unsigned short>(x[i]);
            if (!c1) row[0] = static_cast<unsigned short>(x[i] >> 16);
          }
        }
        row += 2 * ld;
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
    float* to = out + (s.row0 + (s.lane >> 3)) * ld + col0 + q * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + (s.lane >> 3);
      const float4 x = staged(s, r, q);
      if (s.row0 + r < m) *reinterpret_cast<float4*>(to) = x;
      to += 4 * ld;
    }
  } else {  // a column a lane
    const int col = col0 + s.lane;
    if (col < n)
      for (int r = 0; r < 32 && s.row0 + r < m; ++r) out[(s.row0 + r) * ld + col] = staged1(s, r);
  }
}

// Rows of A that a copy brings, where there are m: rows outside of the operand cost time,
// although they are not read (the loss of 4 rows over 130000 tokens of width 2048: 147 us with
// copies of 128 rows, 94 of 4; from 32 rows on 96). What then is left in their place
// in shared memory only goes to rows of the product that there are none of.
template <int CTAS>
__host__ __device__ __forceinline__ int rows_of_box(int m) {
  return CTAS == 1 && m < 128 ? m : 128;
}

// ------------------------------------------------------------------ the kernel

// Parts of a unit's K, and where one of them begins.
template <typename EPI>
__device__ __forceinline__ int parts_of_k(const Unit& t) {
  return EPI::PART ? max(1, (t.kb1 - t.kb0 + EPI::PART / 2) / EPI::PART) : 1;
}
__device__ __forceinline__ int part_begin(const Unit& t, int part, int parts) { return (t.kb1 - t.kb0) * part / parts; }

// A place among the stages, the phase of its barriers, and whether it has been used before.
template <int STAGES>
struct Ring {
  int i = 0;
  unsigned phase = 0, again = 0;
  __device__ __forceinline__ void next() {
    if (++i == STAGES) i = 0, phase ^= 1, again = 1;
  }
};

// EPI: DUAL (B's tiles hold half their columns of each of two operands), WARPS,
// SIDE; US (tiling_for); Params; Units; a State that is constructed for a tile (loads that need no
// accumulator), whose chunk() takes 32 columns, and whose end() all warps call.  PART: 0, or about
// how many stages of K one accumulator sums; a tile's K is then taken in parts of the same length,
// by turns in both accumulators, and the State's hold() keeps the sums of all but the last, 32 columns for
// each of the warp's chunks.
template <typename TILE, typename EPI>
__global__ void __launch_bounds__(TILE::THREADS, 1)
    gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Shape a,
                const __grid_constant__ typename EPI::Params params) {
  constexpr int CTAS = TILE::CTAS, BN = TILE::BN, STAGES = TILE::STAGES;
  constexpr int COLS = EPI::DUAL ? BN / 2 : BN;  // columns of the result
  constexpr int PARTS = EPI::WARPS / 4;          // warps that share 32 rows, each with its share of the chunks
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char* side = smem + STAGES * TILE::STAGE;
  unsigned long long* full = reinterpret_cast<unsigned long long*>(side + TILE::SIDES);
  unsigned long long* empty = full + STAGES;
  unsigned long long* acc_full = empty + STAGES;
  unsigned long long* acc_empty = acc_full + 2;
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(acc_empty + 2);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CTAS == 1 ? 0 : blockIdx.x & 1;
  int first, end, step;
  EPI::Units::range(params, a, blockIdx.x / CTAS, gridDim.x / CTAS, first, end, step);

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&empty[i])));
    }
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&acc_full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&acc_empty[i])), "r"(CTAS * EPI::WARPS));
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
  after_previous();

  if (warp == 0) {
    if (lane == 0) {  // operands
      // what earlier kernels wrote is read through the async proxy
      asm volatile("fence.proxy.async.global;" ::: "memory");
      Ring<TILE::STAGES> ring;
      const unsigned leader = CTAS == 2 ? in_block(smem_u32(full), 0) : smem_u32(full);
      auto load = [&](const CUtensorMap* map, unsigned to, unsigned bar, int x0, int y0) {
        if (CTAS == 1)
          asm volatile(
              "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
                  to),
              "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(x0), "r"(y0)
              : "memory");
        else
          asm volatile(
              "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
              "[%1, {%3, %4}], [%2];" ::"r"(to),
              "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(x0), "r"(y0)
              : "memory");
      };
      for (int u = first; u < end; u += step) {
        const Unit t = EPI::Units::unit(params, a, u);
        const Group g = a.group[t.group];
        const int p0 = t.row * TILE::M + rank * 128;
        const int q0 = EPI::DUAL ? t.col * COLS : t.col * BN + rank * TILE::QN;
        // a run of stages with the same operands
        auto run = [&](auto a_turned, auto b_turned, const CUtensorMap* pa, const CUtensorMap* pb, int kb0, int kb1) {
          constexpr bool AT = decltype(a_turned)::value, BT = decltype(b_turned)::value;
          int k0 = kb0 * BK;
          for (int left = kb1 - kb0; left > 0; --left, ring.next(), k0 += BK) {
            if (ring.again && !bar_wait(&empty[ring.i], ring.phase ^ 1, gave_up)) return false;
            const unsigned st = smem_u32(smem) + ring.i * TILE::STAGE, sq = st + TILE::P_BYTES, bar = leader + ring.i * 8;
            if (rank == 0)
              asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&full[ring.i])),
                           "r"(AT ? CTAS * TILE::STAGE : CTAS * TILE::STAGE - (128 - rows_of_box<CTAS>(g.m)) * 128)
                           : "memory");
            if (AT) {
#pragma unroll
              for (int h = 0; h < 2; ++h) load(pa, st + h * BOX, bar, p0 + h * 64, k0);
            } else {
              load(pa, st, bar, k0, p0);
            }
            if (EPI::DUAL) {
              if (CTAS == 2) {
                load(pb + rank, sq, bar, k0, q0);
              } else {
                load(pb, sq, bar, k0, q0);
                load(pb + 1, sq + TILE::Q_BYTES / 2, bar, k0, q0);
              }
            } else if (BT) {
#pragma unroll
              for (int h = 0; h < TILE::QN / 64; ++h) load(pb, sq + h * BOX, bar, q0 + h * 64, k0);
            } else {
              load(pb, sq, bar, k0, q0);
            }
          }
          return true;
        };
        auto both = [&](const CUtensorMap* pa, const CUtensorMap* pb, int kb0, int kb1) {
          const std::true_type yes;
          const std::false_type no;
          return g.a_turned ? (g.b_turned ? run(yes, yes, pa, pb, kb0, kb1) : run(yes, no, pa, pb, kb0, kb1))
                            : (g.b_turned ? run(no, yes, pa, pb, kb0, kb1) : run(no, no, pa, pb, kb0, kb1));
        };
        const int turn = g.kblocks0;
        if (!both(&maps.a[g.map], &maps.b[g.map], t.kb0, min(t.kb1, turn)) ||
            (t.kb1 > turn && !both(&maps.a[g.map + 1], &maps.b[g.map + 1], max(t.kb0 - turn, 0), t.kb1 - turn))) {
          *gave_up = 1;
          break;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {  // products
      Ring<TILE::STAGES> ring;
      int c = 0;  // accumulators used so far
      for (int u = first; u < end; u += step) {
        const Unit t = EPI::Units::unit(params, a, u);
        const Group& g = a.group[t.group];
        const int parts = parts_of_k<EPI>(t);
        int part = 0;
        auto tile = [&](auto a_turned, auto b_turned) {
          constexpr bool AT = decltype(a_turned)::value, BT = decltype(b_turned)::value;
          // D in 32 bits; operand types (bf16: 1) in bits 7 and 10; across K: bits 15 and 16
          const unsigned idesc = (1u << 4) | (a.half ? 0u : (1u << 7) | (1u << 10)) | (AT ? 1u << 15 : 0u) |
                                 (BT ? 1u << 16 : 0u) | (static_cast<unsigned>(BN >> 3) << 17) |
                                 (static_cast<unsigned>(TILE::M >> 4) << 24);
          if (c >= 2 && !bar_wait(&acc_empty[c & 1], (c / 2 - 1) & 1, gave_up)) return false;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const unsigned acc = tmem + (c & 1) * BN;
          unsigned more = 0;
          const int stages = EPI::PART ? part_begin(t, part + 1, parts) - part_begin(t, part, parts) : t.kb1 - t.kb0;
          for (int left = stages; left > 0; --left, ring.next()) {
            if (!bar_wait(&full[ring.i], ring.phase, gave_up)) return false;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned st = smem_u32(smem) + ring.i * TILE::STAGE;
            const unsigned p = desc_lower<AT>(st), q = desc_lower<BT>(st + TILE::P_BYTES);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              mma<CTAS>(acc, p + k * DESC_STEP<AT>, q + k * DESC_STEP<BT>, idesc, more);
              more = 1;
            }
            commit<CTAS>(smem_u32(&empty[ring.i]));
          }
          commit<CTAS>(smem_u32(&acc_full[c & 1]));
          return true;
        };
        const std::true_type yes;
        const std::false_type no;
        bool fine = true;
        for (; part < parts && fine; ++part, ++c)
          fine = g.a_turned ? (g.b_turned ? tile(yes, yes) : tile(yes, no)) : g.b_turned ? tile(no, yes) : tile(no, no);
        if (!fine) {
          *gave_up = 1;
          break;
        }
      }
    }
  } else {  // epilogues
    const int quad = warp & 3, part = (warp - 2) >> 2;  // 32 rows; which of their chunks
    Spot s;
    s.lane = lane, s.quad = quad, s.part = part;
    s.side = smem_u32(side) + (warp - 2) * EPI::SIDE;
    s.width = COLS, s.stride = PARTS * CHUNK;
    s.dead = false, s.odd = 1;
    int c = 0;
    for (int u = first; u < end; u += step, ++c) {
      const Unit t = EPI::Units::unit(params, a, u);
      s.row0 = t.row * TILE::M + rank * 128 + quad * 32;
      s.unit = t, s.m = a.group[t.group].m, s.n = a.group[t.group].n;
      const int chunks = (min(COLS, s.n - t.col * COLS) + CHUNK - 1) / CHUNK;
      typename EPI::State e(params, a, s);
      // a warp without a row of the result, or a chunk of it, still has to say that it is done
      const bool some = s.row0 < s.m && part < chunks;
      unsigned acc;
      auto filled = [&] {  // the accumulator that comes next
        if (!s.dead && !bar_wait(&acc_full[c & 1], (c / 2) & 1, gave_up)) {
          s.dead = true;
          *gave_up = 1;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        acc = tmem + (static_cast<unsigned>(quad * 32) << 16) + (c & 1) * BN;
        s.free_bar = CTAS == 1 ? smem_u32(&acc_empty[c & 1]) : in_block(smem_u32(&acc_empty[c & 1]), 0);
        if (!some) accumulator_read(s);
      };
      if constexpr (EPI::PART != 0) {
        constexpr int MINE = (COLS / CHUNK + PARTS - 1) / PARTS;  // chunks of a warp, at most: sums that are held stay in registers
        for (int left = parts_of_k<EPI>(t); left > 0; --left, ++c) {
          filled();
#pragma unroll
          for (int i = 0; i < MINE; ++i) {
            const int ch = part + i * PARTS;
            if (!some || ch >= chunks) continue;
            s.last = ch + PARTS >= chunks;
            if (left > 1)
              e.hold(s, acc + ch * CHUNK, i);
            else
              e.chunk(params, a, s, t.col * COLS + ch * CHUNK, acc + ch * CHUNK, i);
          }
        }
        --c;
      } else {
        filled();
        if (some)
          for (int ch = part; ch < chunks; ch += PARTS) {
            s.last = ch + PARTS >= chunks;
            e.chunk(params, a, s, t.col * COLS + ch * CHUNK, acc + ch * CHUNK, COLS);
          }
      }
      s.odd ^= 1;
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

// A product C = A B^T of 16-bit operands: m x n over k.
struct Problem {
  long long m, n, k, k0;  // k0: K of the first operands when there are two in a row (else k)
  bool a_turned, b_turned;
  Mat a[2], b[2];
};
struct Device {
  int device, sms;
};

// The tiling for whole tiles: the one whose rounds take least, a round being a
// tile's products or its epilogue (EPI::US, measured for each tiling), whichever is
// longer.  A large tile's epilogue bounds short K's: dh of 600 x 2048 over 512 took 19 us on
// large tiles, 13 on middle ones and 15 on small ones; of 4095 x 2048 35, 35 and 40.
template <typename EPI, bool DUAL = false>
int tiling_for(long long m, long long n, long long kblocks, int sms) {
  int best = 0;
  double least = 1e30;
  for (int i = 0; i < 3; ++i) {
    const Tiling& t = TILINGS[i];
    const int cols = DUAL ? t.n / 2 : t.n, workers = sms / t.ctas;
    const long long count = ((m + t.m - 1) / t.m) * ((n + cols - 1) / cols);
    const double products = kblocks * t.us, epilogue = EPI::US[i];
    const double us = static_cast<double>((count + workers - 1) / workers) * std::max(products, epilogue) +
                      std::min(products, epilogue) + 4.0;
    if (us < least * 0.97) best = i, least = us;
  }
  return best;
}

// Maps of a group's operands, at `map` of them.  1 with an error set.
template <typename TILE, bool DUAL>
int make_maps(const Problem& p, Maps& maps, int map) {
  const int operands = DUAL || p.k0 < p.k ? 2 : 1;
  for (int i = 0; i < operands; ++i) {
    const long long k = DUAL || p.k0 == p.k ? p.k : i ? p.k - p.k0 : p.k0;
    if (!DUAL || i == 0) {
      if (p.a_turned ? ad_b200_internal::tmap_2d_16(p.a[i].p, k, p.m, p.a[i].ld, 64, 64, &maps.a[map + i])
                     : ad_b200_internal::tmap_2d_16(p.a[i].p, p.m, k, p.a[i].ld,
                                                     rows_of_box<TILE::CTAS>(static_cast<int>(std::min(p.m, 128ll))), 64,
                                                     &maps.a[map + i]))
        return 1;
    }
    const int rows = DUAL && TILE::CTAS == 1 ? TILE::QN / 2 : TILE::QN;
    if (p.b_turned ? ad_b200_internal::tmap_2d_16(p.b[i].p, k, p.n, p.b[i].ld, 64, 64, &maps.b[map + i])
                   : ad_b200_internal::tmap_2d_16(p.b[i].p, p.n, k, p.b[i].ld, rows, 64, &maps.b[map + i]))
      return 1;
  }
  return 0;
}
inline Group group_of(const Problem& p, int map) {
  return {static_cast<int>(p.m), static_cast<int>(p.n), static_cast<int>((p.k0 + BK - 1) / BK), p.a_turned, p.b_turned, map};
}

// Blocks or pairs of them at a time: more would start when others have ended, with
// a whole share of the units each.
template <typename TILE, typename EPI>
cudaError_t workers_of(const Device& d, int* workers) {
  static std::atomic<int> known[64];
  if (d.device < 64 && (*workers = known[d.device])) return cudaSuccess;
  int room = 0;
  cudaError_t e = shared_room<gemm_kernel<TILE, EPI>>(&room);
  if (e != cudaSuccess) return e;
  if (room < TILE::SMEM) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t c = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = TILE::CTAS;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.gridDim = dim3(d.sms / TILE::CTAS * TILE::CTAS);
  c.blockDim = dim3(TILE::THREADS);
  c.dynamicSmemBytes = TILE::SMEM;
  c.attrs = at, c.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(workers, gemm_kernel<TILE, EPI>, &c);
  if (e != cudaSuccess) return e;
  *workers = std::max(1, std::min(*workers, d.sms / TILE::CTAS));
  if (d.device < 64) known[d.device] = *workers;
  return cudaSuccess;
}

template <typename TILE, typename EPI>
cudaError_t launch_gemm(const Maps& maps, const Shape& s, const typename EPI::Params& params, int workers, cudaStream_t st) {
  cudaLaunchConfig_t c = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = TILE::CTAS;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  c.gridDim = dim3(workers * TILE::CTAS);
  c.blockDim = dim3(TILE::THREADS);
  c.dynamicSmemBytes = TILE::SMEM;
  c.stream = st;
  c.attrs = at, c.numAttrs = 2;
  return cudaLaunchKernelEx(&c, gemm_kernel<TILE, EPI>, maps, s, params);
}

template <typename TILE, typename EPI>
int start_tile(const char* who, const Device& d, const Problem& p, int half, const typename EPI::Params& params, cudaStream_t st) {
  Maps maps = {};
  Shape s = {};
  const int cols = EPI::DUAL ? TILE::BN / 2 : TILE::BN;
  s.group[0] = group_of(p, 0);
  s.half = half;
  s.kblocks = kblocks_of(p);
  s.row_tiles = static_cast<int>((p.m + TILE::M - 1) / TILE::M);
  s.col_tiles = static_cast<int>((p.n + cols - 1) / cols);
  // about as many rows as columns under way at a time
  s.band = TILE::M == 256 ? 8 : 16;
  const long long units = static_cast<long long>(s.row_tiles) * s.col_tiles;
  if (units > 0x3fffffffll) return fail("%s: too many tiles in one product", who);
  s.units = static_cast<int>(units);
  if (make_maps<TILE, EPI::DUAL>(p, maps, 0)) return 1;
  int workers = 0;
  cudaError_t e = workers_of<TILE, EPI>(d, &workers);
  if (e == cudaSuccess) e = launch_gemm<TILE, EPI>(maps, s, params, std::min(workers, s.units), st);
  return e == cudaSuccess ? 0 : fail_cuda(who, e);
}

// Launches a product with an epilogue.  0, or 1 with an error set.
template <typename EPI>
int start(const char* who, const Device& d, const Problem& p, int half, int tiling, const typename EPI::Params& params,
          cudaStream_t st) {
  return tiling == 0   ? start_tile<Tile<2, 256, EPI>, EPI>(who, d, p, half, params, st)
         : tiling == 1 ? start_tile<Tile<1, 128, EPI>, EPI>(who, d, p, half, params, st)
                       : start_tile<Tile<1, 64, EPI>, EPI>(who, d, p, half, params, st);
}

// ------------------------------------------------------------------ products to memory (gemm16.cu)

// result = alpha (product + addend) + (accumulate ? result : 0)
struct Result {
  void* p;
  long long ld;
  int type;  // AD_F32 or the operands'
  bool accumulate;
  const float* addend;  // of the result's shape, in 32 bits; NULL: none.  May be the result itself
  long long ld_addend;
  const float* alpha;  // device memory; NULL: 1
};
// Up to MAX_GROUPS products in one go, independent of one another.  `partial`:
// partial_bytes() of memory, 16-byte aligned.
size_t partial_bytes(const Device& d);
int store_products(const char* who, const Device& d, int half, const Problem* p, const Result* r, int count, float* partial,
                   cudaStream_t st);
// Copies of 16-bit matrices whose rows TMA can read (16-byte aligned, of a multiple
// of 8 elements), up to MAX_PACKS of them in one go.
constexpr int MAX_PACKS = 5;
struct Pack {
  const void* from;
  void* to;
  long long rows, cols, ld, ld_to;
};
int pack_rows(const char* who, const Device& d, const Pack* packs, int count, cudaStream_t st);

}  // namespace adgemm

#endif
