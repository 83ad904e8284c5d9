// Products of 16-bit matrices to memory (gemm16.cuh): results in 16 or 32 bits,
// added to others, several products in one launch, and copies of operands whose
// rows are not aligned to the 16 bytes that TMA asks for.
//
// Tiles are dealt out from a list of up to 2048 units that the host makes (schedule.h; with room
// for three parts a block, 1826 tiles of pairs, 1604 of single ones; more go by number): whole tiles, the
// longest first, each to the blocks that are done first, and those that would stick
// out above the others cut along K so that all end together (where that saves more than the partial
// sums' way through memory costs).  The list goes with the kernel's parameters.  What
// it gains: dx, dWg, dWu and dWd of a feed-forward block of 4095 x 512 x 2048 took 88 us
// as three launches with equal splits and their joins, 56 in one (42 since operands are
// issued as gemm16.cuh says).
#include <memory>
#include <new>

#include "gemm16.cuh"

namespace adgemm {

namespace {

template <int N>
struct List {
  Listed unit[N];
  short slot[N];
  short first[MAX_WORKERS + 1];  // of each worker's units
};
template <>
struct List<0> {};

template <int N>
struct ByList {
  template <typename P>
  __device__ static void range(const P& p, const Shape&, int worker, int, int& first, int& end, int& step) {
    first = p.list.first[worker], end = p.list.first[worker + 1], step = 1;
  }
  template <typename P>
  __device__ static Unit unit(const P& p, const Shape&, int u) {
    const Listed l = p.list.unit[u];
    return {static_cast<int>(l.where >> 30), static_cast<int>(l.where >> 15 & 0x7fff), static_cast<int>(l.where & 0x7fff),
            l.kb0, l.kb1, p.list.slot[u]};
  }
};

struct Target {
  void* out;
  const float* addend;
  const float* alpha;
  long long ld, ld_addend;
  int type, accumulate;
  int vec;  // four elements at a time are aligned, and eight of 16 bits
};
struct Targets {
  Target t[MAX_GROUPS];
  float* partial;
};

// Four adjacent elements.
__device__ __forceinline__ void load4(const void* p, int type, long long at, float (&x)[4]) {
  if (type == AD_F32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + at);
    const float2 a = unpack2(v.x, type == AD_F16), b = unpack2(v.y, type == AD_F16);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  }
}
__device__ __forceinline__ void store4(void* p, int type, long long at, const float (&x)[4]) {
  if (type == AD_F32)
    *reinterpret_cast<float4*>(static_cast<float*>(p) + at) = make_float4(x[0], x[1], x[2], x[3]);
  else
    *reinterpret_cast<uint2*>(static_cast<unsigned short*>(p) + at) =
        make_uint2(pack2(x[0], x[1], type == AD_F16), pack2(x[2], x[3], type == AD_F16));
}
// alpha (x + addend) + what is there, to the result.
__device__ __forceinline__ void finish4(const Target& t, float alpha, long long row, int col, float4 v) {
  float x[4] = {v.x, v.y, v.z, v.w}, y[4];
  if (t.addend) {
    load4(t.addend, AD_F32, row * t.ld_addend + col, y);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += y[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] *= alpha;
  if (t.accumulate) {
    load4(t.out, t.type, row * t.ld + col, y);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += y[j];
  }
  store4(t.out, t.type, row * t.ld + col, x);
}
__device__ __forceinline__ void finish1(const Target& t, float alpha, long long row, int col, float x) {
  if (t.addend) x += t.addend[row * t.ld_addend + col];
  x *= alpha;
  if (t.accumulate) x += load_any(t.out, t.type, row * t.ld + col);
  store_any(t.out, t.type, row * t.ld + col, x);
}

// N: the list's room, 0 for units by number.
template <int N>
struct Store {
  static constexpr bool DUAL = false;
  static constexpr int WARPS = 8, SIDE = 4096, PART = 0;
  using Units = std::conditional_t<N == 0, ByNumber, ByList<N>>;
  struct Params {
    Targets to;
    int tile_m, tile_n;
    List<N> list;
  };
  struct State {
    float alpha;
    __device__ State(const Params& p, const Shape&, const Spot& s) {
      const float* a = p.to.t[s.unit.group].alpha;
      alpha = a ? *a : 1.0f;
    }
    __device__ void end(const Params&, const Shape&, const Spot&) {}
    __device__ void chunk(const Params& p, const Shape& a, const Spot& s, int col0, unsigned acc, int) {
      float v[32];
      take32(s, acc, v);
      if (s.unit.slot >= 0) {  // partial sums: tiles of their own
        float* base = p.to.partial + static_cast<long long>(s.unit.slot) * p.tile_m * p.tile_n -
                      static_cast<long long>(s.unit.row) * p.tile_m * p.tile_n - s.unit.col * p.tile_n;
        put32(s, v, base, p.tile_n, s.m, 0x7fffffff, col0, 1);
        return;
      }
      const Target& t = p.to.t[s.unit.group];
      if (t.type != AD_F32 && !t.accumulate && !t.addend) {
        unsigned w[16];
        if (a.half) {
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j] * alpha, v[2 * j + 1] * alpha, 1);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j] * alpha, v[2 * j + 1] * alpha, 0);
        }
        put16(s, w, static_cast<unsigned short*>(t.out), t.ld, s.m, s.n, col0, t.vec);
        return;
      }
      stage32(s, v);
      if (t.vec && col0 + CHUNK <= s.n) {
        const int q = s.lane & 7;
#pragma unroll 4
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (s.lane >> 3);
          const float4 x = staged(s, r, q);
          if (s.row0 + r < s.m) finish4(t, alpha, s.row0 + r, col0 + q * 4, x);
        }
      } else {  // a column a lane, eight rows read ahead of their stores
        const int col = col0 + s.lane;
        const long long at = s.row0 * t.ld + col, from = s.row0 * t.ld_addend + col;
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += 8) {
          float x[8], y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool there = col < s.n && s.row0 + r0 + i < s.m;
            x[i] = staged1(s, r0 + i);
            if (t.addend && there) x[i] += t.addend[from + (r0 + i) * t.ld_addend];
            y[i] = t.accumulate && there ? load_any(t.out, t.type, at + (r0 + i) * t.ld) : 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (col < s.n && s.row0 + r0 + i < s.m)
              store_any(t.out, t.type, at + (r0 + i) * t.ld, t.accumulate ? x[i] * alpha + y[i] : x[i] * alpha);
        }
      }
    }
  };
};

// Tiles that were cut: the sums of their parts, in order, to the result.
struct JoinArgs {
  Targets to;
  Group group[MAX_GROUPS];
  int tile_m, tile_n;
  Cut cut[MAX_WORKERS];
};
constexpr int JOIN_ROWS = 4;   // of a tile a block

__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ JoinArgs a) {
  after_previous();
  const Cut c = a.cut[blockIdx.y];
  const int g = c.where >> 30, row0 = (c.where >> 15 & 0x7fff) * a.tile_m + blockIdx.x * JOIN_ROWS,
            col0 = (c.where & 0x7fff) * a.tile_n;
  const int m = a.group[g].m, n = a.group[g].n;
  const Target& t = a.to.t[g];
  const float alpha = t.alpha ? *t.alpha : 1.0f;
  const long long size = static_cast<long long>(a.tile_m) * a.tile_n;
  const float* part = a.to.partial + c.slot * size + static_cast<long long>(blockIdx.x) * JOIN_ROWS * a.tile_n;
  const int per = a.tile_n / 4;
  for (int i = threadIdx.x; i < JOIN_ROWS * per; i += 256) {
    const int r = i / per, q = (i - r * per) * 4;
    if (row0 + r >= m || col0 + q >= n) continue;
    const float* p = part + r * a.tile_n + q;
    float4 x = *reinterpret_cast<const float4*>(p);
#pragma unroll 4
    for (int k = 1; k < c.parts; ++k) {
      const float4 y = *reinterpret_cast<const float4*>(p + k * size);
      x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    if (t.vec && col0 + q + 4 <= n) {
      finish4(t, alpha, row0 + r, col0 + q, x);
    } else {
      const float v[4] = {x.x, x.y, x.z, x.w};
      for (int j = 0; j < 4 && col0 + q + j < n; ++j) finish1(t, alpha, row0 + r, col0 + q + j, v[j]);
    }
  }
}

struct PackArgs {
  Pack pack[MAX_PACKS];
};
// Eight elements a thread.  Rows start at any element: where that is the upper half
// of a word, five words are read and shifted (four operands of a block of 3001 x 1001
// x 2731, 22 MB: 10.6 us in one launch; element by element 38 in four).
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackArgs a) {
  after_previous();
  const Pack& p = a.pack[blockIdx.y];
  const int per = static_cast<int>((p.cols + 7) / 8);
  const long long total = p.rows * per;
  const unsigned short* from = static_cast<const unsigned short*>(p.from);
  unsigned short* to = static_cast<unsigned short*>(p.to);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = i / per;
    const int c = static_cast<int>(i - r * per) * 8;
    const unsigned short* src = from + r * p.ld + c;
    unsigned w[4];
    if (c + 8 <= p.cols) {
      const bool upper = reinterpret_cast<uintptr_t>(src) & 2;
      const unsigned* words = reinterpret_cast<const unsigned*>(src - upper);
      unsigned x[5];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = words[j];
      x[4] = upper ? words[4] : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = upper ? __funnelshift_r(x[j], x[j + 1], 16) : x[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = c + 2 * j < p.cols ? src[2 * j] : 0u;
        if (c + 2 * j + 1 < p.cols) w[j] |= static_cast<unsigned>(src[2 * j + 1]) << 16;
      }
    }
    *reinterpret_cast<uint4*>(to + r * p.ld_to + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ------------------------------------------------------------------ the list

// The best schedule for products of these sizes, or NULL when there are too many
// tiles for a list.  A program makes the same calls again: a thread keeps the last ones (a
// schedule takes 2 to 50 us to make).
struct Sizes {
  long long m[MAX_GROUPS], n[MAX_GROUPS], k[MAX_GROUPS], k0[MAX_GROUPS];
  int count, workers[3];
};
struct Kept {
  static constexpr int N = 24;
  Sizes sizes[N];
  Schedule schedule[N];
  bool listed[N];
  int used = 0, next = 0;
};
bool best_schedule(const Problem* p, int count, const int (&workers)[3], Schedule& best) {
  bool found = false;
  for (int i = 0; i < 3; ++i) {
    const Tiling& t = TILINGS[i];
    if (found) {  // not if it could not do better with all its workers busy all the time
      double work = 0.0;
      for (int g = 0; g < count; ++g)
        work += static_cast<double>((p[g].m + t.m - 1) / t.m) * ((p[g].n + t.n - 1) / t.n) * kblocks_of(p[g]);
      if (work * t.us / workers[i] + 4.0 > best.us * 0.97) continue;
    }
    Schedule s;
    const bool fits = make_schedule(p, count, i, workers[i], s);
    if (fits && (!found || s.us < 0.97 * best.us)) best = s, found = true;
    if (!found) break;  // too many large tiles: one product at a time, by number
  }
  return found;
}
const Schedule* schedule_for(const Problem* p, int count, const int (&workers)[3], Schedule& room) {
  thread_local std::unique_ptr<Kept> kept(new (std::nothrow) Kept);
  Sizes z;
  memset(&z, 0, sizeof(z));
  z.count = count;
  memcpy(z.workers, workers, sizeof(workers));
  for (int g = 0; g < count; ++g) z.m[g] = p[g].m, z.n[g] = p[g].n, z.k[g] = p[g].k, z.k0[g] = p[g].k0;
  if (!kept) return best_schedule(p, count, workers, room) ? &room : nullptr;
  Kept& c = *kept;
  int at = 0;
  while (at < c.used && memcmp(&c.sizes[at], &z, sizeof(z))) ++at;
  if (at == c.used) {
    at = c.next;
    c.next = (c.next + 1) % Kept::N;
    c.used = std::max(c.used, at + 1);
    c.sizes[at] = z;
    c.listed[at] = best_schedule(p, count, workers, c.schedule[at]);
  }
  return c.listed[at] ? &c.schedule[at] : nullptr;
}

Target target_of(const Result& r, const Problem& p) {
  Target t = {r.p, r.addend, r.alpha, r.ld, r.ld_addend, r.type, r.accumulate, 1};
  const int per = 16 / elem_size(r.type);
  if (!aligned(r.p, 16) || (p.m > 1 && r.ld % per) || (r.addend && (!aligned(r.addend, 16) || (p.m > 1 && r.ld_addend % 4)))) t.vec = 0;
  return t;
}

template <int CTAS, int BN, int N>
int start_listed(const char* who, const Device& d, int half, const Problem* p, const Targets& to, int count, const Schedule& s,
                 cudaStream_t st) {
  using EPI = Store<N>;
  using TILE = Tile<CTAS, BN, EPI>;
  Maps maps = {};
  Shape shape = {};
  shape.half = half;
  typename EPI::Params params;
  params.to = to, params.tile_m = TILE::M, params.tile_n = TILE::BN;
  int map = 0;
  for (int g = 0; g < count; ++g) {
    if (map + 2 > MAX_MAPS) return fail("%s: too many operands in one launch", who);
    if (make_maps<TILE, false>(p[g], maps, map)) return 1;
    shape.group[g] = group_of(p[g], map);
    map += p[g].k0 < p[g].k ? 2 : 1;
  }
  memcpy(params.list.unit, s.unit, sizeof(Listed) * s.units);
  memcpy(params.list.slot, s.slot, sizeof(short) * s.units);
  memcpy(params.list.first, s.first, sizeof(short) * (s.workers + 1));
  int workers = 0;
  cudaError_t e = workers_of<TILE, EPI>(d, &workers);  // its shared memory is allowed on the way
  if (e == cudaSuccess) e = launch_gemm<TILE, EPI>(maps, shape, params, s.workers, st);
  if (e != cudaSuccess) return fail_cuda(who, e);
  if (!s.cuts) return 0;
  JoinArgs j;
  j.to = to, j.tile_m = TILE::M, j.tile_n = TILE::BN;
  for (int g = 0; g < count; ++g) j.group[g] = shape.group[g];
  memcpy(j.cut, s.cut, sizeof(Cut) * s.cuts);
  e = launch_early<join_kernel>(dim3(TILE::M / JOIN_ROWS, s.cuts), 256, 0, st, j);
  return e == cudaSuccess ? 0 : fail_cuda(who, e);
}
template <int CTAS, int BN>
int start_schedule(const char* who, const Device& d, int half, const Problem* p, const Targets& to, int count, const Schedule& s,
                   cudaStream_t st) {
  return s.units <= SMALL_LIST ? start_listed<CTAS, BN, SMALL_LIST>(who, d, half, p, to, count, s, st)
                               : start_listed<CTAS, BN, LARGE_LIST>(who, d, half, p, to, count, s, st);
}

}  // namespace

size_t partial_bytes(const Device& d) {
  return room(sizeof(float) * partial_elements(d.sms));
}

int store_products(const char* who, const Device& d, int half, const Problem* p, const Result* r, int count, float* partial,
                   cudaStream_t st) {
  Targets to = {};
  to.partial = partial;
  for (int g = 0; g < count; ++g) to.t[g] = target_of(r[g], p[g]);
  int workers[3];
  cudaError_t e = workers_of<Tile<2, 256, Store<SMALL_LIST>>, Store<SMALL_LIST>>(d, &workers[0]);
  if (e == cudaSuccess) e = workers_of<Tile<1, 128, Store<SMALL_LIST>>, Store<SMALL_LIST>>(d, &workers[1]);
  if (e == cudaSuccess) e = workers_of<Tile<1, 64, Store<SMALL_LIST>>, Store<SMALL_LIST>>(d, &workers[2]);
  if (e != cudaSuccess) return fail_cuda(who, e);
  Schedule room;
  const Schedule* best = schedule_for(p, count, workers, room);
  if (!best) {
    if (count > 1) {
      for (int g = 0; g < count; ++g)
        if (store_products(who, d, half, p + g, r + g, 1, partial, st)) return 1;
      return 0;
    }
    Store<0>::Params params = {};
    params.to = to;
    return start_tile<Tile<2, 256, Store<0>>, Store<0>>(who, d, p[0], half, params, st);
  }
  const Schedule& b = *best;
  return b.tiling == 0   ? start_schedule<2, 256>(who, d, half, p, to, count, b, st)
         : b.tiling == 1 ? start_schedule<1, 128>(who, d, half, p, to, count, b, st)
                         : start_schedule<1, 64>(who, d, half, p, to, count, b, st);
}

int pack_rows(const char* who, const Device& d, const Pack* packs, int count, cudaStream_t st) {
  if (!count) return 0;
  PackArgs a = {};
  long long most = 0;
  for (int i = 0; i < count; ++i) {
    a.pack[i] = packs[i];
    most = std::max(most, packs[i].rows * ((packs[i].cols + 7) / 8));
  }
  const cudaError_t e = launch_early<pack_kernel>(dim3(static_cast<unsigned>(std::min<long long>((most + 255) / 256, 8 * d.sms)), count), 256, 0, st, a);
  return e == cudaSuccess ? 0 : fail_cuda(who, e);
}

}  // namespace adgemm
