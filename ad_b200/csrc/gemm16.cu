// Products of 16-bit matrices to memory (gemm16.cuh): results in 16 or 32 bits,
// sums over several products, splits of a long K, and copies of operands whose
// rows are not aligned to the 16 bytes that TMA asks for.
#include "gemm16.cuh"

namespace adgemm {

namespace {

struct Store {
  static constexpr bool DUAL = false;
  struct Params {
    void* out[MAX_GROUPS];
    long long ld[MAX_GROUPS];
    long long split_stride;  // elements between the partial sums of two splits
    long long group_stride;  // and of two groups
    int type;                // AD_F32, or the operands'
    int vec;                 // 16-byte stores are aligned
    int accumulate;
    const float* alpha;
  };
  struct State {
    unsigned char* out;
    long long ld;
    float alpha;
    __device__ State(const Params& p, const Shape&, const Spot& s) {
      const int g = p.split_stride ? 0 : s.group;
      ld = p.ld[g];
      out = static_cast<unsigned char*>(p.out[g]) +
            (p.split_stride ? 4 * (s.split * p.split_stride + s.group * p.group_stride) : 0);
      alpha = p.alpha ? *p.alpha : 1.0f;
    }
    __device__ void end(const Params&, const Shape&, const Spot&) {}
    __device__ void chunk(const Params& p, const Shape& a, const Spot& s, int col0, unsigned acc, int) {
      float v[32];
      tmem_ld32(acc, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = s.dead ? __int_as_float(0x7fffffff) : v[j] * alpha;
      if (p.type != AD_F32 && !p.accumulate) {
        unsigned w[16];
        if (a.half) {
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], 1);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], 0);
        }
        put16(s, w, reinterpret_cast<unsigned short*>(out), ld, a.m, a.n, col0, p.vec);
        return;
      }
      stage32(s, v);
      if (p.type == AD_F32) {
        float* o = reinterpret_cast<float*>(out);
        const int q = s.lane & 7, col = col0 + q * 4;
        if (p.vec && col0 + CHUNK <= a.n) {
          float4 old[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (s.lane >> 3);
            old[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (p.accumulate && s.row0 + r < a.m) old[i] = *reinterpret_cast<const float4*>(o + (s.row0 + r) * ld + col);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (s.lane >> 3);
            const float4 x = staged(s, r, q);
            old[i].x += x.x, old[i].y += x.y, old[i].z += x.z, old[i].w += x.w;
            if (s.row0 + r < a.m) *reinterpret_cast<float4*>(o + (s.row0 + r) * ld + col) = old[i];
          }
          return;
        }
      }
      // a column a lane
      const int col = col0 + s.lane;
      if (col >= a.n) return;
      for (int r = 0; r < 32 && s.row0 + r < a.m; ++r) {
        float x = staged1(s, r);
        const long long at = (s.row0 + r) * ld + col;
        if (p.accumulate) x += load_any(out, p.type, at);
        store_any(out, p.type, at, x);
      }
    }
  };
};

struct JoinArgs {
  const float* part;
  long long split_stride, group_stride, ld_part;
  int splits, type, accumulate;
  int m, n;
  void* out[MAX_GROUPS];
  long long ld[MAX_GROUPS];
  const float* alpha;
};

// Partial sums, in order, to the result.  Bound by memory.
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ JoinArgs a) {
  const int g = blockIdx.z;
  const int per = (a.n + 3) / 4;
  const long long total = static_cast<long long>(a.m) * per;
  const float alpha = a.alpha ? *a.alpha : 1.0f;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int r = static_cast<int>(i / per), c = static_cast<int>(i - static_cast<long long>(r) * per) * 4;
    const float* p = a.part + g * a.group_stride + r * a.ld_part + c;
    float4 x = *reinterpret_cast<const float4*>(p);
    for (int s = 1; s < a.splits; ++s) {
      const float4 y = *reinterpret_cast<const float4*>(p + s * a.split_stride);
      x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    const float v[4] = {x.x, x.y, x.z, x.w};
    const long long at = r * a.ld[g] + c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < a.n) {
        float y = v[j] * alpha;
        if (a.accumulate) y += load_any(a.out[g], a.type, at + j);
        store_any(a.out[g], a.type, at + j, y);
      }
  }
}

struct PackArgs {
  const unsigned short* p;
  unsigned short* to;
  long long ld, ld_to, rows;
  int cols;
};
// A row a block and round; what TMA reads past the columns is not read.
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackArgs a) {
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x)
    for (int c = threadIdx.x; c < a.cols; c += 256) a.to[r * a.ld_to + c] = a.p[r * a.ld + c];
}

}  // namespace

Plan store_plan(const Problem& p, int sms) {
  const long long kblocks = (p.k0 + BK - 1) / BK + (p.k - p.k0 + BK - 1) / BK;
  return plan_for(p.m, p.n, kblocks, p.groups, false, true, sms);
}

size_t partial_bytes(const Problem& p, const Plan& plan, bool sums) {
  if (plan.splits == 1 && !sums) return 0;
  return room(sizeof(float) * static_cast<size_t>(plan.splits) * p.groups * p.m * round_up(p.n, 4));
}

int store_product(const char* who, const Problem& p, const Plan& plan, int type, const Out* out, bool accumulate,
                  const float* alpha, float* partial, const Sums* sums, int sms, cudaStream_t st) {
  Store::Params q = {};
  const bool parts = plan.splits > 1 || (sums && !(sums->first && sums->last));
  const long long ld_part = round_up(p.n, 4);
  JoinArgs j = {};
  for (int g = 0; g < p.groups; ++g) j.out[g] = out[g].p, j.ld[g] = out[g].ld;
  if (parts) {
    q.out[0] = partial, q.ld[0] = ld_part;
    q.group_stride = p.m * ld_part, q.split_stride = p.groups * q.group_stride;
    q.type = AD_F32, q.vec = 1;
    q.accumulate = sums && !sums->first;
  } else {
    q.type = type, q.accumulate = accumulate, q.alpha = alpha, q.vec = 1;
    for (int g = 0; g < p.groups; ++g) {
      q.out[g] = out[g].p, q.ld[g] = out[g].ld;
      if (!aligned(out[g].p, 16) || (p.m > 1 && out[g].ld % (16 / elem_size(type)))) q.vec = 0;
    }
  }
  if (start<Store>(who, p, plan, q, sms, st)) return 1;
  if (!parts || (sums && !sums->last)) return 0;
  j.part = partial, j.split_stride = q.split_stride, j.group_stride = q.group_stride, j.ld_part = ld_part;
  j.splits = plan.splits, j.type = type, j.accumulate = accumulate, j.alpha = alpha;
  j.m = static_cast<int>(p.m), j.n = static_cast<int>(p.n);
  const long long blocks = (p.m * (ld_part / 4) + 255) / 256;
  const cudaError_t e = launch<join_kernel>(dim3(static_cast<unsigned>(std::min<long long>(blocks, 8 * sms)), 1, p.groups),
                                            256, 0, st, j);
  return e == cudaSuccess ? 0 : fail_cuda(who, e);
}

int pack_rows(const char* who, const void* p, long long ld, long long rows, long long cols, void* to, long long ld_to,
              cudaStream_t st) {
  PackArgs a = {static_cast<const unsigned short*>(p), static_cast<unsigned short*>(to), ld, ld_to, rows,
                static_cast<int>(cols)};
  const cudaError_t e = launch<pack_kernel>(dim3(static_cast<unsigned>(std::min<long long>(rows, 148 * 8))), 256, 0, st, a);
  return e == cudaSuccess ? 0 : fail_cuda(who, e);
}

}  // namespace adgemm
