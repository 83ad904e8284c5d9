// Log probabilities of given tokens under softmax(scale x W^T) over a large
// vocabulary, without its logits in memory: ad_linear_logprobs and its gradient.
//
//   z = x W^T;  lse = log sum_v exp(scale z_v);  logp = scale z_t - lse
//   dz = scale ((g_lse - g_logp) p + g_logp [v = t]),  p = exp(scale z - lse)
//   dx = dz W,  dW = dz^T x
//
// Bound by the tensor cores (gemm16.cuh).  Forward: a tile's epilogue reduces each
// row of its logits to their largest and the sum of exponents from there, one pass
// over the accumulator with a running maximum; a small kernel joins the tiles'
// pairs.  Backward: pieces of the vocabulary, of each of which the logits are made
// again (a product of three instead of two; kept they would be rows x vocab), turned
// into dz in the epilogue, rounded to the operands' type and used twice: as rows for
// dx, which is summed over the pieces in 32 bits, and across for the piece's rows of dW.
//
// Logits are what the tensor cores sum, which truncate as they add: where terms have one sign and
// size, 1.55e-8 of a sum for each 16 elements that went into it, where the sums fit 24 bits nothing.  It depends
// on the data, so it is not given back, but kept small: widths are summed in parts (WHOLE).
//
// dz in f16 is held times a power of two that puts the largest gradient of a row
// at 2^14: what it loses is below 2^-38 of that.
//
#include <cfloat>
#include <cmath>

#include "gemm16.cuh"

namespace {

using namespace adgemm;

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Logits of a width above WHOLE are summed in parts of about LENGTH (FOLD), joined in registers and
// rounded to nearest there: what the tensor cores truncate grows with the sum that they add to (lse of width
// 4096 over dense states: 1.9e-6 of it in one accumulator, 4.4e-7 in four parts; of 1024 4.6e-7).  The same
// parts forward and backward, or a probability near 1 would be off by the difference.  A part's
// products take longer than an epilogue, which so stays hidden, and what the joins cost is 2 to 8%: 8192 x 2048 over
// 65537 tokens takes 5430 us backward instead of 5180, 2047 x 1600 over 50001 290 forward instead of 272 and 895
// backward instead of 860, 2000 x 4096 over 32000 445 and 1435 instead of 430 and 1400 (medians of three runs by turns;
// forward at 2048 within the noise).  Below 1536 parts would be shorter than an epilogue: of 550, 323 us instead of 295.
constexpr int LENGTH = 1024, WHOLE = 1536;
template <bool FOLD, int WARPS>
struct Held {
  float held[256 / CHUNK / (WARPS / 4)][CHUNK];  // of each of the warp's chunks
  __device__ Held() {
#pragma unroll
    for (auto& h : held)
#pragma unroll
      for (float& x : h) x = 0.0f;
  }
  __device__ __forceinline__ void hold(const Spot& s, unsigned acc, int i) { add32(s, acc, held[i]); }
  // the whole sums of the warp's chunk i
  __device__ __forceinline__ float (&take(const Spot& s, unsigned acc, int i))[32] {
    add32(s, acc, held[i]);
    return held[i];
  }
};
template <int WARPS>
struct Held<false, WARPS> {
  float sums[CHUNK];
  __device__ __forceinline__ float (&take(const Spot& s, unsigned acc, int))[32] {
    take32(s, acc, sums);
    return sums;
  }
};

struct SumParams {
  float2* part;   // [column tiles][rows]
  float* target;  // [rows]
  const void* tokens;
  int tok64;
  float k;  // scale log2(e)
};
// us of a tile's epilogue (tiling_for).
struct SumCosts {
  static constexpr double US[3] = {4.0, 2.2, 1.5};
};
// A row's largest logit and the sum of exponents from there, over a tile's columns.
template <bool FOLD>
struct Sum : SumCosts {
  static constexpr bool DUAL = false;
  static constexpr int WARPS = 8, SIDE = 512, PART = FOLD ? LENGTH / BK : 0;
  using Units = ByNumber;
  using Params = SumParams;
  struct State : Held<FOLD, WARPS> {
    float top, sum;
    int token;  // -1: not in reach
    __device__ State(const Params& p, const Shape&, const Spot& s) {
      top = -INFINITY, sum = 0.0f, token = -1;
      const int row = s.row0 + s.lane;
      if (row < s.m) {
        const long long t = token_at(p.tokens, p.tok64, row);
        if (t >= 0 && t < s.n) token = static_cast<int>(t);
      }
    }
    __device__ void chunk(const Params& p, const Shape&, const Spot& s, int col0, unsigned acc, int i) {
      float(&v)[32] = this->take(s, acc, i);
      if (col0 + CHUNK > s.n) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col0 + j >= s.n) v[j] = -INFINITY;
      }
      const unsigned at = static_cast<unsigned>(token - col0);
      if (__any_sync(0xffffffffu, at < 32u)) {
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (at == j) z = v[j];
        if (at < 32u) p.target[s.row0 + s.lane] = z;
      }
      float most = v[0];
#pragma unroll
      for (int j = 1; j < 32; ++j) most = fmaxf(most, v[j]);
      most = fmaxf(most, top);
      const float from = most == -INFINITY ? 0.0f : most;
      // the difference first: scale times a large logit would lose what tells logits apart
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < 32; ++j) part[j & 3] += ex2((v[j] - from) * p.k);
      sum = sum * ex2((top - from) * p.k) + ((part[0] + part[1]) + (part[2] + part[3]));
      top = most;
    }
    static constexpr int PARTS = WARPS / 4;
    // The warps of the same 32 rows join their pairs.  A warp's place for them is
    // used again two tiles later, when all have met once more.
    __device__ void end(const Params& p, const Shape&, const Spot& s) {
      const int row = s.row0 + s.lane;
      if (s.dead) sum = __int_as_float(0x7fffffff);
      const unsigned at = s.side + s.odd * 256 + s.lane * 8;
      if (s.part) asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(top), "f"(sum) : "memory");
      asm volatile("bar.sync %0, %1;" ::"r"(1 + s.quad), "r"(32 * PARTS) : "memory");
      if (s.part) return;
#pragma unroll
      for (int i = 1; i < PARTS; ++i) {
        float t, u;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(t), "=f"(u) : "r"(at + i * 4 * SIDE) : "memory");
        const float most = fmaxf(top, t), from = most == -INFINITY ? 0.0f : most;
        sum = sum * ex2((top - from) * p.k) + u * ex2((t - from) * p.k);
        top = most;
      }
      if (row < s.m) p.part[static_cast<long long>(s.unit.col) * s.m + row] = make_float2(top, sum);
    }
  };
};

struct FinishArgs {
  const float2* part;
  const float* target;
  const void* tokens;
  int tok64, parts, rows;
  long long vocab;
  float scale, k;
  float *logp, *lse;
  float2* stats;
};

// Joins the tiles' pairs: 8 rows a block, 4 lanes of each of 16 warps a row.
constexpr int FINISH_WARPS = 16, FINISH_ROWS = 8;
__global__ void __launch_bounds__(32 * FINISH_WARPS) finish_kernel(const __grid_constant__ FinishArgs a) {
  after_previous();
  __shared__ float2 buf[FINISH_WARPS][FINISH_ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * FINISH_ROWS + (lane & (FINISH_ROWS - 1));
  float top = -INFINITY, sum = 0.0f;
  auto join = [&](float2 x) {
    const float most = fmaxf(top, x.x), from = most == -INFINITY ? 0.0f : most;
    sum = sum * ex2((top - from) * a.k) + x.y * ex2((x.x - from) * a.k);
    top = most;
  };
  if (row < a.rows) {
#pragma unroll 4
    for (int i = warp * 4 + lane / FINISH_ROWS; i < a.parts; i += FINISH_WARPS * 4) join(a.part[static_cast<long long>(i) * a.rows + row]);
  }
#pragma unroll
  for (int o = FINISH_ROWS; o < 32; o <<= 1)
    join(make_float2(__shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, sum, o)));
  if (lane < FINISH_ROWS) buf[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp || lane >= FINISH_ROWS || row >= a.rows) return;
  for (int w = 1; w < FINISH_WARPS; ++w) join(buf[w][lane]);
  const long long t = token_at(a.tokens, a.tok64, row);
  const float log_sum = logf(sum);
  a.lse[row] = a.scale * top + log_sum;
  a.logp[row] = t < 0          ? 0.0f
                : t >= a.vocab ? __int_as_float(0x7fffffff)
                               : a.scale * (a.target[row] - top) - log_sum;
  a.stats[row] = make_float2(top, sum);
}

// The power of two for f16 (factor[0]) and its reciprocal (factor[1]), from the rows' gradients as
// far as they have a part in any: g_logp not where there is no token, and nothing of a row whose
// token is past the vocabulary, which is NaN whatever the factor is; nor of rows whose gradients are
// infinite or NaN.  In 64 bits: a gradient times the scale may be past 32.
struct RangeArgs {
  const float *g_logp, *g_lse;
  const void* tokens;
  int tok64;
  long long vocab;
  int rows;
  float scale;
  float* factor;
};
__global__ void __launch_bounds__(1024) range_kernel(const __grid_constant__ RangeArgs a) {
  after_previous();
  __shared__ double buf[32];
  double most = 0.0;
  for (int i = threadIdx.x; i < a.rows; i += 1024) {
    const long long t = token_at(a.tokens, a.tok64, i);
    if (t >= a.vocab) continue;
    const double gp = a.g_logp && t >= 0 ? a.g_logp[i] : 0.0f, gl = a.g_lse ? a.g_lse[i] : 0.0f;
    const double size = 2.0 * fabs(gp) + fabs(gl);
    if (size < INFINITY) most = fmax(most, size);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) most = fmax(most, buf[w]);
    most *= a.scale;
    const int e = most > 0.0 ? max(-126, min(126, 14 - ilogb(most))) : 0;
    a.factor[0] = ldexpf(1.0f, e);
    a.factor[1] = ldexpf(1.0f, -e);
  }
}

struct SlopeParams {
  const float2* stats;
  const void* tokens;
  int tok64;
  const float *g_logp, *g_lse;
  const float* factor;
  long long vocab, first;  // of all; the piece's first column
  float k, scale;
  unsigned short* out;
  long long ld;
};
struct SlopeCosts {
  static constexpr double US[3] = {4.5, 2.5, 1.7};
};
// dz of a piece of the vocabulary.
template <bool FOLD>
struct Slope : SlopeCosts {
  static constexpr bool DUAL = false;
  static constexpr int WARPS = 16, SIDE = 2048, PART = FOLD ? LENGTH / BK : 0;
  using Units = ByNumber;
  using Params = SlopeParams;
  struct State : Held<FOLD, WARPS> {
    float top, of_p, of_hot;
    int hot;  // the token's column in the piece
    __device__ State(const Params& p, const Shape&, const Spot& s) {
      top = 0.0f, of_p = 0.0f, of_hot = 0.0f, hot = -1;
      const int row = s.row0 + s.lane;
      if (row >= s.m) return;
      const float2 st = p.stats[row];
      const long long t = token_at(p.tokens, p.tok64, row);
      // in 64 bits until the factor is on: without it they may be past 32
      const double f = p.scale * (p.factor ? static_cast<double>(*p.factor) : 1.0);
      const double gp = p.g_logp && t >= 0 ? p.g_logp[row] : 0.0f, gl = p.g_lse ? p.g_lse[row] : 0.0f;
      top = st.x;
      of_p = t >= p.vocab ? __int_as_float(0x7fffffff) : static_cast<float>((gl - gp) * f) / st.y;
      of_hot = static_cast<float>(gp * f);
      if (t >= p.first && t < p.first + s.n) hot = static_cast<int>(t - p.first);
    }
    __device__ void chunk(const Params& p, const Shape& a, const Spot& s, int col0, unsigned acc, int i) {
      float(&v)[32] = this->take(s, acc, i);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = ex2((v[j] - top) * p.k) * of_p;
      const unsigned at = static_cast<unsigned>(hot - col0);
      if (__any_sync(0xffffffffu, at < 32u)) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (at == j) v[j] += of_hot;
      }
      unsigned w[16];
      if (a.half) {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], 1);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], 0);
      }
      put16(s, w, p.out, p.ld, s.m, s.n, col0, 1);
    }
    __device__ void end(const Params&, const Shape&, const Spot&) {}
  };
};

// ------------------------------------------------------------------ host

// Elements of dz at a time: about half a gigabyte, up to one and a half times that.  Only the vocabulary is
// cut, and a piece has about 1024 columns or more, so that above 2^18 rows dz takes 2 to 4 KB a row, like operands of
// that width (and sums of dx, 4 bytes an element).
constexpr long long PIECE = 1ll << 28;

struct Layout {
  bool pack_x, pack_w;
  long long ld_packed;
  int tiling;  // of the product with an epilogue of its own
  long long piece, pieces;
  size_t x, w, part, target, factor, dz, sum, partial, total;
};

long long parts_of(int tiling, long long vocab) { return (vocab + TILINGS[tiling].n - 1) / TILINGS[tiling].n; }

Layout plan(const Device& d, const void* x, long long ldx, const void* w, long long ldw, long long rows, long long width,
            long long vocab, bool grad) {
  Layout l = {};
  l.pack_x = !tma_ready(x, ldx, rows), l.pack_w = !tma_ready(w, ldw, vocab);
  l.ld_packed = round_up(width, 64);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += room(bytes);
    return here;
  };
  if (l.pack_x) l.x = take(2ull * rows * l.ld_packed);
  if (l.pack_w) l.w = take(2ull * vocab * l.ld_packed);
  const long long kblocks = (width + BK - 1) / BK;
  if (!grad) {
    l.tiling = tiling_for<SumCosts>(rows, vocab, kblocks, d.sms);
    l.part = take(sizeof(float2) * parts_of(l.tiling, vocab) * rows);
    l.target = take(sizeof(float) * rows);
  } else {
    l.pieces = (vocab * rows + PIECE / 2) / PIECE;
    // at least 1024 columns, so that the products with a piece do not fall apart
    l.pieces = std::max(1ll, std::min(l.pieces, (vocab + 1023) / 1024));
    l.piece = std::min(round_up((vocab + l.pieces - 1) / l.pieces, 256), round_up(vocab, 8));
    l.pieces = (vocab + l.piece - 1) / l.piece;
    l.tiling = tiling_for<SlopeCosts>(rows, std::min(l.piece, vocab), kblocks, d.sms);
    l.factor = take(2 * sizeof(float));
    l.dz = take(2ull * rows * l.piece);
    if (l.pieces > 1) l.sum = take(sizeof(float) * rows * round_up(width, 4));
    l.partial = take(partial_bytes(d));
  }
  l.total = at;
  return l;
}

// Copies of the operands that TMA cannot read as they are.
int pack(const char* who, const Device& d, const Layout& l, const void* x, long long ldx, const void* w, long long ldw,
         long long rows, long long width, long long vocab, unsigned char* ws, cudaStream_t st) {
  Pack packs[2];
  int n = 0;
  if (l.pack_x) packs[n++] = {x, ws + l.x, rows, width, ldx, l.ld_packed};
  if (l.pack_w) packs[n++] = {w, ws + l.w, vocab, width, ldw, l.ld_packed};
  return pack_rows(who, d, packs, n, st);
}

int check(const char* who, int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t width,
          int64_t vocab) {
  if (dtype != AD_BF16 && dtype != AD_F16) return fail("%s: unknown element type %d (AD_BF16 or AD_F16)", who, dtype);
  if (rows < 0 || width < 1 || vocab < 1) return fail("%s: %lld rows of %lld, %lld tokens", who, (long long)rows, (long long)width, (long long)vocab);
  if (rows > (1 << 24) || width > (1 << 20) || vocab > (1 << 24))
    return fail("%s: at most 2^24 rows and tokens, of 2^20 elements", who);
  if ((rows > 1 && ldx < width) || (vocab > 1 && ldw < width)) return fail("%s: rows overlap", who);
  if (!aligned({x, w}, 2)) return fail("%s: an operand is not aligned to its elements", who);
  return 0;
}

}  // namespace

extern "C" int ad_linear_logprobs_workspace(int device, int dtype, const void* x, int64_t ldx, const void* weight,
                                            int64_t ldw, int64_t rows, int64_t width, int64_t vocab, int grad,
                                            size_t* bytes) {
  const char* who = "ad_linear_logprobs_workspace";
  if (!bytes) return fail("%s: null operand", who);
  if (check(who, dtype, x, ldx, weight, ldw, rows, width, vocab)) return 1;
  *bytes = 0;
  if (!rows) return 0;
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
  const Device d = {guard.device(), sm_count(guard.device())};
  if (!d.sms) return fail("%s: no device properties", who);
  *bytes = plan(d, x, ldx, weight, ldw, rows, width, vocab, grad != 0).total;
  return 0;
}

extern "C" int ad_linear_logprobs(int device, int dtype, const void* x, int64_t ldx, const void* weight, int64_t ldw,
                                  int64_t rows, int64_t width, int64_t vocab, const void* tokens, int tok64, float scale,
                                  float* logp, float* lse, float* stats, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  const char* who = "ad_linear_logprobs";
  if (check(who, dtype, x, ldx, weight, ldw, rows, width, vocab)) return 1;
  if (!(scale > 0.0f && scale <= FLT_MAX)) return fail("%s: scale %g", who, scale);
  if (!rows) return 0;
  if (!x || !weight || !tokens || !logp || !lse || !stats) return fail("%s: null operand", who);
  if (!aligned(tokens, tok64 ? 8 : 4) || !aligned({logp, lse}, 4) || !aligned(stats, 8))
    return fail("%s: an operand is not aligned to its elements", who);
  const long long tokens_bytes = rows * (tok64 ? 8 : 4), ws_bytes = static_cast<long long>(workspace_bytes);
  if (overlap({{logp, 1, rows * 4, 0, true}, {lse, 1, rows * 4, 0, true}, {stats, 1, rows * 8, 0, true}, {workspace, 1, ws_bytes, 0, true},
               {x, rows, width * 2, ldx * 2, false}, {weight, vocab, width * 2, ldw * 2, false}, {tokens, 1, tokens_bytes, 0, false}}))
    return fail("%s: results overlap operands or one another", who);
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
  const Device d = {guard.device(), sm_count(guard.device())};
  if (!d.sms) return fail("%s: no device properties", who);
  const Layout l = plan(d, x, ldx, weight, ldw, rows, width, vocab, false);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.total)
    return fail("%s: needs %zu bytes of workspace, 256-byte aligned", who, l.total);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  Problem p = {rows, vocab, width, width, false, false, {}, {}};
  p.a[0] = l.pack_x ? Mat{ws + l.x, l.ld_packed} : Mat{x, ldx};
  p.b[0] = l.pack_w ? Mat{ws + l.w, l.ld_packed} : Mat{weight, ldw};
  if (pack(who, d, l, x, ldx, weight, ldw, rows, width, vocab, ws, st)) return 1;
  SumParams q = {};
  q.part = reinterpret_cast<float2*>(ws + l.part);
  q.target = reinterpret_cast<float*>(ws + l.target);
  q.tokens = tokens, q.tok64 = tok64;
  q.k = std::min(scale * LOG2E, FLT_MAX);
  const int half = dtype == AD_F16;
  if (width > WHOLE ? start<Sum<true>>(who, d, p, half, l.tiling, q, st) : start<Sum<false>>(who, d, p, half, l.tiling, q, st)) return 1;
  FinishArgs f = {};
  f.part = q.part, f.target = q.target, f.tokens = tokens, f.tok64 = tok64;
  f.parts = static_cast<int>(parts_of(l.tiling, vocab)), f.rows = static_cast<int>(rows);
  f.vocab = vocab, f.scale = scale, f.k = q.k;
  f.logp = logp, f.lse = lse, f.stats = reinterpret_cast<float2*>(stats);
  const cudaError_t e = launch_early<finish_kernel>(dim3(static_cast<unsigned>((rows + FINISH_ROWS - 1) / FINISH_ROWS)), 32 * FINISH_WARPS, 0, st, f);
  return e == cudaSuccess ? 0 : fail_cuda(who, e);
}

extern "C" int ad_linear_logprobs_grad(int device, int dtype, const void* x, int64_t ldx, const void* weight, int64_t ldw,
                                       int64_t rows, int64_t width, int64_t vocab, const void* tokens, int tok64,
                                       float scale, const float* stats, const float* g_logp, const float* g_lse, void* dx,
                                       int64_t lddx, int dw_type, void* dw, int64_t lddw, int accumulate, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  const char* who = "ad_linear_logprobs_grad";
  if (check(who, dtype, x, ldx, weight, ldw, rows, width, vocab)) return 1;
  if (dw_type != dtype && dw_type != AD_F32) return fail("%s: unknown type %d of the weight's gradient", who, dw_type);
  if (!(scale > 0.0f && scale <= FLT_MAX)) return fail("%s: scale %g", who, scale);
  if (!dw || !aligned(dw, elem_size(dw_type))) return fail("%s: an operand is null or not aligned to its elements", who);
  if ((rows > 1 && lddx < width) || (vocab > 1 && lddw < width)) return fail("%s: rows overlap", who);
  const size_t es = elem_size(dw_type);
  if (!rows) return accumulate ? 0 : ad_clear_rows(device, dw, lddw * es, width * es, vocab, stream);
  if (!x || !weight || !tokens || !stats || !dx) return fail("%s: null operand", who);
  if (!aligned(tokens, tok64 ? 8 : 4) || !aligned({g_logp, g_lse}, 4) || !aligned(stats, 8) || !aligned(dx, 2))
    return fail("%s: an operand is not aligned to its elements", who);
  const long long tokens_bytes = rows * (tok64 ? 8 : 4), ws_bytes = static_cast<long long>(workspace_bytes);
  if (overlap({{dx, rows, width * 2, lddx * 2, true}, {dw, vocab, static_cast<long long>(width * es), static_cast<long long>(lddw * es), true},
               {workspace, 1, ws_bytes, 0, true}, {x, rows, width * 2, ldx * 2, false}, {weight, vocab, width * 2, ldw * 2, false},
               {tokens, 1, tokens_bytes, 0, false}, {stats, 1, rows * 8, 0, false}, {g_logp, 1, rows * 4, 0, false},
               {g_lse, 1, rows * 4, 0, false}}))
    return fail("%s: results overlap operands or one another", who);
  DeviceGuard guard(device);
  if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
  const Device d = {guard.device(), sm_count(guard.device())};
  if (!d.sms) return fail("%s: no device properties", who);
  const int half = dtype == AD_F16;
  const Layout l = plan(d, x, ldx, weight, ldw, rows, width, vocab, true);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.total)
    return fail("%s: needs %zu bytes of workspace, 256-byte aligned", who, l.total);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const Mat mx = l.pack_x ? Mat{ws + l.x, l.ld_packed} : Mat{x, ldx};
  const Mat mw = l.pack_w ? Mat{ws + l.w, l.ld_packed} : Mat{weight, ldw};
  if (pack(who, d, l, x, ldx, weight, ldw, rows, width, vocab, ws, st)) return 1;
  float* factor = half ? reinterpret_cast<float*>(ws + l.factor) : nullptr;
  if (half) {
    const RangeArgs r = {g_logp, g_lse, tokens, tok64, vocab, static_cast<int>(rows), scale, factor};
    const cudaError_t e = launch_early<range_kernel>(1, 1024, 0, st, r);
    if (e != cudaSuccess) return fail_cuda(who, e);
  }
  const Mat dz = {ws + l.dz, l.piece};
  for (long long i = 0; i < l.pieces; ++i) {
    const long long v0 = i * l.piece, n = std::min(l.piece, vocab - v0);
    const Mat w = {static_cast<const unsigned short*>(mw.p) + v0 * mw.ld, mw.ld};
    Problem p = {rows, n, width, width, false, false, {mx, {}}, {w, {}}};
    SlopeParams q = {};
    q.stats = reinterpret_cast<const float2*>(stats);
    q.tokens = tokens, q.tok64 = tok64;
    q.g_logp = g_logp, q.g_lse = g_lse, q.factor = factor;
    q.vocab = vocab, q.first = v0;
    q.k = std::min(scale * LOG2E, FLT_MAX), q.scale = scale;
    q.out = reinterpret_cast<unsigned short*>(ws + l.dz), q.ld = l.piece;
    if (width > WHOLE ? start<Slope<true>>(who, d, p, half, l.tiling, q, st) : start<Slope<false>>(who, d, p, half, l.tiling, q, st)) return 1;
    const Problem products[2] = {{rows, width, n, n, false, true, {dz, {}}, {w, {}}},
                                 {n, width, rows, rows, true, true, {dz, {}}, {mx, {}}}};
    // dx: sums over the pieces stay in 32 bits until the last one's
    float* sum = reinterpret_cast<float*>(ws + l.sum);
    const long long ld_sum = round_up(width, 4);
    const bool first = i == 0, last = i + 1 == l.pieces;
    const float* alpha = factor ? factor + 1 : nullptr;
    const Result results[2] = {
        {last ? dx : sum, last ? lddx : ld_sum, last ? dtype : AD_F32, false, first ? nullptr : sum, ld_sum, last ? alpha : nullptr},
        {static_cast<unsigned char*>(dw) + v0 * lddw * es, lddw, dw_type, accumulate != 0, nullptr, 0, alpha}};
    if (store_products(who, d, half, products, results, 2, reinterpret_cast<float*>(ws + l.partial), st)) return 1;
  }
  return 0;
}
