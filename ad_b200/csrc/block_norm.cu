// The entry points of the norms around a block, and the kernel that adds up the
// gradient's column sums; block_norm.cuh has the formulas and the row kernels.
#include <algorithm>
#include <initializer_list>

#include "block_norm.cuh"

namespace {

using namespace adops;

struct FinishArgs {
  const float* part;
  long long blocks;           // of the whole launch
  long long blocks_per_run;  // consecutive blocks of one gate row
  int width;
  void* out[SUMS];
  int type[SUMS];
  long long ldg;
};

// Columns' sums over the blocks, in their order: 32 columns a block of
// threads, 32 rows of threads each taking a consecutive share of the blocks.
constexpr int FINISH_ROWS = 32;
__global__ void __launch_bounds__(32 * FINISH_ROWS) norm_finish_kernel(const __grid_constant__ FinishArgs a) {
  __shared__ float buf[FINISH_ROWS][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const int sum = blockIdx.y < 4 ? blockIdx.y : SUM_GATE;
  if (!a.out[sum]) return;
  const long long gate = sum == SUM_GATE ? blockIdx.y - 4 : 0;
  const long long b0 = sum == SUM_GATE ? gate * a.blocks_per_run : 0;
  const long long n = sum == SUM_GATE ? a.blocks_per_run : a.blocks;
  const long long share = (n + FINISH_ROWS - 1) / FINISH_ROWS;
  float s = 0.0f;
  if (c < a.width) {
    const long long e = min(n, (threadIdx.y + 1) * share);
#pragma unroll 8
    for (long long b = threadIdx.y * share; b < e; ++b) s += a.part[((b0 + b) * SUMS + sum) * a.width + c];
  }
  buf[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < a.width) {
    for (int k = 1; k < FINISH_ROWS; ++k) s += buf[k][threadIdx.x];
    store_any(a.out[sum], a.type[sum], (sum == SUM_GATE ? gate * a.ldg : 0) + c, s);
  }
}

// How the gradient's rows are shared out: consecutive rows to a block; where a gate is shared by rows, either several
// blocks to a run of such rows or whole runs to a block.
struct Split {
  long long run, blocks_per_run, rows_per_block, blocks;
};
Split split_rows(long long rows, long long rows_per_gate, int width, bool slim, int sms) {
  Split s;
  s.run = rows_per_gate > 1 ? rows_per_gate : rows;
  // 512 or 768 threads with eight elements each to a multiprocessor, in as many blocks as that makes
  const int per_sm = std::max(1, std::min(16, (slim ? 6144 : 4096) / width));
  const long long runs = rows / s.run, want = static_cast<long long>(per_sm) * sms;
  if (runs >= want) {
    s.blocks_per_run = 0;
    s.rows_per_block = (runs + want - 1) / want * s.run;
    s.blocks = (rows + s.rows_per_block - 1) / s.rows_per_block;
    return s;
  }
  long long per = want / runs;  // no more blocks than are resident at a time
  if (per > s.run) per = s.run;
  s.rows_per_block = (s.run + per - 1) / per;
  s.blocks_per_run = (s.run + s.rows_per_block - 1) / s.rows_per_block;
  s.blocks = s.blocks_per_run * runs;
  return s;
}

bool fits(const void* p, long long ld, int size) {
  return !p || (aligned(p, 16) && (ld * size) % 16 == 0);
}

// The checks and the variant that both directions share.
int check(const char* who, int dtype, int wtype, int kind, const void* x, const void* z, const void* gate,
          int64_t rows_per_gate, int64_t rows, int width, float eps, std::initializer_list<int64_t> lds) {
  if (dtype < AD_F32 || dtype > AD_F16) return fail("%s: unknown element type %d", who, dtype);
  if (wtype != AD_F32 && wtype != dtype) return fail("%s: weights of type %d beside elements of type %d", who, wtype, dtype);
  if (kind != 0 && kind != 1) return fail("%s: unknown norm %d", who, kind);
  if (rows < 0 || width < 1 || width > 32768) return fail("%s: %lld rows of %d elements (1 to 32768)", who, (long long)rows, width);
  if (rows > 0x7fffffffll) return fail("%s: %lld rows in one call", who, (long long)rows);
  for (int64_t ld : lds)
    if (ld < 0 || ld > 0x7fffffffll) return fail("%s: rows %lld elements apart", who, (long long)ld);
  if (!(eps >= 0.0f)) return fail("%s: eps %g", who, eps);
  if (rows && (!x || !z)) return fail("%s: null operand", who);
  if (gate && rows && (rows_per_gate < 1 || rows % rows_per_gate))
    return fail("%s: %lld rows cannot share gates of %lld rows", who, (long long)rows, (long long)rows_per_gate);
  return 0;
}

cudaError_t start_any(const NormArgs& a, int dtype, bool grad, bool gen, bool vec, unsigned blocks, int sms, cudaStream_t s) {
  return dtype == AD_F32    ? start_norm_f32(a, grad, gen, vec, blocks, sms, s)
         : dtype == AD_BF16 ? start_norm_bf16(a, grad, gen, vec, blocks, sms, s)
                            : start_norm_f16(a, grad, gen, vec, blocks, sms, s);
}

}  // namespace

extern "C" int ad_block_norm(int device, int dtype, int wtype, int kind, const void* x, int64_t ldx, const void* z,
                             int64_t ldz, const void* gate, int64_t ldg, int64_t rows_per_gate, int gate_sigmoid,
                             const void* wa, const void* ba, const void* wb, const void* bb, float scale, float eps,
                             int64_t rows, int width, void* h, int64_t ldh, void* y, int64_t ldy, float* stats,
                             void* stream) {
  if (check("ad_block_norm", dtype, wtype, kind, x, z, gate, rows_per_gate, rows, width, eps, {ldx, ldz, ldg, ldh, ldy})) return 1;
  if (rows == 0) return 0;
  if (!h || (wb && !y) || !stats || !aligned(stats, 16)) return fail("ad_block_norm: null or unaligned result");
  if ((ba && !wa) || (bb && !wb)) return fail("ad_block_norm: a bias without its weight");
  if (!aligned({x, z, gate, h, y}, elem_size(dtype)) || !aligned({wa, ba, wb, bb}, elem_size(wtype)))
    return fail("ad_block_norm: an operand is not aligned to its elements");
  NormArgs a = {};
  a.x = x, a.z = z, a.gate = gate;
  a.ldx = ldx, a.ldz = ldz, a.ldg = ldg;
  a.wa = wa, a.ba = ba, a.wb = wb, a.bb = bb;
  a.wtype = wtype;
  a.h = h, a.y = y, a.ldh = ldh, a.ldy = ldy;
  a.stats = stats;
  a.rows = rows, a.rows_per_gate = rows_per_gate;
  a.width = width, a.sigmoid = gate_sigmoid, a.layer = kind;
  a.scale = scale, a.eps = eps;
  const int size = elem_size(dtype);
  const bool vec = width % (16 / size) == 0 && fits(x, ldx, size) && fits(z, ldz, size) && fits(gate, ldg, size) &&
                   fits(h, ldh, size) && fits(y, ldy, size) && fits(wa, 0, 1) && fits(ba, 0, 1) && fits(wb, 0, 1) &&
                   fits(bb, 0, 1);
  DeviceGuard g(device);
  if (g.error() != cudaSuccess) return fail_cuda("ad_block_norm", g.error());
  const int sms = sm_count(g.device());
  if (!sms) return fail("ad_block_norm: no device properties");
  const cudaError_t e = start_any(a, dtype, false, kind || ba || bb, vec, 0, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda("ad_block_norm", e);
  return 0;
}

extern "C" int ad_block_norm_grad_workspace(int device, int64_t rows, int width, int64_t rows_per_gate, size_t* bytes) {
  if (!bytes || rows < 0 || width < 1 || rows_per_gate < 0) return fail("ad_block_norm_grad_workspace: bad argument");
  *bytes = 0;
  if (rows == 0) return 0;
  DeviceGuard g(device);
  const int sms = g.error() == cudaSuccess ? sm_count(g.device()) : 0;
  if (!sms) return fail("ad_block_norm_grad_workspace: no device properties");
  if (rows_per_gate && rows % rows_per_gate) return fail("ad_block_norm_grad_workspace: rows cannot share gates so");
  // for the kernels with the most blocks
  *bytes = sizeof(float) * SUMS * static_cast<size_t>(split_rows(rows, rows_per_gate, width, true, sms).blocks) * width;
  return 0;
}

extern "C" int ad_clear_rows(int device, void* p, int64_t row_stride, int64_t row_bytes, int64_t rows, void* stream) {
  if (row_bytes < 0 || rows < 0 || (rows > 1 && row_stride < row_bytes))
    return fail("ad_clear_rows: %lld rows of %lld bytes, %lld apart", (long long)rows, (long long)row_bytes, (long long)row_stride);
  if (rows == 0 || row_bytes == 0) return 0;
  if (!p) return fail("ad_clear_rows: null operand");
  DeviceGuard g(device);
  if (g.error() != cudaSuccess) return fail_cuda("ad_clear_rows", g.error());
  const cudaError_t e = cudaMemset2DAsync(p, std::max(row_stride, row_bytes), 0, row_bytes, rows, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail_cuda("ad_clear_rows", e);
  return 0;
}

extern "C" int ad_block_norm_grad(int device, int dtype, int wtype, int kind, const void* dh, int64_t lddh,
                                  const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* z, int64_t ldz,
                                  const void* gate, int64_t ldg, int64_t rows_per_gate, int gate_sigmoid,
                                  const void* wa, const void* ba, const void* wb, const void* bb, float scale,
                                  const float* stats, int64_t rows, int width, void* dx, int64_t lddx, void* dz,
                                  int64_t lddz, void* dgate, int64_t lddg, void* dwa, void* dba, void* dwb, void* dbb,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (check("ad_block_norm_grad", dtype, wtype, kind, x, z, gate, rows_per_gate, rows, width, 0.0f,
            {lddh, lddy, ldx, ldz, ldg, lddx, lddz, lddg})) return 1;
  if ((ba && !wa) || (bb && !wb)) return fail("ad_block_norm_grad: a bias without its weight");
  if (!aligned({dh, dy, x, z, gate, dx, dz, dgate}, elem_size(dtype)) ||
      !aligned({wa, ba, wb, bb, dwa, dba, dwb, dbb}, elem_size(wtype)))
    return fail("ad_block_norm_grad: an operand is not aligned to its elements");
  if ((wa && !dwa) || (wb && !dwb) || (ba && !dba) || (bb && !dbb))
    return fail("ad_block_norm_grad: a weight without room for its gradient");
  DeviceGuard g(device);
  if (g.error() != cudaSuccess) return fail_cuda("ad_block_norm_grad", g.error());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int wsize = elem_size(wtype);
  if (rows == 0) {  // sums of nothing
    void* sums[4] = {dwa, dba, dwb, dbb};
    const void* of[4] = {wa, ba, wb, bb};
    for (int k = 0; k < 4; ++k)
      if (of[k]) {
        const cudaError_t e = cudaMemsetAsync(sums[k], 0, static_cast<size_t>(width) * wsize, s);
        if (e != cudaSuccess) return fail_cuda("ad_block_norm_grad", e);
      }
    return 0;
  }
  if (!dh || (wb && !dy) || !dx || !dz || (gate && !dgate) || !stats || !aligned(stats, 16))
    return fail("ad_block_norm_grad: null or unaligned operand");
  const int sms = sm_count(g.device());
  if (!sms) return fail("ad_block_norm_grad: no device properties");
  const Split split = split_rows(rows, gate ? rows_per_gate : 0, width,
                                 elem_size(dtype) == 2 && !kind && !ba && !bb, sms);
  const size_t need = sizeof(float) * SUMS * static_cast<size_t>(split.blocks) * width;
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < need)
    return fail("ad_block_norm_grad: needs %zu bytes of workspace, 16-byte aligned", need);
  NormArgs a = {};
  a.x = x, a.z = z, a.gate = gate, a.dh = dh, a.dy = dy;
  a.ldx = ldx, a.ldz = ldz, a.ldg = ldg, a.lddh = lddh, a.lddy = lddy;
  a.wa = wa, a.ba = ba, a.wb = wb, a.bb = bb;
  a.wtype = wtype;
  a.dx = dx, a.dz = dz, a.dgate = dgate;
  a.lddx = lddx, a.lddz = lddz, a.lddg = lddg;
  a.stats = const_cast<float*>(stats);
  a.part = static_cast<float*>(workspace);
  a.rows = rows, a.rows_per_gate = rows_per_gate;
  a.run = split.run, a.blocks_per_run = split.blocks_per_run, a.rows_per_block = split.rows_per_block;
  a.width = width, a.sigmoid = gate_sigmoid, a.layer = kind;
  a.scale = scale;
  const int size = elem_size(dtype);
  const bool vec = width % (16 / size) == 0 && fits(x, ldx, size) && fits(z, ldz, size) && fits(gate, ldg, size) &&
                   fits(dh, lddh, size) && fits(dy, lddy, size) && fits(dx, lddx, size) && fits(dz, lddz, size) &&
                   fits(dgate, lddg, size) && fits(wa, 0, 1) && fits(ba, 0, 1) && fits(wb, 0, 1) && fits(bb, 0, 1);
  cudaError_t e = start_any(a, dtype, true, kind || ba || bb, vec, static_cast<unsigned>(split.blocks), sms, s);
  if (e != cudaSuccess) return fail_cuda("ad_block_norm_grad", e);
  FinishArgs f = {};
  f.part = a.part;
  f.blocks = split.blocks, f.blocks_per_run = split.blocks_per_run;
  f.width = width;
  f.out[SUM_WA] = wa ? dwa : nullptr, f.out[SUM_WB] = wb ? dwb : nullptr;
  f.out[SUM_BA] = ba ? dba : nullptr, f.out[SUM_BB] = bb ? dbb : nullptr;
  for (int k = 0; k < 4; ++k) f.type[k] = wtype;
  const bool shared = gate && rows_per_gate > 1 && split.blocks_per_run;
  f.out[SUM_GATE] = shared ? dgate : nullptr;
  f.type[SUM_GATE] = dtype;
  f.ldg = lddg;
  const long long gates = shared ? rows / rows_per_gate : 0;  // fewer than blocks
  if (f.out[SUM_WA] || f.out[SUM_WB] || shared) {
    e = launch<norm_finish_kernel>(dim3((width + 31) / 32, static_cast<unsigned>(4 + gates)), dim3(32, FINISH_ROWS), 0, s, f);
    if (e != cudaSuccess) return fail_cuda("ad_block_norm_grad", e);
  }
  return 0;
}
