// The norm of many arrays taken together, and their scaling down to a largest
// norm: ad_clip_norm.
//
//   n = sqrt(sum of g^2 over all arrays);  g = g min(1, max_norm / n)
//
// Bound by memory: each array is read for the norm, and once more, backwards so that
// what the first pass has left in L2 comes first, to be scaled.  Where nothing has
// to be scaled and the arrays are their own results, the second pass ends at once.
// Arrays are cut into chunks of 64 KB, dealt out to the blocks of one launch, whose
// table of arrays travels with its parameters: no copy to the device, and a
// captured call replays by itself.  Squares of 16 bytes' elements are summed in 32
// bits where they can neither overflow nor vanish, else in 64, and all sums of
// those in 64, in an order that only the sizes set.
#include <algorithm>
#include <cmath>
#include <vector>

#include "ops_common.cuh"

namespace {

using namespace adops;

constexpr int THREADS = 256, U = 4;            // 16-byte loads of a thread under way
constexpr int ROUNDS = 4, CHUNK = THREADS * U * ROUNDS;  // 16-byte words of a chunk
// Blocks of a multiprocessor, all of them at a time (1.1 GB clipped into another 1.1 GB: 537 us;
// with 8, of which half wait for the others, 555; with 8 resident ones of 32 registers 669, with 2 733).
constexpr int RESIDENT = 4;
constexpr int MAX_BLOCKS = 2048;               // of a launch: partial sums of a table
constexpr long long MAX_ELEMENTS = 1ll << 44;

// Arrays of one launch.  first[i]: the chunks before array i.
template <int N>
struct Table {
  const void* in[N];
  void* out[N];
  long long count[N];
  unsigned first[N + 1];
  unsigned char type[N];
  int arrays;
};
template <int N>
struct ClipArgs {
  Table<N> t;
  double* part;  // of this table
  const double* parts;  // of all tables
  int all_parts;
  double max_norm;
  float* norm;
};

// Elements before the first 16-byte boundary.
__device__ __forceinline__ long long head_of(const void* p, int size, long long count) {
  const long long n = static_cast<long long>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / size;
  return n < count ? n : count;
}
__device__ __forceinline__ void unpack_any(const uint4& q, int type, float (&x)[8]) {
  if (type == AD_F32)
    unpack<float>(q, x);
  else if (type == AD_BF16)
    unpack<__nv_bfloat16>(q, x);
  else
    unpack<__half>(q, x);
}
__device__ __forceinline__ uint4 pack_any(const float (&x)[8], int type) {
  uint4 q;
  if (type == AD_F32) {
    q = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  } else if (type == AD_BF16) {
    Vec<__nv_bfloat16, 8> v;
    round_to<__nv_bfloat16, 8>(x, v);
    memcpy(&q, &v, 16);
  } else {
    Vec<__half, 8> v;
    round_to<__half, 8>(x, v);
    memcpy(&q, &v, 16);
  }
  return q;
}

// The array that a chunk belongs to.
template <int N>
__device__ __forceinline__ int array_of(const Table<N>& t, unsigned chunk) {
  int lo = 0, hi = t.arrays;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Squares of the n elements of 16 bytes.
__device__ __forceinline__ double squares(const float (&x)[8], int n) {
  float q = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) q = fmaf(x[j], x[j], q);
  if (q > 1e-25f && q < 1e37f) return q;
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) s = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), s);
  return s;
}

__device__ __forceinline__ double block_sum(double s, double* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) s += buf[w];
  return s;
}

template <int N>
__global__ void __launch_bounds__(THREADS, RESIDENT) norm_kernel(const __grid_constant__ ClipArgs<N> a) {
  after_previous();
  __shared__ double buf[THREADS / 32];
  const unsigned chunks = a.t.first[a.t.arrays];
  double s = 0.0;
  for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = array_of(a.t, c), type = a.t.type[i], size = type == AD_F32 ? 4 : 2, per = 16 / size;
    const void* p = a.t.in[i];
    const long long count = a.t.count[i], head = head_of(p, size, count), words = (count - head) / per;
    const uint4* body = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(p) + head * size);
    const long long from = static_cast<long long>(c - a.t.first[i]) * CHUNK, end = from + CHUNK < words ? from + CHUNK : words;
    for (long long w0 = from + threadIdx.x; w0 < end; w0 += THREADS * U) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (w0 + u * THREADS < end) q[u] = body[w0 + u * THREADS];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (w0 + u * THREADS < end) {
          float x[8];
          unpack_any(q[u], type, x);
          s += squares(x, per);
        }
      }
    }
    if (c == a.t.first[i]) {  // what lies before the first and behind the last 16 bytes: fewer than 16 elements
      const long long rest = count - head - words * per;
      if (threadIdx.x < head + rest) {
        const long long at = threadIdx.x < head ? threadIdx.x : head + words * per + (threadIdx.x - head);
        const double x = load_any(p, type, at);
        s = fma(x, x, s);
      }
    }
  }
  s = block_sum(s, buf);
  if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

template <int N>
__global__ void __launch_bounds__(THREADS, RESIDENT) scale_kernel(const __grid_constant__ ClipArgs<N> a) {
  after_previous();
  __shared__ double buf[THREADS / 32];
  double s = 0.0;
  for (int i = threadIdx.x; i < a.all_parts; i += THREADS) s += a.parts[i];
  const double norm = sqrt(block_sum(s, buf));
  if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = static_cast<float>(norm);
  // a norm that is no number leaves all as it is
  const bool clip = norm > a.max_norm && norm < INFINITY;
  const double factor = clip ? a.max_norm / norm : 1.0;
  const float f = static_cast<float>(factor);
  const bool wide = factor < 1e-30;  // products in 64 bits, where the factor is no number of 32 in full
  const unsigned chunks = a.t.first[a.t.arrays];
  for (unsigned k = blockIdx.x; k < chunks; k += gridDim.x) {
    const unsigned c = chunks - 1 - k;
    const int i = array_of(a.t, c), type = a.t.type[i], size = type == AD_F32 ? 4 : 2, per = 16 / size;
    const void* p = a.t.in[i];
    void* o = a.t.out[i];
    if (!clip && p == o) continue;
    const long long count = a.t.count[i], head = head_of(p, size, count), words = (count - head) / per;
    const uint4* body = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(p) + head * size);
    unsigned char* to = static_cast<unsigned char*>(o) + head * size;
    const bool vec = (reinterpret_cast<uintptr_t>(to) & 15) == 0;
    const long long from = static_cast<long long>(c - a.t.first[i]) * CHUNK, end = from + CHUNK < words ? from + CHUNK : words;
    for (long long w0 = from + threadIdx.x; w0 < end; w0 += THREADS * U) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (w0 + u * THREADS < end) q[u] = body[w0 + u * THREADS];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long w = w0 + u * THREADS;
        if (w >= end) continue;
        if (clip) {
          float x[8];
          unpack_any(q[u], type, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = wide ? static_cast<float>(x[j] * factor) : x[j] * f;
          q[u] = pack_any(x, type);
        }
        if (vec) {
          reinterpret_cast<uint4*>(to)[w] = q[u];
        } else {
          const unsigned v[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (size == 4) {
              reinterpret_cast<unsigned*>(to)[w * 4 + j] = v[j];
            } else {
              reinterpret_cast<unsigned short*>(to)[w * 8 + 2 * j] = static_cast<unsigned short>(v[j]);
              reinterpret_cast<unsigned short*>(to)[w * 8 + 2 * j + 1] = static_cast<unsigned short>(v[j] >> 16);
            }
          }
        }
      }
    }
    if (c == a.t.first[i]) {
      const long long rest = count - head - words * per;
      if (threadIdx.x < head + rest) {
        const long long at = threadIdx.x < head ? threadIdx.x : head + words * per + (threadIdx.x - head);
        const float x = load_any(p, type, at);
        store_any(o, type, at, wide ? static_cast<float>(x * factor) : x * f);
      }
    }
  }
}

// Launches of at most N arrays each.
template <int N>
int run(const char* who, const std::vector<int>& which, const void* const* in, void* const* out, const int64_t* counts,
        const int* types, double max_norm, float* norm, double* parts, int sms, cudaStream_t st) {
  const int tables = static_cast<int>((which.size() + N - 1) / N);
  std::vector<ClipArgs<N>> args(std::max(tables, 1));
  std::vector<int> blocks(args.size());
  int all = 0;
  for (size_t k = 0; k < args.size(); ++k) {
    ClipArgs<N>& a = args[k];
    memset(&a, 0, sizeof(a));
    unsigned long long chunks = 0;
    for (size_t j = k * N; j < std::min(which.size(), (k + 1) * N); ++j) {
      const int i = which[j], n = a.t.arrays++;
      a.t.in[n] = in[i], a.t.out[n] = out[i];
      a.t.count[n] = counts[i], a.t.type[n] = static_cast<unsigned char>(types[i]);
      a.t.first[n] = static_cast<unsigned>(chunks);
      const long long words = (counts[i] * elem_size(types[i]) + 15) / 16;
      chunks += (words + CHUNK - 1) / CHUNK;
    }
    if (chunks > 0x7fffffffull) return fail("%s: too many elements in one call", who);
    a.t.first[a.t.arrays] = static_cast<unsigned>(chunks);
    blocks[k] = static_cast<int>(std::max(1ull, std::min<unsigned long long>(chunks, std::min(RESIDENT * sms, MAX_BLOCKS))));
    a.part = parts + all;
    all += blocks[k];
  }
  for (size_t k = 0; k < args.size(); ++k) {
    args[k].parts = parts, args[k].all_parts = all;
    args[k].max_norm = max_norm, args[k].norm = k ? nullptr : norm;
    const cudaError_t e = launch_early<norm_kernel<N>>(dim3(blocks[k]), THREADS, 0, st, args[k]);
    if (e != cudaSuccess) return fail_cuda(who, e);
  }
  for (size_t k = args.size(); k-- > 0;) {  // backwards, too
    const cudaError_t e = launch_early<scale_kernel<N>>(dim3(blocks[k]), THREADS, 0, st, args[k]);
    if (e != cudaSuccess) return fail_cuda(who, e);
  }
  return 0;
}

constexpr int SMALL = 64, LARGE = 768;  // arrays of a launch: 1.7 and 20 KB of parameters

}  // namespace

extern "C" int ad_clip_norm_workspace(int64_t count, size_t* bytes) {
  if (!bytes || count < 0) return fail("ad_clip_norm_workspace: bad argument");
  *bytes = sizeof(double) * MAX_BLOCKS * std::max<int64_t>(1, (count + SMALL - 1) / SMALL);
  return 0;
}

extern "C" int ad_clip_norm(int device, int64_t count, const void* const* in, void* const* out, const int64_t* counts,
                            const int* dtypes, double max_norm, float* norm, void* workspace, size_t workspace_bytes,
                            void* stream) {
  const char* who = "ad_clip_norm";
  if (count < 0 || count > (1 << 20)) return fail("%s: %lld arrays (at most 2^20)", who, (long long)count);
  if (count && (!in || !out || !counts || !dtypes)) return fail("%s: null operand", who);
  if (!(max_norm >= 0.0)) return fail("%s: max_norm %g", who, max_norm);
  size_t need = 0;
  if (ad_clip_norm_workspace(count, &need)) return 1;
  if (!norm || !aligned(norm, 4)) return fail("%s: norm is null or not aligned", who);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < need)
    return fail("%s: needs %zu bytes of workspace, 256-byte aligned", who, need);
  try {
    struct Range {
      uintptr_t from, to;
      bool written;
    };
    std::vector<int> which;
    std::vector<Range> ranges;
    which.reserve(count);
    ranges.reserve(2 * count + 2);
    for (int64_t i = 0; i < count; ++i) {
      if (dtypes[i] < AD_F32 || dtypes[i] > AD_F16) return fail("%s: unknown element type %d", who, dtypes[i]);
      if (counts[i] < 0 || counts[i] > MAX_ELEMENTS) return fail("%s: %lld elements", who, (long long)counts[i]);
      if (!counts[i]) continue;
      const int es = elem_size(dtypes[i]);
      if (!in[i] || !out[i]) return fail("%s: null operand", who);
      if (!aligned({in[i], out[i]}, es)) return fail("%s: an operand is not aligned to its elements", who);
      which.push_back(static_cast<int>(i));
      const uintptr_t p = reinterpret_cast<uintptr_t>(in[i]), q = reinterpret_cast<uintptr_t>(out[i]), n = counts[i] * es;
      ranges.push_back({q, q + n, true});
      if (p != q) ranges.push_back({p, p + n, false});
    }
    const uintptr_t w = reinterpret_cast<uintptr_t>(workspace), s = reinterpret_cast<uintptr_t>(norm);
    ranges.push_back({w, w + need, true});
    ranges.push_back({s, s + 4, true});
    // what is written overlaps nothing else: an array that came twice would be scaled twice
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;  // ends so far
    for (const Range& r : ranges) {
      if (r.from < written || (r.written && r.from < any)) return fail("%s: results overlap operands or one another", who);
      any = std::max(any, r.to);
      if (r.written) written = std::max(written, r.to);
    }
    DeviceGuard guard(device);
    if (guard.error() != cudaSuccess) return fail_cuda(who, guard.error());
    const int sms = sm_count(guard.device());
    if (!sms) return fail("%s: no device properties", who);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* parts = static_cast<double*>(workspace);
    return which.size() <= SMALL ? run<SMALL>(who, which, in, out, counts, dtypes, max_norm, norm, parts, sms, st)
                                 : run<LARGE>(who, which, in, out, counts, dtypes, max_norm, norm, parts, sms, st);
  } catch (...) {
    return fail("%s: out of host memory", who);
  }
}
