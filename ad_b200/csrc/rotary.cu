// Rotary positions of queries and keys: ad_rotary.
//
// Each head's first `rotary` elements form rotary / 2 pairs (u, v); pair i of a
// token at position p becomes (u c - v s, v c + u s) with c = cos[p][i] and
// s = sin[p][i] (s negated for the inverse, which is also the gradient).  Pairs
// are (x[i], x[i + rotary/2]) in the half layout and (x[2i], x[2i+1]) in the
// interleaved one; the rest of the head is copied.
//
// Bound by memory: three operations a value.  A thread takes the same vector of
// several heads of one token, so that it reads its cosines and sines once and
// keeps them for all of these heads; the heads' loads are in flight before the
// token's position and its row of the tables are asked for.
//
// Measured: 16288 tokens x 32 heads x 64 fp32 45.2 us (5.9 TB/s); 65536 tokens x
// 40 heads x 128 bf16, half of each head turned in pairs, 264 us (5.1 TB/s);
// all of it in the half layout 250 us, and 438 us with 62 elements turned, whose
// halves of 31 make each partner a load of one element from shared memory.
#include <algorithm>

#include "ops_common.cuh"

namespace {

using namespace adops;

struct RotaryArgs {
  const void* in[2];
  void* out[2];
  long long is[2][3], os[2][3];  // strides in elements: sequence, token, head
  int heads[2];
  const float* cos;
  const float* sin;
  const void* positions;
  long long pos_seq, pos_tok;
  int pos64;
  long long table_rows;
  long long rows, tokens;  // sequences x tokens, tokens
  int dim, half;
  int table_vec;         // rows of the tables are whole 16-byte vectors
  unsigned head_groups;  // a thread takes every so-many-th head
  float sign;
};

// A group of threads, one for each unit of a head, works on a token's every
// so-many-th head; a block has as many groups as 256 threads make.
// HALVES: a unit is two vectors, one from each half of the rotated part, whose
//   halves are whole vectors, or two of what is copied.
// PAIRS: a unit is a vector; interleaved pairs lie within it.
// ACROSS: a unit is a vector of the half layout whose halves are not whole
//   vectors; the group puts its heads into shared memory, where each thread
//   finds its elements' partners.
enum Units { HALVES, PAIRS, ACROSS };

// Heads whose loads a thread has in flight together: four vectors, or what fits
// the registers of 1024 threads a multiprocessor.
template <Units U>
__host__ __device__ constexpr int heads_at_once() {
  return U == HALVES ? 2 : 4;
}

template <typename T, int V, Units U>
__global__ void __launch_bounds__(256, U == HALVES ? 4 : 5) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int N = heads_at_once<U>();
  constexpr int C = U == PAIRS ? V / 2 : V;
  const unsigned group = blockIdx.x * blockDim.y + threadIdx.y;
  const unsigned row = group / a.head_groups, h0 = group - row * a.head_groups;
  const bool here = row < static_cast<unsigned>(a.rows);
  const unsigned tokens = static_cast<unsigned>(a.tokens), seq = here ? row / tokens : 0;
  const long long b = seq, t = here ? row - seq * tokens : 0;
  const unsigned heads = a.heads[0] + a.heads[1];
  const int i = threadIdx.x * V;  // the unit's first element
  const int rot = 2 * a.half;
  const bool copies = U == HALVES ? i >= a.half : i >= rot;
  // HALVES: where the unit's two vectors start; what is copied is shared out by twos as well
  const int left = (a.dim - rot) / V, spread = (left + 1) / 2 * V;
  const int at = U == HALVES && copies ? i + a.half : i;
  const int at2 = copies ? at + spread : at + a.half;
  const bool two = U == HALVES && at2 < a.dim;
  float c[C], s[C];
  Vec<T, V> xu[N], xv[U == HALVES ? N : 1];
  extern __shared__ __align__(16) unsigned char raw[];
  T* const mine = reinterpret_cast<T*>(raw) + threadIdx.y * N * a.dim;  // ACROSS: the group's heads
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const unsigned h = h0 + n * a.head_groups;
    if (!here || h >= heads) continue;
    const int w = h >= static_cast<unsigned>(a.heads[0]);
    const T* x = static_cast<const T*>(a.in[w]) + b * a.is[w][0] + t * a.is[w][1] +
                 static_cast<long long>(w ? h - a.heads[0] : h) * a.is[w][2];
    xu[n] = load_vec<T, V>(x + at);
    if (two) xv[n] = load_vec<T, V>(x + at2);
    if (U == ACROSS) store_vec<T, V>(mine + n * a.dim + i, xu[n]);
  }
  if (here) {  // behind the heads' loads
    const long long pa = b * a.pos_seq + t * a.pos_tok;
    const long long p =
        a.pos64 ? static_cast<const long long*>(a.positions)[pa] : static_cast<const int*>(a.positions)[pa];
    const bool known = p >= 0 && p < a.table_rows;
    const long long at_row = known ? p * a.half : 0;
    const int first = U == PAIRS ? i / 2 : i;
    if (U != ACROSS && C % 4 == 0 && a.table_vec && known && first + C <= a.half) {
#pragma unroll
      for (int j = 0; j < C; j += 4) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(a.cos + at_row + first + j));
        const float4 z = __ldg(reinterpret_cast<const float4*>(a.sin + at_row + first + j));
        c[j % C] = w.x, c[(j + 1) % C] = w.y, c[(j + 2) % C] = w.z, c[(j + 3) % C] = w.w;
        s[j % C] = a.sign * z.x, s[(j + 1) % C] = a.sign * z.y, s[(j + 2) % C] = a.sign * z.z, s[(j + 3) % C] = a.sign * z.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int e = first + j;
        const int k = U == ACROSS && e >= a.half ? e - a.half : e;
        const bool turned = known && (U == ACROSS ? e < rot : e < a.half);
        c[j] = turned ? __ldg(a.cos + at_row + k) : __int_as_float(0x7fffffff);
        s[j] = turned ? a.sign * __ldg(a.sin + at_row + k) : __int_as_float(0x7fffffff);
        if (U == ACROSS && e < a.half) s[j] = -s[j];
      }
    }
  }
  if (U == ACROSS) __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const unsigned h = h0 + n * a.head_groups;
    if (!here || h >= heads) continue;
    const int w = h >= static_cast<unsigned>(a.heads[0]);
    T* y = static_cast<T*>(a.out[w]) + b * a.os[w][0] + t * a.os[w][1] +
           static_cast<long long>(w ? h - a.heads[0] : h) * a.os[w][2];
    if (copies) {
      store_vec<T, V>(y + at, xu[n]);
      if (two) store_vec<T, V>(y + at2, xv[n]);
    } else if (U == HALVES) {
      Vec<T, V> yu, yv;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float fu = to_float(xu[n].v[j]), fv = to_float(xv[n].v[j]);
        yu.v[j] = from_float<T>(fu * c[j] - fv * s[j]);
        yv.v[j] = from_float<T>(fv * c[j] + fu * s[j]);
      }
      store_vec<T, V>(y + at, yu);
      store_vec<T, V>(y + at2, yv);
    } else if (U == PAIRS) {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const float fu = to_float(xu[n].v[2 * j]), fv = to_float(xu[n].v[2 * j + 1]);
        if (i + 2 * j < rot) {
          xu[n].v[2 * j] = from_float<T>(fu * c[j] - fv * s[j]);
          xu[n].v[2 * j + 1] = from_float<T>(fv * c[j] + fu * s[j]);
        }
      }
      store_vec<T, V>(y + at, xu[n]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = i + j;
        if (e >= rot) break;
        const float other = to_float(mine[n * a.dim + (e < a.half ? e + a.half : e - a.half)]);
        xu[n].v[j] = from_float<T>(to_float(xu[n].v[j]) * c[j] + other * s[j]);
      }
      store_vec<T, V>(y + at, xu[n]);
    }
  }
}

// The same an element and its partner at a time, whatever the alignment; a
// block takes one token.
template <typename T, bool HALF>
__global__ void __launch_bounds__(256) rotary_single_kernel(const __grid_constant__ RotaryArgs a) {
  const long long row = blockIdx.x;
  const long long b = row / a.tokens, t = row - b * a.tokens;
  const long long pa = b * a.pos_seq + t * a.pos_tok;
  const long long p =
      a.pos64 ? static_cast<const long long*>(a.positions)[pa] : static_cast<const int*>(a.positions)[pa];
  const bool known = p >= 0 && p < a.table_rows;
  const int units = a.dim - a.half, heads = a.heads[0] + a.heads[1];  // pairs, then what is copied
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    const bool turned = u < a.half;
    const float c = turned && known ? a.cos[p * a.half + u] : __int_as_float(0x7fffffff);
    const float s = turned && known ? a.sign * a.sin[p * a.half + u] : __int_as_float(0x7fffffff);
    for (int h = threadIdx.y; h < heads; h += blockDim.y) {
      const int w = h >= a.heads[0];
      const long long hh = w ? h - a.heads[0] : h;
      const T* x = static_cast<const T*>(a.in[w]) + b * a.is[w][0] + t * a.is[w][1] + hh * a.is[w][2];
      T* y = static_cast<T*>(a.out[w]) + b * a.os[w][0] + t * a.os[w][1] + hh * a.os[w][2];
      if (!turned) {
        y[u + a.half] = x[u + a.half];
      } else {
        const int i = HALF ? u : 2 * u, k = HALF ? u + a.half : 2 * u + 1;
        const float fu = to_float(x[i]), fv = to_float(x[k]);
        y[i] = from_float<T>(fu * c - fv * s);
        y[k] = from_float<T>(fv * c + fu * s);
      }
    }
  }
}

// Whether heads start at multiples of v elements and are made of so many.
bool whole(const RotaryArgs& a, int v, int size) {
  if (a.dim % v) return false;
  for (int w = 0; w < 2; ++w) {
    if (!a.heads[w]) continue;
    if (!aligned(a.in[w], v * size) || !aligned(a.out[w], v * size)) return false;
    for (int d = 0; d < 3; ++d)
      if (a.is[w][d] % v || a.os[w][d] % v) return false;
  }
  return true;
}

template <typename T, int V, Units U>
cudaError_t start(RotaryArgs a, cudaStream_t s) {
  const int units = U == HALVES ? a.half / V + ((a.dim - 2 * a.half) / V + 1) / 2 : a.dim / V;
  const int heads = a.heads[0] + a.heads[1];
  a.head_groups = static_cast<unsigned>((heads + heads_at_once<U>() - 1) / heads_at_once<U>());
  const long long groups = a.rows * a.head_groups;
  if (groups > 0x7fffffffll) return cudaErrorInvalidValue;
  const int by = 256 / units;
  const int bytes = U == ACROSS ? by * heads_at_once<U>() * a.dim * static_cast<int>(sizeof(T)) : 0;
  return launch<rotary_kernel<T, V, U>>(static_cast<unsigned>((groups + by - 1) / by), dim3(units, by), bytes, s, a);
}

template <typename T, int V>
bool try_vectors(const RotaryArgs& a, int layout, cudaStream_t s, cudaError_t& e) {
  if (a.dim / V > 256 || !whole(a, V, sizeof(T))) return false;
  e = layout == 1          ? start<T, V, PAIRS>(a, s)
      : a.half % V == 0    ? start<T, V, HALVES>(a, s)
                           : start<T, V, ACROSS>(a, s);
  return true;
}

// 16-byte vectors where the heads allow them, else 8 bytes, else single elements.
template <typename T>
cudaError_t dispatch(const RotaryArgs& a, int layout, cudaStream_t s) {
  constexpr int M = 16 / sizeof(T);
  cudaError_t e;
  if (try_vectors<T, M>(a, layout, s, e) || try_vectors<T, M / 2>(a, layout, s, e)) return e;
  const int units = a.dim - a.half, bx = std::min(units, 256);
  const int by = std::max(1, std::min(256 / bx, a.heads[0] + a.heads[1]));
  const unsigned blocks = static_cast<unsigned>(a.rows);
  return layout == 0 ? launch<rotary_single_kernel<T, true>>(blocks, dim3(bx, by), 0, s, a)
                     : launch<rotary_single_kernel<T, false>>(blocks, dim3(bx, by), 0, s, a);
}

}  // namespace

extern "C" int ad_rotary(int device, int dtype, const void* q, const int64_t* q_strides, void* q_out,
                         const int64_t* q_out_strides, int q_heads, const void* k, const int64_t* k_strides,
                         void* k_out, const int64_t* k_out_strides, int k_heads, int64_t sequences, int64_t tokens,
                         int dim, int rotary, int layout, int inverse, const float* cos, const float* sin,
                         int64_t table_rows, const void* positions, int pos64, int64_t pos_seq_stride,
                         int64_t pos_tok_stride, void* stream) {
  if (dtype < AD_F32 || dtype > AD_F16) return fail("ad_rotary: unknown element type %d", dtype);
  if (q_heads < 0 || k_heads < 0 || sequences < 0 || tokens < 0 || dim < 0)
    return fail("ad_rotary: negative size");
  if (rotary < 0 || rotary > dim || rotary % 2) return fail("ad_rotary: %d of %d elements cannot be rotated", rotary, dim);
  if (layout != 0 && layout != 1) return fail("ad_rotary: unknown layout %d", layout);
  const long long rows = static_cast<long long>(sequences) * tokens;
  if (rows == 0 || q_heads + k_heads == 0 || dim == 0) return 0;
  if (rows > 0x7fffffffll) return fail("ad_rotary: %lld tokens in one call", rows);
  if ((q_heads && (!q || !q_out || !q_strides || !q_out_strides)) ||
      (k_heads && (!k || !k_out || !k_strides || !k_out_strides)) || !positions ||
      (rotary && table_rows > 0 && (!cos || !sin)))  // an empty table has no address; every position lies outside it
    return fail("ad_rotary: null operand");
  if (!aligned({q, q_out, k, k_out}, elem_size(dtype)) || !aligned({cos, sin}, 4) || !aligned(positions, pos64 ? 8 : 4))
    return fail("ad_rotary: an operand is not aligned to its elements");
  RotaryArgs a;
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t* is[2] = {q_strides, k_strides};
  const int64_t* os[2] = {q_out_strides, k_out_strides};
  a.heads[0] = q_heads;
  a.heads[1] = k_heads;
  for (int w = 0; w < 2; ++w) {
    a.in[w] = in[w];
    a.out[w] = out[w];
    for (int d = 0; d < 3; ++d) {
      a.is[w][d] = a.heads[w] ? is[w][d] : 0;
      a.os[w][d] = a.heads[w] ? os[w][d] : 0;
    }
  }
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.pos_seq = pos_seq_stride;
  a.pos_tok = pos_tok_stride;
  a.pos64 = pos64;
  a.table_rows = table_rows;
  a.rows = rows;
  a.tokens = tokens;
  a.dim = dim;
  a.half = rotary / 2;
  a.table_vec = a.half % 4 == 0 && aligned(cos, 16) && aligned(sin, 16);
  a.sign = inverse ? -1.0f : 1.0f;
  DeviceGuard g(device);
  if (g.error() != cudaSuccess) return fail_cuda("ad_rotary", g.error());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == AD_F32    ? dispatch<float>(a, layout, s)
                        : dtype == AD_BF16 ? dispatch<__nv_bfloat16>(a, layout, s)
                                           : dispatch<__half>(a, layout, s);
  if (e != cudaSuccess) return fail_cuda("ad_rotary", e);
  return 0;
}
