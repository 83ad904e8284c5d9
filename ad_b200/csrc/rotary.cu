// Rotary positions of queries and keys: ad_rotary.
//
// Each head's first `rotary` elements form rotary / 2 pairs (u, v); pair i of a
// token at position p becomes (u c - v s, v c + u s) with c = cos[p][i] and
// s = sin[p][i] (s negated for the inverse, which is also the gradient).  Pairs
// are (x[i], x[i + rotary/2]) in the half layout and (x[2i], x[2i+1]) in the
// interleaved one; the rest of the head is copied.
//
// Bound by memory: three operations a value.  One block takes one token, its
// threads the vectors of a head (x) and the heads (y), so that a thread reads
// its cosines and sines once and keeps them for all its heads.
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
  long long tokens;
  int dim, half;
  float sign;
};

// V: elements a load moves; 1 where sizes or addresses allow no more.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  const long long row = blockIdx.x;
  const long long b = row / a.tokens, t = row - b * a.tokens;
  const long long at = b * a.pos_seq + t * a.pos_tok;
  const long long p =
      a.pos64 ? static_cast<const long long*>(a.positions)[at] : static_cast<const int*>(a.positions)[at];
  const bool known = p >= 0 && p < a.table_rows;
  const float nan = __int_as_float(0x7fffffff);
  // Units of a head: pair units first, then units of copied elements.
  constexpr int PV = HALF ? V : (V > 1 ? V / 2 : 1);  // pairs of a unit
  const int pair_units = a.half / PV;
  const int units = pair_units + (a.dim - 2 * a.half) / V;
  const int heads = a.heads[0] + a.heads[1];
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    const bool turned = u < pair_units;
    float c[PV], s[PV];
    if (turned) {
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        c[j] = known ? a.cos[p * a.half + u * PV + j] : nan;
        s[j] = known ? a.sign * a.sin[p * a.half + u * PV + j] : nan;
      }
    }
    for (int h = threadIdx.y; h < heads; h += blockDim.y) {
      const int w = h >= a.heads[0];
      const int hh = w ? h - a.heads[0] : h;
      const T* x = static_cast<const T*>(a.in[w]) + b * a.is[w][0] + t * a.is[w][1] + hh * a.is[w][2];
      T* y = static_cast<T*>(a.out[w]) + b * a.os[w][0] + t * a.os[w][1] + hh * a.os[w][2];
      if (!turned) {
        const int i = 2 * a.half + (u - pair_units) * V;
        store_vec<T, V>(y + i, load_vec<T, V>(x + i));
      } else if (HALF || V == 1) {
        const int i = HALF ? u * V : 2 * u, k = HALF ? i + a.half : i + 1;
        const Vec<T, V> xu = load_vec<T, V>(x + i), xv = load_vec<T, V>(x + k);
        Vec<T, V> yu, yv;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float fu = to_float(xu.v[j]), fv = to_float(xv.v[j]);
          yu.v[j] = from_float<T>(fu * c[j] - fv * s[j]);
          yv.v[j] = from_float<T>(fv * c[j] + fu * s[j]);
        }
        store_vec<T, V>(y + i, yu);
        store_vec<T, V>(y + k, yv);
      } else {
        const Vec<T, V> xx = load_vec<T, V>(x + u * V);
        Vec<T, V> yy;
#pragma unroll
        for (int j = 0; j < PV; ++j) {
          const float fu = to_float(xx.v[(2 * j) % V]), fv = to_float(xx.v[(2 * j + 1) % V]);
          yy.v[(2 * j) % V] = from_float<T>(fu * c[j] - fv * s[j]);
          yy.v[(2 * j + 1) % V] = from_float<T>(fv * c[j] + fu * s[j]);
        }
        store_vec<T, V>(y + u * V, yy);
      }
    }
  }
}

template <typename T, int V>
cudaError_t launch(const RotaryArgs& a, int layout, long long rows, cudaStream_t s) {
  const int pv = layout == 0 ? V : (V > 1 ? V / 2 : 1);
  const int units = a.half / pv + (a.dim - 2 * a.half) / V;
  const int bx = units < 256 ? units : 256;
  const int heads = a.heads[0] + a.heads[1];
  int by = 256 / bx;
  if (by > heads) by = heads;
  const dim3 block(bx, by);
  if (layout == 0)
    rotary_kernel<T, V, true><<<static_cast<unsigned>(rows), block, 0, s>>>(a);
  else
    rotary_kernel<T, V, false><<<static_cast<unsigned>(rows), block, 0, s>>>(a);
  return cudaGetLastError();
}

// Whether every vector of V elements that the kernel moves is aligned.
bool fits(const RotaryArgs& a, int layout, int v, int size) {
  if (layout == 0 ? a.half % v : (2 * a.half) % v) return false;
  if (a.dim % v) return false;
  for (int w = 0; w < 2; ++w) {
    if (!a.heads[w]) continue;
    if (!aligned(a.in[w], v * size) || !aligned(a.out[w], v * size)) return false;
    for (int d = 0; d < 3; ++d)
      if (a.is[w][d] % v || a.os[w][d] % v) return false;
  }
  return true;
}

template <typename T>
cudaError_t dispatch(const RotaryArgs& a, int layout, long long rows, cudaStream_t s) {
  constexpr int S = sizeof(T), M = 16 / S;
  if (fits(a, layout, M, S)) return launch<T, M>(a, layout, rows, s);
  if (fits(a, layout, M / 2, S)) return launch<T, M / 2>(a, layout, rows, s);
  return launch<T, 1>(a, layout, rows, s);
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
      (k_heads && (!k || !k_out || !k_strides || !k_out_strides)) || !positions || (rotary && (!cos || !sin)))
    return fail("ad_rotary: null operand");
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
  a.tokens = tokens;
  a.dim = dim;
  a.half = rotary / 2;
  a.sign = inverse ? -1.0f : 1.0f;
  DeviceGuard g(device);
  if (g.error() != cudaSuccess) return fail("ad_rotary: %s", cudaGetErrorString(g.error()));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == AD_F32    ? dispatch<float>(a, layout, rows, s)
                        : dtype == AD_BF16 ? dispatch<__nv_bfloat16>(a, layout, rows, s)
                                           : dispatch<__half>(a, layout, rows, s);
  if (e != cudaSuccess) return fail("ad_rotary: %s", cudaGetErrorString(e));
  return 0;
}
