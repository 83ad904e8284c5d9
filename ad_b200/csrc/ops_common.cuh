// What the language-model operators share: element types, vector loads and
// stores, warp reductions, and the checks of their C entry points.
#ifndef AD_B200_OPS_COMMON_CUH
#define AD_B200_OPS_COMMON_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <type_traits>

#include "../../include/ad_b200.h"

namespace ad_b200_internal {
// runtime.cu:
void set_error(const char* msg);  // the message ad_last_error() returns
// TMA descriptor of `count` row-major matrices of 16-bit elements stacked in
// memory (row stride `ld` elements), swizzled over 64 or 128 bytes, boxes of one
// matrix's rows; what lies outside a matrix reads as zero.  0, or 1 with an error set.
int tmap_3d_16(const void* base, uint64_t count, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows,
               uint32_t box_cols, int swizzle_bytes, void* out128);
}

namespace adops {

inline int fail(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  ad_b200_internal::set_error(buf);
  return 1;
}

// The same for an error of the CUDA runtime, which remembers it for the thread's
// next call that asks: it is forgotten here, having been reported.
inline int fail_cuda(const char* who, cudaError_t e) {
  cudaGetLastError();
  return fail("%s: %s", who, cudaGetErrorString(e));
}

// A launch's own status: the last error may be an earlier call's.
template <auto KERNEL, typename A>
cudaError_t launch(dim3 grid, dim3 block, int bytes, cudaStream_t s, const A& a) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = bytes;
  c.stream = s;
  return cudaLaunchKernelEx(&c, KERNEL, a);
}

// Makes `device` current for one call (-1: the current one) and puts the
// caller's device back at its end.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    err_ = cudaGetDevice(&prev_);
    dev_ = device < 0 ? prev_ : device;
    if (err_ == cudaSuccess && dev_ != prev_) {
      err_ = cudaSetDevice(dev_);
      moved_ = err_ == cudaSuccess;
    }
  }
  ~DeviceGuard() {
    if (moved_) cudaSetDevice(prev_);
  }
  cudaError_t error() const { return err_; }
  int device() const { return dev_; }

 private:
  int prev_ = 0, dev_ = 0;
  bool moved_ = false;
  cudaError_t err_ = cudaSuccess;
};

// Multiprocessors of a device, asked for once; 0 with an error set on failure.
inline int sm_count(int device) {
  static std::atomic<int> known[64];
  if (device >= 0 && device < 64 && known[device]) return known[device];
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    cudaGetLastError();  // reported by the caller
    return 0;
  }
  if (device >= 0 && device < 64) known[device] = n;
  return n;
}

// Dynamic shared memory that a block of KERNEL can have on the current device.  It
// is allowed to the kernel once and for good: set to what each launch asks for, the
// limit could be lowered by another thread's launch before this one's.
template <auto KERNEL>
cudaError_t shared_room(int* room) {
  static std::atomic<int> known[64];
  int device = 0, most = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device < 64 && (*room = known[device])) return cudaSuccess;
  cudaFuncAttributes f;
  e = cudaFuncGetAttributes(&f, KERNEL);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
  if (e != cudaSuccess) return e;
  *room = most - static_cast<int>(f.sharedSizeBytes);
  e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, *room);
  if (e == cudaSuccess && device < 64) known[device] = *room;
  return e;
}

inline int elem_size(int dtype) { return dtype == AD_F32 ? 4 : 2; }
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// A load or store of an element elsewhere would be a fault of the device.
inline bool aligned(std::initializer_list<const void*> all, size_t n) {
  for (const void* p : all)
    if (!aligned(p, n)) return false;
  return true;
}

// ---------------------------------------------------------------- elements
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// V elements moved by one load or store (V * sizeof(T) <= 16 bytes).
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};
// One instruction each: a copy of 16-bit elements as a structure can fall apart
// into single ones (rotary positions of 16-bit heads ran at half their speed).
template <int BYTES>
struct Word;
template <>
struct Word<2> { typedef unsigned short type; };
template <>
struct Word<4> { typedef unsigned type; };
template <>
struct Word<8> { typedef uint2 type; };
template <>
struct Word<16> { typedef uint4 type; };
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  typedef typename Word<sizeof(T) * V>::type W;
  const W w = *reinterpret_cast<const W*>(p);
  Vec<T, V> x;
  memcpy(&x, &w, sizeof(w));
  return x;
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& x) {
  typedef typename Word<sizeof(T) * V>::type W;
  W w;
  memcpy(&w, &x, sizeof(w));
  *reinterpret_cast<W*>(p) = w;
}

// The elements of 16 bytes as floats: an instruction each (two for a pair of
// halves); taken out of a structure of 16-bit elements they cost two.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float* o) {
  const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      o[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      o[2 * i] = f.x;
      o[2 * i + 1] = f.y;
    } else {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// V values rounded to elements, two by one instruction where there are two.
template <typename T, int V>
__device__ __forceinline__ void round_to(const float* x, Vec<T, V>& y) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      unsigned w;
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x[j], x[j + 1]);
        memcpy(&w, &h, 4);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[j], x[j + 1]);
        memcpy(&w, &h, 4);
      }
      memcpy(&y.v[j], &w, 4);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) y.v[j] = from_float<T>(x[j]);
  }
}

// Element i of an array whose type (AD_F32, AD_BF16, AD_F16) is known at run
// time only: parameters that are read a few times a block.
__device__ __forceinline__ float load_any(const void* p, int dtype, long long i) {
  if (dtype == AD_F32) return static_cast<const float*>(p)[i];
  if (dtype == AD_BF16) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, long long i, float x) {
  if (dtype == AD_F32)
    static_cast<float*>(p)[i] = x;
  else if (dtype == AD_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(x);
  else
    static_cast<__half*>(p)[i] = from_float<__half>(x);
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

}  // namespace adops

#endif
