// What the operators for sequence models share: activations of three types read and written four channels at a time, the
// caller's device put back, messages, and the checks of their arguments.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdio.h>

#include <type_traits>

#include "common.cuh"

namespace myea {

constexpr uint64_t kSequenceMost = uint64_t(1) << 30;   // of any one dimension
constexpr int kSms = 148;

inline int refuse(char *dst, size_t cap, int code, const char *msg) {
  if (dst != nullptr && cap > 0) snprintf(dst, cap, "%s", msg);
  return code;
}
inline int launched(char *dst, size_t cap, const char *what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return MYEA_OK;
  if (dst != nullptr && cap > 0) snprintf(dst, cap, "%s: %s", what, cudaGetErrorString(e));
  return MYEA_E_CUDA;
}

// makes `device` current for the call and puts the caller's device back
struct DeviceScope {
  int previous = -1;
  bool ok = false;
  explicit DeviceScope(int device) {
    int now = -1;
    if (device < 0 || cudaGetDevice(&now) != cudaSuccess) return;
    if (now != device) {
      if (cudaSetDevice(device) != cudaSuccess) return;
      previous = now;
    }
    ok = true;
  }
  ~DeviceScope() { if (previous >= 0) cudaSetDevice(previous); }
};

inline size_t type_bytes(uint32_t type) { return type == MYEA_TYPE_F32 ? 4 : 2; }
inline bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }
// whether four channels at a time can be accessed as one word of 4 * type_bytes
inline bool view_takes_vectors(const myea_view &v, uint32_t type) {
  return aligned(v.data, 4 * type_bytes(type)) && v.stride_batch % 4 == 0 && v.stride_time % 4 == 0;
}
inline size_t round_up_256(size_t n) { return (n + 255) / 256 * 256; }

#ifdef __CUDACC__
// four neighbouring elements as they lie in memory
template <typename T> struct Raw4 { uint2 v; };
template <> struct Raw4<float> { float4 v; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ float4 widen(const Raw4<float> &r) { return r.v; }
__device__ __forceinline__ float4 widen(const Raw4<__nv_bfloat16> &r) {   // the upper half of a float
  return make_float4(__uint_as_float(r.v.x << 16), __uint_as_float(r.v.x & 0xffff0000u), __uint_as_float(r.v.y << 16), __uint_as_float(r.v.y & 0xffff0000u));
}
__device__ __forceinline__ float4 widen(const Raw4<__half> &r) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&r.v.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&r.v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ Raw4<float> narrow(float4 x, float) { return {x}; }
__device__ __forceinline__ Raw4<__nv_bfloat16> narrow(float4 x, __nv_bfloat16) {
  Raw4<__nv_bfloat16> r;
  const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
  r.v = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
  return r;
}
__device__ __forceinline__ Raw4<__half> narrow(float4 x, __half) {
  Raw4<__half> r;
  const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
  r.v = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
  return r;
}
template <typename T> __device__ __forceinline__ Raw4<T> zero4() {
  Raw4<T> r;
  r.v = {};
  return r;
}
// the first n (0..4) of four elements at p, the others 0; vec: p is aligned to four of them
template <typename T> __device__ __forceinline__ Raw4<T> load4(const T *p, int n, bool vec) {
  Raw4<T> r = zero4<T>();
  if (vec && n >= 4) {
    r = *reinterpret_cast<const Raw4<T> *>(p);
  } else {
    T *e = reinterpret_cast<T *>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) e[i] = p[i];
  }
  return r;
}
template <typename T> __device__ __forceinline__ void store4(T *p, float4 x, int n, bool vec) {
  const Raw4<T> r = narrow(x, T());
  if (vec && n >= 4) {
    *reinterpret_cast<Raw4<T> *>(p) = r;
  } else {
    const T *e = reinterpret_cast<const T *>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = e[i];
  }
}
// the same for parameters, whose arrays may lie anywhere
__device__ __forceinline__ float4 parameters4(const float *p, int n, float none = 0.f) {
  float4 r = make_float4(none, none, none, none);
  if (p != nullptr) {
    if (n > 0) r.x = p[0];
    if (n > 1) r.y = p[1];
    if (n > 2) r.z = p[2];
    if (n > 3) r.w = p[3];
  }
  return r;
}
// (a denominator beyond 2^126 divides to 0, which is the limit)
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
__device__ __forceinline__ int sequence_length(const int32_t *lengths, long long b, int time) {
  return lengths == nullptr ? time : min(max(lengths[b], 0), time);
}

__device__ __forceinline__ bool aligned_16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// over all threads of a block of at most 512, in a fixed order; memory: 17 floats that nothing else uses meanwhile
__device__ __forceinline__ float block_sum(float x, float *memory) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) memory[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0.f;
  for (int k = 0; k < static_cast<int>(blockDim.x >> 5); ++k) x += memory[k];
  return x;
}
__device__ __forceinline__ float block_max(float x, float *memory) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) memory[threadIdx.x >> 5] = x;
  __syncthreads();
  x = memory[0];
  for (int k = 1; k < static_cast<int>(blockDim.x >> 5); ++k) x = fmaxf(x, memory[k]);
  return x;
}

// store(column, sum over rows of part[row][column]): partial sums of blocks that ran side by side, 32 columns and 8 strands of
// rows per block of 256 threads, the strands joined in their order
template <typename Store>
__device__ __forceinline__ void sum_partials_block(const float *part, long long rows, long long columns, long long block, Store store) {
  __shared__ float strand[8][32];
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5;
  const long long c = block * 32 + lane;
  float sum = 0.f;
  if (c < columns) {
    long long r = s;
    for (; r + 24 < rows; r += 32) {   // four loads in flight
      const float a = part[r * columns + c], b = part[(r + 8) * columns + c], d = part[(r + 16) * columns + c], e = part[(r + 24) * columns + c];
      sum += (a + b) + (d + e);
    }
    for (; r < rows; r += 8) sum += part[r * columns + c];
  }
  strand[s][lane] = sum;
  __syncthreads();
  if (s == 0 && c < columns) {
#pragma unroll
    for (int k = 1; k < 8; ++k) sum += strand[k][lane];
    store(c, sum);
  }
}
#endif

// f(value of the C++ type that a MYEA_TYPE_* stands for)
template <typename F> inline void with_type(uint32_t type, F f) {
  if (type == MYEA_TYPE_F32) f(float());
  else if (type == MYEA_TYPE_BF16) f(__nv_bfloat16());
  else f(__half());
}

}  // namespace myea
