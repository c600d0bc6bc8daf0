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
constexpr float kLog2e = 1.4426950408889634f;

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
// 2^x and 1 / x to two steps, denormals as 0
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float inverse(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two values in one instruction
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 lo(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 exp2_fast(float2 x) { return make_float2(exp2_fast(x.x), exp2_fast(x.y)); }
__device__ __forceinline__ float2 inverse2(float2 x) { return make_float2(inverse(x.x), inverse(x.y)); }
// z * sigmoid(z), and sigmoid(z)  (beyond the range of e^-z it is 0, the limit)
__device__ __forceinline__ float2 gate2(float2 z, float2 &sig) {
  sig = inverse2(add2(exp2_fast(mul2(z, both(-kLog2e))), both(1.f)));
  return mul2(z, sig);
}
__device__ __forceinline__ float sigmoid(float x) { return inverse(1.f + exp2_fast(x * -kLog2e)); }
__device__ __forceinline__ int sequence_length(const int32_t *lengths, long long b, int time) {
  return lengths == nullptr ? time : min(max(lengths[b], 0), time);
}

__device__ __forceinline__ bool aligned_16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
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
