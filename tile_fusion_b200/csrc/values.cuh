// The dense operators' value types: fp32, bf16 and fp16 in memory, fp32 in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "tile_fusion_b200.h"

namespace tfk {

constexpr int kMaxRows = 0x7f000000;  // of rows, columns and classes: an index and a grid's step beyond it stay below 2^31
__host__ __device__ constexpr int value_bytes(int dtype) { return dtype == TF_F32 ? 4 : 2; }
__host__ __device__ constexpr bool known_dtype(int dtype) { return dtype == TF_F32 || dtype == TF_BF16 || dtype == TF_F16; }

// Polls of a bounded wait (tf_dense_set_wait_limit), and after one has run out, for copies and products under way that take microseconds.
int dense_wait_limit();
constexpr int kInFlightPolls = 1 << 16;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Element i of an array whose type is known at run time only.
__device__ __forceinline__ float load_value(const void *p, int dtype, long long i) {
  if (dtype == TF_F32) return __ldg(static_cast<const float *>(p) + i);
  const unsigned short b = __ldg(static_cast<const unsigned short *>(p) + i);
  return dtype == TF_BF16 ? __uint_as_float((unsigned)b << 16) : __half2float(__ushort_as_half(b));
}
__device__ __forceinline__ void store_value(void *p, int dtype, long long i, float v) {
  if (dtype == TF_F32) static_cast<float *>(p)[i] = v;
  else if (dtype == TF_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half *>(p)[i] = __float2half_rn(v);
}
// Two values as the 16-bit pair that tensor memory copies and tensor cores read, the first in the low half.
__device__ __forceinline__ unsigned pack_pair(float a, float b, bool f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&h);
}

// N consecutive values (N a power of two, the address a multiple of their size) in one access.
template <class T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };
template <class T, int N> __device__ __forceinline__ void store_pack(T *p, const float (&v)[N]) {
  Pack<T, N> a;
#pragma unroll
  for (int i = 0; i < N; ++i) a.v[i] = from_float<T>(v[i]);
  *reinterpret_cast<Pack<T, N> *>(p) = a;
}

// As they lie in memory, up to 32 bytes at a time.
template <class T, int N> __device__ __forceinline__ Pack<T, N> load_raw(const T *p) {
  if constexpr (sizeof(T) * N == 32) {
    Pack<T, N> a;
    unsigned *u = reinterpret_cast<unsigned *>(&a);
    asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]) : "l"(p));
    return a;
  } else return *reinterpret_cast<const Pack<T, N> *>(p);
}
template <class T, int N> __device__ __forceinline__ void store_raw(T *p, const Pack<T, N> &a) {
  if constexpr (sizeof(T) * N == 32) {
    const unsigned *u = reinterpret_cast<const unsigned *>(&a);
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
                 "r"(u[6]), "r"(u[7]) : "memory");
  } else *reinterpret_cast<Pack<T, N> *>(p) = a;
}
// The largest of |a|, |b|, |c|, or a NaN if one of them is; and of a, b, c.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The largest of |a|, |b|, |c| that are numbers.
__device__ __forceinline__ float max3_abs_numbers(float a, float b, float c) {
  float d;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace tfk
