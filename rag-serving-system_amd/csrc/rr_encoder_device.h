// rr_encoder_device.h — device helpers of the embedding encoder's operators (rr_encoder_*.hip): element types, unaligned
// vector loads, sums and maxima over a wave or a workgroup, the 8-bit row rule.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "rr_encoder.h"

namespace rr {
namespace enc {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int TY> struct Elem;
template <> struct Elem<T_F32> { using type = float; };
template <> struct Elem<T_BF16> { using type = __bf16; };
template <> struct Elem<T_F16> { using type = _Float16; };

// A launch's workgroups: one for each piece of work up to 2^22 (a grid holds below 2^32 threads); they loop over the rest.
inline dim3 grid_of(int64_t pieces) { return dim3((unsigned)(pieces < (1 << 22) ? pieces : 1 << 22)); }

// N elements from an address that is aligned to one element only (one vector load: the hardware takes such addresses).
template <class V>
__device__ __forceinline__ V load_as(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <class V>
__device__ __forceinline__ void store_as(void* p, V v) {
  __builtin_memcpy(p, &v, sizeof(V));
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const unsigned t = __shfl_xor(v, o);
    v = v > t ? v : t;
  }
  return v;
}
// over a workgroup of W waves; `red` W words of LDS, free again after the call's last barrier
template <int W>
__device__ __forceinline__ float group_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (W == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) s += red[i];
  return s;
}
template <int W>
__device__ __forceinline__ unsigned group_max(unsigned v, float* red) {
  v = wave_max(v);
  if constexpr (W == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __uint_as_float(v);
  __syncthreads();
  unsigned s = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const unsigned t = __float_as_uint(red[i]);
    s = s > t ? s : t;
  }
  return s;
}

// The 8-bit row rule. The row's largest magnitude travels as its bit pattern: patterns of |x| order as their values do,
// infinities above every finite value and NaNs above those.
__device__ __forceinline__ unsigned mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float row_scale(unsigned m) {
  return m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(m) / 127.0f;
}
// the divisor that goes with it: rows of zeros, of non-finite values and of a scale that underflows give q = 0
__device__ __forceinline__ float row_divisor(float scale) { return scale > 0.f ? scale : __uint_as_float(0x7f800000u); }
__device__ __forceinline__ int to_i8(float v, float divisor) {
  const float t = fminf(fmaxf(rintf(v / divisor), -127.0f), 127.0f);
  return (int)t;
}

}  // namespace enc
}  // namespace rr
