// rr_encoder_device.h — device helpers of the embedding encoder's operators (rr_encoder_*.hip): element types, unaligned
// vector loads, sums and maxima over a wave or a workgroup, the 8-bit row rule.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "rr_device.h"
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

// A launch's workgroups of so many threads: one for each piece of work up to 2^22 and below 2^32 threads in all, which is what a
// grid holds; they loop over the rest.
inline dim3 grid_of(int64_t pieces, int threads) {
  const int64_t hold = ((int64_t(1) << 32) - 1) / threads, most = hold < (1 << 22) ? hold : 1 << 22;
  return dim3((unsigned)(pieces < most ? pieces : most));
}

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
// The same past the caches (non-temporal): for results that are too many to be found there when they are read.
template <class V>
__device__ __forceinline__ void store_past(void* p, V v) {
  typedef V any __attribute__((aligned(1)));
  __builtin_nontemporal_store(v, static_cast<any*>(p));
}
constexpr int64_t kCacheBytes = 32 << 20;   // eight XCDs' L2 of 4 MiB

// Sums and maxima over the W waves of a row, every lane gets them. `red`: LDS words, 2 W for each row of the workgroup, used
// in turn (the first half, the second, ...): one barrier a call, since a half is written again only after a barrier that
// follows its last reads. A short row (W = 1) may have G lanes of a wave only, aligned.
template <int W, int G = 64>
struct RowReduce {
  static_assert(W == 1 || G == 64, "whole waves");
  float* red;
  int turn = 0;
  __device__ __forceinline__ float sum(float v) {
    if constexpr (G < 64) {
      v = dpp_add_f32<0xB1>(v);                         // quad_perm [1,0,3,2]
      v = dpp_add_f32<0x4E>(v);                         // quad_perm [2,3,0,1]
      v = dpp_add_f32<0x141>(v);                        // row_half_mirror
      if constexpr (G >= 16) v = dpp_add_f32<0x140>(v); // row_mirror
      if constexpr (G >= 32) v += __shfl_xor(v, 16);
      return v;
    }
    v = wave_sum_f32(v);
    if constexpr (W == 1) return v;
    float* r = put(v);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += r[i];
    return s;
  }
  __device__ __forceinline__ unsigned max(unsigned v) {
    if constexpr (G < 64) {
      v = group_max_u32<(G < 16 ? G : 16)>(v);
      if constexpr (G >= 32) {
        const unsigned t = __shfl_xor(v, 16);
        v = v > t ? v : t;
      }
      return v;
    }
    v = wave_max_u32(v);
    if constexpr (W == 1) return v;
    float* r = put(__uint_as_float(v));
    unsigned s = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const unsigned t = __float_as_uint(r[i]);
      s = s > t ? s : t;
    }
    return s;
  }

 private:
  __device__ __forceinline__ float* put(float v) {
    float* r = red + turn * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x / 64 % W] = v;
    __syncthreads();
    return r;
  }
};

// 16 bytes of a row in registers: N values of type E, of which those at and behind `left` are not read (zeros) or written.
template <class E>
struct Chunk {
  static constexpr int N = 16 / sizeof(E);
  u32x4 raw;
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(E) == 4) return __uint_as_float(raw[i]);
    const unsigned h = i % 2 ? raw[i / 2] >> 16 : raw[i / 2] & 0xffffu;
    if constexpr (std::is_same<E, __bf16>::value) return __uint_as_float(h << 16);
    else return (float)__builtin_bit_cast(_Float16, (unsigned short)h);
  }
  __device__ __forceinline__ void load(const E* p, int left) {
    if (left >= N) {
      raw = load_as<u32x4>(p);
    } else {
      E v[N] = {};
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < left) v[i] = p[i];
      __builtin_memcpy(&raw, v, 16);
    }
  }
  __device__ __forceinline__ void fill(float x) {
    E v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (E)x;
    __builtin_memcpy(&raw, v, 16);
  }
};
template <class E>
__device__ __forceinline__ void store_chunk(E* p, const float* v, int left, bool past) {
  constexpr int N = 16 / sizeof(E);
  E o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = (E)v[i];
  if (left >= N) {
    u32x4 raw;
    __builtin_memcpy(&raw, o, 16);
    if (past) store_past(p, raw);
    else store_as(p, raw);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = o[i];
  }
}

// The 8-bit row rule: scale = max|x| times the fp32 neighbour of 1/127. (One multiplication, as torch divides a GPU tensor by 127. An
// IEEE quotient, which the index's int8 copies take, is another number in the last bit in one row of twenty.) The row's largest
// magnitude travels as its bit pattern: patterns of |x| order as their values do, infinities above every finite value and NaNs above
// those.
__device__ __forceinline__ unsigned mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float row_scale(unsigned m) {
  return m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(m) * (1.0f / 127.0f);
}
// the divisor that goes with it: rows of zeros, of non-finite values and of a scale that underflows give q = 0
__device__ __forceinline__ float row_divisor(float scale) { return scale > 0.f ? scale : __uint_as_float(0x7f800000u); }
__device__ __forceinline__ int to_i8(float v, float divisor) {
  const float t = fminf(fmaxf(rintf(v / divisor), -127.0f), 127.0f);
  return (int)t;
}
// N values to N bytes; values at and behind `left` are not written
template <int N>
__device__ __forceinline__ void store_i8(int8_t* p, const float* v, float divisor, int left) {
  unsigned o[N / 4];
#pragma unroll
  for (int w = 0; w < N / 4; ++w) {
    o[w] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[w] |= (unsigned)(to_i8(v[4 * w + i], divisor) & 255) << (8 * i);
  }
  if (left >= N) {
    __builtin_memcpy(p, o, N);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = (int8_t)(o[i / 4] >> (8 * (i % 4)));
  }
}

}  // namespace enc
}  // namespace rr
