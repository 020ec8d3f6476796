// rr_encoder_norm.hip — the norms around a block, fused with its gate, residual scale and 8-bit rows (rr_block_norm).
#include "rr_encoder_device.h"

namespace rr {
namespace enc {
namespace {

// Bandwidth is all there is to it: a row is read once, stays in the registers of its W waves in fp32 (S times 16 bytes of
// its type a lane; W = 1: no barriers, and a short row has G lanes of a wave), and each result is written once. The variance is a second sum
// over the registers, of centred values. Workgroups loop over rows, so that weights and biases are loaded once each.
// 32768 x 4096 bf16, norms on both sides, 211 us: 5.1 TB/s, what a large copy reaches; 4097 x 1001 fp32 (rows at odd
// addresses) 13.0 us, 5.05 TB/s; 613 x 1024 with 8-bit rows 4.2 us, a launch and four memory and reduction latencies.
template <int TY, int W, int S, int G = 64>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void block_norm_kernel(NormArgs a) {
  using E = typename Elem<TY>::type;
  constexpr int N = Chunk<E>::N, kLanes = W == 1 ? G : 64 * W, kGroups = W == 1 ? 256 / G : 1;
  __shared__ float red[2 * W];
  RowReduce<W, G> over{red};
  const int t = threadIdx.x % kLanes, cols = a.cols;

  auto vector = [&](Chunk<E>* c, const void* p, float none) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int at = (s * kLanes + t) * N;
      if (p) c[s].load(static_cast<const E*>(p) + at, cols - at);
      else c[s].fill(none);
    }
  };
  // Weights and biases stay in registers over the rows, in their own type, where that leaves room for the rows themselves
  // (at most two chunks a lane); otherwise each row takes them from cache.
  constexpr bool kHold = S <= 2;
  Chunk<E> pw[S], pb[S], nw[S], nb[S];
  if (kHold && a.post) {
    vector(pw, a.post_w, 1.f);
    vector(pb, a.post_b, 0.f);
  }
  if (kHold && a.next) {
    vector(nw, a.next_w, 1.f);
    vector(nb, a.next_b, 0.f);
  }
  // v in place; columns behind the row's end hold zeros and are kept out of the centred sum
  auto norm = [&](float (*v)[N], int kind, Chunk<E>* w, Chunk<E>* b, const void* wp, const void* bp) {
    if constexpr (kHold) {
#pragma unroll
      for (int s = 0; s < S; ++s) asm volatile("" : "+v"(w[s].raw), "+v"(b[s].raw));   // (not widened ahead of the loop)
    } else {
      vector(w, wp, 1.f);
      vector(b, bp, 0.f);
    }
    float mean = 0.f;
    if (kind == 1) {
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < N; ++i) sum += v[s][i];
      mean = over.sum(sum) / (float)cols;
    }
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[s][i] = (s * kLanes + t) * N + i < cols ? v[s][i] - mean : 0.f;
        sum = fmaf(v[s][i], v[s][i], sum);
      }
    const float r = 1.0f / sqrtf(over.sum(sum) / (float)cols + a.eps);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < N; ++i) v[s][i] = fmaf(v[s][i] * r, w[s][i], b[s][i]);
  };

  for (int64_t r = (int64_t)blockIdx.x * kGroups + threadIdx.x / kLanes; r < a.rows; r += (int64_t)gridDim.x * kGroups) {
    Chunk<E> y[S], x[S], g[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int at = (s * kLanes + t) * N;
      y[s].load(static_cast<const E*>(a.y) + r * a.ldy + at, cols - at);
      if (a.x) x[s].load(static_cast<const E*>(a.x) + r * a.ldx + at, cols - at);
    }
    if (a.gate) vector(g, static_cast<const E*>(a.gate) + r / a.rows_per_gate * a.ldg, 1.f);
    float v[S][N];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < N; ++i) v[s][i] = y[s][i];
    if (a.post) norm(v, a.post, pw, pb, a.post_w, a.post_b);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int at = (s * kLanes + t) * N;
      if (a.gate)
#pragma unroll
        for (int i = 0; i < N; ++i) v[s][i] *= g[s][i];
      if (a.x)
#pragma unroll
        for (int i = 0; i < N; ++i) v[s][i] = fmaf(a.residual_scale, x[s][i], v[s][i]);
      if (a.stream) store_chunk(static_cast<E*>(a.stream) + r * a.lds + at, v[s], cols - at, a.past);
    }
    if (!a.next) continue;
    norm(v, a.next, nw, nb, a.next_w, a.next_b);
    if (a.normed)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int at = (s * kLanes + t) * N;
        store_chunk(static_cast<E*>(a.normed) + r * a.ldn + at, v[s], cols - at, a.past);
      }
    if (!a.q) continue;
    unsigned m = 0;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if ((s * kLanes + t) * N + i >= cols) v[s][i] = 0.f;
        m = mag(v[s][i]) > m ? mag(v[s][i]) : m;
      }
    const float sc = row_scale(over.max(m));
    const float div = row_divisor(sc);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int at = (s * kLanes + t) * N;
#pragma unroll
      for (int i = 0; i < N; ++i) v[s][i] = sc == sc ? v[s][i] : 0.f;
      store_i8<N>(a.q + r * a.ldq + at, v[s], div, cols - at);
    }
    if (t == 0) a.q_scale[r] = sc;
  }
}

template <int W>
__device__ __forceinline__ void norm_in_place(float* v, int cols, int kind, float eps, RowReduce<W>& over) {
  float mean = 0.f;
  if (kind == 1) {
    float s = 0.f;
    for (int c = threadIdx.x; c < cols; c += 64 * W) s += v[c];
    mean = over.sum(s) / (float)cols;
  }
  float s2 = 0.f;
  for (int c = threadIdx.x; c < cols; c += 64 * W) s2 += (v[c] - mean) * (v[c] - mean);
  const float r = 1.0f / sqrtf(over.sum(s2) / (float)cols + eps);
  for (int c = threadIdx.x; c < cols; c += 64 * W) v[c] = (v[c] - mean) * r;
}

// Rows that do not fit the registers: one workgroup per row, which lies in LDS in fp32 between the steps, each thread at its
// own columns, element by element. 4096 x 20000 with both norms: bf16 486 us, 1.3 TB/s; fp32 539 us, 2.4 TB/s (of the 5.2 that a
// large copy and the rows in registers reach).
template <int TY>
__global__ __launch_bounds__(1024) void block_norm_wide_kernel(NormArgs a) {
  using E = typename Elem<TY>::type;
  extern __shared__ float v[];
  __shared__ float red[32];
  RowReduce<16> over{red};
  const int cols = a.cols;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const E* y = static_cast<const E*>(a.y) + r * a.ldy;
    for (int c = threadIdx.x; c < cols; c += 1024) v[c] = (float)y[c];
    if (a.post) norm_in_place<16>(v, cols, a.post, a.eps, over);
    const E* x = a.x ? static_cast<const E*>(a.x) + r * a.ldx : nullptr;
    const E* g = a.gate ? static_cast<const E*>(a.gate) + r / a.rows_per_gate * a.ldg : nullptr;
    for (int c = threadIdx.x; c < cols; c += 1024) {
      float u = v[c];
      if (a.post_w) u *= (float)static_cast<const E*>(a.post_w)[c];
      if (a.post_b) u += (float)static_cast<const E*>(a.post_b)[c];
      if (g) u *= (float)g[c];
      if (x) u += a.residual_scale * (float)x[c];
      v[c] = u;
      if (a.stream) static_cast<E*>(a.stream)[r * a.lds + c] = (E)u;
    }
    if (!a.next) continue;
    norm_in_place<16>(v, cols, a.next, a.eps, over);
    unsigned m = 0;
    for (int c = threadIdx.x; c < cols; c += 1024) {
      float u = v[c];
      if (a.next_w) u *= (float)static_cast<const E*>(a.next_w)[c];
      if (a.next_b) u += (float)static_cast<const E*>(a.next_b)[c];
      v[c] = u;
      if (a.normed) static_cast<E*>(a.normed)[r * a.ldn + c] = (E)u;
      m = mag(u) > m ? mag(u) : m;
    }
    if (!a.q) continue;
    const float s = row_scale(over.max(m));
    const float div = row_divisor(s);
    const bool dead = !(s == s);
    for (int c = threadIdx.x; c < cols; c += 1024) a.q[r * a.ldq + c] = dead ? 0 : (int8_t)to_i8(v[c], div);
    if (threadIdx.x == 0) a.q_scale[r] = s;
  }
}

template <int TY>
hipError_t run(NormArgs a, hipStream_t s) {
  constexpr int N = Chunk<typename Elem<TY>::type>::N;
  // What a call reads and writes, beyond the caches: its results are written past them (32768 x 4096 bf16, both norms 246 us
  // with plain stores, 212 so; 4097 x 1001 fp32 14.9 and 13.0). Below that the next operator finds them in L2.
  const int64_t values = (1 + (a.x != nullptr) + (a.stream != nullptr) + (a.normed != nullptr)) * a.rows * a.cols;
  a.past = values * (int64_t)sizeof(typename Elem<TY>::type) > kCacheBytes;
  auto go = [&](auto kernel, int waves, int lanes = 64) {
    const int groups = waves == 1 ? 256 / lanes : 1;
    const int64_t wgs = (a.rows + groups - 1) / groups, most = 256 * 8;
    kernel<<<dim3((unsigned)(wgs < most ? wgs : most)), waves == 1 ? 256 : 64 * waves, 0, s>>>(a);
    return hipGetLastError();
  };
  // Lanes in proportion to the row, so that few idle (16000 x 192 bf16 with 8-bit rows: a wave a row 14.6 us, half a wave 9.8;
  // x 50 14.2, with eight lanes 5.1; 2712 x 4608 with both norms and 8-bit rows: 1024 lanes' room 50 us, 768 43)
  const int chunks = (a.cols + N - 1) / N;
  if (chunks <= 8) return go(block_norm_kernel<TY, 1, 1, 8>, 1, 8);
  if (chunks <= 16) return go(block_norm_kernel<TY, 1, 1, 16>, 1, 16);
  if (chunks <= 32) return go(block_norm_kernel<TY, 1, 1, 32>, 1, 32);
  if (chunks <= 64) return go(block_norm_kernel<TY, 1, 1>, 1);
  if (chunks <= 64 * 2) return go(block_norm_kernel<TY, 1, 2>, 1);
  if (chunks <= 64 * 3) return go(block_norm_kernel<TY, 1, 3>, 1);
  if (chunks <= 64 * 4) return go(block_norm_kernel<TY, 1, 4>, 1);
  if (chunks <= 64 * 6) return go(block_norm_kernel<TY, 3, 2>, 3);
  if (chunks <= 64 * 8) return go(block_norm_kernel<TY, 4, 2>, 4);
  if (chunks <= 64 * 12) return go(block_norm_kernel<TY, 3, 4>, 3);
  if (chunks <= 64 * 16) return go(block_norm_kernel<TY, 8, 2>, 8);
  if (chunks <= 64 * 24) return go(block_norm_kernel<TY, 12, 2>, 12);
  if (chunks <= 64 * 32) return go(block_norm_kernel<TY, 16, 2>, 16);
  const size_t lds = (size_t)a.cols * 4;
  auto wide = block_norm_wide_kernel<TY>;
  if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(wide), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds))
    return e;
  wide<<<grid_of(a.rows, 1024), 1024, lds, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_norm(int type, const NormArgs& a, hipStream_t s) {
  return type == T_F32 ? run<T_F32>(a, s) : type == T_BF16 ? run<T_BF16>(a, s) : run<T_F16>(a, s);
}

}  // namespace enc
}  // namespace rr
