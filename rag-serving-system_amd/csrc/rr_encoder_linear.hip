// rr_encoder_linear.hip — 8-bit rows and the 8-bit matrix product (rr_quantize_rows, rr_linear_i8).
#include "rr_encoder_device.h"

namespace rr {
namespace enc {
namespace {

// ---- 8-bit rows ----------------------------------------------------------------------------------------------------
// A row in the registers of W waves, S times 16 bytes a lane; W = 1: four rows a workgroup. cols_pad: columns written, zeros
// behind the row's own.
template <int TY, int W, int S>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void quantize_rows_kernel(const void* xv, int64_t ldx, int64_t rows,
                                                                             int cols, int cols_pad, int8_t* q, int64_t ldq,
                                                                             float* scale) {
  using E = typename Elem<TY>::type;
  constexpr int N = Chunk<E>::N, kGroups = W == 1 ? 4 : 1;
  __shared__ float red[2 * W];
  RowReduce<W> over{red};
  const int t = threadIdx.x % (64 * W);
  for (int64_t r = (int64_t)blockIdx.x * kGroups + threadIdx.x / (64 * W); r < rows; r += (int64_t)gridDim.x * kGroups) {
    const E* x = static_cast<const E*>(xv) + r * ldx;
    Chunk<E> c[S];
#pragma unroll
    for (int s = 0; s < S; ++s) c[s].load(x + (s * 64 * W + t) * N, cols - (s * 64 * W + t) * N);
    unsigned m = 0;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < N; ++i) m = mag(c[s][i]) > m ? mag(c[s][i]) : m;
    const float sc = row_scale(over.max(m));
    const float div = row_divisor(sc);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = sc == sc ? c[s][i] : 0.f;
      store_i8<N>(q + r * ldq + (s * 64 * W + t) * N, v, div, cols_pad - (s * 64 * W + t) * N);
    }
    if (t == 0) scale[r] = sc;
  }
}

// Rows of any length: one workgroup per row, two passes over it (the second one from cache).
template <int TY>
__global__ __launch_bounds__(256) void quantize_long_rows_kernel(const void* xv, int64_t ldx, int64_t rows, int cols,
                                                                 int cols_pad, int8_t* q, int64_t ldq, float* scale) {
  using E = typename Elem<TY>::type;
  __shared__ float red[8];
  RowReduce<4> over{red};
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const E* x = static_cast<const E*>(xv) + r * ldx;
    unsigned m = 0;
    for (int c = threadIdx.x; c < cols; c += 256) {
      const unsigned t = mag((float)x[c]);
      m = t > m ? t : m;
    }
    const float s = row_scale(over.max(m));
    const float div = row_divisor(s);
    for (int c = threadIdx.x; c < cols_pad; c += 256)
      q[r * ldq + c] = c < cols && s == s ? (int8_t)to_i8((float)x[c], div) : 0;
    if (threadIdx.x == 0) scale[r] = s;
  }
}

// ---- the product ---------------------------------------------------------------------------------------------------
// out^T = w x^T: the matrix instruction's rows are output channels and its columns rows of x, so a lane holds four
// consecutive channels of one row and stores them together.
__device__ __forceinline__ float activate(float y, int act) {
  return act == 1 ? 0.5f * y * (1.0f + erff(y * 0.70710678118654752f)) : y;
}

template <int OT>
__device__ __forceinline__ void store4(const LinearArgs& a, int64_t m, int n, i32x4 c) {
  using O = typename Elem<OT>::type;
  const float sx = a.x_scale[m];
  O* out = static_cast<O*>(a.out) + m * a.ldo + n;
  typedef O o4 __attribute__((ext_vector_type(4)));
  o4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ni = n + i < a.n ? n + i : a.n - 1;
    float y = (float)c[i] * (sx * a.w_scale[ni]);
    if (a.bias) y += a.bias[ni];
    v[i] = (O)activate(y, a.act);
  }
  if (n + 4 <= a.n) {
    store_as(out, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.n) out[i] = v[i];
  }
}

// 16 bytes of a row of `k`, zeros behind its end
__device__ __forceinline__ u32x4 load_row16(const int8_t* row, int at, int k) {
  u32x4 v = {0, 0, 0, 0};
  if (at + 16 <= k) return load_as<u32x4>(row + at);
  if (at < k) {
    int8_t b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = at + i < k ? row[at + i] : 0;
    __builtin_memcpy(&v, b, 16);
  }
  return v;
}

// 64 x 64 tiles, 64 bytes of k at a time, any size and alignment.
constexpr int kPad = 80;   // bytes from one LDS row to the next
template <int OT>
__global__ __launch_bounds__(256) void linear_any_kernel(LinearArgs a, int64_t tiles_n, int64_t tiles) {
  __shared__ __align__(16) int8_t lw[64 * kPad], lx[64 * kPad];
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
  const int n0 = (int)(tile % tiles_n) * 64;
  const int64_t m0 = tile / tiles_n * 64;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int row = t >> 2, col = (t & 3) * 16;
  const int8_t* wr = a.w + (int64_t)(n0 + row < a.n ? n0 + row : a.n - 1) * a.ldw;
  const int8_t* xr = a.x + (m0 + row < a.m ? m0 + row : a.m - 1) * a.ldx;
  i32x4 acc[2][2] = {};
  const int wn = (wave & 1) * 32, wm = (wave >> 1) * 32;
  for (int k0 = 0; k0 < a.k; k0 += 64) {
    const u32x4 vw = load_row16(wr, k0 + col, a.k), vx = load_row16(xr, k0 + col, a.k);
    __syncthreads();
    *reinterpret_cast<u32x4*>(lw + row * kPad + col) = vw;
    *reinterpret_cast<u32x4*>(lx + row * kPad + col) = vx;
    __syncthreads();
    i32x4 fw[2], fx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fw[i] = *reinterpret_cast<const i32x4*>(lw + (wn + 16 * i + (lane & 15)) * kPad + (lane >> 4) * 16);
      fx[i] = *reinterpret_cast<const i32x4*>(lx + (wm + 16 * i + (lane & 15)) * kPad + (lane >> 4) * 16);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fx[j], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t m = m0 + wm + 16 * j + (lane & 15);
      const int n = n0 + wn + 16 * i + 4 * (lane >> 4);
      if (m < a.m && n < a.n) store4<OT>(a, m, n, acc[i][j]);
    }
  }
}

}  // namespace

namespace {
template <int TY>
hipError_t quantize(const void* x, int64_t ldx, int64_t rows, int cols, int cols_pad, int8_t* q, int64_t ldq, float* scale,
                    hipStream_t s) {
  constexpr int N = Chunk<typename Elem<TY>::type>::N;
  auto go = [&](auto kernel, int waves) {
    const int groups = waves == 1 ? 4 : 1;
    kernel<<<grid_of((rows + groups - 1) / groups), 64 * waves * groups, 0, s>>>(x, ldx, rows, cols, cols_pad, q, ldq, scale);
    return hipGetLastError();
  };
  const int chunks = (cols_pad + N - 1) / N;
  if (chunks <= 64) return go(quantize_rows_kernel<TY, 1, 1>, 1);
  if (chunks <= 64 * 2) return go(quantize_rows_kernel<TY, 1, 2>, 1);
  if (chunks <= 64 * 4) return go(quantize_rows_kernel<TY, 1, 4>, 1);
  if (chunks <= 64 * 8) return go(quantize_rows_kernel<TY, 4, 2>, 4);
  if (chunks <= 64 * 16) return go(quantize_rows_kernel<TY, 4, 4>, 4);
  if (chunks <= 64 * 32) return go(quantize_rows_kernel<TY, 8, 4>, 8);
  quantize_long_rows_kernel<TY><<<grid_of(rows), 256, 0, s>>>(x, ldx, rows, cols, cols_pad, q, ldq, scale);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_quantize_rows(int type, const void* x, int64_t ldx, int64_t rows, int cols, int cols_pad, int8_t* q,
                                int64_t ldq, float* scale, hipStream_t s) {
  return type == T_F32    ? quantize<T_F32>(x, ldx, rows, cols, cols_pad, q, ldq, scale, s)
         : type == T_BF16 ? quantize<T_BF16>(x, ldx, rows, cols, cols_pad, q, ldq, scale, s)
                          : quantize<T_F16>(x, ldx, rows, cols, cols_pad, q, ldq, scale, s);
}

hipError_t launch_linear(const LinearArgs& a, hipStream_t s) {
  const int64_t tiles_n = ((int64_t)a.n + 63) / 64, tiles = tiles_n * (((int64_t)a.m + 63) / 64);
  auto kernel = a.out_type == T_F32 ? linear_any_kernel<T_F32> : a.out_type == T_BF16 ? linear_any_kernel<T_BF16>
                                                                                      : linear_any_kernel<T_F16>;
  kernel<<<grid_of(tiles), 256, 0, s>>>(a, tiles_n, tiles);
  return hipGetLastError();
}

}  // namespace enc
}  // namespace rr
