// rr_encoder_linear.hip — 8-bit rows and the 8-bit matrix product (rr_quantize_rows, rr_linear_i8).
#include "rr_encoder_device.h"

namespace rr {
namespace enc {
namespace {

// ---- 8-bit rows ----------------------------------------------------------------------------------------------------
// One workgroup per row, two passes over it (the second one from cache).
template <int TY>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* xv, int64_t ldx, int64_t rows, int cols, int cols_pad,
                                                            int8_t* q, int64_t ldq, float* scale) {
  using E = typename Elem<TY>::type;
  __shared__ float red[4];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const E* x = static_cast<const E*>(xv) + r * ldx;
    unsigned m = 0;
    for (int c = threadIdx.x; c < cols; c += 256) {
      const unsigned t = mag((float)x[c]);
      m = t > m ? t : m;
    }
    const float s = row_scale(group_max<4>(m, red));
    const float div = row_divisor(s);
    const bool dead = !(s == s);
    for (int c = threadIdx.x; c < cols_pad; c += 256)
      q[r * ldq + c] = c < cols && !dead ? (int8_t)to_i8((float)x[c], div) : 0;
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

hipError_t launch_quantize_rows(int type, const void* x, int64_t ldx, int64_t rows, int cols, int cols_pad, int8_t* q,
                                int64_t ldq, float* scale, hipStream_t s) {
  auto kernel = type == T_F32 ? quantize_rows_kernel<T_F32> : type == T_BF16 ? quantize_rows_kernel<T_BF16>
                                                                             : quantize_rows_kernel<T_F16>;
  kernel<<<grid_of(rows), 256, 0, s>>>(x, ldx, rows, cols, cols_pad, q, ldq, scale);
  return hipGetLastError();
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
