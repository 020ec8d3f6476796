// rr_encoder_norm.hip — the norms around a block, fused with its gate, residual scale and 8-bit rows (rr_block_norm).
#include "rr_encoder_device.h"

namespace rr {
namespace enc {
namespace {

template <int W>
__device__ __forceinline__ void norm_in_place(float* v, int cols, int kind, float eps, float* red) {
  float mean = 0.f;
  if (kind == 1) {
    float s = 0.f;
    for (int c = threadIdx.x; c < cols; c += 64 * W) s += v[c];
    mean = group_sum<W>(s, red) / (float)cols;
  }
  float s2 = 0.f;
  for (int c = threadIdx.x; c < cols; c += 64 * W) s2 += (v[c] - mean) * (v[c] - mean);
  const float r = 1.0f / sqrtf(group_sum<W>(s2, red) / (float)cols + eps);
  for (int c = threadIdx.x; c < cols; c += 64 * W) v[c] = (v[c] - mean) * r;
}

// One workgroup per row; the row lies in LDS in fp32 between the steps, each thread at its own columns.
template <int TY>
__global__ __launch_bounds__(256) void block_norm_kernel(NormArgs a) {
  using E = typename Elem<TY>::type;
  extern __shared__ float v[];
  __shared__ float red[4];
  const int cols = a.cols;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
  const E* y = static_cast<const E*>(a.y) + r * a.ldy;
  for (int c = threadIdx.x; c < cols; c += 256) v[c] = (float)y[c];
  if (a.post) norm_in_place<4>(v, cols, a.post, a.eps, red);
  const E* x = a.x ? static_cast<const E*>(a.x) + r * a.ldx : nullptr;
  const E* g = a.gate ? static_cast<const E*>(a.gate) + r / a.rows_per_gate * a.ldg : nullptr;
  for (int c = threadIdx.x; c < cols; c += 256) {
    float u = v[c];
    if (a.post_w) u *= (float)static_cast<const E*>(a.post_w)[c];
    if (a.post_b) u += (float)static_cast<const E*>(a.post_b)[c];
    if (g) u *= (float)g[c];
    if (x) u += a.residual_scale * (float)x[c];
    v[c] = u;
    if (a.stream) static_cast<E*>(a.stream)[r * a.lds + c] = (E)u;
  }
  if (!a.next) continue;
  norm_in_place<4>(v, cols, a.next, a.eps, red);
  unsigned m = 0;
  for (int c = threadIdx.x; c < cols; c += 256) {
    float u = v[c];
    if (a.next_w) u *= (float)static_cast<const E*>(a.next_w)[c];
    if (a.next_b) u += (float)static_cast<const E*>(a.next_b)[c];
    v[c] = u;
    if (a.normed) static_cast<E*>(a.normed)[r * a.ldn + c] = (E)u;
    m = mag(u) > m ? mag(u) : m;
  }
  if (!a.q) continue;
  const float s = row_scale(group_max<4>(m, red));
  const float div = row_divisor(s);
  const bool dead = !(s == s);
  for (int c = threadIdx.x; c < cols; c += 256) a.q[r * a.ldq + c] = dead ? 0 : (int8_t)to_i8(v[c], div);
  if (threadIdx.x == 0) a.q_scale[r] = s;
  }
}

}  // namespace

hipError_t launch_block_norm(int type, const NormArgs& a, hipStream_t s) {
  auto kernel = type == T_F32 ? block_norm_kernel<T_F32> : type == T_BF16 ? block_norm_kernel<T_BF16> : block_norm_kernel<T_F16>;
  const size_t lds = (size_t)a.cols * 4;
  if (lds > 48 * 1024)
    if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds)) return e;
  kernel<<<grid_of(a.rows), 256, lds, s>>>(a);
  return hipGetLastError();
}

}  // namespace enc
}  // namespace rr
