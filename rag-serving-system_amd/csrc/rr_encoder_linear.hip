// rr_encoder_linear.hip — 8-bit rows and the 8-bit matrix product (rr_quantize_rows, rr_linear_i8).
#include "rr_encoder_device.h"

#include <algorithm>

namespace rr {
namespace enc {
namespace {

// ---- rows at any address ---------------------------------------------------------------------------------------------
// Rows of `k` bytes that may start anywhere, `ld` apart, as a buffer of dwords: the loads' addresses are multiples of four
// (16-byte loads at odd ones take 128 cycles an instruction here, which made 48 rows of 3769 take 20 us), and what lies behind
// the last row is read as zeros. Rows are less than RR_LINEAR_LDMOST = 2^22 bytes apart and at most 514 here: offsets below 2^32.
struct RowBytes {
  __amdgpu_buffer_rsrc_t r;
  unsigned first, ld;   // first: where row 0 starts in the buffer
  bool odd;             // whether a row may start between dwords
  __device__ __forceinline__ RowBytes(const int8_t* rows, int64_t ld, int64_t count, int k)
      : first((unsigned)(reinterpret_cast<uintptr_t>(rows) & 3)), ld((unsigned)ld), odd(first | (ld & 3)) {
    r = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(rows - first), 0,
                                          (int)((first + (unsigned)(count - 1) * this->ld + k + 3) & ~3u), 0x00020000);
  }
  __device__ __forceinline__ unsigned start(int row) const { return first + row * ld; }
  // 16 bytes of the row that starts at `start`, in two parts: what is loaded (nothing behind column k) ...
  struct Sixteen {
    u32x4 four;
    unsigned fifth;
  };
  __device__ __forceinline__ void load(Sixteen& to, unsigned start, int at, int k) const {
    const unsigned from = at < k ? (start & ~3u) + at : ~31u;
    to.four = __builtin_amdgcn_raw_buffer_load_b128(r, from, 0, 0);
    if (odd) to.fifth = __builtin_amdgcn_raw_buffer_load_b32(r, from + 16, 0, 0);
  }
  // ... and the bytes. Those behind column k may be anything: one factor of a product has to have zeros there, see below.
  __device__ __forceinline__ u32x4 get(const Sixteen& of, unsigned start) const {
    if (!odd) return of.four;
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbyte(i < 3 ? of.four[i + 1] : of.fifth, of.four[i], start & 3);
    return v;
  }
};
// zeros behind column k
__device__ __forceinline__ u32x4 cut(u32x4 v, int at, int k) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = k - at - 4 * i;
    v[i] = left >= 4 ? v[i] : left <= 0 ? 0u : v[i] & ((1u << 8 * left) - 1);
  }
  return v;
}

// ---- copies for the tiled product -------------------------------------------------------------------------------------
// A matrix of `k` columns copied to rows of `kp` = k rounded up to 16, zeros behind k. A thread a 16-byte column; block `b`
// takes the b-th columns, as many as it has threads.
struct Repack {
  const int8_t* from;
  int64_t ld, rows;
  int8_t* to;
  int k, kp;
  __host__ __device__ int64_t blocks(int threads) const { return from ? (rows * (kp / 16) + threads - 1) / threads : 0; }
};
__device__ __forceinline__ void repack(const Repack& p, int64_t b) {
  const unsigned cols = p.kp / 16;
  const int64_t at = b * blockDim.x;
  const unsigned in = (unsigned)(at % cols) + threadIdx.x;
  const int64_t r = at / cols + in / cols;
  const int c = (int)(in % cols) * 16;
  const int64_t r0 = at / cols, most = blockDim.x / cols + 2;
  const RowBytes rows(p.from + r0 * p.ld, p.ld, p.rows - r0 < most ? p.rows - r0 : most, p.k);
  if (r >= p.rows) return;
  const unsigned start = rows.start((int)(r - r0));
  RowBytes::Sixteen v;
  rows.load(v, start, c, p.k);
  store_as(p.to + r * p.kp + c, cut(rows.get(v, start), c, p.k));
}
__global__ __launch_bounds__(256) void repack_kernel(Repack one, Repack two, int64_t blocks_one, int64_t blocks) {
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x)
    if (b < blocks_one) repack(one, b);
    else repack(two, b - blocks_one);
}

// ---- 8-bit rows ----------------------------------------------------------------------------------------------------
// A row in the registers of W waves, or of G lanes of one, S times 16 bytes a lane. cols_pad: columns written, zeros behind the
// row's own. Bandwidth: 16384 x 4096 bf16 46 us, 4.4 TB/s (of 5.2 that a large copy reaches; a wave a row instead of
// four changes nothing).
template <int TY, int W, int S, int G = 64>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void quantize_rows_kernel(const void* xv, int64_t ldx, int64_t rows,
                                                                             int cols, int cols_pad, int8_t* q, int64_t ldq,
                                                                             float* scale, unsigned blocks, Repack also) {
  using E = typename Elem<TY>::type;
  constexpr int N = Chunk<E>::N, kLanes = W == 1 ? G : 64 * W, kGroups = W == 1 ? 256 / G : 1;
  if (blockIdx.x >= blocks) {
    const int64_t all = also.blocks(blockDim.x);
    for (int64_t b = blockIdx.x - blocks; b < all; b += gridDim.x - blocks) repack(also, b);
    return;
  }
  __shared__ float red[2 * W];
  RowReduce<W, G> over{red};
  const int t = threadIdx.x % kLanes;
  for (int64_t r = (int64_t)blockIdx.x * kGroups + threadIdx.x / kLanes; r < rows; r += (int64_t)blocks * kGroups) {
    const E* x = static_cast<const E*>(xv) + r * ldx;
    Chunk<E> c[S];
#pragma unroll
    for (int s = 0; s < S; ++s) c[s].load(x + (s * kLanes + t) * N, cols - (s * kLanes + t) * N);
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
      store_i8<N>(q + r * ldq + (s * kLanes + t) * N, v, div, cols_pad - (s * kLanes + t) * N);
    }
    if (t == 0) scale[r] = sc;
  }
}

// Rows of any length: one workgroup per row, two passes over it (the second one from cache). Columns up to 2^31 - 1 are counted
// in unsigned, where the step behind the last one still fits. 4096 x 40000 bf16 320 us, 1.5 TB/s, fp32 417 us, 2.0 TB/s (element
// by element, of 5.2 that a large copy reaches); a single row is one CU's work: 2^25 columns 83 ms.
template <int TY>
__global__ __launch_bounds__(256) void quantize_long_rows_kernel(const void* xv, int64_t ldx, int64_t rows, int cols,
                                                                 int cols_pad, int8_t* q, int64_t ldq, float* scale,
                                                                 unsigned blocks, Repack also) {
  using E = typename Elem<TY>::type;
  __shared__ float red[8];
  if (blockIdx.x >= blocks) {
    const int64_t all = also.blocks(blockDim.x);
    for (int64_t b = blockIdx.x - blocks; b < all; b += gridDim.x - blocks) repack(also, b);
    return;
  }
  RowReduce<4> over{red};
  for (int64_t r = blockIdx.x; r < rows; r += blocks) {
    const E* x = static_cast<const E*>(xv) + r * ldx;
    unsigned m = 0;
    for (unsigned c = threadIdx.x; c < (unsigned)cols; c += 256) {
      const unsigned t = mag((float)x[c]);
      m = t > m ? t : m;
    }
    const float s = row_scale(over.max(m));
    const float div = row_divisor(s);
    for (unsigned c = threadIdx.x; c < (unsigned)cols_pad; c += 256)
      q[r * ldq + c] = c < (unsigned)cols && s == s ? (int8_t)to_i8((float)x[c], div) : 0;
    if (threadIdx.x == 0) scale[r] = s;
  }
}

// ---- the product ---------------------------------------------------------------------------------------------------
// out^T = w x^T: the matrix instruction's rows are output channels and its columns rows of x, so a lane holds four
// consecutive channels of one row and stores them together.
template <int OT>
__device__ __forceinline__ float gelu(float y) {
  if constexpr (OT == T_F32) return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
  // 16-bit results: erf to 1.5e-7 by Abramowitz and Stegun 7.1.26, a third of erff's instructions
  // (613 x 4096 results of a 1024-long product: 18.2 us with erff, 10.2 with this); relative to 1 - erf it is off by
  // 5e-5 at y = -3 and 4e-3 at -6, where 1 + erf in fp32 has lost all of it
  const float z = fabsf(y) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, z, 1.0f));
  const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
  const float e = p * __builtin_amdgcn_exp2f(z * z * -1.4426950408889634f);   // 1 - erf(z)
  return 0.5f * y * (y < 0.f ? e : 2.0f - e);
}
template <int OT>
__device__ __forceinline__ float activate(float y, int act) {
  return act == 1 ? gelu<OT>(y) : y;
}

// Four channels of one row: sums to results.
template <int OT>
__device__ __forceinline__ void store4(const LinearArgs& a, int64_t m, int n, i32x4 c, float sx, const float* sw,
                                       const float* bias) {
  using O = typename Elem<OT>::type;
  O* out = static_cast<O*>(a.out) + m * a.ldo + n;
  typedef O o4 __attribute__((ext_vector_type(4)));
  o4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (O)activate<OT>((float)c[i] * (sx * sw[i]) + bias[i], a.act);
  if (n + 4 <= a.n) {
    store_as(out, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.n) out[i] = v[i];
  }
}

// 64 x 64 tiles, rows at any byte: through registers into LDS, the next two steps' loads in flight during a step's matrix
// instructions. Two groups of four waves take every other 128 bytes of k, since such calls have few tiles and wait for their
// chain of steps; each group then finishes half of the tile, with scales that it asked for before the first step
// (1031 rows of 1000 -> 777, GPU time: 10.3 us with one group and scales read at the end, 8.1 so; rows at 4-byte addresses take
// the tiled product, 6.3).
constexpr int kAnyStep = 128, kAnyGroups = 2, kPad = kAnyStep + 16;   // kPad: bytes from one LDS row to the next
template <int OT>
__global__ __launch_bounds__(256 * kAnyGroups) void linear_any_kernel(LinearArgs a, int64_t tiles_n, int64_t tiles) {
  __shared__ __align__(16) int8_t lds[kAnyGroups][2][64 * kPad];
  const int t = threadIdx.x & 255, lane = t & 63, wave = t >> 6, group = threadIdx.x >> 8;
  const int row = t >> 2, col = (t & 3) * 16;
  const int wn = (wave & 1) * 32, wm = (wave >> 1) * 32;
  int8_t *lw = lds[group][0], *lx = lds[group][1];
  struct Step {
    RowBytes::Sixteen w[2], x[2];
  };
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int n0 = (int)(tile % tiles_n) * 64;
    const int64_t m0 = tile / tiles_n * 64;
    const RowBytes rw(a.w + n0 * a.ldw, a.ldw, a.n - n0 < 64 ? a.n - n0 : 64, a.k);
    const RowBytes rx(a.x + m0 * a.ldx, a.ldx, a.m - m0 < 64 ? a.m - m0 : 64, a.k);
    const unsigned w_at = rw.start(row), x_at = rx.start(row);
    auto fetch = [&](Step& s, int k0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        rw.load(s.w[h], w_at, k0 + 64 * h + col, a.k);
        rx.load(s.x[h], x_at, k0 + 64 * h + col, a.k);
      }
    };
    i32x4 acc[2][2] = {};
    auto take = [&](Step& s, int k0, int next) {   // and asks for the step at `next`
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<u32x4*>(lw + row * kPad + 64 * h + col) = rw.get(s.w[h], w_at);
        *reinterpret_cast<u32x4*>(lx + row * kPad + 64 * h + col) = cut(rx.get(s.x[h], x_at), k0 + 64 * h + col, a.k);
      }
      __syncthreads();
      fetch(s, next);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        i32x4 fw[2], fx[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          fw[i] = *reinterpret_cast<const i32x4*>(lw + (wn + 16 * i + (lane & 15)) * kPad + 64 * kk + (lane >> 4) * 16);
          fx[i] = *reinterpret_cast<const i32x4*>(lx + (wm + 16 * i + (lane & 15)) * kPad + 64 * kk + (lane >> 4) * 16);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fx[j], acc[i][j], 0, 0, 0);
      }
    };
    constexpr int kRound = kAnyGroups * kAnyStep;   // what all groups take in a step; both go through the same steps
    Step one, two;
    const int first = group * kAnyStep;
    fetch(one, first);
    fetch(two, first + kRound);
    // group g finishes channels 16 g .. 16 g + 15 of every wave's 32; what that takes is asked for now
    const int n = n0 + wn + 16 * group + 4 * (lane >> 4);
    float scale[4], bias[4], row_scales[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ni = n + i < a.n ? n + i : a.n - 1;
      scale[i] = a.w_scale[ni];
      bias[i] = a.bias ? a.bias[ni] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t m = m0 + wm + 16 * j + (lane & 15);
      row_scales[j] = a.x_scale[m < a.m ? m : a.m - 1];
    }
    for (int k0 = 0; k0 < a.k; k0 += 2 * kRound) {
      take(one, first + k0, first + k0 + 2 * kRound);
      if (k0 + kRound < a.k) take(two, first + k0 + kRound, first + k0 + 3 * kRound);
    }
    __syncthreads();
    i32x4* other = reinterpret_cast<i32x4*>(lds[0][0]);   // [group][wave][j][lane]
#pragma unroll
    for (int j = 0; j < 2; ++j) other[(((1 - group) * 4 + wave) * 2 + j) * 64 + lane] = group ? acc[0][j] : acc[1][j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const i32x4 c = (group ? acc[1][j] : acc[0][j]) + other[((group * 4 + wave) * 2 + j) * 64 + lane];
      const int64_t m = m0 + wm + 16 * j + (lane & 15);
      if (m < a.m && n < a.n) store4<OT>(a, m, n, c, row_scales[j], scale, bias);
    }
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------
// Up to 16 R rows of x: the weights' bytes are all there is. A workgroup holds 16 channels; its eight waves take every eighth
// 64 bytes of k, straight from memory into the matrix instruction's operands, and their integer sums, exact in any order, meet
// in LDS. FUSED: x is floating point and every workgroup makes its own 8-bit rows in LDS while its first weights arrive: one
// launch, where a short row would wait for two.
// One row 4096 -> 1024 4.3 us (its 4 MiB of weights would take 0.8 at copy speed: the rest is a launch and three memory
// latencies in a row), 16 rows 5.6; 1024 -> 4096 3.4 and 3.6.
constexpr int kFewWaves = 8, kFewRows = 48;
constexpr int kFusedRow = 8192;    // columns of a single row that every workgroup converts for itself, all waves at it,
constexpr int kFusedWave = 1024;   // and of up to eight rows, a wave each

// A row's 8-bit row by W waves, of which this is lane t: the row's values are asked for first, then the rest is done.
template <int XT, int W>
struct Row8 {
  using E = typename Elem<XT>::type;
  static constexpr int N = Chunk<E>::N, S = (W == 1 ? kFusedWave : kFusedRow) / (64 * W * N);
  Chunk<E> c[S];
  __device__ __forceinline__ void load(const E* x, int k, int t) {
#pragma unroll
    for (int s = 0; s < S; ++s) c[s].load(x + (s * 64 * W + t) * N, k - (s * 64 * W + t) * N);
  }
  __device__ __forceinline__ void put(int8_t* to, int kp, float* scale, int t, float* red) {
    unsigned top = 0;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int e = 0; e < N; ++e) top = mag(c[s][e]) > top ? mag(c[s][e]) : top;
    RowReduce<W> over{red};
    const float s8 = row_scale(over.max(top));
    const float div = row_divisor(s8);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int at = (s * 64 * W + t) * N;
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = s8 == s8 ? c[s][e] : 0.f;
      if (at < kp) store_i8<N>(to + at, v, div, N);
    }
    if (t == 0) *scale = s8;
  }
};

// SINGLE: of a fused kernel, that x is one row.
template <int OT, int R, int XT, bool SINGLE = false>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few_kernel(LinearArgs a) {
  constexpr bool kFused = XT != T_I8;
  constexpr int kAhead = R == 1 ? 8 : 4;   // steps of 64 bytes, of weights and rows, loaded together
  __shared__ __align__(16) i32x4 sums[kFewWaves][R][64];
  __shared__ __align__(16) int8_t x8[kFused ? kFusedRow : 16];   // (eight rows of kFusedWave columns are as many)
  __shared__ float sc[16];
  __shared__ float red[2 * kFewWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * R, kp = (a.k + 63) / 64 * 64;   // (fused: one block of rows)
  const RowBytes rw(a.w + (int64_t)n0 * a.ldw, a.ldw, a.n - n0 < 16 ? a.n - n0 : 16, a.k);
  const RowBytes rx(a.x + m0 * a.ldx, a.ldx, a.m - m0 < 16 * R ? a.m - m0 : 16 * R, a.k);   // (not fused)
  const unsigned w_at = rw.start(i);
  i32x4 acc[R] = {};
  float scale[4], bias[4];   // of the four channels that this lane finishes
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int n = n0 + 4 * g + x < a.n ? n0 + 4 * g + x : a.n - 1;
    scale[x] = a.w_scale[n];
    bias[x] = a.bias ? a.bias[n] : 0.f;
  }
  Row8<kFused ? XT : T_F32, SINGLE ? kFewWaves : 1> rows;
  const int t = SINGLE ? threadIdx.x : lane, mine = SINGLE ? 0 : wave;
  if constexpr (kFused)
    if (mine < a.m) rows.load(reinterpret_cast<const typename Elem<XT>::type*>(a.x) + mine * a.ldx, a.k, t);
  for (int k0 = wave * 64; k0 < kp || (kFused && k0 == wave * 64); k0 += kAhead * kFewWaves * 64) {
    RowBytes::Sixteen w[kAhead], x[kFused ? 1 : kAhead][R];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) rw.load(w[s], w_at, k0 + s * kFewWaves * 64 + 16 * g, a.k);
    if constexpr (!kFused)
#pragma unroll
      for (int s = 0; s < kAhead; ++s)
#pragma unroll
        for (int r = 0; r < R; ++r) rx.load(x[s][r], rx.start(16 * r + i), k0 + s * kFewWaves * 64 + 16 * g, a.k);
    if constexpr (kFused) {
      if (k0 == wave * 64) {   // (every wave comes here once, with or without weights to multiply)
        if (mine < a.m) rows.put(x8 + mine * kp, kp, sc + mine, t, red);
        __syncthreads();
      }
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const int at = k0 + s * kFewWaves * 64 + 16 * g;
      const u32x4 ws = rw.get(w[s], w_at);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        u32x4 v;
        if constexpr (kFused) {
          v = u32x4{0, 0, 0, 0};
          if (i < a.m && at < kp) v = *reinterpret_cast<const u32x4*>(x8 + i * kp + at);
        } else {
          v = cut(rx.get(x[s][r], rx.start(16 * r + i)), at, a.k);
        }
        acc[r] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, ws), __builtin_bit_cast(i32x4, v), acc[r], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) sums[wave][r][lane] = acc[r];
  __syncthreads();
  for (int r = wave; r < R; r += kFewWaves) {
    i32x4 c = sums[0][r][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) c += sums[w][r][lane];
    const int m = m0 + 16 * r + i, n = n0 + 4 * g;
    if (m < a.m && n < a.n) store4<OT>(a, m, n, c, kFused ? sc[16 * r + i] : a.x_scale[m], scale, bias);
  }
}

// ---- the tiled product -----------------------------------------------------------------------------------------------
// Workgroup tile: TN channels x TM rows, 128 bytes of k a step, both operands brought into LDS by the loads' LDS form (no
// registers, no ds_write) into BUFS buffers in turn: BUFS - 1 steps are in flight while one is multiplied, one barrier a step.
// Waves: WN x WM, each (TN / WN) x (TM / WM) in 32 x 32 x 32 instructions. LDS rows hold a step; the 16-byte column c of row r
// lies at column c ^ swizzle(r), so that the 16 lanes that read a column of 16 rows at once meet all 64 banks.
// Wants rows at 4-byte addresses. What lies behind the last row is out of the buffer's range and read as zeros, and so is a
// 16-byte column that starts behind k; the one that k ends in is cut in LDS, in the rows of x alone: zeros in one factor do.
// 16384 x 4096 -> 1024 (int8 rows, bf16 results) in 256 x 256 tiles: 70 us, 1.95 POP/s (the library's i8 product of these
// sizes takes 75). A step's 2048 cycles of matrix instructions need as many of LDS (192 KiB of reads, 64 KiB of arriving
// rows); tried and dropped: four waves of 128 x 128 (fewer LDS reads, 87 us), 64-byte steps in four buffers (87), operands
// read one part ahead with the barrier inside the step (78). A quarter of the tiles on a quarter of the CUs take 51 us, so
// the rest is the whole chip's clock under matrix load.
constexpr int kStep = 128, kCols = kStep / 16;
__device__ __forceinline__ int swizzle(int r) { return r / 2 % 8; }   // (two rows fill the banks once)

__device__ __forceinline__ i32x4 buffer_of(const void* p, unsigned bytes) {
  const uint64_t at = (uint64_t)p;
  return i32x4{__builtin_amdgcn_readfirstlane((int)(unsigned)at), __builtin_amdgcn_readfirstlane((int)(unsigned)(at >> 32)),
               __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
// 16 bytes a lane from buffer + at to LDS address `to` + 16 * lane
__device__ __forceinline__ void load_to_lds(i32x4 buffer, unsigned at, unsigned to) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
      : "=&s"(keep)
      : "v"(at), "s"(buffer), "s"(to)
      : "memory");
}
// all but this wave's last N loads have landed, its LDS reads are done, and so are the other waves'
template <int N>
__device__ __forceinline__ void step_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

template <int OT, int ACT, int TN, int TM, int WN, int WM, int BUFS>
__global__ __launch_bounds__(64 * WN * WM, 1) void linear_tile_kernel(LinearArgs a, int tiles_n, int64_t tiles) {
  constexpr int kWaves = WN * WM, kN = TN / WN / 32, kM = TM / WM / 32;
  constexpr int kBuf = (TN + TM) * kStep, kLoadsN = TN * kStep / (1024 * kWaves), kLoadsM = TM * kStep / (1024 * kWaves);
  using O = typename Elem<OT>::type;
  constexpr int kOutLd = kN * 32 * sizeof(O) + 16;   // bytes of an output row in LDS
  constexpr int kLds = BUFS * kBuf > kWaves * 32 * kOutLd ? BUFS * kBuf : kWaves * 32 * kOutLd;
  __shared__ __align__(1024) char lds[kLds];
  __shared__ __align__(16) float chan[2][TN];   // the tile's channel scales and biases
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const unsigned lds0 = (unsigned)(uintptr_t)lds;
  // Workgroups go to the 8 XCDs in turn: each XCD takes a contiguous run of tiles, channels first, so that the tiles that
  // share rows of x meet in one XCD's cache.
  const int64_t per = tiles / 8, more = tiles % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
  const int64_t tile = xcd * per + (xcd < more ? xcd : more) + at;
  const int n0 = (int)(tile % tiles_n) * TN;
  const int64_t m0 = tile / tiles_n * TM;
  const int rows_n = a.n - n0 < TN ? a.n - n0 : TN, rows_m = a.m - m0 < TM ? (int)(a.m - m0) : TM;
  const i32x4 bw = buffer_of(a.w + (int64_t)n0 * a.ldw, (unsigned)((rows_n - 1) * a.ldw + a.k + 3) & ~3u);
  const i32x4 bx = buffer_of(a.x + m0 * a.ldx, (unsigned)((rows_m - 1) * a.ldx + a.k + 3) & ~3u);
  for (int c = threadIdx.x; c < TN; c += 64 * kWaves) {
    const int n = n0 + c < a.n ? n0 + c : a.n - 1;
    chan[0][c] = a.w_scale[n];
    chan[1][c] = a.bias ? a.bias[n] : 0.f;
  }

  // this lane's 16 bytes of load j: row (64 / kCols) (j waves + wave) + lane / kCols, LDS column lane % kCols
  unsigned from_w[kLoadsN], from_x[kLoadsM];
  int col_w[kLoadsN], col_x[kLoadsM];
#pragma unroll
  for (int j = 0; j < kLoadsN; ++j) {
    const int r = 64 / kCols * (j * kWaves + wave) + lane / kCols;
    col_w[j] = 16 * (lane % kCols ^ swizzle(r));
    from_w[j] = (unsigned)(r * a.ldw + col_w[j]);
  }
#pragma unroll
  for (int j = 0; j < kLoadsM; ++j) {
    const int r = 64 / kCols * (j * kWaves + wave) + lane / kCols;
    col_x[j] = 16 * (lane % kCols ^ swizzle(r));
    from_x[j] = (unsigned)(r * a.ldx + col_x[j]);
  }
  auto fetch = [&](int k0, int buf) {
    const unsigned to = lds0 + buf * kBuf + wave * 1024;
#pragma unroll
    for (int j = 0; j < kLoadsN; ++j)
      load_to_lds(bw, k0 + col_w[j] < a.k ? from_w[j] + k0 : ~15u, to + j * kWaves * 1024);
#pragma unroll
    for (int j = 0; j < kLoadsM; ++j)
      load_to_lds(bx, k0 + col_x[j] < a.k ? from_x[j] + k0 : ~15u, to + TN * kStep + j * kWaves * 1024);
  };
  i32x16 acc[kN][kM] = {};
  const int row = lane % 32, half = lane / 32, swz = swizzle(row);
  float sx[kM];
#pragma unroll
  for (int j = 0; j < kM; ++j) {
    const int64_t m = m0 + (wm * kM + j) * 32 + row;
    sx[j] = a.x_scale[m < a.m ? m : a.m - 1];
  }
  const int steps = (a.k + kStep - 1) / kStep;
#pragma unroll
  for (int s = 0; s < BUFS - 1; ++s)
    if (s < steps) fetch(s * kStep, s);
  int buf = 0, next = BUFS - 1;
  for (int s = 0; s < steps; ++s) {
    if (s + BUFS - 2 < steps) step_barrier<(BUFS - 2) * (kLoadsN + kLoadsM)>();
    else step_barrier<0>();
    if (s + BUFS - 1 < steps) fetch((s + BUFS - 1) * kStep, next);   // (its buffer was last read before this barrier)
    if (s + 1 == steps && a.k % 16) {
      for (int r = threadIdx.x; r < TM; r += 64 * kWaves) {
        const int c = a.k % kStep / 16;
        u32x4* at = reinterpret_cast<u32x4*>(lds + buf * kBuf + TN * kStep + r * kStep + 16 * (c ^ swizzle(r)));
        *at = cut(*at, 16 * c, a.k % kStep);
      }
      __syncthreads();
    }
    const char* lw = lds + buf * kBuf + (wn * kN * 32 + row) * kStep;
    const char* lx = lds + buf * kBuf + TN * kStep + (wm * kM * 32 + row) * kStep;
#pragma unroll
    for (int kk = 0; kk < kStep / 32; ++kk) {
      const int c = 16 * ((2 * kk + half) ^ swz);
      i32x4 fw[kN], fx[kM];
#pragma unroll
      for (int i = 0; i < kN; ++i) fw[i] = *reinterpret_cast<const i32x4*>(lw + i * 32 * kStep + c);
#pragma unroll
      for (int j = 0; j < kM; ++j) fx[j] = *reinterpret_cast<const i32x4*>(lx + j * 32 * kStep + c);
#pragma unroll
      for (int i = 0; i < kN; ++i)
#pragma unroll
        for (int j = 0; j < kM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[i], fx[j], acc[i][j], 0, 0, 0);
    }
    buf = buf + 1 == BUFS ? 0 : buf + 1;
    next = next + 1 == BUFS ? 0 : next + 1;
  }
  step_barrier<0>();   // the buffers are free: each wave turns its results into rows there, 32 rows of x at a time
  char* out = lds + wave * 32 * kOutLd;
#pragma unroll
  for (int j = 0; j < kM; ++j) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int nl = i * 32 + 8 * g + 4 * half;
        const f32x4 sw = *reinterpret_cast<const f32x4*>(&chan[0][wn * kN * 32 + nl]);
        const f32x4 bias = *reinterpret_cast<const f32x4*>(&chan[1][wn * kN * 32 + nl]);
        typedef O o4 __attribute__((ext_vector_type(4)));
        o4 v;
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = (O)activate<OT>((float)acc[i][j][4 * g + x] * (sx[j] * sw[x]) + bias[x], ACT);
        *reinterpret_cast<o4*>(out + row * kOutLd + nl * sizeof(O)) = v;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (a wave's own LDS: no barrier)
    constexpr int kPer = 16 / sizeof(O), kLanes = kN * 32 / kPer, kRowsAtOnce = 64 / kLanes;
#pragma unroll
    for (int r = 0; r < 32; r += kRowsAtOnce) {
      const int rr = r + lane / kLanes, nl = lane % kLanes * kPer, n = n0 + wn * kN * 32 + nl;
      const int64_t mm = m0 + (wm * kM + j) * 32 + rr;
      const u32x4 v = *reinterpret_cast<const u32x4*>(out + rr * kOutLd + nl * sizeof(O));
      if (mm < a.m && n < a.n) {
        O* to = static_cast<O*>(a.out) + mm * a.ldo + n;
        if (n + kPer <= a.n) {
          store_as(to, v);
        } else {
          O e[kPer];
          __builtin_memcpy(e, &v, 16);
#pragma unroll
          for (int x = 0; x < kPer; ++x)
            if (n + x < a.n) to[x] = e[x];
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

}  // namespace

namespace {
template <int TY>
hipError_t quantize(const void* x, int64_t ldx, int64_t rows, int cols, int cols_pad, int8_t* q, int64_t ldq, float* scale,
                    const Repack& also, hipStream_t s) {
  constexpr int N = Chunk<typename Elem<TY>::type>::N;
  auto go = [&](auto kernel, int waves, int lanes = 64) {
    const int groups = waves == 1 ? 256 / lanes : 1, threads = waves == 1 ? 256 : 64 * waves;
    const unsigned blocks = grid_of((rows + groups - 1) / groups, threads).x, more = (unsigned)std::min<int64_t>(also.blocks(threads), 1 << 16);
    kernel<<<dim3(blocks + more), threads, 0, s>>>(x, ldx, rows, cols, cols_pad, q, ldq, scale, blocks, also);
    return hipGetLastError();
  };
  const int chunks = cols_pad / N + (cols_pad % N != 0);
  if (chunks <= 8) return go(quantize_rows_kernel<TY, 1, 1, 8>, 1, 8);
  if (chunks <= 16) return go(quantize_rows_kernel<TY, 1, 1, 16>, 1, 16);
  if (chunks <= 32) return go(quantize_rows_kernel<TY, 1, 1, 32>, 1, 32);
  if (chunks <= 64) return go(quantize_rows_kernel<TY, 1, 1>, 1);
  if (chunks <= 64 * 2) return go(quantize_rows_kernel<TY, 1, 2>, 1);
  if (chunks <= 64 * 3) return go(quantize_rows_kernel<TY, 1, 3>, 1);
  if (chunks <= 64 * 4) return go(quantize_rows_kernel<TY, 1, 4>, 1);
  if (chunks <= 64 * 6) return go(quantize_rows_kernel<TY, 3, 2>, 3);
  if (chunks <= 64 * 8) return go(quantize_rows_kernel<TY, 4, 2>, 4);
  if (chunks <= 64 * 12) return go(quantize_rows_kernel<TY, 3, 4>, 3);
  if (chunks <= 64 * 16) return go(quantize_rows_kernel<TY, 4, 4>, 4);
  if (chunks <= 64 * 32) return go(quantize_rows_kernel<TY, 8, 4>, 8);
  return go(quantize_long_rows_kernel<TY>, 4);
}
}  // namespace

hipError_t launch_quantize_rows(int type, const void* x, int64_t ldx, int64_t rows, int cols, int cols_pad, int8_t* q,
                                int64_t ldq, float* scale, const WeightCopy& copy, hipStream_t s) {
  const Repack also{copy.w, copy.ldw, copy.n, copy.to, cols, cols_pad};
  return type == T_F32    ? quantize<T_F32>(x, ldx, rows, cols, cols_pad, q, ldq, scale, also, s)
         : type == T_BF16 ? quantize<T_BF16>(x, ldx, rows, cols, cols_pad, q, ldq, scale, also, s)
                          : quantize<T_F16>(x, ldx, rows, cols, cols_pad, q, ldq, scale, also, s);
}

namespace {
template <int OT, int ACT, int TN, int TM, int WN, int WM, int BUFS>
hipError_t tiled(const LinearArgs& a, hipStream_t s) {
  const int tiles_n = (a.n + TN - 1) / TN;
  const int64_t tiles = (int64_t)tiles_n * ((a.m + TM - 1) / TM);
  linear_tile_kernel<OT, ACT, TN, TM, WN, WM, BUFS><<<dim3((unsigned)tiles), 64 * WN * WM, 0, s>>>(a, tiles_n, tiles);
  return hipGetLastError();
}
template <int OT, int ACT>
hipError_t linear(const LinearArgs& a, hipStream_t s) {
  auto tiles_of = [&](int64_t tn, int64_t tm) { return ((a.n + tn - 1) / tn) * ((a.m + tm - 1) / tm); };
  const bool rows4 = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | a.ldx | a.ldw) & 3) == 0;
  // More rows in blocks of 48, as long as every workgroup has a CU: where the tiles' chain of steps is longer (4096 columns
  // 11.6 us against 9.9, 3008 9.8 / 7.2, 1024 5.3 / 5.2, 400 4.3 / 4.6), or the rows fit no
  // tile (192 x 3769 -> 1024 18.9 / 13.5, x 1001 9.1 / 6.7).
  const int64_t blocks = ((int64_t)a.m + kFewRows - 1) / kFewRows, few = ((int64_t)a.n + 15) / 16 * blocks;
  if (a.m <= kFewRows || (few <= 256 && (!rows4 || a.k >= 1024))) {
    const dim3 grid((a.n + 15) / 16, (unsigned)blocks);
    if (a.m <= 16) linear_few_kernel<OT, 1, T_I8><<<grid, 64 * kFewWaves, 0, s>>>(a);
    else if (a.m <= 32) linear_few_kernel<OT, 2, T_I8><<<grid, 64 * kFewWaves, 0, s>>>(a);
    else linear_few_kernel<OT, 3, T_I8><<<grid, 64 * kFewWaves, 0, s>>>(a);
    return hipGetLastError();
  }
  // The largest tile that still gives the 256 CUs one each, or nearly (int8 rows, GPU time; channels x rows, waves, buffers):
  //   16384 x 4096 -> 1024   256 x 256  70 us    128 x 128  85    64 x 64  125
  //    4096 x 4096 -> 1024   128 x 128, four buffers 24, two 27;  64 x 64  32
  //    2048 x 1024 -> 4096   128 x 128, four buffers 19, two 15;  64 x 64  22   (two tiles a CU: they fill each other's waits)
  //     613 x 1024 -> 4096   64 x 128  9.0 (with GELU two buffers 9.9, three 10.2, four 13.4; in an
  //                          encoder, whose weights come from memory, two 13.1, three 11.3)  128 x 128  9.5  64 x 64  10.0
  //     613 x 4096 -> 1024   64 x 64  11.5 (four or six buffers change nothing)  128 x 128 19
  // Short rows are mostly results: two tiles a CU store while the other multiplies (256 x 256 / 128 x 128, two buffers):
  //   14500 x 512 -> 3530   51.8 / 43.1, with GELU 80.7 / 58.1;  16384 x 512 -> 4096 with GELU 82 / 71, x 768 94 / 97
  if (rows4 && tiles_of(64, 64) < (1 << 22)) {
    if (tiles_of(256, 256) >= 192 && a.k > 512) return tiled<OT, ACT, 256, 256, 2, 4, 2>(a, s);
    if (tiles_of(128, 128) > 256) return tiled<OT, ACT, 128, 128, 2, 4, 2>(a, s);
    if (tiles_of(128, 128) >= 224) return tiled<OT, ACT, 128, 128, 2, 4, 4>(a, s);
    if (tiles_of(64, 128) >= 256) return tiled<OT, ACT, 64, 128, 2, 4, 3>(a, s);
    return tiled<OT, ACT, 64, 64, 2, 2, 3>(a, s);
  }
  const int64_t tiles = tiles_of(64, 64);
  linear_any_kernel<OT><<<grid_of(tiles, 256 * kAnyGroups), 256 * kAnyGroups, 0, s>>>(a, (a.n + 63) / 64, tiles);
  return hipGetLastError();
}
template <int OT, int XT>
hipError_t fused(const LinearArgs& a, hipStream_t s) {
  const dim3 grid((a.n + 15) / 16);
  if (a.m == 1) linear_few_kernel<OT, 1, XT, true><<<grid, 64 * kFewWaves, 0, s>>>(a);
  else linear_few_kernel<OT, 1, XT, false><<<grid, 64 * kFewWaves, 0, s>>>(a);
  return hipGetLastError();
}
template <int OT>
hipError_t fused(int x_type, const LinearArgs& a, hipStream_t s) {
  return x_type == T_F32 ? fused<OT, T_F32>(a, s) : x_type == T_BF16 ? fused<OT, T_BF16>(a, s) : fused<OT, T_F16>(a, s);
}
}  // namespace

hipError_t launch_linear(const LinearArgs& a, hipStream_t s) {
  if (a.act) return a.out_type == T_F32 ? linear<T_F32, 1>(a, s) : a.out_type == T_BF16 ? linear<T_BF16, 1>(a, s) : linear<T_F16, 1>(a, s);
  return a.out_type == T_F32 ? linear<T_F32, 0>(a, s) : a.out_type == T_BF16 ? linear<T_BF16, 0>(a, s) : linear<T_F16, 0>(a, s);
}

// Inner sizes that are no multiple of 4, whose contiguous rows start between dwords: the tiled product of copies, where it saves
// more than they cost (int8 rows, GPU time, any sizes / copies and tiles). The choice is made by k, since the workspace's
// size depends on it and k is all that the function that tells it sees: rows of such a k that lie on dwords are copied too, and
// rows of another k that do not go to the kernel of any alignment.
//   613 x 4001 -> 1024   20.4 / 21.1 us     613 x 1307 -> 3637   25.1 / 21.1
//   16000 x 4001 -> 1024  249 / 93          2000 x 1307 -> 3637  57.8 / 27.6
// Floating-point rows are made with the padding, and the launch that makes them copies the weights beside them.
bool linear_repacks(int x_type, int64_t m, int n, int k) {
  const int64_t tiles = ((int64_t)n + 63) / 64 * ((m + 63) / 64);
  return k % 4 && m > kFewRows && tiles < (1 << 22) && m * n * k >= (x_type == T_I8 ? (int64_t)1 << 31 : 0);
}

hipError_t launch_repack(const int8_t* x, int64_t ldx, int64_t m, int8_t* to_x, const WeightCopy& copy, int k, hipStream_t s) {
  const int kp = (int)round_up(k, 16);
  const Repack one{x, ldx, m, to_x, k, kp}, two{copy.w, copy.ldw, copy.n, copy.to, k, kp};
  const int64_t blocks = one.blocks(256) + two.blocks(256);
  repack_kernel<<<grid_of(blocks, 256), 256, 0, s>>>(one, two, one.blocks(256), blocks);
  return hipGetLastError();
}

// One launch instead of two, as long as every workgroup's own conversion costs less than the second launch (bf16, GPU time
// alone): one row 4096 -> 1024 4.5 us against 7.1, eight rows 1024 -> 4096 4.8 against 6.2; but sixteen rows, two a wave, 7.6
// against 6.3 and two rows of 4096 8.9 against 7.2.
bool linear_fuses_rows(int64_t m, int k) { return k <= (m == 1 ? kFusedRow : kFusedWave) && m <= kFewWaves; }

hipError_t launch_linear_fused(int x_type, const LinearArgs& a, hipStream_t s) {
  return a.out_type == T_F32 ? fused<T_F32>(x_type, a, s) : a.out_type == T_BF16 ? fused<T_BF16>(x_type, a, s) : fused<T_F16>(x_type, a, s);
}

}  // namespace enc
}  // namespace rr
