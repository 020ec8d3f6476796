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


// ---- the tiled product -----------------------------------------------------------------------------------------------
// Workgroup tile: TN channels x TM rows, 128 bytes of k a step, both operands brought into LDS by the loads' LDS form (no
// registers, no ds_write), two buffers in turn: one barrier a step, the next step's loads in flight during this step's matrix
// instructions. Waves: WN x WM, each (TN / WN) x (TM / WM) in 32 x 32 x 32 instructions. LDS: rows of 128 bytes, the
// 16-byte column c of row r at column c ^ (r / 2 % 8): the 16 lanes that read a column of 16 rows at once meet all 64 banks.
// Wants rows at 16-byte addresses and k a multiple of 16 (the loads' unit); columns behind k and rows behind the end are out
// of the buffer's range and read as zeros.
constexpr int kStep = 128;

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
// every load of this wave has landed, its LDS reads are done, and so are the other waves'
__device__ __forceinline__ void step_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int OT, int ACT, int TN, int TM, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM, 2) void linear_tile_kernel(LinearArgs a, int tiles_n, int64_t tiles) {
  constexpr int kWaves = WN * WM, kN = TN / WN / 32, kM = TM / WM / 32;
  constexpr int kBuf = (TN + TM) * kStep, kLoadsN = TN * kStep / (1024 * kWaves), kLoadsM = TM * kStep / (1024 * kWaves);
  using O = typename Elem<OT>::type;
  constexpr int kOutLd = kN * 32 * sizeof(O) + 16;   // bytes of an output row in LDS
  constexpr int kLds = 2 * kBuf > kWaves * 32 * kOutLd ? 2 * kBuf : kWaves * 32 * kOutLd;
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
  const i32x4 bw = buffer_of(a.w + (int64_t)n0 * a.ldw, (unsigned)((rows_n - 1) * a.ldw + a.k));
  const i32x4 bx = buffer_of(a.x + m0 * a.ldx, (unsigned)((rows_m - 1) * a.ldx + a.k));

  // this lane's 16 bytes of load j: row 8 (j waves + wave) + lane / 8, LDS column lane % 8
  unsigned from_w[kLoadsN], from_x[kLoadsM];
  int col_w[kLoadsN], col_x[kLoadsM];
#pragma unroll
  for (int j = 0; j < kLoadsN; ++j) {
    const int r = 8 * (j * kWaves + wave) + lane / 8;
    col_w[j] = 16 * (lane % 8 ^ (r / 2 % 8));
    from_w[j] = (unsigned)(r * a.ldw + col_w[j]);
  }
#pragma unroll
  for (int j = 0; j < kLoadsM; ++j) {
    const int r = 8 * (j * kWaves + wave) + lane / 8;
    col_x[j] = 16 * (lane % 8 ^ (r / 2 % 8));
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
  const int row = lane % 32, half = lane / 32, swz = row / 2 % 8;
  fetch(0, 0);
  for (int c = threadIdx.x; c < TN; c += 64 * kWaves) {
    const int n = n0 + c < a.n ? n0 + c : a.n - 1;
    chan[0][c] = a.w_scale[n];
    chan[1][c] = a.bias ? a.bias[n] : 0.f;
  }
  int buf = 0;
  for (int k0 = 0; k0 < a.k; k0 += kStep, buf ^= 1) {
    step_barrier();
    if (k0 + kStep < a.k) fetch(k0 + kStep, buf ^ 1);
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
  }
  step_barrier();   // the buffers are free: each wave turns its results into rows there, 32 rows of x at a time
  char* out = lds + wave * 32 * kOutLd;
#pragma unroll
  for (int j = 0; j < kM; ++j) {
    const int64_t m = m0 + (wm * kM + j) * 32 + row;
    const float sx = a.x_scale[m < a.m ? m : a.m - 1];
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
        for (int x = 0; x < 4; ++x) v[x] = (O)activate((float)acc[i][j][4 * g + x] * (sx * sw[x]) + bias[x], ACT);
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

namespace {
template <int OT>
hipError_t linear(const LinearArgs& a, hipStream_t s) {
  auto tiles_of = [&](int tn, int tm) { return (((int64_t)a.n + tn - 1) / tn) * (((int64_t)a.m + tm - 1) / tm); };
  const bool rows16 = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | a.ldx | a.ldw | a.k) & 15) == 0 &&
                      a.ldx < (1 << 22) && a.ldw < (1 << 22);
  auto tile = [&](auto kernel, int tn, int tm, int threads) {
    const int64_t tiles = tiles_of(tn, tm);
    kernel<<<dim3((unsigned)tiles), threads, 0, s>>>(a, (a.n + tn - 1) / tn, tiles);
    return hipGetLastError();
  };
  if (rows16 && tiles_of(256, 256) < (1 << 22)) {
    if (tiles_of(256, 256) >= 192)
      return tile(a.act ? linear_tile_kernel<OT, 1, 256, 256, 2, 4> : linear_tile_kernel<OT, 0, 256, 256, 2, 4>, 256, 256, 512);
    if (tiles_of(128, 128) >= 96)
      return tile(a.act ? linear_tile_kernel<OT, 1, 128, 128, 2, 2> : linear_tile_kernel<OT, 0, 128, 128, 2, 2>, 128, 128, 256);
  }
  const int64_t tiles = tiles_of(64, 64);
  linear_any_kernel<OT><<<grid_of(tiles), 256, 0, s>>>(a, (a.n + 63) / 64, tiles);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_linear(const LinearArgs& a, hipStream_t s) {
  return a.out_type == T_F32 ? linear<T_F32>(a, s) : a.out_type == T_BF16 ? linear<T_BF16>(a, s) : linear<T_F16>(a, s);
}

}  // namespace enc
}  // namespace rr
