// rr_encoder_attn.hip — attention of queries to an encoder's states (rr_cross_attention).
//
// One pass over a sequence's keys with the running maximum m and sum l of the softmax (in powers of two: the scores are
// scaled by scale * log2 e), S^T = K Q^T and O^T = V^T P^T: in both products a lane's column is one query, so the softmax
// weights a lane computes are the ones the second product takes from it, and no value changes lanes between the two.
#include "rr_encoder_device.h"

namespace rr {
namespace enc {
namespace {

constexpr int kRows = 16;   // query rows of a tile: (query, head of the key head's group) pairs

struct AttnParams {
  AttnArgs a;
  float c;          // |scale| * log2 e
  bool flip;        // scale below 0: the queries change sign instead, so that larger scores are larger here too
  unsigned group;   // heads per key head
  unsigned tiles;   // row tiles of a key head the launch was sized for
  unsigned units;   // tiles * key heads * batch
  unsigned splits;  // pieces of the keys, each a workgroup's; joined by attn_join_kernel when more than one
};

struct Span {
  int64_t first;    // packed row, 0 for dense
  int n;
};
// (the same for a whole wave, and known to the compiler as such: what follows from them stays in scalar registers)
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Span span_of(const int32_t* offsets, int64_t total, int b) {
  int64_t lo = uniform(offsets[b]), hi = uniform(offsets[b + 1]);
  lo = lo < 0 ? 0 : lo > total ? total : lo;
  hi = hi < lo ? lo : hi > total ? total : hi;
  return {lo, (int)(hi - lo)};
}
__device__ __forceinline__ Span queries_of(const AttnArgs& a, int b) {
  return a.q_offsets ? span_of(a.q_offsets, a.total_q, b) : Span{0, a.max_q};
}
__device__ __forceinline__ Span keys_of(const AttnArgs& a, int b) {
  Span s = a.k_offsets ? span_of(a.k_offsets, a.total_k, b) : Span{0, a.max_k};
  if (a.key_lengths) {
    const int len = uniform(a.key_lengths[b]);
    s.n = len < 0 ? 0 : len < s.n ? len : s.n;
  }
  return s;
}

// Keys of a mask's row up to the last one that takes part: a padded batch's masks end long before their rows do, and a step
// without keys costs a wave nearly what one with keys waits for. 1024 keys at a time from the end, 16 a lane, as dwords
// (none that holds no byte of the row).
__device__ __forceinline__ int mask_end(const uint8_t* mask, int n) {
  const int lane = threadIdx.x & 63, sh = (int)(reinterpret_cast<uintptr_t>(mask) & 3);   // byte 0 of the row in the buffer
  const auto row = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(mask - sh), 0, (sh + n + 3) & ~3, 0x00020000);
  for (int c0 = n > 0 ? (sh + n - 1) & ~1023 : -1; c0 >= 0; c0 -= 1024) {
    const int at = c0 + 16 * lane;
    const u32x4 bytes = __builtin_amdgcn_raw_buffer_load_b128(row, at, 0, 0);
    int last = -1;   // this lane's last byte that is set, counted in the buffer
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int left = sh + n - (at + 4 * j);   // bytes of this dword before the row's end
      unsigned v = left >= 4 ? bytes[j] : left <= 0 ? 0u : bytes[j] & ((1u << 8 * left) - 1);
      if (at + 4 * j < sh) v &= ~0u << 8 * sh;
      if (v) last = at + 4 * j + (31 - __builtin_clz(v)) / 8;
    }
    const uint64_t any = __ballot(last >= 0);
    if (any) return __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(any)) - sh + 1;
  }
  return 0;
}

// Rows [first, first + count) of a tensor whose rows lie `ts` elements apart, as a buffer: reads behind the last row's end give
// zeros, so that no lane has to ask whether its key is there, and 32-bit offsets reach every row of a block of keys (the
// caller keeps ts below 2^23).
template <class E>
struct RowBuffer {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ RowBuffer(const E* base, int64_t ts, int first, int count, int d)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(base + first * ts), 0,
                                            count > 0 ? (int)(((count - 1) * (int)ts + d) * (int)sizeof(E)) : 0, 0x00020000)) {}
  template <int BYTES>
  __device__ __forceinline__ auto load(unsigned at) const {
    if constexpr (BYTES == 16) return __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0);
    else if constexpr (BYTES == 8) return __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0);
    else return __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
  }
  // 16 bytes a lane to LDS address `to` + 16 * lane
  __device__ __forceinline__ void to_lds(unsigned at, unsigned to) const {
    unsigned keep;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
        : "=&s"(keep)
        : "v"(at), "s"(r), "s"(to)
        : "memory");
  }
};
constexpr unsigned kNowhere = 0xfffffff0u;   // an offset behind every buffer

// ---- the two products of one wave over a block of keys ------------------------------------------------------------
// Lane (i = lane % 16, g = lane / 16). DP: the head size rounded up to a whole tile.
template <int TY, int DP> struct Core;

// Two 16-bit values with infinities (and NaNs) as the largest finite number: what the second part of a weight multiplies, which
// may be 0 or of the other sign and would make a NaN of the infinity that the first part's product has.
template <int TY>
__device__ __forceinline__ unsigned finite2(unsigned v) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  constexpr unsigned short kMost = TY == T_BF16 ? 0x7f7f : 0x7bff;
  const s16x2 up = __builtin_elementwise_min(__builtin_bit_cast(s16x2, v), s16x2{(short)kMost, (short)kMost});
  constexpr unsigned short kLeast = kMost | 0x8000;
  return __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(u16x2, up), u16x2{kLeast, kLeast}));
}
template <int TY>
__device__ __forceinline__ u32x4 finite8(u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = finite2<TY>(v[i]);
  return v;
}

// 16-bit types: 32 keys a block. Lane i, g holds the scores of query i with keys 4g + r and 16 + 4g + r (r < 4): the eight
// keys that its slots 8g .. 8g + 7 of the second product's contraction stand for.
template <int TY, int DP>
struct Core16 {
  static constexpr int kKeys = 32, kMine = 8, kTiles = DP / 16, kSteps = DP / 32;
  static constexpr int kRun = kTiles;
  static constexpr int VW = DP / 16;   // values of a V row a lane loads: tile t's row i is dimension VW i + t
  using E = typename Elem<TY>::type;
  typedef E e8 __attribute__((ext_vector_type(8)));
  struct Keys {   // a block's keys and values, on their way or there
    u32x4 k[2][kSteps];
    unsigned v[8][VW / 2];
  };
  u32x4 q[kSteps];

  static __device__ __forceinline__ int key(int g, int j) { return (j < 4 ? 0 : 12) + 4 * g + j; }
  static __device__ __forceinline__ int dim(int t, int i) { return VW * i + t; }
  static __device__ __forceinline__ f32x4 mma(u32x4 x, u32x4 y, f32x4 c) {
    if constexpr (TY == T_BF16)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
  }
  __device__ __forceinline__ void load_q(const E* row, bool there, bool flip, int d, int g) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      q[s] = u32x4{0, 0, 0, 0};
      if (there && 32 * s + 8 * g < d) q[s] = load_as<u32x4>(row + 32 * s + 8 * g);
      if (flip) q[s] ^= 0x80008000u;
    }
  }
  // byte offsets in a block: of this lane's part of K rows 0 .. 15 (+ 32 bytes a step) and of V rows 4g (+ a row each)
  static __device__ __forceinline__ unsigned k_offset(unsigned ts, int i, int g) { return 2 * (i * ts + 8 * g); }
  static __device__ __forceinline__ unsigned v_offset(unsigned ts, int i, int g, int d) {
    return VW * i < d ? 2 * (4 * g * ts + VW * i) : kNowhere;
  }
  static __device__ __forceinline__ void load_k(Keys& to, const RowBuffer<E>& k, unsigned at, unsigned ts, int d, int g) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        to.k[h][s] = k.template load<16>(32 * s + 32 <= d || 32 * s + 8 * g < d ? at + 32 * h * ts + 64 * s : kNowhere);
  }
  // (ts: 0 in lanes that have no part of a row, which stay at kNowhere)
  static __device__ __forceinline__ void load_v(Keys& to, const RowBuffer<E>& v, unsigned at, unsigned ts) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const auto x = v.template load<2 * VW>(at + 2 * key(0, j) * ts);
#pragma unroll
      for (int p = 0; p < VW / 2; ++p) {
        if constexpr (VW == 2) to.v[j][p] = x;
        else to.v[j][p] = x[p];
      }
    }
  }
  __device__ __forceinline__ void scores(const Keys& of, float* s) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 c = {0, 0, 0, 0};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) c = mma(of.k[h][st], q[st], c);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[4 * h + r] = c[r];
    }
  }
  // valid: bit j says whether key j of this lane takes part; the V rows of the others may hold anything and become zeros
  static __device__ __forceinline__ void accumulate(Keys& of, const float* p, unsigned valid, f32x4* acc) {
    e8 pe, rest;   // the weights in two parts, as kFewRows' kernel takes them
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      pe[j] = (E)p[j];
      rest[j] = (E)(p[j] - (float)pe[j]);
    }
    const u32x4 pb = __builtin_bit_cast(u32x4, pe), pr = __builtin_bit_cast(u32x4, rest);
    if (valid != 0xffu) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int w = 0; w < VW / 2; ++w) of.v[j][w] = (valid >> j & 1) ? of.v[j][w] : 0u;
    }
#pragma unroll
    for (int w = 0; w < VW / 2; ++w) {
      u32x4 lo, hi;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        lo[x] = __builtin_amdgcn_perm(of.v[2 * x + 1][w], of.v[2 * x][w], 0x05040100u);
        hi[x] = __builtin_amdgcn_perm(of.v[2 * x + 1][w], of.v[2 * x][w], 0x07060302u);
      }
      acc[2 * w] = mma(finite8<TY>(lo), pr, mma(lo, pb, acc[2 * w]));
      acc[2 * w + 1] = mma(finite8<TY>(hi), pr, mma(hi, pb, acc[2 * w + 1]));
    }
  }
};
template <int DP> struct Core<T_BF16, DP> : Core16<T_BF16, DP> {};
template <int DP> struct Core<T_F16, DP> : Core16<T_F16, DP> {};

// fp32: 16 keys a block, contractions of four; lane i, g holds the scores of query i with keys 4g + r.
template <int DP>
struct Core<T_F32, DP> {
  // a V row's dimensions: kWide times 64, of which a lane loads four, then kPair times 32, of which it loads two
  static constexpr int kKeys = 16, kMine = 4, kTiles = DP / 16, kSteps = DP / 16, kWide = DP / 64, kPair = DP / 32 % 2;
  static constexpr int kRun = 4;
  using E = float;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  struct Keys {
    f32x4 k[kSteps], v[4][kWide ? kWide : 1];
    f32x2 pair[kPair ? 4 : 1];
  };
  f32x4 q[kSteps];

  static __device__ __forceinline__ int key(int g, int j) { return 4 * g + j; }
  static __device__ __forceinline__ int dim(int t, int i) {
    return t < 4 * kWide ? 64 * (t / 4) + 4 * i + t % 4 : 64 * kWide + 2 * i + t % 2;
  }
  __device__ __forceinline__ void load_q(const float* row, bool there, bool flip, int d, int g) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      q[s] = f32x4{0, 0, 0, 0};
      if (there && 16 * s + 4 * g < d) q[s] = load_as<f32x4>(row + 16 * s + 4 * g);
      if (flip) q[s] = -q[s];
    }
  }
  static __device__ __forceinline__ unsigned k_offset(unsigned ts, int i, int g) { return 4 * (i * ts + 4 * g); }
  static __device__ __forceinline__ unsigned v_offset(unsigned ts, int i, int g, int d) { return 4 * (4 * g * ts + 4 * i); }
  static __device__ __forceinline__ void load_k(Keys& to, const RowBuffer<float>& k, unsigned at, unsigned ts, int d, int g) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      to.k[s] = __builtin_bit_cast(f32x4, k.load<16>(16 * s + 16 <= d || 16 * s + 4 * g < d ? at + 64 * s : kNowhere));
  }
  // (columns behind d are the next head's: they end up in columns of the result that are not stored)
  static __device__ __forceinline__ void load_v(Keys& to, const RowBuffer<float>& v, unsigned at, unsigned ts) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int w = 0; w < kWide; ++w) to.v[j][w] = __builtin_bit_cast(f32x4, v.load<16>(at + 4 * j * ts + 256 * w));
    if constexpr (kPair)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        to.pair[j] = __builtin_bit_cast(f32x2, v.load<8>(at - 8 * (threadIdx.x & 15) + 4 * j * ts + 256 * kWide));
  }
  __device__ __forceinline__ void scores(const Keys& of, float* s) const {
    f32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int x = 0; x < 4; ++x) c = __builtin_amdgcn_mfma_f32_16x16x4f32(of.k[st][x], q[st][x], c, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = c[r];
  }
  static __device__ __forceinline__ void accumulate(Keys& of, const float* p, unsigned valid, f32x4* acc) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const float x = t < 4 * kWide ? of.v[j][t < 4 * kWide ? t / 4 : 0][t % 4] : of.pair[kPair ? j : 0][t % 2];
        const float v = (valid >> j & 1) ? x : 0.f;
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[j], acc[t], 0, 0, 0);
      }
  }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The softmax's weights are 2^(c score - m). The reference m follows the running maximum: it moves when a score passes it by
// kTop + kLag, and then to kTop below that score, so that a row's largest weight is at least 2^kTop and none above 2^(kTop + kLag).
// Near 1 is right for types with fp32's exponents. fp16 weights begin at 2^13 and stay below its largest, 2^16: steps relative to
// the weight reach down to 2^-14, 27 powers of two (18.7 nats) below the largest; what is smaller still is off by 2^-38 of it.
template <int TY> constexpr float kTop = TY == T_F16 ? 13.f : 0.f;
template <int TY> constexpr float kLag = TY == T_F16 ? 2.9f : 8.f;
template <int TY>
__device__ __forceinline__ bool passes(float top, float m) { return top - m > kTop<TY> + kLag<TY>; }   // (an exact difference)
template <int TY>
__device__ __forceinline__ float moved(float m, float top) {
  float to = top - kTop<TY>;
  if (kTop<TY> != 0.f && passes<TY>(top, to)) to = top;   // (a score so large that the difference was rounded)
  return fmaxf(m, to);
}
// Scores whose next fp32 number is far away are rounded to powers of two before the reference is taken off. In one step with the
// subtraction they would keep what the reference lost to its rounding, which at 2^28 overflows fp16 and at 2^32 fp32.
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) >= 0x1p20f && m != -INFINITY; }
__device__ __forceinline__ float in_powers(float s, float c) {
#pragma clang fp contract(off)
  return s * c;
}

// where the row's results go, null if the row is not there
template <class E>
__device__ __forceinline__ E* out_row(const AttnParams& p, const Span& sq, int b, int kvh, unsigned row) {
  const AttnArgs& a = p.a;
  const unsigned qi = row / p.group, h = kvh * p.group + row % p.group;
  if ((int)qi >= sq.n) return nullptr;
  return static_cast<E*>(a.out) + (a.q_offsets ? sq.first * a.o_ts : b * a.o_bs) + qi * a.o_ts + h * a.o_hs;
}

// A row of sums times `scale`, dimensions below d (a multiple of 8)
template <class C>
__device__ __forceinline__ void store_row(typename C::E* to, const f32x4* acc, float scale, int d, int g) {
  using E = typename C::E;
  // tiles whose rows are neighbouring dimensions; kLeft: the narrower run of fp32's last two
  constexpr int kRun = C::kRun, kLeft = C::kTiles % kRun;
  typedef E run __attribute__((ext_vector_type(kRun)));
  typedef E left __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int t = 0; t < C::kTiles - kLeft; t += kRun) {
      run v;
#pragma unroll
      for (int x = 0; x < kRun; ++x) v[x] = (E)(acc[t + x][r] * scale);
      const int at = C::dim(t, 4 * g + r);
      if (at < d) store_as(to + at, v);
    }
    if constexpr (kLeft != 0) {
      const int at = C::dim(C::kTiles - 2, 4 * g + r);
      const left v = {(E)(acc[C::kTiles - 2][r] * scale), (E)(acc[C::kTiles - 1][r] * scale)};
      if (at < d) store_as(to + at, v);
    }
  }
}

// Tiles of 16 query rows. WK = 1: four tiles a workgroup, a wave each, which takes all keys of its own; nothing is shared. WK
// waves: one tile and one piece of the keys a workgroup, each wave every WK-th block of keys, their sums joined in LDS. Either
// way a wave has its next block of keys on the way while it works on one, straight from memory into registers.
// Short sequences and fp32. 32 x 20 queries x 20 keys, 16 heads of 64: bf16 4.2 us, fp32 6.1 (a launch and the latencies of
// offsets, rows and result); fp32 41 x 70 x 1668, 16 heads of 32: 178 us, 55 TFLOP/s; fp32 one query x 16384 keys x 4, 16 heads
// of 128: 184 us, 5.8 TB/s.
template <int TY, int DP, int WK>
__global__ __launch_bounds__(WK == 1 ? 256 : 64 * WK) void attn_rows_kernel(AttnParams p) {
  using C = Core<TY, DP>;
  using E = typename C::E;
  constexpr int kLd = DP + 4;
  __shared__ float so[WK == 1 ? 1 : WK][kRows][kLd];
  __shared__ float sm[WK][kRows], sl[WK][kRows];
  const AttnArgs& a = p.a;
  const int lane = threadIdx.x & 63, first = uniform(threadIdx.x >> 6), wave = WK == 1 ? 0 : first, i = lane & 15, g = lane >> 4;
  const unsigned unit = WK == 1 ? blockIdx.x * 4 + first : blockIdx.x / p.splits;
  const int split = WK == 1 ? 0 : blockIdx.x % p.splits;
  if (unit >= p.units) return;
  const int tile0 = unit % p.tiles, kvh = unit / p.tiles % a.kv_heads, b = unit / p.tiles / a.kv_heads;
  const Span sq = queries_of(a, b);
  Span sk = keys_of(a, b);
  const int rows = sq.n * p.group;
  const E* kbase = static_cast<const E*>(a.k) + (a.k_offsets ? sk.first * a.k_ts : b * a.k_bs) + kvh * a.k_hs;
  const E* vbase = static_cast<const E*>(a.v) + (a.k_offsets ? sk.first * a.v_ts : b * a.v_bs) + kvh * a.v_hs;
  const uint8_t* mask = a.key_mask ? a.key_mask + b * a.mask_stride : nullptr;
  if (mask) sk.n = mask_end(mask, sk.n);

  // tiles behind the ones the launch was sized for (a sequence longer than max_q) take all keys in one piece
  const unsigned k_ts = (unsigned)a.k_ts, v_ts = (unsigned)a.v_ts;
  const unsigned k_at = C::k_offset(k_ts, i, g), v_at = C::v_offset(v_ts, i, g, a.d), v_step = v_at == kNowhere ? 0 : v_ts;
  for (int tile = tile0; tile < (rows + kRows - 1) / kRows; tile += p.tiles) {
    const bool whole = p.splits == 1 || tile >= (int)p.tiles;
    if (whole && split) break;
    const int pieces = whole ? 1 : p.splits;
    C core;
    {
      const unsigned row = tile * kRows + i, qi = row / p.group, h = kvh * p.group + row % p.group;
      const E* q = static_cast<const E*>(a.q) + (a.q_offsets ? sq.first * a.q_ts : b * a.q_bs) + qi * a.q_ts + h * a.q_hs;
      core.load_q(q, (int)qi < sq.n, p.flip, a.d, g);
    }
    f32x4 acc[C::kTiles] = {};
    float m = -INFINITY, l = 0.f;
    bool far = false;   // (of the whole wave)
    struct Block {
      typename C::Keys keys;
      unsigned char there;   // of key `lane`, if there is a mask
    } one, two;
    auto load = [&](Block& to, int kb) {
      to.there = 1;
      if (mask) to.there = mask[kb + lane < sk.n ? kb + lane : sk.n - 1];
      const int n = sk.n - kb < C::kKeys ? sk.n - kb : C::kKeys;
      C::load_k(to.keys, RowBuffer<E>(kbase, a.k_ts, kb, n, a.d), k_at, k_ts, a.d, g);
      C::load_v(to.keys, RowBuffer<E>(vbase, a.v_ts, kb, n, a.d), v_at, v_step);
    };
    auto take = [&](Block& of, int kb) {
      const uint64_t all = __ballot(kb + lane < sk.n && of.there);
      unsigned valid = 0;
#pragma unroll
      for (int j = 0; j < C::kMine; ++j) valid |= (unsigned)(all >> C::key(g, j) & 1) << j;
      float s[C::kMine];
      core.scores(of.keys, s);
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < C::kMine; ++j) {
        s[j] = (valid >> j & 1) ? s[j] : -INFINITY;
        top = fmaxf(top, s[j]);
      }
      top = in_powers(top, p.c);
      if (__any(passes<TY>(top, m))) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = moved<TY>(m, top);
        const float f = to == m ? 1.f : exp2_fast(m - to);
        m = to;
        far = __any(is_far(m));
        l *= f;
#pragma unroll
        for (int t = 0; t < C::kTiles; ++t) acc[t] *= f;
      }
      const float ref = m == -INFINITY ? 0.f : m, c = far ? 1.f : p.c;
      if (far)
#pragma unroll
        for (int j = 0; j < C::kMine; ++j) s[j] = in_powers(s[j], p.c);
      float w[C::kMine];
#pragma unroll
      for (int j = 0; j < C::kMine; ++j) {
        w[j] = exp2_fast(fmaf(s[j], c, -ref));
        l += w[j];
      }
      C::accumulate(of.keys, w, valid, acc);
    };
    const int step = pieces * WK * C::kKeys;
    int kb = (split * WK + wave) * C::kKeys;
    if (kb < sk.n) load(one, kb);
    for (; kb < sk.n; kb += 2 * step) {
      const int next = kb + step, after = next + step;
      if (next < sk.n) load(two, next);
      take(one, kb);
      if (next >= sk.n) break;
      if (after < sk.n) load(one, after);
      take(two, next);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if constexpr (WK == 1) {
      E* to = out_row<E>(p, sq, b, kvh, tile * kRows + i);
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      if (to) store_row<C>(to, acc, inv, a.d, g);
    } else {
      __syncthreads();   // (a tile before this one may still be read)
#pragma unroll
      for (int t = 0; t < C::kTiles; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) so[wave][i][C::dim(t, 4 * g + r)] = acc[t][r];
      if (g == 0) {
        sm[wave][i] = m;
        sl[wave][i] = l;
      }
      __syncthreads();
      float* ws = whole ? nullptr : a.ws + ((int64_t)unit * p.splits + split) * kRows * (DP + 2);
      for (int x = threadIdx.x; x < kRows * DP; x += 64 * WK) {
        const int row = x / DP, d = x % DP;
        float top = sm[0][row];
#pragma unroll
        for (int w = 1; w < WK; ++w) top = fmaxf(top, sm[w][row]);
        float o = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float f = sm[w][row] == top ? 1.f : exp2_fast(sm[w][row] - top);
          o += f * so[w][row][d];
          sum += f * sl[w][row];
        }
        if (whole) {
          E* to = out_row<E>(p, sq, b, kvh, tile * kRows + row);
          if (to && d < a.d) to[d] = (E)(sum == 0.f ? 0.f : o / sum);
        } else {
          ws[2 * kRows + x] = o;
          if (d == 0) {
            ws[row] = top;
            ws[kRows + row] = sum;
          }
        }
      }
    }
  }
}

// ---- 16-bit types, keys through LDS -----------------------------------------------------------------------------------
// A workgroup of four waves brings a step's K and V rows into LDS (whole rows at a time, two buffers: one barrier a step, the
// next step's rows are on their way during this one) and multiplies them in 32 x 32 x 16 instructions, 32 query rows and 32
// keys at a time. WK = 1: 128 query rows, 32 a wave; every wave takes every key, 64 a step. WK = 4: 32 query rows, of which
// every wave takes another 32 of 128 keys a step, and their sums are joined in LDS: for few rows, where bandwidth counts.
// Keys that do not take part are read as zeros, whatever they held. Lane (i = lane % 32, half = lane / 32) holds the scores
// of query i with keys 8 (r / 4) + 4 half + r % 4 of a 32-key block, r < 16; eight of them in a row (r / 8 = t) are its slots
// of the second product's 16-key contraction t. V lies in LDS as in memory; the transposing LDS read hands each lane four keys
// of one dimension. The weights enter the second product rounded to the type: off by at most half a step of each, which is half
// a step of sum p |v| in the result, while their sum and the statistics are of the unrounded ones in fp32. Few rows, which
// wait for memory and not for arithmetic, add what the rounding left in a product of its own (small fp16 rests in steps of 2^-24);
// for many rows it costs more than the precision is worth: 32 x 512 x 512 by mask 46 -> 62 us.
// DMA: rows at 16-byte addresses go to LDS by the loads themselves; others through registers.
// WK = 4 is bound by bandwidth: one query x 65536 keys x 4, 32 heads over 8 of 128, bf16: 199 us, 5.4 TB/s; x 40 to 512 keys x 32,
// 16 heads of 64: 12.4 us (a launch and four steps' latency). WK = 1 is bound by the softmax's instructions (a 32-key block's 16 exponentials, multiply-adds and
// sums a lane take longer than its eight matrix instructions): 32 x 512 x 512, 16 heads of 64, bf16: 53 us, 650 TFLOP/s, of
// which 19 are there with 64 keys too (queries in, results out, latencies); 8 x 2048 x 2048, 16 heads of 128: 300 us, 915
// TFLOP/s. fp16, whose reference moves more often: 56 and 322 us.
// Four workgroups a CU at 128 registers a wave (32 keys at a time) beat two with 64 at a time (54 against 68 us).
constexpr int kTileRows = 128, kFewRows = 32;

// The 16-byte column of key row r that lies at column c of its LDS row (and the other way round): the 16 lanes that read a
// column of 16 K rows at once, and the 32 lanes that read 64 bytes of four V rows at once, each meet all 64 banks.
template <int DP>
__device__ __forceinline__ unsigned k_column(unsigned r, unsigned c) {
  constexpr unsigned kCols = DP / 8, kPerCycle = 16 / kCols;
  return c ^ (r / kPerCycle % kCols);
}
template <int DP>
__device__ __forceinline__ unsigned v_column(unsigned r, unsigned c) {
  return DP == 128 ? c ^ 4 * (r % 4) : DP == 64 ? c ^ 4 * (r / 2 % 2) : c;
}

template <int TY>
__device__ __forceinline__ f32x16 mma32(u32x4 x, u32x4 y, f32x16 c) {
  if constexpr (TY == T_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}
__device__ __forceinline__ u32x2 read_transposed(const char* lds) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lds));
}

template <int TY, int DP, int WK, bool DMA>
__global__ __launch_bounds__(256, DP == 128 ? 2 : 4) void attn_tile_kernel(AttnParams p) {
  using E = typename Elem<TY>::type;
  typedef E e8 __attribute__((ext_vector_type(8)));
  constexpr int kRowsHere = WK == 1 ? kTileRows : kFewRows, kKeys = WK == 1 ? 64 : 128, kWords = kKeys / 64;
  constexpr int kCols = DP / 8, kLoads = kKeys * kCols / 256, kHalf = kKeys * DP * 2, kBuf = 2 * kHalf;
  constexpr int kLd = DP + 4;
  constexpr int kJoin = WK == 1 ? 0 : WK * kFewRows * (kLd + 2) * 4;
  __shared__ __align__(1024) char lds[2 * kBuf > kJoin ? 2 * kBuf : kJoin];
  const AttnArgs& a = p.a;
  // Workgroups go to the 8 XCDs in turn: those of one key head, which read the same keys, stay in one XCD's cache
  // (where the heads divide evenly).
  const unsigned each = p.tiles * p.splits, heads = p.units / p.tiles;
  const unsigned at = heads % 8 ? blockIdx.x : (blockIdx.x / 8 / each * 8 + blockIdx.x % 8) * each + blockIdx.x / 8 % each;
  const int split = at % p.splits, tile0 = at / p.splits % p.tiles;
  const int kvh = at / each % a.kv_heads, b = at / each / a.kv_heads;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), i = lane & 31, half = lane >> 5;
  const Span sq = queries_of(a, b);
  Span sk = keys_of(a, b);
  const int rows = sq.n * p.group;
  const E* kbase = static_cast<const E*>(a.k) + (a.k_offsets ? sk.first * a.k_ts : b * a.k_bs) + kvh * a.k_hs;
  const E* vbase = static_cast<const E*>(a.v) + (a.k_offsets ? sk.first * a.v_ts : b * a.v_bs) + kvh * a.v_hs;
  const uint8_t* mask = a.key_mask ? a.key_mask + b * a.mask_stride : nullptr;
  if (mask) sk.n = mask_end(mask, sk.n);
  // A step's keys as bits. The mask's bytes are asked for two steps ahead, before that step's rows, so that nothing waits
  // for more than the bytes themselves.
  struct Bytes {
    unsigned char there[kWords];
  };
  struct Bits {
    uint64_t word[kWords];
  };
  auto bytes_of = [&](int kb) {
    Bytes r;
#pragma unroll
    for (int w = 0; w < kWords; ++w) r.there[w] = mask && kb + 64 * w + lane < sk.n ? mask[kb + 64 * w + lane] : 1;
    return r;
  };
  auto bits_of = [&](int kb, const Bytes& of) {
    Bits r;
#pragma unroll
    for (int w = 0; w < kWords; ++w) r.word[w] = __ballot(kb + 64 * w + lane < sk.n && of.there[w]);
    return r;
  };
  // this lane's 16 bytes of load j: key row (4 j + wave) 64 / kCols + lane / kCols, at LDS column lane % kCols
  const unsigned r0 = wave * (64 / kCols) + lane / kCols, c0 = lane % kCols;
  constexpr unsigned kApart = 256 / kCols;   // (a multiple of the swizzles' periods: the columns are the same for every j)
  const unsigned ck = k_column<DP>(r0, c0), cv = v_column<DP>(r0, c0);
  const unsigned from_k = 2 * (r0 * (unsigned)a.k_ts + 8 * ck), from_v = 2 * (r0 * (unsigned)a.v_ts + 8 * cv);
  const bool in_k = (int)(8 * ck) < a.d, in_v = (int)(8 * cv) < a.d;
  const unsigned lds0 = (unsigned)(uintptr_t)lds;

  for (int tile = tile0; tile < (rows + kRowsHere - 1) / kRowsHere; tile += p.tiles) {
    const bool whole = p.splits == 1 || tile >= (int)p.tiles;
    if (whole && split) break;
    const int pieces = whole ? 1 : p.splits;
    const unsigned row = tile * kRowsHere + (WK == 1 ? wave * 32 : 0) + i;
    const bool busy = WK > 1 || tile * kRowsHere + wave * 32 < rows;   // (of this wave)
    u32x4 kr[DMA ? 1 : kLoads], vr[DMA ? 1 : kLoads];
    auto fetch = [&](int kb, const Bits& bits, int buf) {
      const int n = sk.n - kb < kKeys ? sk.n - kb : kKeys;
      const RowBuffer<E> k(kbase, a.k_ts, kb, n, a.d), v(vbase, a.v_ts, kb, n, a.d);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const unsigned r = r0 + kApart * j;
        const bool there = (kWords == 1 || 64 / kCols * (4 * j + wave) < 64 ? bits.word[0] : bits.word[kWords - 1]) >> (r % 64) & 1;
        const unsigned at_k = there && in_k ? from_k + 2 * kApart * j * (unsigned)a.k_ts : kNowhere;
        const unsigned at_v = there && in_v ? from_v + 2 * kApart * j * (unsigned)a.v_ts : kNowhere;
        if constexpr (DMA) {
          const unsigned to = lds0 + buf * kBuf + (4 * j + wave) * 1024;
          k.to_lds(at_k, to);
          v.to_lds(at_v, to + kHalf);
        } else {
          kr[j] = k.template load<16>(at_k);
          vr[j] = v.template load<16>(at_v);
        }
      }
    };
    auto keep = [&](int buf) {
      if constexpr (!DMA)
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          char* to = lds + buf * kBuf + (4 * j + wave) * 1024 + lane * 16;
          *reinterpret_cast<u32x4*>(to) = kr[j];
          *reinterpret_cast<u32x4*>(to + kHalf) = vr[j];
        }
    };
    const int step = pieces * kKeys;
    int kb = split * kKeys, buf = 0;
    Bytes ahead = bytes_of(kb + step);
    Bits valid = bits_of(kb, bytes_of(kb));
    u32x4 q[DP / 16];
    {
      const unsigned qi = row / p.group, h = kvh * p.group + row % p.group;
      const E* from = static_cast<const E*>(a.q) + (a.q_offsets ? sq.first * a.q_ts : b * a.q_bs) + qi * a.q_ts + h * a.q_hs;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        q[s] = u32x4{0, 0, 0, 0};
        if ((int)qi < sq.n && 16 * s + 8 * half < a.d) q[s] = load_as<u32x4>(from + 16 * s + 8 * half);
      }
    }
    if (kb < sk.n) {
      fetch(kb, valid, 0);
      keep(0);
    }
    if (p.flip)
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) q[s] ^= 0x80008000u;
    f32x16 acc[DP / 32] = {};
    float m = -INFINITY, l = 0.f;
    bool far = false;   // (of the whole wave)
    // 32 keys of the buffer, rows key0 and on, `here` those that take part
    auto take = [&](const char* k_rows, int key0, unsigned here) {
      // K is read before the first product, V before the softmax that its product waits for: the reads' latency is hidden
      // behind arithmetic, not met once for each instruction
      u32x4 kf[DP / 16];
#pragma unroll
      for (int st = 0; st < DP / 16; ++st) {
        const unsigned r = key0 + i;
        kf[st] = *reinterpret_cast<const u32x4*>(k_rows + (r * kCols + k_column<DP>(r, 2 * st + half)) * 16);
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x16 s = {};
#pragma unroll
      for (int st = 0; st < DP / 16; ++st) s = mma32<TY>(kf[st], q[st], s);
      u32x4 vf[2][DP / 32];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
          const unsigned r = key0 + 16 * t + 4 * half + i % 16 / 4, c = 4 * dt + 2 * (i / 16) + i % 4 / 2;
          const char* v_rows = k_rows + kHalf + 8 * (i % 2);
          const u32x2 lo = read_transposed(v_rows + (r * kCols + v_column<DP>(r, c)) * 16);
          const u32x2 hi = read_transposed(v_rows + ((r + 8) * kCols + v_column<DP>(r + 8, c)) * 16);
          vf[t][dt] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      __builtin_amdgcn_sched_barrier(0);
      if (here != ~0u) {
        const unsigned mine = here >> 4 * half;   // bits 8 (r / 4) + r % 4
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (mine >> (8 * (r / 4) + r % 4) & 1) ? s[r] : -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
      top = in_powers(top, p.c);
      if (__any(passes<TY>(top, m))) {
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = moved<TY>(m, top);
        const float f = to == m ? 1.f : exp2_fast(m - to);
        m = to;
        far = __any(is_far(m));
        l *= f;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) acc[t] *= f;
      }
      const float ref = m == -INFINITY ? 0.f : m, c = far ? 1.f : p.c;
      if (far)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = in_powers(s[r], p.c);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        e8 w, rest;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float e = exp2_fast(fmaf(s[8 * t + x], c, -ref));
          l += e;
          w[x] = (E)e;
          if constexpr (WK > 1) rest[x] = (E)(e - (float)w[x]);
        }
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
          acc[dt] = mma32<TY>(vf[t][dt], __builtin_bit_cast(u32x4, w), acc[dt]);
          if constexpr (WK > 1) acc[dt] = mma32<TY>(finite8<TY>(vf[t][dt]), __builtin_bit_cast(u32x4, rest), acc[dt]);
        }
      }
    };
    for (; kb < sk.n; kb += step, buf ^= 1) {
      if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // (this step's rows are in LDS)
      else __syncthreads();
      const bool more = kb + step < sk.n;
      const Bits next = bits_of(kb + step, ahead);
      if (more) {
        ahead = bytes_of(kb + 2 * step);
        fetch(kb + step, next, buf ^ 1);   // (last read before the barrier above)
      }
      const char* k_rows = lds + buf * kBuf;
      if constexpr (WK == 1) {
        if (busy)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (const unsigned here = (unsigned)(valid.word[0] >> 32 * h)) take(k_rows, 32 * h, here);
      } else {
        const unsigned here = (unsigned)((wave < 2 ? valid.word[0] : valid.word[kWords - 1]) >> 32 * (wave % 2));
        if (here) take(k_rows, 32 * wave, here);
      }
      if (more) keep(buf ^ 1);
      valid = next;
    }
    __syncthreads();   // (the buffers are written again: by the join, or by a tile after this one)
    l += __shfl_xor(l, 32);
    const int64_t unit = ((int64_t)b * a.kv_heads + kvh) * p.tiles + tile;
    float* ws = whole ? nullptr : a.ws + (unit * p.splits + split) * kRowsHere * (DP + 2);
    if constexpr (WK == 1) {
      if (!busy) continue;
      if (whole) {
        E* to = out_row<E>(p, sq, b, kvh, row);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        if (to) {
#pragma unroll
          for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              typedef E e4 __attribute__((ext_vector_type(4)));
              const int d = 32 * dt + 8 * r + 4 * half;
              e4 v;
#pragma unroll
              for (int x = 0; x < 4; ++x) v[x] = (E)(acc[dt][4 * r + x] * inv);
              if (d < a.d) store_as(to + d, v);
            }
        }
      } else {
        const int mine = wave * 32 + i;
        if (half == 0) {
          ws[mine] = m;
          ws[kRowsHere + mine] = l;
        }
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            store_as(ws + 2 * kRowsHere + mine * DP + 32 * dt + 8 * r + 4 * half,
                     f32x4{acc[dt][4 * r], acc[dt][4 * r + 1], acc[dt][4 * r + 2], acc[dt][4 * r + 3]});
      }
    } else {
      float* so = reinterpret_cast<float*>(lds);             // [WK][kFewRows][kLd]
      float* sm = so + WK * kFewRows * kLd;                  // [WK][kFewRows]
      float* sl = sm + WK * kFewRows;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *reinterpret_cast<f32x4*>(so + (wave * kFewRows + i) * kLd + 32 * dt + 8 * r + 4 * half) =
              f32x4{acc[dt][4 * r], acc[dt][4 * r + 1], acc[dt][4 * r + 2], acc[dt][4 * r + 3]};
      if (half == 0) {
        sm[wave * kFewRows + i] = m;
        sl[wave * kFewRows + i] = l;
      }
      __syncthreads();
      const int last = rows - tile * kRowsHere < kRowsHere ? rows - tile * kRowsHere : kRowsHere;
      for (int x = threadIdx.x; x < last * DP / 4; x += 256) {   // four dimensions of a row
        const int r = x / (DP / 4), d = x % (DP / 4) * 4;
        float top = sm[r];
#pragma unroll
        for (int w = 1; w < WK; ++w) top = fmaxf(top, sm[w * kFewRows + r]);
        f32x4 o = {0, 0, 0, 0};
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float mw = sm[w * kFewRows + r], f = mw == top ? 1.f : exp2_fast(mw - top);
          o += f * *reinterpret_cast<const f32x4*>(so + (w * kFewRows + r) * kLd + d);
          sum += f * sl[w * kFewRows + r];
        }
        if (whole) {
          typedef E e4 __attribute__((ext_vector_type(4)));
          E* to = out_row<E>(p, sq, b, kvh, tile * kRowsHere + r);
          const float inv = sum == 0.f ? 0.f : 1.0f / sum;
          e4 v;
#pragma unroll
          for (int y = 0; y < 4; ++y) v[y] = (E)(o[y] * inv);
          if (to && d < a.d) store_as(to + d, v);
        } else {
          store_as(ws + 2 * kRowsHere + r * DP + d, o);
          if (d == 0) {
            ws[r] = top;
            ws[kRowsHere + r] = sum;
          }
        }
      }
      __syncthreads();   // (a tile after this one writes the buffers again)
    }
  }
}

// ---- fp32, keys through LDS ---------------------------------------------------------------------------------------------
// 64 query rows a workgroup, 16 a wave; every wave takes every key, 32 a step, in the products of Core<T_F32>: K and V rows lie in
// LDS (two buffers, as above), where 16 lanes read a column of 16 K rows, or a V row's 16 columns, in all 64 banks at once.
// Bound by the matrix instructions, in whose chains few workgroups wait: 8 x 512 x 512, 16 heads of 64: 80 us, 108 of the 153
// TFLOP/s that an fp32 library product reaches (98 us with a wave for itself); 8 x 1024 x 1024, 8 heads of 128: 290 us, 118 (415).
// Reading K and V ahead of the products, as the 16-bit kernel does, changes nothing where four workgroups share a CU.
constexpr int kTileRows32 = 64;

template <int DP, bool DMA>
__global__ __launch_bounds__(256, DP > 64 ? 2 : 4) void attn_tile32_kernel(AttnParams p) {
  using C = Core<T_F32, DP>;
  constexpr int kKeys = 32, kCols = DP / 4, kLoads = kKeys * kCols / 256, kHalf = kKeys * DP * 4, kBuf = 2 * kHalf;
  __shared__ __align__(1024) char lds[2 * kBuf];
  const AttnArgs& a = p.a;
  const unsigned each = p.tiles * p.splits, heads = p.units / p.tiles;   // (the 8 XCDs' caches, as above)
  const unsigned at = heads % 8 ? blockIdx.x : (blockIdx.x / 8 / each * 8 + blockIdx.x % 8) * each + blockIdx.x / 8 % each;
  const int split = at % p.splits, tile0 = at / p.splits % p.tiles;
  const int kvh = at / each % a.kv_heads, b = at / each / a.kv_heads;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const Span sq = queries_of(a, b);
  Span sk = keys_of(a, b);
  const int rows = sq.n * p.group;
  const float* kbase = static_cast<const float*>(a.k) + (a.k_offsets ? sk.first * a.k_ts : b * a.k_bs) + kvh * a.k_hs;
  const float* vbase = static_cast<const float*>(a.v) + (a.k_offsets ? sk.first * a.v_ts : b * a.v_bs) + kvh * a.v_hs;
  const uint8_t* mask = a.key_mask ? a.key_mask + b * a.mask_stride : nullptr;
  if (mask) sk.n = mask_end(mask, sk.n);
  auto byte_of = [&](int kb) -> unsigned char { return mask && lane < 32 && kb + lane < sk.n ? mask[kb + lane] : 1; };
  auto bits_of = [&](int kb, unsigned char there) { return (unsigned)__ballot(lane < 32 && kb + lane < sk.n && there); };
  auto column = [](unsigned r, unsigned c) { return c ^ (DP % 64 ? r / 2 % 8 : r % 16); };
  // this lane's 16 bytes of load j: key row `key` at LDS column chunk % kCols
  unsigned key[kLoads], from_k[kLoads], from_v[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const unsigned chunk = (4 * j + wave) * 64 + lane, c = column(chunk / kCols, chunk % kCols);
    key[j] = chunk / kCols;
    const bool in = (int)(4 * c) < a.d;
    from_k[j] = in ? 4 * (key[j] * (unsigned)a.k_ts + 4 * c) : kNowhere;
    from_v[j] = in ? 4 * (key[j] * (unsigned)a.v_ts + 4 * c) : kNowhere;
  }
  const unsigned lds0 = (unsigned)(uintptr_t)lds;

  for (int tile = tile0; tile < (rows + kTileRows32 - 1) / kTileRows32; tile += p.tiles) {
    const bool whole = p.splits == 1 || tile >= (int)p.tiles;
    if (whole && split) break;
    const int pieces = whole ? 1 : p.splits;
    const unsigned row = tile * kTileRows32 + wave * 16 + i;
    const bool busy = tile * kTileRows32 + wave * 16 < rows;   // (of this wave)
    u32x4 kr[DMA ? 1 : kLoads], vr[DMA ? 1 : kLoads];
    auto fetch = [&](int kb, unsigned bits, int buf) {
      const int n = sk.n - kb < kKeys ? sk.n - kb : kKeys;
      const RowBuffer<float> k(kbase, a.k_ts, kb, n, a.d), v(vbase, a.v_ts, kb, n, a.d);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const bool there = bits >> key[j] & 1;
        const unsigned at_k = there ? from_k[j] : kNowhere, at_v = there ? from_v[j] : kNowhere;
        if constexpr (DMA) {
          const unsigned to = lds0 + buf * kBuf + (4 * j + wave) * 1024;
          k.to_lds(at_k, to);
          v.to_lds(at_v, to + kHalf);
        } else {
          kr[j] = k.template load<16>(at_k);
          vr[j] = v.template load<16>(at_v);
        }
      }
    };
    auto keep = [&](int buf) {
      if constexpr (!DMA)
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          char* to = lds + buf * kBuf + (4 * j + wave) * 1024 + lane * 16;
          *reinterpret_cast<u32x4*>(to) = kr[j];
          *reinterpret_cast<u32x4*>(to + kHalf) = vr[j];
        }
    };
    const int step = pieces * kKeys;
    int kb = split * kKeys, buf = 0;
    unsigned char ahead = byte_of(kb + step);
    unsigned valid = bits_of(kb, byte_of(kb));
    C core;
    {
      const unsigned qi = row / p.group, h = kvh * p.group + row % p.group;
      const float* q = static_cast<const float*>(a.q) + (a.q_offsets ? sq.first * a.q_ts : b * a.q_bs) + qi * a.q_ts + h * a.q_hs;
      core.load_q(q, (int)qi < sq.n, p.flip, a.d, g);
    }
    if (kb < sk.n) {
      fetch(kb, valid, 0);
      keep(0);
    }
    f32x4 acc[C::kTiles] = {};
    float m = -INFINITY, l = 0.f;
    bool far = false;   // (of the whole wave)
    auto take = [&](const char* k_rows, unsigned here) {
      f32x4 s[2] = {};
#pragma unroll
      for (int st = 0; st < C::kSteps; ++st) {
        f32x4 kf[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          kf[h] = *reinterpret_cast<const f32x4*>(k_rows + ((16 * h + i) * kCols + column(16 * h + i, 4 * st + g)) * 16);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[h][x], core.q[st][x], s[h], 0, 0, 0);
      }
      if (here != ~0u) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[h][r] = (here >> (16 * h + 4 * g + r) & 1) ? s[h][r] : -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[h][r]);
      top = in_powers(top, p.c);
      if (__any(passes<T_F32>(top, m))) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = moved<T_F32>(m, top);
        const float f = to == m ? 1.f : exp2_fast(m - to);
        m = to;
        far = __any(is_far(m));
        l *= f;
#pragma unroll
        for (int t = 0; t < C::kTiles; ++t) acc[t] *= f;
      }
      const float ref = m == -INFINITY ? 0.f : m, c = far ? 1.f : p.c;
      if (far)
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r / 4][r % 4] = in_powers(s[r / 4][r % 4], p.c);
      float w[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          w[h][r] = exp2_fast(fmaf(s[h][r], c, -ref));
          l += w[h][r];
        }
      const char* v_rows = k_rows + kHalf;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned r = 16 * h + 4 * g + j;
#pragma unroll
          for (int x = 0; x < C::kWide; ++x) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(v_rows + (r * kCols + column(r, 16 * x + i)) * 16);
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[4 * x + t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t], w[h][j], acc[4 * x + t], 0, 0, 0);
          }
          if constexpr (C::kPair) {
            const typename C::f32x2 v = *reinterpret_cast<const typename C::f32x2*>(
                v_rows + (r * kCols + column(r, 16 * C::kWide + i / 2)) * 16 + 8 * (i % 2));
#pragma unroll
            for (int t = 0; t < 2; ++t)
              acc[4 * C::kWide + t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t], w[h][j], acc[4 * C::kWide + t], 0, 0, 0);
          }
        }
    };
    for (; kb < sk.n; kb += step, buf ^= 1) {
      if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // (this step's rows are in LDS)
      else __syncthreads();
      const bool more = kb + step < sk.n;
      const unsigned next = bits_of(kb + step, ahead);
      if (more) {
        ahead = byte_of(kb + 2 * step);
        fetch(kb + step, next, buf ^ 1);   // (last read before the barrier above)
      }
      if (busy && valid) take(lds + buf * kBuf, valid);
      if (more) keep(buf ^ 1);
      valid = next;
    }
    __syncthreads();   // (a tile after this one writes the buffers again)
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (!busy) continue;
    const int mine = wave * 16 + i;
    float* to = out_row<float>(p, sq, b, kvh, row);
    float scale = l == 0.f ? 0.f : 1.0f / l;
    int d = a.d;
    if (!whole) {   // this piece's part of the sums
      const int64_t unit = ((int64_t)b * a.kv_heads + kvh) * p.tiles + tile;
      float* ws = a.ws + (unit * p.splits + split) * kTileRows32 * (DP + 2);
      if (g == 0) {
        ws[mine] = m;
        ws[kTileRows32 + mine] = l;
      }
      to = ws + 2 * kTileRows32 + mine * DP;
      scale = 1.f;
      d = DP;
    }
    if (to) store_row<C>(to, acc, scale, d, g);
  }
}

// Joins the pieces of the tiles: a wave each row, the pieces' weights first (a lane each piece), then the pieces' sums, eight on
// the way at a time.
template <int TY, int DP, int ROWS>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnParams p) {
  using E = typename Elem<TY>::type;
  const AttnArgs& a = p.a;
  constexpr int kPiece = ROWS * (DP + 2), kPer = (DP + 63) / 64;
  const int lane = threadIdx.x & 63, row = blockIdx.x % (ROWS / 4) * 4 + threadIdx.x / 64;
  const unsigned unit = blockIdx.x / (ROWS / 4);
  const int tile = unit % p.tiles, kvh = unit / p.tiles % a.kv_heads, b = unit / p.tiles / a.kv_heads;
  E* to = out_row<E>(p, queries_of(a, b), b, kvh, tile * ROWS + row);
  if (!to) return;
  const int splits = p.splits;
  const float* ws = a.ws + (int64_t)unit * splits * kPiece;
  float m[4], l = 0.f, top = -INFINITY;   // (at most 256 pieces)
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int s = 64 * x + lane;
    m[x] = s < splits ? ws[(int64_t)s * kPiece + row] : -INFINITY;
    top = fmaxf(top, m[x]);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int s = 64 * x + lane;
    m[x] = s >= splits ? 0.f : m[x] == top ? 1.f : exp2_fast(m[x] - top);
    if (s < splits) l += m[x] * ws[(int64_t)s * kPiece + ROWS + row];
  }
  const float sum = wave_sum_f32(l);
  typedef float vec __attribute__((ext_vector_type(kPer)));
  vec o = 0.f;
  const int d = lane * kPer;
  const float* at = ws + 2 * ROWS + row * DP + (d < DP ? d : 0);
#pragma unroll
  for (int x = 0; x < 4; ++x)
    for (int s0 = 64 * x; s0 < splits && s0 < 64 * x + 64; s0 += 8) {
      vec v[8];
#pragma unroll
      for (int y = 0; y < 8; ++y) v[y] = load_as<vec>(at + (int64_t)(s0 + y < splits ? s0 + y : s0) * kPiece);
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const float f = __shfl(m[x], s0 + y - 64 * x);
        o += s0 + y < splits ? f * v[y] : vec(0.f);
      }
    }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
  for (int x = 0; x < kPer; ++x)
    if (d + x < a.d) to[d + x] = (E)(o[x] * inv);
}

int padded_d(int type, int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 && type == T_F32 ? 96 : 128; }

// How a launch is cut up.
//   16-bit types  128-row tiles where a key head has more than 32 query rows, else 32-row tiles
//   fp32          64-row tiles where a key head has more than 32 query rows and there is much to multiply, else 16-row tiles,
//                 eight waves each (8 x 512 x 512, 16 heads of 64: 77 / 98 us; 1 x 512 x 512, 8 heads: 21 / 13, few workgroups
//                 waiting for their chain of steps); heads of up to 32 are quicker without LDS (41 x 70 x 1668: 195 / 178)
//   alone         16-row tiles, a wave each: so few keys that a wave is done with them before a join would be (16-bit types: and
//                 at most 32 query rows a key head), or, fp32, tiles enough for two waves on each of 1024 SIMDs
// and, where those leave CUs idle, pieces of the keys, each at least 256 long, up to what the CUs hold at once (one more in a
// round of its own: 1 x 686 x 6136, 4 heads over 1 of 80, fp32: 473 workgroups 74 us, 516 98).
enum class Way { kAlone, kRows, kFew, kTile };
struct Plan {
  Way way;
  int tiles, splits, rows;
  int64_t units;
};
Plan plan(int type, int batch, int heads, int kv_heads, int d, int max_q, int max_k) {
  Plan p;
  if (max_q < 1) max_q = 1;   // (a hint, for packed queries: there may be some all the same)
  const int64_t rows = (int64_t)max_q * (heads / kv_heads);
  const int64_t sixteens = (rows + kRows - 1) / kRows * batch * kv_heads;
  const bool much = max_k <= 128 || (double)rows * batch * kv_heads * max_k * d >= 1 << 28;
  if (rows > kFewRows && (type != T_F32 || (d > 32 && much))) p.way = Way::kTile;
  else if (type == T_F32) p.way = max_k <= 128 || sixteens >= 2048 ? Way::kAlone : Way::kRows;
  else p.way = max_k <= 128 ? Way::kAlone : Way::kFew;
  p.rows = p.way == Way::kTile ? (type == T_F32 ? kTileRows32 : kTileRows) : p.way == Way::kFew ? kFewRows : kRows;
  const int64_t tiles = (rows + p.rows - 1) / p.rows, most = ((int64_t)1 << 22) / ((int64_t)batch * kv_heads) + 1;
  p.tiles = (int)(tiles < most ? tiles : most);   // (a grid holds below 2^32 threads; workgroups loop over the rest)
  p.units = (int64_t)p.tiles * batch * kv_heads;
  // What 256 CUs hold at once; tiles of short heads are four a CU, which 16-bit types' need only where two would leave many of
  // them empty (14 x 83 x 3593, 32 heads over 8 of 64, lengths from 31: 66 us whole, 61 in pieces; 8 x 128 x 2000, 16 heads:
  // four pieces 27.5, seven 29.6; fp32 11 x 251 x 4844, 8 heads: 302 with one, 230 with two).
  const bool four = p.way == Way::kTile && d <= 64 && (type == T_F32 || p.units > 256);
  const int at_once = p.way == Way::kRows ? 256 : four ? 1024 : 512;
  int64_t n = p.units && p.way != Way::kAlone ? at_once / p.units : 1;
  const int64_t pieces = (int64_t)max_k / 256;
  n = n < pieces ? n : pieces;
  p.splits = (int)(n < 1 ? 1 : n > 256 ? 256 : n);
  return p;
}

template <int TY, int DP, int ROWS>
hipError_t join(const AttnParams& p, hipStream_t s) {
  if (hipError_t e = hipGetLastError()) return e;
  if (p.splits == 1) return hipSuccess;
  attn_join_kernel<TY, DP, ROWS><<<dim3((unsigned)(p.units * (ROWS / 4))), 256, 0, s>>>(p);
  return hipGetLastError();
}
template <int TY, int DP>
hipError_t run(const AttnParams& p, const Plan& n, hipStream_t s) {
  const dim3 grid((unsigned)(p.units * p.splits));
  if (n.way == Way::kAlone) {
    attn_rows_kernel<TY, DP, 1><<<dim3((unsigned)((p.units + 3) / 4)), 256, 0, s>>>(p);
    return hipGetLastError();
  }
  const AttnArgs& a = p.a;
  constexpr int kBytes = sizeof(typename Elem<TY>::type);
  const bool dma = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                     kBytes * (a.k_ts | a.k_hs | a.v_ts | a.v_hs | (a.k_offsets ? 0 : a.k_bs | a.v_bs))) & 15) == 0;
  if constexpr (TY == T_F32) {
    if constexpr (DP > 32)
      if (n.way == Way::kTile) {
        if (dma) attn_tile32_kernel<DP, true><<<grid, 256, 0, s>>>(p);
        else attn_tile32_kernel<DP, false><<<grid, 256, 0, s>>>(p);
        return join<TY, DP, kTileRows32>(p, s);
      }
    attn_rows_kernel<TY, DP, 8><<<grid, 512, 0, s>>>(p);
    return join<TY, DP, kRows>(p, s);
  } else {
    if (n.way == Way::kTile) {
      if (dma) attn_tile_kernel<TY, DP, 1, true><<<grid, 256, 0, s>>>(p);
      else attn_tile_kernel<TY, DP, 1, false><<<grid, 256, 0, s>>>(p);
      return join<TY, DP, kTileRows>(p, s);
    }
    if (dma) attn_tile_kernel<TY, DP, 4, true><<<grid, 256, 0, s>>>(p);
    else attn_tile_kernel<TY, DP, 4, false><<<grid, 256, 0, s>>>(p);
    return join<TY, DP, kFewRows>(p, s);
  }
}

}  // namespace

int64_t attention_workspace(int type, int batch, int heads, int kv_heads, int d, int max_q, int max_k) {
  if (batch == 0) return 0;
  const Plan p = plan(type, batch, heads, kv_heads, d, max_q, max_k);
  return p.splits == 1 ? 0 : p.units * p.splits * p.rows * (padded_d(type, d) + 2) * 4;
}

hipError_t launch_attention(int type, const AttnArgs& a, hipStream_t s) {
  const Plan n = plan(type, a.batch, a.heads, a.kv_heads, a.d, a.max_q, a.max_k);
  // (never 0: a masked score of -inf stays one)
  const float c = fmaxf((float)(fabs((double)a.scale) * 1.4426950408889634), __FLT_DENORM_MIN__);
  const AttnParams p{a, c, a.scale < 0, (unsigned)(a.heads / a.kv_heads), (unsigned)n.tiles, (unsigned)n.units, (unsigned)n.splits};
  const int dp = padded_d(type, a.d);
  if (type == T_F32)
    return dp == 32   ? run<T_F32, 32>(p, n, s)
           : dp == 64 ? run<T_F32, 64>(p, n, s)
           : dp == 96 ? run<T_F32, 96>(p, n, s)
                      : run<T_F32, 128>(p, n, s);
  if (type == T_BF16) return dp == 32 ? run<T_BF16, 32>(p, n, s) : dp == 64 ? run<T_BF16, 64>(p, n, s) : run<T_BF16, 128>(p, n, s);
  return dp == 32 ? run<T_F16, 32>(p, n, s) : dp == 64 ? run<T_F16, 64>(p, n, s) : run<T_F16, 128>(p, n, s);
}

}  // namespace enc
}  // namespace rr
