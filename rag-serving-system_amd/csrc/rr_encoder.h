// rr_encoder.h — the embedding encoder's operators: arguments and launchers shared between their C-ABI checks
// (rr_encoder_api.cpp) and their kernels (rr_encoder_*.hip). Not part of the public ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rr {

int fail(int code, const char* fmt, ...);   // rr_api.cpp: sets rr_last_error(), returns code

namespace enc {

constexpr int T_F32 = 0, T_BF16 = 1, T_F16 = 2, T_I8 = 3;   // RR_TYPE_*

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// ---- 8-bit rows and the 8-bit product (rr_encoder_linear.hip) ------------------------------------------------------
struct WeightCopy {   // weights to copy to rows of k rounded up to 16, zeros behind k (w null: none)
  const int8_t* w;
  int64_t ldw;
  int n;
  int8_t* to;
};
// cols_pad: the columns of q that are written, zeros behind cols; with a copy, k rounded up to 16 of k = cols
hipError_t launch_quantize_rows(int type, const void* x, int64_t ldx, int64_t rows, int cols, int cols_pad, int8_t* q,
                                int64_t ldq, float* scale, const WeightCopy& copy, hipStream_t s);

struct LinearArgs {
  const int8_t* x;       // [m][k]
  int64_t ldx;
  const float* x_scale;  // [m]
  const int8_t* w;       // [n][k]
  int64_t ldw;
  const float* w_scale;  // [n]
  const float* bias;     // [n] or null
  int act;
  int out_type;
  void* out;
  int64_t ldo;
  int m, n, k;
};
hipError_t launch_linear(const LinearArgs& a, hipStream_t s);
// Inner sizes that are no multiple of 4: whether the product takes copies of its weights, and of 8-bit rows, padded to 16.
bool linear_repacks(int x_type, int64_t m, int n, int k);
hipError_t launch_repack(const int8_t* x, int64_t ldx, int64_t m, int8_t* to_x, const WeightCopy& copy, int k, hipStream_t s);
// Few short floating-point rows: one launch makes their 8-bit rows too (x holds the floating-point rows, x_scale is unused).
bool linear_fuses_rows(int64_t m, int k);
hipError_t launch_linear_fused(int x_type, const LinearArgs& a, hipStream_t s);

// ---- norms (rr_encoder_norm.hip) -----------------------------------------------------------------------------------
struct NormArgs {
  int64_t rows;
  int cols;
  const void *y, *x, *gate;
  int64_t ldy, ldx, ldg, rows_per_gate;
  float residual_scale, eps;
  int post, next;
  const void *post_w, *post_b, *next_w, *next_b;
  void *stream, *normed;
  int64_t lds, ldn;
  int8_t* q;
  int64_t ldq;
  float* q_scale;
  bool past;   // (set by the launcher) results are written past the caches
};
hipError_t launch_block_norm(int type, const NormArgs& a, hipStream_t s);

// ---- attention (rr_encoder_attn.hip) -------------------------------------------------------------------------------
struct AttnArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, o_bs, o_ts, o_hs;
  int batch, heads, kv_heads, d, max_q, max_k;
  int64_t total_q, total_k;
  const int32_t *q_offsets, *k_offsets, *key_lengths;
  const uint8_t* key_mask;
  int64_t mask_stride;
  float scale;
  float* ws;
};
int64_t attention_workspace(int type, int batch, int heads, int kv_heads, int d, int max_q, int max_k);
hipError_t launch_attention(int type, const AttnArgs& a, hipStream_t s);

}  // namespace enc
}  // namespace rr
