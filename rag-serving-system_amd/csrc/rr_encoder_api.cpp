// rr_encoder_api.cpp — C-ABI host side of the embedding encoder's operators (include/rag_retrieval.h): argument checks,
// the device scope, and the launchers of rr_encoder_*.hip. Nothing here owns device memory or waits.
#include "rag_retrieval.h"
#include "rr_encoder.h"

#include <climits>
#include <cmath>

using rr::fail;
using namespace rr::enc;

namespace {

bool float_type(int t) { return t == RR_TYPE_F32 || t == RR_TYPE_BF16 || t == RR_TYPE_F16; }
int bytes_of(int t) { return t == RR_TYPE_F32 ? 4 : t == RR_TYPE_I8 ? 1 : 2; }
bool misaligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// The calling thread's device is `device` inside the scope and what it was after it.
struct DeviceScope {
  int before = -1;
  hipError_t err;
  explicit DeviceScope(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) err = hipSetDevice(device);
    else if (err == hipSuccess) before = -1;
    if (err != hipSuccess) {
      before = -1;
      (void)hipGetLastError();   // (reported here: the next launch's check is not to find it)
    }
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

template <class F>
int enqueue(const char* what, int device, F&& f) {
  DeviceScope on(device);
  if (on.err != hipSuccess) return fail(RR_E_HIP, "%s: device %d: %s", what, device, hipGetErrorString(on.err));
  if (hipError_t e = f()) return fail(RR_E_HIP, "%s: launch failed: %s", what, hipGetErrorString(e));
  return RR_OK;
}

int bad_device(const char* what, int device) {
  if (device < 0) return fail(RR_E_INVALID, "%s: device=%d", what, device);
  return RR_OK;
}

// rows of `cols` elements of `bytes` each, `ld` elements apart
int bad_rows(const char* what, const char* name, const void* p, int64_t ld, int64_t cols, int bytes) {
  if (!p) return fail(RR_E_INVALID, "%s: %s is null", what, name);
  if (misaligned(p, bytes)) return fail(RR_E_INVALID, "%s: %s is not aligned to its %d-byte elements", what, name, bytes);
  if (ld < cols) return fail(RR_E_INVALID, "%s: row stride %lld of %s below its %lld columns", what, (long long)ld, name,
                             (long long)cols);
  return RR_OK;
}

int bad_scratch(const char* what, const void* ws, int64_t have, int64_t need) {
  if (need <= 0) return RR_OK;
  if (!ws || have < need)
    return fail(RR_E_INVALID, "%s: workspace of %lld bytes, %lld needed", what, (long long)(ws ? have : 0), (long long)need);
  if (misaligned(ws, 16)) return fail(RR_E_INVALID, "%s: workspace is not 16-byte aligned", what);
  return RR_OK;
}

#define TRY(expr)                                \
  do {                                           \
    if (int _rc = (expr); _rc != RR_OK) return _rc; \
  } while (0)

int linear_sizes(int x_type, int64_t m, int32_t n, int32_t k) {
  if (x_type != RR_TYPE_I8 && !float_type(x_type)) return fail(RR_E_INVALID, "rr_linear_i8: bad x_type %d", x_type);
  if (m < 0 || n < 1 || k < 1)
    return fail(RR_E_INVALID, "rr_linear_i8: m=%lld n=%d k=%d", (long long)m, n, k);
  if (k > RR_LINEAR_KMAX)
    return fail(RR_E_UNSUPPORTED, "rr_linear_i8: k=%d above %d (the 32-bit sum would no longer be exact)", k, RR_LINEAR_KMAX);
  if (m > INT_MAX) return fail(RR_E_UNSUPPORTED, "rr_linear_i8: m=%lld above 2^31 - 1", (long long)m);
  if (n > 1 << 26) return fail(RR_E_UNSUPPORTED, "rr_linear_i8: n=%d above 2^26", n);
  return RR_OK;
}

// What a product's workspace holds, each part on 256 bytes: the rows' scales, the 8-bit rows, the weights' copy.
struct LinearScratch {
  bool fused, rows, repack;
  int64_t kp, x_at, w_at, bytes;
};
LinearScratch linear_scratch(int x_type, int64_t m, int32_t n, int32_t k) {
  LinearScratch l{};
  l.fused = x_type != RR_TYPE_I8 && linear_fuses_rows(m, k);
  l.rows = x_type != RR_TYPE_I8 && !l.fused && m > 0;
  l.repack = linear_repacks(x_type, m, n, k);
  l.kp = round_up(k, 16);
  l.x_at = l.rows ? round_up(m * 4, 256) : 0;
  l.w_at = l.x_at + (l.rows || l.repack ? round_up(m * l.kp, 256) : 0);
  l.bytes = l.w_at + (l.repack ? n * l.kp : 0);
  return l;
}

constexpr int64_t kTsMost = (1 << 23) - 1;   // 64 rows of up to 4-byte elements within 32-bit byte offsets

int attention_sizes(int type, int32_t batch, int32_t heads, int32_t kv_heads, int32_t d, int32_t max_q, int32_t max_k) {
  const char* me = "rr_cross_attention";
  if (!float_type(type)) return fail(RR_E_INVALID, "%s: bad type %d", me, type);
  if (batch < 0 || heads < 1 || kv_heads < 1 || max_q < 0 || max_k < 0)
    return fail(RR_E_INVALID, "%s: batch=%d heads=%d kv_heads=%d max_q=%d max_k=%d", me, batch, heads, kv_heads, max_q, max_k);
  if (heads % kv_heads) return fail(RR_E_INVALID, "%s: %d heads over %d key heads", me, heads, kv_heads);
  if (d < 8 || d % 8 || d > RR_ATTN_DMAX)
    return fail(RR_E_UNSUPPORTED, "%s: head size %d (a multiple of 8 up to %d)", me, d, RR_ATTN_DMAX);
  if (batch > 65535 || kv_heads > 65535)
    return fail(RR_E_UNSUPPORTED, "%s: batch=%d kv_heads=%d above 65535", me, batch, kv_heads);
  if ((int64_t)batch * kv_heads > 1 << 22)
    return fail(RR_E_UNSUPPORTED, "%s: %d sequences of %d key heads above 2^22", me, batch, kv_heads);
  if (max_q > 1 << 30 || max_k > 1 << 30)
    return fail(RR_E_UNSUPPORTED, "%s: max_q=%d max_k=%d above 2^30", me, max_q, max_k);
  if ((int64_t)max_q * (heads / kv_heads) > 1 << 30)
    return fail(RR_E_UNSUPPORTED, "%s: %d queries of %d heads a key head above 2^30 rows", me, max_q, heads / kv_heads);
  return RR_OK;
}

}  // namespace

extern "C" {

int rr_quantize_rows(int device, void* stream, int type, const void* x, int64_t ldx, int64_t rows, int32_t cols, int8_t* q,
                     int64_t ldq, float* scale) {
  const char* me = "rr_quantize_rows";
  TRY(bad_device(me, device));
  if (!float_type(type)) return fail(RR_E_INVALID, "%s: bad type %d", me, type);
  if (rows < 0 || cols < 1) return fail(RR_E_INVALID, "%s: rows=%lld cols=%d", me, (long long)rows, cols);
  if (rows > INT_MAX) return fail(RR_E_UNSUPPORTED, "%s: rows=%lld above 2^31 - 1", me, (long long)rows);
  if (rows == 0) return RR_OK;
  TRY(bad_rows(me, "x", x, ldx, cols, bytes_of(type)));
  TRY(bad_rows(me, "q", q, ldq, cols, 1));
  TRY(bad_rows(me, "scale", scale, 1, 1, 4));
  return enqueue(me, device, [&] {
    return launch_quantize_rows(type, x, ldx, rows, cols, cols, q, ldq, scale, {}, static_cast<hipStream_t>(stream));
  });
}

int64_t rr_linear_i8_workspace(int x_type, int64_t m, int32_t n, int32_t k) {
  if (int rc = linear_sizes(x_type, m, n, k); rc != RR_OK) return rc;
  return linear_scratch(x_type, m, n, k).bytes;
}

int rr_linear_i8(int device, void* stream, int x_type, const void* x, int64_t ldx, const float* x_scale, const int8_t* w,
                 int64_t ldw, const float* w_scale, const float* bias, int act, int out_type, void* out, int64_t ldo,
                 int64_t m, int32_t n, int32_t k, void* workspace, int64_t workspace_bytes) {
  const char* me = "rr_linear_i8";
  TRY(bad_device(me, device));
  TRY(linear_sizes(x_type, m, n, k));
  if (act != RR_ACT_NONE && act != RR_ACT_GELU) return fail(RR_E_INVALID, "%s: bad act %d", me, act);
  if (!float_type(out_type)) return fail(RR_E_INVALID, "%s: bad out_type %d", me, out_type);
  if (m == 0) return RR_OK;
  TRY(bad_rows(me, "x", x, ldx, k, bytes_of(x_type)));
  TRY(bad_rows(me, "w", w, ldw, k, 1));
  if ((n > 1 && ldw >= RR_LINEAR_LDMOST) || (x_type == RR_TYPE_I8 && m > 1 && ldx >= RR_LINEAR_LDMOST))
    return fail(RR_E_UNSUPPORTED, "%s: 8-bit rows %lld and weights %lld bytes apart, not below %d", me, (long long)ldx,
                (long long)ldw, RR_LINEAR_LDMOST);
  TRY(bad_rows(me, "w_scale", w_scale, 1, 1, 4));
  if (bias) TRY(bad_rows(me, "bias", bias, 1, 1, 4));
  TRY(bad_rows(me, "out", out, ldo, n, bytes_of(out_type)));
  if ((x_type == RR_TYPE_I8) != (x_scale != nullptr))
    return fail(RR_E_INVALID, "%s: x_scale goes with 8-bit rows, and only with them", me);
  if (x_scale) TRY(bad_rows(me, "x_scale", x_scale, 1, 1, 4));
  const LinearScratch l = linear_scratch(x_type, m, n, k);
  TRY(bad_scratch(me, workspace, workspace_bytes, l.bytes));
  hipStream_t s = static_cast<hipStream_t>(stream);
  return enqueue(me, device, [&]() -> hipError_t {
    LinearArgs a{static_cast<const int8_t*>(x), ldx, x_scale, w, ldw, w_scale, bias, act, out_type, out, ldo, (int)m, n, k};
    if (l.fused) return launch_linear_fused(x_type, a, s);
    int8_t* at = static_cast<int8_t*>(workspace);
    const WeightCopy copy = l.repack ? WeightCopy{w, ldw, n, at + l.w_at} : WeightCopy{};
    if (l.rows) {
      float* sc = static_cast<float*>(workspace);
      if (hipError_t e = launch_quantize_rows(x_type, x, ldx, m, k, (int)l.kp, at + l.x_at, l.kp, sc, copy, s))
        return e;
      a.x = at + l.x_at;
      a.ldx = l.kp;
      a.x_scale = sc;
    }
    if (l.repack) {
      if (!l.rows)
        if (hipError_t e = launch_repack(a.x, ldx, m, at + l.x_at, copy, k, s)) return e;
      a.x = at + l.x_at;
      a.w = at + l.w_at;
      a.ldx = a.ldw = l.kp;
      a.k = (int)l.kp;
    }
    return launch_linear(a, s);
  });
}

int rr_block_norm(int device, void* hip_stream, int type, int64_t rows, int32_t cols, const void* y, int64_t ldy,
                  const void* x, int64_t ldx, float residual_scale, const void* gate, int64_t ldg, int64_t gate_rows,
                  int64_t rows_per_gate, int post_norm, const void* post_weight, const void* post_bias, int next_norm,
                  const void* next_weight, const void* next_bias, float eps, void* stream, int64_t lds, void* normed,
                  int64_t ldn, int8_t* q, int64_t ldq, float* q_scale) {
  const char* me = "rr_block_norm";
  TRY(bad_device(me, device));
  if (!float_type(type)) return fail(RR_E_INVALID, "%s: bad type %d", me, type);
  if (rows < 0 || cols < 1) return fail(RR_E_INVALID, "%s: rows=%lld cols=%d", me, (long long)rows, cols);
  if (cols > RR_NORM_COLMAX) return fail(RR_E_UNSUPPORTED, "%s: cols=%d above %d", me, cols, RR_NORM_COLMAX);
  if (rows > INT_MAX) return fail(RR_E_UNSUPPORTED, "%s: rows=%lld above 2^31 - 1", me, (long long)rows);
  for (int kind : {post_norm, next_norm})
    if (kind != RR_NORM_NONE && kind != RR_NORM_LAYER && kind != RR_NORM_RMS)
      return fail(RR_E_INVALID, "%s: bad norm %d", me, kind);
  if (!(eps >= 0.f) || std::isinf(eps)) return fail(RR_E_INVALID, "%s: eps=%g", me, eps);
  if (!stream && !normed && !q) return fail(RR_E_INVALID, "%s: no output asked for", me);
  if ((q != nullptr) != (q_scale != nullptr)) return fail(RR_E_INVALID, "%s: q and q_scale go together", me);
  if (next_norm == RR_NORM_NONE && (normed || q || next_weight || next_bias))
    return fail(RR_E_INVALID, "%s: normed, q and the next norm's weights need a next norm", me);
  if (post_norm == RR_NORM_NONE && (post_weight || post_bias))
    return fail(RR_E_INVALID, "%s: weights of a post norm that is not there", me);
  const int eb = bytes_of(type);
  if (gate && (rows_per_gate < 1 || gate_rows < rows / rows_per_gate + (rows % rows_per_gate != 0)))
    return fail(RR_E_INVALID, "%s: %lld gate rows of %lld rows each for %lld rows", me, (long long)gate_rows,
                (long long)rows_per_gate, (long long)rows);
  if (rows == 0) return RR_OK;
  TRY(bad_rows(me, "y", y, ldy, cols, eb));
  if (x) TRY(bad_rows(me, "x", x, ldx, cols, eb));
  if (gate) TRY(bad_rows(me, "gate", gate, ldg, cols, eb));
  for (const void* p : {post_weight, post_bias, next_weight, next_bias})
    if (p) TRY(bad_rows(me, "a weight or bias", p, cols, cols, eb));
  if (stream) TRY(bad_rows(me, "stream", stream, lds, cols, eb));
  if (normed) TRY(bad_rows(me, "normed", normed, ldn, cols, eb));
  if (q) {
    TRY(bad_rows(me, "q", q, ldq, cols, 1));
    TRY(bad_rows(me, "q_scale", q_scale, 1, 1, 4));
  }
  const NormArgs a{rows, cols, y, x, gate, ldy, ldx, ldg, gate ? rows_per_gate : 1, residual_scale, eps, post_norm,
                   next_norm, post_weight, post_bias, next_weight, next_bias, stream, normed, lds, ldn, q, ldq, q_scale, false};
  return enqueue(me, device, [&] { return launch_block_norm(type, a, static_cast<hipStream_t>(hip_stream)); });
}

int64_t rr_cross_attention_workspace(int type, int32_t batch, int32_t heads, int32_t kv_heads, int32_t d, int32_t max_q,
                                     int32_t max_k) {
  if (int rc = attention_sizes(type, batch, heads, kv_heads, d, max_q, max_k); rc != RR_OK) return rc;
  return attention_workspace(type, batch, heads, kv_heads, d, max_q, max_k);
}

int rr_cross_attention(int device, void* stream, int type, const void* q, int64_t q_bs, int64_t q_ts, int64_t q_hs,
                       const void* k, int64_t k_bs, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_bs, int64_t v_ts,
                       int64_t v_hs, void* out, int64_t o_bs, int64_t o_ts, int64_t o_hs, int32_t batch, int32_t heads,
                       int32_t kv_heads, int32_t d, int32_t max_q, int32_t max_k, int64_t total_q, int64_t total_k,
                       const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* key_lengths,
                       const uint8_t* key_mask, int64_t mask_stride, float scale, void* workspace,
                       int64_t workspace_bytes) {
  const char* me = "rr_cross_attention";
  TRY(bad_device(me, device));
  TRY(attention_sizes(type, batch, heads, kv_heads, d, max_q, max_k));
  if (!std::isfinite(scale)) return fail(RR_E_INVALID, "%s: scale=%g", me, scale);
  if (key_mask && k_offsets) return fail(RR_E_INVALID, "%s: key_mask goes with dense keys", me);
  if (key_mask && mask_stride < max_k)
    return fail(RR_E_INVALID, "%s: mask row stride %lld below max_k=%d", me, (long long)mask_stride, max_k);
  if (q_offsets && (total_q < 0 || total_q > 1 << 30)) return fail(RR_E_INVALID, "%s: total_q=%lld", me, (long long)total_q);
  if (k_offsets && (total_k < 0 || total_k > 1 << 30)) return fail(RR_E_INVALID, "%s: total_k=%lld", me, (long long)total_k);
  if (q_offsets && total_q * (heads / kv_heads) > 1 << 30)
    return fail(RR_E_UNSUPPORTED, "%s: %lld queries of %d heads a key head above 2^30 rows", me, (long long)total_q,
                heads / kv_heads);
  if ((k_offsets ? total_k : max_k) <= 1) k_ts = v_ts = d;   // (no step from key to key: its size may be anything)
  if (k_ts > kTsMost || v_ts > kTsMost)
    return fail(RR_E_UNSUPPORTED, "%s: keys %lld and values %lld elements apart, above %lld", me, (long long)k_ts,
                (long long)v_ts, (long long)kTsMost);
  const int eb = bytes_of(type);
  for (int64_t st : {q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs, q_offsets ? 0 : q_bs, q_offsets ? 0 : o_bs,
                     k_offsets ? 0 : k_bs, k_offsets ? 0 : v_bs})
    if (st < 0) return fail(RR_E_INVALID, "%s: negative stride %lld", me, (long long)st);
  for (const void* p : {static_cast<const void*>(q_offsets), static_cast<const void*>(k_offsets),
                        static_cast<const void*>(key_lengths)})
    if (misaligned(p, 4)) return fail(RR_E_INVALID, "%s: offsets or lengths are not aligned to their 4-byte elements", me);
  if (batch == 0 || (q_offsets ? total_q : max_q) == 0) return RR_OK;
  TRY(bad_rows(me, "q", q, d, d, eb));
  TRY(bad_rows(me, "out", out, d, d, eb));
  if ((k_offsets ? total_k : max_k) > 0) {
    TRY(bad_rows(me, "k", k, d, d, eb));
    TRY(bad_rows(me, "v", v, d, d, eb));
  }
  TRY(bad_scratch(me, workspace, workspace_bytes, attention_workspace(type, batch, heads, kv_heads, d, max_q, max_k)));
  const AttnArgs a{q, k, v, out, q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, o_bs, o_ts, o_hs, batch, heads,
                   kv_heads, d, max_q, max_k, q_offsets ? total_q : 0, k_offsets ? total_k : 0, q_offsets, k_offsets,
                   key_lengths, key_mask, mask_stride, scale, static_cast<float*>(workspace)};
  return enqueue(me, device, [&] { return launch_attention(type, a, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
