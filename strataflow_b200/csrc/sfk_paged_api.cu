// sfk_paged_api.cu -- C entries of the paged-cache operators (include/sfk.h):
// sfk_qk_norm_rope_append, sfk_attn_decode_window, sfk_attn_prefill_window and
// sfk_device_status.  They check their arguments, launch on the caller's
// stream and return without waiting: no allocation, no state between calls.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/sfk.h"
#include "sfk_kernels.cuh"
#include "sfk_paged.cuh"
#include "sfk_rows.h"

using namespace sfk;

namespace {

sfk_status pfail(sfk_status st, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return st;
}
sfk_status cuda_result(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return SFK_OK;
  cudaGetLastError();  // reported here, and to no later call
  return pfail(e == cudaErrorMemoryAllocation ? SFK_ERR_OUT_OF_MEMORY : SFK_ERR_RUNTIME, "%s: %s", what,
               cudaGetErrorString(e));
}
#define BAD(...) return pfail(SFK_ERR_INVALID_ARGUMENT, __VA_ARGS__)

// SFK_TYPE_* of activation rows / SFK_KV_* of the cache -> Elem, -1 if neither
int row_elem(int t) { return t == SFK_TYPE_F32 ? EL_F32 : t == SFK_TYPE_F16 ? EL_F16 : t == SFK_TYPE_BF16 ? EL_BF16 : -1; }
int kv_elem(int t) { return t == SFK_KV_F32 ? EL_F32 : t == SFK_KV_F16 ? EL_F16 : t == SFK_KV_BF16 ? EL_BF16 : -1; }

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// rows of `stride` elements from p keep 16-byte alignment
bool vec_rows(const void* p, int64_t stride, int elem) { return aligned16(p) && stride * elem_size(elem) % 16 == 0; }

Rows rows_of(const void* at, int64_t stride, int64_t width, int64_t n, int elem) {
  return {at, stride * elem_size(elem), width * elem_size(elem), n};
}

int current_sms() {
  static int cached[64];  // multiprocessors of each device; every writer writes the same number
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 64 && cached[dev] > 0) return cached[dev];
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  if (dev >= 0 && dev < 64) cached[dev] = n;
  return n;
}

constexpr int MAX_PAGES = 1 << 27;  // positions stay below 2^31

constexpr float LOG2_E = 1.44269504088896340736f;

// What the two attention entries share.
sfk_status attn_args(const char* who, WindowAttnParams& a, int* kv, int32_t io_type, const void* q, int64_t q_stride,
                     int32_t kv_type, const void* kp, const void* vp, int32_t n_pages, const int32_t* table,
                     int32_t max_pages, int32_t n_head, int32_t n_head_kv, int32_t hd, float scale, int32_t window,
                     int32_t n_sink, void* out) {
  const int io = row_elem(io_type);
  *kv = kv_elem(kv_type);
  if (io < 0 || *kv < 0) BAD("%s: element type (rows %d, cache %d)", who, io_type, kv_type);
  if (io != EL_F32 && io != *kv) BAD("%s: 16-bit rows need a cache of their own type", who);
  if (hd != 32 && hd != 64 && hd != 128 && hd != 256) BAD("%s: head_dim %d (32, 64, 128 or 256)", who, hd);
  if (n_head < 1 || n_head_kv < 1 || n_head % n_head_kv || n_head > 65535)
    BAD("%s: %d heads over %d kv heads", who, n_head, n_head_kv);
  if (n_pages < 1 || max_pages < 1 || max_pages > MAX_PAGES) BAD("%s: pages (pool %d, table %d)", who, n_pages, max_pages);
  if (window < 0 || n_sink < 0) BAD("%s: window %d, sinks %d", who, window, n_sink);
  if (!std::isfinite(scale * LOG2_E) || scale < 0.f) BAD("%s: scale %g", who, (double)scale);
  if (!q || !kp || !vp || !table || !out) BAD("%s: null pointer", who);
  if (!aligned16(kp) || !aligned16(vp)) BAD("%s: page pools start on 16-byte boundaries", who);
  if (q_stride < (int64_t)n_head * hd) BAD("%s: q_stride %lld", who, (long long)q_stride);
  a.q = q;
  a.q_stride = q_stride;
  a.io = io;
  a.q_vec = vec_rows(q, q_stride, io);
  a.out_vec = aligned16(out);
  a.k_pages = kp;
  a.v_pages = vp;
  a.n_pages = n_pages;
  a.max_pages = max_pages;
  a.n_head = n_head;
  a.n_head_kv = n_head_kv;
  a.page_table = table;
  a.scale_log2 = (scale == 0.f ? 1.0f / sqrtf((float)hd) : scale) * LOG2_E;
  a.window = window;
  a.n_sink = n_sink;
  a.out = out;
  return SFK_OK;
}

}  // namespace

extern "C" {

sfk_status sfk_qk_norm_rope_append(int32_t io_type, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                   const void* v, int64_t v_stride, int32_t n_tok, int32_t n_head, int32_t n_head_kv,
                                   int32_t hd, const float* q_norm, const float* k_norm, float eps, int32_t neox,
                                   int32_t n_rot, const float* freqs, const int32_t* rope_pos, int32_t n_axes,
                                   const uint8_t* rope_axis, int32_t kv_type, void* kp, void* vp, int32_t n_pages,
                                   const int32_t* table, int32_t n_seq, int32_t max_pages, const int32_t* seq,
                                   const int32_t* pos, void* q_out, int64_t q_out_stride, int32_t* status, void* stream) {
  const char* who = "qk_norm_rope_append";
  const int io = row_elem(io_type), kv = kv_elem(kv_type);
  if (io < 0 || kv < 0) BAD("%s: element type (rows %d, cache %d)", who, io_type, kv_type);
  if (hd < 8 || hd > 256 || hd % 8) BAD("%s: head_dim %d (a multiple of 8 up to 256)", who, hd);
  if (n_head < 1 || n_head_kv < 1 || n_head > 65535 || n_head_kv > 65535) BAD("%s: %d and %d heads", who, n_head, n_head_kv);
  if (n_rot < 0 || n_rot > hd || n_rot % (neox ? 16 : 8)) BAD("%s: n_rot %d of %d", who, n_rot, hd);
  if (n_tok < 0 || n_seq < 0 || n_pages < 1 || max_pages < 1 || max_pages > MAX_PAGES)
    BAD("%s: sizes (%d tokens, %d sequences, pool %d, table %d)", who, n_tok, n_seq, n_pages, max_pages);
  if ((q_norm || k_norm) && !(eps >= 0.f && std::isfinite(eps))) BAD("%s: eps %g", who, (double)eps);
  if (rope_pos ? (n_axes < 1 || n_axes > 8) : (n_axes > 1 || rope_axis != nullptr))
    BAD("%s: %d position axes need rope_pos", who, n_axes);
  if (rope_axis)
    for (int i = 0; i < n_rot / 2; ++i)
      if (rope_axis[i] >= n_axes) BAD("%s: pair %d is on axis %d of %d", who, i, rope_axis[i], n_axes);
  if (n_tok == 0) return SFK_OK;
  if (!q || !k || !v || !kp || !vp || !table || !pos || !q_out || (n_rot > 0 && !freqs)) BAD("%s: null pointer", who);
  if (!seq && n_seq < n_tok) BAD("%s: %d tokens of %d sequences without a sequence list", who, n_tok, n_seq);
  if (!aligned16(kp) || !aligned16(vp)) BAD("%s: page pools start on 16-byte boundaries", who);
  const int64_t nq = (int64_t)n_head * hd, nk = (int64_t)n_head_kv * hd;
  if (q_stride < nq || k_stride < nk || v_stride < nk || q_out_stride < nq) BAD("%s: strides below a token's row", who);
  // in place a warp has read the row that it writes; a row of another token, or of k or v, may still be waited for
  const Rows qr = rows_of(q, q_stride, nq, n_tok, io), outr = rows_of(q_out, q_out_stride, nq, n_tok, io);
  if (!same_rows(qr, outr) && rows_meet(qr, outr)) BAD("%s: q_out overlaps q (only q itself, in q's stride, may be)", who);
  if (rows_meet(rows_of(k, k_stride, nk, n_tok, io), outr) || rows_meet(rows_of(v, v_stride, nk, n_tok, io), outr))
    BAD("%s: q_out overlaps k or v", who);
  AppendParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.out_stride = q_out_stride;
  p.n_tok = n_tok;
  p.n_head = n_head;
  p.n_head_kv = n_head_kv;
  p.hd = hd;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.eps = eps;
  p.neox = neox != 0;
  p.n_rot = n_rot;
  p.freqs = freqs;
  p.rope_pos = rope_pos;
  p.n_axes = n_axes;
  p.k_pages = kp;
  p.v_pages = vp;
  p.page_table = table;
  p.n_seq = n_seq;
  p.max_pages = max_pages;
  p.n_pages = n_pages;
  p.seq = seq;
  p.pos = pos;
  p.status = status;
  p.vec = (vec_rows(q, q_stride, io) ? 1 : 0) | (vec_rows(k, k_stride, io) ? 2 : 0) | (vec_rows(v, v_stride, io) ? 4 : 0) |
          (vec_rows(q_out, q_out_stride, io) ? 8 : 0);
  if (rope_axis) memcpy(p.axis, rope_axis, (size_t)(n_rot / 2));
  return cuda_result(launch_append(p, io, kv, current_sms(), (cudaStream_t)stream), who);
}

sfk_status sfk_attn_decode_window(int32_t io_type, const void* q, int64_t q_stride, int32_t kv_type, const void* kp,
                                  const void* vp, int32_t n_pages, const int32_t* table, int32_t max_pages,
                                  const int32_t* positions, int32_t n_seq, int32_t n_head, int32_t n_head_kv, int32_t hd,
                                  float scale, int32_t window, int32_t n_sink, void* out, void* workspace,
                                  size_t workspace_bytes, int32_t* status, void* stream) {
  const char* who = "attn_decode_window";
  if (n_seq < 0 || n_seq > 65535) BAD("%s: %d sequences (at most 65535)", who, n_seq);
  if (n_seq == 0) return SFK_OK;
  WindowAttnParams a{};
  int kv = 0;
  if (sfk_status s = attn_args(who, a, &kv, io_type, q, q_stride, kv_type, kp, vp, n_pages, table, max_pages, n_head,
                               n_head_kv, hd, scale, window, n_sink, out))
    return s;
  if (!positions) BAD("%s: null pointer", who);
  if (!aligned16(workspace)) BAD("%s: the workspace starts on a 16-byte boundary", who);
  // in place a CTA reads the heads that it writes, and no others; else one sequence's output would be another's query
  const int64_t width = (int64_t)n_head * hd;
  const Rows qr = rows_of(q, q_stride, width, n_seq, a.io), outr = rows_of(out, width, width, n_seq, a.io);
  if (!same_rows(qr, outr) && rows_meet(qr, outr)) BAD("%s: out overlaps q (only its own rows, contiguous, may be)", who);
  a.partial = static_cast<float*>(workspace);
  a.ws_bytes = workspace ? workspace_bytes : 0;
  a.pos = positions;
  a.n_seq = n_seq;
  a.status = status;
  return cuda_result(launch_window_decode(a, kv, hd, current_sms(), (cudaStream_t)stream), who);
}

size_t sfk_attn_decode_window_workspace(int32_t n_seq, int32_t n_head, int32_t n_head_kv, int32_t hd, int32_t max_pages,
                                        int32_t window, int32_t n_sink) {
  if (n_seq < 1 || n_seq > 65535 || n_head < 1 || n_head_kv < 1 || n_head % n_head_kv || hd < 1 || hd > 256 ||
      max_pages < 1 || max_pages > MAX_PAGES || window < 0 || n_sink < 0)
    return 0;
  WindowAttnParams a{};
  a.n_seq = n_seq;
  a.n_head = n_head;
  a.n_head_kv = n_head_kv;
  a.max_pages = max_pages;
  a.window = window;
  a.n_sink = n_sink;
  return window_decode_workspace(a, hd, current_sms());
}

sfk_status sfk_attn_prefill_window(int32_t io_type, const void* q, int64_t q_stride, int32_t n_tok, int32_t kv_type,
                                   const void* kp, const void* vp, int32_t n_pages, const int32_t* table,
                                   int32_t max_pages, const int32_t* q_start, const int32_t* kv_len, int32_t n_seq,
                                   int32_t n_head, int32_t n_head_kv, int32_t hd, float scale, int32_t window,
                                   int32_t n_sink, void* out, int32_t* status, void* stream) {
  const char* who = "attn_prefill_window";
  if (n_seq < 0 || n_tok < 0 || n_seq > 65535) BAD("%s: sizes (%d tokens, %d sequences)", who, n_tok, n_seq);
  if (n_seq == 0 || n_tok == 0) return SFK_OK;
  WindowAttnParams a{};
  int kv = 0;
  if (sfk_status s = attn_args(who, a, &kv, io_type, q, q_stride, kv_type, kp, vp, n_pages, table, max_pages, n_head,
                               n_head_kv, hd, scale, window, n_sink, out))
    return s;
  if (!q_start || !kv_len) BAD("%s: null pointer", who);
  if (n_head_kv > 65535 || (int64_t)n_tok * (n_head / n_head_kv) > (1ll << 30))
    BAD("%s: %d tokens of %d heads in one call", who, n_tok, n_head);
  // a row may be read again after others of its tile are written
  const int64_t width = (int64_t)n_head * hd;
  if (rows_meet(rows_of(q, q_stride, width, n_tok, a.io), rows_of(out, width, width, n_tok, a.io)))
    BAD("%s: out is q, or overlaps it", who);
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.n_seq = n_seq;
  a.n_tok = n_tok;
  a.status = status;
  return cuda_result(launch_window_prefill(a, kv, hd, current_sms(), (cudaStream_t)stream), who);
}

sfk_status sfk_device_status(int32_t* status, void* stream) {
  if (!status) BAD("device_status: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  int32_t h = 0;
  cudaError_t e = cudaMemcpyAsync(&h, status, sizeof(h), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(status, 0, sizeof(h), st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return cuda_result(e, "device_status");
  if (h == ERR_NONE) return SFK_OK;
  return pfail(SFK_ERR_RUNTIME, "device reported error %d (%s)", h,
               h == ERR_TIMEOUT    ? "bounded wait expired"
               : h == ERR_BAD_ID   ? "sequence id out of range"
               : h == ERR_BAD_PAGE ? "page id outside the KV pool"
                                   : "position or length outside the page table");
}

}  // extern "C"
