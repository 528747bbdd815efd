// sfk_paged.cuh -- parameter blocks, launch entry points and shared device
// code of the operator-level paged-cache kernels: rotated append
// (sfk_paged_append.cu), windowed attention of single tokens
// (sfk_paged_decode.cu) and of prompts (sfk_paged_prefill.cu).
//
// The cache is the engine's: pools of 16-token pages [page][Hkv][16][hd] for
// K and V and a table of page ids per sequence.  Key j is seen from position
// p when j <= p and (window == 0, or j > p - window, or j < n_sink).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

#include "sfk_device.cuh"

namespace sfk {

constexpr int PG = 16;  // tokens per page

// element types of the rows (SFK_TYPE_*) and of the cache (SFK_KV_*), as one enum
enum Elem : int { EL_F32 = 0, EL_F16 = 1, EL_BF16 = 2 };
inline int elem_size(int e) { return e == EL_F32 ? 4 : 2; }

constexpr int APPEND_MAX_PAIRS = 128;  // rotated pairs per head (head_dim <= 256)

struct AppendParams {
  const void *q, *k, *v;
  void* q_out;
  int64_t q_stride, k_stride, v_stride, out_stride;  // elements between tokens
  int n_tok, n_head, n_head_kv, hd;
  const float *q_norm, *k_norm;  // [hd] or null
  float eps;
  int neox, n_rot;
  const float* freqs;      // [n_rot / 2]
  const int* rope_pos;     // [n_axes][n_tok] or null: the cache positions
  int n_axes;
  void *k_pages, *v_pages;
  const int* page_table;  // [n_seq][max_pages]
  int n_seq, max_pages, n_pages;
  const int* seq;  // [n_tok] or null: token t is sequence t's
  const int* pos;  // [n_tok]
  int* status;     // or null
  int vec;         // 16-byte accesses: bit 0 q, 1 k, 2 v, 3 q_out
  int share;       // warps that share a token's heads
  uint8_t axis[APPEND_MAX_PAIRS];
};
cudaError_t launch_append(AppendParams& p, int io, int kv, int sm_count, cudaStream_t st);

struct WindowAttnParams {
  const void* q;
  int64_t q_stride;  // elements between tokens
  int io;            // Elem of q and out
  int q_vec, out_vec;  // rows are 16-byte aligned
  const void *k_pages, *v_pages;
  int n_pages, max_pages, n_head, n_head_kv;
  const int* page_table;
  float scale_log2;  // softmax scale * log2(e)
  int window, n_sink;
  void* out;         // [tokens][n_head * hd]
  int* status;       // or null
  // decode
  const int* pos;    // [n_seq]
  int n_seq;
  int parts;         // CTAs that share one (sequence, kv head, row tile)
  float* partial;    // where they join: null, a cluster; else this workspace
  size_t ws_bytes;
  // prefill
  const int* q_start;  // [n_seq + 1]
  const int* kv_len;   // [n_seq]
  int n_tok;
  int tile_rows;   // rows per CTA (tensor-core form)
  int key_parts;   // CTAs of a cluster that share a row tile's keys (tensor-core form)
};
cudaError_t launch_window_decode(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st);
// p.partial / p.ws_bytes: the caller's workspace, or null
size_t window_decode_workspace(const WindowAttnParams& p, int hd, int sm_count);
cudaError_t launch_window_prefill(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st);
// the tensor-core form: whether it takes these types and sizes, and its launch
bool prefill_tc_takes(const WindowAttnParams& p, int kv, int hd);
cudaError_t launch_prefill_tc(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st);

// Dynamic shared memory above 48 KB has to be allowed once per kernel and device (two threads may do it twice).
template <auto Kernel>
inline cudaError_t allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};  // a bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

#ifdef __CUDACC__
// A launch and its own status: cudaGetLastError after it would also return what an earlier call of another kind left
// behind (an engine that did not fit the card).
template <class P>
inline cudaError_t launch_own(void (*kernel)(P), dim3 grid, int threads, size_t smem, cudaStream_t st, const P& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// ---- element access -----------------------------------------------------------
template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
// one rounding to nearest even
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <class T>
struct Raw8 {  // eight elements as loaded
  uint4 w[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ void load8(Raw8<T>& r, const T* p, bool vec) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
    T* e = reinterpret_cast<T*>(r.w);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
  }
}
template <class T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&x)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8], bool vec) {
  Raw8<T> r;
  uint32_t* w = reinterpret_cast<uint32_t*>(r.w);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
  }
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
  } else {
    const T* e = reinterpret_cast<const T*>(r.w);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = e[i];
  }
}
// element i of a row of `io` elements, and its store (the type is the same for the whole launch)
__device__ __forceinline__ float load_elem(const void* p, int64_t i, int io) {
  if (io == EL_F32) return static_cast<const float*>(p)[i];
  if (io == EL_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int64_t i, float x, int io) {
  if (io == EL_F32) static_cast<float*>(p)[i] = x;
  else if (io == EL_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

// 2^x, at most 2 ulp off; 0 for -inf
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- two f32 at a time ----------------------------------------------------------
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t both(float x) { return pair(x, x); }
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// numbers below 2^-126 become 0
__device__ __forceinline__ uint64_t mul2_ftz(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ void report(int* status, int code) {
  if (status) atomicExch(status, code);
}

// The pages a query position (or a run of them) can see: pages 0 .. n_sink_pages-1
// and pages first .. last, as one list of n entries.
struct SeenPages {
  int sink;   // leading pages that only the sinks need (0 when the window reaches them)
  int first;  // first page of the window
  int n;      // entries
  __device__ __forceinline__ int page(int i) const { return i < sink ? i : first + i - sink; }
};
// positions lo_pos .. hi_pos (0 <= lo_pos <= hi_pos)
__device__ __forceinline__ SeenPages seen_pages(int lo_pos, int hi_pos, int window, int n_sink) {
  SeenPages s;
  const int lo = window > 0 && lo_pos >= window ? lo_pos - window + 1 : 0;
  const int last = hi_pos / PG;
  s.first = lo / PG;
  const int sp = min((int64_t)last + 1, ((int64_t)n_sink + PG - 1) / PG);
  s.sink = min(sp, s.first);
  if (s.sink == s.first) s.sink = s.first = 0;  // one run from page 0
  s.n = s.sink + last - s.first + 1;
  return s;
}
__device__ __forceinline__ bool key_seen(int j, int p, int window, int n_sink) {
  return j <= p && (window == 0 || j > p - window || j < n_sink);
}

// Where q_start descends: bits of the lane's four starts that lie below one before them, in this lane, in the lanes
// before it or (top) in an earlier step, and the largest start so far.  Out of line, it is never called for a q_start
// that ascends.
static __device__ __noinline__ int2 begin_below(int a0, int a1, int a2, int a3, int top) {
  const int lane = threadIdx.x & 31, a[4] = {a0, a1, a2, a3};
  int upto = max(max(a0, a1), max(a2, a3));  // of this lane and those before it
  for (int d = 1; d < 32; d *= 2) {
    const int v = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto = max(upto, v);
  }
  int before = __shfl_up_sync(0xffffffffu, upto, 1);
  before = lane ? max(before, top) : top;
  unsigned below = 0;
  for (int i = 0; i < 4; ++i) {
    if (a[i] < before) below |= 1u << i;
    before = max(before, a[i]);
  }
  return make_int2((int)below, max(top, __shfl_sync(0xffffffffu, upto, 31)));
}

// Tile `idx` of the ragged batch: tiles of RT rows, sequence by sequence, the
// last tile of a sequence first (its rows see the most keys).  All lanes of
// the warp call it and get the same answer; seq = -1 past the last tile.
struct Tile {
  int seq, q0, n_q, row0;  // first token of the sequence, its tokens, first row
  int past;                // position of its first token
};
__device__ __forceinline__ Tile find_tile(const WindowAttnParams& p, int64_t idx, int RT) {
  constexpr int V = 4;  // sequences of a lane: one round trip to memory for 128 of them
  const int lane = threadIdx.x & 31;
  const int64_t group = p.n_head / p.n_head_kv;
  Tile t;
  t.seq = -1;
  bool descends = false;  // q_start went back: what begins below a start before it shares rows, and counts as bad
  int top = 0;            // then: the largest start so far
  for (int s0 = 0; s0 < p.n_seq; s0 += 32 * V) {
    const int s = s0 + lane * V;
    int at[V + 1], len[V], n[V];
    int64_t tiles[V], sum = 0;
#pragma unroll
    for (int i = 0; i <= V; ++i) at[i] = s + i <= p.n_seq ? p.q_start[s + i] : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) len[i] = s + i < p.n_seq ? p.kv_len[s + i] : 0;
    unsigned below = 0;  // bit i: begins below a start before it
    bool back = false;
#pragma unroll
    for (int i = 0; i < V; ++i) back = back || (s + i < p.n_seq && at[i + 1] < at[i]);
    descends = __any_sync(0xffffffffu, back) || descends;
    if (descends) {
      const int2 r = begin_below(at[0], at[1], at[2], at[3], top);
      below = r.x;
      top = r.y;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      n[i] = 0;
      if (s + i < p.n_seq) {
        if (at[i] < 0 || (below >> i & 1) || at[i + 1] < at[i] || at[i + 1] > p.n_tok || len[i] < 0 || (len[i] + (int64_t)PG - 1) / PG > p.max_pages)
          report(p.status, ERR_BAD_POS);  // nothing of this sequence is read or written
        else
          n[i] = at[i + 1] - at[i];
      }
      tiles[i] = (n[i] * group + RT - 1) / RT;
      sum += tiles[i];
    }
    int64_t incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, idx < incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      // the lane that holds it picks the sequence
      int64_t left = idx - (incl - sum), cnt = 0;
      int seq = 0, q0 = 0, nq = 0, kv = 0;
      bool found = false;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!found && left < tiles[i]) {
          found = true;
          seq = s + i;
          q0 = at[i];
          nq = n[i];
          kv = len[i];
          cnt = tiles[i];
        }
        if (!found) left -= tiles[i];
      }
      t.seq = __shfl_sync(0xffffffffu, seq, src);
      t.q0 = __shfl_sync(0xffffffffu, q0, src);
      t.n_q = __shfl_sync(0xffffffffu, nq, src);
      t.past = __shfl_sync(0xffffffffu, kv, src) - t.n_q;
      t.row0 = (int)((__shfl_sync(0xffffffffu, cnt, src) - 1 - __shfl_sync(0xffffffffu, left, src)) * RT);
      return t;
    }
    idx -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return t;
}
#endif

}  // namespace sfk
