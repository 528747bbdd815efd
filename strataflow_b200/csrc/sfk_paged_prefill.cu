// sfk_paged_prefill.cu -- attention of a ragged batch of prompts over the
// paged cache (causal, with an optional window and sinks).
//
//   token i of sequence s sits at position p = kv_len[s] - n_q(s) + i and sees
//   the keys of key_seen(): out = softmax(scale q K^T) V over them
//
// The query heads of one kv head read the same keys, so they are rows of one
// matrix: row r of a (sequence, kv head) is token r / G, head r % G.  A CTA
// takes a tile of rows and walks the key tiles its rows see with a running
// maximum, sum and output per row (f32).
#include "sfk_paged.cuh"

namespace sfk {
namespace {

// ---- CUDA cores: any cache type ------------------------------------------------------
// For f32 caches, and 32-bit rows over a bf16 cache or with heads of 256; the other
// prompts go to sfk_paged_prefill_tc.cu.  Bound by the multiply-adds and their shared loads
// (8 loads of 16 bytes to 64 multiply-adds): 2048 tokens, 32 heads of 128 over 8, f32:
// 1.51 ms, 23 TFLOP/s.
// 64 rows x 64 keys per step, 256 threads as 16 x 16: thread (ty, tx) owns rows
// ty + 16 i, keys tx + 16 j of the scores and dims 4 tx .. 4 tx + 3 of each 64
// of the output.  Everything is f32 in shared memory, rows padded by 16 bytes.
constexpr int FR = 64, FK = 64, FT = 256;

template <int HD>
struct FmaSmem {
  float q[FR][HD + 4], k[FK][HD + 4], v[FK][HD + 4];
  float p[FR][FK + 4];
};

template <class KV, int HD>
__global__ void __launch_bounds__(FT) prefill_fma_kernel(const __grid_constant__ WindowAttnParams p) {
  using Smem = FmaSmem<HD>;
  constexpr int NC = (HD + 63) / 64;  // chunks of 64 output dims
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int hk = blockIdx.y, G = p.n_head / p.n_head_kv;
  const Tile t = find_tile(p, blockIdx.x, FR);
  if (t.seq < 0) return;
  const int n_rows = (int)min((int64_t)FR, (int64_t)t.n_q * G - t.row0);
  for (int i = tid; i < FR * HD; i += FT) {
    const int r = i / HD, d = i % HD;
    float x = 0.f;
    if (r < n_rows) {
      const int tok = (t.row0 + r) / G, h = hk * G + (t.row0 + r) % G;
      x = load_elem(p.q, (int64_t)(t.q0 + tok) * p.q_stride + (int64_t)h * HD + d, p.io);
    }
    sm.q[r][d] = x;
  }
  const int p_lo = max(t.past + t.row0 / G, 0), p_hi = t.past + (t.row0 + n_rows - 1) / G;
  SeenPages sp;
  sp.n = 0;
  if (p_hi >= 0) sp = seen_pages(p_lo, p_hi, p.window, p.n_sink);
  int pos[4];
  float m[4], l[4], o[4][NC][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty + 16 * i;
    pos[i] = r < n_rows ? t.past + (t.row0 + r) / G : -1;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
  }
  for (int i0 = 0; i0 < sp.n; i0 += FK / PG) {
    __syncthreads();
    // four pages of keys and values; what no row sees is zero
    for (int i = tid; i < FK * HD / 8; i += FT) {
      const int key = i / (HD / 8), d = i % (HD / 8) * 8;
      float a[8] = {}, b[8] = {};
      const int e = i0 + key / PG;
      if (e < sp.n && sp.page(e) * PG + key % PG <= p_hi) {
        const int id = p.page_table[(int64_t)t.seq * p.max_pages + sp.page(e)];
        if (id >= 0 && id < p.n_pages) {
          const int64_t off = (((int64_t)id * p.n_head_kv + hk) * PG + key % PG) * HD + d;
          Raw8<KV> ra, rb;
          load8(ra, static_cast<const KV*>(p.k_pages) + off, true);
          load8(rb, static_cast<const KV*>(p.v_pages) + off, true);
          unpack8(ra, a);
          unpack8(rb, b);
        } else {
          report(p.status, ERR_BAD_PAGE);
        }
      }
#pragma unroll
      for (int x = 0; x < 8; x += 4) {
        *reinterpret_cast<float4*>(&sm.k[key][d + x]) = make_float4(a[x], a[x + 1], a[x + 2], a[x + 3]);
        *reinterpret_cast<float4*>(&sm.v[key][d + x]) = make_float4(b[x], b[x + 1], b[x + 2], b[x + 3]);
      }
    }
    __syncthreads();
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
      float4 q[4], k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(&sm.q[ty + 16 * i][d]);
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(&sm.k[tx + 16 * j][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = fmaf(q[i].x, k[j].x, s[i][j]);
          s[i][j] = fmaf(q[i].y, k[j].y, s[i][j]);
          s[i][j] = fmaf(q[i].z, k[j].z, s[i][j]);
          s[i][j] = fmaf(q[i].w, k[j].w, s[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = i0 + j;  // key tx of page entry i0 + j
        const bool see = e < sp.n && key_seen(sp.page(e) * PG + tx, pos[i], p.window, p.n_sink);
        s[i][j] = see ? s[i][j] * p.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int d = 1; d < 16; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float ms = mx == -INFINITY ? 0.f : mx;
      const float f = exp2_approx(m[i] - ms);
      m[i] = mx;
      l[i] *= f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][c][e] *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float pr = exp2_approx(s[i][j] - ms);
        l[i] += pr;
        sm.p[ty + 16 * i][tx + 16 * j] = pr;
      }
    }
    __syncwarp();  // rows ty + 16 i belong to one half of a warp
    for (int k0 = 0; k0 < FK; k0 += 4) {
      float pr[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(pr[i]) = *reinterpret_cast<const float4*>(&sm.p[ty + 16 * i][k0]);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (HD < 64 && tx >= HD / 4) continue;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const float4 v = *reinterpret_cast<const float4*>(&sm.v[k0 + kk][c * 64 + tx * 4]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (pr[i][kk] != 0.f) {  // a masked key's value, whatever it holds, is not used
              o[i][c][0] = fmaf(pr[i][kk], v.x, o[i][c][0]);
              o[i][c][1] = fmaf(pr[i][kk], v.y, o[i][c][1]);
              o[i][c][2] = fmaf(pr[i][kk], v.z, o[i][c][2]);
              o[i][c][3] = fmaf(pr[i][kk], v.w, o[i][c][3]);
            }
          }
        }
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int d = 1; d < 16; d *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
    const int r = ty + 16 * i;
    if (r >= n_rows) continue;
    const int tok = (t.row0 + r) / G, h = hk * G + (t.row0 + r) % G;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (HD < 64 && tx >= HD / 4) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        store_elem(p.out, ((int64_t)(t.q0 + tok) * p.n_head + h) * HD + c * 64 + tx * 4 + e,
                   pos[i] >= 0 ? o[i][c][e] / l[i] : 0.f, p.io);
    }
  }
}

template <class KV, int HD>
cudaError_t launch_fma(WindowAttnParams& p, cudaStream_t st) {
  const size_t smem = sizeof(FmaSmem<HD>);
  cudaError_t e = allow_smem<prefill_fma_kernel<KV, HD>>(smem);
  if (e != cudaSuccess) return e;
  const int64_t group = p.n_head / p.n_head_kv;
  const dim3 grid((unsigned)(p.n_tok * group / FR + p.n_seq), (unsigned)p.n_head_kv);
  prefill_fma_kernel<KV, HD><<<grid, FT, smem, st>>>(p);
  return cudaGetLastError();
}

template <class KV>
cudaError_t launch_kv(WindowAttnParams& p, int hd, cudaStream_t st) {
  switch (hd) {
    case 32: return launch_fma<KV, 32>(p, st);
    case 64: return launch_fma<KV, 64>(p, st);
    case 128: return launch_fma<KV, 128>(p, st);
    case 256: return launch_fma<KV, 256>(p, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_window_prefill(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st) {
  if (prefill_tc_takes(p, kv, hd)) return launch_prefill_tc(p, kv, hd, sm_count, st);
  if (kv == EL_F32) return launch_kv<float>(p, hd, st);
  if (kv == EL_F16) return launch_kv<__half>(p, hd, st);
  return launch_kv<__nv_bfloat16>(p, hd, st);
}

}  // namespace sfk
