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
#include <type_traits>

#include "sfk_paged.cuh"

namespace sfk {
namespace {

// ---- CUDA cores: any cache type ------------------------------------------------------
// For f32 caches, and 32-bit rows over a bf16 cache or with heads of 256; the other
// prompts go to sfk_paged_prefill_tc.cu.  Bound by the multiply-adds, two to an
// instruction, and the softmax between them: 2048 tokens, 32 heads of 128 over 8, f32:
// 1.30 ms, 27 TFLOP/s; at 8048 keys 6.9 ms, 34 TFLOP/s.  (One multiply-add an instruction
// and one CTA to an SM: 1.52 and 9.0 ms.)
// 64 rows x 64 keys per step, 256 threads as 16 x 16: thread (ty, tx) owns rows
// ty + 16 i, keys tx + 16 j of the scores and dims 4 tx .. 4 tx + 3 of each 64
// of the output.  Everything is f32 in shared memory, rows padded by 16 bytes.
constexpr int FR = 64, FK = 64, FT = 256;

template <int HD>
struct FmaSmem {
  // Of wide heads K and V take turns in one place, so that two CTAs of 128 fit an SM and one loads while the other
  // multiplies; of narrow ones they arrive together, in one round trip.
  static constexpr bool TURNS = HD >= 128;
  float q[FR][HD + 4], k[FK][HD + 4], v_own[TURNS ? 1 : FK][HD + 4];
  float p[FR][FK + 4];
  __device__ float (*v())[HD + 4] { return TURNS ? k : v_own; }
};

template <class KV, int HD>
__global__ void __launch_bounds__(FT, HD > 128 ? 1 : 2) prefill_fma_kernel(const __grid_constant__ WindowAttnParams p) {
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
  float m[4], l[4];
  uint64_t o[4][NC][2];  // two dims each
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty + 16 * i;
    pos[i] = r < n_rows ? t.past + (t.row0 + r) / G : -1;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[i][c][0] = o[i][c][1] = both(0.f);
  }
  // Four pages of one pool, or of both; what no row sees is zero.  Returns whether a number of this thread's last pool
  // is infinite or NaN.
  auto load = [&](int i0, const void* pages, float (*dst)[HD + 4], auto both_pools) {
    constexpr int N = decltype(both_pools)::value ? 2 : 1;
    bool odd = false;
#pragma unroll 2
    for (int i = tid; i < FK * HD / 8; i += FT) {
      const int key = i / (HD / 8), d = i % (HD / 8) * 8;
      float a[N][8] = {};
      const int e = i0 + key / PG;
      if (e < sp.n && sp.page(e) * PG + key % PG <= p_hi) {
        const int id = p.page_table[(int64_t)t.seq * p.max_pages + sp.page(e)];
        if (id >= 0 && id < p.n_pages) {
          const int64_t off = (((int64_t)id * p.n_head_kv + hk) * PG + key % PG) * HD + d;
          Raw8<KV> raw[N];
#pragma unroll
          for (int k = 0; k < N; ++k) load8(raw[k], static_cast<const KV*>(k ? p.v_pages : pages) + off, true);
#pragma unroll
          for (int k = 0; k < N; ++k) unpack8(raw[k], a[k]);
        } else {
          report(p.status, ERR_BAD_PAGE);
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float* to = k ? &sm.v()[key][d] : &dst[key][d];
        *reinterpret_cast<float4*>(to) = make_float4(a[k][0], a[k][1], a[k][2], a[k][3]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(a[k][4], a[k][5], a[k][6], a[k][7]);
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) odd = odd || !(fabsf(a[N - 1][x]) < INFINITY);
    }
    return odd;
  };
  const int row_lo = n_rows < FR ? -1 : t.past + t.row0 / G;  // a row of the tile that is none sees nothing
  for (int i0 = 0; i0 < sp.n; i0 += FK / PG) {
    __syncthreads();
    bool odd = load(i0, p.k_pages, sm.k, std::bool_constant<!Smem::TURNS>());
    odd = __syncthreads_or(odd);
    uint64_t s2[4][4];  // the sums of even and of odd dims
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s2[i][j] = both(0.f);
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
      ulonglong2 q[4], k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const ulonglong2*>(&sm.q[ty + 16 * i][d]);
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const ulonglong2*>(&sm.k[tx + 16 * j][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s2[i][j] = fma2(q[i].y, k[j].y, fma2(q[i].x, k[j].x, s2[i][j]));
    }
    if (Smem::TURNS) {
      __syncthreads();
      odd = load(i0, p.v_pages, sm.v(), std::false_type());
    }
    // all keys seen by all rows (7.2 ms for the 8048 keys below where each key asks)
    const bool inner = i0 >= sp.sink && i0 + FK / PG <= sp.n && sp.page(i0 + FK / PG - 1) * PG + PG - 1 <= row_lo &&
                       (p.window == 0 || sp.page(i0) * PG > p_hi - p.window);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = m[i], s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = i0 + j;  // key tx of page entry i0 + j
        const bool see = inner || (e < sp.n && key_seen(sp.page(e) * PG + tx, pos[i], p.window, p.n_sink));
        float even, odd;
        unpair(s2[i][j], even, odd);
        s[j] = see ? (even + odd) * p.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[j]);
      }
#pragma unroll
      for (int d = 1; d < 16; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float ms = mx == -INFINITY ? 0.f : mx;
      const float f = exp2_approx(m[i] - ms);
      m[i] = mx;
      l[i] *= f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        o[i][c][0] = mul2(o[i][c][0], both(f));
        o[i][c][1] = mul2(o[i][c][1], both(f));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float pr = exp2_approx(s[j] - ms);
        l[i] += pr;
        sm.p[ty + 16 * i][tx + 16 * j] = pr;
      }
    }
    if (Smem::TURNS) odd = __syncthreads_or(odd);  // V has arrived
    else __syncwarp();                             // rows ty + 16 i belong to one half of a warp
    // A masked key's weight is 0, which takes its value out unless that is infinite or NaN: only then each product
    // asks (2048 tokens at 8048 keys, 32 heads of 128, f32: 6.8 ms, 8.7 ms where all ask).
    auto add = [&](auto ask) {
#pragma unroll 1
      for (int k0 = 0; k0 < FK; k0 += 4) {
        float pr[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(pr[i]) = *reinterpret_cast<const float4*>(&sm.p[ty + 16 * i][k0]);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            if (HD < 64 && tx >= HD / 4) continue;
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.v()[k0 + kk][c * 64 + tx * 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!decltype(ask)::value || pr[i][kk] != 0.f) {
                o[i][c][0] = fma2(both(pr[i][kk]), v.x, o[i][c][0]);
                o[i][c][1] = fma2(both(pr[i][kk]), v.y, o[i][c][1]);
              }
          }
        }
      }
    };
    if (odd) add(std::true_type());
    else add(std::false_type());
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
      float x[4];
      unpair(o[i][c][0], x[0], x[1]);
      unpair(o[i][c][1], x[2], x[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        store_elem(p.out, ((int64_t)(t.q0 + tok) * p.n_head + h) * HD + c * 64 + tx * 4 + e,
                   pos[i] >= 0 ? x[e] / l[i] : 0.f, p.io);
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
  return launch_own(prefill_fma_kernel<KV, HD>, grid, FT, smem, st, p);
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
