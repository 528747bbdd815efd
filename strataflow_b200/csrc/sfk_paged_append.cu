// sfk_paged_append.cu -- the write side of a paged KV cache: the per-head norm
// of q and k, the position rotation, and the append of k and v, in one pass.
//
//   x' = x * rsqrt(mean_i x_i^2 + eps) * w                  (q and k, if w is given)
//   angle_i = position[axis_i] * freq_i                     i < n_rot / 2
//   (a, b) -> (a cos - b sin, a sin + b cos)                pairs (2i, 2i+1) or (i, i + n_rot/2)
//   q -> q_out; k, v -> row pos % 16 of page table[seq][pos / 16]
//
// Bound by memory: every element is read once and written once, a few
// operations on each.  The angles of a token are the same for all of its
// heads, so a CTA takes all heads of its tokens (or a share of them when
// there are few tokens) and computes each cosine and sine once.  The angle is
// formed and reduced in turns, in 64 bits: at position 1e5 an f32 product is
// already off by up to 4e-3 radians, and the 64-bit product and subtraction
// cost one thread per pair a few instructions.  A head row is spread over
// hd / 8 lanes of one warp, 16 bytes each for 16-bit types, so the norm and
// the partner of a half-split pair are warp shuffles.
#include "sfk_paged.cuh"

namespace sfk {
namespace {

constexpr int AT = 256;  // threads
constexpr int TPC_MAX = 16;

template <class IO, class KV, int P>
__global__ void __launch_bounds__(AT) append_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ float2 cs[];  // [tpc][n_rot / 2] cosine, sine
  __shared__ int s_pos[TPC_MAX], s_page[TPC_MAX];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * p.tpc;
  const int nt = min(p.tpc, p.n_tok - t0);
  const int rows = p.n_head + 2 * p.n_head_kv;
  const int lpr = p.lpr, sub = tid & (lpr - 1), e0 = sub * 8;
  const int rpp = AT / lpr;  // rows per pass
  const bool lane_on = e0 < p.hd;

  // 1. every row this thread takes is requested before anything waits
  Raw8<IO> raw[P];
  int tok[P], row[P];  // token within the CTA (-1: none), row within the token
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int slot = (i * gridDim.y + blockIdx.y) * rpp + tid / lpr;
    tok[i] = slot < nt * rows ? slot / rows : -1;
    row[i] = slot % rows;
    if (tok[i] >= 0 && lane_on) {
      const int64_t t = t0 + tok[i];
      if (row[i] < p.n_head)
        load8(raw[i], static_cast<const IO*>(p.q) + t * p.q_stride + (int64_t)row[i] * p.hd + e0, p.vec & 1);
      else if (row[i] < p.n_head + p.n_head_kv)
        load8(raw[i], static_cast<const IO*>(p.k) + t * p.k_stride + (int64_t)(row[i] - p.n_head) * p.hd + e0, p.vec & 2);
      else
        load8(raw[i], static_cast<const IO*>(p.v) + t * p.v_stride + (int64_t)(row[i] - p.n_head - p.n_head_kv) * p.hd + e0,
              p.vec & 4);
    }
  }
  // 2. the slot of each token, and its angles
  if (tid < nt) {
    const int t = t0 + tid;
    const int pos = p.pos[t];
    const int s = p.seq ? p.seq[t] : t;
    int page = -1, keep = pos;
    if (pos >= 0) {
      if (s < 0 || s >= p.n_seq) {
        report(p.status, ERR_BAD_ID);
        keep = -1;
      } else if (pos / PG >= p.max_pages) {
        report(p.status, ERR_BAD_POS);
        keep = -1;
      } else {
        page = p.page_table[(int64_t)s * p.max_pages + pos / PG];
        if (page < 0 || page >= p.n_pages) {
          report(p.status, ERR_BAD_PAGE);
          page = -1;
        }
      }
    }
    s_pos[tid] = keep;
    s_page[tid] = page;
  }
  const int half = p.n_rot / 2;
  for (int i = tid; i < nt * half; i += AT) {
    const int t = t0 + i / half, c = i % half;
    const int where = p.rope_pos ? p.rope_pos[(int64_t)p.axis[c] * p.n_tok + t] : p.pos[t];
    double turns = (double)where * (double)p.freqs[c] * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, co;
    sincospif(2.0f * (float)turns, &s, &co);
    cs[i] = make_float2(co, s);
  }
  __syncthreads();
  // 3. norm, rotation, stores.  The lanes of a row agree on every branch.
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const bool mine = tok[i] >= 0 && s_pos[max(tok[i], 0)] >= 0;
    const int tk = max(tok[i], 0);
    float x[8];
    if (mine && lane_on) {
      unpack8(raw[i], x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    }
    const bool is_q = row[i] < p.n_head, is_v = row[i] >= p.n_head + p.n_head_kv;
    const float* w = is_v ? nullptr : (is_q ? p.q_norm : p.k_norm);
    if (p.q_norm || p.k_norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
      for (int o = lpr / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (w && lane_on) {
        const float r = 1.0f / sqrtf(ss / (float)p.hd + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e0 + e];
      }
    }
    if (p.n_rot > 0) {
      const float2* a = cs + tk * half;
      if (p.neox) {
        // e0 .. e0+7 is wholly in the first or the second half (half % 8 == 0)
        const bool lo = e0 < half;
        const int d = half / 8;
        const int from = (lo ? sub + d : sub - d) & (lpr - 1);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(0xffffffffu, x[e], from, lpr);
        if (!is_v && mine && e0 < p.n_rot) {
          const float2* ae = a + (lo ? e0 : e0 - half);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = lo ? x[e] * ae[e].x - y[e] * ae[e].y : y[e] * ae[e].y + x[e] * ae[e].x;
        }
      } else if (!is_v && mine && e0 < p.n_rot) {
        const float2* ae = a + e0 / 2;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = x[2 * e], v = x[2 * e + 1];
          x[2 * e] = u * ae[e].x - v * ae[e].y;
          x[2 * e + 1] = u * ae[e].y + v * ae[e].x;
        }
      }
    }
    if (!mine || !lane_on) continue;
    const int64_t t = t0 + tk;
    if (is_q) {
      store8(static_cast<IO*>(p.q_out) + t * p.out_stride + (int64_t)row[i] * p.hd + e0, x, p.vec & 8);
    } else if (s_page[tk] >= 0) {
      const int h = row[i] - p.n_head - (is_v ? p.n_head_kv : 0);
      KV* base = static_cast<KV*>(is_v ? p.v_pages : p.k_pages);
      store8(base + (((int64_t)s_page[tk] * p.n_head_kv + h) * PG + s_pos[tk] % PG) * p.hd + e0, x, true);
    }
  }
}

template <class IO, class KV>
cudaError_t launch_t(AppendParams& p, int sm_count, cudaStream_t st) {
  const int rows = p.n_head + 2 * p.n_head_kv;
  p.lpr = 1;
  while (p.lpr * 8 < p.hd) p.lpr *= 2;
  const int rpp = AT / p.lpr;
  // Few rows per token: several tokens to a CTA, as long as every SM has work
  p.tpc = 1;
  while (p.tpc < TPC_MAX && (p.tpc + 1) * rows <= 2 * rpp && (int64_t)p.n_tok > (int64_t)(p.tpc + 1) * 4 * sm_count) ++p.tpc;
  const int passes = (p.tpc * rows + rpp - 1) / rpp;
  const int64_t groups = (p.n_tok + p.tpc - 1) / p.tpc;
  // Many tokens: up to four rows per thread in flight; few: one pass per CTA,
  // so that the heads of a token spread over the SMs.
  const int P = groups * passes <= 4 * sm_count ? 1 : (passes >= 3 ? 4 : passes);
  const dim3 grid((unsigned)groups, (unsigned)((passes + P - 1) / P));
  const size_t smem = sizeof(float2) * p.tpc * (p.n_rot / 2);
  if (P == 1) append_kernel<IO, KV, 1><<<grid, AT, smem, st>>>(p);
  else if (P == 2) append_kernel<IO, KV, 2><<<grid, AT, smem, st>>>(p);
  else append_kernel<IO, KV, 4><<<grid, AT, smem, st>>>(p);
  return cudaGetLastError();
}

template <class IO>
cudaError_t launch_io(AppendParams& p, int kv, int sm_count, cudaStream_t st) {
  if (kv == EL_F32) return launch_t<IO, float>(p, sm_count, st);
  if (kv == EL_F16) return launch_t<IO, __half>(p, sm_count, st);
  return launch_t<IO, __nv_bfloat16>(p, sm_count, st);
}

}  // namespace

cudaError_t launch_append(AppendParams& p, int io, int kv, int sm_count, cudaStream_t st) {
  if (io == EL_F32) return launch_io<float>(p, kv, sm_count, st);
  if (io == EL_F16) return launch_io<__half>(p, kv, sm_count, st);
  return launch_io<__nv_bfloat16>(p, kv, sm_count, st);
}

}  // namespace sfk
