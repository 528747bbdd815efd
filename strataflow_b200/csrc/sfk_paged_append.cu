// sfk_paged_append.cu -- the write side of a paged KV cache: the per-head norm
// of q and k, the position rotation, and the append of k and v, in one pass.
//
//   x' = x * rsqrt(mean_i x_i^2 + eps) * w                  (q and k, if w is given)
//   angle_i = position[axis_i] * freq_i                     i < n_rot / 2
//   (a, b) -> (a cos - b sin, a sin + b cos)                pairs (2i, 2i+1) or (i, i + n_rot/2)
//   q -> q_out; k, v -> row pos % 16 of page table[seq][pos / 16]
//
// Bound by memory: every element is read once and written once.  What stands in
// the way is the arithmetic, so it is folded: with r the row's reciprocal norm and
// y the partner of x, the weight and the rotation are
//   out_e = r (x_e A_e + y_e B_e),  A_e = w_e cos, B_e = -+ w_partner sin
// and A, B depend on the token alone.  A warp takes the heads of one token (or a
// share of them when there are few tokens): it makes the token's table in shared
// memory while its first rows are on their way, then walks the q, k and v heads, a
// row on hd / 8 lanes, 16 bytes each for 16-bit types, with the next PF loads under
// way.  The norm and the partner of a half-split pair are warp shuffles (of the
// words as loaded).  No warp waits for another, every address is a constant step
// from the last.  (A CTA to a token or several, rows dealt out by an index that
// runs over tokens and heads: 262 instructions a step and 147 us where this takes
// 66, 8192 tokens of 64 + 8 + 8 heads of 128 in bf16, both norms.)
// The angle is formed and reduced in turns, in 64 bits: at position 1e5 an f32
// product is already off by up to 4e-3 radians, and the 64-bit product and
// subtraction cost one lane per pair a few instructions.
#include "sfk_paged.cuh"

namespace sfk {
namespace {

constexpr int AW = 4;  // warps per CTA
constexpr int PF = 4;  // loads ahead

// LPR: lanes per row (8 elements each)
template <class IO, class KV, int LPR>
__global__ void __launch_bounds__(AW * 32) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int R = 32 / LPR;  // rows per step
  extern __shared__ __align__(16) float4 tables[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t item = (int64_t)blockIdx.x * AW + warp;
  const int64_t t = item / p.share;
  if (t >= p.n_tok) return;
  const int sub = lane % LPR, e0 = sub * 8, rr = lane / LPR;
  const bool lane_on = e0 < p.hd;
  const int nq = (p.n_head + R - 1) / R, nk = (p.n_head_kv + R - 1) / R, steps = nq + 2 * nk;

  const IO* qp = static_cast<const IO*>(p.q) + t * p.q_stride + rr * p.hd + e0;
  const IO* kp = static_cast<const IO*>(p.k) + t * p.k_stride + rr * p.hd + e0;
  const IO* vp = static_cast<const IO*>(p.v) + t * p.v_stride + rr * p.hd + e0;
  auto load = [&](Raw8<IO>& raw, int i) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(IO) / 2; ++k) raw.w[k] = make_uint4(0, 0, 0, 0);
    if (i < nq) {
      if (lane_on && i * R + rr < p.n_head) load8(raw, qp + i * R * p.hd, p.vec & 1);
    } else if (i < nq + nk) {
      if (lane_on && (i - nq) * R + rr < p.n_head_kv) load8(raw, kp + (i - nq) * R * p.hd, p.vec & 2);
    } else if (i < steps) {
      if (lane_on && (i - nq - nk) * R + rr < p.n_head_kv) load8(raw, vp + (i - nq - nk) * R * p.hd, p.vec & 4);
    }
  };
  const int first = (int)(item % p.share);
  Raw8<IO> next[PF];
#pragma unroll
  for (int k = 0; k < PF; ++k) load(next[k], first + k * p.share);

  // the token's slot
  const int pos = p.pos[t];
  if (pos < 0) return;
  const int sq = p.seq ? p.seq[t] : (int)t;
  if (sq < 0 || sq >= p.n_seq || pos / PG >= p.max_pages) {
    report(p.status, sq < 0 || sq >= p.n_seq ? ERR_BAD_ID : ERR_BAD_POS);
    return;
  }
  const int page = p.page_table[(int64_t)sq * p.max_pages + pos / PG];
  const bool page_ok = page >= 0 && page < p.n_pages;
  if (!page_ok) report(p.status, ERR_BAD_PAGE);
  // its table: (A, B) of element 8 i + j is float2 j % 2 of entry [j / 2][i], so that lanes read side by side
  const int half = p.n_rot / 2, lanes = p.hd / 8;
  const int kinds = p.q_norm == p.k_norm ? 1 : 2;
  float4* table = tables + warp * kinds * p.hd / 2;
  auto entry = [&](int k, int e) {
    return reinterpret_cast<float2*>(table + k * p.hd / 2 + (e % 8 / 2) * lanes + e / 8) + e % 2;
  };
  for (int c = lane; c < half; c += 32) {
    const int where = p.rope_pos ? p.rope_pos[(int64_t)p.axis[c] * p.n_tok + t] : pos;
    double turns = (double)where * (double)p.freqs[c] * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float sn, co;
    sincospif(2.0f * (float)turns, &sn, &co);
    const int a = p.neox ? c : 2 * c, b = p.neox ? c + half : 2 * c + 1;
    for (int k = 0; k < kinds; ++k) {
      const float* w = k ? p.k_norm : p.q_norm;
      const float wa = w ? w[a] : 1.f, wb = w ? w[b] : 1.f;
      *entry(k, a) = make_float2(wa * co, -wb * sn);
      *entry(k, b) = make_float2(wb * co, wa * sn);
    }
  }
  for (int e = p.n_rot + lane; e < p.hd; e += 32)
    for (int k = 0; k < kinds; ++k) {
      const float* w = k ? p.k_norm : p.q_norm;
      *entry(k, e) = make_float2(w ? w[e] : 1.f, 0.f);
    }
  __syncwarp();

  const float inv_hd = 1.0f / (float)p.hd;
  const bool turned = e0 < p.n_rot;  // past n_rot the partner, whatever it is, has no part
  // e0 .. e0+7 is wholly in the first or the second half (half % 8 == 0)
  const int from = (e0 < half ? sub + half / 8 : sub - half / 8) & (LPR - 1);
  IO* op = static_cast<IO*>(p.q_out) + t * p.out_stride + rr * p.hd + e0;
  const int64_t at = (((int64_t)page * p.n_head_kv + rr) * PG + pos % PG) * p.hd + e0;
  KV* kd = static_cast<KV*>(p.k_pages) + at;
  KV* vd = static_cast<KV*>(p.v_pages) + at;
  for (int i0 = first; i0 < steps; i0 += PF * p.share) {
    Raw8<IO> raw[PF];
#pragma unroll
    for (int k = 0; k < PF; ++k) raw[k] = next[k];
#pragma unroll
    for (int k = 0; k < PF; ++k) load(next[k], i0 + (PF + k) * p.share);
#pragma unroll
    for (int k = 0; k < PF; ++k) {
      const int i = i0 + k * p.share;
      if (i >= steps) break;
      float x[8];
      unpack8(raw[k], x);
      if (i >= nq + nk) {  // v: as it is
        const int h = (i - nq - nk) * R;
        if (lane_on && page_ok && h + rr < p.n_head_kv) store8(vd + (int64_t)h * PG * p.hd, x, true);
        continue;
      }
      const bool is_q = i < nq;
      float r = 1.f;
      if (is_q ? p.q_norm != nullptr : p.k_norm != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        r = rsqrtf(fmaf(ss, inv_hd, p.eps));
      }
      float y[8];  // partners
      if (p.neox && half > 0) {
        Raw8<IO> other;
#pragma unroll
        for (int j = 0; j < (int)sizeof(IO) / 2; ++j) {
          other.w[j].x = __shfl_sync(0xffffffffu, raw[k].w[j].x, from, LPR);
          other.w[j].y = __shfl_sync(0xffffffffu, raw[k].w[j].y, from, LPR);
          other.w[j].z = __shfl_sync(0xffffffffu, raw[k].w[j].z, from, LPR);
          other.w[j].w = __shfl_sync(0xffffffffu, raw[k].w[j].w, from, LPR);
        }
        unpack8(other, y);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
      }
      if (!lane_on) continue;
      const float4* ab = table + (is_q ? 0 : kinds - 1) * p.hd / 2 + sub;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 z = ab[e * lanes];
        x[2 * e] *= z.x;
        x[2 * e + 1] *= z.z;
        if (turned) {
          x[2 * e] = fmaf(y[2 * e], z.y, x[2 * e]);
          x[2 * e + 1] = fmaf(y[2 * e + 1], z.w, x[2 * e + 1]);
        }
        x[2 * e] *= r;
        x[2 * e + 1] *= r;
      }
      if (is_q) {
        if (i * R + rr < p.n_head) store8(op + i * R * p.hd, x, p.vec & 8);
      } else {
        const int h = (i - nq) * R;
        if (page_ok && h + rr < p.n_head_kv) store8(kd + (int64_t)h * PG * p.hd, x, true);
      }
    }
  }
}

template <class IO, class KV>
cudaError_t launch_t(AppendParams& p, int sm_count, cudaStream_t st) {
  const int lpr = p.hd <= 32 ? 4 : p.hd <= 64 ? 8 : p.hd <= 128 ? 16 : 32;
  const int R = 32 / lpr, steps = (p.n_head + R - 1) / R + 2 * ((p.n_head_kv + R - 1) / R);
  // warps per token: enough for 32 warps on every SM, a step each at least
  p.share = 1;
  while (p.share < steps && (int64_t)p.n_tok * p.share < (int64_t)32 * sm_count) ++p.share;
  const int64_t ctas = ((int64_t)p.n_tok * p.share + AW - 1) / AW;
  const size_t smem = (size_t)AW * (p.q_norm == p.k_norm ? 1 : 2) * p.hd * sizeof(float2);
  if (lpr == 4) append_kernel<IO, KV, 4><<<(unsigned)ctas, AW * 32, smem, st>>>(p);
  else if (lpr == 8) append_kernel<IO, KV, 8><<<(unsigned)ctas, AW * 32, smem, st>>>(p);
  else if (lpr == 16) append_kernel<IO, KV, 16><<<(unsigned)ctas, AW * 32, smem, st>>>(p);
  else append_kernel<IO, KV, 32><<<(unsigned)ctas, AW * 32, smem, st>>>(p);
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
