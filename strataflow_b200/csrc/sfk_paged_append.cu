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
// 63, 8192 tokens of 64 + 8 + 8 heads of 128 in bf16, both norms: 5.3 TB/s.)
// The angle is formed and reduced in turns, in 64 bits: at position 1e5 an f32
// product is already off by up to 4e-3 radians, and the 64-bit product and
// subtraction cost one lane per pair a few instructions.
#include "sfk_paged.cuh"

namespace sfk {
namespace {

constexpr int AW = 4;  // warps per CTA

// The heads of one kind (q, k or v) that a warp takes: steps first, first + share, ..., R rows each, a row on
// LPR lanes.  The loads of PF steps are under way before the caller's other work, PF more while PF are worked on.
template <class IO, class Out, int LPR, int PF>
struct HeadLoop {
  static constexpr int R = 32 / LPR;
  const IO* src;    // this lane's elements of its row of the first step
  Out* dst;
  int64_t src_step, dst_step;  // elements from step to step
  int left, left_step;         // rows from this lane's row on, this one included (<= 0: none), and their change
  bool in_vec, out_vec;
  Raw8<IO> next[PF];

  __device__ __forceinline__ void load(Raw8<IO>& raw, int ahead) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(IO) / 2; ++k) raw.w[k] = make_uint4(0, 0, 0, 0);
    if (left - ahead * left_step > 0) load8(raw, src + ahead * src_step, in_vec);
  }
  // n rows of hd elements, `src` / `dst` of this lane's row of step 0; a lane that has no part of a row: on = false
  __device__ __forceinline__ void start(const IO* src0, Out* dst0, int64_t dst_row, int n, int hd, int first, int share,
                                        int rr, bool on, bool iv, bool ov) {
    src = src0 + (int64_t)first * R * hd;
    dst = dst0 + (int64_t)first * R * dst_row;
    src_step = (int64_t)share * R * hd;
    dst_step = (int64_t)share * R * dst_row;
    left = on ? n - first * R - rr : 0;
    left_step = share * R;
    in_vec = iv;
    out_vec = ov;
#pragma unroll
    for (int k = 0; k < PF; ++k) load(next[k], k);
  }
  // f(words as loaded, out[8]) of every row; the whole warp runs as many steps as its first row has
  template <class F>
  __device__ __forceinline__ void run(bool store_on, F f) {
    while (__any_sync(0xffffffffu, left > 0)) {
      Raw8<IO> raw[PF];
#pragma unroll
      for (int k = 0; k < PF; ++k) raw[k] = next[k];
#pragma unroll
      for (int k = 0; k < PF; ++k) load(next[k], PF + k);
#pragma unroll
      for (int k = 0; k < PF; ++k) {
        float x[8];
        f(raw[k], x);
        if (store_on && left > 0) store8(dst, x, out_vec);
        left -= left_step;
        src += src_step;
        dst += dst_step;
      }
    }
  }
};

// LPR: lanes per row (8 elements each); FULL: hd is 8 LPR
template <class IO, class KV, int LPR, bool FULL>
__global__ void __launch_bounds__(AW * 32, 5) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int R = 32 / LPR, PF = sizeof(IO) == 2 ? 4 : 2;
  extern __shared__ __align__(16) float4 tables[];
  const int hd = FULL ? 8 * LPR : p.hd;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t item = (int64_t)blockIdx.x * AW + warp;
  const int64_t t = item / p.share;
  if (t >= p.n_tok) return;
  const int sub = lane % LPR, e0 = sub * 8, rr = lane / LPR;
  const bool lane_on = FULL || e0 < hd;
  // the steps of the three kinds are dealt out over the `share` warps of the token as one list
  const int share = p.share, first = (int)(item % share);
  const int nq = (p.n_head + R - 1) / R, nk = (p.n_head_kv + R - 1) / R;
  const int first_k = (first + share - nq % share) % share, first_v = (first_k + share - nk % share) % share;
  const int own = rr * hd + e0;
  const int pos = p.pos[t];
  HeadLoop<IO, KV, LPR, PF> k, v;
  HeadLoop<IO, IO, LPR, PF> q;
  v.start(static_cast<const IO*>(p.v) + t * p.v_stride + own, nullptr, (int64_t)PG * hd, p.n_head_kv, hd, first_v, share,
          rr, lane_on, p.vec & 4, true);
  k.start(static_cast<const IO*>(p.k) + t * p.k_stride + own, nullptr, (int64_t)PG * hd, p.n_head_kv, hd, first_k, share,
          rr, lane_on, p.vec & 2, true);
  q.start(static_cast<const IO*>(p.q) + t * p.q_stride + own, static_cast<IO*>(p.q_out) + t * p.out_stride + own, hd,
          p.n_head, hd, first, share, rr, lane_on, p.vec & 1, p.vec & 8);

  // the token's slot
  if (pos < 0) return;
  const int sq = p.seq ? p.seq[t] : (int)t;
  if (sq < 0 || sq >= p.n_seq || pos / PG >= p.max_pages) {
    report(p.status, sq < 0 || sq >= p.n_seq ? ERR_BAD_ID : ERR_BAD_POS);
    return;
  }
  const int page = p.page_table[(int64_t)sq * p.max_pages + pos / PG];
  const bool page_ok = page >= 0 && page < p.n_pages;
  if (!page_ok) report(p.status, ERR_BAD_PAGE);
  // its table: entry [j / 2][i] is A of elements 8 i + j and 8 i + j + 1 (j even), then their B: lanes read side by side
  const int half = p.n_rot / 2, lanes = hd / 8;
  const int kinds = p.q_norm == p.k_norm ? 1 : 2;
  float4* table = tables + warp * kinds * hd / 2;
  auto put = [&](int kind, int e, float a, float b) {
    float* at = reinterpret_cast<float*>(table + kind * hd / 2 + (e % 8 / 2) * lanes + e / 8) + e % 2;
    at[0] = a;
    at[2] = b;
  };
#pragma unroll 2
  for (int c = lane; c < half; c += 32) {
    const int a = p.neox ? c : 2 * c, b = p.neox ? c + half : 2 * c + 1;
    // every load before the arithmetic
    const float qa = p.q_norm ? __ldg(p.q_norm + a) : 1.f, qb = p.q_norm ? __ldg(p.q_norm + b) : 1.f;
    const float ka = kinds > 1 && p.k_norm ? __ldg(p.k_norm + a) : 1.f, kb = kinds > 1 && p.k_norm ? __ldg(p.k_norm + b) : 1.f;
    const float freq = __ldg(p.freqs + c);
    const int where = p.rope_pos ? __ldg(p.rope_pos + (int64_t)p.axis[c] * p.n_tok + t) : pos;
    double turns = (double)where * (double)freq * 0.15915494309189533577;  // 1 / (2 pi)
    turns -= rint(turns);
    float sn, co;
    sincospif(2.0f * (float)turns, &sn, &co);
    put(0, a, qa * co, -qb * sn);
    put(0, b, qb * co, qa * sn);
    if (kinds > 1) {
      put(1, a, ka * co, -kb * sn);
      put(1, b, kb * co, ka * sn);
    }
  }
  for (int e = p.n_rot + lane; e < hd; e += 32)
    for (int kind = 0; kind < kinds; ++kind) {
      const float* w = kind ? p.k_norm : p.q_norm;
      put(kind, e, w ? __ldg(w + e) : 1.f, 0.f);
    }
  __syncwarp();

  const int64_t at = (((int64_t)page * p.n_head_kv + rr) * PG + pos % PG) * hd + e0;
  v.dst = static_cast<KV*>(p.v_pages) + at + (int64_t)first_v * R * PG * hd;
  v.run(page_ok, [](const Raw8<IO>& raw, float (&x)[8]) { unpack8(raw, x); });

  const float inv_hd = 1.0f / (float)hd, eps = p.eps;
  const bool turned = e0 < p.n_rot;  // past n_rot the partner, whatever it is, has no part
  const bool apart = p.neox && half > 0;
  // e0 .. e0+7 is wholly in the first or the second half (half % 8 == 0)
  const int from = (e0 < half ? sub + half / 8 : sub - half / 8) & (LPR - 1);
  auto turn = [&](const Raw8<IO>& raw, float (&x)[8], bool norm, const float4* ab) {
    unpack8(raw, x);
    float r = 1.f;
    if (norm) {
      uint64_t s2 = mul2(pair(x[0], x[1]), pair(x[0], x[1]));
#pragma unroll
      for (int e = 2; e < 8; e += 2) s2 = fma2(pair(x[e], x[e + 1]), pair(x[e], x[e + 1]), s2);
      float ss, s1;
      unpair(s2, ss, s1);
      ss += s1;
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      r = rsqrtf(fmaf(ss, inv_hd, eps));
    }
    float y[8];  // partners
    if (apart) {
      Raw8<IO> other;
#pragma unroll
      for (int j = 0; j < (int)sizeof(IO) / 2; ++j) {
        other.w[j].x = __shfl_sync(0xffffffffu, raw.w[j].x, from, LPR);
        other.w[j].y = __shfl_sync(0xffffffffu, raw.w[j].y, from, LPR);
        other.w[j].z = __shfl_sync(0xffffffffu, raw.w[j].z, from, LPR);
        other.w[j].w = __shfl_sync(0xffffffffu, raw.w[j].w, from, LPR);
      }
      unpack8(other, y);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
    }
    const uint64_t rr2 = both(r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 z = lane_on ? ab[e * lanes] : make_float4(0.f, 0.f, 0.f, 0.f);
      uint64_t o = mul2(pair(x[2 * e], x[2 * e + 1]), pair(z.x, z.y));
      if (turned) o = fma2(pair(y[2 * e], y[2 * e + 1]), pair(z.z, z.w), o);
      unpair(mul2(o, rr2), x[2 * e], x[2 * e + 1]);
    }
  };
  const float4* ab_q = table + sub;
  const float4* ab_k = ab_q + (kinds - 1) * hd / 2;
  k.dst = static_cast<KV*>(p.k_pages) + at + (int64_t)first_k * R * PG * hd;
  const bool norm_k = p.k_norm != nullptr, norm_q = p.q_norm != nullptr;
  k.run(page_ok, [&](const Raw8<IO>& raw, float (&x)[8]) { turn(raw, x, norm_k, ab_k); });
  q.run(true, [&](const Raw8<IO>& raw, float (&x)[8]) { turn(raw, x, norm_q, ab_q); });
}

template <class IO, class KV>
cudaError_t launch_t(AppendParams& p, int sm_count, cudaStream_t st) {
  const int lpr = p.hd <= 32 ? 4 : p.hd <= 64 ? 8 : p.hd <= 128 ? 16 : 32;
  const int R = 32 / lpr, steps = (p.n_head + R - 1) / R + 2 * ((p.n_head_kv + R - 1) / R);
  // warps per token: one wave of 20 warps on every SM, two steps each at least (each warp makes the table)
  const int64_t wave = (int64_t)20 * sm_count / p.n_tok;
  p.share = (int)(wave < 1 ? 1 : wave < (steps + 1) / 2 ? wave : (steps + 1) / 2);
  const int64_t ctas = ((int64_t)p.n_tok * p.share + AW - 1) / AW;
  const size_t smem = (size_t)AW * (p.q_norm == p.k_norm ? 1 : 2) * p.hd * sizeof(float2);
  auto launch = [&](void (*kernel)(AppendParams)) {
    return launch_own(kernel, dim3((unsigned)ctas), AW * 32, smem, st, p);
  };
  if (p.hd == 64) return launch(append_kernel<IO, KV, 8, true>);
  if (p.hd == 128) return launch(append_kernel<IO, KV, 16, true>);
  if (lpr == 4) return launch(append_kernel<IO, KV, 4, false>);
  if (lpr == 8) return launch(append_kernel<IO, KV, 8, false>);
  if (lpr == 16) return launch(append_kernel<IO, KV, 16, false>);
  return launch(append_kernel<IO, KV, 32, false>);
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
