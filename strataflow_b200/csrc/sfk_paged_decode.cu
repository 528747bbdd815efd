// sfk_paged_decode.cu -- attention of one new token of each sequence over the
// keys it sees in the paged cache (window and sinks), split over the keys and
// joined.
//
//   s_j = scale q . k_j  for the seen keys j;  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
//
// Bound by memory: each seen key and value is read once for 8 query heads of its
// kv head (of more, every 8 read it again).  The seen pages of one (sequence, kv
// head, 8 query heads) are split over CTAs; each warp takes every W-th page of its
// CTA's run with a running maximum, sum and output of its own (f32).  The partials
// of the warps meet in shared memory, those of the CTAs
//   - in the distributed shared memory of a cluster of up to 8 (no scratch, one
//     launch), or,
//   - where the batch is too small for such clusters to fill the GPU, in the
//     caller's workspace, joined by a second kernel that is already resident when
//     the first ends.
#include <cooperative_groups.h>

#include <type_traits>

#include "sfk_paged.cuh"
#include "sfk_paged_map.cuh"

namespace sfk {
namespace {

namespace cg = cooperative_groups;


// Bounded wait of a whole warp for a slot (about a second); one answer for all lanes.
__device__ __forceinline__ bool wait_slot(uint64_t* bar, uint32_t parity, int* status) {
  bool ok = mbar_try_wait(bar, parity);
  if (!ok) {
    const long long t0 = clock64();
    while (!(ok = mbar_try_wait(bar, parity)) && clock64() - t0 < (1ll << 31)) {
    }
    if (!ok) report(status, ERR_TIMEOUT);
  }
  return __all_sync(0xffffffffu, ok);
}

// The workspace: o [n_seq * n_head][parts][HD], then (m, l) [n_seq * n_head][parts]
template <int HD>
__device__ __forceinline__ float* partial_o(const WindowAttnParams& p, int seq, int head, int part) {
  return p.partial + (((int64_t)seq * p.n_head + head) * p.parts + part) * HD;
}
template <int HD>
__device__ __forceinline__ float2* partial_ml(const WindowAttnParams& p, int seq, int head, int part) {
  return reinterpret_cast<float2*>(p.partial + (int64_t)p.n_seq * p.n_head * p.parts * HD) +
         ((int64_t)seq * p.n_head + head) * p.parts + part;
}
// One query head: warp w adds parts w, w + 8, ..., the warps meet in shared memory
// (a fixed order: the same bits each time).  Launched while the parts are
// computed (programmatic dependent launch); waits for all of them.
constexpr int JW = 8;  // warps
template <int HD>
__global__ void __launch_bounds__(JW * 32) join_kernel(const __grid_constant__ WindowAttnParams p) {
  constexpr int E = HD / 32;
  extern __shared__ float weight[];  // [parts]
  __shared__ float red[JW], lsum[JW], os[JW][HD];
  const int seq = blockIdx.x / p.n_head, head = blockIdx.x % p.n_head;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int pos = p.pos[seq];
  pdl_wait();
  const float2* ml = partial_ml<HD>(p, seq, head, 0);
  const float* po = partial_o<HD>(p, seq, head, 0) + lane * E;
  float m = -INFINITY;
  for (int c = tid; c < p.parts; c += JW * 32) m = fmaxf(m, ml[c].x);
  m = warp_max(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < JW; ++w) m = fmaxf(m, red[w]);
  if (m == -INFINITY) m = 0.f;
  float l = 0.f;
  for (int c = tid; c < p.parts; c += JW * 32) {
    const float2 x = ml[c];
    const float f = exp2_approx(x.x - m);
    weight[c] = f;
    l += x.y * f;
  }
  l = warp_sum(l);
  if (lane == 0) lsum[warp] = l;
  __syncthreads();
  float o[E] = {};
#pragma unroll 4
  for (int c = warp; c < p.parts; c += JW) {
    float x[E];
    if constexpr (E % 4 == 0) {
#pragma unroll
      for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(x + e) = *reinterpret_cast<const float4*>(po + (int64_t)c * HD + e);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = po[(int64_t)c * HD + e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(x[e], weight[c], o[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) os[warp][lane * E + e] = o[e];
  __syncthreads();
  if (tid < HD) {
    float sum = 0.f, ls = 0.f;
#pragma unroll
    for (int w = 0; w < JW; ++w) {
      sum += os[w][tid];
      ls += lsum[w];
    }
    store_elem(p.out, ((int64_t)seq * p.n_head + head) * HD + tid, pos >= 0 && pos / PG < p.max_pages ? sum / ls : 0.f, p.io);
  }
}

// ---- join -----------------------------------------------------------------------
// Every warp's partial (m, l, o) of R rows to the output.  m is in units of
// log2; a partial without keys has m = -inf, l = 0, o = 0.
template <int R, int HD, int DW>
struct JoinSmem {
  float o[DW][R][HD];
  float m[DW][R], l[DW][R];
  float co[R][HD];  // the CTA's partial
  float cm[R], cl[R];
};

template <int R, int HD, int DW>
__device__ void join_and_store(JoinSmem<R, HD, DW>& sm, const WindowAttnParams& p, int seq, int head0, int n_rows, bool any) {
  constexpr int DT = DW * 32;
  cg::cluster_group cl = cg::this_cluster();
  const int C = p.partial ? 1 : p.parts, rank = C > 1 ? (int)cl.block_rank() : 0;
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid < R) {
    float m = -INFINITY;
    for (int w = 0; w < DW; ++w) m = fmaxf(m, sm.m[w][tid]);
    const float ms = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int w = 0; w < DW; ++w) {
      const float f = exp2_approx(sm.m[w][tid] - ms);
      l += sm.l[w][tid] * f;
      sm.m[w][tid] = f;
    }
    sm.cm[tid] = m;
    sm.cl[tid] = l;
  }
  __syncthreads();
  for (int i = tid; i < n_rows * HD; i += DT) {
    const int r = i / HD, d = i % HD;
    float o = 0.f;
    for (int w = 0; w < DW; ++w) o += sm.o[w][r][d] * sm.m[w][r];
    if (p.partial) partial_o<HD>(p, seq, head0 + r, blockIdx.x % p.parts)[d] = o;
    else sm.co[r][d] = o;
  }
  if (p.partial) {
    if (tid < n_rows) *partial_ml<HD>(p, seq, head0 + tid, blockIdx.x % p.parts) = make_float2(sm.cm[tid], sm.cl[tid]);
    return;
  }
  if (C > 1) cl.sync();
  else __syncthreads();
  // output i of the rows belongs to CTA i / per, which adds the partials in rank order
  const int n = n_rows * HD, per = (n + C - 1) / C;
  for (int i = rank * per + tid; i < min(n, rank * per + per); i += DT) {
    const int r = i / HD, d = i % HD;
    float o, l;
    if (C == 1) {
      o = sm.co[r][d];
      l = sm.cl[r];
    } else {
      float m = -INFINITY;
      for (int c = 0; c < C; ++c) m = fmaxf(m, *cl.map_shared_rank(&sm.cm[r], c));
      if (m == -INFINITY) m = 0.f;
      o = l = 0.f;
      for (int c = 0; c < C; ++c) {
        const float f = exp2_approx(*cl.map_shared_rank(&sm.cm[r], c) - m);
        l += *cl.map_shared_rank(&sm.cl[r], c) * f;
        o += *cl.map_shared_rank(&sm.co[r][d], c) * f;
      }
    }
    store_elem(p.out, ((int64_t)seq * p.n_head + head0 + r) * HD + d, any ? o / l : 0.f, p.io);
  }
  if (C > 1) cl.sync();  // nobody leaves while its shared memory is read
}

// What a CTA works on.
struct Work {
  int seq, hk, head0, n_rows;  // query heads head0 .. head0 + n_rows - 1
  int pos;                     // -1: sees nothing
  SeenPages sp;
  int i0, i1;                  // entries of the page list
};
template <int R>
__device__ __forceinline__ Work find_work(const WindowAttnParams& p) {
  Work w;
  const int group = p.n_head / p.n_head_kv, tiles = (group + R - 1) / R;
  const int rank = blockIdx.x % p.parts;
  const int pair = blockIdx.x / p.parts;
  w.hk = pair / tiles;
  const int tile = pair % tiles;
  w.head0 = w.hk * group + tile * R;
  w.n_rows = min(R, group - tile * R);
  w.seq = blockIdx.y;
  w.pos = p.pos[w.seq];
  w.sp.n = w.sp.sink = w.sp.first = 0;
  if (w.pos >= 0 && w.pos / PG >= p.max_pages) {  // outside the table: no access, report
    report(p.status, ERR_BAD_POS);
    w.pos = -1;
  }
  if (w.pos >= 0) w.sp = seen_pages(w.pos, w.pos, p.window, p.n_sink);
  // runs that differ by a page at most
  w.i0 = (int)((int64_t)w.sp.n * rank / p.parts);
  w.i1 = (int)((int64_t)w.sp.n * (rank + 1) / p.parts);
  return w;
}
// the page id of list entry i, or -1
__device__ __forceinline__ int page_id(const WindowAttnParams& p, const Work& w, int i) {
  const int id = p.page_table[(int64_t)w.seq * p.max_pages + w.sp.page(i)];
  if (id >= 0 && id < p.n_pages) return id;
  report(p.status, ERR_BAD_PAGE);
  return -1;
}

// ---- CUDA cores: any cache type -----------------------------------------------------
// A warp takes a page at a time.  K and V of a page and head are contiguous: each
// arrives by one bulk copy in a ring of slots that the warp has to itself (K, V, K,
// V, ...).  Scores: lane (g, t) multiplies four dims of every 16 of keys g and g + 8
// by the query rows in shared memory; odd g take the two halves of 32 dims in the
// other order, so that two keys' rows never meet in a bank.  Values: the lane owns
// HD / 32 output dims.  64 multiply-adds to 10 shared loads.
// Sixteen sequences of 4096 keys, 32 heads of 128 over 8, f32: 133 us, 4.0 TB/s; a bf16
// cache of half the bytes 129 us.  So memory is not what binds it: the ring leaves room
// for two CTAs to an SM, two warps to a scheduler, which wait for shared loads and fixed
// latencies half of the time (issue slots 0.47 busy), 8 query rows are computed where four
// heads need 4, and 256 CTAs on 296 places leave a seventh of them empty.
template <class KV, int HD>
struct CcCfg {
  static constexpr int R = 8, DW = 4;
  static constexpr int UNIT = PG * HD * (int)sizeof(KV);  // bytes of a page's K or V
  static constexpr int SLOTS = UNIT <= 4096 ? 6 : 3;
};
template <class KV, int HD>
struct CcSmem {
  using C = CcCfg<KV, HD>;
  union {
    uint8_t ring[C::DW][C::SLOTS][C::UNIT];
    JoinSmem<C::R, HD, C::DW> join;
  };
  float q[C::R][HD];
  float p[C::DW][C::R][PG];
  uint64_t full[C::DW][C::SLOTS];
};
template <class KV>
__device__ __forceinline__ float4 lds4(const KV* p) {
  if constexpr (sizeof(KV) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    if constexpr (std::is_same<KV, __nv_bfloat16>::value)
      return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                         __uint_as_float(w.y & 0xffff0000u));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

template <class KV, int HD>
__global__ void __launch_bounds__(CcCfg<KV, HD>::DW * 32) decode_cc_kernel(const __grid_constant__ WindowAttnParams p) {
  using C = CcCfg<KV, HD>;
  using Smem = CcSmem<KV, HD>;
  constexpr int R = C::R, E = HD / 32, DW = C::DW, DT = DW * 32, S = C::SLOTS;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  if (p.partial) pdl_launch_dependents();
  const Work w = find_work<R>(p);
  const int mine = (w.i1 - w.i0 - warp + DW - 1) / DW;  // pages of this warp (<= 0: none)
  if (lane == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  // ids of this warp's entries i0 + warp + DW k, k = ids_at .. ids_at + 31; -1: outside the pool
  int ids = -1, ids_at = -32;
  unsigned bad = 0;  // bit k % 8: page k is outside the pool
  auto issue = [&](int j) {  // unit j: K (even) or V (odd) of page j / 2
    const int k = j / 2;
    if (k >= mine) return;
    if (k - ids_at >= 32) {
      const int i = w.i0 + warp + DW * (k + lane);
      ids = i < w.i1 ? page_id(p, w, i) : -1;
      ids_at = k;
    }
    const int id = __shfl_sync(0xffffffffu, ids, k - ids_at);
    bad = id < 0 ? bad | 1u << (k % 8) : bad & ~(1u << (k % 8));
    if (lane == 0) {
      uint64_t* bar = &sm.full[warp][j % S];
      if (id < 0) {
        mbar_arrive(bar);
      } else {
        mbar_arrive_expect_tx(bar, C::UNIT);
        bulk_g2s(sm.ring[warp][j % S],
                 static_cast<const KV*>(j & 1 ? p.v_pages : p.k_pages) + ((int64_t)id * p.n_head_kv + w.hk) * PG * HD,
                 C::UNIT, bar);
      }
    }
  };
  for (int j = 0; j < S; ++j) issue(j);
  for (int i = tid; i < R * HD; i += DT) {
    const int r = i / HD;
    sm.q[r][i % HD] = r < w.n_rows ? load_elem(p.q, w.seq * p.q_stride + (int64_t)(w.head0 + r) * HD + i % HD, p.io) : 0.f;
  }
  __syncthreads();
  float m[R], l[R], o[R][E];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[r][e] = 0.f;
  }
  bool expired = false;
  for (int k = 0; k < mine; ++k) {
    const int j0 = w.sp.page(w.i0 + warp + DW * k) * PG;
    const bool gone = bad >> (k % 8) & 1;
    bool ok = wait_slot(&sm.full[warp][2 * k % S], (uint32_t)(2 * k / S) & 1, p.status);
    const KV* kp = reinterpret_cast<const KV*>(sm.ring[warp][2 * k % S]) + g * HD + t * 4;
    float s[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = 0.f;
#pragma unroll 2
    for (int c = 0; c < HD / 16; ++c) {
      const int d = (c ^ (g & 1)) * 16;
      const float4 a = lds4<KV>(kp + d), b = lds4<KV>(kp + 8 * HD + d);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 q = *reinterpret_cast<const float4*>(&sm.q[r][d + t * 4]);
        s[r][0] = fmaf(q.x, a.x, fmaf(q.y, a.y, fmaf(q.z, a.z, fmaf(q.w, a.w, s[r][0]))));
        s[r][1] = fmaf(q.x, b.x, fmaf(q.y, b.y, fmaf(q.z, b.z, fmaf(q.w, b.w, s[r][1]))));
      }
    }
    __syncwarp();
    issue(2 * k + S);
    const bool see0 = !gone && key_seen(j0 + g, w.pos, p.window, p.n_sink);
    const bool see1 = !gone && key_seen(j0 + g + 8, w.pos, p.window, p.n_sink);
    float f[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[r][h] += __shfl_xor_sync(0xffffffffu, s[r][h], 1);
        s[r][h] += __shfl_xor_sync(0xffffffffu, s[r][h], 2);
      }
      s[r][0] = see0 ? s[r][0] * p.scale_log2 : -INFINITY;
      s[r][1] = see1 ? s[r][1] * p.scale_log2 : -INFINITY;
      float mx = fmaxf(s[r][0], s[r][1]);
#pragma unroll
      for (int d = 4; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      mx = fmaxf(mx, m[r]);
      const float ms = mx == -INFINITY ? 0.f : mx;
      f[r] = exp2_approx(m[r] - ms);
      m[r] = mx;
      const float p0 = exp2_approx(s[r][0] - ms), p1 = exp2_approx(s[r][1] - ms);
      l[r] = l[r] * f[r] + (p0 + p1);  // of this lane's two keys
      if (t == 0) {
        sm.p[warp][r][g] = p0;
        sm.p[warp][r][g + 8] = p1;
      }
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) o[r][e] *= f[r];
    ok = ok && wait_slot(&sm.full[warp][(2 * k + 1) % S], (uint32_t)((2 * k + 1) / S) & 1, p.status);
    if (!ok) {
      const long long t0 = clock64();  // the copies still under way end before their memory is used again
      while (clock64() - t0 < 1 << 20) {
      }
      expired = true;
      break;
    }
    const KV* vp = reinterpret_cast<const KV*>(sm.ring[warp][(2 * k + 1) % S]) + lane * E;
    const bool edge = gone || j0 + PG - 1 > w.pos || (p.window > 0 && j0 <= w.pos - p.window);
#pragma unroll
    for (int j = 0; j < PG; j += 4) {
      float v[4][E];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // what a masked place holds is never used
        const bool see = !edge || (!gone && key_seen(j0 + j + i, w.pos, p.window, p.n_sink));
        if constexpr (E % 4 == 0) {
#pragma unroll
          for (int e = 0; e < E; e += 4) {
            const float4 x = lds4<KV>(vp + (j + i) * HD + e);
            v[i][e] = see ? x.x : 0.f;
            v[i][e + 1] = see ? x.y : 0.f;
            v[i][e + 2] = see ? x.z : 0.f;
            v[i][e + 3] = see ? x.w : 0.f;
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) v[i][e] = see ? to_f32<KV>(vp[(j + i) * HD + e]) : 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 x = *reinterpret_cast<const float4*>(&sm.p[warp][r][j]);
#pragma unroll
        for (int e = 0; e < E; ++e)
          o[r][e] = fmaf(x.w, v[3][e], fmaf(x.z, v[2][e], fmaf(x.y, v[1][e], fmaf(x.x, v[0][e], o[r][e]))));
      }
    }
    __syncwarp();
    issue(2 * k + 1 + S);
  }
  __syncthreads();  // the ring becomes the join's memory
#pragma unroll
  for (int r = 0; r < R; ++r) {
    for (int d = 4; d < 32; d *= 2) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
    if (lane == 0) {
      sm.join.m[warp][r] = m[r];
      sm.join.l[warp][r] = expired ? NAN : l[r];  // NaN: so is every output that this is a part of
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm.join.o[warp][r][lane * E + e] = o[r][e];
  }
  join_and_store(sm.join, p, w.seq, w.head0, w.n_rows, w.pos >= 0);
}

// ---- tensor cores (mma.sync): 16-bit caches ------------------------------------------
// A warp takes a page (16 keys) at a time.  Each warp has a ring of its own of
// page slots in shared memory, filled by one tensor-map copy for K and one for V
// (4 KB each at hd 128, 128-byte swizzle): only lanes of one warp wait for one
// another, and the bytes under way do not depend on registers.  The operands of
// the m16n8k16 products come from the slots with 16-byte loads free of bank
// conflicts, without ldmatrix, because the inner index may be permuted:
//   S (8 heads x 16 keys): lane (g, t) loads 16-byte chunk 2t + h of each 128
//   bytes of keys g and g + 8; q follows the same permutation of head dims.
//   O (8 heads x hd): lane (g, t) loads chunk g of keys 2t, 2t+1, 2t+8, 2t+9; a
//   byte permute of two keys' words gives the operand, column g of product e
//   being dim 8 g + e.
// The product has 16 rows and a CTA takes 8 heads: the other 8 rows carry what f32
// has below 16 bits.  Rows 0-7 hold the first term of q (32-bit rows: q scaled by a
// power of two per head, as two f16 terms) and of P, rows 8-15 the second; the two
// halves of S and of O are added.  The running maximum moves when a row outgrows it
// by 2^RAISE; P is 2^BIAS at it.  Over f16 that is 2^11, 2^15 at most, so that P's
// second term keeps clear of f16's smallest step; values reach 2^16 there and sums
// stay far inside f32.  bf16 has the range of f32, values too: P is at most 1, so that
// a finite value stays finite under it, as under the softmax's own weights.
// The product's f32 sum drops what falls below its last bits, each time, towards 0: of
// values of one sign 2.1e-4 was gone after the 2048 pages that a warp of a full batch takes
// at 131072 keys.  So a warp of many pages (RUNS) sums O in runs, which it adds to a kept O by
// f32 additions that round to nearest: runs of 8 pages for 32-bit rows (4e-7 of the result, as
// prompts have it), of 512 for f16 rows (5e-5, a tenth of f16's half step).  A warp of at
// most 12 pages of 32-bit rows (8e-7), or of 512, does without: one sequence of 32768, 32-bit
// rows: 30.0 us, 31.3 with runs.  bf16 rows do without up to 2048 pages: those 2.1e-4 are a
// twentieth of their half step, and runs took 673 us where one sum takes 667 (eight long
// sequences).
// Eight sequences of 131072 keys, 64 heads of 128 over 8, bf16: 645 us, 6.66 TB/s, what a
// copy reaches (operands straight from global memory: 1190 us).  One sequence of
// 32768, f32 rows over f16: 30.0 us, of which 20.5 are the bytes and the rest the chain
// before the first page and behind the last one.  Three CTAs of two slots a warp,
// not two of three: 38 and 49 us for 48 ragged windows of 1024, 645 and 647 for the
// eight long ones.
constexpr int MMA_R = 8;

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (x, y) rounded to 16 bits in one word, and what the rounding left, in another
template <bool BF16>
__device__ __forceinline__ void two_terms(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  }
}

// The sum of the two terms' products.  An infinite key or value times the second term is infinite of either sign, or
// NaN: the first term's product alone is what the formula gives.
__device__ __forceinline__ float add_terms(float first, float second) {
  return fabsf(first) < INFINITY ? first + second : first;
}

// One query head's part of one warp again, in f32, key by key: o to `out`, (m, l) returned, weights `one` at m.  For a
// part that came out as NaN over an f16 cache: a weight (or a number of q) whose first term rounds to 0 makes NaN of an
// infinite value (or key), where the formula has an infinite output (or a weight of 0).
template <class KV, int HD, int DW>
__device__ __noinline__ float2 recompute_part(const WindowAttnParams& p, const Work w, int row, float one, float* out) {
  constexpr int E = HD / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, key = lane % PG, half = lane / PG * (HD / 2);
  const int64_t q0 = w.seq * p.q_stride + (int64_t)(w.head0 + row) * HD + half;
  float m = -INFINITY, l = 0.f, o[E] = {};
  for (int i = w.i0 + warp; i < w.i1; i += DW) {
    const int id = page_id(p, w, i);
    if (id < 0) continue;  // the same for all lanes
    const int64_t page = ((int64_t)id * p.n_head_kv + w.hk) * PG * HD;
    const KV* k = static_cast<const KV*>(p.k_pages) + page + key * HD + half;
    const KV* v = static_cast<const KV*>(p.v_pages) + page + lane * E;
    float s = 0.f;
#pragma unroll 8
    for (int d = 0; d < HD / 2; ++d) s = fmaf(load_elem(p.q, q0 + d, p.io), to_f32<KV>(k[d]), s);
    s += __shfl_xor_sync(0xffffffffu, s, PG);
    const bool see = key_seen(w.sp.page(i) * PG + key, w.pos, p.window, p.n_sink);
    s = see ? s * p.scale_log2 : -INFINITY;
    float mx = s;
#pragma unroll
    for (int d = 1; d < PG; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    mx = fmaxf(mx, m);
    const float ms = mx == -INFINITY ? 0.f : mx;
    const float f = exp2_approx(m - ms), x = exp2_approx(s - ms);
    m = mx;
    l = l * f + x;  // of this lane's key
    const unsigned seen = __ballot_sync(0xffffffffu, see);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= f;
    for (int j = 0; j < PG; ++j) {
      const float xj = __shfl_sync(0xffffffffu, x, j);
      if (!(seen >> j & 1)) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(xj, to_f32<KV>(v[j * HD + e]), o[e]);
    }
  }
#pragma unroll
  for (int d = 1; d < PG; d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane * E + e] = o[e] * one;
  return make_float2(m, l * one);
}

template <int HD, int DW>
struct MmaCfg {
  static constexpr int HDP = HD < 64 ? 64 : HD;    // head width in a slot (the copy fills with zeros)
  static constexpr int PAGE = PG * HDP * 2;        // bytes of a page's K or V
  static constexpr int STAGES = HDP == 64 ? 4 : 2;  // slots per warp: 16 KB (32 KB at hd 256)
  static constexpr int RING = DW * STAGES * 2 * PAGE;
};
template <int HD, int DW>
struct MmaSmem {
  using C = MmaCfg<HD, DW>;
  union {
    uint8_t ring[C::RING];  // [warp][stage][K | V][64-dim block][16 keys][128 B]
    JoinSmem<MMA_R, HD, DW> join;
  };
  uint4 q[C::HDP / 16][32];  // A operands of q, by lane
  float up[MMA_R];           // scale of each head's scores
  uint64_t full[DW][C::STAGES];
};

// Pages of a run, and the most that a warp may take without runs.
template <bool SPLIT>
constexpr int RUN = SPLIT ? 8 : 512;
template <bool SPLIT, bool BF16>
constexpr int MAX_RUN = SPLIT ? 12 : BF16 ? 2048 : 512;

template <class KV, int HD, bool SPLIT, int DW, bool RUNS>
__global__ void __launch_bounds__(DW * 32, HD <= 128 ? 3 : 1)
    decode_mma_kernel(const __grid_constant__ WindowAttnParams p, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap) {
  constexpr bool BF16 = std::is_same<KV, __nv_bfloat16>::value;
  using C = MmaCfg<HD, DW>;
  using Smem = MmaSmem<HD, DW>;
  constexpr int DT = DW * 32, NB = C::HDP / 64, S = C::STAGES;
  constexpr float RAISE = 4.f, BIAS = BF16 ? -RAISE : 11.f;
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  static_assert(DT == MMA_R * 16, "16 threads to a query head");
  if (p.partial) pdl_launch_dependents();
  if (tid == 0) {
    prefetch_map(&kmap);
    prefetch_map(&vmap);
  }
  // q is on its way while the position and the page ids are looked up
  constexpr int QC = (C::HDP / 8 + 15) / 16;
  const int qr = tid / 16, qi = tid % 16;
  float qx[QC][8] = {};
  {
    const int group = p.n_head / p.n_head_kv, tiles = (group + MMA_R - 1) / MMA_R, pair = blockIdx.x / p.parts;
    const int r = pair % tiles * MMA_R + qr;
    if (r < group) {
      const int64_t at = blockIdx.y * p.q_stride + (int64_t)(pair / tiles * group + r) * HD;
#pragma unroll
      for (int c = 0; c < QC; ++c)
        if ((qi + 16 * c) * 8 < HD) {
          using Row = typename std::conditional<SPLIT, float, KV>::type;
          Raw8<Row> raw;
          load8(raw, static_cast<const Row*>(p.q) + at + (qi + 16 * c) * 8, p.q_vec);
          unpack8(raw, qx[c]);
        }
    }
  }
  const Work w = find_work<MMA_R>(p);
  const int mine = (w.i1 - w.i0 - warp + DW - 1) / DW;  // pages of this warp (<= 0: none)

  // ids of this warp's entries i0 + warp + DW k, k = ids_at .. ids_at + 31; -1: outside the pool
  int ids = -1, ids_at = 0;
  auto fetch_ids = [&](int k0) {
    const int i = w.i0 + warp + DW * (k0 + lane);
    ids = i < w.i1 ? page_id(p, w, i) : -1;
    ids_at = k0;
  };
  uint8_t* slots = sm.ring + warp * S * 2 * C::PAGE;
  // A page outside the pool comes as zeros (a row past the map's end); its keys count as masked.
  auto issue = [&](int k) {
    if (k - ids_at == 32) fetch_ids(k);
    const int id = __shfl_sync(0xffffffffu, ids, k - ids_at);
    if (lane == 0) {
      const int y = id < 0 ? p.n_pages * p.n_head_kv * PG : (id * p.n_head_kv + w.hk) * PG;
      uint64_t* bar = &sm.full[warp][k % S];
      uint8_t* dst = slots + k % S * 2 * C::PAGE;
      mbar_arrive_expect_tx(bar, 2 * C::PAGE);
      tma_page(smem_u32(dst), &kmap, y, bar);
      tma_page(smem_u32(dst + C::PAGE), &vmap, y, bar);
    }
    return id;
  };
  unsigned bad = 0;  // bit k % S: the page in that slot is outside the pool
  auto issue_noting = [&](int k) {
    const unsigned bit = 1u << (k % S);
    bad = issue(k) < 0 ? bad | bit : bad & ~bit;
  };
  if (lane == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  if (mine > 0) fetch_ids(0);
  for (int k = 0; k < min(mine, S); ++k) issue_noting(k);

  // q as A operands: step 4 b + 2 h + u, lane (g, t): dims 64 b + 8 (2 t + h) + 4 u + 0..3 of head g
  float mx = 0.f;
#pragma unroll
  for (int c = 0; c < QC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(qx[c][e]));
  float up = 1.f;  // the head's largest |q| to [1, 2): a power of two, exact
  if (SPLIT) {
#pragma unroll
    for (int d = 1; d < 16; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const int e = (int)(__float_as_uint(mx) >> 23) - 127;
    if (mx > 0.f && e < 128) up = __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
    if (qi == 0) sm.up[qr] = up;
  }
  const float down = 1.f / up;
#pragma unroll
  for (int c = 0; c < QC; ++c) {
    const int ch = qi + 16 * c;  // 8 dims
    if (ch < C::HDP / 8) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint4 a;
        two_terms<BF16>(qx[c][4 * u] * down, qx[c][4 * u + 1] * down, a.x, a.y);  // 16-bit rows: the second term is 0
        two_terms<BF16>(qx[c][4 * u + 2] * down, qx[c][4 * u + 3] * down, a.z, a.w);
        sm.q[ch / 8 * 4 + ch % 2 * 2 + u][qr * 4 + ch % 8 / 2] = a;
      }
    }
  }
  __syncthreads();
  const float scale = p.scale_log2 * (SPLIT ? sm.up[g] : 1.f);

  float o[NB * 8][4];
#pragma unroll
  for (int i = 0; i < NB * 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m = -INFINITY, l = 0.f;  // of head g; l of this lane's keys
  bool expired = false;
  // The first terms' sums of whole runs, in units of 2^kept_m: in registers, or, where the runs are long,
  // in local memory (asm: so that they take no registers from the loop) from the first whole run on.
  float kept_here[NB * 8 * 2], kept_m = -INFINITY;
  float* kept = kept_here;
  if constexpr (RUNS && SPLIT) {
#pragma unroll
    for (int i = 0; i < NB * 8 * 2; ++i) kept[i] = 0.f;
  } else if constexpr (RUNS) {
    asm volatile("" : "+l"(kept)::"memory");
  }
  auto fold = [&](bool any) {  // any: there are kept sums
    const float f = kept_m == -INFINITY ? 0.f : exp2_approx(kept_m - m);
    kept_m = m;
#pragma unroll
    for (int i = 0; i < NB * 8; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        kept[2 * i + h] = SPLIT || any ? fmaf(kept[2 * i + h], f, o[i][h]) : o[i][h];
        o[i][h] = 0.f;
      }
  };
  for (int k = 0; k < mine; ++k) {
    const int j0 = w.sp.page(w.i0 + warp + DW * k) * PG;
    if (!wait_slot(&sm.full[warp][k % S], (uint32_t)(k / S) & 1, p.status)) {
      const long long t0 = clock64();  // the copies still under way end before their memory is used again
      while (clock64() - t0 < 1 << 20) {
      }
      expired = true;
      break;
    }
    const uint8_t* ks = slots + k % S * 2 * C::PAGE;
    const uint8_t* vs = ks + C::PAGE;
    float s0[4] = {}, s1[4] = {};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* at = ks + b * (PG * 128) + g * 128 + (((2 * t + h) ^ g) * 16);
        const uint4 k0 = lds128(at), k1 = lds128(at + 8 * 128);
        const uint4 qa = sm.q[4 * b + 2 * h][lane], qb = sm.q[4 * b + 2 * h + 1][lane];
        const uint32_t a0[4] = {qa.x, qa.y, qa.z, qa.w}, a1[4] = {qb.x, qb.y, qb.z, qb.w};
        mma16816<BF16>(s0, a0, k0.x, k0.y);
        mma16816<BF16>(s1, a0, k1.x, k1.y);
        mma16816<BF16>(s0, a1, k0.z, k0.w);
        mma16816<BF16>(s1, a1, k1.z, k1.w);
      }
    // keys 2t, 2t+1, 2t+8, 2t+9 of head g
    float x[4] = {add_terms(s0[0], s0[2]), add_terms(s0[1], s0[3]), add_terms(s1[0], s1[2]), add_terms(s1[1], s1[3])};
    const bool gone = bad >> (k % S) & 1;
    const bool edge = gone || j0 + PG - 1 > w.pos || (p.window > 0 && j0 <= w.pos - p.window);
    bool see[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      see[j] = !edge || (!gone && key_seen(j0 + 2 * t + (j & 1) + (j & 2) * 4, w.pos, p.window, p.n_sink));
      if (!see[j]) x[j] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * scale;
    if (__any_sync(0xffffffffu, mx > m + RAISE || m == -INFINITY)) {
      const float mn = fmaxf(mx, m);
      const float f = m == -INFINITY ? 0.f : exp2_approx(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < NB * 8; ++i) {
        o[i][0] *= f;
        o[i][1] *= f;
        o[i][2] *= f;
        o[i][3] *= f;
      }
    }
    const float neg = BIAS - (m == -INFINITY ? 0.f : m);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = exp2_approx(fmaf(x[j], scale, neg));
    l += (x[0] + x[1]) + (x[2] + x[3]);
    uint32_t a[4];
    two_terms<BF16>(x[0], x[1], a[0], a[1]);
    two_terms<BF16>(x[2], x[3], a[2], a[3]);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t v[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = 2 * t + (j & 1) + (j & 2) * 4;
        const uint4 r = lds128(vs + b * (PG * 128) + key * 128 + ((g ^ (key & 7)) * 16));
        // whatever a masked place holds is not used
        v[j][0] = see[j] ? r.x : 0;
        v[j][1] = see[j] ? r.y : 0;
        v[j][2] = see[j] ? r.z : 0;
        v[j][3] = see[j] ? r.w : 0;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = e & 1 ? 0x7632 : 0x5410;
        mma16816<BF16>(o[b * 8 + e], a, __byte_perm(v[0][e / 2], v[1][e / 2], sel),
                       __byte_perm(v[2][e / 2], v[3][e / 2], sel));
      }
    }
    __syncwarp();  // every lane is done with the slot
    if (k + S < mine) issue_noting(k + S);
    if (RUNS && k % RUN<SPLIT> == RUN<SPLIT> - 1) fold(k >= RUN<SPLIT>);
  }
  if (RUNS && (SPLIT || mine >= RUN<SPLIT>)) {
    const float f = kept_m == -INFINITY ? 0.f : exp2_approx(kept_m - m);
#pragma unroll
    for (int i = 0; i < NB * 8; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) o[i][h] = fmaf(kept[2 * i + h], f, o[i][h]);
  }
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncthreads();  // the ring becomes the join's memory
  if (t == 0) {
    sm.join.m[warp][g] = m;
    sm.join.l[warp][g] = expired ? NAN : l;  // NaN: so is every output that this is a part of
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = b * 64 + 16 * t + e;  // and d + 8
      if (d < HD) sm.join.o[warp][g][d] = add_terms(o[b * 8 + e][0], o[b * 8 + e][2]);
      if (d + 8 < HD) sm.join.o[warp][g][d + 8] = add_terms(o[b * 8 + e][1], o[b * 8 + e][3]);
    }
  if constexpr (!BF16) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < NB * 8; ++i) nan = nan || o[i][0] != o[i][0] || o[i][1] != o[i][1];
    // rows of one term of q: a sum of weights that is not finite is the formula's
    unsigned again = __ballot_sync(0xffffffffu, nan && !expired && g < w.n_rows && (SPLIT || l < INFINITY));
    while (again) {
      const int r = (__ffs(again) - 1) / 4;
      again &= ~(0xfu << (4 * r));
      __syncwarp();
      const float2 ml = recompute_part<KV, HD, DW>(p, w, r, 1 << (int)BIAS, sm.join.o[warp][r]);
      if (lane == 0) {
        sm.join.m[warp][r] = ml.x;
        sm.join.l[warp][r] = ml.y;
      }
    }
  }
  join_and_store(sm.join, p, w.seq, w.head0, w.n_rows, w.pos >= 0);
}

template <auto Kernel, class... Maps>
cudaError_t launch_parts(const WindowAttnParams& p, int tiles, int threads, size_t smem, cudaStream_t st,
                         const Maps&... maps) {
  cudaError_t e = allow_smem<Kernel>(smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.n_head_kv * tiles * p.parts), (unsigned)p.n_seq);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)(p.partial ? 1 : p.parts);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, Kernel, p, maps...);
}

template <int HD>
cudaError_t launch_join(const WindowAttnParams& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.n_seq * p.n_head));
  cfg.blockDim = dim3(JW * 32);
  cfg.dynamicSmemBytes = sizeof(float) * p.parts;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<HD>, p);
}

// pages that the longest possible context of this call sees
int64_t max_seen_pages(const WindowAttnParams& p) {
  if (p.window <= 0) return p.max_pages;
  const int64_t n = (p.window + (int64_t)PG - 1) / PG + 1 + ((int64_t)p.n_sink + PG - 1) / PG;
  return n < p.max_pages ? n : p.max_pages;
}

constexpr int DEC_R = 8, DEC_W = 4;  // query heads and warps of a CTA
int row_tiles(const WindowAttnParams& p) { return (p.n_head / p.n_head_kv + DEC_R - 1) / DEC_R; }

// How many CTAs share a (sequence, kv head, row tile), and where they join.
// Short contexts: a cluster of up to 8, doubled until the GPU has two CTAs for
// every SM, as long as each warp keeps a page or more.  Where a warp would still
// walk more than LONG pages that way, the pages are split into one wave of `occ`
// CTAs per SM, joined through the workspace (one sequence, 8 kv heads: 12.4 us in clusters and
// 8.8 split at 4096 keys; 6.3 and 7.5 at 1024).
constexpr int LONG = 2;
struct Parts {
  int cluster;    // CTAs per cluster without a workspace
  int64_t split;  // CTAs with one, 0: not worth it
  size_t bytes;   // the workspace
};
Parts count_parts(const WindowAttnParams& p, int occ, int hd, int sm_count) {
  const int64_t pages = max_seen_pages(p), pairs = (int64_t)p.n_seq * p.n_head_kv * row_tiles(p);
  Parts r{1, 0, 0};
  while (r.cluster < 8 && pairs * r.cluster < 2 * sm_count && pages > (int64_t)r.cluster * DEC_W) r.cluster *= 2;
  int64_t n = occ * sm_count / pairs;
  n = n < pages / (2 * DEC_W) ? n : pages / (2 * DEC_W);
  if (n > 1 && pages > (int64_t)r.cluster * DEC_W * LONG) {
    r.split = n;
    r.bytes = (size_t)(n * p.n_seq * p.n_head * (hd + 2)) * sizeof(float);
  }
  return r;
}
void pick_parts(WindowAttnParams& p, int occ, int hd, int sm_count) {
  const Parts r = count_parts(p, occ, hd, sm_count);
  const bool split = r.split && p.partial && p.ws_bytes >= r.bytes;
  p.parts = split ? (int)r.split : r.cluster;
  if (!split) p.partial = nullptr;
}

template <class KV, int HD>
cudaError_t launch_cc(WindowAttnParams& p, int sm_count, cudaStream_t st) {
  using Smem = CcSmem<KV, HD>;
  using C = CcCfg<KV, HD>;
  static_assert(C::R == DEC_R && C::DW == DEC_W, "pick_parts counts these");
  pick_parts(p, sizeof(Smem) > 113 * 1024 ? 1 : 2, HD, sm_count);
  return launch_parts<decode_cc_kernel<KV, HD>>(p, row_tiles(p), DEC_W * 32, sizeof(Smem), st);
}

template <class KV, int HD, bool SPLIT>
cudaError_t launch_mma(WindowAttnParams& p, int kv, int sm_count, cudaStream_t st) {
  using Smem = MmaSmem<HD, DEC_W>;
  CUtensorMap km, vm;
  const int64_t rows = (int64_t)p.n_pages * p.n_head_kv * PG;
  cudaError_t e = pool_map(&km, p.k_pages, kv, HD, rows, (HD + 63) / 64);
  if (e == cudaSuccess) e = pool_map(&vm, p.v_pages, kv, HD, rows, (HD + 63) / 64);
  if (e != cudaSuccess) return e;
  pick_parts(p, HD <= 128 ? 3 : 1, HD, sm_count);
  const auto launch = [&](auto runs) {
    return launch_parts<decode_mma_kernel<KV, HD, SPLIT, DEC_W, decltype(runs)::value>>(p, row_tiles(p), DEC_W * 32,
                                                                                       sizeof(Smem) + 1024, st, km, vm);
  };
  constexpr int most = MAX_RUN<SPLIT, std::is_same<KV, __nv_bfloat16>::value>;
  return max_seen_pages(p) > (int64_t)p.parts * DEC_W * most ? launch(std::true_type()) : launch(std::false_type());
}
template <class KV, int HD>
cudaError_t launch_16(WindowAttnParams& p, int kv, int sm_count, cudaStream_t st) {
  if ((int64_t)p.n_pages * p.n_head_kv * PG >= 0x7fffffff) return launch_cc<KV, HD>(p, sm_count, st);  // beyond a map's rows
  if constexpr (std::is_same<KV, __half>::value)
    if (p.io == EL_F32) return launch_mma<KV, HD, true>(p, kv, sm_count, st);
  return launch_mma<KV, HD, false>(p, kv, sm_count, st);
}

template <int HD>
cudaError_t launch_hd(WindowAttnParams& p, int kv, int sm_count, cudaStream_t st) {
  cudaError_t e;
  if (kv == EL_F32) e = launch_cc<float, HD>(p, sm_count, st);
  else if (kv == EL_F16) e = launch_16<__half, HD>(p, kv, sm_count, st);
  // 32-bit rows over a bf16 cache: two bf16 terms hold 16 bits only, so these stay on the CUDA cores
  else if (p.io == EL_F32) e = launch_cc<__nv_bfloat16, HD>(p, sm_count, st);
  else e = launch_16<__nv_bfloat16, HD>(p, kv, sm_count, st);
  return e == cudaSuccess && p.partial ? launch_join<HD>(p, st) : e;
}

}  // namespace

size_t window_decode_workspace(const WindowAttnParams& p, int hd, int sm_count) {
  // of the kernel with the most CTAs per SM, and so the most parts
  return count_parts(p, 3, hd, sm_count).bytes;
}

cudaError_t launch_window_decode(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st) {
  switch (hd) {
    case 32: return launch_hd<32>(p, kv, sm_count, st);
    case 64: return launch_hd<64>(p, kv, sm_count, st);
    case 128: return launch_hd<128>(p, kv, sm_count, st);
    case 256: return launch_hd<256>(p, kv, sm_count, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace sfk
