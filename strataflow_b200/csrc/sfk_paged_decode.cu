// sfk_paged_decode.cu -- attention of one new token of each sequence over the
// keys it sees in the paged cache (window and sinks), split over the keys and
// joined inside a thread-block cluster.
//
//   s_j = scale q . k_j  for the seen keys j;  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
//
// Bound by memory: each seen key and value is read once for all query heads
// of its kv head.  A cluster takes one (sequence, kv head); each CTA takes a
// run of its seen pages, each warp every W-th page of the run with a running
// maximum, sum and output of its own (f32).  The partials of the warps meet in
// shared memory, those of the CTAs in distributed shared memory: no scratch
// in global memory, no second launch, and calls on several streams or in
// several graphs have nothing in common.
#include <cooperative_groups.h>

#include "sfk_paged.cuh"

namespace sfk {
namespace {

namespace cg = cooperative_groups;

constexpr int DW = 4;         // warps per CTA
constexpr int DT = DW * 32;

// ---- join -----------------------------------------------------------------------
// Every warp's partial (m, l, o) of R rows to the output.  m is in units of
// log2; a partial without keys has m = -inf, l = 0, o = 0.
template <int R, int HD>
struct JoinSmem {
  float o[DW][R][HD];
  float m[DW][R], l[DW][R];
  float co[R][HD];  // the CTA's partial
  float cm[R], cl[R];
};

template <int R, int HD>
__device__ void join_and_store(JoinSmem<R, HD>& sm, const WindowAttnParams& p, int seq, int head0, int n_rows, bool any) {
  cg::cluster_group cl = cg::this_cluster();
  const int C = p.cluster, rank = C > 1 ? (int)cl.block_rank() : 0;
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
    sm.co[r][d] = o;
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
  const int rank = blockIdx.x % p.cluster;
  const int pair = blockIdx.x / p.cluster;
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
  const int per = (w.sp.n + p.cluster - 1) / p.cluster;
  w.i0 = min(w.sp.n, rank * per);
  w.i1 = min(w.sp.n, w.i0 + per);
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
// A warp takes a page at a time.  Scores: lane (g, t) = (lane / 4, lane % 4)
// multiplies dims 8 t .. 8 t + 7 of each 32 of keys g and g + 8 by the query
// rows in shared memory.  Values: the lane owns HD / 32 output dims.
template <class KV, int HD>
struct CcSmem {
  static constexpr int R = 8;
  float q[R][HD];
  float p[DW][R][PG];
  JoinSmem<R, HD> join;
};

template <class KV, int HD>
__global__ void __launch_bounds__(DT) decode_cc_kernel(const __grid_constant__ WindowAttnParams p) {
  using Smem = CcSmem<KV, HD>;
  constexpr int R = Smem::R, E = HD / 32;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const Work w = find_work<R>(p);
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
  for (int i = w.i0 + warp; i < w.i1; i += DW) {
    const int id = page_id(p, w, i);
    if (id < 0) continue;
    const int64_t off = ((int64_t)id * p.n_head_kv + w.hk) * PG * HD;
    const KV* kp = static_cast<const KV*>(p.k_pages) + off;
    const KV* vp = static_cast<const KV*>(p.v_pages) + off;
    const int j0 = w.sp.page(i) * PG;
    float s[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = 0.f;
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) {
      Raw8<KV> ra, rb;
      load8(ra, kp + g * HD + c * 32 + t * 8, true);
      load8(rb, kp + (g + 8) * HD + c * 32 + t * 8, true);
      float a[8], b[8];
      unpack8(ra, a);
      unpack8(rb, b);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float q[8];
        *reinterpret_cast<float4*>(q) = *reinterpret_cast<const float4*>(&sm.q[r][c * 32 + t * 8]);
        *reinterpret_cast<float4*>(q + 4) = *reinterpret_cast<const float4*>(&sm.q[r][c * 32 + t * 8 + 4]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[r][0] = fmaf(q[e], a[e], s[r][0]);
          s[r][1] = fmaf(q[e], b[e], s[r][1]);
        }
      }
    }
    const bool see0 = key_seen(j0 + g, w.pos, p.window, p.n_sink), see1 = key_seen(j0 + g + 8, w.pos, p.window, p.n_sink);
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
#pragma unroll 4
    for (int j = 0; j < PG; ++j) {
      if (!key_seen(j0 + j, w.pos, p.window, p.n_sink)) continue;  // what a masked place holds is never used
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = to_f32<KV>(vp[j * HD + lane * E + e]);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] = fmaf(sm.p[warp][r][j], v[e], o[r][e]);
    }
    __syncwarp();
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    for (int d = 4; d < 32; d *= 2) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
    if (lane == 0) {
      sm.join.m[warp][r] = m[r];
      sm.join.l[warp][r] = l[r];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm.join.o[warp][r][lane * E + e] = o[r][e];
  }
  join_and_store(sm.join, p, w.seq, w.head0, w.n_rows, w.pos >= 0);
}

template <class K>
cudaError_t launch_clusters(K kernel, const WindowAttnParams& p, int tiles, size_t smem, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  if (p.cluster > 8) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.n_head_kv * tiles * p.cluster), (unsigned)p.n_seq);
  cfg.blockDim = dim3(DT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)p.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// CTAs per (sequence, kv head, row tile): enough for two on every SM, as long
// as each of a CTA's warps has a page or more.
int pick_cluster(const WindowAttnParams& p, int tiles, int sm_count) {
  int64_t pages = p.max_pages;
  if (p.window > 0)
    pages = pages < (p.window + PG - 1) / PG + 1 + ((int64_t)p.n_sink + PG - 1) / PG
                ? pages
                : (p.window + PG - 1) / PG + 1 + ((int64_t)p.n_sink + PG - 1) / PG;
  const int64_t pairs = (int64_t)p.n_seq * p.n_head_kv * tiles;
  int c = 1;
  while (c < 16 && pairs * c < 2 * sm_count && pages > (int64_t)c * DW) c *= 2;
  return c;
}

template <class KV, int HD>
cudaError_t launch_cc(WindowAttnParams& p, int sm_count, cudaStream_t st) {
  using Smem = CcSmem<KV, HD>;
  const int tiles = (p.n_head / p.n_head_kv + Smem::R - 1) / Smem::R;
  p.cluster = pick_cluster(p, tiles, sm_count);
  return launch_clusters(decode_cc_kernel<KV, HD>, p, tiles, sizeof(Smem), st);
}

template <class KV>
cudaError_t launch_kv(WindowAttnParams& p, int hd, int sm_count, cudaStream_t st) {
  switch (hd) {
    case 32: return launch_cc<KV, 32>(p, sm_count, st);
    case 64: return launch_cc<KV, 64>(p, sm_count, st);
    case 128: return launch_cc<KV, 128>(p, sm_count, st);
    case 256: return launch_cc<KV, 256>(p, sm_count, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_window_decode(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st) {
  if (kv == EL_F32) return launch_kv<float>(p, hd, sm_count, st);
  if (kv == EL_F16) return launch_kv<__half>(p, hd, sm_count, st);
  return launch_kv<__nv_bfloat16>(p, hd, sm_count, st);
}

}  // namespace sfk
