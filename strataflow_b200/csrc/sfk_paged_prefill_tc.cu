// sfk_paged_prefill_tc.cu -- attention of a ragged batch of prompts over the
// paged cache on the tensor cores (tcgen05), for 16-bit caches.
//
//   S = Q K^T;  P = 2^(scale S - m);  O = sum over key tiles of P V;  out = O / sum P
//
// A CTA takes two tiles of 128 rows (rows: tokens x the query heads of one kv
// head) and walks the pages its rows see in tiles of 128 keys:
//   warps 0-3, 4-7  softmax of row tile 0 and 1: thread = TMEM lane = row.
//                   Reads its S row, updates the running maximum, writes P over
//                   S in TMEM as 16-bit A operands.
//   warp 8          brings K and V tiles in, eight pages each, by tensor-map
//                   copies (128-byte swizzle) into a ring of tile slots.
//   warp 9          one thread issues the products: P V of one row tile and the
//                   next Q K^T of the same tile, then the other tile's, so the
//                   tensor core works on one tile while the other is in softmax.
//   warps 10, 11    fill the third warpgroup, which hands registers to the softmax.
// S and O live in TMEM (2 x 128 and 2 x head_dim columns).  The products of one
// thread run in order, so S(n + 1) of a row tile is complete only after its
// P V(n): the softmax threads may touch O as soon as S(n + 1) has arrived.
//
// The running maximum m is only raised when a row outgrows it by 2^8: O is
// rescaled then, by the row's own thread.  P then reaches 2^8, far inside both
// 16-bit types, and the sum stays in 32 bits.
//
// 32-bit rows over an f16 cache (SPLIT): q, scaled by a power of two per row,
// is the sum of two f16 numbers and so is each P (22 bits), and each product
// is two.  P is held up to 2^15 so that its second part stays above f16's
// smallest step.  A bf16 pair holds 16 bits only: that cache takes the
// CUDA-core kernel.
//
// What a masked place holds does not matter: K only reaches its own column of
// S, which is replaced; V rows past the sequence's length are zeroed in shared
// memory; a V row that some rows of a tile see and others do not reaches the
// others as 0 * v, which is NaN for an infinite v: rows whose output is not
// finite are computed again key by key (recompute_row).
#include <type_traits>

#include "sfk_paged.cuh"
#include "sfk_paged_map.cuh"

namespace sfk {
namespace {

constexpr int TM = 128;       // rows per tile
constexpr int TK = 128;       // keys per tile
constexpr int TC_ROWS = 256;  // rows per CTA
constexpr int TT = 384;       // threads: three warpgroups, 168 registers each at launch
// Registers after the split: 2 x 128 x 200 + 128 x 104 = 384 x 168, what the launch holds
constexpr int REG_SOFTMAX = 200, REG_OTHER = 104;
static_assert(2 * 128 * REG_SOFTMAX + 128 * REG_OTHER <= TT * 168, "register split above the launch's");
constexpr int PPT = TK / PG;  // pages per key tile

template <int HD, bool SPLIT>
struct Cfg {
  static constexpr int HDP = HD < 64 ? 64 : HD;  // head width in shared memory (the copy fills with zeros)
  static constexpr int HALVES = HDP / 64;        // 128-byte column blocks
  static constexpr int TILE = TK * HDP * 2;      // bytes of a K, V or Q tile
  static constexpr int NS = SPLIT ? 2 : 1;       // terms of q and P
  static constexpr int QB = 2 * NS * TILE;
  static constexpr int FIT = (224 * 1024 - QB) / TILE;
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int SMEM = 1024 + QB + STAGES * TILE + 512;
};

struct Ctl {
  uint64_t full[8], empty[8];
  uint64_t tail;     // the last V tile, before its rows past the end are zeroed
  uint64_t q_ready[2], s_full[2], p_full[2], o_full[2];
  uint64_t drain;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Ctl* c, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 15) == 0) {
      if (*(volatile int*)&c->abort) return false;
      if (clock64() - t0 > (1ll << 31)) {  // about a second
        *(volatile int*)&c->abort = 1;
        report(status, ERR_TIMEOUT);
        return false;
      }
    }
  }
}

// the same for all lanes of a warp, which leave it together and with one answer
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, Ctl* c, int* status) {
  return __all_sync(0xffffffffu, wait(bar, parity, c, status));
}

// ---- tcgen05 ------------------------------------------------------------------------
#define R8(c, v, o) c(v[o]), c(v[o + 1]), c(v[o + 2]), c(v[o + 3]), c(v[o + 4]), c(v[o + 5]), c(v[o + 6]), c(v[o + 7])
#define R32(c, v, o) R8(c, v, o), R8(c, v, o + 8), R8(c, v, o + 16), R8(c, v, o + 24)
// 32 columns of the warp's lanes; the wait is in the same statement, so no use moves above it
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n tcgen05.wait::ld.sync.aligned;"
      : R32("=f", v, 0)
      : "r"(addr)
      : "memory");
}
#define R16(c, v, o) R8(c, v, o), R8(c, v, o + 8)
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      " tcgen05.wait::ld.sync.aligned;"
      : R16("=f", v, 0)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      R16("f", v, 0)
      : "memory");
}
__device__ __forceinline__ void tmem_ld64(uint32_t addr, float (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,"
      "%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : R32("=f", v, 0), R32("=f", v, 32)
      : "r"(addr), "r"(addr + 32)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      R32("r", v, 0)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// D += A B with A in shared memory / in TMEM, B in shared memory; f32 accumulator
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(
                   d),
               "l"(a), "l"(b), "r"(idesc), "r"(acc)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle, version 1.  K-major: 8-row
// groups 1024 bytes apart (the leading offset is not used).  MN-major: 64-element
// column blocks `lbo` bytes apart, groups of 8 k-rows 1024 bytes apart.
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 |
         2ull << 61;
}
// instruction descriptor, kind::f16: D f32, A and B f16 (0) or bf16 (1), B K-major or MN-major
__host__ __device__ constexpr uint32_t idesc_f16(int bf16, int n, int b_mn) {
  return 1u << 4 | (uint32_t)bf16 << 7 | (uint32_t)bf16 << 10 | (uint32_t)b_mn << 16 | (uint32_t)(n >> 3) << 17 |
         (uint32_t)(TM >> 4) << 24;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---- rows with a non-finite output ------------------------------------------------------
// One row by one warp, key by key, touching the values of seen keys alone.
template <class KV, int HD>
__device__ __noinline__ void recompute_row(const WindowAttnParams& p, const Tile& t, int hk, int r) {
  const int lane = threadIdx.x & 31, G = p.n_head / p.n_head_kv;
  const int tok = r / G, h = hk * G + r % G, pos = t.past + tok;
  const int64_t q0 = (int64_t)(t.q0 + tok) * p.q_stride + (int64_t)h * HD;
  const SeenPages sp = seen_pages(pos, pos, p.window, p.n_sink);
  constexpr int E = HD / 32;
  float m = -INFINITY, l = 0.f, o[E] = {};
  for (int i0 = 0; i0 < sp.n; i0 += 2) {  // two pages: a key per lane
    const int i = i0 + lane / PG;
    int id = -1;
    float s = -INFINITY;
    if (i < sp.n && key_seen(sp.page(i) * PG + lane % PG, pos, p.window, p.n_sink)) {
      id = p.page_table[(int64_t)t.seq * p.max_pages + sp.page(i)];
      if (id >= p.n_pages) id = -1;
    }
    const int64_t off = id < 0 ? -1 : (((int64_t)id * p.n_head_kv + hk) * PG + lane % PG) * HD;
    if (off >= 0) {
      s = 0.f;
      for (int d = 0; d < HD; ++d)
        s = fmaf(load_elem(p.q, q0 + d, p.io), to_f32<KV>(static_cast<const KV*>(p.k_pages)[off + d]), s);
      s *= p.scale_log2;
    }
    float mx = s;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    mx = fmaxf(mx, m);
    const float ms = mx == -INFINITY ? 0.f : mx;
    const float f = exp2_approx(m - ms), w = exp2_approx(s - ms);
    m = mx;
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= f;
    for (int k = 0; k < 32; ++k) {
      const int64_t at = __shfl_sync(0xffffffffu, off, k);
      const float wk = __shfl_sync(0xffffffffu, w, k);
      if (at < 0) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(wk, to_f32<KV>(static_cast<const KV*>(p.v_pages)[at + lane * E + e]), o[e]);
    }
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
  for (int e = 0; e < E; ++e)
    store_elem(p.out, ((int64_t)(t.q0 + tok) * p.n_head + h) * HD + lane * E + e, o[e] / l, p.io);
}

// ---- the kernel ----------------------------------------------------------------------------
template <class KV, int HD, bool SPLIT>
__global__ void __launch_bounds__(TT, 1)
    prefill_tc_kernel(const __grid_constant__ WindowAttnParams p, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<HD, SPLIT>;
  constexpr bool BF16 = std::is_same<KV, __nv_bfloat16>::value;
  constexpr int HDP = C::HDP, NS = C::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = base;                   // [tile][term][half][128 rows][128 B]
  uint8_t* ring = base + C::QB;         // [stage][half][128 keys][128 B]
  Ctl* c = reinterpret_cast<Ctl*>(base + C::QB + C::STAGES * C::TILE);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int G = p.n_head / p.n_head_kv, hk = blockIdx.x % p.n_head_kv;

  const Tile t = find_tile<TC_ROWS>(p, blockIdx.x / p.n_head_kv);
  if (t.seq < 0) return;  // the whole CTA
  const int n_rows = (int)min((int64_t)TC_ROWS, (int64_t)t.n_q * G - t.row0);
  const int n_tiles = n_rows > TM ? 2 : 1;
  const int p_lo = max(t.past + t.row0 / G, 0), p_hi = t.past + (t.row0 + n_rows - 1) / G;
  SeenPages sp;
  sp.n = sp.sink = sp.first = 0;
  if (p_hi >= 0) sp = seen_pages(p_lo, p_hi, p.window, p.n_sink);
  const int nk = (sp.n + PPT - 1) / PPT;

  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&c->full[i], 1);
      mbar_init(&c->empty[i], 1);
    }
    mbar_init(&c->tail, 1);
    mbar_init(&c->drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c->q_ready[i], TM);
      mbar_init(&c->s_full[i], 1);
      mbar_init(&c->p_full[i], TM);
      mbar_init(&c->o_full[i], 1);
    }
    c->abort = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c->tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  __syncthreads();
  fence_after();
  const uint32_t tmem = c->tmem;  // S tiles at 0 and 128, O tiles at 256 and 256 + HDP

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_SOFTMAX));
    // ---- softmax: thread = row ----
    const int w = warp / 4;  // row tile
    if (w < n_tiles) {
      const int row = w * TM + (warp % 4) * 32 + lane;  // row of the CTA
      const bool live = row < n_rows;
      const int r = t.row0 + row, tok = r / G, h = hk * G + r % G;
      const int pos = live ? t.past + tok : -1;
      // positions of the tile's first and last live rows
      const int t_lo = t.past + (t.row0 + w * TM) / G;
      const int t_hi = t.past + (t.row0 + min(n_rows, w * TM + TM) - 1) / G;
      float scale = p.scale_log2;
      {
        // q into shared memory, swizzled: 16-byte chunk i of the row's 128-byte block at i ^ (row % 8)
        const int lr = row % TM;
        uint8_t* q0 = qs + w * NS * C::TILE + lr * 128;
        const int64_t at = (int64_t)(t.q0 + tok) * p.q_stride + (int64_t)h * HD;
        float up = 1.f;
        if (SPLIT && live) {
          float mx = 0.f;
          for (int d = 0; d < HD; d += 8) {
            Raw8<float> raw;
            float x[8];
            load8(raw, static_cast<const float*>(p.q) + at + d, p.q_vec);
            unpack8(raw, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
          }
          // largest |q| to [1, 2): exact, and undone in the scale
          int e = (int)(__float_as_uint(mx) >> 23) - 127;
          if (mx > 0.f && e < 128) {
            e = max(e, -126);
            up = exp2f((float)-e);  // a power of two: exact
            scale *= exp2f((float)e);
          }
        }
#pragma unroll 2
        for (int d = 0; d < HDP; d += 8) {
          uint8_t* dst = q0 + (d / 64) * (TM * 128) + ((((d % 64) / 8) ^ (lr & 7)) * 16);
          if constexpr (SPLIT) {
            float x[8] = {};
            if (live && d < HD) {
              Raw8<float> raw;
              load8(raw, static_cast<const float*>(p.q) + at + d, p.q_vec);
              unpack8(raw, x);
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float a = x[2 * e] * up, b = x[2 * e + 1] * up;
              hi[e] = pack2<false>(a, b);
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
              lo[e] = pack2<false>(a - f.x, b - f.y);
            }
            *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(dst + C::TILE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          } else {
            Raw8<KV> raw;
            raw.w[0] = make_uint4(0, 0, 0, 0);
            if (live && d < HD) load8(raw, static_cast<const KV*>(p.q) + at + d, p.q_vec);
            *reinterpret_cast<uint4*>(dst) = raw.w[0];
          }
        }
        fence_async_smem();
        mbar_arrive(&c->q_ready[w]);
      }
      const uint32_t lanes = (uint32_t)(warp % 4) * 32 << 16;
      const uint32_t ts = tmem + lanes + w * 128, to = tmem + lanes + 256 + w * HDP;
      constexpr float RAISE = SPLIT ? 0.f : 8.f;   // log2 by which a row may outgrow m
      constexpr float BIAS = SPLIT ? 15.f : 0.f;   // P = 2^BIAS at the maximum
      float m = -INFINITY, l = 0.f;  // m in scaled log2 units
      bool ok = true;
      for (int n = 0; n < nk; ++n) {
        if (!(ok = wait_warp(&c->s_full[w], n & 1, c, p.status))) break;
        fence_after();
        // every key of the tile seen by every row: whole pages, none past the first row's position, all in the last row's window
        const int e0 = n * PPT;
        const bool inner = e0 >= sp.sink && e0 + PPT <= sp.n && sp.page(e0 + PPT - 1) * PG + PG - 1 <= t_lo &&
                           (p.window == 0 || sp.page(e0) * PG > t_hi - p.window);
        // keys 64 b .. 64 b + 63 of the tile that the row does not see become -inf
        auto mask = [&](float (&s)[64], int b) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int e = e0 + 4 * b + g;
            const int jb = e < sp.n ? sp.page(e) * PG : 0x7fffff00;
            const int hi = pos - jb, lo = p.window ? hi - p.window : -1, sk = p.window ? p.n_sink - jb : 0;
#pragma unroll
            for (int k = 0; k < PG; ++k) {
              const bool see = k <= hi && (k > lo || k < sk);
              s[g * PG + k] = see ? s[g * PG + k] : -INFINITY;
            }
          }
        };
        // S is read twice, for the maximum and for P: 128 values held over would not leave registers for P
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          float s[64];
          tmem_ld64(ts + b * 64, s);
          if (!inner) mask(s, b);
          float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int k = 4; k < 64; k += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) m4[i] = fmaxf(m4[i], s[k + i]);
          mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
        }
        mx *= scale;
        if (__any_sync(0xffffffffu, mx > m + RAISE || m == -INFINITY)) {
          const float mn = fmaxf(mx, m);
          const float f = m == -INFINITY ? 0.f : exp2_approx(m - mn);
          m = mn;
          l *= f;
          if (n > 0) {  // O is complete: S(n) came after P V(n - 1)
#pragma unroll 1
            for (int d = 0; d < HDP; d += 16) {
              float o[16];
              tmem_ld16(to + d, o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] *= f;
              tmem_st16(to + d, o);
            }
          }
        }
        const float neg = BIAS - (m == -INFINITY ? 0.f : m);
        float l0 = 0.f, l1 = 0.f;
        uint32_t lo[SPLIT ? 64 : 1];
#pragma unroll
        for (int b = 0; b < 2; ++b) {  // 64 keys: 32 columns of P, over S columns already read
          float s[64];
          tmem_ld64(ts + b * 64, s);
          if (!inner) mask(s, b);
          uint32_t hi[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const float x = exp2_approx(fmaf(s[2 * k], scale, neg));
            const float y = exp2_approx(fmaf(s[2 * k + 1], scale, neg));
            l0 += x;
            l1 += y;
            hi[k] = pack2<BF16>(x, y);
            if constexpr (SPLIT) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
              lo[b * 32 + k] = pack2<false>(x - f.x, y - f.y);
            }
          }
          tmem_st32(ts + b * 32, hi);
        }
        if constexpr (SPLIT) {
#pragma unroll
          for (int b = 0; b < 2; ++b) tmem_st32(ts + 64 + b * 32, reinterpret_cast<const uint32_t(&)[32]>(lo[b * 32]));
        }
        l += l0 + l1;
        tmem_st_wait();
        fence_before();
        mbar_arrive(&c->p_full[w]);
      }
      // ---- out = O / l ----
      if (nk > 0 && ok) {
        ok = wait_warp(&c->o_full[w], 0, c, p.status);
        fence_after();
      }
      if (ok) {
        const float inv = 1.0f / l;
        bool finite = true;
#pragma unroll 1
        for (int d = 0; d < HD; d += 32) {
          float o[32];
          __syncwarp();
          if (nk > 0) tmem_ld32(to + d, o);
          if (live) {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              finite = finite && fabsf(o[k]) < INFINITY;
              o[k] = pos >= 0 ? o[k] * inv : 0.f;
            }
            const int64_t at = ((int64_t)(t.q0 + tok) * p.n_head + h) * HD + d;
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              const float(&x)[8] = *reinterpret_cast<const float(*)[8]>(&o[k]);
              if (SPLIT) store8(static_cast<float*>(p.out) + at + k, x, p.out_vec);
              else store8(static_cast<KV*>(p.out) + at + k, x, p.out_vec);
            }
          }
        }
        __syncwarp();
        // an infinite or NaN value that this row may not see; a sum that is not finite is the row's own
        unsigned again = __ballot_sync(0xffffffffu, live && pos >= 0 && !finite && l < INFINITY);
        while (again) {
          const int src = __ffs(again) - 1;
          again &= again - 1;
          recompute_row<KV, HD>(p, t, hk, __shfl_sync(0xffffffffu, r, src));
        }
      }
    }
  } else {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_OTHER));
  if (warp == 8) {
    // ---- K and V tiles ----
    const int64_t rows = (int64_t)p.n_pages * p.n_head_kv * PG;
    const int* table = p.page_table + (int64_t)t.seq * p.max_pages;
    const int kv_end = t.past + t.n_q;  // keys of the sequence
    bool ok = true;
    for (int n = 0; n < nk && ok; ++n) {
      // lane i < 8: row of page i in the map; outside it (zeros) where there is none
      int y = (int)rows;
      if (lane < PPT && n * PPT + lane < sp.n) {
        const int id = table[sp.page(n * PPT + lane)];
        if (id >= 0 && id < p.n_pages) y = (id * p.n_head_kv + hk) * PG;
        else report(p.status, ERR_BAD_PAGE);
      }
      // rows of the last page past the sequence's end
      const int n_tail = n == nk - 1 ? (sp.page(sp.n - 1) + 1) * PG - kv_end : 0;
      for (int v = 0; v < 2 && ok; ++v) {
        const int i = 2 * n + v, slot = i % C::STAGES;
        if (i >= C::STAGES && !(ok = wait_warp(&c->empty[slot], (uint32_t)(i / C::STAGES - 1) & 1, c, p.status))) break;
        const bool fix = v && n_tail > 0;
        uint64_t* bar = fix ? &c->tail : &c->full[slot];
        if (lane == 0) mbar_arrive_expect_tx(bar, C::TILE);
        __syncwarp();
        const uint32_t dst = smem_u32(ring + slot * C::TILE);
        const int yy = __shfl_sync(0xffffffffu, y, lane % PPT);
        if (lane < PPT * C::HALVES)
          tma_page(dst + (lane / PPT) * (TK * 128) + (lane % PPT) * (PG * 128), v ? &vmap : &kmap, yy, bar, lane / PPT);
        __syncwarp();
        if (fix) {
          ok = wait_warp(&c->tail, 0, c, p.status);
          const int key0 = (sp.n - 1 - n * PPT) * PG + PG - n_tail;
          for (int x = lane; x < n_tail * 8 * C::HALVES; x += 32) {
            const int key = key0 + x / 8 % n_tail, half = x / 8 / n_tail;
            *reinterpret_cast<uint4*>(ring + slot * C::TILE + half * (TK * 128) + key * 128 + x % 8 * 16) =
                make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&c->full[slot]);
        }
      }
    }
  } else if (warp == 9 && lane == 0) {
    // ---- products ----
    constexpr uint32_t QK = idesc_f16(BF16, TK, 0), PV = idesc_f16(BF16, HDP, 1);
    const uint32_t q_addr = smem_u32(qs), ring_addr = smem_u32(ring);
    auto qk = [&](int w, int n) {
      const uint32_t k_addr = ring_addr + (2 * n % C::STAGES) * C::TILE;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int k = 0; k < HDP / 16; ++k) {
          const uint32_t off = (k / 4) * (TM * 128) + (k % 4) * 32;
          mma_ss(tmem + w * 128, desc128(q_addr + (w * NS + s) * C::TILE + off, 16), desc128(k_addr + off, 16), QK, s + k > 0);
        }
      commit(&c->s_full[w]);
    };
    auto pv = [&](int w, int n) {
      const uint32_t v_addr = ring_addr + ((2 * n + 1) % C::STAGES) * C::TILE;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int k = 0; k < TK / 16; ++k)
          mma_ts(tmem + 256 + w * HDP, tmem + w * 128 + s * 64 + k * 8, desc128(v_addr + k * 2048, TK * 128), PV,
                 n > 0 || s + k > 0);
    };
    bool ok = nk > 0;
    for (int w = 0; w < n_tiles && ok; ++w) {
      ok = wait(&c->q_ready[w], 0, c, p.status);
      if (ok && w == 0) ok = wait(&c->full[0], 0, c, p.status);
      if (!ok) break;
      fence_after();
      qk(w, 0);
    }
    if (ok) commit(&c->empty[0]);
    for (int n = 0; n < nk && ok; ++n) {
      const int iv = 2 * n + 1, ik = 2 * n + 2;
      if (!(ok = wait(&c->full[iv % C::STAGES], (uint32_t)(iv / C::STAGES) & 1, c, p.status))) break;
      for (int w = 0; w < n_tiles; ++w) {
        if (!(ok = wait(&c->p_full[w], n & 1, c, p.status))) break;
        fence_after();
        pv(w, n);
        if (w == n_tiles - 1) commit(&c->empty[iv % C::STAGES]);
        if (n + 1 < nk) {
          if (w == 0 && !(ok = wait(&c->full[ik % C::STAGES], (uint32_t)(ik / C::STAGES) & 1, c, p.status))) break;
          qk(w, n + 1);
          if (w == n_tiles - 1) commit(&c->empty[ik % C::STAGES]);
        } else {
          commit(&c->o_full[w]);
        }
      }
    }
  }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (*(volatile int*)&c->abort) {
    // a wait ran out: the products and copies still under way end before the memory goes
    if (warp == 9 && lane == 0) {
      commit(&c->drain);
      for (int i = 0; i < 1 << 14 && !mbar_try_wait(&c->drain, 0); ++i) {
      }
    }
    const long long t0 = clock64();
    while (clock64() - t0 < 1 << 20) {
    }
    __syncthreads();
  }
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---- host -----------------------------------------------------------------------------------
template <class KV, int HD, bool SPLIT>
cudaError_t launch_t(WindowAttnParams& p, int kv, cudaStream_t st) {
  using C = Cfg<HD, SPLIT>;
  CUtensorMap km, vm;
  const int64_t rows = (int64_t)p.n_pages * p.n_head_kv * PG;
  cudaError_t e = pool_map(&km, p.k_pages, kv, HD, rows, 1);
  if (e == cudaSuccess) e = pool_map(&vm, p.v_pages, kv, HD, rows, 1);
  if (e != cudaSuccess) return e;
  const auto kernel = prefill_tc_kernel<KV, HD, SPLIT>;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  const int64_t group = p.n_head / p.n_head_kv;
  const int64_t tiles = p.n_tok * group / TC_ROWS + p.n_seq;
  kernel<<<(unsigned)(tiles * p.n_head_kv), TT, C::SMEM, st>>>(p, km, vm);
  return cudaGetLastError();
}

template <class KV, bool SPLIT>
cudaError_t launch_hd(WindowAttnParams& p, int kv, int hd, cudaStream_t st) {
  if (hd == 32) return launch_t<KV, 32, SPLIT>(p, kv, st);
  if (hd == 64) return launch_t<KV, 64, SPLIT>(p, kv, st);
  return launch_t<KV, 128, SPLIT>(p, kv, st);
}

}  // namespace

bool prefill_tc_takes(const WindowAttnParams& p, int kv, int hd) {
  const int64_t rows = (int64_t)p.n_pages * p.n_head_kv * PG;
  const int64_t tiles = (int64_t)p.n_tok * (p.n_head / p.n_head_kv) / TC_ROWS + p.n_seq;
  if (hd > 128 || rows >= 0x7fffffff || tiles * p.n_head_kv > 0x7fffffff) return false;
  return kv == EL_F16 || (kv == EL_BF16 && p.io == EL_BF16);
}

cudaError_t launch_prefill_tc(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st) {
  (void)sm_count;
  if (kv == EL_BF16) return launch_hd<__nv_bfloat16, false>(p, kv, hd, st);
  if (p.io == EL_F32) return launch_hd<__half, true>(p, kv, hd, st);
  return launch_hd<__half, false>(p, kv, hd, st);
}

}  // namespace sfk
