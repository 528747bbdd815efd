// sfk_paged_prefill_tc.cu -- attention of a ragged batch of prompts over the
// paged cache on the tensor cores (tcgen05), for 16-bit caches.
//
//   S = Q K^T;  P = 2^(scale S - m);  O = sum over key tiles of P V;  out = O / sum P
//
// A CTA takes two tiles of 128 rows (rows: tokens x the query heads of one kv
// head) and walks the pages its rows see in tiles of TK keys:
//   warps 0-3, 4-7  softmax of row tile 0 and 1: thread = TMEM lane = row.
//                   Reads its S row into registers, updates the running maximum,
//                   writes P to TMEM as 16-bit A operands.
//   warps 8 and 10  bring K and V tiles in, page by page, by tensor-map copies
//                   (128-byte swizzle), into a ring of tiles each.
//   warps 9 and 11  one thread each issues Q K^T and P V of both row tiles.
// S, P and O of both row tiles live in TMEM side by side: S(n + 1) is computed as
// soon as S(n) is in registers, under the exponentials of S(n), so a softmax warp
// goes from tile to tile without waiting for the tensor core.  That sets TK: 80 keys
// at head width 128 (S 2 x 80, P 2 x 40, O 2 x 128 of 512 columns); at 64 there would
// be room for 128, and 96 were faster (245 and 252 us for a ragged batch of 7308
// tokens of 32 heads, 123 GFLOP): a row of 128 leaves too few registers.
// (P over S with 128 keys, the products of a tile in one chain with its softmax, took
// 892 us for 2048 tokens at 30000 keys, 32 heads of 128.)
// One thread issues in about 30 cycles a product and 100 a wait: Q K^T and P V
// by one thread were what the kernel waited for.
//
// Heads of 256 take one row tile: its O is half of TMEM, and q and two stages of K and
// V of 80 keys fill shared memory.  4096 tokens, 16 heads over 8 (137 GFLOP): 157 us,
// 0.87 PFLOP/s, where the CUDA cores reach 13 TFLOP/s.
//
// Bound by the tensor core and the exponentials, which take about as long, under
// the card's power limit: 2048 tokens at 30000 keys, 32 heads of 128 over 8, bf16
// (974 GFLOP): 810 us in a burst (1.20 PFLOP/s), 920 back to back at 1.6 GHz and 1000 W
// (1.06 PFLOP/s, 0.75 of what a library product sustains there).  8192 tokens through
// a window of 2048 (241 GFLOP): 262 us; a CTA walks 27 key tiles there and spends
// a sixth of its time before the first and after the last.
//
// The running maximum m is only raised when a row outgrows it, in bf16 by 2^8: O
// is rescaled then, by the row's own thread.  P is rounded once to the cache's
// type, and the sum stays in 32 bits.  bf16 has the range of f32: P is 1 at m and
// 2^8 at most.  f16's smallest step is 2^-24, and a long tail of weights far below
// the row's largest would fall under it while the sum keeps them (one key 18 nats
// above 30000 others: 0.95 of the tail lost): P is 2^11 at m, 2^15 at most, and a
// weight is held to half a step of f16 or 2^-36 of the largest.
//
// The accumulator of a product drops what falls below its last bits, each time, towards
// 0: 8.3e-4 of values of one sign were gone after 131072 keys, more than half a step of
// f16.  So f16 rows start O anew every 10240 keys and keep the sum in local memory, added
// to the nearest (6.7e-5; 2048 tokens at 30000 keys, 32 heads of 128: 875 us with and
// without, heads of 64: 858 and 832).  bf16 rows do so every 81920 keys where a CTA may
// walk more than 131072: up to there one accumulator loses a fifth of their half step, and
// the second loop around the tiles takes 2 %.
//
// 32-bit rows over an f16 cache (SPLIT): q, scaled by a power of two per row,
// is the sum of two f16 numbers and so is each P (22 bits), and each product
// is two.  P's range is that of f16 rows, so that its second part too stays above
// f16's smallest step.  A bf16 pair holds 16 bits only: that cache takes the
// CUDA-core kernel.  One row tile per CTA then, and the second warpgroup keeps the
// sum of the key tiles' O (below, at the sum).  512 tokens at 1012 keys, 32 heads of
// 128 over 8: 29 us, a CTA to each of the 128 row tiles; 2048 at 8048 keys 465 us, 0.51
// PFLOP/s of the formula's products, half of those it does.  (Two softmax threads to a row and
// the sum in a third warpgroup: 45 and 851 us, its registers no longer fit.)
//
// What a masked place holds does not matter: K only reaches its own column of
// S, which is replaced; V rows past the sequence's length are zeroed in shared
// memory; a V row that some rows of a tile see and others do not reaches the
// others as 0 * v, which is NaN for an infinite v: rows whose output is not
// finite are computed again key by key (recompute_row).
#include <cooperative_groups.h>

#include <type_traits>

#include "sfk_paged.cuh"
#include "sfk_paged_map.cuh"

namespace sfk {
namespace {

namespace cg = cooperative_groups;

constexpr int TM = 128;       // rows per tile
constexpr int TT = 384;       // threads: three warpgroups, 168 registers each at launch
template <int HD, bool SPLIT>
struct Cfg {
  static constexpr int HDP = HD < 64 ? 64 : HD;  // head width in shared memory (the copy fills with zeros)
  static constexpr int HALVES = HDP / 64;        // 128-byte column blocks
  static constexpr int NS = SPLIT ? 2 : 1;       // terms of q and P
  static constexpr int TILES = SPLIT || HD > 128 ? 1 : 2;  // row tiles per CTA
  static constexpr int OBUF = SPLIT ? 2 : TILES;           // O tiles
  static constexpr int ROWS = TILES * TM;
  // Keys per tile: S (TK columns), P (TK / 2 a term) and O (HDP) of two row tiles, or of one (with a second O; with an
  // O of 256), share the 512 columns of TMEM
  static constexpr int TK = HDP == 64 || SPLIT ? 96 : 80;
  static constexpr int PPT = TK / PG;            // pages per key tile
  static constexpr int TILE = TK * HDP * 2;      // bytes of a K or V tile
  static constexpr int QTILE = TM * HDP * 2;     // bytes of a q term of a row tile
  static constexpr int QB = TILES * NS * QTILE;
  static constexpr int FIT = (224 * 1024 - QB) / (2 * TILE);
  static constexpr int STAGES = FIT > 4 ? 4 : FIT;  // K tiles, and V tiles, under way
  static constexpr int SMEM = 1024 + QB + 2 * STAGES * TILE + (SPLIT ? 4096 : 512);
  static constexpr int FIRST = (PPT + 1) / 2 * PG;  // keys of the first part of P
  // Of 8 exponentials, how many go to the multiply-add unit (0 / 1 / 2 / 3: 1003 / 946 / 933 / 944 us at width 128,
  // 2048 tokens at 30000 keys; 1 / 2 / 3: 233 / 238 / 253 at 64, the ragged batch)
  static constexpr int POLY_OF_8 = SPLIT ? 0 : HDP == 64 ? 1 : 2;
  // Registers after the split: 384 x 168 is what the launch holds.  A softmax thread holds a row of S.
  static constexpr int REG_SOFTMAX = 184, REG_OTHER = 136;
  static_assert(2 * 128 * REG_SOFTMAX + 128 * REG_OTHER <= TT * 168, "register split above the launch's");
  // TMEM columns
  static constexpr int P0 = TILES * TK, PCOLS = TK / 2 * NS, O0 = 512 - OBUF * HDP;
  static_assert(P0 + TILES * PCOLS <= O0 && STAGES >= 2 && TK % PG == 0, "tile sizes");
};

// Keys that meet in one accumulator of 16-bit rows, and how many may without a kernel of RUNS
template <class KV>
constexpr int RUN_KEYS = std::is_same<KV, __nv_bfloat16>::value ? 81920 : 10240;
template <class KV>
constexpr int64_t MAX_RUN_KEYS = std::is_same<KV, __nv_bfloat16>::value ? 131072 : 0;

struct Ctl {
  uint64_t full[2][4], empty[2][4];  // [K, V][stage]
  uint64_t tail;                     // the last V tile, before its rows past the end are zeroed
  uint64_t q_ready[2];
  uint64_t s_full[2], s_free[2];     // S of a row tile is complete / is in registers
  uint64_t p_full[2][2];             // [row tile][part of the keys]: P is written
  uint64_t pv_done[2];               // O is complete and P is free
  // SPLIT: O of tile n is complete in buffer n % 2 / has been added; the factor of tile n is in slot n % 4
  uint64_t o_full[2], o_free[2], f_full[4];
  uint64_t drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Ctl) <= 512, "the control block's place");

// Bounded: false after about a second, or once another warp gave up.  Little code, for the loops that call it.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, Ctl* c) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity))
    if (clock64() - t0 > (1ll << 31) || *(volatile int*)&c->abort) {
      *(volatile int*)&c->abort = 1;
      return false;
    }
  return true;
}
// the same for all lanes of a warp, which leave it together and with one answer
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, Ctl* c) {
  return __all_sync(0xffffffffu, wait(bar, parity, c));
}
// one lane of the warp, always the same
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(on));
  return on;
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
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[80]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%80];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%81];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79},"
      " [%82];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : R32("=f", v, 0), R32("=f", v, 32), R16("=f", v, 64)
      : "r"(addr), "r"(addr + 32), "r"(addr + 64)
      : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[96]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%96];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%97];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
      "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95}, [%98];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : R32("=f", v, 0), R32("=f", v, 32), R32("=f", v, 64)
      : "r"(addr), "r"(addr + 32), "r"(addr + 64)
      : "memory");
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), R8("r", v, 0)
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Shared-memory matrix descriptor, 128-byte swizzle, version 1.  K-major: 8-row
// groups 1024 bytes apart (the leading offset is not used).  MN-major: 64-element
// column blocks `lbo` bytes apart, groups of 8 k-rows 1024 bytes apart.
constexpr uint32_t DESC_HI = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3FFFu) | lbo >> 4 << 16; }
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// D += A B with A in shared memory / in TMEM, B in shared memory; f32 accumulator.  a, b: low descriptor words.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI)
      : "memory");
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

// 2^x of a pair without the special-function unit, which has 4 lanes where the
// multiply-add unit has 32: x = n + f with n the nearest whole number (the low
// bits of x + 1.5 2^23), 2^f on [-1/2, 1/2] by a polynomial of least relative
// error (Lawson's iteration), n added to the exponent.  Relative error 7.5e-5 at
// degree 3, 2.7e-6 at degree 4: well below the rounding of P to bf16 (2^-8) and
// f16 (2^-11).  x below -126 gives 2^-126, which is 0 in f16.  bf16 holds it, and a masked key's value may be
// 3e38: there x2 comes 24 larger, and the factor 2^-24 at the end flushes all below 2^-126 to 0.
constexpr float POLY_UP = 24.f;
template <bool BF16>
__device__ __forceinline__ void exp2_poly(uint64_t x2, float& x, float& y) {
  unpair(x2, x, y);
  x2 = pair(fmaxf(x, -126.f), fmaxf(y, -126.f));
  const uint64_t t = add2(x2, both(12582912.f));
  const uint64_t f = fma2(add2(t, both(-12582912.f)), both(-1.f), x2);
  uint64_t r;
  if constexpr (BF16) {
    r = fma2(both(0.0551716685295105f), f, both(0.2426111251115799f));
    r = fma2(r, f, both(0.6932609677314758f));
    r = fma2(r, f, both(0.9999280571937561f));
  } else {
    r = fma2(both(0.009570102207362652f), f, both(0.05591785907745361f));
    r = fma2(r, f, both(0.240247443318367f));
    r = fma2(r, f, both(0.6931217908859253f));
    r = fma2(r, f, both(0.9999992847442627f));
  }
  float a, b, u, v;
  unpair(r, a, b);
  unpair(t, u, v);
  x = __int_as_float(__float_as_int(a) + (__float_as_int(u) << 23));
  y = __int_as_float(__float_as_int(b) + (__float_as_int(v) << 23));
  if constexpr (BF16) unpair(mul2_ftz(pair(x, y), both(1.f / (1 << (int)POLY_UP))), x, y);
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
template <class KV, int HD, bool SPLIT, bool RUNS>  // RUNS: O is the sum of several accumulators
__global__ void __launch_bounds__(TT, 1)
    prefill_tc_kernel(const __grid_constant__ WindowAttnParams p, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<HD, SPLIT>;
  constexpr bool BF16 = std::is_same<KV, __nv_bfloat16>::value;
  constexpr int HDP = C::HDP, NS = C::NS, TK = C::TK, PPT = C::PPT;
  constexpr int RUN = RUNS ? RUN_KEYS<KV> / TK : 1 << 30;  // key tiles of one
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* qs = base;                   // [tile][term][half][128 rows][128 B]
  uint8_t* ring = base + C::QB;         // [K, V][stage][half][TK keys][128 B]
  Ctl* c = reinterpret_cast<Ctl*>(base + C::QB + 2 * C::STAGES * C::TILE);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int parts = p.key_parts, part = blockIdx.x % parts, job = blockIdx.x / parts;
  const int G = p.n_head / p.n_head_kv, hk = job % p.n_head_kv;

  const Tile t = find_tile(p, job / p.n_head_kv, p.tile_rows);
  if (t.seq < 0) return;  // the whole cluster
  const int n_rows = (int)min((int64_t)p.tile_rows, (int64_t)t.n_q * G - t.row0);
  const int n_tiles = n_rows > TM ? 2 : 1;  // row tiles
  const int p_lo = max(t.past + t.row0 / G, 0), p_hi = t.past + (t.row0 + n_rows - 1) / G;
  SeenPages sp;
  sp.n = sp.sink = sp.first = 0;
  if (p_hi >= 0) sp = seen_pages(p_lo, p_hi, p.window, p.n_sink);
  // this CTA's key tiles: n_first .. n_first + nk - 1 of n_all
  const int n_all = (sp.n + PPT - 1) / PPT;
  const int n_first = (int)((int64_t)n_all * part / parts), nk = (int)((int64_t)n_all * (part + 1) / parts) - n_first;

  if (tid == 0) {
    for (int v = 0; v < 2; ++v)
      for (int i = 0; i < C::STAGES; ++i) {
        mbar_init(&c->full[v][i], 1);
        mbar_init(&c->empty[v][i], 1);
      }
    mbar_init(&c->tail, 1);
    mbar_init(&c->drain, 2);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&c->q_ready[i], TM);
      mbar_init(&c->s_full[i], 1);
      mbar_init(&c->s_free[i], 4);  // warps
      mbar_init(&c->p_full[i][0], 4);
      mbar_init(&c->p_full[i][1], 4);
      mbar_init(&c->pv_done[i], 1);
      mbar_init(&c->o_full[i], 1);
      mbar_init(&c->o_free[i], 4);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&c->f_full[i], 4);
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
  const uint32_t tmem = c->tmem;
  float* stage = reinterpret_cast<float*>(base);                // [ROWS][HD]: a part's O
  float2* ml = reinterpret_cast<float2*>(stage + C::ROWS * HD);  // [ROWS]: its m and l
  float* factor = reinterpret_cast<float*>(c) + 128;            // SPLIT: [4][TM] factors of tiles, then m and l [TM]
  float2* last = reinterpret_cast<float2*>(factor + 4 * TM);

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REG_SOFTMAX));
    // ---- softmax: thread = row ----
    const int w = SPLIT ? 0 : warp / 4;  // row tile
    const bool adds = SPLIT && warp >= 4;  // the warpgroup that keeps the sum of the tiles' O
    if (w < n_tiles) {
      const int row = w * TM + (warp % 4) * 32 + lane;  // row of the CTA
      const bool live = row < n_rows;
      const int r = t.row0 + row, tok = r / G, h = hk * G + r % G;
      const int pos = live ? t.past + tok : -1;
      // positions of the tile's first and last live rows
      const int t_lo = t.past + (t.row0 + w * TM) / G;
      const int t_hi = t.past + (t.row0 + min(n_rows, w * TM + TM) - 1) / G;
      float scale = p.scale_log2;
      const int wrow = w * TM + (warp % 4) * 32;  // first row of the warp
      // A row of q by HD / 8 lanes, 16 bytes of a 16-bit type each, two or more rows at a time (thread by row
      // instead, the loads of a warp go to 32 rows: measured 10k cycles for the tile, and this is before the
      // first product).  Into shared memory swizzled: 16-byte chunk i of the row's 128-byte block at i ^ (row % 8).
      constexpr int LR = HD / 8, RI = 32 / LR;  // lanes per row, rows per step
      const int64_t my_q = live ? (int64_t)(t.q0 + tok) * p.q_stride + (int64_t)h * HD : -1;
      if (nk > 0 && !adds) {
        const int ch = lane % LR;
        auto slot = [&](int lr, int c) {  // row of the tile, chunk of the row
          return qs + w * NS * C::QTILE + lr * 128 + c / 8 * (TM * 128) + ((c % 8) ^ (lr & 7)) * 16;
        };
        if constexpr (SPLIT) {
#pragma unroll 1
          for (int i0 = 0; i0 < LR; i0 += (LR < 8 ? LR : 8)) {
            constexpr int B = LR < 8 ? LR : 8;
            Raw8<float> raw[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
              const int64_t at = __shfl_sync(0xffffffffu, my_q, (i0 + i) * RI + lane / LR);
              raw[i].w[0] = raw[i].w[1] = make_uint4(0, 0, 0, 0);
              if (at >= 0) load8(raw[i], static_cast<const float*>(p.q) + at + ch * 8, p.q_vec);
            }
#pragma unroll
            for (int i = 0; i < B; ++i) {
              const int rr = (i0 + i) * RI + lane / LR;  // row of the warp
              float x[8], mx = 0.f;
              unpack8(raw[i], x);
#pragma unroll
              for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
#pragma unroll
              for (int d = 1; d < LR; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
              // the row's largest |q| to [1, 2): a power of two, exact, undone in the row's scale
              int e = (int)(__float_as_uint(mx) >> 23) - 127;
              e = mx > 0.f && e < 128 ? min(max(e, -126), 126) : 0;
              const float up = __uint_as_float((uint32_t)(127 - e) << 23);
              const int er = __shfl_sync(0xffffffffu, e, lane % RI * LR);
              if (lane / RI == i0 + i) scale = p.scale_log2 * __uint_as_float((uint32_t)(er + 127) << 23);
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float u = x[2 * k] * up, v = x[2 * k + 1] * up;
                hi[k] = pack2<false>(u, v);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
                lo[k] = pack2<false>(u - f.x, v - f.y);
              }
              uint8_t* dst = slot(wrow % TM + rr, ch);
              *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              *reinterpret_cast<uint4*>(dst + C::QTILE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
          }
        } else {
          constexpr int B = LR < 16 ? LR : 16;
#pragma unroll 1
          for (int i0 = 0; i0 < LR; i0 += B) {
            Raw8<KV> raw[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {
              const int64_t at = __shfl_sync(0xffffffffu, my_q, (i0 + i) * RI + lane / LR);
              raw[i].w[0] = make_uint4(0, 0, 0, 0);
              if (at >= 0) load8(raw[i], static_cast<const KV*>(p.q) + at + ch * 8, p.q_vec);
            }
#pragma unroll
            for (int i = 0; i < B; ++i)
              *reinterpret_cast<uint4*>(slot(wrow % TM + (i0 + i) * RI + lane / LR, ch)) = raw[i].w[0];
          }
        }
        if constexpr (HDP > HD) {  // dims past the head
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int k = HD / 8; k < HDP / 8; ++k)
              *reinterpret_cast<uint4*>(slot(wrow % TM + lane, k) + s * C::QTILE) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        mbar_arrive(&c->q_ready[w]);
      }
      const uint32_t lanes = (uint32_t)(warp % 4) * 32 << 16;
      const uint32_t ts = tmem + lanes + w * TK, tp = tmem + lanes + C::P0 + w * C::PCOLS, to = tmem + lanes + C::O0 + w * HDP;
      constexpr float RAISE = BF16 ? 8.f : 4.f;  // log2 by which a row may outgrow m
      constexpr float BIAS = BF16 ? 0.f : 11.f;  // P = 2^BIAS at m
      bool ok = true;
      auto done = [&](uint64_t* bar) {  // what this warp's lanes did in TMEM so far
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
      };
      // ---- out = O / l, columns(d, o) being 32 columns of O from d on ----
      auto finish = [&](auto columns, float m, float l) {
        if (parts > 1) {
        // A part of the keys: O, m and l to shared memory (over q and the ring),
        // 16-byte chunk i of a row at i ^ (row % 8); the cluster adds the parts below.
        float* o_row = stage + (w * TM + (warp % 4) * 32 + lane) * HD;
        if (nk > 0) {
#pragma unroll(SPLIT ? HD / 32 : 1)
          for (int d = 0; d < HD; d += 32) {
            float o[32];
            __syncwarp();
            columns(d, o);
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<float4*>(o_row + (((d + k) / 4) ^ (lane & 7)) * 4) =
                  make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
        }
          ml[w * TM + (warp % 4) * 32 + lane] = make_float2(m, l);
          return;
        }
        // Through shared memory (the tile's q, whose products are done), so that a warp writes whole rows: 16-byte
        // chunk i of a row at i ^ (row % 8).
        constexpr int ES = SPLIT ? 4 : 2, CH = HD * ES / 16;  // bytes of an output element, chunks of a row
        constexpr int X = CH < 8 ? CH - 1 : 7;
        uint8_t* rows = qs + w * NS * C::QTILE + wrow % TM * (HD * ES);
        // a row whose every seen score is -inf has no weights: NaN, where the polynomial's 2^-126 would leave a sum
        const float inv = 1.0f / (m == -INFINITY ? 0.f : l);
        bool finite = true;
#pragma unroll(SPLIT ? HD / 32 : 1)
        for (int d = 0; d < HD; d += 32) {
          float o[32];
          if (nk > 0) columns(d, o);
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            finite = finite && fabsf(o[k]) < INFINITY;
            o[k] = pos >= 0 ? o[k] * inv : 0.f;
          }
          uint8_t* mine = rows + lane * (HD * ES);
#pragma unroll
          for (int k = 0; k < 32; k += 16 / ES) {
            uint4 v;
            if constexpr (SPLIT)
              v = make_uint4(__float_as_uint(o[k]), __float_as_uint(o[k + 1]), __float_as_uint(o[k + 2]), __float_as_uint(o[k + 3]));
            else
              v = make_uint4(pack2<BF16>(o[k], o[k + 1]), pack2<BF16>(o[k + 2], o[k + 3]), pack2<BF16>(o[k + 4], o[k + 5]),
                             pack2<BF16>(o[k + 6], o[k + 7]));
            *reinterpret_cast<uint4*>(mine + ((((d + k) * ES / 16) ^ (lane & X)) * 16)) = v;
          }
        }
        __syncwarp();
        const int64_t my_out = live ? ((int64_t)(t.q0 + tok) * p.n_head + h) * HD : -1;
        constexpr int RO = 32 / CH;  // rows per step
#pragma unroll 4
        for (int i = 0; i < CH; ++i) {
          const int rr = i * RO + lane / CH, ch = lane % CH;
          const int64_t at = __shfl_sync(0xffffffffu, my_out, rr);
          const uint4 v = *reinterpret_cast<const uint4*>(rows + rr * (HD * ES) + ((ch ^ (rr & X)) * 16));
          if (at >= 0) {
            uint8_t* dst = static_cast<uint8_t*>(p.out) + (at * ES + ch * 16);
            if (p.out_vec) {
              *reinterpret_cast<uint4*>(dst) = v;
            } else {  // rows off 16-byte boundaries
              const uint16_t* e = reinterpret_cast<const uint16_t*>(&v);
#pragma unroll
              for (int k = 0; k < 8; ++k) reinterpret_cast<uint16_t*>(dst)[k] = e[k];
            }
          }
        }
        __syncwarp();
        // an infinite or NaN value that this row may not see; a sum that is not finite is the row's own, unless the two
        // terms of q met an infinite key with two signs
        unsigned again = __ballot_sync(0xffffffffu, live && pos >= 0 && !finite && (SPLIT || l < INFINITY));
        while (again) {
          const int src = __ffs(again) - 1;
          again &= again - 1;
          recompute_row<KV, HD>(p, t, hk, __shfl_sync(0xffffffffu, r, src));
        }
      };
      if (!adds) {
        float m = -INFINITY, l = 0.f;  // m in scaled log2 units
        // O of whole runs of RUN key tiles, in units of 2^kept_m: in local memory, touched once a run
        volatile float kept[RUNS ? HDP : 1];
        float kept_m = -INFINITY;
        auto fold = [&](bool any) {  // any: there are kept sums.  O is complete, and 0 from here on.
          const float f = kept_m == -INFINITY ? 0.f : exp2_approx(kept_m - m);
          kept_m = m;
#pragma unroll 1
          for (int d = 0; d < HDP; d += 16) {
            float o[16];
            tmem_ld16(to + d, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              kept[d + k] = any ? fmaf(kept[d + k], f, o[k]) : o[k];
              o[k] = 0.f;
            }
            tmem_st16(to + d, o);
          }
          tmem_st_wait();
        };
        for (int n0 = 0; n0 < (RUNS ? nk : 1) && ok; n0 += RUN) {
          if (RUNS && n0 > 0) {
            if (!(ok = wait_warp(&c->pv_done[w], (n0 - 1) & 1, c))) break;
            fence_after();
            fold(n0 > RUN);
          }
          const int n1 = RUNS ? min(n0 + RUN, nk) : nk;
          for (int n = n0; n < n1; ++n) {
            if (!(ok = wait_warp(&c->s_full[w], n & 1, c))) break;
            fence_after();
            // every key of the tile seen by every row: whole pages, none past the first row's position, all in the last row's window
            const int e0 = (n_first + n) * PPT;
            const bool inner = e0 >= sp.sink && e0 + PPT <= sp.n && sp.page(e0 + PPT - 1) * PG + PG - 1 <= t_lo &&
                               (p.window == 0 || sp.page(e0) * PG > t_hi - p.window);
            if (!inner) {
              // what the row does not see becomes -inf, in place
#pragma unroll 1
              for (int g = 0; g < PPT; ++g) {
                const int jb = e0 + g < sp.n ? sp.page(e0 + g) * PG : 0x7fffff00;
                if (jb + PG - 1 <= t_lo && (p.window == 0 || jb > t_hi - p.window)) continue;  // every row sees the page
                const int hi = pos - jb, lo = p.window ? hi - p.window : -1, sk = p.window ? p.n_sink - jb : 0;
                float s[16];
                tmem_ld16(ts + g * PG, s);
#pragma unroll
                for (int k = 0; k < PG; ++k) s[k] = k <= hi && (k > lo || k < sk) ? s[k] : -INFINITY;
                tmem_st16(ts + g * PG, s);
              }
              tmem_st_wait();
            }
            float s[TK];
            tmem_ld(ts, s);
            if (n + 1 < nk) done(&c->s_free[w]);  // the next Q K^T may begin
            float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int k = 4; k < TK; k += 4)
#pragma unroll
              for (int i = 0; i < 4; ++i) m4[i] = max_nan(m4[i], s[k + i]);
            float mx = max_nan(max_nan(m4[0], m4[1]), max_nan(m4[2], m4[3]));
            // O is complete and P may be written again (mostly long since)
            if (n > 0) {
              if (!(ok = wait_warp(&c->pv_done[w], (n - 1) & 1, c))) break;
              fence_after();
            }
            mx *= scale;
            float f = 1.f;
            if (__any_sync(0xffffffffu, !(mx <= m + RAISE))) {
              // a row that saw a score of NaN or +inf is NaN, by its m: the polynomial below does not carry these on
              const float mn = max_nan(mx, m) < INFINITY ? fmaxf(mx, m) : NAN;
              f = m == -INFINITY ? 0.f : exp2_approx(m - mn);
              m = mn;
              l *= f;
              if (!SPLIT && n > 0) {
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
            if constexpr (SPLIT) {  // the other warpgroup rescales
              factor[n % 4 * TM + row] = f;
              __syncwarp();
              if (lane == 0) mbar_arrive(&c->f_full[n % 4]);
            }
            const float neg = BIAS - (m == -INFINITY ? 0.f : m);
            const uint64_t scale2 = both(scale), neg2 = both(neg), up2 = both(neg + POLY_UP);
            uint64_t sum2 = 0;
#pragma unroll
            for (int b = 0; b < PPT; ++b) {  // 16 keys: 8 columns of P
              uint32_t hi[8], lo[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const bool poly = (k * 3) % 8 < C::POLY_OF_8;
                const uint64_t x2 = fma2(pair(s[b * 16 + 2 * k], s[b * 16 + 2 * k + 1]), scale2, BF16 && poly ? up2 : neg2);
                float x, y;
                if (poly) {
                  exp2_poly<BF16>(x2, x, y);
                } else {
                  unpair(x2, x, y);
                  x = exp2_approx(x);
                  y = exp2_approx(y);
                }
                sum2 = add2(sum2, pair(x, y));
                hi[k] = pack2<BF16>(x, y);
                if constexpr (SPLIT) {
                  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
                  lo[k] = pack2<false>(x - f.x, y - f.y);
                }
              }
              tmem_st8(tp + b * 8, hi);
              if constexpr (SPLIT) tmem_st8(tp + TK / 2 + b * 8, lo);
              if ((b + 1) * PG == C::FIRST) {  // the product of these keys may begin
                tmem_st_wait();
                done(&c->p_full[w][0]);
              }
            }
            float l0, l1;
            unpair(sum2, l0, l1);
            l += l0 + l1;
            tmem_st_wait();
            done(&c->p_full[w][1]);
          }
        }
        if constexpr (SPLIT) {
          last[row] = make_float2(m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(&c->f_full[nk % 4]);
        } else {
          if (nk > 0 && ok) {
            ok = wait_warp(&c->pv_done[w], (nk - 1) & 1, c);
            fence_after();
          }
          if (parts > 1) asm volatile("bar.sync 1, %0;" ::"r"(n_tiles * TM) : "memory");  // both row tiles are through
          if (ok)
            finish(
                [&](int d, float(&o)[32]) {
                  tmem_ld32(to + d, o);
                  if (RUNS && nk > RUN) {
                    const float f = kept_m == -INFINITY ? 0.f : exp2_approx(kept_m - m);
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = fmaf(kept[d + k], f, o[k]);
                  }
                },
                m, l);
        }
      } else if constexpr (SPLIT) {
        // Each tile's O is a product of its own, added here: the tensor core's f32 accumulator drops what falls below
        // its last bit, a loss that grows with the products on one accumulator (-7.6e-6 of the result over 440 of them).
        float acc[HD];
#pragma unroll
        for (int k = 0; k < HD; ++k) acc[k] = 0.f;
        for (int n = 0; n < nk; ++n) {
          if (!(ok = wait_warp(&c->f_full[n % 4], n / 4 & 1, c))) break;
          const float f = factor[n % 4 * TM + row];
          if (!(ok = wait_warp(&c->o_full[n % 2], n / 2 & 1, c))) break;
          fence_after();
#pragma unroll
          for (int d = 0; d < HD; d += 32) {
            float o[32];
            tmem_ld32(to + n % 2 * HDP + d, o);
#pragma unroll
            for (int k = 0; k < 32; ++k) acc[d + k] = fmaf(acc[d + k], f, o[k]);
          }
          done(&c->o_free[n % 2]);
        }
        if (ok && (ok = wait_warp(&c->f_full[nk % 4], nk / 4 & 1, c))) {
          const float2 x = last[row];
          finish(
              [&](int d, float(&o)[32]) {
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = acc[d + k];
              },
              x.x, x.y);
        }
      }
    }
  } else {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REG_OTHER));
  if (warp == 8 || warp == 10) {
    // ---- K tiles (warp 8) and V tiles (warp 10) ----
    const int v = warp == 10;
    const CUtensorMap* map = v ? &vmap : &kmap;
    const int past_end = p.n_pages * p.n_head_kv * PG;  // a row outside the map: zeros
    const int* table = p.page_table + (int64_t)t.seq * p.max_pages;
    const int kv_end = t.past + t.n_q;  // keys of the sequence
    // lane i: row in the map of page entry e + i, for as many whole tiles as 32 lanes hold
    constexpr int AHEAD = 32 / PPT;
    auto rows_from = [&](int e) {
      int y = past_end;
      if (e + lane < sp.n) {
        const int id = table[sp.page(e + lane)];
        if (id >= 0 && id < p.n_pages) y = (id * p.n_head_kv + hk) * PG;
        else report(p.status, ERR_BAD_PAGE);
      }
      return y;
    };
    int ahead = rows_from(n_first * PPT), y = past_end, in = 0, slot = 0;
    uint32_t use = 0;  // how often the slot was filled before
    bool ok = true;
    for (int n = 0; n < nk && ok; ++n) {
      if (in == 0) {
        y = ahead;
        ahead = rows_from((n_first + n + AHEAD) * PPT);
      }
      // rows of the last page past the sequence's end
      const int n_tail = v && n_first + n == n_all - 1 ? (sp.page(sp.n - 1) + 1) * PG - kv_end : 0;
      if (use > 0 && !(ok = wait_warp(&c->empty[v][slot], (use - 1) & 1, c))) break;
      uint64_t* bar = n_tail > 0 ? &c->tail : &c->full[v][slot];
      if (lane == 0) mbar_arrive_expect_tx(bar, C::TILE);
      __syncwarp();
      uint8_t* tile = ring + (v * C::STAGES + slot) * C::TILE;
      const int yy = __shfl_sync(0xffffffffu, y, in * PPT + lane % PPT);
      if (lane < PPT * C::HALVES)
        tma_page(smem_u32(tile) + (lane / PPT) * (TK * 128) + (lane % PPT) * (PG * 128), map, yy, bar, lane / PPT);
      __syncwarp();
      if (n_tail > 0) {
        ok = wait_warp(&c->tail, 0, c);
        const int key0 = (sp.n - 1 - (n_first + n) * PPT) * PG + PG - n_tail;
        for (int x = lane; x < n_tail * 8 * C::HALVES; x += 32) {
          const int key = key0 + x / 8 % n_tail, half = x / 8 / n_tail;
          *reinterpret_cast<uint4*>(tile + half * (TK * 128) + key * 128 + x % 8 * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c->full[v][slot]);
      }
      if (++slot == C::STAGES) slot = 0, ++use;
      if (++in == AHEAD) in = 0;
    }
  } else if (elect_one()) {
    // ---- products, one thread each: Q K^T (warp 9), P V (warp 11) ----
    // One thread for a whole loop: a vote or a warp barrier at each wait would cost more than the wait.
    if (warp == 9) {
      constexpr uint32_t QK = idesc_f16(BF16, TK, 0);
      const uint32_t q_lo = desc_lo(smem_u32(qs), 16), k_lo = desc_lo(smem_u32(ring), 16);
      int slot = 0;
      uint32_t use = 0;
      bool ok = true;
      for (int n = 0; n < nk && ok; ++n) {
        if (!(ok = wait(&c->full[0][slot], use & 1, c))) break;
#pragma unroll 1
        for (int w = 0; w < n_tiles; ++w) {
          if (!(ok = n == 0 ? wait(&c->q_ready[w], 0, c) : wait(&c->s_free[w], (n - 1) & 1, c))) break;
          fence_after();
          const uint32_t a = q_lo + w * (NS * C::QTILE >> 4), b = k_lo + slot * (C::TILE >> 4), d = tmem + w * TK;
#pragma unroll
          for (int s = NS - 1; s >= 0; --s)
#pragma unroll
            for (int k = 0; k < HDP / 16; ++k)
              mma_ss(d, a + ((s * C::QTILE + k / 4 * (TM * 128) + k % 4 * 32) >> 4),
                     b + ((k / 4 * (TK * 128) + k % 4 * 32) >> 4), QK, NS - 1 - s + k > 0);
          commit(&c->s_full[w]);
          if (w == n_tiles - 1) commit(&c->empty[0][slot]);
        }
        if (++slot == C::STAGES) slot = 0, ++use;
      }
    } else if (warp == 11) {
      constexpr uint32_t PV = idesc_f16(BF16, HDP, 1);
      const uint32_t v_lo = desc_lo(smem_u32(ring + C::STAGES * C::TILE), TK * 128);
      int slot = 0;
      uint32_t use = 0;
      bool ok = true;
      for (int n = 0; n < nk && ok; ++n) {
        if (!(ok = wait(&c->full[1][slot], use & 1, c))) break;
#pragma unroll 1
        for (int w = 0; w < n_tiles; ++w) {
          const uint32_t a = tmem + C::P0 + w * C::PCOLS, b = v_lo + slot * (C::TILE >> 4);
          const uint32_t d = tmem + C::O0 + (SPLIT ? n % 2 : w) * HDP;
          if (SPLIT && n > 1 && !(ok = wait(&c->o_free[n % 2], (n / 2 - 1) & 1, c))) break;
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            if (!(ok = wait(&c->p_full[w][part], n & 1, c))) break;
            fence_after();
            // the small terms first: they lose nothing to a large sum
#pragma unroll
            for (int s = NS - 1; s >= 0; --s)
#pragma unroll
              for (int k = part ? C::FIRST / 16 : 0; k < (part ? TK : C::FIRST) / 16; ++k)
                mma_ts(d, a + s * (TK / 2) + k * 8, b + (k * 2048 >> 4), PV,
                       part + (NS - 1 - s) + k > 0 ? 1 : !SPLIT && n > 0);
          }
          if (!ok) break;
          commit(&c->pv_done[w]);
          if (SPLIT) commit(&c->o_full[n % 2]);
          if (w == n_tiles - 1) commit(&c->empty[1][slot]);
        }
        if (++slot == C::STAGES) slot = 0, ++use;
      }
    }
  }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (*(volatile int*)&c->abort) {
    if (tid == 0) report(p.status, ERR_TIMEOUT);
    // a wait ran out: the products and copies still under way end before the memory goes
    if ((warp == 9 || warp == 11) && elect_one()) {
      commit(&c->drain);
      for (int i = 0; i < 1 << 14 && !mbar_try_wait(&c->drain, 0); ++i) {
      }
    }
    const long long t0 = clock64();
    while (clock64() - t0 < 1 << 20) {
    }
    __syncthreads();
    // the CTA's rows are NaN: alone, or by their part's sum
    if (parts > 1) {
      for (int i = tid; i < C::ROWS; i += TT) ml[i] = make_float2(-INFINITY, NAN);
    } else {
      for (int i = tid; i < n_rows * HD; i += TT) {
        const int r = t.row0 + i / HD;
        store_elem(p.out, ((int64_t)(t.q0 + r / G) * p.n_head + hk * G + r % G) * HD + i % HD, NAN, p.io);
      }
    }
  }
  if (parts > 1) {
    // Each CTA adds the parts of its share of the rows, in order, each warp a run of rows; lane = (row, part) for the
    // statistics.  A wait that ran out anywhere leaves garbage, not a wait here: every CTA comes by.
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    constexpr int E = HD / 32, B = 4;  // rows whose reads are under way at a time
    if (warp < 8) {
      const int rpw = p.tile_rows / (8 * parts), row0 = (part * 8 + warp) * rpw;
      float2 x = make_float2(-INFINITY, 0.f);
      if (lane < rpw * parts && row0 + lane / parts < n_rows) x = *cl.map_shared_rank(&ml[row0 + lane / parts], lane % parts);
      float m = x.x;
      for (int d = 1; d < parts; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      if (m == -INFINITY) m = 0.f;
      float f = exp2_approx(x.x - m);  // 0 for a part without keys of the row
      float l = x.y * f;
      for (int d = 1; d < parts; d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
      for (int i0 = 0; i0 < rpw && row0 + i0 < n_rows; i0 += B) {
        float o[B][E] = {};
        for (int i = 0; i < parts; ++i) {
          float v[B][E];
#pragma unroll
          for (int j = 0; j < B; ++j) {
            const int row = row0 + i0 + j;
            const float* po = cl.map_shared_rank(stage + min(row, n_rows - 1) * HD, i);
            if constexpr (E == 4) {
              *reinterpret_cast<float4*>(v[j]) = *reinterpret_cast<const float4*>(po + (lane ^ (row & 7)) * 4);
            } else {
#pragma unroll
              for (int e = 0; e < E; ++e) v[j][e] = po[(((lane * E + e) / 4) ^ (row & 7)) * 4 + (lane * E + e) % 4];
            }
          }
#pragma unroll
          for (int j = 0; j < B; ++j) {
            const int from = min(i0 + j, rpw - 1) * parts + i;
            const float fi = __shfl_sync(0xffffffffu, f, from);
            if (__shfl_sync(0xffffffffu, x.x, from) == -INFINITY) continue;  // what is there was never written
#pragma unroll
            for (int e = 0; e < E; ++e) o[j][e] = fmaf(v[j][e], fi, o[j][e]);
          }
        }
#pragma unroll
        for (int j = 0; j < B; ++j) {
          const int row = row0 + i0 + j;
          const float lr = __shfl_sync(0xffffffffu, l, min(i0 + j, rpw - 1) * parts);
          if (i0 + j >= rpw || row >= n_rows) continue;  // the same for the warp
          const int r = t.row0 + row, tok = r / G, h = hk * G + r % G;
          const bool sees = t.past + tok >= 0;
          bool finite = true;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            finite = finite && fabsf(o[j][e]) < INFINITY;
            store_elem(p.out, ((int64_t)(t.q0 + tok) * p.n_head + h) * HD + lane * E + e, sees ? o[j][e] / lr : 0.f, p.io);
          }
          if (__any_sync(0xffffffffu, !finite) && sees && (SPLIT || lr < INFINITY)) recompute_row<KV, HD>(p, t, hk, r);
        }
      }
    }
    cl.sync();  // nobody leaves while its shared memory is read
  }
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---- host -----------------------------------------------------------------------------------
template <class KV, int HD, bool SPLIT>
cudaError_t launch_t(WindowAttnParams& p, int kv, int sm_count, cudaStream_t st) {
  using C = Cfg<HD, SPLIT>;
  CUtensorMap km, vm;
  const int64_t rows = (int64_t)p.n_pages * p.n_head_kv * PG;
  cudaError_t e = pool_map(&km, p.k_pages, kv, HD, rows, 1);
  if (e == cudaSuccess) e = pool_map(&vm, p.v_pages, kv, HD, rows, 1);
  if (e != cudaSuccess) return e;
  // Few row tiles: their keys are split over clusters of 2, 4 or 8, as long as all clusters fit the GPU at a time
  // (clusters of 8 with one CTA to an SM: 15 of them were seen to fit 148 SMs) and a CTA keeps four key tiles; row
  // tiles of 128 then, if that still leaves half of the SMs without work.
  const int64_t rows_all = (int64_t)p.n_tok * (p.n_head / p.n_head_kv);
  auto jobs = [&](int rt) { return ((rows_all + rt - 1) / rt + p.n_seq - 1) * p.n_head_kv; };
  int64_t pages = p.max_pages;
  if (p.window > 0) {
    const int64_t seen = ((int64_t)p.window + p.n_sink + p.n_tok) / PG + 3;
    pages = seen < pages ? seen : pages;
  }
  p.tile_rows = C::ROWS;
  p.key_parts = 1;
  while (p.key_parts < 8 && pages >= (int64_t)p.key_parts * 8 * C::PPT &&
         jobs(C::ROWS) * p.key_parts * 2 <= (p.key_parts == 4 ? sm_count * 8 / 10 : p.key_parts == 2 ? sm_count * 9 / 10 : sm_count))
    p.key_parts *= 2;
  if (C::ROWS > TM && jobs(TM) * p.key_parts <= sm_count * 8 / 10) p.tile_rows = TM;
  const int64_t tiles = rows_all / p.tile_rows + p.n_seq;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * p.n_head_kv * p.key_parts));
  cfg.blockDim = dim3(TT);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)p.key_parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const auto launch = [&](auto runs) {
    constexpr auto kernel = prefill_tc_kernel<KV, HD, SPLIT, decltype(runs)::value>;
    const cudaError_t e = allow_smem<kernel>(C::SMEM);
    return e == cudaSuccess ? cudaLaunchKernelEx(&cfg, kernel, p, km, vm) : e;
  };
  if constexpr (!SPLIT)
    if (pages * PG > p.key_parts * MAX_RUN_KEYS<KV>) return launch(std::true_type());
  if constexpr (SPLIT || MAX_RUN_KEYS<KV> > 0) return launch(std::false_type());
  return cudaErrorInvalidValue;  // f16 rows: a table has a page or more
}

template <class KV, bool SPLIT>
cudaError_t launch_hd(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st) {
  if (hd == 32) return launch_t<KV, 32, SPLIT>(p, kv, sm_count, st);
  if (hd == 64) return launch_t<KV, 64, SPLIT>(p, kv, sm_count, st);
  if constexpr (!SPLIT)
    if (hd == 256) return launch_t<KV, 256, false>(p, kv, sm_count, st);
  return launch_t<KV, 128, SPLIT>(p, kv, sm_count, st);
}

}  // namespace

bool prefill_tc_takes(const WindowAttnParams& p, int kv, int hd) {
  const int64_t rows = (int64_t)p.n_pages * p.n_head_kv * PG;
  const int64_t tiles = (int64_t)p.n_tok * (p.n_head / p.n_head_kv) / TM + p.n_seq;
  if ((hd > 128 && p.io == EL_F32) || rows >= 0x7fffffff || tiles * p.n_head_kv * 8 > 0x7fffffff) return false;
  return kv == EL_F16 || (kv == EL_BF16 && p.io == EL_BF16);
}

cudaError_t launch_prefill_tc(WindowAttnParams& p, int kv, int hd, int sm_count, cudaStream_t st) {
  if (kv == EL_BF16) return launch_hd<__nv_bfloat16, false>(p, kv, hd, sm_count, st);
  if (p.io == EL_F32) return launch_hd<__half, true>(p, kv, hd, sm_count, st);
  return launch_hd<__half, false>(p, kv, hd, sm_count, st);
}

}  // namespace sfk
