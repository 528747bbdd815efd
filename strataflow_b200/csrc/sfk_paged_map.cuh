// sfk_paged_map.cuh -- tensor maps of a 16-bit page pool, and the copy of a page.
//
// The pool [n_pages][Hkv][16][hd] is a matrix of n_pages * Hkv * 16 rows of hd
// elements; one page of one head is 16 rows.  The map sees it as [64-dim block]
// [row][64 dims], so that a copy takes whole 128-byte rows of one or more blocks
// into the 128-byte swizzle.  hd 32: the block's upper half lies outside the map
// and arrives as zeros, as does a page whose first row lies past the last.
#pragma once
#include <cuda.h>

#include "sfk_paged.cuh"

namespace sfk {

#ifdef __CUDACC__
// a page's rows from row y of the map, blocks from `block` on, to shared memory [block][16][128 B]
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, int y, uint64_t* bar, int block = 0) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(0), "r"(y), "r"(block), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
#endif

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}
// The map of a pool of `rows` rows; a copy takes 16 rows of `blocks` 64-dim blocks.
inline cudaError_t pool_map(CUtensorMap* m, const void* pool, int kv, int hd, int64_t rows, int blocks) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)(hd < 64 ? hd : 64), (cuuint64_t)rows, (cuuint64_t)((hd + 63) / 64)};
  const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, 128};
  const cuuint32_t box[3] = {64, PG, (cuuint32_t)blocks}, step[3] = {1, 1, 1};
  return fn(m, kv == EL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
            const_cast<void*>(pool), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? cudaSuccess
             : cudaErrorInvalidValue;
}

}  // namespace sfk
