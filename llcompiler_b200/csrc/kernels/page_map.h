// Tensor maps of a paged cache: host side of the TMA loads in the paged-attention kernels.
#pragma once
#include "paged_attention.cuh"
#include "tensor_map.h"

namespace llc {

// Cache [pages, page_size, kv_heads, d] as a 4-D map (d, slot, head, page); box = 64 elements x boxRows slots, 128-byte swizzle.  A
// load whose page coordinate is num_pages lies outside the tensor and reads as zeros.
inline bool makePageMap(CUtensorMap* map, const void* base, int dtype, const PagedArgs& p, long long sPage, long long sSlot, long long sHead, int boxRows) {
  EncodeTiledFn enc = encodeTiled();
  if (!enc) return false;
  cuuint64_t dims[4] = {(cuuint64_t)p.d, (cuuint64_t)p.pageSize, (cuuint64_t)p.kvHeads, (cuuint64_t)p.numPages};
  cuuint64_t strides[3] = {(cuuint64_t)sSlot * 2, (cuuint64_t)sHead * 2, (cuuint64_t)sPage * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)boxRows, 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(map, dtype == LLC_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace llc
