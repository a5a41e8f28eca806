// asmllm_b200/csrc/tensor_map.cuh -- tensor maps of the paged key-value view
// and the tensor copies that use them.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <stdint.h>

#include <mutex>

#include "serving.cuh"

namespace asmllm {

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// A 16-bit array [n3][n2][n1][n0] (strides in elements, the innermost dense)
// copied in boxes of 64 x rows with the 128-byte swizzle; what is outside
// reads as zeros.
inline bool encode_4d(CUtensorMap* map, int dtype, const void* base, uint64_t n0, uint64_t n1, uint64_t n2, uint64_t n3,
                      uint64_t s1, uint64_t s2, uint64_t s3, uint32_t box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encode_fn();
  if (!encode) return false;
  const cuuint64_t dim[4] = {n0, n1, n2, n3};
  const cuuint64_t stride[3] = {s1 * 2, s2 * 2, s3 * 2};
  const cuuint32_t box[4] = {64u, box_rows, 1u, 1u}, step[4] = {1u, 1u, 1u, 1u};
  return encode(map, dtype == kDtF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                const_cast<void*>(base), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Keys or values: (value, offset in page, KV head, page).
inline bool encode_kv_map(CUtensorMap* map, const KvArgs& kv, const void* base, int box_rows) {
  return encode_4d(map, kv.dtype, base, (uint64_t)kv.head_dim, (uint64_t)kv.page_size, (uint64_t)kv.n_kv,
                   (uint64_t)kv.n_pages, (uint64_t)kv.token_stride, (uint64_t)kv.head_stride, (uint64_t)kv.page_stride,
                   (uint32_t)box_rows);
}

#ifdef __CUDACC__
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3,
                                            uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(mbar)
      : "memory");
}
#endif

}  // namespace asmllm
