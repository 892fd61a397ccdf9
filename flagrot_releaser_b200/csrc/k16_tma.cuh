// Tensor maps over the 16-bit pool and the host lookup of the driver's encoder.
//
// The pool is mapped as [D / 64][rows][64] with rows = num_pages * Hkv * 2 * page, so that one copy of a box of 64 x BR x D / 64
// elements brings BR whole rows as D / 64 tiles of BR rows x 128 bytes, each in the 128-byte swizzle (16-byte piece c of row r
// at piece c ^ (r & 7)): what ldmatrix reads without bank conflicts and tcgen05.mma takes as an operand.  A box that starts at
// row `rows` lies outside and arrives as zeros.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "fr_tc5.cuh"

namespace k16 {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// box of 64 elements x `mid` x `outer`; dims and byte strides of the two outer axes
inline cudaError_t encode3(CUtensorMap* m, int dtype, const void* base, uint64_t d1, uint64_t s1, uint64_t d2, uint64_t s2,
                           uint32_t mid, uint32_t outer) {
  EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {64, d1, d2}, strides[2] = {s1, s2};
  const cuuint32_t box[3] = {64, mid, outer}, es[3] = {1, 1, 1};
  const CUresult r = fn(m, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
                        dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
// box of 64 elements x b1 x b2 x 1
inline cudaError_t encode4(CUtensorMap* m, int dtype, const void* base, uint64_t d1, uint64_t s1, uint64_t d2, uint64_t s2, uint64_t d3,
                           uint64_t s3, uint32_t b1, uint32_t b2) {
  EncodeFn fn = encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[4] = {64, d1, d2, d3}, strides[3] = {s1, s2, s3};
  const cuuint32_t box[4] = {64, b1, b2, 1}, es[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base),
                        dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
inline cudaError_t pool_map(CUtensorMap* m, int dtype, const void* pool, long long rows, int D, uint32_t box_rows) {
  return encode3(m, dtype, pool, static_cast<uint64_t>(rows), static_cast<uint64_t>(D) * 2, static_cast<uint64_t>(D / 64), 128, box_rows,
                 static_cast<uint32_t>(D / 64));
}

FR_DEVI void tma3(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint32_t mbar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
               "l"(m), "r"(x), "r"(y), "r"(z), "r"(mbar)
               : "memory");
}
FR_DEVI void tma4(uint32_t dst, const CUtensorMap* m, int x, int y, int z, int w, uint32_t mbar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(dst),
               "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(mbar)
               : "memory");
}
FR_DEVI void tma_prefetch_map(const CUtensorMap* m) { asm volatile("prefetch.tensormap [%0];\n" ::"l"(m) : "memory"); }

}  // namespace k16
