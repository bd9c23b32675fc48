// Maps of arrays for the tensor copies.
#include <atomic>

#include "rows.cuh"
#include "tensor.cuh"

namespace plx {
namespace {

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                            const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                            CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                            CUtensorMapFloatOOBfill);
// The driver's encoder, found once.
int encoder(Encode* out) {
  static std::atomic<void*> found{nullptr};
  void* f = found.load(std::memory_order_acquire);
  if (!f) {
    cudaDriverEntryPointQueryResult q;
    PLX_TRY_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q));
    if (q != cudaDriverEntryPointSuccess || !f)
      return set_error(PLX_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    found.store(f, std::memory_order_release);
  }
  *out = reinterpret_cast<Encode>(f);
  return PLX_OK;
}

}  // namespace

int tensor_map(CUtensorMap* map, int dtype, const void* p, uint64_t inner, uint64_t outer,
               int64_t ld, uint32_t box_inner, uint32_t box_outer, bool swizzle) {
  Encode encode = nullptr;
  if (int rc = encoder(&encode)) return rc;
  const cuuint64_t dims[2] = {inner, outer};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * dtype_bytes(dtype)};
  const cuuint32_t box[2] = {box_inner, box_outer}, elem[2] = {1, 1};
  const CUtensorMapDataType type = dtype == PLX_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == PLX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult e = encode(map, type, 2, const_cast<void*>(p), dims, strides, box, elem,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (e != CUDA_SUCCESS)
    return set_error(PLX_ERR_CUDA, "cuTensorMapEncodeTiled: error %d for %llu x %llu values, "
                     "stride %lld", (int)e, (unsigned long long)outer, (unsigned long long)inner,
                     (long long)ld);
  return PLX_OK;
}

}  // namespace plx
