// Host side: tensor maps of K-major operands.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "mg_common.h"

namespace mg {

inline int get_encoder(PFN_cuTensorMapEncodeTiled_v12000* out) {
  static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
  static std::once_flag g_encode_once;
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  *out = g_encode;
  return g_encode ? MG_OK : MG_ERR_CUDA;
}

// 2-D K-major operand: `kdim` elements of type `dt` per row, `rows` rows, `pitch` bytes.
inline int make_map(CUtensorMap* m, CUtensorMapDataType dt, const void* ptr, uint64_t kdim, uint64_t rows,
                    uint64_t pitch, uint32_t box_k, uint32_t box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc;
  if (get_encoder(&enc) != MG_OK) return MG_ERR_CUDA;
  cuuint64_t dims[2] = {kdim, rows};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {box_k, box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(m, dt, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    mg::note_cuda_error(cudaErrorInvalidValue);
    return MG_ERR_CUDA;
  }
  return MG_OK;
}

}  // namespace mg
