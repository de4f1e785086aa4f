// Host side shared by the paged-cache entry points: errors, tensor maps of the pools, the SM count.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <string>

#include "../../include/vpass.h"

void vp_set_last_error(const std::string& msg);

namespace {

constexpr int PG_MAX_CTAS = 160;       // CTAs of an attention launch, one per SM (148 on a B200)
constexpr size_t WORK_HEAD = 1024;     // counters at the head of the work buffer
static_assert(PG_MAX_CTAS * sizeof(unsigned) <= WORK_HEAD, "counters");

int pfail(int code, const char* msg) {
  vp_set_last_error(msg);
  return code;
}
int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return VP_OK;
  vp_set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
  return VP_ERR_CUDA;
}

// SMs of the current device, at most PG_MAX_CTAS.
int sm_count(int* out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return pfail(VP_ERR_CUDA, cudaGetErrorString(e));
  if (*out > PG_MAX_CTAS) *out = PG_MAX_CTAS;
  return VP_OK;
}

// Maps of both pools as [page][head][slot][element] with boxes of 64 elements x `rows` slots of one
// page and head, 128-byte swizzle, zeros outside.
int pool_maps(const vp_paged& c, int rows, CUtensorMap* mk, CUtensorMap* mv) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess) f = nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  if (!encode) return pfail(VP_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.n_kv, (cuuint64_t)c.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)c.slot_stride * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = c.type == VP_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int i = 0; i < 2; ++i)
    if (encode(i ? mv : mk, type, 4, i ? c.v : c.k, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return pfail(VP_ERR_ARG, "the pools' strides or extents cannot be mapped");
  return VP_OK;
}

}  // namespace
