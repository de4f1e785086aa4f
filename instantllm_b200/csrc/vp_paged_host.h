// Host side shared by the paged-cache entry points: errors, tensor maps of the pools, the SM count.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <string>
#include <utility>

#include "vp_paged.cuh"

void vp_set_last_error(const std::string& msg);

namespace {

using namespace vp;

constexpr int PG_MAX_CTAS = 160;       // CTAs of an attention launch, one per SM (148 on a B200)
constexpr size_t WORK_HEAD = VP_PAGED_WORK_ZEROED;  // counters at the head of the work buffer

int pfail(int code, const char* msg) {
  vp_set_last_error(msg);
  return code;
}
bool off16(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

int check_cache(const vp_paged* c) {
  if (!c) return pfail(VP_ERR_ARG, "null cache");
  if (c->type != VP_T_F16 && c->type != VP_T_BF16) return pfail(VP_ERR_ARG, "the cache's type must be f16 or bf16");
  if (c->head_dim != 64 && c->head_dim != 128) return pfail(VP_ERR_ARG, "head_dim must be 64 or 128");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return pfail(VP_ERR_ARG, "page_size must be 16, 32, 64, 128 or 256");
  if (c->n_kv < 1 || c->n_kv > 4096) return pfail(VP_ERR_ARG, "n_kv out of range");
  if (c->n_pages < 1 || c->n_seqs < 0 || c->max_pages < 1 || (long long)c->max_pages * c->page_size > (1 << 30))
    return pfail(VP_ERR_ARG, "n_pages, n_seqs or max_pages out of range");
  if (!c->k || !c->v || !c->table) return pfail(VP_ERR_ARG, "null pool or table");
  if (off16(c->k) || off16(c->v)) return pfail(VP_ERR_ARG, "pools must be 16-byte aligned");
  const int64_t s[3] = {c->page_stride, c->head_stride, c->slot_stride};
  for (int64_t x : s)
    if (x <= 0 || x % 8 || x >= (1ll << 39)) return pfail(VP_ERR_ARG, "pool strides must be positive multiples of 8 elements below 2^39");
  if (c->table_stride < c->max_pages) return pfail(VP_ERR_ARG, "table_stride below max_pages");
  return VP_OK;
}

bool bad_strides(int64_t a, int64_t b, int unit) { return a % unit || b % unit; }

// prompts: q_start names the rows, and what only a decode call has (request strides, masks) is not looked at
int check_attn(const vp_paged* c, const vp_paged_attn* a, bool prompts) {
  if (const int e = check_cache(c)) return e;
  if (!a) return pfail(VP_ERR_ARG, "null arguments");
  if (a->n < 0 || a->rows < 0 || a->n > (1 << 24)) return pfail(VP_ERR_ARG, "n or rows out of range");
  if (a->n_q < 1 || a->n_q % c->n_kv) return pfail(VP_ERR_ARG, "n_q must be a multiple of n_kv");
  if (a->n_q / c->n_kv > PG_MAX_GROUP) return pfail(VP_ERR_ARG, "more than 64 query heads per cache head");
  if (a->window < 0 || a->sinks < 0) return pfail(VP_ERR_ARG, "window and sinks must not be negative");
  if (!(a->scale > 0.f && a->scale < 3e38f)) return pfail(VP_ERR_ARG, "scale must be positive and finite");
  if (a->n == 0 || a->rows == 0) return VP_OK;
  if (!a->q || !a->out || !a->lens) return pfail(VP_ERR_ARG, "null q, out or lens");
  if (off16(a->q) || off16(a->out)) return pfail(VP_ERR_ARG, "q and out must be 16-byte aligned");
  if (bad_strides(a->q_row, a->q_head, 8) || bad_strides(a->out_row, a->out_head, 8) ||
      (!prompts && bad_strides(a->q_seq, a->out_seq, 8)))
    return pfail(VP_ERR_ARG, "strides of q and out must be multiples of 8 elements");
  if (!a->work || (reinterpret_cast<uintptr_t>(a->work) & 255)) return pfail(VP_ERR_ARG, "work must be 256-byte aligned");
  if (a->work_bytes < vp_paged_work_bytes(c->head_dim, a->n_q, c->n_kv, a->rows))
    return pfail(VP_ERR_ARG, "work is smaller than vp_paged_work_bytes");
  return VP_OK;
}

// A window past every position is none, and sinks past every position are all: the kernels subtract positions from them.
vp_paged_attn in_range(const vp_paged_attn& a) {
  vp_paged_attn t = a;
  if (t.window > (1 << 30)) t.window = 0;
  if (t.sinks > (1 << 30)) t.sinks = 1 << 30;
  return t;
}

// Launches a kernel whose prologue may run while the kernel before it in the stream ends
// (griddepcontrol.wait in the kernel stands before its first access to global memory).
template <typename... P, typename... A>
int pg_launch(const char* what, void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, A&&... args) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return pfail(VP_ERR_CUDA, cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
  if (e == cudaSuccess) return VP_OK;
  cudaGetLastError();
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

// Maps of both pools as [page][head][panel of 64 elements][slot][element] with boxes of `panels` panels
// x `rows` slots of one page and head, 128-byte swizzle, zeros outside.
int pool_maps(const vp_paged& c, int rows, int panels, CUtensorMap* mk, CUtensorMap* mv) {
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
  const cuuint64_t dims[5] = {64, (cuuint64_t)c.page_size, (cuuint64_t)c.head_dim / 64, (cuuint64_t)c.n_kv, (cuuint64_t)c.n_pages};
  const cuuint64_t strides[4] = {(cuuint64_t)c.slot_stride * 2, 128, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
  const cuuint32_t box[5] = {64, (cuuint32_t)rows, (cuuint32_t)panels, 1, 1}, step[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType type = c.type == VP_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int i = 0; i < 2; ++i)
    if (encode(i ? mv : mk, type, 5, i ? c.v : c.k, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return pfail(VP_ERR_ARG, "the pools' strides or extents cannot be mapped");
  return VP_OK;
}

}  // namespace
