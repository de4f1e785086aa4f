// Attention of prompts over the paged cache (include/vpass.h, vp_paged_prefill).
#include <exception>

#include "vp_paged_host.h"
#include "vp_paged_prefill.cuh"

namespace {

template <typename T, int HD>
int prefill_launch(const vp_paged& c, const vp_paged_attn& a, cudaStream_t st) {
  using Sh = PfShape<HD>;
  PfParams p;
  p.c = c;
  p.a = a;
  p.group = a.n_q / c.n_kv;
  CUtensorMap mk, mv;
  if (const int e = pool_maps(c, c.page_size < PF_TS ? c.page_size : PF_TS, &mk, &mv)) return e;
  // every request's last block may be short
  const long long blocks = ((long long)a.rows * p.group + PF_ROWS - 1) / PF_ROWS + a.n;
  if (blocks * c.n_kv > 0x7fffffffll) return pfail(VP_ERR_ARG, "more rows than a launch holds");
  const cudaError_t e = cudaFuncSetAttribute(k_paged_prefill<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Sh::SMEM);
  if (e != cudaSuccess) return pfail(VP_ERR_CUDA, cudaGetErrorString(e));
  k_paged_prefill<T, HD><<<(unsigned)(blocks * c.n_kv), PF_THREADS, Sh::SMEM, st>>>(p, mk, mv);
  return launched("vp_paged_prefill");
}

}  // namespace

extern "C" int vp_paged_prefill(const vp_paged* c, const vp_paged_attn* a, void* stream) try {
  if (const int e = check_attn(c, a)) return e;
  if (a->n == 0 || a->rows == 0) return VP_OK;
  if (!a->q_start) return pfail(VP_ERR_ARG, "null q_start");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (c->type == VP_T_F16) return c->head_dim == 64 ? prefill_launch<__half, 64>(*c, *a, st) : prefill_launch<__half, 128>(*c, *a, st);
  return c->head_dim == 64 ? prefill_launch<__nv_bfloat16, 64>(*c, *a, st) : prefill_launch<__nv_bfloat16, 128>(*c, *a, st);
} catch (const std::exception&) {
  return VP_ERR_NOMEM;
}
