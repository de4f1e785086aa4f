// Attention of prompts over the paged cache (include/vpass.h, vp_paged_prefill).
#include <exception>

#include "vp_paged_host.h"
#include "vp_paged_prefill.cuh"

namespace {

static_assert(PF_RECORDS >= 4 * PG_MAX_CTAS && (4 * PF_RECORDS + 2) * sizeof(unsigned) <= WORK_HEAD, "records and their counters");

template <typename T, int HD>
int tiles_launch(const vp_paged& c, const vp_paged_attn& a, cudaStream_t st) {
  using Sh = PfShape<HD>;
  PfParams p;
  p.c = c;
  p.a = a;
  p.group = a.n_q / c.n_kv;
  const long long rows = (long long)a.rows * p.group;  // packed, of a request (tree) or of all
  if (rows > 0x7fffff00ll) return pfail(VP_ERR_ARG, "more rows than a launch holds");
  if (const int e = sm_count(&p.sms)) return e;
  // at most this many blocks of 256 rows: every request's last block may be short. Where they leave half of
  // the SMs idle, 128 rows make a block: twice the CTAs, each with one row tile (a prompt of 1,024 rows
  // of 14 query and 2 key-value heads: 21.8 us with 256, 16.3 with 128).
  auto blocks_of = [&](int of) { return (a.q_start ? rows / of + a.n : (rows + of - 1) / of * a.n) * c.n_kv; };
  p.rows = blocks_of(PF_ROWS) * 2 <= p.sms ? PF_ROWS / 2 : PF_ROWS;
  p.block_rows = rows < p.rows ? (int)rows : p.rows;
  p.tickets = static_cast<unsigned*>(a.work);
  p.rec = reinterpret_cast<float*>(static_cast<char*>(a.work) + WORK_HEAD);
  // the warpgroups trade registers: what the softmax takes on must have been launched with
  static const int regs = [] {
    cudaFuncAttributes f{};
    return cudaFuncGetAttributes(&f, k_paged_tiles<T, HD>) == cudaSuccess ? f.numRegs : 0;
  }();
  if (regs * PF_THREADS < 2 * 128 * PF_SOFTMAX_REGS + 128 * PF_OTHER_REGS) return pfail(VP_ERR_CUDA, "the kernel was built with too few registers");
  CUtensorMap mk, mv;
  if (const int e = pool_maps(c, c.page_size < PF_TS ? c.page_size : PF_TS, 1, &mk, &mv)) return e;
  // at most this many pieces: the cuts add two CTAs per SM at most, or as many as the table's longest request
  // allows
  const long long pairs = blocks_of(p.rows), tiles = ((long long)c.max_pages * c.page_size + PF_TS - 1) / PF_TS;
  const long long cuts = (tiles + PF_LEAST - 1) / PF_LEAST - 1;
  p.cuts = 2 * tiles > 3 * PF_LEAST;
  const long long more = !p.cuts ? 0 : pairs * cuts < 2 * p.sms ? pairs * cuts : 2 * p.sms;
  if (pairs + more >= 0x7fffffffll) return pfail(VP_ERR_ARG, "more rows than a launch holds");
  p.most = (int)(pairs + more);
  return pg_launch(a.q_start ? "vp_paged_prefill" : "vp_paged_decode", k_paged_tiles<T, HD>, p.most < p.sms ? p.most : p.sms, PF_THREADS,
                   Sh::SMEM, st, p, mk, mv);
}

}  // namespace

// Prompts (q_start set), or the new rows of vp_paged_decode.
int pg_tiles(const vp_paged& c, const vp_paged_attn& a, cudaStream_t st) {
  if (c.type == VP_T_F16) return c.head_dim == 64 ? tiles_launch<__half, 64>(c, a, st) : tiles_launch<__half, 128>(c, a, st);
  return c.head_dim == 64 ? tiles_launch<__nv_bfloat16, 64>(c, a, st) : tiles_launch<__nv_bfloat16, 128>(c, a, st);
}

extern "C" int vp_paged_prefill(const vp_paged* c, const vp_paged_attn* a, void* stream) try {
  if (const int e = check_attn(c, a, true)) return e;
  if (a->n == 0 || a->rows == 0) return VP_OK;
  if (!a->q_start) return pfail(VP_ERR_ARG, "null q_start");
  vp_paged_attn t = in_range(*a);
  t.q_seq = t.out_seq = 0;
  t.mask = nullptr;
  return pg_tiles(*c, t, static_cast<cudaStream_t>(stream));
} catch (const std::exception&) {
  return VP_ERR_NOMEM;
}
