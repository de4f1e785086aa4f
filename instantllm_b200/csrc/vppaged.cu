// Paged key-value cache operators (include/vpass.h, vp_paged_*): appending rotated rows, attention of
// the newest rows of many requests, attention of prompts.
#include <cuda_runtime.h>

#include <exception>
#include <string>

#include "vp_paged.cuh"
#include "vp_paged_decode.cuh"
#include "vp_paged_host.h"
#include "vp_paged_prefill.cuh"

int pg_tiles(const vp_paged& c, const vp_paged_attn& a, cudaStream_t st);  // vpprefill.cu

using namespace vp;

namespace vp {

// ---- append ----
// One CTA per row, HD / 16 threads per head: each turns two runs of 8 elements (or copies 16), so a
// thread keeps its 8 (cos, sin) pairs in registers over the heads it serves. 16-byte accesses. Bytes
// bound it: each row is read and written once, 452 MB of 32 + 2 x 8 heads of 128 in 75 us (6.05 TB/s,
// 93% of the measured copy), one row in 2.1 us. A call of more than APPEND_STREAM bytes cannot leave
// its rows in L2 for the attention behind it, so it marks them as passing through, in CTAs of two warps
// (88 us with the accesses and CTAs of a small call, which in turn takes 3.4 us for 5 MB against 3.75).
constexpr int APPEND_THREADS = 128;
constexpr int64_t APPEND_STREAM = 64 << 20;

template <typename TI, bool STREAM>
__device__ __forceinline__ void load8(const TI* p, float (&x)[8]) {
  if constexpr (sizeof(TI) == 4) {
    const float4* q = reinterpret_cast<const float4*>(p);
    const float4 a = STREAM ? __ldcs(q) : q[0], b = STREAM ? __ldcs(q + 1) : q[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4* q = reinterpret_cast<const uint4*>(p);
    const uint4 w = STREAM ? __ldcs(q) : *q;
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = PgType<TI>::up(u[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <typename T, bool STREAM>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 w;
  w.x = PgType<T>::down(x[0], x[1]);
  w.y = PgType<T>::down(x[2], x[3]);
  w.z = PgType<T>::down(x[4], x[5]);
  w.w = PgType<T>::down(x[6], x[7]);
  if (STREAM) __stcs(reinterpret_cast<uint4*>(p), w);
  else *reinterpret_cast<uint4*>(p) = w;
}

template <typename TI, typename T, int HD, bool STREAM>
__global__ void __launch_bounds__(APPEND_THREADS) k_paged_append(const vp_paged c, const vp_paged_rows r) {
  constexpr int J = HD / 16;
  pdl_launch_dependents();
  pdl_wait();
  const long long t = blockIdx.x;
  const int j = threadIdx.x % J;
  const int seq = r.seq[t], slot = r.slot[t];
  const int pos = r.rot_dim ? r.pos[t] : 0;
  const bool turns = 16 * j < r.rot_dim;
  const bool pos_ok = !r.rot_dim || (pos >= 0 && pos < r.rope_rows);
  // runs a and b of the head: the two halves of 8 rotation pairs, or 16 elements in a row
  const bool half = turns && !r.interleaved;
  const int da = half ? 8 * j : 16 * j, db = half ? r.rot_dim / 2 + 8 * j : 16 * j + 8;
  float cs[8], sn[8];
  if (turns && pos_ok) {
    const float4* p = reinterpret_cast<const float4*>(r.rope + ((long long)pos * (r.rot_dim / 2) + 8 * j) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = __ldg(p + i);
      cs[2 * i] = f.x, sn[2 * i] = f.y, cs[2 * i + 1] = f.z, sn[2 * i + 1] = f.w;
    }
  }
  bool keep = seq >= 0 && pos_ok;
  long long at = 0;
  if (seq >= 0) {
    bool ok = seq < c.n_seqs && slot >= 0 && slot / c.page_size < c.max_pages;
    int page = -1;
    if (ok) page = c.table[seq * c.table_stride + slot / c.page_size];
    const bool page_ok = page >= 0 && page < c.n_pages;
    if (threadIdx.x == 0 && !(ok && page_ok && pos_ok))
      pg_status(c.status, !ok || !pos_ok ? VP_DEV_ERR_SLOT : VP_DEV_ERR_PAGE);
    keep = keep && ok && page_ok;
    at = (long long)page * c.page_stride + (long long)(slot % c.page_size) * c.slot_stride;
  } else if (threadIdx.x == 0 && !pos_ok) {
    pg_status(c.status, VP_DEV_ERR_SLOT);
  }
  const int heads = r.n_q + 2 * c.n_kv, step = blockDim.x / J;
#pragma unroll 4
  for (int h = threadIdx.x / J; h < heads; h += step) {
    const bool is_q = h < r.n_q, is_v = h >= r.n_q + c.n_kv;
    const int hh = is_q ? h : is_v ? h - r.n_q - c.n_kv : h - r.n_q;
    if (!is_q && !keep) continue;
    const TI* src = is_q ? static_cast<const TI*>(r.q) + t * r.q_row + hh * r.q_head
                  : is_v ? static_cast<const TI*>(r.v) + t * r.v_row + hh * r.v_head
                         : static_cast<const TI*>(r.k) + t * r.k_row + hh * r.k_head;
    T* dst = is_q ? static_cast<T*>(r.q_out) + t * r.out_row + hh * r.out_head
                  : static_cast<T*>(is_v ? c.v : c.k) + at + hh * c.head_stride;
    float a[8], b[8];
    if (is_v) {
      load8<TI, STREAM>(src + 16 * j, a);
      load8<TI, STREAM>(src + 16 * j + 8, b);
      store8<T, STREAM>(dst + 16 * j, a);
      store8<T, STREAM>(dst + 16 * j + 8, b);
      continue;
    }
    load8<TI, STREAM>(src + da, a);
    load8<TI, STREAM>(src + db, b);
    if (!pos_ok) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
    } else if (half) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = a[i], y = b[i];
        a[i] = x * cs[i] - y * sn[i];
        b[i] = y * cs[i] + x * sn[i];
      }
    } else if (turns) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], w = b[2 * i + 1];
        a[2 * i] = x * cs[i] - y * sn[i];
        a[2 * i + 1] = y * cs[i] + x * sn[i];
        b[2 * i] = z * cs[4 + i] - w * sn[4 + i];
        b[2 * i + 1] = w * cs[4 + i] + z * sn[4 + i];
      }
    }
    store8<T, STREAM>(dst + da, a);
    store8<T, STREAM>(dst + db, b);
  }
}

}  // namespace vp

namespace {

template <typename TI, typename T, int HD>
int append_launch(const vp_paged& c, const vp_paged_rows& r, cudaStream_t st) {
  const int heads = r.n_q + 2 * c.n_kv, want = heads * (HD / 16);
  if ((int64_t)r.rows * heads * HD * (sizeof(TI) + sizeof(T)) > APPEND_STREAM)
    return pg_launch("vp_paged_append", k_paged_append<TI, T, HD, true>, r.rows, 64, 0, st, c, r);
  const int threads = want < APPEND_THREADS ? (want + 31) / 32 * 32 : APPEND_THREADS;
  return pg_launch("vp_paged_append", k_paged_append<TI, T, HD, false>, r.rows, threads, 0, st, c, r);
}
template <typename TI, typename T>
int append_launch(const vp_paged& c, const vp_paged_rows& r, cudaStream_t st) {
  return c.head_dim == 64 ? append_launch<TI, T, 64>(c, r, st) : append_launch<TI, T, 128>(c, r, st);
}

template <typename T, int HD>
int decode_launch(const vp_paged& c, const vp_paged_attn& a, cudaStream_t st) {
  using Sh = DcShape<HD>;
  DcParams p;
  p.c = c;
  p.a = a;
  p.group = a.n_q / c.n_kv;
  p.M = p.group * a.rows;
  // a CTA's ring: all of it flies at once (one request of 257 slots: 6.7 us; 7.6 with half as many, which cut its heads, 6.7
  // with twice as many; 64 requests of 130 to 2,048, in even shares of tiles: 12.7, 12.7 and 15.2; 16 of 300: 7.3, 8.4, 7.3)
  p.min_tiles = DC_WARPS * DC_STAGES;
  p.page_shift = __builtin_ctz(c.page_size);
  p.tickets = static_cast<unsigned*>(a.work);
  p.rec = reinterpret_cast<float*>(static_cast<char*>(a.work) + WORK_HEAD);
  CUtensorMap mk, mv;
  if (const int e = pool_maps(c, c.page_size < Sh::TS ? c.page_size : Sh::TS, HD / 64, &mk, &mv)) return e;
  int sms = 0;
  if (const int e = sm_count(&sms)) return e;
  const int tiles = (int)(((long long)c.max_pages * c.page_size + Sh::TS - 1) / Sh::TS);
  const long long pairs = (long long)a.n * c.n_kv, most = pairs * tiles;
  if (most + DC_RUN * pairs > 0x7fffffff) return pfail(VP_ERR_ARG, "more slots than a launch holds");
  return pg_launch("vp_paged_decode", k_paged_decode<T, HD>, (unsigned)(most < sms ? most : sms), DC_THREADS, Sh::SMEM, st, p, mk, mv);
}

}  // namespace

extern "C" {

int vp_paged_append(const vp_paged* c, const vp_paged_rows* r, void* stream) try {
  if (const int e = check_cache(c)) return e;
  if (!r) return pfail(VP_ERR_ARG, "null rows");
  if (r->type != c->type && r->type != VP_T_F32) return pfail(VP_ERR_ARG, "rows must have the cache's type or f32");
  if (r->rows < 0 || r->n_q < 1 || r->n_q > 4096) return pfail(VP_ERR_ARG, "rows or n_q out of range");
  if (r->rot_dim < 0 || r->rot_dim % 16 || r->rot_dim > c->head_dim)
    return pfail(VP_ERR_ARG, "rot_dim must be a multiple of 16, at most head_dim");
  if (r->rot_dim && r->rope_rows < 1) return pfail(VP_ERR_ARG, "empty rotation table");
  if (r->rows == 0) return VP_OK;
  if (!r->q || !r->k || !r->v || !r->q_out || !r->seq || !r->slot) return pfail(VP_ERR_ARG, "null buffer");
  if (r->rot_dim && (!r->pos || !r->rope || off16(r->rope))) return pfail(VP_ERR_ARG, "null or unaligned pos or rope");
  if (off16(r->q) || off16(r->k) || off16(r->v) || off16(r->q_out)) return pfail(VP_ERR_ARG, "rows must be 16-byte aligned");
  const int unit = r->type == VP_T_F32 ? 4 : 8;
  if (bad_strides(r->q_row, r->q_head, unit) || bad_strides(r->k_row, r->k_head, unit) ||
      bad_strides(r->v_row, r->v_head, unit) || bad_strides(r->out_row, r->out_head, 8))
    return pfail(VP_ERR_ARG, "strides of rows must be multiples of 16 bytes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (c->type == VP_T_F16)
    return r->type == VP_T_F32 ? append_launch<float, __half>(*c, *r, st) : append_launch<__half, __half>(*c, *r, st);
  return r->type == VP_T_F32 ? append_launch<float, __nv_bfloat16>(*c, *r, st) : append_launch<__nv_bfloat16, __nv_bfloat16>(*c, *r, st);
} catch (const std::exception&) {
  return VP_ERR_NOMEM;
}

size_t vp_paged_work_bytes(int32_t head_dim, int32_t n_q, int32_t n_kv, int32_t rows) {
  if ((head_dim != 64 && head_dim != 128) || n_kv < 1 || n_q < 1 || n_q % n_kv || n_q / n_kv > PG_MAX_GROUP || rows < 1)
    return 0;
  const long long m = (long long)n_q / n_kv * rows;
  const size_t few = PG_MAX_CTAS * 2 * DC_LEVELS * pg_record(m < DC_ROWS ? (int)m : DC_ROWS, head_dim);
  const size_t many = PF_RECORDS * pg_record(m < PF_ROWS ? (int)m : PF_ROWS, head_dim);
  return WORK_HEAD + (few > many ? few : many) * sizeof(float);
}

int vp_paged_decode(const vp_paged* c, const vp_paged_attn* a, void* stream) try {
  if (const int e = check_attn(c, a, false)) return e;
  if (a->rows > PG_MAX_ROWS) return pfail(VP_ERR_ARG, "a decode call takes 1 to 16 rows per request");
  if (a->n == 0 || a->rows == 0) return VP_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  vp_paged_attn t = in_range(*a);
  t.q_start = nullptr;
  if (a->n_q / c->n_kv * a->rows > DC_ROWS) return pg_tiles(*c, t, st);
  if (c->type == VP_T_F16) return c->head_dim == 64 ? decode_launch<__half, 64>(*c, t, st) : decode_launch<__half, 128>(*c, t, st);
  return c->head_dim == 64 ? decode_launch<__nv_bfloat16, 64>(*c, t, st) : decode_launch<__nv_bfloat16, 128>(*c, t, st);
} catch (const std::exception&) {
  return VP_ERR_NOMEM;
}

}  // extern "C"
