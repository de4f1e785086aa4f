// Shared parts of the paged-cache operators (include/vpass.h, vp_paged_*): device views of the
// cache and of a call, visibility of slots, element conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "vp_common.cuh"

namespace vp {

constexpr int PG_MAX_ROWS = VP_MAX_ROWS;  // new rows per request of a decode call
constexpr int PG_MAX_GROUP = 64;          // query heads per cache head

__device__ __forceinline__ void pg_status(int32_t* status, int bits) {
  if (status) atomicOr(status, bits);
}

// A request's row of the table and its length, clipped to what the table holds.
struct PgSeq {
  const int32_t* pages;
  int len;
};
__device__ __forceinline__ PgSeq pg_seq(const vp_paged& c, const int32_t* seqs, const int32_t* lens, int i) {
  const int s = seqs ? seqs[i] : i;
  int len = lens[i];
  const long long cap = (long long)c.max_pages * c.page_size;
  if (s < 0 || s >= c.n_seqs || len < 0 || len > cap) {
    pg_status(c.status, VP_DEV_ERR_SLOT);
    len = s < 0 || s >= c.n_seqs || len < 0 ? 0 : (int)cap;
  }
  return {c.table + (s < 0 || s >= c.n_seqs ? 0 : (long long)s * c.table_stride), len};
}

// Whether a row of a decode call sees a slot. base: slots before the new rows; bits: the row's
// mask; anc: masks of all new rows (for their positions when a window is set).
__device__ __forceinline__ bool pg_sees(int slot, int len, int base, uint32_t bits, const uint32_t* anc, int window,
                                        int sinks) {
  if (slot >= len) return false;
  int place = slot;
  if (slot >= base) {
    if (!((bits >> (slot - base)) & 1)) return false;
    if (window) place = base + __popc(anc[slot - base]) - 1;
  }
  return !window || base + __popc(bits) - 1 - place < window || place < sinks;
}

template <typename T>
struct PgType;
template <>
struct PgType<__half> {
  using Pair = __half2;
  static __device__ __forceinline__ float2 up(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ uint32_t down(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct PgType<__nv_bfloat16> {
  using Pair = __nv_bfloat162;
  static __device__ __forceinline__ float2 up(uint32_t w) {
    return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  }
  static __device__ __forceinline__ uint32_t down(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

}  // namespace vp
