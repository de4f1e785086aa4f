// Shared parts of the paged-cache operators (include/vpass.h, vp_paged_*): lengths of requests, copies, waits,
// element conversions.
#pragma once
#include <cuda.h>
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

// A request's length, clipped to what its row of the table holds; zero for a request outside the table.
__device__ __forceinline__ int pg_len(const vp_paged& c, const int32_t* seqs, const int32_t* lens, int i) {
  const int s = seqs ? seqs[i] : i, len = lens[i];
  const long long cap = (long long)c.max_pages * c.page_size;
  const bool there = s >= 0 && s < c.n_seqs && len >= 0;
  if (!there || len > cap) pg_status(c.status, VP_DEV_ERR_SLOT);
  return !there ? 0 : len > cap ? (int)cap : len;
}

// One box of a pool into shared memory: the map's box of slots from `slot` of a page, in panels of 64
// elements, 128 bytes a slot with the 128-byte swizzle: the 16-byte piece i of line l lies at piece
// i ^ (l & 7). pg_box: one panel of the box; pg_box5: all its panels. A page outside the pool fills zeros.
__device__ __forceinline__ void pg_box(void* dst, const CUtensorMap* map, int panel, int slot, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(slot), "r"(panel), "r"(head), "r"(page)
      : "memory");
}
__device__ __forceinline__ void pg_box5(void* dst, const CUtensorMap* map, int slot, int head, int page, uint64_t* bar) {
  pg_box(dst, map, 0, slot, head, page, bar);
}
__device__ __forceinline__ void pg_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// 16 bytes global -> shared without a register; pg_cp_arrive: the barrier counts this thread once its
// copies so far are there.
__device__ __forceinline__ void pg_cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void pg_cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pg_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Wait of a whole warp that ends early once `dead` (shared memory) is set; false if the phase is not complete. The lanes
// leave on a vote, as in mbar_wait_warp.
__device__ __forceinline__ bool pg_wait(uint64_t* bar, uint32_t parity, const int* dead) {
  const unsigned long long t0 = globaltimer();
  for (uint32_t i = 0; i < (1u << 26); ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((i & 63) == 0 && __any_sync(0xffffffffu, *(const volatile int*)dead || globaltimer() - t0 > WAIT_NS)) return false;
  }
  return false;
}
__device__ __forceinline__ float pg_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct PgType;
template <>
struct PgType<__half> {
  static constexpr bool BF16 = false;
  static __device__ __forceinline__ float2 up(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ uint32_t down(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct PgType<__nv_bfloat16> {
  static constexpr bool BF16 = true;
  static __device__ __forceinline__ float2 up(uint32_t w) {
    return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
  }
  static __device__ __forceinline__ uint32_t down(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void pg_ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void pg_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

}  // namespace vp
