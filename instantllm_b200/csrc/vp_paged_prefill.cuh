// Attention of prompt rows over the paged cache (vp_paged_prefill).
//
// Mathematics as in vp_paged_decode.cuh: a running maximum m and sum l over tiles of 128 slots. The
// maximum that the weights are taken against only moves when the tile's is more than 2^8 above it
// (weights then reach 2^8 at most, and out = o / l does not depend on it), so o is rarely rescaled.
//
// Bound: the tensor cores at head_dim 128, the exponentials (16 a clock and SM against 4,096 products)
// at 64. The query rows of one cache head are packed as row G + g, 256 of them to a CTA as two
// tiles of 128, so K and V are read once for 256 rows and the heads of a group share them. Tensor
// memory holds S of both tiles (128 columns each, the weights P written over them as pairs) and both
// o (head_dim columns each). One warp brings K and V tiles (TMA boxes of one page each), one thread
// issues the products, and two warpgroups, one tile each and one row a thread, do the softmax: while
// one of them works on its tile, the tensor cores work on the other's.
#pragma once
#include "vp_paged.cuh"

namespace vp {

constexpr int PF_TS = 128;                 // slots per tile
constexpr int PF_ROWS = 256;               // packed query rows per CTA
constexpr int PF_THREADS = 384;            // two softmax warpgroups, then one: producer, issuer, two idle warps
constexpr int PF_PRODUCER = 8, PF_ISSUER = 9;
constexpr uint32_t PF_TMEM = 512;          // columns
constexpr float PF_SLACK = 8.f;            // log2 of the largest weight

template <int HD>
struct PfShape {
  static constexpr int PANELS = HD / 64;                        // 128-byte wide columns of a tile
  static constexpr int TILE = PF_TS * HD * 2;                   // bytes of a K, V or Q tile
  static constexpr int SLOTS = HD == 64 ? 8 : 5;                // ring of K and V tiles
  static constexpr size_t SMEM = 1024 + 2 * TILE + (size_t)SLOTS * TILE;
};

struct PfParams {
  vp_paged c;
  vp_paged_attn a;
  int group;
};

__device__ __forceinline__ uint64_t pf_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  // shared-memory operand, 128-byte swizzle: address and offsets in 16-byte units
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)((stride >> 4) & 0x3fff) << 32 |
         1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void pf_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void pf_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void pf_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pf_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pf_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pf_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// The registers of loads issued before are valid from here on (the empty statements keep their uses behind).
template <int N>
__device__ __forceinline__ void pf_loaded(uint32_t (&r)[N]) {
  pf_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void pf_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the warp's 32 lanes, one lane a thread.
__device__ __forceinline__ void pf_ld32(uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void pf_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}

// Slots that a run of rows at positions [p0, p1] sees, as tiles: [0, ns) hold sinks, then [ws, end).
struct PfSpan {
  int ns, ws, tiles;
  __device__ __forceinline__ int at(int t) const { return t < ns ? t : ws + t - ns; }
  // tiles of this list whose first slot is at or below p
  __device__ __forceinline__ int upto(int p) const {
    if (p < 0) return 0;
    const int end = p / PF_TS + 1;
    return min(tiles, end <= ns ? end : ns + max(0, end - ws));
  }
};
__device__ __forceinline__ PfSpan pf_span(int p0, int p1, int window, int sinks) {
  PfSpan s;
  const int end = p1 < 0 ? 0 : p1 / PF_TS + 1, lo = window ? max(0, p0 - window + 1) : 0;
  s.ns = window ? min((min(sinks, p1 + 1) + PF_TS - 1) / PF_TS, end) : 0;
  s.ws = lo / PF_TS;
  if (s.ws <= s.ns) s.ws = s.ns = 0;
  s.tiles = s.ns + end - s.ws;
  return s;
}

template <typename T, int HD>
__global__ void __launch_bounds__(PF_THREADS, 1)
    k_paged_prefill(const __grid_constant__ PfParams p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
  using Sh = PfShape<HD>;
  constexpr int TILE = Sh::TILE, SLOTS = Sh::SLOTS, PANELS = Sh::PANELS, PANEL = PF_TS * 128;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* qs = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* ring = qs + 2 * TILE;
  __shared__ uint64_t kv_full[SLOTS], kv_empty[SLOTS], s_full[2], p_full[2], q_full, edge, drained;
  __shared__ uint32_t tmem_base;
  __shared__ int warp_sums[PF_THREADS / 32], my_seq, my_tile, dead;

  const vp_paged& c = p.c;
  const vp_paged_attn& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(&q_full, 8);
    mbar_init(&edge, 1);
    mbar_init(&drained, 1);
    fence_barrier_init();
    dead = 0;
    my_seq = -1;
  }
  // which request and block of rows: blocks are counted over the requests, the last ones (with the
  // most slots to see) first
  const int run = (a.n + PF_THREADS - 1) / PF_THREADS, i0 = min(a.n, tid * run), i1 = min(a.n, i0 + run);
  auto new_rows = [&](int i) {
    const int x = min(max(a.q_start[i], 0), a.rows), y = min(max(a.q_start[i + 1], 0), a.rows);
    return max(0, y - x);
  };
  auto blocks_of = [&](int i) { return (int)(((long long)new_rows(i) * p.group + PF_ROWS - 1) / PF_ROWS); };
  int mine = 0;
  for (int i = i0; i < i1; ++i) mine += blocks_of(i);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl;
  cta_sync();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < PF_THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  const int block = total - 1 - (int)(blockIdx.x / c.n_kv), head = blockIdx.x % c.n_kv;
  if (block < 0) return;
  int at = before + incl - mine;
  if (at <= block && block < at + mine) {
    for (int i = i0; i < i1; ++i) {
      const int n = blocks_of(i);
      if (block < at + n) {
        my_seq = i;
        my_tile = block - at;
        break;
      }
      at += n;
    }
  }
  __syncwarp();
  if (warp == PF_ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(PF_TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pf_fence_before();
  cta_sync();
  pf_fence_after();
  const uint32_t tmem = tmem_base;
  const int seq = my_seq, f0 = my_tile * PF_ROWS, n_new = new_rows(seq), first = min(max(a.q_start[seq], 0), a.rows);
  const PgSeq sq = pg_seq(c, a.seqs, a.lens, seq);
  const int base = sq.len - n_new;
  const int f_end = (int)min((long long)n_new * p.group, (long long)f0 + PF_ROWS);
  const int p_lo = base + f0 / p.group, p_hi = base + (f_end - 1) / p.group;
  const PfSpan sp = pf_span(p_lo, p_hi, a.window, a.sinks);
  // tiles of the two row tiles: the first ends earlier
  const int p_hi0 = base + (min(f_end, f0 + 128) - 1) / p.group;
  const int n0 = sp.upto(p_hi0), n1 = f_end > f0 + 128 ? sp.tiles : 0, n_max = max(n0, n1);

  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {  // whole warp
    __syncwarp();
    if (*(volatile int*)&dead) return;
    if (!mbar_wait_warp(bar, parity)) {
      pg_status(c.status, VP_DEV_ERR_TIMEOUT);
      *(volatile int*)&dead = 1;
    }
    __syncwarp();
  };
  auto wait_one = [&](uint64_t* bar, uint32_t parity) {  // one thread
    if (*(volatile int*)&dead) return;
    if (!mbar_wait_bounded(bar, parity)) {
      pg_status(c.status, VP_DEV_ERR_TIMEOUT);
      *(volatile int*)&dead = 1;
    }
  };

  if (warp < 8) {
    // ---- softmax: warpgroup i has row tile i, a thread row f ----
    const int i = warp >> 2, row = tid & 127, f = f0 + tid;
    const int n_t = i ? n1 : n0;
    const bool valid = f < f_end;
    const int qrow = f / p.group, h = head * p.group + f % p.group;
    {
      const T* q = static_cast<const T*>(a.q) + (long long)(first + qrow) * a.q_row + h * a.q_head;
      unsigned char* dst = qs + i * TILE + row * 128;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        const uint4 v = valid ? *reinterpret_cast<const uint4*>(q + d * 8) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + (d / 8) * PANEL + (((d & 7) ^ (row & 7)) << 4)) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) pg_arrive(&q_full);
    }
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // the warp's 32 lanes of tensor memory
    const uint32_t ts = tmem + lanes + i * 128, to = tmem + lanes + 256 + i * HD;
    const int pos = base + qrow;
    const int hi = valid ? pos + 1 : 1 << 30, lo = valid && a.window ? pos - a.window + 1 : 0;
    // the tile of rows: every row sees below hi_all, and from lo_all on
    const int hi_all = base + (f0 + i * 128) / p.group + 1, lo_all = a.window ? base + (f0 + i * 128 + 127) / p.group - a.window + 1 : 0;
    const float cexp = a.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < n_t; ++j) {
      const int s0 = sp.at(j) * PF_TS;
      wait_warp(&s_full[i], j & 1);
      pf_fence_after();
      uint32_t s[128];
#pragma unroll
      for (int k = 0; k < 4; ++k) pf_ld32(s + 32 * k, ts + 32 * k);
      pf_loaded(s);
      if (s0 + PF_TS > hi_all || (s0 < lo_all && s0 + PF_TS > a.sinks)) {
        const int h_r = hi - s0, l_r = lo - s0, k_r = a.sinks - s0;
#pragma unroll
        for (int k = 0; k < 128; ++k)
          if (k >= h_r || (k < l_r && k >= k_r)) s[k] = 0xff800000u;
      }
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < 128; ++k) top = fmaxf(top, __uint_as_float(s[k]));
      top *= cexp;
      const bool move = top > m + PF_SLACK || (m == -INFINITY && top > m);
      if (__any_sync(0xffffffffu, move)) {
        const float mn = fmaxf(m, top), fac = m == -INFINITY ? 0.f : pg_exp2(m - mn);
        l *= fac;
        m = mn;
        if (j > 0) {
#pragma unroll 1
          for (int k = 0; k < HD; k += 32) {
            uint32_t o[32];
            pf_ld32(o, to + k);
            pf_loaded(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fac);
            pf_st32(to + k, o);
          }
          pf_wait_st();
        }
      }
      const float use = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t w[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float x = pg_exp2(fmaf(__uint_as_float(s[64 * b + 2 * k]), cexp, -use));
          const float y = pg_exp2(fmaf(__uint_as_float(s[64 * b + 2 * k + 1]), cexp, -use));
          sum[k & 1] += x;
          sum[2 + (k & 1)] += y;
          w[k] = PgType<T>::down(x, y);
        }
        pf_st32(ts + 32 * b, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      pf_wait_st();
      pf_fence_before();
      __syncwarp();
      if (lane == 0) pg_arrive(&p_full[i]);
    }
    if (n_t > 0) {
      wait_warp(&s_full[i], n_t & 1);  // the last product into o
      pf_fence_after();
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    T* out = static_cast<T*>(a.out) + (long long)(first + qrow) * a.out_row + h * a.out_head;
#pragma unroll 1
    for (int k = 0; k < HD; k += 32) {
      uint32_t o[32];
      if (n_t > 0) {
        pf_ld32(o, to + k);
        pf_loaded(o);
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0;
      }
      if (valid) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint4 v;
          uint32_t* w = &v.x;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float y0 = __uint_as_float(o[e + 2 * x]), y1 = __uint_as_float(o[e + 2 * x + 1]);
            w[x] = PgType<T>::down(inv == 0.f ? 0.f : y0 * inv, inv == 0.f ? 0.f : y1 * inv);
          }
          *reinterpret_cast<uint4*>(out + k + e) = v;
        }
      }
      __syncwarp();
    }
    if (a.lse && valid)
      a.lse[(long long)(first + qrow) * a.n_q + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    pf_fence_before();
  } else if (warp == PF_PRODUCER) {
    // ---- K and V tiles, in the order of their use: K0 V0 K1 V1 ... ----
    const int box = min(c.page_size, PF_TS), boxes = PF_TS / box;
    int issued = 0;
    uint32_t edges = 0;
    for (int j = 0; j < n_max; ++j) {
      const int s0 = sp.at(j) * PF_TS, slot = s0 + lane * box;
      int page = c.n_pages;  // a box that nobody sees fills zeros
      const int w_lo = a.window ? p_lo - a.window + 1 : 0;
      if (lane < boxes && slot <= p_hi && (slot + box > w_lo || slot < a.sinks)) {
        page = sq.pages[slot / c.page_size];
        if (page < 0 || page >= c.n_pages) {
          pg_status(c.status, VP_DEV_ERR_PAGE);
          page = c.n_pages;
        }
      }
      // slots of the tile that no row of the CTA sees: their values may be NaN, which a zero weight
      // does not silence, so they are zeroed before the product may read them
      const bool ragged = s0 + PF_TS > p_hi + 1 || (s0 < w_lo && s0 + PF_TS > a.sinks);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv, ++issued) {
        const int st = issued % SLOTS;
        if (issued >= SLOTS) wait_warp(&kv_empty[st], (issued / SLOTS - 1) & 1);
        if (*(volatile int*)&dead) break;
        const bool patch = kv && ragged;
        uint64_t* bar = patch ? &edge : &kv_full[st];
        unsigned char* tile = ring + (size_t)st * TILE;
        if (lane == 0) mbar_arrive_expect_tx(bar, TILE);
        __syncwarp();
        if (lane < boxes) {
#pragma unroll
          for (int d = 0; d < PANELS; ++d)
            pg_box(tile + d * PANEL + lane * box * 128, kv ? &mv : &mk, d * 64, slot % c.page_size, head, page, bar);
        }
        if (patch) {
          wait_warp(&edge, edges & 1);
          ++edges;
          for (int x = lane; x < PF_TS; x += 32) {
            const int sl = s0 + x;
            if (sl > p_hi || (sl < w_lo && sl >= a.sinks)) {
#pragma unroll
              for (int d = 0; d < PANELS; ++d)
#pragma unroll
                for (int e = 0; e < 8; ++e) *reinterpret_cast<uint4*>(tile + d * PANEL + x * 128 + e * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) pg_arrive(&kv_full[st]);
        }
      }
      if (*(volatile int*)&dead) break;
    }
    // copies still in flight land before the CTA may end (they have, unless a wait ran out)
    for (int k = max(0, issued - SLOTS); k < issued; ++k) mbar_wait_warp(&kv_full[k % SLOTS], (k / SLOTS) & 1);
  } else if (warp == PF_ISSUER && lane == 0 && n_max > 0) {
    // ---- products ----
    constexpr uint32_t FMT = PgType<T>::BF16 ? 1u : 0u;
    constexpr uint32_t ID_S = 1u << 4 | FMT << 7 | FMT << 10 | (PF_TS / 8) << 17 | (128 / 16) << 24;
    constexpr uint32_t ID_O = 1u << 4 | FMT << 7 | FMT << 10 | 1u << 16 | (HD / 8) << 17 | (128 / 16) << 24;
    const uint32_t qb = smem_u32(qs), rb = smem_u32(ring);
    auto scores = [&](int i, int j) {  // S_i = Q_i K_j^T
      const uint32_t kb = rb + (2 * j % SLOTS) * TILE, qa = qb + i * TILE;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const uint32_t off = (k / 4) * PANEL + (k & 3) * 32;
        pf_mma_ss(tmem + i * 128, pf_desc(qa + off, 16, 1024), pf_desc(kb + off, 16, 1024), ID_S, k > 0);
      }
      pf_commit(&s_full[i]);
    };
    wait_one(&q_full, 0);
    wait_one(&kv_full[0], 0);
    pf_fence_after();
    if (n0 > 0) scores(0, 0);
    if (n1 > 0) scores(1, 0);
    pf_commit(&kv_empty[0]);
    for (int j = 0; j < n_max; ++j) {
      const int v = 2 * j + 1, vs = v % SLOTS, kn = 2 * j + 2;
      wait_one(&kv_full[vs], (v / SLOTS) & 1);
      bool k_there = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n_t = i ? n1 : n0;
        if (j >= n_t) continue;
        wait_one(&p_full[i], j & 1);
        if (*(volatile int*)&dead) break;
        pf_fence_after();
        const uint32_t vb = rb + vs * TILE;
#pragma unroll
        for (int k = 0; k < PF_TS / 16; ++k)
          pf_mma_ts(tmem + 256 + i * HD, tmem + i * 128 + k * 8, pf_desc(vb + k * 2048, PANEL, 1024), ID_O, j > 0 || k > 0);
        if (j + 1 < n_t) {
          if (!k_there) wait_one(&kv_full[kn % SLOTS], (kn / SLOTS) & 1), k_there = true;
          pf_fence_after();
          scores(i, j + 1);
        } else {
          pf_commit(&s_full[i]);
        }
      }
      if (*(volatile int*)&dead) break;
      pf_commit(&kv_empty[vs]);
      if (j + 1 < n_max) pf_commit(&kv_empty[kn % SLOTS]);
    }
    pf_commit(&drained);
    mbar_wait_bounded(&drained, 0);
    pf_fence_before();
  }
  cta_sync();
  pf_fence_after();
  if (warp == PF_ISSUER)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PF_TMEM) : "memory");
}

}  // namespace vp
