// Attention of many query rows per cache head over the paged cache: prompts (vp_paged_prefill), and
// vp_paged_decode where the new rows of a request and the heads of a group make more than 16.
//
// Mathematics as in vp_paged_decode.cuh: a running maximum m and sum l over tiles of 128 slots. The
// maximum that the weights are taken against only moves when the tile's is more than 2^PF_SLACK above it
// (out = o / l does not depend on it), so o is rarely rescaled. In fp16 it is taken PF_LIFT below: weights
// reach 2^(PF_SLACK + PF_LIFT), within its range, and those lost to o are below 2^-32 of the largest, in all
// 2^-15 of it over 2^17 slots.
//
// Bound: the tensor cores at head_dim 128, the exponentials (16 a clock and SM against 4,096 products)
// at 64. The query rows of one cache head are packed as row G + g, 256 of them to a block as two
// tiles of 128, so K and V are read once for 256 rows and the heads of a group share them. Tensor
// memory holds three buffers of S (two at head_dim 128; 128 columns each, the weights P written over
// them as pairs) and both o (head_dim columns each). A unit is a row tile with a tile of slots; units go
// round the buffers in order, first row tile, second row tile, next slots, so with three buffers the
// next S of a row tile is there before its present weights are. A block of one row tile has both
// warpgroups too: they take its tiles of slots in turns and join their two records at the end. One warp
// brings K and V tiles (TMA boxes of one page each), one thread issues the products, and two
// warpgroups, one row a thread, do the softmax: while one of them works on its tile, the tensor
// cores work on the other's.
//
// Work: one piece per (request, block, head), dealt out to one CTA per SM, the blocks with the most slots
// first. Where that gives a CTA more than its share, a block's tiles are cut into pieces of about an
// even share of all tiles (PF_LEAST at least); the pieces leave records in the work buffer and the
// one that finishes last (a counter per row tile, back at zero afterwards) joins them in order. A
// scheduler warp looks up the next piece, and its K and V arrive, while the present one is computed.
//
// Measured: a prompt of 8,192 rows, 32 + 2 x 8 heads of 128, bf16: 488 us, 1,128 TFLOP/s (68% of cuBLAS at bf16); of 64:
// 372 us, where the exponentials alone are 50% of the tensor rate. 16 prompts of 186 to 2,048 rows, 14 + 2 x 2 heads of 64:
// 82 us; one of 256: 10.5 us; 64 requests with 16 rows each over 151 to 2,064 slots: 25 us. Calls of equal blocks of 2 to
// 16 tiles, head_dim 64: 7.2 us + 4.8 a block of a CTA + 1.46 a 256 x 128 tile of scores; at 128: 9.5 + 5.5 + 2.0 to 2.3. Of a
// tile in a traced run, 1.76 us at 64: load and maximum 0.37, exponentials of both warpgroups 1.1, next S 0.25; 2.25 at
// 128: 0.37, 0.83, then its own two products 0.55 and 0.45 to be told.
#pragma once
#include "vp_paged_decode.cuh"

namespace vp {

constexpr int PF_TS = 128;                 // slots per tile
constexpr int PF_ROWS = 256;               // packed query rows per CTA
constexpr int PF_THREADS = 384;            // two softmax warpgroups, then one: producer, issuer, scheduler, an idle warp
constexpr int PF_PRODUCER = 8, PF_ISSUER = 9, PF_SCHEDULER = 10;
constexpr int PF_SOFTMAX_REGS = 208, PF_OTHER_REGS = 88;  // of the 168 a thread that the block is launched with
constexpr uint32_t PF_TMEM = 512;          // columns
constexpr float PF_SLACK = 8.f;            // log2 (with 4 and a lift of 11, 2,048 rows over 6,001 to 8,191 slots with a window and 4 sinks: 96 us, 89 with these)
constexpr float PF_LIFT = 7.f;             // log2, in fp16

template <int HD>
struct PfShape {
  static constexpr int PANELS = HD / 64;                        // 128-byte wide columns of a tile
  static constexpr int TILE = PF_TS * HD * 2;                   // bytes of a K, V or Q tile
  static constexpr int SLOTS = HD == 64 ? 8 : 4;                // ring of K and V tiles
  static constexpr int BUFS = HD == 64 ? 3 : 2;                 // buffers of S in tensor memory, beside both o
  static constexpr size_t SMEM = 1024 + 2 * TILE + (size_t)SLOTS * TILE;
};

constexpr int PF_RECORDS = 640;            // records at most: four per SM, for 160
constexpr int PF_AHEAD = 3;                // tiles of slots before a piece's end that the next piece is taken (two pieces
                                           // ahead: 4,096 rows 76 us instead of 60, as the CTAs no longer even out)
constexpr int PF_SORT = 128;               // requests that are sorted by length, at most (16 prompts: 87 us unsorted, 82
                                           // sorted; the sort is n steps a thread, 0.5 us at 128)
constexpr int PF_JOIN = 8;                 // records joined at a time (16 rows over 60,000 slots, 14 + 2 x 2 heads of 64: 46 us, all 74 at once 64)
constexpr int PF_LEAST = 16;               // tiles of a piece, at least (64 trees: 25.1 us, one over 2,000 slots 22.5; with 8, whose joins cost
                                           // more than they save: 27.7 and 26.3, but 16 rows over 60,000 slots 42 instead of 46)

struct PfParams {
  vp_paged c;
  vp_paged_attn a;
  float* rec;         // records of block_rows rows, one per piece of a cut block
  unsigned* tickets;  // [2 steps of a join][records][2 row tiles], then the scheduler's two
  int group, block_rows, sms, most;  // most: pieces that a call can have
  int rows;                          // packed rows of a block: 256, or 128 where there are few blocks
  int cuts;                          // whether the table's longest request may be cut
};

__device__ __forceinline__ uint64_t pf_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  // shared-memory operand, 128-byte swizzle: address and offsets in 16-byte units
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)((stride >> 4) & 0x3fff) << 32 |
         1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ bool pf_elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
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

// Slots [0, min(sinks, end)) and [lo, end) as tiles: [0, ns) hold the sinks, then [ws, ..).
struct PfSpan {
  int ns, ws, tiles;
  __device__ __forceinline__ int at(int t) const { return t < ns ? t : ws + t - ns; }
  // tiles of the list that start below `stop`
  __device__ __forceinline__ int upto(int stop) const {
    const int end = stop <= 0 ? 0 : (stop - 1) / PF_TS + 1;
    return min(tiles, end <= ns ? end : ns + max(0, end - ws));
  }
};
__device__ __forceinline__ PfSpan pf_span(int lo, int end, int sinks) {
  PfSpan s;
  const int all = end <= 0 ? 0 : (end - 1) / PF_TS + 1;
  s.ns = lo > 0 ? min((min(sinks, max(end, 0)) + PF_TS - 1) / PF_TS, all) : 0;
  s.ws = min(max(lo, 0) / PF_TS, all);
  if (s.ws <= s.ns) s.ws = s.ns = 0;
  s.tiles = s.ns + all - s.ws;
  return s;
}
// The request's part of a call: its new rows, and the slots that packed rows [f, g) of it see.
struct PfSeq {
  int index, first, n_new, len, base, blocks, least, row;  // index: of the request; least: fewest mask bits of a row (trees); row: of the table
  int lo, end;                                 // of the last range asked for
  __device__ __forceinline__ void see(const PfParams& p, int f, int g) {
    const bool tree = !p.a.q_start;
    const int p_lo = tree ? base + min(least, p.a.window) - 1 : base + f / p.group;  // a tree's new slots go by its masks, not by lo
    end = tree ? len : base + (g - 1) / p.group + 1;
    lo = p.a.window ? max(0, p_lo - p.a.window + 1) : 0;
  }
  __device__ __forceinline__ int last_tiles(const PfParams& p) {  // of the last block, which has the most
    see(p, (blocks - 1) * p.rows, n_new * p.group);
    return pf_span(lo, end, p.a.sinks).tiles;
  }
};
__device__ __forceinline__ PfSeq pf_seq(const PfParams& p, int i) {
  PfSeq s;
  s.index = i;
  s.first = 0;
  s.n_new = p.a.rows;
  s.least = 1;
  if (p.a.q_start) {
    const int x = p.a.q_start[i], y = p.a.q_start[i + 1];
    s.first = min(max(x, 0), p.a.rows);
    const int next = min(max(y, 0), p.a.rows);
    if (s.first != x || next != y || next < s.first) pg_status(p.c.status, VP_DEV_ERR_SLOT);
    s.n_new = max(0, next - s.first);
  } else if (p.a.window && p.a.mask) {
    s.least = p.a.rows;
    for (int r = 0; r < p.a.rows; ++r)
      s.least = min(s.least, __popc((uint32_t)p.a.mask[(long long)i * p.a.rows + r] & ((1u << p.a.rows) - 1)));
  }
  s.len = pg_len(p.c, p.a.seqs, p.a.lens, i);
  s.row = p.a.seqs ? p.a.seqs[i] : i;
  s.base = s.len - s.n_new;
  s.blocks = (int)(((unsigned)s.n_new * (unsigned)p.group + p.rows - 1) / p.rows);
  return s;
}
// Cuts of each of a request's blocks: none as long as the largest is not half as much again as the share.
__device__ __forceinline__ int pf_cuts(int last, int share) { return 2 * last > 3 * share ? (last + share - 1) / share : 1; }
__device__ __forceinline__ uint32_t pf_low(int x) { return x <= 0 ? 0u : x >= 32 ? ~0u : (1u << x) - 1; }

// A piece as the scheduler hands it to the other roles.
struct PfPiece {
  int seq, row, head, f0, f_end, first, base, cut, cuts, live, record0, j0, n0, n1, see_lo, see_end, ns, ws;  // seq < 0: no more
  uint32_t any;                 // trees: new slots that a row sees
  uint32_t masks[PG_MAX_ROWS];  // bits 0-15: new slots that the row sees, 16-20: the row's mask bits
};

__device__ __forceinline__ float2 pf_fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 pf_add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}

// Number of the unit (warpgroup i, its j-th tile of slots) in its piece. Two row tiles: one to a warpgroup, the
// first has n0 tiles of slots, the second as many or more. One: the warpgroups take turns.
__device__ __forceinline__ int pf_unit(bool two, int i, int j, int n0) { return !two || j < n0 ? 2 * j + i : n0 + j; }

// Named barriers of the warpgroups with one row tile: the second one's part of o is there, is taken.
constexpr int PF_PART = 3, PF_TAKEN = 4;
__device__ __forceinline__ void pf_sync(int bar) {
  __syncwarp();
  asm volatile("barrier.sync %0, 256;" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pf_arrive(int bar) {
  __threadfence_block();
  __syncwarp();
  asm volatile("barrier.arrive %0, 256;" ::"r"(bar) : "memory");
}

template <typename T, int HD>
__global__ void __launch_bounds__(PF_THREADS, 1)
    k_paged_tiles(const __grid_constant__ PfParams p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
  using Sh = PfShape<HD>;
  constexpr int TILE = Sh::TILE, SLOTS = Sh::SLOTS, PANELS = Sh::PANELS, PANEL = PF_TS * 128, BUFS = Sh::BUFS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* qs = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* ring = qs + 2 * TILE;
  // of a buffer: its S is there, its weights are, its product into o is done; of a row tile: the piece's last product is
  __shared__ uint64_t kv_full[SLOTS], kv_empty[SLOTS], s_full[BUFS], p_full[BUFS], o_done[BUFS], o_last[2], q_full, edge, drained, info_full[2], info_empty[2], wanted;
  __shared__ uint32_t tmem_base;
  __shared__ long long tile_sums[PF_THREADS / 32];
  __shared__ int sums[PF_THREADS / 32][2], starts[PF_THREADS], rec_starts[PF_THREADS], dead, last_s[2];
  __shared__ PfPiece info[2];
  __shared__ float2 part_ml[128];  // m and l of the second warpgroup's records
  __shared__ PfSeq seqs_s[PF_THREADS];  // the requests, where there are no more than threads

  const vp_paged& c = p.c;
  const vp_paged_attn& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool tree = !a.q_start;

  pdl_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < BUFS; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&o_last[i], 1);
      mbar_init(&info_full[i], 1);
      mbar_init(&info_empty[i], 10);  // the softmax warps, the producer, the issuer
    }
    mbar_init(&q_full, 9);  // the softmax warps and the issuer
    mbar_init(&edge, 1);
    mbar_init(&drained, 1);
    mbar_init(&wanted, 1);
    fence_barrier_init();
    dead = 0;
    info[0].seq = info[1].seq = -1;
  }
  if (warp == PF_PRODUCER && lane == 0) {
    pg_prefetch_map(&mk);
    pg_prefetch_map(&mv);
  }
  pdl_wait();
  // Pieces of all requests, in two sums: all tiles, which give the share of a CTA (left out where no
  // request can be long enough to be cut); pieces and records.
  const int chunk = (a.n + PF_THREADS - 1) / PF_THREADS, i0 = min(a.n, tid * chunk), i1 = min(a.n, i0 + chunk);
  long long tiles = 0;
  int one_blocks = 0, one_last = 0;  // of the thread's last request
  if (chunk == 1 && i0 < i1) seqs_s[tid] = pf_seq(p, tid);
  if (a.n > 1 && a.n <= PF_SORT) {  // longest requests last: pieces are taken from the end
    __shared__ int ranks_s[PF_SORT];
    if (i0 < i1) ranks_s[tid] = seqs_s[tid].blocks ? seqs_s[tid].last_tiles(p) : 0;
    const PfSeq s = seqs_s[min(tid, a.n - 1)];
    cta_sync();
    if (i0 < i1) {
      int rank = 0;
      for (int k = 0; k < a.n; ++k) rank += ranks_s[k] < ranks_s[tid] || (ranks_s[k] == ranks_s[tid] && k < tid);
      seqs_s[rank] = s;
    }
    cta_sync();
  }
  for (int i = i0; i < i1; ++i) {
    PfSeq s = chunk == 1 ? seqs_s[tid] : pf_seq(p, i);
    one_blocks = s.blocks;
    if (!s.blocks || !p.cuts) continue;
    one_last = s.last_tiles(p);
    s.see(p, 0, min(p.rows, s.n_new * p.group));
    tiles = min(tiles + (long long)s.blocks * (one_last + pf_span(s.lo, s.end, a.sinks).tiles), 1ll << 50);
  }
  // Tensor memory is taken here, beside the reads above, not in the prologue: the kernel before may be one that still waits
  // for its own, on this SM, while this one would hold all of it and wait for its end.
  __syncwarp();
  if (warp == PF_ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(PF_TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  int share = 1 << 30;
  if (p.cuts) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    if (lane == 0) tile_sums[warp] = tiles;
    cta_sync();
    long long all = 0;
#pragma unroll
    for (int w = 0; w < PF_THREADS / 32; ++w) all += tile_sums[w];
    // the mean of its first and last block stands for a request's blocks: `all` is twice the tiles per
    // cache head. Rounded up by two so that the float division cannot make it less than an even half.
    share = max(PF_LEAST, (int)fminf((float)all * c.n_kv / (2 * p.sms), 1e8f) + 2);
  }
  // Requests whose rows overlap can have more pieces than a word counts: the sums stop at PF_MANY, which is more than
  // any call may have.
  constexpr unsigned PF_MANY = 0x7fffffff;
  unsigned pieces = 0;
  int records = 0;
  for (int i = i0; i < i1; ++i) {
    int blocks = one_blocks, last = one_last;
    if (chunk > 1) {
      PfSeq s = pf_seq(p, i);
      blocks = s.blocks;
      if (blocks && p.cuts) last = s.last_tiles(p);
    }
    if (!blocks) continue;
    const int n = p.cuts ? pf_cuts(last, share) : 1;
    pieces = (unsigned)min(pieces + (unsigned long long)blocks * n * c.n_kv, (unsigned long long)PF_MANY);
    if (n > 1) records += blocks * n * c.n_kv;
  }
  unsigned incl = pieces;
  int incl_r = records;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
    const int x = __shfl_up_sync(0xffffffffu, incl_r, o);
    if (lane >= o) incl = min(incl + v, PF_MANY), incl_r += x;
  }
  if (lane == 31) sums[warp][0] = (int)incl, sums[warp][1] = incl_r;
  cta_sync();
  unsigned at0 = incl - pieces, total = 0;
  int at_r0 = incl_r - records;
#pragma unroll
  for (int w = 0; w < PF_THREADS / 32; ++w) {
    if (w < warp) at0 += sums[w][0], at_r0 += sums[w][1];
    total = min(total + sums[w][0], PF_MANY);
  }
  starts[tid] = (int)at0;
  rec_starts[tid] = at_r0;
  pf_fence_before();
  cta_sync();
  pf_fence_after();
  const uint32_t tmem = tmem_base;

  // Waits of a whole warp. After one that ran out none waits any more, and the call ends with an error status: the
  // scheduler hands out no more pieces, and everybody goes through those that are out, without waiting, to the end. No role
  // leaves before: the softmax warps meet at named barriers, which have no limit and want all of them. So the hand-over
  // of pieces itself is always waited for. Its limit is many times that of the others: no role passes more than one wait that
  // runs out.
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
    __syncwarp();
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const bool there = pg_wait(bar, parity, &dead);
    if (!there) {
      pg_status(c.status, VP_DEV_ERR_TIMEOUT);
      *(volatile int*)&dead = 1;
    }
    __syncwarp();
    return there;
  };
  auto wait_piece = [&](uint64_t* bar, uint32_t parity) {
    __syncwarp();
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
#pragma unroll 1
    for (int k = 0; k < 8; ++k)
      if (mbar_wait_warp(bar, parity)) return;
    pg_status(c.status, VP_DEV_ERR_TIMEOUT);
    *(volatile int*)&dead = 1;
    __syncwarp();
  };

  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PF_OTHER_REGS));
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PF_SOFTMAX_REGS));
    // ---- softmax: warpgroup i has row tile i (or every other tile of slots), a thread row f ----
    const int i = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // the warp's 32 lanes of tensor memory
    const uint32_t to = tmem + lanes + BUFS * 128 + i * HD;
    const float cexp = a.scale * 1.4426950408889634f;
    const size_t rec_floats = pg_record(p.block_rows, HD);
    const int m_at = p.block_rows * HD, l_at = m_at + p.block_rows;
    uint32_t units = 0, n_last = 0;  // units of all pieces so far, phases of o_last so far
    // Queries of piece r on their way into the row tile's buffer, once the last product that reads it is done.
    auto fetch = [&](int r) {
      wait_piece(&info_full[r & 1], (r >> 1) & 1);
      const PfPiece& in = info[r & 1];
      const int f = in.f0 + tid;  // with one row tile the second warpgroup has none to bring
      if (in.seq >= 0 && f < in.f_end) {
        const T* q = static_cast<const T*>(a.q) + in.seq * a.q_seq + (long long)(in.first + f / p.group) * a.q_row +
                     (in.head * p.group + f % p.group) * a.q_head;
        unsigned char* dst = qs + i * TILE + row * 128;
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) pg_cp16(dst + (d / 8) * PANEL + (((d & 7) ^ (row & 7)) << 4), q + d * 8);
      }
      __syncwarp();
    };
    auto hand_over = [&] {  // they are there: the issuer may start the piece
      asm volatile("cp.async.wait_all;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) pg_arrive(&q_full);
    };
    bool fetched = false, handed = false, lent = false;  // lent: the row tile's buffer holds a part of o
    for (int r = 0;; ++r) {
      if (lent) pf_sync(PF_TAKEN);  // the buffer is the queries' again
      lent = false;
      if (!fetched) fetch(r);
      fetched = false;
      const PfPiece& in = info[r & 1];
      const int seq = in.seq, f_end = in.f_end, f0 = in.f0, head = in.head, first = in.first, base = in.base;
      if (seq < 0) break;
      const bool two = f_end > f0 + 128;  // row tiles
      const int i_row = two ? i : 0, f = f0 + i_row * 128 + row;
      const int n_t = !two ? (in.n0 + 1 - i) / 2 : i ? in.n1 : in.n0, j0 = in.j0, cuts = in.cuts, cut = in.cut, live = in.live, record0 = in.record0;
      const int n0 = in.n0, n1 = in.n1;
      PfSpan sp;
      sp.ns = in.ns;
      sp.ws = in.ws;
      const bool valid = f < f_end;
      const int qrow = f / p.group, h = head * p.group + f % p.group;
      // the row sees old slots [lo, hi), the sinks below hi, and new slot j of a tree where bit j is set
      uint32_t bits = 0;
      int hi = 0, lo = 0;
      if (valid && base + qrow >= 0) {
        const uint32_t mask = tree ? in.masks[qrow] : 0;
        bits = mask & 0xffffu;
        hi = tree ? base : base + qrow + 1;
        if (a.window) lo = (tree ? base + (int)(mask >> 16) : base + qrow + 1) - a.window;
      }
      __syncwarp();
      if (lane == 0) pg_arrive(&info_empty[r & 1]);
      if (!handed) hand_over();
      handed = false;
      {
        // Everybody starts the piece together: a warp ahead of the others would wait for phases of barriers
        // whose earlier phases, the other warpgroup's, are still to come, and take one for another.
        wait_warp(&q_full, r & 1);
      }
      // every row of the tile sees [lo_all, hi_all)
      const int hi_all = tree ? base : base + (f0 + i_row * 128) / p.group + 1;
      const int lo_all = !a.window ? 0 : tree ? base + a.rows - a.window : base + (f0 + i_row * 128 + 127) / p.group - a.window + 1;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n_t; ++j) {
        const int s0 = sp.at(j0 + (two ? j : 2 * j + i)) * PF_TS;
        const uint32_t u = units + pf_unit(two, i, j, n0), buf = u % BUFS;
        const uint32_t ts = tmem + lanes + buf * 128;
        wait_warp(&s_full[buf], (u / BUFS) & 1);
        pf_fence_after();
        uint32_t s[128];
#pragma unroll
        for (int k = 0; k < 4; ++k) pf_ld32(s + 32 * k, ts + 32 * k);
        if (j + 1 == n_t && two) {  // the row tile's last scores are there: the next piece's queries may come
          fetch(r + 1);
          fetched = true;
        }
        pf_loaded(s);
        if (s0 + PF_TS > hi_all || (s0 < lo_all && s0 + PF_TS > a.sinks)) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int b = s0 + 32 * k, fresh = base - b;
            uint32_t see = (pf_low(hi - b) & ~pf_low(lo - b)) | pf_low(min(a.sinks, hi) - b);
            if (__any_sync(0xffffffffu, bits != 0)) see |= fresh >= 32 || fresh <= -32 ? 0u : fresh >= 0 ? bits << fresh : bits >> -fresh;
            if (__all_sync(0xffffffffu, see == ~0u)) continue;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((see >> e) & 1)) s[32 * k + e] = 0xff800000u;
          }
        }
        float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains: a single one is 128 steps long
#pragma unroll
        for (int k = 0; k < 128; k += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            t4[e] = fmaxf(fmaxf(t4[e], __uint_as_float(s[k + 2 * e])), __uint_as_float(s[k + 2 * e + 1]));
        const float top = fmaf(fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])), cexp, PgType<T>::BF16 ? 0.f : -PF_LIFT);
        const bool move = top > m + PF_SLACK || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, move)) {
          // a row's maximum moves by its own scores alone: what the other rows of the warp hold (rows past the
          // block's end: anything) must not show in its bits
          const float mn = move ? top : m, fac = m == -INFINITY ? 0.f : pg_exp2(m - mn);
          l *= fac;
          m = mn;
          if (j > 0) {
            const uint32_t before = units + pf_unit(two, i, j - 1, n0);
            if (u - before < BUFS) {  // the last product into o may be under way: this S did not wait for it
              wait_warp(&o_done[before % BUFS], (before / BUFS) & 1);
              pf_fence_after();
            }
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
        const float2 c2 = make_float2(cexp, cexp), u2 = make_float2(-use, -use);
        float2 sum[4] = {};
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t w[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            float2 x = make_float2(__uint_as_float(s[64 * b + 2 * k]), __uint_as_float(s[64 * b + 2 * k + 1]));
            x = pf_fma2(x, c2, u2);
            x = make_float2(pg_exp2(x.x), pg_exp2(x.y));
            sum[k & 3] = pf_add2(sum[k & 3], x);
            w[k] = PgType<T>::down(x.x, x.y);
          }
          pf_st32(ts + 32 * b, w);
        }
        sum[0] = pf_add2(pf_add2(sum[0], sum[1]), pf_add2(sum[2], sum[3]));
        l += sum[0].x + sum[0].y;
        pf_wait_st();
        pf_fence_before();
        __syncwarp();
        if (lane == 0) pg_arrive(&p_full[buf]);
      }
      if (n_t > 0) {
        wait_warp(&o_last[i], n_last & 1);
        ++n_last;
        pf_fence_after();
        if (fetched) {
          hand_over();  // the next piece's first scores are made beside this one's epilogue
          handed = true;
        } else if (i == 0) {  // one row tile: before this product the other warpgroup's last scores were made too
          fetch(r + 1);
          fetched = true;
        }
      }
      units += two ? n0 + n1 : n0;
      T* out = static_cast<T*>(a.out) + seq * a.out_seq + (long long)(first + qrow) * a.out_row + h * a.out_head;
      float* lse = a.lse ? a.lse + ((tree ? (long long)seq * a.rows : (long long)first) + qrow) * a.n_q + h : nullptr;
      float* rec = p.rec + (size_t)(record0 + cut) * rec_floats;
      // The warpgroup's writes are out, and it is told whether it is the last of n to come (and the counter is reset).
      auto arrive_last = [&](unsigned* ticket, int n) {
        __threadfence();
        __syncwarp();
        asm volatile("barrier.sync %0, 128;" ::"r"(1 + i) : "memory");
        if (row == 0) {
          last_s[i] = atomicAdd(ticket, 1u) == (unsigned)(n - 1);
          if (last_s[i]) *ticket = 0;
        }
        __syncwarp();
        asm volatile("barrier.sync %0, 128;" ::"r"(1 + i) : "memory");
        const bool last = last_s[i];
        if (last) __threadfence();
        return last;
      };
      // Records first, first + step, .. (n of them) of the row tile joined into the output, or into the first one:
      // a thread a row, the weights in place of the maxima; then 4 elements a thread and turn, four turns'
      // reads of 4 records in flight.
      auto join = [&](int from, int n, int step, bool to_out) {
        float* rec0 = p.rec + (size_t)(record0 + from) * rec_floats;
        const size_t stride = step * rec_floats;
        const int n_rows = min(128, f_end - f0 - i * 128);
        float top = -INFINITY, sm = 0.f;
        if (row < n_rows) {
#pragma unroll 8
          for (int k = 0; k < n; ++k) top = fmaxf(top, __ldcg(rec0 + k * stride + m_at + tid));
          const float us = top == -INFINITY ? 0.f : top;
#pragma unroll 8
          for (int k = 0; k < n; ++k) sm += __ldcg(rec0 + k * stride + l_at + tid) * pg_exp2(__ldcg(rec0 + k * stride + m_at + tid) - us);
          const float iv = !to_out ? 1.f : sm > 0.f ? 1.f / sm : sm == 0.f ? 0.f : sm;
#pragma unroll 8
          for (int k = 0; k < n; ++k) {
            float* x = rec0 + k * stride + m_at + tid;
            *x = pg_exp2(__ldcg(x) - us) * iv;
          }
          if (to_out && lse) *lse = sm == 0.f ? -INFINITY : (top + log2f(sm)) * 0.6931471805599453f;
        }
        __threadfence();
        __syncwarp();
        asm volatile("barrier.sync %0, 128;" ::"r"(1 + i) : "memory");
        constexpr int W = 4;
        for (int x0 = row; x0 < n_rows * (HD / 4); x0 += 128 * W) {
          float4 acc[W] = {};
          int mm[W], d[W];
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const int x = min(x0 + 128 * e, n_rows * (HD / 4) - 1);
            mm[e] = i * 128 + x / (HD / 4), d[e] = x % (HD / 4) * 4;
          }
          for (int k0 = 0; k0 < n; k0 += 4) {
            float4 v[W][4];
            float w[W][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float* x = rec0 + min(k0 + k, n - 1) * stride;
#pragma unroll
              for (int e = 0; e < W; ++e) {
                v[e][k] = __ldcg(reinterpret_cast<const float4*>(x + (size_t)mm[e] * HD + d[e]));
                w[e][k] = __ldcg(x + m_at + mm[e]);
              }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int e = 0; e < W; ++e) {
                const float f1 = k0 + k < n ? w[e][k] : 0.f;
                acc[e].x += v[e][k].x * f1, acc[e].y += v[e][k].y * f1, acc[e].z += v[e][k].z * f1, acc[e].w += v[e][k].w * f1;
              }
          }
#pragma unroll
          for (int e = 0; e < W; ++e) {
            if (x0 + 128 * e >= n_rows * (HD / 4)) break;
            if (!to_out) {
              *reinterpret_cast<float4*>(rec0 + (size_t)mm[e] * HD + d[e]) = acc[e];
              continue;
            }
            const int r2 = (f0 + mm[e]) / p.group, h2 = head * p.group + (f0 + mm[e]) % p.group;
            uint2 v2;
            v2.x = PgType<T>::down(acc[e].x, acc[e].y);
            v2.y = PgType<T>::down(acc[e].z, acc[e].w);
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + seq * a.out_seq + (long long)(first + r2) * a.out_row + h2 * a.out_head + d[e]) = v2;
          }
        }
        if (!to_out) {
          __syncwarp();
          asm volatile("barrier.sync %0, 128;" ::"r"(1 + i) : "memory");
          if (row < n_rows) rec0[m_at + tid] = top, rec0[l_at + tid] = sm;
        }
        __syncwarp();
      };
      // one row tile: the second warpgroup hands its record over, 32 elements at a time, in its row tile's buffer
      unsigned char* part = qs + TILE + row * 128;
      float mine = 1.f, other = 0.f;
      if (!two && i == 1) {
        part_ml[row] = make_float2(m, l);
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
          if (k > 0) pf_sync(PF_TAKEN);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(part + ((e ^ (row & 7)) << 4)) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          pf_arrive(PF_PART);
        }
        lent = true;
      }
      if (f_end > f0 + i * 128) {
        float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
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
          if (!two) {
            pf_sync(PF_PART);
            if (k == 0) {
              const float2 ml = part_ml[row];
              const float top = fmaxf(m, ml.x), use = top == -INFINITY ? 0.f : top;
              mine = pg_exp2(m - use);
              other = pg_exp2(ml.x - use);
              l = l * mine + ml.y * other;
              m = top;
              inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 v = *reinterpret_cast<const float4*>(part + ((e ^ (row & 7)) << 4));
              o[4 * e] = __float_as_uint(__uint_as_float(o[4 * e]) * mine + v.x * other);
              o[4 * e + 1] = __float_as_uint(__uint_as_float(o[4 * e + 1]) * mine + v.y * other);
              o[4 * e + 2] = __float_as_uint(__uint_as_float(o[4 * e + 2]) * mine + v.z * other);
              o[4 * e + 3] = __float_as_uint(__uint_as_float(o[4 * e + 3]) * mine + v.w * other);
            }
            pf_arrive(PF_TAKEN);
          }
          if (valid && cuts > 1) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(rec + (size_t)tid * HD + k + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          } else if (valid) {
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
        if (valid && cuts > 1) rec[m_at + tid] = m, rec[l_at + tid] = l;
        if (valid && cuts == 1 && lse) *lse = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        pf_fence_before();
        if (cuts > 1) {
          // A few pieces are joined by the one that finishes last; of many, every PF_JOIN by their last one into
          // the first one's record, and those by the last of all.
          unsigned* t1 = p.tickets + 2 * (record0 + cut / PF_JOIN * PF_JOIN) + i;
          unsigned* t2 = p.tickets + 2 * PF_RECORDS + 2 * record0 + i;
          const bool deep = cuts > PF_JOIN + PF_JOIN / 2;
          const int k_first = deep ? cut / PF_JOIN * PF_JOIN : 0, k_last = deep ? min(cuts, k_first + PF_JOIN) : cuts;
          bool last = arrive_last(deep ? t1 : t2, k_last - k_first);
          if (last && deep) {
            join(k_first, max(0, min(k_last, live) - k_first), 1, false);
            last = arrive_last(t2, (cuts + PF_JOIN - 1) / PF_JOIN);
          }
          if (last) join(0, deep ? (live + PF_JOIN - 1) / PF_JOIN : live, deep ? PF_JOIN : 1, true);
        }
      }
      pf_fence_before();
    }
  } else if (warp == PF_SCHEDULER) {
    // ---- the CTA's pieces: one for each CTA, then whoever comes first has the next, from the last request's
    // last block on. Which CTA has a piece does not show in the results. ----
    unsigned* next = p.tickets + 4 * PF_RECORDS;  // and the number of CTAs that have come to the end
    for (int r = 0;; ++r) {
      if (r >= 2) wait_piece(&info_empty[r & 1], ((r >> 1) - 1) & 1);
      unsigned idx = blockIdx.x;
      if (r > 0) {  // taken when the last copies of the piece before are under way, not earlier: whoever is ahead takes more
        wait_warp(&wanted, (r - 1) & 1);
        if (lane == 0) idx = gridDim.x + atomicAdd(next, 1u);
        idx = __shfl_sync(0xffffffffu, idx, 0);
      }
      int piece = idx < total ? (int)(total - 1 - idx) : -1;
      if (total > (unsigned)p.most) {  // requests whose rows overlap
        if (lane == 0) pg_status(c.status, VP_DEV_ERR_SLOT);
        piece = -1;
      }
      PfPiece& in = info[r & 1];
      if (__any_sync(0xffffffffu, piece < 0 || *(volatile int*)&dead)) {
        if (lane == 0) {
          in.seq = -1;
          pg_arrive(&info_full[r & 1]);
          if (atomicAdd(next + 1, 1u) == gridDim.x - 1) next[0] = next[1] = 0;  // the last one leaves them as it found them
        }
        break;
      }
      // the thread whose run of requests has the piece: 32 threads at a time
      int owner = 0;
#pragma unroll
      for (int b = 0; b < PF_THREADS; b += 32) {
        const uint32_t under = __ballot_sync(0xffffffffu, starts[b + lane] <= piece);
        owner += __popc(under);
      }
      owner -= 1;
      int at = starts[owner], at_r = rec_starts[owner], seq = owner * chunk;
      PfSeq s = chunk == 1 ? seqs_s[seq] : pf_seq(p, seq);
      int cuts = 1;
      for (;; s = pf_seq(p, ++seq)) {
        if (s.blocks) {
          cuts = p.cuts ? pf_cuts(s.last_tiles(p), share) : 1;
          const int k = s.blocks * cuts * c.n_kv;
          if (piece < at + k) break;
          at += k;
          if (cuts > 1) at_r += k;
        }
      }
      // pieces of a request: block, then head, then cut
      const int mine = piece - at, pair = mine / cuts, cut = mine - pair * cuts, block = pair / c.n_kv;
      const int f0 = block * p.rows, f_end = min(s.n_new * p.group, f0 + p.rows);
      s.see(p, f0, f_end);
      const PfSpan sp = pf_span(s.lo, s.end, a.sinks);
      const int live = max(1, min(cuts, sp.tiles)), per = sp.tiles / live, odd = sp.tiles % live;
      const int j0 = cut * per + min(cut, odd), j1 = cut < live ? j0 + per + (cut < odd) : j0;
      const int stop0 = tree ? s.end : s.base + (min(f_end, f0 + 128) - 1) / p.group + 1;
      if (tree) {
        const uint32_t all_rows = (1u << a.rows) - 1;
        uint32_t anc = 0, keep = 0;
        if (lane < a.rows) anc = a.mask ? (uint32_t)a.mask[(long long)s.index * a.rows + lane] & all_rows : (2u << lane) - 1;
        const int pos = s.base + __popc(anc) - 1;
        for (int j = 0; j < a.rows; ++j) {  // less the new slots that have left the row's window
          const int place = s.base + __popc(__shfl_sync(0xffffffffu, anc, j)) - 1;
          if (!a.window || pos - place < a.window || place < a.sinks) keep |= 1u << j;
        }
        const uint32_t any = __reduce_or_sync(0xffffffffu, s.base + lane >= 0 ? anc & keep : 0u);
        if (lane < PG_MAX_ROWS) in.masks[lane] = (anc & keep) | (uint32_t)__popc(anc) << 16;
        if (lane == 0) in.any = any;
      }
      if (lane == 0) {
        in.seq = s.index, in.row = s.row, in.head = pair - block * c.n_kv, in.f0 = f0, in.f_end = f_end, in.first = s.first, in.base = s.base;
        in.cut = cut, in.cuts = cuts, in.live = live, in.record0 = at_r + mine - cut;
        in.j0 = j0, in.n0 = max(0, min(j1, sp.upto(stop0)) - j0), in.n1 = f_end > f0 + 128 ? j1 - j0 : 0;
        in.see_lo = s.lo, in.see_end = s.end, in.ns = sp.ns, in.ws = sp.ws;
      }
      __threadfence_block();
      __syncwarp();
      if (lane == 0) pg_arrive(&info_full[r & 1]);
    }
  } else if (warp == PF_PRODUCER) {
    // ---- K and V tiles, in the order of their use: K0 V0 K1 V1 ... ----
    const int box = min(c.page_size, PF_TS), boxes = PF_TS / box;
    uint32_t issued = 0, edges = 0;
    bool gone = false;  // a wait ran out: nothing is refilled any more
    for (int r = 0;; ++r) {
      wait_piece(&info_full[r & 1], (r >> 1) & 1);
      const PfPiece& in = info[r & 1];
      const int seq = in.seq, table_row = in.row, head = in.head, j0 = in.j0, n_max = max(in.n0, in.n1), see_lo = in.see_lo, see_end = in.see_end, base = in.base;
      const uint32_t any = in.any;
      PfSpan sp;
      sp.ns = in.ns;
      sp.ws = in.ws;
      if (seq < 0) break;
      __syncwarp();
      if (lane == 0) pg_arrive(&info_empty[r & 1]);
      // a request outside the table has no slots, and no page is looked up for it
      const int32_t* pages = c.table + table_row * c.table_stride;
      for (int j = 0; j < n_max && !gone; ++j) {
        if (j == max(0, n_max - PF_AHEAD) && lane == 0) pg_arrive(&wanted);
        const int s0 = sp.at(j0 + j) * PF_TS, slot = s0 + lane * box;
        int page = c.n_pages;  // a box that nobody sees fills zeros
        if (lane < boxes && slot < see_end && (slot + box > see_lo || slot < a.sinks)) {
          page = pages[slot / c.page_size];
          if (page < 0 || page >= c.n_pages) {
            pg_status(c.status, VP_DEV_ERR_PAGE);
            page = c.n_pages;
          }
        }
        // slots of the tile that no row of the block sees: their values may be NaN, which a zero weight
        // does not silence, so they are zeroed before the product may read them
        const bool ragged = s0 + PF_TS > (tree ? base : see_end) || (s0 < see_lo && s0 + PF_TS > a.sinks);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++issued) {
          const uint32_t st = issued % SLOTS;
          if (issued >= SLOTS && !gone) gone = !wait_warp(&kv_empty[st], (issued / SLOTS - 1) & 1);
          if (gone) break;
          const bool patch = kv && ragged;
          uint64_t* bar = patch ? &edge : &kv_full[st];
          unsigned char* tile = ring + (size_t)st * TILE;
          if (lane == 0) mbar_arrive_expect_tx(bar, TILE);
          __syncwarp();
          if (lane < boxes) {
#pragma unroll
            for (int d = 0; d < PANELS; ++d)
              pg_box(tile + d * PANEL + lane * box * 128, kv ? &mv : &mk, d, slot & (c.page_size - 1), head, page, bar);
          }
          if (patch) {
            gone = !wait_warp(&edge, edges & 1);
            ++edges;
            for (int x = lane; x < PF_TS; x += 32) {
              const int sl = s0 + x;
              if (sl >= see_end || (sl < see_lo && sl >= a.sinks) || (tree && sl >= base && !((any >> (sl - base)) & 1))) {
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
      }
      if (n_max == 0 && lane == 0) pg_arrive(&wanted);
    }
    // copies still in flight land before the CTA may end (they have, unless a wait ran out)
    if (edges) mbar_wait_warp(&edge, (edges - 1) & 1);
    for (uint32_t k = issued > SLOTS ? issued - SLOTS : 0; k < issued; ++k) mbar_wait_warp(&kv_full[k % SLOTS], (k / SLOTS) & 1);
  } else if (warp == PF_ISSUER) {
    // ---- products. The whole warp walks, one elected lane issues: what the operands' descriptors come from
    // is the same in every lane and known to be (shuffles), so that they live in uniform registers. With
    // one lane walking alone every product took 100 clocks to issue, more than it takes to compute. ----
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const bool lead = pf_elect();
    constexpr uint32_t FMT = PgType<T>::BF16 ? 1u : 0u;
    constexpr uint32_t ID_S = 1u << 4 | FMT << 7 | FMT << 10 | (PF_TS / 8) << 17 | (128 / 16) << 24;
    constexpr uint32_t ID_O = 1u << 4 | FMT << 7 | FMT << 10 | 1u << 16 | (HD / 8) << 17 | (128 / 16) << 24;
    const uint32_t qb = __shfl_sync(0xffffffffu, smem_u32(qs), 0), rb = __shfl_sync(0xffffffffu, smem_u32(ring), 0);
    auto scores = [&](int i, int buf, uint32_t st) {  // S buffer = Q_i K^T
      const uint64_t kd = pf_desc(rb + st * TILE, 16, 1024), qd = pf_desc(qb + i * TILE, 16, 1024);
      if (!lead) return;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const uint32_t off = ((k / 4) * PANEL + (k & 3) * 32) >> 4;
        pf_mma_ss(tm + buf * 128, qd + off, kd + off, ID_S, k > 0);
      }
      pf_commit(&s_full[buf]);
    };
    auto values = [&](int i, int buf, uint32_t st, bool add, bool last) {  // o_i += P buffer V
      const uint64_t vd = pf_desc(rb + st * TILE, PANEL, 1024);
      if (!lead) return;
#pragma unroll
      for (int k = 0; k < PF_TS / 16; ++k) pf_mma_ts(tm + BUFS * 128 + i * HD, tm + buf * 128 + k * 8, vd + k * 128, ID_O, add || k > 0);
      pf_commit(&o_done[buf]);
      if (last) pf_commit(&o_last[i]);
    };
    auto free_tile = [&](uint32_t k) {
      if (lead) pf_commit(&kv_empty[k % SLOTS]);
    };
    uint32_t used = 0, units = 0;  // K and V tiles, and units, of all pieces so far
    for (int r = 0;; ++r) {
      wait_piece(&info_full[r & 1], (r >> 1) & 1);
      const PfPiece& in = info[r & 1];
      const int seq = __shfl_sync(0xffffffffu, in.seq, 0), n0 = __shfl_sync(0xffffffffu, in.n0, 0), n1 = __shfl_sync(0xffffffffu, in.n1, 0);
      const bool two = __shfl_sync(0xffffffffu, in.f_end - in.f0, 0) > 128;
      if (seq < 0) break;
      __syncwarp();
      if (lead) {
        pg_arrive(&info_empty[r & 1]);
        pg_arrive(&q_full);
      }
      wait_warp(&q_full, r & 1);
      pf_fence_after();
      const int n = two ? n0 + n1 : n0;
      int next_k = 0, next_v = 0;  // tiles of slots whose K, whose V, have been waited for
      auto tile_of = [&](int u, int& i) {  // warpgroup and tile of slots of unit u
        i = two && u >= 2 * n0 ? 1 : u & 1;
        return !two ? u : u < 2 * n0 ? u >> 1 : u - n0;
      };
      auto start = [&](int u) {  // S of unit u
        int i;
        const int j = tile_of(u, i);
        const uint32_t k = used + 2 * j;
        if (j >= next_k) {
          wait_warp(&kv_full[k % SLOTS], (k / SLOTS) & 1);
          pf_fence_after();
          next_k = j + 1;
        }
        scores(two ? i : 0, (units + u) % BUFS, k % SLOTS);
        if (!two || i) free_tile(k);  // the second row tile sees every tile of slots that the first does
      };
      for (int u = 0; u < min(n, BUFS); ++u) start(u);
      for (int u = 0; u < n; ++u) {
        int i;
        const int j = tile_of(u, i);
        const uint32_t g = units + u, v = used + 2 * j + 1;
        if (j >= next_v) {
          wait_warp(&kv_full[v % SLOTS], (v / SLOTS) & 1);
          next_v = j + 1;
        }
        wait_warp(&p_full[g % BUFS], (g / BUFS) & 1);
        pf_fence_after();
        values(i, g % BUFS, v % SLOTS, two ? j > 0 : u > 1, two ? j + 1 == (i ? n1 : n0) : u + 2 >= n);
        if (!two || i) free_tile(v);
        if (u + BUFS < n) start(u + BUFS);
      }
      units += n;
      used += 2 * max(n0, n1);
    }
    if (lead) pf_commit(&drained);
    mbar_wait_warp(&drained, 0);
    pf_fence_before();
  }
  cta_sync();
  pf_fence_after();
  if (warp == PF_ISSUER)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PF_TMEM) : "memory");
}

}  // namespace vp
