// Attention of the newest rows of many requests over the paged cache (vp_paged_decode), up to 16 query
// rows (heads of a group x new rows) per cache head; more go to the tensor-memory kernel.
//
// Mathematics. Per request and cache head: S = scale q K^T over the visible slots,
// p = 2^(S log2 e - m) with the running maximum m, l = sum p, o = sum p v; two such records (m, l, o)
// over disjoint slots join as m* = max, l* = sum l 2^(m - m*), o* likewise, and out = o / l. The second product's operand, p,
// is rounded to the cache's type, as the tensor cores take it: an output is then off by up to one unit of that rounding more
// than the exact result's own (l adds up the unrounded p). fp16 has nothing below 2^-24, so there m is taken DC_LIFT below the
// maximum: weights reach 2^DC_LIFT, and those lost to o are below 2^-39 of the largest, which 2^17 slots do not add up.
//
// Bound: the bytes of K and V, each read once, and for small calls the chain of dependent reads
// (length, page, K, V). So the query rows of one cache head (G heads x R rows, packed as m = r G + g)
// share one read of the cache, and the work is cut into tiles of 8 KB (32 slots of 64, 16 of 128)
// dealt out evenly: the tiles of all (request, head) pairs are numbered in order and every CTA takes
// about the same number of consecutive ones. One CTA per SM, two roles:
//  * eight consumer warps take turns over the tiles. Each has two stages of its own and refills a
//    stage itself (TMA boxes of one page each) once it has computed on it (mma.sync), so the warps never
//    wait for one another;
//  * four joiner warps bring the queries of the next pair, and at the end of a pair's run add up the
//    warps' records while the warps are on the next pair. A pair that several CTAs share leaves records
//    in the work buffer; the CTA that finishes last (a counter per first CTA, back at zero afterwards)
//    joins them in the order of the slots, so results do not depend on which CTA that is. Of many records,
//    each eight are first joined by the last CTA of those, in the buffer that the warps' records were in.
// Measured: 4 requests of 103,871 to 131,072 slots, 32 + 2 x 8 heads of 128, bf16: 270 us, 6.8 TB/s (a plain copy: 6.5;
// calls on one input leave part of it in L2; with a producer warp filling a ring for all warps: 430 us). 64 requests of
// 130 to 2,048 slots, 14 + 2 x 2 heads of 64: 12.7 us; 128 requests with a window of 1,024: 17.9 us; one request of 257
// slots: 6.7 us, of which 2.9 us pass before the first tile is asked for (lengths, shares, pages), 0.9 until it is there,
// 0.65 a tile, 0.8 for the join.
#pragma once
#include "vp_paged.cuh"

namespace vp {

constexpr int DC_WARPS = 8;                         // consumer warps
constexpr int DC_JOINERS = 128;                     // threads
constexpr int DC_THREADS = DC_WARPS * 32 + DC_JOINERS;
// Packed query rows of a pair: one MMA tile, which reads the cache at HBM speed. With more tiles a pair (this kernel for up
// to 128 rows, one 16-row tile a warp) 64 requests of 112 rows took 62 us, on the tensor-memory kernel 25.
constexpr int DC_ROWS = 16;
constexpr int DC_TILE = 4096;                       // bytes of K (and of V) per tile
constexpr int DC_STAGES = 2;                        // per warp
constexpr int DC_LENS = 2048;                       // lengths kept in shared memory
// Tiles that a run costs beside its own, in the even shares (64 requests of 130 to 2,048 slots: 12.7 us then, 14.2 without,
// 13.5 with 24; 200 of 20 to 4,000: 23.3, 36.2, 25.5; 30 of 100 to 4,000, 32 + 2 x 8 heads of 128: 32.2, 51, 35).
constexpr int DC_RUN = 12;
// Tiles of a CTA's share, at most, for whole pairs: past it the joins they save cost less than CTAs without a last pair
// (32 + 2 x 8 heads of 128, 40 requests of 2,000 slots: 57 us, 70 with whole pairs; 16 of 16,000: 160.2 and 161.5).
constexpr int DC_SHORT = 64;
// Rounds of reads (8 records, 128 items of 4 elements), at most, in which the last CTA joins a pair's records by itself;
// more records go eight at a time. 8 records of 4 rows of 128: 9.8 us a call, 10.9 by eights; 18 of them (3 rounds): 29.8
// and 31; 18 of 16 rows of 128 (12 rounds): 21.5 by eights, 25.9 otherwise; 49 of 8 rows of 128 (14): 15.7 and 22.5.
constexpr int DC_FLAT = 3;
constexpr int DC_LEVELS = 3;                        // of joins that leave a record: 8^3 parts a pair, more than CTAs

constexpr float DC_LIFT = 14.f;                     // log2 of the largest weight in fp16 (2^16 is past its range)

template <int HD>
struct DcShape {
  static constexpr int TS = DC_TILE / (HD * 2);     // slots per tile
  static constexpr int PITCH = HD + 4;              // floats per row of the join buffer
  static constexpr int QBUF = DC_ROWS * HD * 2;
  static constexpr size_t RING = (size_t)DC_WARPS * DC_STAGES * 2 * DC_TILE;
  static constexpr size_t JOIN = (size_t)DC_WARPS * DC_ROWS * PITCH * 4;
  static constexpr size_t SMEM = 1024 + RING + 2 * QBUF + JOIN + DC_WARPS * DC_ROWS * 8 + DC_LENS * 4;
};

// Floats of one record of `rows` rows: o, then (m, l) of each row; a multiple of 16 bytes.
__host__ __device__ constexpr size_t pg_record(int rows, int hd) { return ((size_t)rows * (hd + 2) + 3) / 4 * 4; }

struct DcParams {
  vp_paged c;
  vp_paged_attn a;
  float* rec;         // [grid][DC_LEVELS][2] records of M rows
  unsigned* tickets;  // [grid][DC_LEVELS][2]
  int group, M, min_tiles, page_shift;  // G, G R, fewest tiles per CTA, log2 of the page size
};

// Slots of a request that the rows of a call see, as tiles: [0, ns) hold the sinks, [ws, end) the rest.
struct DcSpan {
  int len, base, ns, ws, tiles, lo, lo_all;  // lo: no row sees a non-sink slot below it; lo_all: all rows see those at or above
};
template <int TS>
__device__ __forceinline__ DcSpan dc_span(int len, int rows, int window, int sinks) {
  DcSpan s;
  s.len = len;
  s.base = len - rows;
  s.lo = window ? max(0, s.base - window) : 0;
  s.lo_all = window ? s.base + rows - window : 0;
  const int end = (len + TS - 1) / TS;
  s.ns = window ? min((min(sinks, len) + TS - 1) / TS, end) : 0;
  s.ws = s.lo / TS;
  if (s.ws <= s.ns) s.ws = s.ns = 0;
  s.tiles = max(1, s.ns + end - s.ws);  // one for an empty request: it has zeros to write
  return s;
}

// Even shares of N tiles: the first N % G of G CTAs take one more.
struct PgShare {
  int per, more;
  __device__ __forceinline__ PgShare(int N, int G) : per(N / G), more(N % G) {}
  __device__ __forceinline__ int first(int c) const { return c * per + min(c, more); }
  __device__ __forceinline__ int owner(int t) const {
    const int big = more * (per + 1);
    return t < big ? t / (per + 1) : more + (t - big) / per;
  }
};

// Bits a .. b - 1 of a tile's 64 (all relative to its first slot).
__device__ __forceinline__ uint64_t dc_bits(int a, int b) {
  const uint64_t hi = b >= 64 ? ~0ull : b <= 0 ? 0ull : (1ull << b) - 1;
  const uint64_t lo = a >= 64 ? ~0ull : a <= 0 ? 0ull : (1ull << a) - 1;
  return hi & ~lo;
}
// Slots of a tile that a row sees: the old ones [lo, base) and the sinks, and its new ones.
__device__ __forceinline__ uint64_t dc_seen(int s0, int base, int lo, int sinks, uint32_t bits) {
  const int b = base - s0;
  const uint64_t fresh = b >= 64 ? 0ull : b >= 0 ? (uint64_t)bits << b : b > -32 ? (uint64_t)(bits >> -b) : 0ull;
  return dc_bits(lo - s0, b) | dc_bits(-s0, min(sinks - s0, b)) | fresh;
}

// Named barriers between consumers and joiners: the join buffer is filled, is free.
constexpr int DC_FILLED = 2, DC_FREE = 3;
__device__ __forceinline__ void dc_sync(int bar) {
  __syncwarp();
  asm volatile("barrier.sync %0, 384;" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void dc_arrive(int bar) {
  __syncwarp();
  asm volatile("barrier.arrive %0, 384;" ::"r"(bar) : "memory");
}
static_assert(DC_THREADS == 384, "barrier counts");

// A walk over the CTA's tiles: the request and head that tile t belongs to.
template <int TS>
struct DcWalk {
  const DcParams& p;
  const int* lens_s;
  int seq, head, u, t, t1;  // tile t is tile u of this head
  DcSpan sp;
  // at: the number of seq's first tile
  __device__ __forceinline__ DcWalk(const DcParams& p_, const int* l, int s, int at, int t_, int t1_)
      : p(p_), lens_s(l), seq(s), t(at), t1(t1_) {
    span();
    const int skip = t_ - at;  // seq has the CTA's first tile, so few requests are passed over
    head = 0;
    u = 0;
    if (skip >= sp.tiles && t_ < t1) {
      head = min(skip / sp.tiles, p.c.n_kv - 1);
      t += head * sp.tiles;
    }
    advance(t_ - t);
  }
  __device__ __forceinline__ void span() {
    const int len = seq < DC_LENS ? lens_s[seq] : pg_len(p.c, p.a.seqs, p.a.lens, seq);
    sp = dc_span<TS>(len, p.a.rows, p.a.window, p.a.sinks);
  }
  __device__ __forceinline__ bool more() const { return t < t1; }
  __device__ __forceinline__ void advance(int k) {
    t += k;
    if (t >= t1) return;
    u += k;
    while (u >= sp.tiles) {
      u -= sp.tiles;
      if (++head == p.c.n_kv) {
        head = 0;
        ++seq;
        span();
      }
    }
  }
  __device__ __forceinline__ int run() const { return min(sp.tiles - u, t1 - t); }  // tiles of this head from t on
  __device__ __forceinline__ int slot(int v) const { return (v < sp.ns ? v : sp.ws + v - sp.ns) * TS; }
};

template <typename T, int HD>
__global__ void __launch_bounds__(DC_THREADS, 1)
    k_paged_decode(const __grid_constant__ DcParams p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
  using Sh = DcShape<HD>;
  constexpr int TS = Sh::TS, NT = TS / 8, KS = HD / 16, PITCH = Sh::PITCH, QP = DC_ROWS * 128;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* qbuf = ring + Sh::RING;
  float* join = reinterpret_cast<float*>(qbuf + 2 * Sh::QBUF);
  float2* join_ml = reinterpret_cast<float2*>(join + DC_WARPS * DC_ROWS * PITCH);
  int* lens_s = reinterpret_cast<int*>(join_ml + DC_WARPS * DC_ROWS);
  __shared__ uint64_t full[DC_WARPS][DC_STAGES], q_full[2];
  __shared__ int warp_sums[DC_THREADS / 32], warp_most[DC_THREADS / 32], warp_least[DC_THREADS / 32];
  __shared__ int first_seq, first_tile, t0_s, t1_s, dead, last_flag;  // first_tile: number of first_seq's first tile
  __shared__ int gave_up[DC_WARPS];  // the first tile of a warp whose wait ran out

  const vp_paged& c = p.c;
  const vp_paged_attn& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = a.rows;

  pdl_launch_dependents();
  if (tid < DC_WARPS * DC_STAGES) mbar_init(&full[0][0] + tid, 1);
  if (tid < 2) mbar_init(&q_full[tid], DC_JOINERS);
  if (tid == 0) dead = 0;
  if (tid < DC_WARPS) gave_up[tid] = -1;
  if (tid < 32) fence_barrier_init();
  for (int i = tid; i < 2 * Sh::QBUF / 16; i += DC_THREADS) reinterpret_cast<uint4*>(qbuf)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 32) {
    pg_prefetch_map(&mk);
    pg_prefetch_map(&mv);
  }
  pdl_wait();

  // tiles of all requests: every thread counts a run of them, then a scan over the CTA
  const int chunk = (a.n + DC_THREADS - 1) / DC_THREADS;
  const int i0 = min(a.n, tid * chunk), i1 = min(a.n, i0 + chunk);
  int mine = 0, most = 0, least = 1 << 30;
  for (int i = i0; i < i1; ++i) {
    const int len = pg_len(c, a.seqs, a.lens, i);
    if (i < DC_LENS) lens_s[i] = len;
    const int tiles = dc_span<TS>(len, rows, a.window, a.sinks).tiles;
    mine += tiles * c.n_kv;
    most = max(most, tiles);
    least = min(least, tiles);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  least = __reduce_min_sync(0xffffffffu, least);
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl, warp_most[warp] = most, warp_least[warp] = least;
  cta_sync();
  int before = 0, N = 0;
#pragma unroll
  for (int w = 0; w < DC_THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    N += warp_sums[w];
    most = max(most, warp_most[w]);
    least = min(least, warp_least[w]);
  }
  // Even shares of the tiles; or, where the requests are about equally long and the shares small, whole pairs
  // (cuts == 1) or even cuts of them: a pair that ends inside a CTA's share costs a join (16 requests of 300
  // slots: 7.3 us, 10.6 with even shares; 64 of 1,000: 10.8 and 13.2; 128 with a window of 1,024: 17.9 and 19.5).
  const int cta = blockIdx.x, pairs = a.n * c.n_kv;
  int G = min((N + p.min_tiles - 1) / p.min_tiles, (int)gridDim.x), cuts = 0;
  if (4ll * most <= 5ll * least && N <= DC_SHORT * (int)gridDim.x) {
    cuts = 2 * pairs > (int)gridDim.x ? 1 : min((int)gridDim.x / pairs, (most + p.min_tiles - 1) / p.min_tiles);
    G = min((int)gridDim.x, pairs * cuts);
  }
  if (cta >= G) return;
  // A run of tiles of one pair costs about as much as DC_RUN tiles more, so shares are even in tiles and DC_RUN
  // for each pair, which stand before its tiles in this count.
  const PgShare share(cuts ? pairs : N + DC_RUN * pairs, G);  // of tiles, or of pairs
  int at = before + incl - mine;
  if (!cuts) {
    const int v0 = share.first(cta), v1 = share.first(cta + 1);
    if (tid == 0 && cta + 1 == G) t1_s = N;
    __syncwarp();
    for (int i = i0, v = at + DC_RUN * c.n_kv * i0; i < i1; ++i) {
      const int len = i < DC_LENS ? lens_s[i] : pg_len(c, a.seqs, a.lens, i);
      const int tiles = dc_span<TS>(len, rows, a.window, a.sinks).tiles, width = tiles + DC_RUN, end = v + width * c.n_kv;
      auto tile_at = [&](int x) {  // tiles before place x of the count
        const int h = (x - v) / width;
        return at + h * tiles + max(0, x - v - h * width - DC_RUN);
      };
      if (v <= v0 && v0 < end) {
        first_seq = i;
        first_tile = at;
        t0_s = tile_at(v0);
      }
      if (v <= v1 && v1 < end) t1_s = tile_at(v1);
      at += tiles * c.n_kv;
      v = end;
    }
  } else {
    const int q0 = cuts == 1 ? share.first(cta) : cta / cuts, q1 = cuts == 1 ? share.first(cta + 1) : q0 + 1;
    const int s0 = q0 / c.n_kv, s1 = q1 / c.n_kv;  // their requests
    if (cuts == 1 && tid == 0 && s1 == a.n) t1_s = N;
    __syncwarp();
    for (int i = i0; i < i1; ++i) {
      const int len = i < DC_LENS ? lens_s[i] : pg_len(c, a.seqs, a.lens, i);
      const int tiles = dc_span<TS>(len, rows, a.window, a.sinks).tiles;
      if (i == s0) {
        const int t = at + (q0 - s0 * c.n_kv) * tiles, k = cuts == 1 ? 0 : cta - q0 * cuts;
        first_seq = i;
        first_tile = at;
        t0_s = t + k * tiles / cuts;
        if (cuts > 1) t1_s = t + (k + 1) * tiles / cuts;
      }
      if (cuts == 1 && i == s1) t1_s = at + (q1 - s1 * c.n_kv) * tiles;
      at += tiles * c.n_kv;
    }
  }
  cta_sync();
  const int t0 = t0_s, t1 = t1_s;
  if (t0 == t1) return;

  // Waits of a whole warp: whether the phase is complete. After one that ran out none waits any more, and the call ends with an
  // error status; everybody goes on to the end, as the roles meet at named barriers that want all of them.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    __syncwarp();
    const bool there = pg_wait(bar, parity, &dead);
    if (!there) {
      pg_status(c.status, VP_DEV_ERR_TIMEOUT);
      *(volatile int*)&dead = 1;
    }
    __syncwarp();
    return there;
  };

  if (warp < DC_WARPS) {
    // ---- consumers: warp w has tiles t0 + w, t0 + w + 8, ... ----
    const int g = lane >> 2, q4 = lane & 3;
    const float cexp = a.scale * 1.4426950408889634f;
    const uint32_t stage0 = smem_u32(ring) + warp * DC_STAGES * 2 * DC_TILE;
    // Loads run ahead of the computation. A tile is looked up (lane b < boxes: the page of box b) well
    // before it is fetched, so that the table's answer is there.
    const int box = min(c.page_size, TS), boxes = TS / box;
    struct Tile {
      int page, slot, head;
      bool any, seen;
    };
    DcWalk<TS> ahead(p, lens_s, first_seq, first_tile, t0 + warp, t1);
    auto look = [&] {
      Tile x;
      x.any = ahead.more();
      x.page = c.n_pages;  // a box that nobody sees fills zeros
      x.slot = ahead.slot(ahead.u) + lane * box;
      x.head = ahead.head;
      x.seen = x.any && lane < boxes && x.slot < ahead.sp.len && (x.slot + box > ahead.sp.lo || x.slot < a.sinks);
      if (x.seen) {
        const int s = a.seqs ? a.seqs[ahead.seq] : ahead.seq;  // a request outside the table has no slots
        x.page = c.table[s * c.table_stride + (x.slot >> p.page_shift)];
      }
      ahead.advance(DC_WARPS);
      return x;
    };
    auto fetch = [&](const Tile& x, int st) {
      if (!x.any) return;
      if (lane == 0) mbar_arrive_expect_tx(&full[warp][st], 2 * DC_TILE);
      __syncwarp();
      if (lane < boxes) {
        int page = x.page;
        if (x.seen && (page < 0 || page >= c.n_pages)) {
          pg_status(c.status, VP_DEV_ERR_PAGE);
          page = c.n_pages;
        }
        unsigned char* dst = ring + (size_t)((warp * DC_STAGES + st) * 2) * DC_TILE + lane * box * 128;
        pg_box5(dst, &mk, x.slot & (c.page_size - 1), x.head, page, &full[warp][st]);
        pg_box5(dst + DC_TILE, &mv, x.slot & (c.page_size - 1), x.head, page, &full[warp][st]);
      }
    };
    Tile coming;
    {
      const Tile x = look(), y = look();
      fetch(x, 0);
      fetch(y, 1);
      coming = look();
    }
    static_assert(DC_STAGES == 2, "first tiles");
    const int row_of[2] = {g / p.group, (g + 8) / p.group};
    const bool plain = rows == 1 && !a.mask;  // one row that sees all up to its own slot
    uint32_t k_th = 0;  // tiles computed
    int next = t0 + warp;
    DcWalk<TS> w(p, lens_s, first_seq, first_tile, t0, t1);
    for (int r = 0; w.more(); ++r) {
      const DcSpan& sp = w.sp;
      const int n = w.run(), seq = w.seq;
      // masks of the request's rows (lane i: row i); this thread's two rows, and their union
      uint32_t bits[2] = {1, 1}, any = 1;
      int lo[2];  // first old slot beside the sinks that the row sees
      int least = 1;
      const bool there[2] = {g < p.M && sp.base + row_of[0] >= 0, g + 8 < p.M && sp.base + row_of[1] >= 0};
      if (plain) {
        lo[0] = lo[1] = a.window ? sp.base + 1 - a.window : 0;
      } else {
        uint32_t anc = 0;
        if (lane < rows)
          anc = a.mask ? (uint32_t)a.mask[(long long)seq * rows + lane] & ((1u << rows) - 1) : (2u << lane) - 1;
        least = __reduce_min_sync(0xffffffffu, lane < rows ? __popc(anc) : 32);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          bits[h] = __shfl_sync(0xffffffffu, anc, min(row_of[h], 31));
          lo[h] = a.window ? sp.base + __popc(bits[h]) - a.window : 0;
        }
        if (a.window) {  // new slots that have left a row's window
          uint32_t keep[2] = {0, 0};
          for (int j = 0; j < rows; ++j) {
            const int place = sp.base + __popc(__shfl_sync(0xffffffffu, anc, j)) - 1;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (place >= lo[h] || place < a.sinks) keep[h] |= 1u << j;
          }
          bits[0] &= keep[0];
          bits[1] &= keep[1];
        }
        any = __reduce_or_sync(0xffffffffu, (there[0] ? bits[0] : 0u) | (there[1] ? bits[1] : 0u));
      }
      const int first_seen = a.window ? sp.base + least - a.window : 0;  // beside the sinks, by any row
      uint32_t qf[KS][4];
      wait(&q_full[r & 1], (r >> 1) & 1);
      {
        const int m = lane & 15;
        const uint32_t qa = smem_u32(qbuf) + (r & 1) * Sh::QBUF + m * 128;
#pragma unroll
        for (int k = 0; k < KS; ++k) pg_ldsm(qf[k], qa + (k / 4) * QP + ((((k & 3) * 2 + (lane >> 4)) ^ (m & 7)) << 4));
      }
      float o[HD / 8][4] = {};
      float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
      for (; next < w.t + n; next += DC_WARPS, ++k_th) {
        const int st = k_th % DC_STAGES, s0 = w.slot(w.u + next - w.t);
        if (!wait(&full[warp][st], (k_th / DC_STAGES) & 1)) {
          if (lane == 0 && gave_up[warp] < 0) gave_up[warp] = k_th;
          coming.any = false;  // nothing is asked for any more: a stage whose copy was not waited for is not refilled
          ahead.t = t1;
        }
        const uint32_t kb = stage0 + st * 2 * DC_TILE, vb = kb + DC_TILE;
        float s[NT][4], s2[NT][4];
        // lanes 0-7 .. 24-31 point at the lines of four 8 x 8 matrices: 8 slots, 32 elements; two sums
        // side by side halve the chain of dependent products
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
          const int line = nt * 8 + (lane & 7);
#pragma unroll
          for (int k = 0; k < KS; k += 2) {
            uint32_t f[4];
            pg_ldsm(f, kb + (k / 4) * TS * 128 + line * 128 + ((((k & 3) * 2 + (lane >> 3)) ^ (line & 7)) << 4));
            PgType<T>::mma(s[nt], qf[k], f[0], f[1]);
            PgType<T>::mma(s2[nt], qf[k + 1], f[2], f[3]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] += s2[nt][e];
        }
        const bool whole = s0 + TS <= sp.base && (s0 >= sp.lo_all || s0 + TS <= a.sinks);
        if (!whole) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t see = there[h] ? (uint32_t)dc_seen(s0, sp.base, lo[h], a.sinks, bits[h]) >> (2 * q4) : 0u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (!((see >> (nt * 8 + e)) & 1)) s[nt][2 * h + e] = -INFINITY;
          }
        }
        float mn[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mn[0] = fmaxf(mn[0], fmaxf(s[nt][0], s[nt][1]));
          mn[1] = fmaxf(mn[1], fmaxf(s[nt][2], s[nt][3]));
        }
        float use[2], f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mn[h] = fmaxf(mn[h], __shfl_xor_sync(0xffffffffu, mn[h], 1));
          mn[h] = fmaxf(mn[h], __shfl_xor_sync(0xffffffffu, mn[h], 2));
          mn[h] = fmaxf(mx[h], fmaf(mn[h], cexp, PgType<T>::BF16 ? 0.f : -DC_LIFT));
          use[h] = mn[h] == -INFINITY ? 0.f : mn[h];
          f[h] = pg_exp2(mx[h] - use[h]);
          mx[h] = mn[h];
          sum[h] *= f[h];
        }
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) {
          o[d][0] *= f[0], o[d][1] *= f[0];
          o[d][2] *= f[1], o[d][3] *= f[1];
        }
        uint32_t pf[TS / 16][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) e[i] = pg_exp2(fmaf(s[nt][i], cexp, -use[i >> 1]));
          sum[0] += e[0] + e[1];
          sum[1] += e[2] + e[3];
          pf[nt / 2][(nt & 1) * 2] = PgType<T>::down(e[0], e[1]);
          pf[nt / 2][(nt & 1) * 2 + 1] = PgType<T>::down(e[2], e[3]);
        }
        // values of slots that no row sees may be NaN, which a zero weight does not silence
        const uint32_t live = whole ? ~0u : (uint32_t)dc_seen(s0, sp.base, first_seen, a.sinks, any) >> (2 * q4);
#pragma unroll
        for (int kk = 0; kk < TS / 16; ++kk) {
          uint32_t w0 = 0xffffffffu, w1 = 0xffffffffu;
          if (!whole) {
            const uint32_t x = live >> (kk * 16);
            w0 = (x & 1 ? 0xffffu : 0u) | (x & 2 ? 0xffff0000u : 0u);
            w1 = (x & 0x100 ? 0xffffu : 0u) | (x & 0x200 ? 0xffff0000u : 0u);
          }
          const int line = kk * 16 + (lane & 15);
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            uint32_t f4[4];
            pg_ldsm_t(f4, vb + (d / 4) * TS * 128 + line * 128 + ((((d & 3) * 2 + (lane >> 4)) ^ (line & 7)) << 4));
            PgType<T>::mma(o[2 * d], pf[kk], f4[0] & w0, f4[1] & w1);
            PgType<T>::mma(o[2 * d + 1], pf[kk], f4[2] & w0, f4[3] & w1);
          }
        }
        __syncwarp();
        fetch(coming, st);
        coming = look();
      }
      if (r > 0) dc_sync(DC_FREE);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        if (g + 8 * h < p.M) {
          const int m = warp * DC_ROWS + g + 8 * h;
#pragma unroll
          for (int d = 0; d < HD / 8; ++d)
            *reinterpret_cast<float2*>(join + m * PITCH + d * 8 + 2 * q4) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
          if (q4 == 0) join_ml[m] = make_float2(mx[h], sum[h]);
        }
      }
      dc_arrive(DC_FILLED);
      w.advance(n);
    }
    // copies still in flight land before the CTA may end (they have, unless a wait ran out)
    __syncwarp();
    const int left = gave_up[warp];
    if (left >= 0)
      for (int k = left; k < left + DC_STAGES && t0 + warp + k * DC_WARPS < t1; ++k) mbar_wait_warp(&full[warp][k % DC_STAGES], (k / DC_STAGES) & 1);
    return;
  }

  // ---- joiners ----
  const int jt = tid - DC_WARPS * 32;
  const size_t rec_floats = pg_record(p.M, HD);
  auto queries = [&](int seq, int head, int r) {
    unsigned char* qd = qbuf + (r & 1) * Sh::QBUF;
    for (int x = jt; x < p.M * (HD / 8); x += DC_JOINERS) {
      const int m = x / (HD / 8), ch = x % (HD / 8);
      const T* q = static_cast<const T*>(a.q) + seq * a.q_seq + m / p.group * a.q_row + (head * p.group + m % p.group) * a.q_head;
      pg_cp16(qd + (ch / 8) * QP + m * 128 + (((ch & 7) ^ (m & 7)) << 4), q + ch * 8);
    }
    pg_cp_arrive(&q_full[r & 1]);
  };
  auto put = [&](int seq, int head, int m, int d, float top, float l, const float4& acc) {
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    const int row = m / p.group, h = head * p.group + m % p.group;
    T* out = static_cast<T*>(a.out) + seq * a.out_seq + row * a.out_row + h * a.out_head + d;
    uint2 v;
    v.x = PgType<T>::down(acc.x * inv, acc.y * inv);
    v.y = PgType<T>::down(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(out) = v;
    if (a.lse && d == 0) a.lse[((long long)seq * rows + row) * a.n_q + h] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
  };
  // Records of a CTA's part of a pair (level 0), and of the parts from it on that were joined first and second. A CTA has at most one pair that begins
  // in it and ends elsewhere, and one that began elsewhere.
  auto record = [&](int cc, bool begins, int level) { return p.rec + (size_t)(2 * DC_LEVELS * cc + 2 * level + begins) * rec_floats; };
  // Whether this CTA is the last of n whose records are out; the counter is back at zero then. The barriers carry the
  // order of one thread's atomic to the others' records.
  auto last = [&](unsigned* ticket, int n) {
    __syncwarp();
    asm volatile("barrier.sync 1, 128;" ::: "memory");
    if (jt == 0) {
      unsigned before;
      asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
      last_flag = before == (unsigned)(n - 1);
      if (last_flag) *ticket = 0;
    }
    __syncwarp();
    asm volatile("barrier.sync 1, 128;" ::: "memory");
    return last_flag != 0;
  };
  DcWalk<TS> w(p, lens_s, first_seq, first_tile, t0, t1);
  queries(w.seq, w.head, 0);
  bool more = true;
  for (int r = 0; more; ++r) {
    const int seq = w.seq, head = w.head, u0 = w.u, n = w.run(), tiles = w.sp.tiles, pair_at = w.t - w.u;
    const bool alone = n == tiles;
    w.advance(n);
    more = w.more();
    if (more) queries(w.seq, w.head, r + 1);  // the warps are done with the queries of run r - 1
    const int pair = seq * c.n_kv + head, place = pair_at + DC_RUN * (pair + 1);  // of the pair's first tile
    const int c0 = alone ? cta : cuts ? pair * cuts : share.owner(place);
    const int c1 = alone ? cta : cuts ? c0 + cuts - 1 : share.owner(place + tiles - 1);
    dc_sync(DC_FILLED);
    // Joins the first n records of the buffer; item: row m, 4 elements.
    auto joined = [&](int n_rec, float* rec) {
      for (int it = jt; it < p.M * (HD / 4); it += DC_JOINERS) {
        const int m = it / (HD / 4), d = it % (HD / 4) * 4;
        float2 ml[DC_WARPS];
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < DC_WARPS; ++k) {
          ml[k] = k < n_rec ? join_ml[k * DC_ROWS + m] : make_float2(-INFINITY, 0.f);
          top = fmaxf(top, ml[k].x);
        }
        const float use = top == -INFINITY ? 0.f : top;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int k = 0; k < DC_WARPS; ++k) {
          if (k >= n_rec) continue;
          const float f = pg_exp2(ml[k].x - use);
          const float4 v = *reinterpret_cast<const float4*>(join + (k * DC_ROWS + m) * PITCH + d);
          l += ml[k].y * f;
          acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
        }
        if (!rec) {
          put(seq, head, m, d, top, l, acc);
        } else {
          *reinterpret_cast<float4*>(rec + (size_t)m * HD + d) = acc;
          if (d == 0) *reinterpret_cast<float2*>(rec + (size_t)p.M * HD + 2 * m) = make_float2(top, l);
        }
      }
    };
    joined(DC_WARPS, alone ? nullptr : record(cta, u0 == 0, 0));
    const int parts = c1 - c0 + 1;
    if (alone || (parts + 7) / 8 * ((p.M * (HD / 4) + DC_JOINERS - 1) / DC_JOINERS) <= DC_FLAT) {
      if (more) dc_arrive(DC_FREE);  // the warps come for it before each further run
      if (alone || !last(&p.tickets[2 * DC_LEVELS * c0 + 1], parts)) continue;
#pragma unroll 1
      for (int it = jt; it < p.M * (HD / 4); it += DC_JOINERS) {
        const int m = it / (HD / 4), d = it % (HD / 4) * 4;
        float top = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int k0 = 0; k0 < parts; k0 += 8) {  // 8 records at a time: their reads fly together
          float2 ml[8];
          float4 v8[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int kk = min(k0 + k, parts - 1);
            const float* x = record(c0 + kk, kk == 0, 0);
            ml[k] = __ldcg(reinterpret_cast<const float2*>(x + (size_t)p.M * HD + 2 * m));
            v8[k] = __ldcg(reinterpret_cast<const float4*>(x + (size_t)m * HD + d));
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (k0 + k >= parts) continue;
            const float nt = fmaxf(top, ml[k].x), use = nt == -INFINITY ? 0.f : nt;
            const float fo = pg_exp2(top - use), fn = pg_exp2(ml[k].x - use);
            l = l * fo + ml[k].y * fn;
            acc.x = acc.x * fo + v8[k].x * fn, acc.y = acc.y * fo + v8[k].y * fn;
            acc.z = acc.z * fo + v8[k].z * fn, acc.w = acc.w * fo + v8[k].w * fn;
            top = nt;
          }
        }
        put(seq, head, m, d, top, l, acc);
      }
      continue;
    }
    // 8 parts at a time through the buffer, then 8 times 8, and all; each time in the last CTA of those that add to it
    for (int level = 0, span = 1;; ++level) {
      const int from = c0 + (cta - c0) / (8 * span) * (8 * span);
      const int n_rec = (min(8 * span, c1 + 1 - from) + span - 1) / span;
      if (!last(&p.tickets[2 * DC_LEVELS * from + 2 * level + (from == c0)], n_rec)) break;
#pragma unroll 1
      for (int k = 0; k < n_rec; ++k) {
        const float* x = record(from + k * span, from == c0 && k == 0, level);
        for (int it = jt; it < p.M * (HD / 4); it += DC_JOINERS)
          pg_cp16(join + (k * DC_ROWS + it / (HD / 4)) * PITCH + it % (HD / 4) * 4, x + it * 4);
        if (2 * jt < p.M) pg_cp16(join_ml + k * DC_ROWS + 2 * jt, x + p.M * HD + 4 * jt);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      asm volatile("barrier.sync 1, 128;" ::: "memory");
      span *= 8;
      const bool all = from == c0 && from + span > c1;
      joined(n_rec, all ? nullptr : record(from, from == c0, level + 1));
      if (all) break;
    }
    if (more) dc_arrive(DC_FREE);
  }
}

}  // namespace vp
