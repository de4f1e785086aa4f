// Attention of the newest rows of many requests over the paged cache (vp_paged_decode).
//
// Mathematics. Per request, cache head and block of query rows: S = scale q K^T over the visible slots,
// p = 2^(S log2 e - m) with the running maximum m, l = sum p, o = sum p v; two such records (m, l, o)
// over disjoint slots join as m* = max, l* = sum l 2^(m - m*), o* likewise, and out = o / l.
//
// Bound: the bytes of K and V, each read once. So the query rows of one cache head (G heads x R
// rows, packed as m = r G + g, up to 128 per block) share one read of the cache, and the work is cut
// into tiles of 16 KB (64 slots of 64, 32 of 128) dealt out evenly: the tiles of all (request, row
// block, head) pairs are numbered in order, and CTA c of G' takes tiles [c N / G', (c + 1) N / G').
// One CTA per SM: a producer warp keeps a ring of tiles in flight (TMA boxes of one page each), eight
// consumer warps compute on mma.sync. MT warps hold the 16-row tiles of the block; the 8 / MT groups of
// them take turns over the tiles, so that no CTA barrier stands in the loop: a warp waits for its
// tile, computes and frees it. At the end of a pair's run the groups join in shared memory. A pair
// that several CTAs share leaves records in the work buffer; the CTA that finishes last (a counter
// per first CTA, back at zero afterwards) joins them in the order of the slots, so results do not
// depend on which CTA that is.
#pragma once
#include "vp_paged.cuh"

namespace vp {

constexpr int DC_WARPS = 8;                         // consumer warps
constexpr int DC_THREADS = (DC_WARPS + 1) * 32;     // and the producer
constexpr int DC_BLOCK_ROWS = DC_WARPS * 16;        // packed query rows per block
constexpr int DC_TILE = 8192;                       // bytes of K (and of V) per tile
constexpr int DC_LENS = 2048;                       // lengths kept in shared memory

template <int HD>
struct DcShape {
  static constexpr int TS = DC_TILE / (HD * 2);     // slots per tile
  static constexpr int PITCH = HD + 4;              // floats per row of the join buffer
  // a multiple of every number of groups (8, 4, 2, 1): a stage then always goes to the same group,
  // whose warps saw its previous tile. A warp that came to a stage whose previous tile, another
  // group's, is still on its way would take that phase's parity for its own.
  static constexpr int STAGES = DC_WARPS;
  static constexpr size_t RING = (size_t)STAGES * 2 * DC_TILE;
  static constexpr size_t JOIN = (size_t)DC_BLOCK_ROWS * PITCH * 4;
  static constexpr size_t SMEM = 1024 + RING + JOIN + DC_BLOCK_ROWS * 8 + DC_LENS * 4;
  // floats of one record: DC_BLOCK_ROWS rows at most, o then m then l; a multiple of 16 bytes
  static __host__ __device__ constexpr size_t record(int rows) { return ((size_t)rows * (HD + 2) + 3) / 4 * 4; }
};

struct DcParams {
  vp_paged c;
  vp_paged_attn a;
  float* rec;         // [grid][2] records of min(M, 128) rows
  unsigned* tickets;  // [grid]
  int group, blocks, block_rows, mt, min_tiles;  // G, row blocks per pair, rows of a full block, 16-row tiles of one, tiles per CTA
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

__device__ __forceinline__ void dc_bar() {  // the consumer warps
  __syncwarp();
  asm volatile("barrier.sync 1, 256;" ::: "memory");
}

template <typename T, int HD>
__global__ void __launch_bounds__(DC_THREADS, 1)
    k_paged_decode(const __grid_constant__ DcParams p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
  using Sh = DcShape<HD>;
  constexpr int TS = Sh::TS, ST = Sh::STAGES, NT = TS / 8, KS = HD / 16, PITCH = Sh::PITCH;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float* join = reinterpret_cast<float*>(ring + Sh::RING);
  float2* join_ml = reinterpret_cast<float2*>(join + DC_BLOCK_ROWS * PITCH);
  int* lens_s = reinterpret_cast<int*>(join_ml + DC_BLOCK_ROWS);
  __shared__ uint64_t full[ST], empty[ST];
  __shared__ long long warp_sums[DC_THREADS / 32];
  __shared__ int first_seq, dead, last_flag;
  __shared__ long long first_tile;  // number of first_seq's first tile

  const vp_paged& c = p.c;
  const vp_paged_attn& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = a.rows, per_seq = c.n_kv * p.blocks;  // pairs per request

  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], p.mt);
    }
    fence_barrier_init();
    dead = 0;
  }
  // tiles of all requests: every thread counts a run of them, then a scan over the CTA
  const int run = (a.n + DC_THREADS - 1) / DC_THREADS;
  const int i0 = min(a.n, tid * run), i1 = min(a.n, i0 + run);
  long long mine = 0;
  for (int i = i0; i < i1; ++i) {
    const int len = pg_seq(c, a.seqs, a.lens, i).len;
    if (i < DC_LENS) lens_s[i] = len;
    mine += (long long)dc_span<TS>(len, rows, a.window, a.sinks).tiles * per_seq;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sums[warp] = incl;
  cta_sync();
  long long before = 0, N = 0;
#pragma unroll
  for (int w = 0; w < DC_THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    N += warp_sums[w];
  }
  const long long want = (N + p.min_tiles - 1) / p.min_tiles;
  const int G = (int)(want < (long long)gridDim.x ? want : (long long)gridDim.x);
  const int cta = blockIdx.x;
  if (cta >= G) return;
  const long long t0 = cta * N / G, t1 = (cta + 1) * N / G;
  long long at = before + incl - mine;
  if (at <= t0 && t0 < at + mine) {
    for (int i = i0; i < i1; ++i) {
      const int len = i < DC_LENS ? lens_s[i] : pg_seq(c, a.seqs, a.lens, i).len;
      const long long n = (long long)dc_span<TS>(len, rows, a.window, a.sinks).tiles * per_seq;
      if (t0 < at + n) {
        first_seq = i;
        first_tile = at;
        break;
      }
      at += n;
    }
  }
  cta_sync();

  // the CTA's runs: (request, pair, tiles [u0, u1) of the pair), the same walk in every warp
  int seq = first_seq;
  long long seq_at = first_tile, t = t0;
  const int box = min(c.page_size, TS), boxes = TS / box;

  if (warp == DC_WARPS) {  // producer
    const int per_batch = 32 / boxes;
    uint32_t n_issued = 0;
    bool ok = true;
    while (t < t1 && ok) {
      const PgSeq s = pg_seq(c, a.seqs, a.lens, seq);
      const DcSpan sp = dc_span<TS>(s.len, rows, a.window, a.sinks);
      const long long end = seq_at + (long long)sp.tiles * per_seq;
      while (t < t1 && t < end && ok) {
        const int pair = (int)((t - seq_at) / sp.tiles), u0 = (int)((t - seq_at) % sp.tiles);
        const int n = (int)min((long long)(sp.tiles - u0), t1 - t);
        const int head = pair % c.n_kv;
        for (int b = 0; b < n && ok; b += per_batch) {
          // lane: tile b + lane / boxes of the run, box lane % boxes
          const int u = u0 + b + lane / boxes;
          const int slot = (u < sp.ns ? u : sp.ws + u - sp.ns) * TS + (lane % boxes) * box;
          int page = c.n_pages;  // a box that nobody sees fills zeros
          if (b + lane / boxes < n && slot < s.len && (slot + box > sp.lo || slot < a.sinks)) {
            page = s.pages[slot / c.page_size];
            if (page < 0 || page >= c.n_pages) {
              pg_status(c.status, VP_DEV_ERR_PAGE);
              page = c.n_pages;
            }
          }
          const int m = min(per_batch, n - b);
          for (int k = 0; k < m; ++k) {
            const int st = n_issued % ST;
            if (n_issued >= ST && !mbar_wait_warp(&empty[st], (n_issued / ST - 1) & 1)) {
              pg_status(c.status, VP_DEV_ERR_TIMEOUT);
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * DC_TILE);
            __syncwarp();
            if (lane / boxes == k) {
              unsigned char* dst = ring + (size_t)st * 2 * DC_TILE + (lane % boxes) * box * 128;
#pragma unroll
              for (int d = 0; d < HD / 64; ++d) {
                pg_box(dst + d * TS * 128, &mk, d * 64, slot % c.page_size, head, page, &full[st]);
                pg_box(dst + DC_TILE + d * TS * 128, &mv, d * 64, slot % c.page_size, head, page, &full[st]);
              }
            }
            ++n_issued;
          }
        }
        t += n;
      }
      seq_at = end;
      ++seq;
    }
    return;
  }

  // consumers
  const int mt = warp % p.mt, ks = warp / p.mt, groups = DC_WARPS / p.mt;
  const bool active = ks < groups;
  const int g = lane >> 2, q4 = lane & 3;
  const float cexp = a.scale * 1.4426950408889634f;
  uint32_t n_seen = 0;  // tiles of the CTA so far
  while (t < t1) {
    const int len = seq < DC_LENS ? lens_s[seq] : pg_seq(c, a.seqs, a.lens, seq).len;
    const DcSpan sp = dc_span<TS>(len, rows, a.window, a.sinks);
    const long long end = seq_at + (long long)sp.tiles * per_seq;
    while (t < t1 && t < end) {
      const int pair = (int)((t - seq_at) / sp.tiles), u0 = (int)((t - seq_at) % sp.tiles);
      const int n = (int)min((long long)(sp.tiles - u0), t1 - t);
      const int head = pair % c.n_kv, m0 = pair / c.n_kv * DC_BLOCK_ROWS;
      const int M = min(rows * p.group - m0, DC_BLOCK_ROWS);
      // masks of the request's rows (lane r: row r), this thread's two rows
      uint32_t anc = 0;
      if (lane < rows)
        anc = a.mask ? (uint32_t)a.mask[(long long)seq * rows + lane] & ((1u << rows) - 1) : (2u << lane) - 1;
      uint32_t any = anc;
      int least = lane < rows ? __popc(anc) : 32;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        any |= __shfl_xor_sync(0xffffffffu, any, o);
        least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      }
      const int first_seen = a.window ? sp.base + least - a.window : 0;  // beside the sinks, by any row
      uint32_t qf[KS][4];
      uint32_t bits[2];
      bool there[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int m = mt * 16 + g + 8 * h, r = (m0 + m) / p.group;
        there[h] = m < M && sp.base + r >= 0;
        bits[h] = __shfl_sync(0xffffffffu, anc, min(r, 31));
        const T* q = static_cast<const T*>(a.q) + seq * a.q_seq + r * a.q_row + (head * p.group + (m0 + m) % p.group) * a.q_head;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          qf[k][h] = m < M ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * q4) : 0u;
          qf[k][2 + h] = m < M ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 8 + 2 * q4) : 0u;
        }
      }
      float o[HD / 8][4] = {};
      float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
      if (active) {
        for (int b = (ks + groups - (int)(n_seen % groups)) % groups; b < n; b += groups) {
          const uint32_t k_th = n_seen + b;
          const int st = k_th % ST, u = u0 + b;
          const int s0 = (u < sp.ns ? u : sp.ws + u - sp.ns) * TS;
          __syncwarp();
          if (!*(volatile int*)&dead && !mbar_wait_warp(&full[st], (k_th / ST) & 1)) {
            pg_status(c.status, VP_DEV_ERR_TIMEOUT);
            *(volatile int*)&dead = 1;
          }
          __syncwarp();
          const uint32_t kb = smem_u32(ring) + st * 2 * DC_TILE, vb = kb + DC_TILE;
          float s[NT][4];
          // lanes 0-7 .. 24-31 point at the lines of four 8 x 8 matrices: 8 slots, 32 elements
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
            const int line = nt * 8 + (lane & 7);
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
              uint32_t f[4];
              pg_ldsm(f, kb + (k / 4) * TS * 128 + line * 128 + ((((k & 3) * 2 + (lane >> 3)) ^ (line & 7)) << 4));
              PgType<T>::mma(s[nt], qf[k], f[0], f[1]);
              PgType<T>::mma(s[nt], qf[k + 1], f[2], f[3]);
            }
          }
          const bool whole = s0 + TS <= sp.base && (s0 >= sp.lo_all || s0 + TS <= a.sinks);
          if (!whole) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int slot = s0 + nt * 8 + 2 * q4 + (e & 1), h = e >> 1;
                bool see = there[h] && slot < len;
                int place = slot;
                const int j = slot - sp.base;
                const uint32_t aj = __shfl_sync(0xffffffffu, anc, j & 15);
                if (j >= 0) {
                  see = see && ((bits[h] >> (j & 31)) & 1);
                  place = sp.base + __popc(aj) - 1;
                }
                if (a.window) see = see && (sp.base + __popc(bits[h]) - 1 - place < a.window || place < a.sinks);
                if (!see) s[nt][e] = -INFINITY;
              }
          }
          float mn[2] = {mx[0], mx[1]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mn[0] = fmaxf(mn[0], fmaxf(s[nt][0], s[nt][1]) * cexp);
            mn[1] = fmaxf(mn[1], fmaxf(s[nt][2], s[nt][3]) * cexp);
          }
          float use[2], f[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mn[h] = fmaxf(mn[h], __shfl_xor_sync(0xffffffffu, mn[h], 1));
            mn[h] = fmaxf(mn[h], __shfl_xor_sync(0xffffffffu, mn[h], 2));
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
#pragma unroll
          for (int kk = 0; kk < TS / 16; ++kk) {
            uint32_t w0 = 0xffffffffu, w1 = 0xffffffffu;
            if (!whole) {  // values of slots that no row sees may be NaN: a zero weight does not silence those
              w0 = w1 = 0;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int slot = s0 + kk * 16 + 2 * q4 + (e & 1) + (e >> 1) * 8;
                const bool live = slot < len && (slot >= first_seen || slot < a.sinks) &&
                                  (slot < sp.base || ((any >> ((slot - sp.base) & 31)) & 1));
                if (live) (e >> 1 ? w1 : w0) |= e & 1 ? 0xffff0000u : 0xffffu;
              }
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
          if (lane == 0) pg_arrive(&empty[st]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
          sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
          const int m = warp * 16 + g + 8 * h;
#pragma unroll
          for (int d = 0; d < HD / 8; ++d)
            *reinterpret_cast<float2*>(join + m * PITCH + d * 8 + 2 * q4) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
          if (q4 == 0) join_ml[m] = make_float2(mx[h], sum[h]);
        }
      }
      n_seen += n;
      dc_bar();

      // join the groups: item (row m of the block, 4 elements); group k's rows lie p.mt * 16 further on
      const bool alone = n == sp.tiles;
      const long long pair_at = seq_at + (long long)pair * sp.tiles;
      const int c0 = (int)(((pair_at + 1) * G - 1) / N), c1 = (int)(((pair_at + sp.tiles) * G - 1) / N);
      const size_t rec_floats = Sh::record(p.block_rows);
      float* rec = p.rec + (size_t)(u0 == 0 ? 2 * cta + 1 : 2 * cta) * rec_floats;
      auto finish = [&](bool to_out) {
        for (int it = tid; it < M * (HD / 4); it += DC_WARPS * 32) {
          const int m = it / (HD / 4), d = it % (HD / 4) * 4;
          float top = -INFINITY;
          for (int k = 0; k < groups; ++k) top = fmaxf(top, join_ml[k * p.mt * 16 + m].x);
          const float use = top == -INFINITY ? 0.f : top;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float l = 0.f;
          for (int k = 0; k < groups; ++k) {
            const int mm = k * p.mt * 16 + m;
            const float2 ml = join_ml[mm];
            const float w = pg_exp2(ml.x - use);
            const float4 v = *reinterpret_cast<const float4*>(join + mm * PITCH + d);
            l += ml.y * w;
            acc.x += v.x * w, acc.y += v.y * w, acc.z += v.z * w, acc.w += v.w * w;
          }
          if (!to_out) {
            *reinterpret_cast<float4*>(rec + (size_t)m * HD + d) = acc;
            if (d == 0) {
              rec[(size_t)p.block_rows * HD + m] = top;
              rec[(size_t)p.block_rows * (HD + 1) + m] = l;
            }
            continue;
          }
          const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
          const int r = (m0 + m) / p.group, h = head * p.group + (m0 + m) % p.group;
          T* out = static_cast<T*>(a.out) + seq * a.out_seq + r * a.out_row + h * a.out_head + d;
          uint2 w2;
          w2.x = PgType<T>::down(acc.x * inv, acc.y * inv);
          w2.y = PgType<T>::down(acc.z * inv, acc.w * inv);
          *reinterpret_cast<uint2*>(out) = w2;
          if (a.lse && d == 0)
            a.lse[((long long)seq * rows + r) * a.n_q + h] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
        }
      };
      finish(alone);
      if (!alone) {
        __threadfence();
        dc_bar();
        if (tid == 0) last_flag = atomicAdd(&p.tickets[c0], 1u) == (unsigned)(c1 - c0);
        dc_bar();
        if (last_flag) {  // all records of the pair are there: each group joins every groups-th of them
          __threadfence();
          if (active) {
            const int rows_here = min(16, M - mt * 16);
            for (int it = lane; it < rows_here * (HD / 4); it += 32) {
              const int m = mt * 16 + it / (HD / 4), d = it % (HD / 4) * 4;
              float top = -INFINITY, l = 0.f;
              float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
              for (int k = c0 + ks; k <= c1; k += groups) {
                const float* x = p.rec + (size_t)(k == c0 ? 2 * k + 1 : 2 * k) * rec_floats;
                const float mk2 = __ldcg(x + (size_t)p.block_rows * HD + m), lk = __ldcg(x + (size_t)p.block_rows * (HD + 1) + m);
                const float4 v = __ldcg(reinterpret_cast<const float4*>(x + (size_t)m * HD + d));
                const float nt = fmaxf(top, mk2), use = nt == -INFINITY ? 0.f : nt;
                const float fo = pg_exp2(top - use), fn = pg_exp2(mk2 - use);
                l = l * fo + lk * fn;
                acc.x = acc.x * fo + v.x * fn, acc.y = acc.y * fo + v.y * fn;
                acc.z = acc.z * fo + v.z * fn, acc.w = acc.w * fo + v.w * fn;
                top = nt;
              }
              const int mm = warp * 16 + it / (HD / 4);
              *reinterpret_cast<float4*>(join + mm * PITCH + d) = acc;
              if (d == 0) join_ml[mm] = make_float2(top, l);
            }
          }
          dc_bar();
          finish(true);
          if (tid == 0) p.tickets[c0] = 0;
        }
      }
      dc_bar();  // the join buffer is free
      t += n;
    }
    seq_at = end;
    ++seq;
  }
}

}  // namespace vp
