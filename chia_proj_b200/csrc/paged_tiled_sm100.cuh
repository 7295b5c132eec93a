// paged_tiled_sm100.cuh -- attention of many queries over the paged 8-bit K/V
// cache: chunked prefill, on the 5th-generation tensor cores.
//
// A unit is up to 256 rows (queries x the heads of a group) of a request with
// one K/V head, as two query tiles of 128 rows; keys come in tiles of 64. With
// hundreds of rows to a key the work is bound by the tensor cores and the
// exponentials, and the conversion of the cache to halves, done once for both
// query tiles, hides behind them. One CTA an SM takes an equal piece of the
// line of tiles; units that are cut leave parts in the workspace, which a small
// kernel behind this one merges with the whole GPU.
//
//   warps 0-3, 4-7  softmax of query tile 0 and 1, a thread a row
//   warps 8, 10     issue the UMMAs of query tile 0 and 1, warp 9 looks up pages
//                   and loads by TMA
//   warps 12-15     convert 8-bit tiles to halves
//
// Tensor memory: two S buffers of 64 columns for each query tile (P, in halves,
// takes the first 32 of its S, the rest of its rounding the others), O0 O1. Shared memory: Q0 Q1 | a ring of
// converted K and V tiles, all in the 128-byte swizzle | a ring of 8-bit tiles
// as TMA brings them.
//
// The UMMAs of a CTA execute in the order of their issue, so S_w(t + 2) is
// issued right behind PV_w(t), which reads P_w(t) out of its columns, while the
// softmax works on S_w(t + 1): it finds the next S ready. (With tiles of 128
// keys one S buffer a query tile is all that fits beside O, and each softmax
// waited some 2000 of 5200 cycles for PV and the next S.)
//
// Measured (D 128, e4m3, bf16, 32 query and 8 K/V heads): 4 requests x 1024
// queries over 8192 keys 602 us, 0.86 PFLOP/s, 52% of the rate of a plain matrix
// product; up to that many each, ragged, 265 us, 39% (the fullest CTA has 185 tiles where the mean is 150).
// Bound by the softmax warps: of a tile's 2,550 cycles the UMMAs take 1,024; 500 go to scores and
// maximum, 1,150 to exponentials, sums and packing (64 a thread, two warps a
// scheduler: issue and latency), 700 to barriers and tensor memory. fp16: 700 us.
// Tried: two threads a row on 16 warps 282 us ragged where this had 273; the two
// query tiles' exponentials in turns 290.
//
// Numbers as in the split kernel: Q times a power of two per row and the
// cache's values are halves exactly; a key scale multiplies the scores of its
// 16 columns, the logarithm of a value scale is part of the running maximum.
#pragma once
#include "paged_line_sm100.cuh"

namespace chia {

constexpr int kTiledThreads = 512;
constexpr float kTiledPTop = 7.f;  // P is 2^7 at the running maximum, and at most 2^15 (a half's range)
// The pieces (32 query heads, 8 K/V heads, D 128 unless said; us, requests x queries / keys).
// What a unit costs beside its tiles of 64 keys: 6 against 2: 1 x 4000 / 4000 230, 370;
// 3 x 128 / 20000 93, 97; 4 x 1024 / 8192 601, 603.
constexpr int kTiledCost = 6;
// Units of up to this cost, and of no more than a CTA's share, are not cut: a cut is a part of
// 128 KB to write and to read and another start. 48 against 12: 16 x 100 / 900 67, 85. Without
// the share 1 x 2000 / 2000 (8 query heads to one K/V head) takes 58, with it 38; never whole,
// 64 x 32 / 400 takes 103 in place of 82.
constexpr int kTiledWhole = 48;
// The least cost of a piece: 1, 4, 12 and 40 on 1 x 64 / 700: 24, 25, 41, 83; on
// 30 x 256 / 2000 119.2, 118.7 (1 and 4).
constexpr int kTiledPiece = 4;

template <int D>
struct TiledConfig {
  static constexpr int ROWS = 256;             // rows of a unit
  static constexpr int TK = 64;                // keys of a tile
  static constexpr int GROUPS = TK / 16;       // of keys that share their scales
  static constexpr int Q_TILE = 128 * D * 2;
  static constexpr int Q_CHUNK = 128 * 128;    // 64 channels of a query tile
  static constexpr int CHUNK = TK * 128;       // 64 channels of a key tile
  static constexpr int KV = TK * D * 2;        // a converted K or V tile
  static constexpr int SLOTS = 6;
  static constexpr int STAGE = TK * D;         // an 8-bit one
  static constexpr int STAGES = 4;
  static constexpr int SETS = 8;             // tiles whose scales are held
  static constexpr int OFF_KV = 2 * Q_TILE;
  static constexpr int OFF_ST = OFF_KV + SLOTS * KV;
  static constexpr int OFF_SC = OFF_ST + STAGES * STAGE;
  static constexpr int SMEM = 1024 + OFF_SC + SETS * GROUPS * 16;
  // registers a thread: 512 threads begin with 128
  static constexpr int REG_SOFTMAX = 160, REG_OTHER = 96;
  static_assert(256 * REG_SOFTMAX + 256 * REG_OTHER == 65536, "register split");
};

// A unit that a CTA begins and later ones, up to `last`, go on with; rows 0: none.
struct CutUnit {
  Unit un;
  int last;
};

// Merges the parts of the units that are cut: CTA (c, y) some rows of the unit that
// CTA c of the tiled kernel began, its parts in the order of the line, eight of
// them in flight at once.
constexpr int kMergeThreads = 256, kMergeSlices = 16;
template <int D, int KIND, bool BF16>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const PagedArgs a, const CutUnit *cuts) {
  constexpr int ROWS = TiledConfig<D>::ROWS;
  follow();
  const int first = blockIdx.x;
  const CutUnit cu = cuts[first];
  for (int e = blockIdx.y * kMergeThreads + threadIdx.x; e < cu.un.rows * (D / 4);
       e += kMergeSlices * kMergeThreads) {
    const int r = e / (D / 4), c4 = e % (D / 4);
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    merge_parts<ROWS, D>(a, first, cu.last, r, c4, M, L, acc);
    float f;
    uint16_t *dst = row_out<KIND>(a, cu.un, r, M, L, c4 == 0, f);
    store4<BF16>(a, dst + 4 * c4, f, acc.x, acc.y, acc.z, acc.w);
  }
}

// Channels (bits) in which a visible key of tiles [t0, t1) of the unit holds
// NaN, where the tile is not visible as a whole (pages out of range are not): the
// converters leave NaN out of such tiles, since a P of zero would spread it to rows
// that do not see it. Tree: the first key of the row's tree, and the row's word.
template <int D, class... Tree>
__device__ __noinline__ void nan_channels(const PagedArgs &a, const uint8_t *v_cache, int b, int hk,
                                          const Tiles &tl, int t0, int t1, int i, int len, int lo_max,
                                          int hi_min, uint32_t *mask, Tree... tree) {
  int lo, hi;
  band32(a, i, len, lo, hi);
  int pf = min(a.prefix, len);
  auto sees = [&](int j) { return j < pf || (j >= lo && j <= hi && (a.dil == 1 || divides(a.dil, i - j))); };
  auto sees_node = [&](int j, int first, unsigned long long word) {
    return j < first ? sees(j) : j - first < 64 && ((word >> (j - first)) & 1) != 0;
  };
  if constexpr (sizeof...(Tree) > 0) {
    const auto clip = [&](int first, unsigned long long) { pf = max(0, min(pf, first)); };
    clip(tree...);
  }
  for (int t = t0; t < t1; ++t) {
    constexpr int TK = TiledConfig<D>::TK;
    const int j0 = tl.key_tile(t) * TK;
    bool whole = (a.dil == 1 && j0 >= lo_max && j0 + TK - 1 <= hi_min) || j0 <= pf - TK;
    for (int x = 0; x < TK && whole; x += 16) {
      const int pg = a.block_table[b * a.table_stride + (j0 + x) / a.page];
      whole = pg >= 0 && pg < a.num_pages;
    }
    if (whole) continue;
    for (int j = j0; j - j0 < TK && j < len; ++j) {
      if constexpr (sizeof...(Tree) > 0) {
        if (!sees_node(j, tree...)) continue;
      } else if (!sees(j)) {
        continue;
      }
      const int pg = a.block_table[b * a.table_stride + j / a.page];
      if (pg < 0 || pg >= a.num_pages) continue;
      const uint8_t *v = v_cache + ((static_cast<int64_t>(pg) * a.heads_kv + hk) * a.page + j % a.page) * D;
      for (int c = 0; c < D; ++c)
        if ((v[c] & 0x7f) == 0x7f) mask[c / 32] |= 1u << (c % 32);
    }
  }
}

// TREE: requests of up to kTreeNodes queries are trees of drafted tokens, as in the split kernel.
// Measured (D 128, e4m3, bf16, 8 K/V heads): 8 x 64 nodes of 64 heads over 4,096 keys 118 us, 16 x 25
// of 32 over 16,000 313 to 323, 32 x 1 to 64 of 64 over up to 16,384 keys, capped, 315. A tile takes
// 2,400 to 3,500 cycles where its unit has up to 128 rows (1,140 of the conversion, 700 of waits for
// copies, 1,700 to 2,150 of the softmax), up to 5,000 in a full unit with capped scores; the line
// counts them alike, so the CTA with most full units is the last: 123 tiles of 5,000 cycles are 313
// us. Tried for units of up to 128 rows: both halves of the softmax warps with the same rows, a key
// tile each by turns, joined at the end: 291 us on 16 x 25 nodes, where warps without rows that did no
// arithmetic took 300; capped 337 and 330. Without that skipping, as it is now, the capped trees took
// 314 us for 325 and the 16 x 25 nodes 313 to 323 for 300.
template <int D, int CT, int KIND, bool BF16, bool TREE>
__global__ void __launch_bounds__(kTiledThreads, 1)
paged_tiled_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                   const PagedArgs a, const uint8_t *v_cache, CutUnit *cuts) {
  using C = TiledConfig<D>;
  constexpr int TK = C::TK, ROWS = C::ROWS, SLOTS = C::SLOTS, STAGES = C::STAGES, SETS = C::SETS,
                GROUPS = C::GROUPS;
  constexpr bool SOFTMAX = KIND <= KIND_ALIBI;
  constexpr float LOG2E = 1.4426950408889634f;
  using L = Line<TK, ROWS, kTiledThreads, kTiledCost, kTiledWhole, true, TREE>;
  extern __shared__ uint8_t dyn[];
  uint8_t *sm = dyn + ((1024u - (ptx::smem_u32(dyn) & 1023u)) & 1023u);
  const uint32_t sb = ptx::smem_u32(sm);
  float4 *scales = reinterpret_cast<float4 *>(sm + C::OFF_SC);  // [SETS][GROUPS]: ks, value factor, its inverse
  __shared__ typename L::Shared line_sm;
  // st_full st_empty | kv_full kv_empty | q (2) | s p (2 buffers x 2) | pv o o_empty (2 each) | scales full empty | drain
  enum { ST_FULL = 0, ST_EMPTY = ST_FULL + STAGES, KV_FULL = ST_EMPTY + STAGES, KV_EMPTY = KV_FULL + SLOTS,
         Q_FULL = KV_EMPTY + SLOTS, S_FULL = Q_FULL + 2, P_FULL = S_FULL + 4, PV_DONE = P_FULL + 4,
         O_FULL = PV_DONE + 2, O_EMPTY = O_FULL + 2, SC_FULL = O_EMPTY + 2, SC_EMPTY = SC_FULL + SETS,
         DRAIN = SC_EMPTY + SETS, BARS = DRAIN + 2 };
  __shared__ __align__(8) uint64_t bars[BARS];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag, nan_flag;
  __shared__ float q_scale[256];  // of the rows of Q, undone in the scores
  __shared__ unsigned long long s_word[TREE ? 256 : 1];  // the nodes that each row sees
  // of a tile: all rows see the whole of it; keys there are; bits, 16 keys each: their page
  // is out of range, so that nothing is loaded and no row sees them
  __shared__ int tile_full[SETS], tile_live[SETS], tile_lost[SETS];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  auto bar = [&](int i) { return ptx::smem_u32(bars) + 8 * i; };
  if (t == 0) {
    for (int i = 0; i < BARS; ++i) {
      const bool four = (i >= ST_EMPTY && i < KV_EMPTY) || (i >= Q_FULL && i < S_FULL) ||
                        (i >= P_FULL && i < PV_DONE) || (i >= O_EMPTY && i < SC_FULL);
      ptx::mbar_init(bar(i), i >= KV_EMPTY && i < Q_FULL ? 2 : four ? 4 : i >= SC_EMPTY && i < DRAIN ? 8 : 1);
    }
    abort_flag = nan_flag = 0;
    ptx::tma_prefetch_desc(&mk);
    ptx::tma_prefetch_desc(&mv);
  }
  ptx::fence_barrier_init();
  follow();
  const L line(line_sm, a, kTiledPiece);
  if (static_cast<int>(blockIdx.x) >= line.ctas) {
    if (t == 0) cuts[blockIdx.x].un.rows = 0;
    return;
  }
  int c0, nk;  // this CTA's tiles
  {
    int tile, entry;
    line.place(line.even(blockIdx.x + (lane & 1)), true, tile, entry);
    c0 = __shfl_sync(0xffffffffu, tile, 0);
    nk = __shfl_sync(0xffffffffu, tile, 1) - c0;
  }
  if (warp == 8) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](int i, uint32_t parity) { return paged_wait(bar(i), parity, &abort_flag, a); };

  // both of two: asked for together, since an answer takes some 100 cycles
  auto wait2 = [&](int i, uint32_t pi, int j, uint32_t pj) {
    const bool x = ptx::mbar_test_wait(bar(i), pi), y = ptx::mbar_test_wait(bar(j), pj);
    if (x && y) return true;
#pragma unroll 1  // (one copy of the code)
    for (int second = 0; second < 2; ++second)
      if (!wait(second ? j : i, second ? pj : pi)) return false;
    return true;
  };

  // the unit of this CTA's tile k
  struct Here {
    Unit un;
    Request rq;
    int ut0, nt, p0, lo_max, hi_min;
  };
  // the first key of a request's tree (none: the largest number)
  auto tree_first = [](const Request &r) { return TREE && r.n <= kTreeNodes ? r.len - r.n : 0x7fffffff; };
  auto unit_at = [&](int k) {
    Here h;
    const int e = line.entry_at(c0 + k);
    h.rq = line_sm.req[e];
    h.un = line.unit_at(c0 + k, e, h.rq, h.ut0);
    h.nt = min(h.un.n - h.ut0, nk - k);
    h.p0 = h.rq.len - h.rq.n;
    int x;
    band32(a, h.p0 + div_group(a, h.un.row0), h.rq.len, x, h.hi_min);
    band32(a, h.p0 + div_group(a, h.un.row0 + h.un.rows - 1), h.rq.len, h.lo_max, x);
    if (TREE && h.rq.n <= kTreeNodes) {
      band32(a, h.p0, h.rq.len, x, h.hi_min);
      band32(a, h.rq.len - 1, h.rq.len, h.lo_max, x);
      h.hi_min = min(h.hi_min, h.p0 - 1);
    }
    return h;
  };
  auto prefix_of = [&](const Here &h) {  // keys that every row sees
    const int pf = min(a.prefix, h.rq.len);
    return TREE ? max(0, min(pf, tree_first(h.rq))) : pf;
  };
  auto sees_all = [&](const Here &h, int j0) {  // every row of the unit sees keys [j0, j0 + TK)
    return (a.dil == 1 && j0 >= h.lo_max && j0 + TK - 1 <= h.hi_min) ||
           j0 <= prefix_of(h) - TK;
  };

  if (warp >= 8) {
    ptx::setmaxnreg_dec<C::REG_OTHER>();
    if (warp == 9) {
      // ==================================================== pages and TMA
      const int pshift = 31 - __clz(a.page), rows = min(a.page, TK);
      struct Keys {
        int key, pg;
        int hk, all, live;  // all: bit 0 every row sees the tile, 1 no row these keys, 2 there are such keys
      };
      int issued = 0;
      if constexpr (TREE) {
        // Trees: a lane looks up 16 keys of a tile, four lanes a tile, so eight tiles at a time: the pages
        // of the next eight are asked for while the first of these are loaded, their scales four tiles
        // later. (16 x 25 nodes over 16,000 keys 326 us, with the way below 348; without trees 302 and 296.)
        static_assert(GROUPS == 4, "four lanes a tile");
        const int grp = lane & 3;
        auto page_of = [&](int k) {
          Keys x{0, -1, 0, 0, 0};
          if (k >= nk) return x;
          const Here h = unit_at(k);
          int y, lo_min, hi_max;
          band32(a, h.p0 + div_group(a, h.un.row0), h.rq.len, lo_min, y);
          band32(a, h.p0 + div_group(a, h.un.row0 + h.un.rows - 1), h.rq.len, y, hi_max);
          if (h.rq.n <= kTreeNodes) {
            band32(a, h.p0, h.rq.len, lo_min, y);
            band32(a, h.rq.len - 1, h.rq.len, y, hi_max);
          }
          const int j0 = h.rq.tl.key_tile(h.ut0) * TK;
          x.key = j0 + 16 * grp;
          x.hk = h.un.hk;
          x.all = sees_all(h, j0);
          x.live = h.rq.len - j0;
          // (the scales of 16 keys that no row sees may be anything)
          if (!(x.key < prefix_of(h) || (x.key <= hi_max && x.key + 15 >= lo_min))) x.all |= 2;
          if (x.key < h.rq.len) x.pg = a.block_table[h.rq.b * a.table_stride + (x.key >> pshift)], x.all |= 4;
          return x;
        };
        Keys now, next = page_of(lane >> 2);
        int row = -1, next_row = -1;
        float ks = 0.f, vs = 0.f, next_ks = 0.f, next_vs = 0.f;
        auto ask_scales = [&] {
          next_row = -1;
          if (next.pg >= 0 && next.pg < a.num_pages) {
            next_row = next.pg * a.heads_kv + next.hk;
            next_ks = a.k_scale[next_row];
            next_vs = a.v_scale[next_row];
          }
        };
        ask_scales();
        for (int k = 0; k < nk; ++k) {
          const int in = k & 7;
          if (in == 0) now = next, row = next_row, ks = next_ks, vs = next_vs;
          // A softmax warp may be far behind: a query tile without rows takes part in no other wait
          // for these tiles, and its warps may still be writing the unit before.
          if (!warp_all(wait(SC_EMPTY + k % SETS, ((k / SETS) & 1) ^ 1))) break;
          const bool me = (lane >> 2) == in;  // this lane's keys are of the tile
          const bool bad = me && row < 0 && (now.all & 6) == 4;
          const int lost = static_cast<int>(__ballot_sync(0xffffffffu, bad)) >> (4 * in) & 15;
          if (bad) report(a.status, kStatusBadIndex);
          if (me && grp == 0)
            tile_full[k % SETS] = lost == 0 && (now.all & 1), tile_live[k % SETS] = now.live, tile_lost[k % SETS] = lost;
          __syncwarp();
          const bool leads = me && row >= 0 && (16 * grp) % rows == 0;
          const int bytes = __popc(__ballot_sync(0xffffffffu, leads)) * rows * D;
          bool ok = true;
          for (int v = 0; v < 2 && ok; ++v) {
            const int item = 2 * k + v, st = item % STAGES;
            ok = warp_all(wait(ST_EMPTY + st, ((item / STAGES) & 1) ^ 1));
            if (!ok) break;
            if (lane == 0) ptx::mbar_arrive_expect_tx(bar(ST_FULL + st), bytes);
            __syncwarp();
            if (leads)
              tma_load_3d(sb + C::OFF_ST + st * C::STAGE + 16 * grp * D, v ? &mv : &mk, bar(ST_FULL + st), 0,
                          now.key & (a.page - 1), row);
            ++issued;
          }
          if (!ok) break;
          if (me) {
            float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row >= 0 && !(now.all & 2)) {
              sc.x = ks;
              sc.y = value_factor<SOFTMAX>(vs);
              sc.z = SOFTMAX ? ptx::ex2(-sc.y) : 0.f;
            }
            scales[(k % SETS) * GROUPS + grp] = sc;
          }
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(SC_FULL + k % SETS));
          if (in == 1) next = page_of(k - 1 + 8 + (lane >> 2));
          if (in == 5) ask_scales();
        }
      } else {
        // Of the tile's keys 16 lane .. + 15 (lanes 0-3). What a tile needs from
        // memory is asked for a tile or two ahead and looked at when its turn
        // comes: the page of tile k + 2, the scales of tile k + 1.
        Here h;
        int left = 0, lo_min = 0, hi_max = 0;  // tiles of the unit still to look up
        auto page_of = [&](int k) {
          Keys x{0, -1, 0, 0, 0};
          if (k >= nk) return x;
          if (left == 0) {
            h = unit_at(k), left = h.nt;
            int y;
            band32(a, h.p0 + div_group(a, h.un.row0), h.rq.len, lo_min, y);
            band32(a, h.p0 + div_group(a, h.un.row0 + h.un.rows - 1), h.rq.len, y, hi_max);
          }
          const int j0 = h.rq.tl.key_tile(h.ut0 + h.nt - left) * TK;
          --left;
          x.key = j0 + 16 * lane;
          x.hk = h.un.hk;
          x.all = sees_all(h, j0);
          x.live = h.rq.len - j0;
          // (the scales of 16 keys that no row sees may be anything)
          if (!(x.key < min(a.prefix, h.rq.len) || (x.key <= hi_max && x.key + 15 >= lo_min))) x.all |= 2;
          if (lane < GROUPS && x.key < h.rq.len) 
            x.pg = a.block_table[h.rq.b * a.table_stride + (x.key >> pshift)], x.all |= 4;
          return x;
        };
        Keys k1 = page_of(0);
        int row1 = -1, row = -1;
        float ks1 = 0.f, vs1 = 0.f, ks = 0.f, vs = 0.f;
        auto scales_of = [&](const Keys &x) {
          row1 = -1;
          if (x.pg >= 0 && x.pg < a.num_pages) {
            row1 = x.pg * a.heads_kv + x.hk;
            ks1 = a.k_scale[row1];
            vs1 = a.v_scale[row1];
          }
        };
        scales_of(k1);
        Keys k2 = page_of(1);
        for (int k = 0; k < nk; ++k) {
          // A softmax warp may be far behind: a query tile without rows takes part in no other wait
          // for these tiles, and its warps may still be writing the unit before.
          if (!warp_all(wait(SC_EMPTY + k % SETS, ((k / SETS) & 1) ^ 1))) break;
          const Keys now = k1;
          row = row1, ks = ks1, vs = vs1;
          const bool bad = row < 0 && (now.all & 6) == 4;
          const int lost = static_cast<int>(__ballot_sync(0xffffffffu, bad));
          if (bad) report(a.status, kStatusBadIndex);
          if (lane < GROUPS) {
            float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row >= 0 && !(now.all & 2)) {
              sc.x = ks;
              sc.y = value_factor<SOFTMAX>(vs);
              sc.z = SOFTMAX ? ptx::ex2(-sc.y) : 0.f;
            }
            scales[(k % SETS) * GROUPS + lane] = sc;
          }
          if (lane == 0)
            tile_full[k % SETS] = lost == 0 && (now.all & 1), tile_live[k % SETS] = now.live, tile_lost[k % SETS] = lost;
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(SC_FULL + k % SETS));
          k1 = k2;
          scales_of(k1);
          k2 = page_of(k + 2);
          const bool leads = lane < GROUPS && row >= 0 && (16 * lane) % rows == 0;
          const int bytes = __popc(__ballot_sync(0xffffffffu, leads)) * rows * D;
          bool ok = true;
          for (int v = 0; v < 2 && ok; ++v) {
            const int item = 2 * k + v, st = item % STAGES;
            ok = warp_all(wait(ST_EMPTY + st, ((item / STAGES) & 1) ^ 1));
            if (!ok) break;
            if (lane == 0) ptx::mbar_arrive_expect_tx(bar(ST_FULL + st), bytes);
            __syncwarp();
            if (leads)
              tma_load_3d(sb + C::OFF_ST + st * C::STAGE + 16 * lane * D, v ? &mv : &mk, bar(ST_FULL + st), 0,
                          now.key & (a.page - 1), row);
            ++issued;
          }
          if (!ok) break;
        }
      }
      // no copy is in flight when the CTA exits
      PagedArgs d = a;
      d.timeout_ns = a.drain_ns;
      int none = 0;
      for (int i = max(0, issued - STAGES); i < issued; ++i)
        paged_wait(bar(ST_FULL + i % STAGES), (i / STAGES) & 1, &none, d);
    } else if (warp == 8 || warp == 10) {
      // ==================================================== UMMA issue
      // A warp a query tile: one warp's issue (some 40 cycles a UMMA) would be
      // the limit, since a UMMA of 64 keys runs for 32.
      const int w = warp == 10;
      constexpr uint32_t IDESC_QK = ptx::make_idesc_f16(128, TK, false, false, false);
      constexpr uint32_t IDESC_PV = ptx::make_idesc_f16(128, D, false, false, true);
      const uint64_t dq = ptx::make_sdesc_sw128(sb + w * C::Q_TILE, 16, 1024);
      const uint64_t dk = ptx::make_sdesc_sw128(sb + C::OFF_KV, 16, 1024);
      const uint64_t dv = ptx::make_sdesc_sw128(sb + C::OFF_KV, C::CHUNK, 1024);
      const uint32_t tS = tmem + w * 128, tO = tmem + 256 + w * 128;
      auto issue_s = [&](int buf, int slot) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint64_t q0 = dq + ((c * C::Q_CHUNK) >> 4), k0 = dk + ((slot * C::KV + c * C::CHUNK) >> 4);
          const uint64_t qa[4] = {q0, q0 + 2, q0 + 4, q0 + 6}, kb[4] = {k0, k0 + 2, k0 + 4, k0 + 6};
          ptx::umma_ss_x4_warp(tS + buf * 64, qa, kb, IDESC_QK, c > 0 ? 1u : 0u);
        }
        ptx::umma_commit_warp(bar(S_FULL + 2 * w + buf));
        ptx::umma_commit_warp(bar(KV_EMPTY + slot));
      };
      auto issue_pv = [&](int buf, int slot, bool first, bool last) {
        static_assert(TK == 64, "four steps of 16 keys");
        const uint32_t p0 = tS + buf * 64, pa[4] = {p0, p0 + 8, p0 + 16, p0 + 24};
        const uint64_t v0 = dv + ((slot * C::KV) >> 4), vb[4] = {v0, v0 + 128, v0 + 256, v0 + 384};
        ptx::umma_ts_x4_warp(tO, pa, vb, IDESC_PV, first ? 0u : 1u);
        if (!BF16) {  // what P's rounding left
          const uint32_t pb[4] = {p0 + 32, p0 + 40, p0 + 48, p0 + 56};
          ptx::umma_ts_x4_warp(tO, pb, vb, IDESC_PV, 1u);
        }
        ptx::umma_commit_warp(bar(PV_DONE + w));
        ptx::umma_commit_warp(bar(KV_EMPTY + slot));
        if (last) ptx::umma_commit_warp(bar(O_FULL + w));
      };
      uint32_t tiles = 0, units = 0;
      bool ok = true;
      for (int k = 0; k < nk && ok;) {
        const Here h = unit_at(k);
        if (h.un.rows <= 128 * w) {  // no second query tile: the slots are let go as they come
          for (int i = 2 * k; i < 2 * (k + h.nt) && ok; ++i) {
            ok = warp_all(wait(KV_FULL + i % SLOTS, (i / SLOTS) & 1));
            if (ok && lane == 0) ptx::mbar_arrive(bar(KV_EMPTY + i % SLOTS));
          }
          k += h.nt;
          continue;
        }
        ok = warp_all(wait(Q_FULL + w, units & 1));
        // S of the unit's first two tiles, then behind each PV the S two tiles on
        auto next_s = [&](int i) {
          const int ki = 2 * (k + i);
          if (!warp_all(wait(KV_FULL + ki % SLOTS, (ki / SLOTS) & 1))) return false;
          ptx::tc_fence_after();
          issue_s((tiles + i) & 1, ki % SLOTS);
          return true;
        };
        for (int i = 0; i < min(2, h.nt) && ok; ++i) ok = next_s(i);
        for (int i = 0; i < h.nt && ok; ++i) {
          const int vi = 2 * (k + i) + 1;
          const uint32_t n = tiles + i;
          ok = warp_all(wait(KV_FULL + vi % SLOTS, (vi / SLOTS) & 1) &&
                        wait(P_FULL + 2 * w + (n & 1), (n >> 1) & 1) &&
                        (i > 0 || units == 0 || wait(O_EMPTY + w, (units - 1) & 1)));
          if (!ok) break;
          ptx::tc_fence_after();
          issue_pv(n & 1, vi % SLOTS, i == 0, i == h.nt - 1);
          if (i + 2 < h.nt) ok = next_s(i + 2);
        }
        tiles += h.nt;
        ++units;
        k += h.nt;
      }
      // all UMMAs are complete before tensor memory is freed
      ptx::umma_commit_warp(bar(DRAIN + w));
      PagedArgs d = a;
      d.timeout_ns = a.drain_ns;
      int none = 0;
      paged_wait(bar(DRAIN + w), 0, &none, d);
    } else if (warp >= 12) {
      // ==================================================== conversion
      const int c = t - 384;
      for (int item = 0; item < 2 * nk; ++item) {
        const int st = item % STAGES, sl = item % SLOTS;
        // (after a wait that ran out what is read and stored is anything; the vote below ends the work)
        const bool got = wait2(ST_FULL + st, (item / STAGES) & 1, KV_EMPTY + sl, ((item / SLOTS) & 1) ^ 1);
        const int set = (item / 2) % SETS;
        const bool sift = CT == CACHE_E4M3 && (item & 1) && !tile_full[set];
        bool nan_seen = false;
        // Eight lanes read 128 bytes of two neighbouring rows, 64 of each, that
        // fall into different banks, and store to units of the two rows' swizzled
        // lines that do so too: the rows' swizzles differ in the lowest bit.
        constexpr int PER = TK * D / 16 / 128;  // 16-byte pieces a thread
        const int half = (lane >> 2) & 1, r0 = (c >> 5) * (TK / 4) + 2 * (lane >> 3) + half;
        auto row_of = [&](int x) { return r0 + 8 * (D == 128 ? x >> 1 : x); };
        auto piece_of = [&](int x) { return (lane & 3) + (D == 128 ? 4 * (half ^ (x & 1)) : 0); };
        uint4 q[PER];
#pragma unroll
        for (int x = 0; x < PER; ++x)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(q[x].x), "=r"(q[x].y), "=r"(q[x].z), "=r"(q[x].w)
                       : "r"(sb + C::OFF_ST + st * C::STAGE + row_of(x) * D + piece_of(x) * 16));
#pragma unroll
        for (int x = 0; x < PER; ++x) {
          const int row = row_of(x), v = piece_of(x);
          if (sift) {
            const bool live = row < tile_live[set];
            auto clean = [&](uint32_t &w) {
              const uint32_t nan = (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
              nan_seen |= live && nan != 0;
              w &= ~(nan * 0xffu);
            };
            clean(q[x].x), clean(q[x].y), clean(q[x].z), clean(q[x].w);
          }
          uint32_t h[8];
          cache4_to_f16<CT>(q[x].x, h[0], h[1]);
          cache4_to_f16<CT>(q[x].y, h[2], h[3]);
          cache4_to_f16<CT>(q[x].z, h[4], h[5]);
          cache4_to_f16<CT>(q[x].w, h[6], h[7]);
          // channels 16 v .. + 15: units 2 v, 2 v + 1 of the row, four pieces a chunk
          const uint32_t base = sb + C::OFF_KV + sl * C::KV + (v / 4) * C::CHUNK + row * 128;
          const int u = 2 * (v % 4), sw = row & 7;
          ptx::st_shared_v4(base + ((u ^ sw) << 4), h[0], h[1], h[2], h[3]);
          ptx::st_shared_v4(base + (((u + 1) ^ sw) << 4), h[4], h[5], h[6], h[7]);
        }
        if (sift && nan_seen) nan_flag = 1;
        ptx::fence_proxy_async_smem();  // the UMMAs read what was stored
        __syncwarp();
        if (!warp_all(got)) break;
        if (lane == 0) {
          ptx::mbar_arrive(bar(KV_FULL + sl));
          ptx::mbar_arrive(bar(ST_EMPTY + st));
        }
      }
    }
    __syncwarp();
  } else {
    ptx::setmaxnreg_inc<C::REG_SOFTMAX>();
    // ======================================================= softmax
    const int w = warp >> 2, row = t & 127;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS0 = tmem + lane_off + w * 128, tO = tmem + lane_off + 256 + w * 128;
    uint32_t cnt = 0, units = 0;
    bool ok = true;
    if (t == 0) cuts[blockIdx.x].un.rows = 0;
    for (int k = 0; k < nk && ok;) {
      const Here h = unit_at(k);
      const bool begun = h.ut0 == 0, ended = h.ut0 + h.nt == h.un.n, whole = begun && ended;
      const int64_t slot = 2ll * blockIdx.x + (begun ? 1 : 0);
      const int r = w * 128 + row;  // row of the unit
      const bool real = r < h.un.rows;
      if (h.un.rows > w * 128) {
        const int rr = h.un.row0 + min(r, h.un.rows - 1);
        const int qi = div_group(a, rr), head = h.un.hk * a.group + rr - qi * a.group;
        const int first = tree_first(h.rq);
        // (asked for here, looked at behind Q)
        int pos = h.p0 + qi;
        unsigned long long word = 0;
        if (TREE && first != 0x7fffffff) pos = a.tree_pos[h.rq.t0 + qi], word = a.tree_word[h.rq.t0 + qi];
        // ---- the row of Q, as halves
        // (16 bytes a lane, neighbouring lanes along a row, four loads on their way
        // while four are converted: unrolled further, fetching the code takes longer)
        float rowmul = a.score_scale;
        {
          constexpr int UPR = D / 8, RPI = 32 / UPR, IT = 32 / RPI, AHEAD = 4;
          const int u = lane % UPR, q0 = w * 128 + (warp & 3) * 32 + lane / UPR;  // row of the first load
          uint4 raw[AHEAD];
          auto load = [&](int x) {
            const int q = q0 + x * RPI, qr = h.un.row0 + q;
            const int qt = div_group(a, qr), qh = h.un.hk * a.group + qr - qt * a.group;
            return q < h.un.rows
                       ? *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) +
                                                          static_cast<int64_t>(h.un.t0 + qt) * a.q_st +
                                                          qh * a.q_sh + 8 * u)
                       : make_uint4(0, 0, 0, 0);
          };
#pragma unroll
          for (int x = 0; x < AHEAD; ++x) raw[x] = load(x);
#pragma unroll 1
          for (int x0 = 0; x0 < IT; x0 += AHEAD) {
#pragma unroll
            for (int x = 0; x < AHEAD; ++x) {
              const uint32_t v[4] = {raw[x].x, raw[x].y, raw[x].z, raw[x].w};
              if (x0 + AHEAD < IT) raw[x] = load(x0 + AHEAD + x);
              float2 f[4];
              float mx = 0.f;
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                f[y] = in16x2_to_float2<BF16>(v[y]);
                mx = ptx::max3(mx, fabsf(f[y].x), fabsf(f[y].y));
              }
#pragma unroll
              for (int d = 1; d < UPR; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
              int e = static_cast<int>(__float_as_uint(mx) >> 23) - 127;
              e = max(-100, min(127, e));
              const float up = pow2f(14 - e);
              const int q = q0 + (x0 + x) * RPI;
              ptx::st_shared_v4(sb + w * C::Q_TILE + (u / 8) * C::Q_CHUNK + (q & 127) * 128 +
                                    (((u % 8) ^ (q & 7)) << 4),
                                ptx::pack_f16(f[0].x * up, f[0].y * up), ptx::pack_f16(f[1].x * up, f[1].y * up),
                                ptx::pack_f16(f[2].x * up, f[2].y * up), ptx::pack_f16(f[3].x * up, f[3].y * up));
              if (u == 0) q_scale[q] = pow2f(e - 14);
            }
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(Q_FULL + w));
          rowmul *= q_scale[r];
        }
        const float hp = a.head_param != nullptr ? a.head_param[head] : 1.f;
        float slope = 0.f;
        if (KIND == KIND_SOFTMAX) rowmul *= LOG2E * hp;
        if (KIND == KIND_SOFTCAP) rowmul *= 2.f * LOG2E / a.softcap;
        if (KIND == KIND_ALIBI) rowmul *= LOG2E, slope = hp * LOG2E;
        if (KIND == KIND_SIGMOID) rowmul *= -LOG2E;
        if (TREE && first != 0x7fffffff) {
          pos = max(h.p0, min(h.rq.len - 1, pos));
          s_word[t] = tree_word_of(a, word, h.rq.t0, h.rq.n, pos, h.rq.len);
        }
        int lo, hi;
        band32(a, pos, h.rq.len, lo, hi);
        const int pf = prefix_of(h);
        float m_run = SOFTMAX ? -INFINITY : -100.f, l_run = 0.f;
        for (int i = 0; i < h.nt; ++i, ++cnt) {
          const int n = k + i;
          // (after a wait that ran out S is anything; the vote below ends the work before P is stored)
          const bool got =
              wait2(SC_FULL + n % SETS, (n / SETS) & 1, S_FULL + 2 * w + (cnt & 1), (cnt >> 1) & 1);
          ptx::tc_fence_after();
          const uint32_t tS = tS0 + (cnt & 1) * 64;
          uint32_t sr[2][32];
          ptx::tmem_ld32(tS, sr[0]);
          ptx::tmem_ld32(tS + 32, sr[1]);
          const int j0 = h.rq.tl.key_tile(h.ut0 + i) * TK;
          const float4 *sc = scales + (n % SETS) * GROUPS;
          const bool all = tile_full[n % SETS];
          uint32_t vis[2] = {~0u, ~0u};  // the keys of the tile that this row sees
          if (!all) {
            auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; };
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int k0 = j0 + 32 * c;
              uint32_t m = lo > hi ? 0u : below(hi + 1 - k0) & ~below(lo - k0);
              if (a.dil != 1) {
                uint32_t every = 0;
                const int first = (pos - k0) % a.dil;
                const int by = min(a.dil, 32);  // (a step of up to 2^31 - 1 would wrap around and come back)
                for (int e = first < 0 ? first + a.dil : first; e < 32; e += by) every |= 1u << e;
                m &= every;
              }
              m |= below(pf - k0);
              // (differences from the largest number do not fit: no tree's keys are near)
              if (TREE && first - 32 < k0) m = (m & below(first - k0)) | tree_bits(s_word[t], k0, first);
              vis[c] = real ? m : 0u;
              const int lost = tile_lost[n % SETS] >> (2 * c);
              vis[c] &= (lost & 1 ? 0u : 0xffffu) | (lost & 2 ? 0u : 0xffff0000u);
            }
          }
          ptx::tmem_wait_ld();
          ptx::reg_fence(sr[0]);
          ptx::reg_fence(sr[1]);
          const float rel = static_cast<float>(j0 - pos);
          const bool at_tree = TREE && KIND == KIND_ALIBI && first < j0 + TK;
          float mx = SOFTMAX ? -INFINITY : 0.f;
          auto pass1 = [&](auto masked) {
            constexpr bool MASKED = decltype(masked)::value;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
              const float4 s4 = sc[g];
              const float f = rowmul * s4.x;
              const uint64_t F2 = ptx::f2(f, f), V2 = ptx::f2(s4.y, s4.y);
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const int col = 16 * g + e;
                uint32_t &ra = sr[g / 2][(g & 1) * 16 + e], &rb = sr[g / 2][(g & 1) * 16 + e + 1];
                uint64_t x2 = ptx::f2(__uint_as_float(ra), __uint_as_float(rb));
                float x, y;
                if (KIND == KIND_SOFTCAP) {
                  ptx::f2_split(ptx::mul2(x2, F2), x, y);
                  x = fmaf(a.softcap * LOG2E, fmaf(-2.f, ptx::rcp_fast(ptx::ex2(x) + 1.f), 1.f), s4.y);
                  y = fmaf(a.softcap * LOG2E, fmaf(-2.f, ptx::rcp_fast(ptx::ex2(y) + 1.f), 1.f), s4.y);
                } else if (KIND == KIND_SIGMOID) {
                  const float bias = -a.sig_bias * LOG2E;
                  ptx::f2_split(ptx::fma2(x2, F2, ptx::f2(bias, bias)), x, y);
                  x = s4.y * ptx::rcp_fast(1.f + ptx::ex2(x));
                  y = s4.y * ptx::rcp_fast(1.f + ptx::ex2(y));
                } else if (KIND == KIND_RELU) {
                  ptx::f2_split(ptx::mul2(x2, F2), x, y);
                  x = x < 0.f ? 0.f : x * s4.y;
                  y = y < 0.f ? 0.f : y * s4.y;
                } else {
                  x2 = ptx::fma2(x2, F2, V2);
                  if (KIND == KIND_ALIBI) {
                    const float c = static_cast<float>(col);
                    float d0 = rel + c, d1 = rel + c + 1.f;
                    if (MASKED && at_tree) {  // a tree's nodes have positions of their own
                      const int j = j0 + col;
                      if (j >= first && j < h.rq.len)
                        d0 = static_cast<float>(tree_position(a, h.rq.t0, j - first, h.p0, h.rq.len) - pos);
                      if (j + 1 >= first && j + 1 < h.rq.len)
                        d1 = static_cast<float>(tree_position(a, h.rq.t0, j + 1 - first, h.p0, h.rq.len) - pos);
                    }
                    x2 = ptx::fma2(ptx::f2(slope, slope), ptx::f2(d0, d1), x2);
                  }
                  ptx::f2_split(x2, x, y);
                }
                if (MASKED) {
                  if (!((vis[g / 2] >> ((g & 1) * 16 + e)) & 1)) x = SOFTMAX ? -INFINITY : 0.f;
                  if (!((vis[g / 2] >> ((g & 1) * 16 + e + 1)) & 1)) y = SOFTMAX ? -INFINITY : 0.f;
                }
                mx = ptx::max3(mx, x, y);
                ra = __float_as_uint(x), rb = __float_as_uint(y);
              }
            }
          };
          if (all)
            pass1(std::false_type{});
          else
            pass1(std::true_type{});
          if (!SOFTMAX) mx = static_cast<float>(static_cast<int>(__float_as_uint(mx) >> 23) - 126);
          // the maximum moves only by more than 2^8: P stays below 2^(8 + kTiledPTop)
          const float m_new = fmaxf(m_run, mx);
          const bool need = m_new > m_run + 8.f;
          float alpha = 1.f;
          if (need) {
            alpha = ptx::ex2(m_run - m_new);
            l_run *= alpha;
            m_run = m_new;
          }
          if (__any_sync(0xffffffffu, !got || (need && i > 0))) {
            // O is rescaled once the tile before is in it
            if (!warp_all(got && (i == 0 || wait(PV_DONE + w, (cnt - 1) & 1)))) {
              ok = false;
              break;
            }
            ptx::tc_fence_after();
            rescale_rows<D>(tO, alpha);
          }
          const float mu = m_run == -INFINITY ? 0.f : m_run - kTiledPTop;
          const uint64_t NM2 = ptx::f2(-mu, -mu);
          const float down = SOFTMAX ? 0.f : ptx::ex2(-mu);
          const uint64_t DN2 = ptx::f2(down, down);
          // P as halves. Beside outputs of 8 bits (bf16) that rounding, 2^-12, is nothing;
          // outputs of 11 bits get what it left as halves too, in the other columns of S.
          {
            constexpr bool BOTH = !BF16;
            constexpr int AT = BOTH ? 16 : 32;  // columns of P that are stored at once
#pragma unroll
            for (int part = 0; part < 32 / AT; ++part) {
              uint32_t pk[AT], rest[AT];
#pragma unroll
              for (int g = part * AT / 8; g < (part + 1) * AT / 8; ++g) {
                uint64_t sum = ptx::f2(0.f, 0.f);
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                  uint64_t x2 = ptx::f2(__uint_as_float(sr[g / 2][(g & 1) * 16 + e]),
                                        __uint_as_float(sr[g / 2][(g & 1) * 16 + e + 1]));
                  float x, y;
                  if (SOFTMAX) {
                    ptx::f2_split(ptx::add2(x2, NM2), x, y);
                    x = ptx::ex2(x), y = ptx::ex2(y);
                    sum = ptx::add2(sum, ptx::f2(x, y));
                  } else {
                    ptx::f2_split(ptx::mul2(x2, DN2), x, y);
                  }
                  uint32_t &h = pk[(g * 8 + e / 2) % AT];
                  h = ptx::pack_f16(x, y);
                  if (BOTH) {
                    const float2 f = f16x2_to_float2(h);
                    rest[(g * 8 + e / 2) % AT] = ptx::pack_f16(x - f.x, y - f.y);
                  }
                }
                if (SOFTMAX) {
                  float x, y;
                  ptx::f2_split(sum, x, y);
                  l_run = fmaf(x + y, sc[g].z, l_run);
                }
              }
              if constexpr (BOTH) {
                ptx::tmem_st16(tS + AT * part, pk);
                ptx::tmem_st16(tS + 32 + AT * part, rest);
              } else {
                ptx::tmem_st32(tS, pk);
              }
            }
          }
          ptx::tmem_wait_st();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            ptx::mbar_arrive(bar(P_FULL + 2 * w + (cnt & 1)));
            ptx::mbar_arrive(bar(SC_EMPTY + n % SETS));
          }
        }
        if (!ok) break;
        // ---- O
        if (!warp_all(wait(O_FULL + w, units & 1))) {
          ok = false;
          break;
        }
        ++units;
        ptx::tc_fence_after();
        m_run -= kTiledPTop;  // what O and the sum are relative to
        uint32_t nan[D / 32] = {};
        if (CT == CACHE_E4M3 && nan_flag && real) {
          auto find = [&](auto... tree) {
            nan_channels<D>(a, v_cache, h.rq.b, h.un.hk, h.rq.tl, h.ut0, h.ut0 + h.nt, pos, h.rq.len, h.lo_max,
                            h.hi_min, nan, tree...);
          };
          if constexpr (TREE)
            find(first, s_word[t]);
          else
            find();
        }
        float f = 1.f;
        row_out<KIND>(a, h.un, min(r, h.un.rows - 1), m_run, l_run, whole && real, f);
        // Through this warp's rows of Q's memory (free: the unit's UMMAs are
        // complete), so that neighbouring lanes write along a row: a pass is 128
        // bytes of each of 32 rows, 64 channels as halves or 32 as fp32.
        {
          const int base = (warp & 3) * 32, cols = whole ? 64 : 32;
          auto unit16 = [&](int lr, int u) {
            return sb + w * C::Q_TILE + (base + lr) * 128 + (((u ^ lr) & 7) << 4);
          };
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += cols) {
#pragma unroll 1
            for (int c = 0; c < cols; c += 16) {
              uint32_t o[16];
              ptx::tmem_ld16(tO + c0 + c, o);
              ptx::tmem_wait_ld();
              ptx::reg_fence16(o);
              if (CT == CACHE_E4M3 && nan_flag) {
                const uint32_t nn = nan[(c0 + c) / 32] >> ((c0 + c) % 32);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] |= (nn >> e) & 1 ? 0x7fffffffu : 0u;
              }
              if (whole) {
                uint32_t x[8];
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                  const float p = __uint_as_float(o[2 * y]) * f, q = __uint_as_float(o[2 * y + 1]) * f;
                  x[y] = BF16 ? ptx::pack_bf16(p, q) : ptx::pack_f16(p, q);
                }
                ptx::st_shared_v4(unit16(lane, c / 8), x[0], x[1], x[2], x[3]);
                ptx::st_shared_v4(unit16(lane, c / 8 + 1), x[4], x[5], x[6], x[7]);
              } else {
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                  ptx::st_shared_v4(unit16(lane, (c + e) / 4), o[e], o[e + 1], o[e + 2], o[e + 3]);
              }
            }
            __syncwarp();
#pragma unroll 4
            for (int x = 0; x < 32; x += 4) {
              const int lr = x + lane / 8, u = lane % 8, q = w * 128 + base + lr;
              uint4 v;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                           : "r"(unit16(lr, u)));
              const int ch = c0 + u * (whole ? 8 : 4);
              if (q < h.un.rows) {
                if (whole) {
                  const int qr = h.un.row0 + q, qt = div_group(a, qr), qh = h.un.hk * a.group + qr - qt * a.group;
                  *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.o) +
                                             static_cast<int64_t>(h.un.t0 + qt) * a.o_st + qh * a.o_sh + ch) = v;
                } else {
                  *reinterpret_cast<uint4 *>(a.part_o + (slot * ROWS + q) * D + ch) = v;
                }
              }
            }
            __syncwarp();
          }
        }
        if (!whole && real)
          *reinterpret_cast<float2 *>(a.part_ml + (slot * ROWS + r) * 2) = make_float2(m_run, l_run);
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(O_EMPTY + w));
      } else {  // no rows for this query tile: it keeps step, so that no phase of the scales is passed by
        for (int n = k; n < k + h.nt && ok; ++n) {
          ok = warp_all(wait(SC_FULL + n % SETS, (n / SETS) & 1));
          if (ok && lane == 0) ptx::mbar_arrive(bar(SC_EMPTY + n % SETS));
        }
        if (!ok) break;
      }
      k += h.nt;
      // a unit that begins here and goes on in later CTAs
      if (t == 0 && begun && !ended)
        cuts[blockIdx.x] = CutUnit{h.un, line.cta_of(h.un, h.un.n - 1)};
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// Launches of one head size and cache type; each has a source file of its own, and so have
// those of trees.
template <int D, int CT>
cudaError_t launch_tiled(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a,
                         const uint8_t *v_cache, void *cuts, int kind, int grid, int device, cudaStream_t s);
template <int D, int CT>
cudaError_t launch_tiled_tree(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a,
                              const uint8_t *v_cache, void *cuts, int kind, int grid, int device, cudaStream_t s);

template <int D, int CT, int KIND, bool BF16, bool TREE>
cudaError_t launch_tiled_one(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a,
                             const uint8_t *v_cache, void *cuts, int grid, int device, cudaStream_t s) {
  static std::atomic<uint64_t> set{0};
  constexpr int bytes = TiledConfig<D>::SMEM;
  cudaError_t e = allow_smem(reinterpret_cast<const void *>(&paged_tiled_kernel<D, CT, KIND, BF16, TREE>), bytes,
                             device, set);
  if (e != cudaSuccess) return e;
  e = launch_after(paged_tiled_kernel<D, CT, KIND, BF16, TREE>, dim3(grid), kTiledThreads, bytes, s, mk, mv, a, v_cache,
                   static_cast<CutUnit *>(cuts));
  if (e != cudaSuccess) return e;
  return launch_after(paged_merge_kernel<D, KIND, BF16>, dim3(grid, kMergeSlices), kMergeThreads, 0, s, a,
                      static_cast<const CutUnit *>(cuts));
}

template <int D, int CT, bool BF16, bool TREE = false>
cudaError_t launch_tiled_kind(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a,
                              const uint8_t *v_cache, void *cuts, int kind, int grid, int device, cudaStream_t s) {
  switch (kind) {
    case KIND_SOFTCAP: return launch_tiled_one<D, CT, KIND_SOFTCAP, BF16, TREE>(mk, mv, a, v_cache, cuts, grid, device, s);
    case KIND_ALIBI: return launch_tiled_one<D, CT, KIND_ALIBI, BF16, TREE>(mk, mv, a, v_cache, cuts, grid, device, s);
    case KIND_SIGMOID: return launch_tiled_one<D, CT, KIND_SIGMOID, BF16, TREE>(mk, mv, a, v_cache, cuts, grid, device, s);
    case KIND_RELU: return launch_tiled_one<D, CT, KIND_RELU, BF16, TREE>(mk, mv, a, v_cache, cuts, grid, device, s);
    default: return launch_tiled_one<D, CT, KIND_SOFTMAX, BF16, TREE>(mk, mv, a, v_cache, cuts, grid, device, s);
  }
}

#define CHIA_INSTANTIATE_TILED(D, CT)                                                          \
  template <>                                                                                  \
  cudaError_t chia::launch_tiled<D, CT>(const CUtensorMap &mk, const CUtensorMap &mv,          \
                                        const PagedArgs &a, const uint8_t *v_cache,            \
                                        void *cuts, int kind, int grid, int device,            \
                                        cudaStream_t s) {                                      \
    return a.bf16 ? launch_tiled_kind<D, CT, true>(mk, mv, a, v_cache, cuts, kind, grid, device, s)   \
                  : launch_tiled_kind<D, CT, false>(mk, mv, a, v_cache, cuts, kind, grid, device, s); \
  }
#define CHIA_INSTANTIATE_TILED_TREE(D, CT)                                                          \
  template <>                                                                                  \
  cudaError_t chia::launch_tiled_tree<D, CT>(const CUtensorMap &mk, const CUtensorMap &mv,          \
                                        const PagedArgs &a, const uint8_t *v_cache,            \
                                        void *cuts, int kind, int grid, int device,            \
                                        cudaStream_t s) {                                      \
    return a.bf16 ? launch_tiled_kind<D, CT, true, true>(mk, mv, a, v_cache, cuts, kind, grid, device, s)   \
                  : launch_tiled_kind<D, CT, false, true>(mk, mv, a, v_cache, cuts, kind, grid, device, s); \
  }

}  // namespace chia
