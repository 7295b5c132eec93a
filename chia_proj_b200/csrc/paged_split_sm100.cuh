// paged_split_sm100.cuh -- attention of few queries over the paged 8-bit K/V
// cache: decode steps and drafted tokens.
//
// Every key and value byte is read once and used by group * queries rows, so
// the work is bound by HBM as long as nothing else is in its way. All (request,
// K/V head, block of up to 16 rows) units with their 32-key tiles form one line
// of tiles. A worker is a warp: one CTA of eight an SM, and each takes an equal
// piece of the line whatever the lengths, a unit counting as kUnitCost tiles
// more than it has (its queries, its output). A worker has a ring of its own,
// which its lane 0 fills by TMA (tiled copies with a swizzle that keeps the
// reads below free of bank conflicts), after it looked up 32 tiles' pages and
// scales at a time, a tile a lane. So no warp waits for another until all of a
// CTA's are done. A unit within one worker's piece goes straight to the output;
// units that are cut leave parts, which the CTA merges in shared memory, and the
// last CTA of a unit merges the CTAs' parts, always in the order of the line.
//
// A tile is computed transposed, keys and channels on the 16-row side of
// m16n8k16 and query rows on the 8-column side, so that a group of up to eight
// rows wastes no work; a 5th-generation MMA would need 64 rows or more.
//   S^T (keys x rows)     = K  (A: 16 bytes of a key's row a lane) * Q^T
//   O^T (channels x rows) = V^T (A: ldmatrix.trans of byte pairs)  * P^T
// The contraction over channels may run in any order: lane t of a quad takes
// the 16-byte pieces 2t, 2t + 1 of a key row as its channels of eight steps,
// and Q's fragments are laid out to match. P^T is S^T's accumulators, packed
// and turned by movmatrix. The cache's numbers are halves exactly (e4m3 by one
// conversion a pair; int8 by a byte permutation and a subtraction); Q, brought
// to [2^14, 2^15) by a power of two per row, is a half exactly down to 2^-29
// of its row's largest value; so products lose nothing. P is rounded to a half
// (11 bits) with its page's value scale in it: the softmax's running maximum is
// that of s + log2(scale), so the largest P of a row is 2^15 whatever the scales
// are, and its sum takes the scale out again. Sigmoid and ReLU divide by a
// running power of two instead. Outputs of 11 bits (fp16) get what P's rounding
// left through a second product.
//
// Measured (D 128, e4m3, bf16 unless said): 64 requests x 32,768 keys, 64 query
// and 8 K/V heads 640 to 705 us from GPU to GPU, 6.7 to 6.1 TB/s (a plain copy
// has 6.5, reading alone 6.9); 96 x up to 16,384, pages of 16, 65 us, 4.9 TB/s;
// 8 x 8192, 4 K/V heads, capped, 23.5 us, 2.9 TB/s; one of 601 keys 10.0 us. What is beside HBM there is a chain of some 6 us before the
// first tile (lengths, the line, page, scales; half of it the fetch of the code,
// run once a call) and 2 us of joining parts.
#pragma once
#include "decode_sm100.cuh"
#include "paged_line_sm100.cuh"

namespace chia {

constexpr int kSplitWarps = 8;
constexpr int kSplitThreads = 32 * kSplitWarps;
// The largest P is 2^kPTop: a half keeps 11 bits of a P down to 2^-14, so of one
// that is 2^-29 of its row's largest.
constexpr float kPTop = 15.f;
// What a unit costs beside its tiles, in tiles: 2, 4, 6, 9 on 96 requests of up to 16,384 keys
// 75, 68, 67, 69 us, on 48 with a window of 1024 keys 17.0, 18.0, 17.8, 18.6.
constexpr int kUnitCost = 4;
// Units of up to this cost are not cut between CTAs: 0, 64, 160 on one request of 601 keys 12.8,
// 10.1, 10.1 us, on 24 with five queries each over up to 4,100 keys 22.4, 22.6, 39. It does
// not ask for a CTA's share: of those 24 the fullest CTA has 50 tiles where the mean is 17.
constexpr int kWholeUnit = 64;

// D (16x8, fp32) += A (16x16, halves) * B (16x8). Not volatile: the compiler may
// interleave products with the conversions of the next operands.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 8x8 16-bit matrix, one row a quad of lanes: transposed
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

template <int D, int NT>
struct SplitConfig {
  static constexpr int TK = 32;                   // keys of a tile
  static constexpr int STAGE = 2 * TK * D;        // bytes: K, then V
  static constexpr int NST = 3 * (128 / D);       // stages of a worker: 24 KB of tiles
  static constexpr int ROWS = 8 * NT;             // rows of a unit
  static constexpr int PITCH = D + 4;             // floats of a row in the merge buffer
  static constexpr int SCALES = 64;               // tiles whose scales a worker holds
  static constexpr int RING = kSplitWarps * NST * STAGE;
  static constexpr int SMEM = 1024 + RING + kSplitWarps * SCALES * 16;
  static_assert(kSplitWarps * ROWS * PITCH * 4 <= RING, "the parts fit the spent ring");
};

// KIND: score modification and normaliser.
template <int D, int CT, int NT, int KIND, bool BF16>
__global__ void __launch_bounds__(kSplitThreads, 1)
paged_split_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                   const PagedArgs a) {
  using C = SplitConfig<D, NT>;
  constexpr int TK = C::TK, NST = C::NST, ROWS = C::ROWS, PITCH = C::PITCH;
  constexpr int H = D / 64;   // 16-byte pieces of a key row a lane
  constexpr int MT = D / 16;  // channel tiles of the output
  constexpr bool SOFTMAX = KIND <= KIND_ALIBI;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ uint8_t dyn[];
  uint8_t *sm = dyn + ((1024u - (ptx::smem_u32(dyn) & 1023u)) & 1023u);
  float *parts = reinterpret_cast<float *>(sm);  // [warps][ROWS][PITCH], in the spent ring
  using L = Line<TK, ROWS, kSplitThreads, kUnitCost, kWholeUnit, false>;
  __shared__ typename L::Shared line_sm;
  __shared__ __align__(8) uint64_t bars[kSplitWarps * NST];
  __shared__ float part_ml[kSplitWarps][ROWS][2];
  __shared__ __align__(2) uint8_t s_lost[kSplitWarps][C::SCALES];  // beside the scales: see `lost`
  __shared__ Unit s_head[kSplitWarps], s_end[kSplitWarps];
  __shared__ int s_has_head[kSplitWarps], s_has_end[kSplitWarps];  // end: 1 begun here, 2 before
  __shared__ volatile int abort_flag;
  // A unit's parts in this CTA: what workers first..last have of it. `before`,
  // `after`: it began in an earlier CTA, goes on in a later one.
  struct Group {
    int first, last;
    bool before, after, last_is_head;
  };
  __shared__ Group s_group[kSplitWarps + 1];
  __shared__ int s_groups, s_last[2], s_first_cta[2], s_last_cta[2];
  __shared__ uint32_t s_ends;

  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int gid = lane >> 2, tig = lane & 3;
  const uint32_t bar0 = ptx::smem_u32(bars) + warp * NST * 8;
  const uint32_t ring = ptx::smem_u32(sm) + warp * NST * C::STAGE;
  float4 *scales = reinterpret_cast<float4 *>(sm + C::RING) + warp * C::SCALES;  // ks and the
                                                             // value factor of keys 0-15, 16-31
  if (t < kSplitWarps * NST) ptx::mbar_init(ptx::smem_u32(bars) + 8 * t, 1);
  static_assert(kSplitWarps * C::SCALES == 2 * kSplitThreads, "two a thread");
  reinterpret_cast<uint16_t *>(s_lost)[t] = 0;
  if (t == 0) {
    abort_flag = 0;
    ptx::tma_prefetch_desc(&mk);
    ptx::tma_prefetch_desc(&mv);
  }

  ptx::fence_barrier_init();
  follow();
  const L line(line_sm, a, kSplitWarps);  // (its barriers also order the set-up above)
  if (static_cast<int>(blockIdx.x) >= line.ctas) return;
  const int me = blockIdx.x * kSplitWarps + warp;
  int c0, nk, e0;  // first tile and number of tiles of this worker, the first one's entry
  {
    int tile;  // lane 0: this border, lane 1: the next one
    int x = line.even(blockIdx.x + (lane & 1));
#pragma unroll 1  // (one copy of the code: fetching it is most of the time)
    for (int own = 0; own < 2; ++own) {  // the CTA's borders, then the worker's within them
      const int y = line.place(x, own == 0, tile, e0);
      const int y0 = __shfl_sync(0xffffffffu, y, 0), y1 = __shfl_sync(0xffffffffu, y, 1);
      x = y0 + static_cast<int>(static_cast<long long>(y1 - y0) * (warp + (lane & 1)) / kSplitWarps);
    }
    e0 = __shfl_sync(0xffffffffu, e0, 0);
    c0 = __shfl_sync(0xffffffffu, tile, 0);
    nk = __shfl_sync(0xffffffffu, tile, 1) - c0;
  }
  if (lane == 0) s_has_head[warp] = s_has_end[warp] = 0;
  auto head_o = [&](int w) { return a.part_o + (2ll * gridDim.x + w) * ROWS * D; };
  auto head_ml = [&](int w) { return a.part_ml + (2ll * gridDim.x + w) * ROWS * 2; };
  auto rings_spent = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };

  // ---- loads
  // Of tile 32 * (k / 32) + lane: rows of the tensor map (page * heads_kv + head), first token.
  // The next 32 tiles' pages are asked for while the first of these 32 are
  // computed, their scales a while later, and both are looked at when they are
  // needed: with HBM busy a load takes longer than the ring lasts.
  const int pshift = 31 - __clz(a.page);
  int row0 = -1, row1 = -1, tok = 0;
  int lost = 0;           // bits: keys 0-15, 16-31 have a page out of range: nothing is loaded, no row sees them
  bool any_lost = false;  // so far: from then on no tile counts as one that all rows see
  int next_pg0 = -1, next_pg1 = -1, next_hk = 0, next_tok = 0;  // pages
  int wanted = 0;                                                // bits: that there are such keys
  float next_ks0 = 0.f, next_vs0 = 0.f, next_ks1 = 0.f, next_vs1 = 0.f;
  auto ask_pages = [&](int k, bool one_entry) {  // one_entry: the 32 tiles are all of entry e0
    next_pg0 = next_pg1 = -1, wanted = 0;
    if (k + lane < nk) {
      const int g = c0 + k + lane;
      const int b = one_entry ? e0 : line.entry_at(g);
      const Request r = line_sm.req[b];
      int ut;
      next_hk = line.unit_at(g, b, r, ut).hk;
      const int key = r.tl.key_tile(ut) * TK;
      const int32_t *table = a.block_table + b * a.table_stride + (key >> pshift);
      next_tok = key & (a.page - 1);
      if (key < r.len) next_pg0 = table[0], wanted = 1;
      if (a.page == 16 && key + 16 < r.len) next_pg1 = table[1], wanted = 3;
    }
  };
  auto row_at = [&](int pg) { return pg >= 0 && pg < a.num_pages ? pg * a.heads_kv + next_hk : -1; };
  auto ask_scales = [&] {
    const int r0 = row_at(next_pg0), r1 = row_at(next_pg1);
    if (r0 >= 0) next_ks0 = a.k_scale[r0], next_vs0 = a.v_scale[r0];
    if (r1 >= 0) next_ks1 = a.k_scale[r1], next_vs1 = a.v_scale[r1];
  };
  auto take_rows = [&] {
    row0 = row_at(next_pg0), row1 = row_at(next_pg1), tok = next_tok;
    lost = row0 < 0 && (wanted & 1) ? (a.page == 16 ? 1 : 3) : 0;
    if (row1 < 0 && (wanted & 2)) lost |= 2;
  };
  // all rows of the unit see keys [lo_max, hi_min] and tiles that begin up to pf_all
  int lo_max = 0, hi_min = 0, pf_all = 0;
  auto take_scales = [&](int k) {  // to shared memory
    float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row0 >= 0) sc.x = next_ks0, sc.y = value_factor<SOFTMAX>(next_vs0);
    if (a.page != 16)
      sc.z = sc.x, sc.w = sc.y;
    else if (row1 >= 0)
      sc.z = next_ks1, sc.w = value_factor<SOFTMAX>(next_vs1);
    scales[(k + lane) % C::SCALES] = sc;  // (those of 64 tiles ago are long used)
    if (__any_sync(0xffffffffu, lost != 0)) any_lost = true, hi_min = pf_all = -1;
    if (any_lost) s_lost[warp][(k + lane) % C::SCALES] = static_cast<uint8_t>(lost);
    __syncwarp();
  };
  auto issue = [&](int k) {  // start the copies of tile k, whose stage is free
    if (k >= nk) return;
    const int in = k % 32;
    if (in == 0 && k > 0) {
      take_rows();
      take_scales(k);
    }
    const int r0 = __shfl_sync(0xffffffffu, row0, in);
    const int r1 = __shfl_sync(0xffffffffu, row1, in);
    const int tk = __shfl_sync(0xffffffffu, tok, in);
    if (lane == 0) {
      const uint32_t dst = ring + (k % NST) * C::STAGE, bar = bar0 + 8 * (k % NST);
      const int rows = a.page == 16 ? 16 : TK;
      ptx::mbar_arrive_expect_tx(bar, ((r0 >= 0) + (r1 >= 0)) * 2 * rows * D);
      if (r0 >= 0) {
        tma_load_3d(dst, &mk, bar, 0, tk, r0);
        tma_load_3d(dst + TK * D, &mv, bar, 0, tk, r0);
      }
      if (r1 >= 0) {
        tma_load_3d(dst + 16 * D, &mk, bar, 0, 0, r1);
        tma_load_3d(dst + TK * D + 16 * D, &mv, bar, 0, 0, r1);
      }
    }
    if (in == 12 && k + 20 < nk) ask_pages(k + 20, false);
    if (in == 22 && k + 10 < nk) ask_scales();
  };

  // ---- units of the piece: the one that tile k belongs to, and its queries
  Unit un;
  Tiles tl;
  int len = 0, p0 = 0, ut0 = 0, nt = 0;
  uint4 raw[NT][H * 2];  // row 8 n + gid, channels 16 H tig .. + 16 H - 1
  float hp[NT][2];       // of rows 8 n + 2 tig + e, as in the columns of S^T
  auto begin_unit = [&](int k, int b) {  // b: the entry
    const int g = c0 + k;
    const Request rq = line_sm.req[b];
    len = rq.len;
    p0 = len - rq.n;
    tl = rq.tl;
    un = line.unit_at(g, b, rq, ut0);
    nt = min(tl.n - ut0, nk - k);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int rr = 8 * n + gid, row = un.row0 + rr;
      if (rr < un.rows) {
        const int qi = div_group(a, row);
        const uint16_t *src = static_cast<const uint16_t *>(a.q) +
                              static_cast<int64_t>(rq.t0 + qi) * a.q_st +
                              (un.hk * a.group + row - qi * a.group) * a.q_sh + H * 16 * tig;
#pragma unroll
        for (int c = 0; c < H * 2; ++c) raw[n][c] = *reinterpret_cast<const uint4 *>(src + 8 * c);
      } else {
#pragma unroll
        for (int c = 0; c < H * 2; ++c) raw[n][c] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = min(8 * n + 2 * tig + x, un.rows - 1) + un.row0;
        hp[n][x] = a.head_param != nullptr
                       ? a.head_param[un.hk * a.group + r - div_group(a, r) * a.group]
                       : 1.f;
      }
    }
  };
  if (nk > 0) {
    ask_pages(0, line_sm.tiles_pre[e0 + 1] >= c0 + min(nk, 32));
    begin_unit(0, e0);
    take_rows();
    ask_scales();
    for (int k = 0; k < NST; ++k) issue(k);
    take_scales(0);
  }

  bool aborted = false, has_end = false;
  for (int k = 0; k < nk;) {
    int lo_min, hi_max;  // no row sees a key outside of them and the prefix
    band32(a, p0 + div_group(a, un.row0), len, lo_min, hi_min);
    band32(a, p0 + div_group(a, un.row0 + un.rows - 1), len, lo_max, hi_max);
    const int pf = min(a.prefix, len);
    pf_all = pf - TK;
    if (any_lost) hi_min = pf_all = -1;

    // Q as fragments: channels 16 (H tig + h) + 4 s .. + 3 of step (h, s)
    uint32_t qf[NT][H * 4][2];
    float rowmul[NT][2], slope[NT][2];
    int posn[NT][2];
    uint32_t real = 0;  // bit 2 n + e: that row exists
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float mx = 0.f;
      auto get = [&](int w, float2 &x) {  // 32-bit word w of the lane's channels
        const uint4 &r4 = raw[n][w / 4];
        const uint32_t v = w % 4 == 0 ? r4.x : w % 4 == 1 ? r4.y : w % 4 == 2 ? r4.z : r4.w;
        x = in16x2_to_float2<BF16>(v);
      };
#pragma unroll
      for (int w = 0; w < H * 8; ++w) {
        float2 x;
        get(w, x);
        mx = fmaxf(mx, fmaxf(fabsf(x.x), fabsf(x.y)));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int e = static_cast<int>(__float_as_uint(mx) >> 23) - 127;  // 2^e <= mx < 2^(e + 1)
      e = max(-100, min(127, e));
      const float up = pow2f(14 - e);
#pragma unroll
      for (int w = 0; w < H * 8; ++w) {
        float2 x;
        get(w, x);
        qf[n][w / 2][w % 2] = ptx::pack_f16(x.x * up, x.y * up);
      }
      const float down = pow2f(e - 14);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f = __shfl_sync(0xffffffffu, down, (2 * tig + x) * 4);
        const int r = min(8 * n + 2 * tig + x, un.rows - 1) + un.row0;
        posn[n][x] = p0 + div_group(a, r);
        real |= (8 * n + 2 * tig + x < un.rows ? 1u : 0u) << (2 * n + x);
        float mul = a.score_scale * f;
        slope[n][x] = 0.f;
        if (KIND == KIND_SOFTMAX) mul *= LOG2E * hp[n][x];
        if (KIND == KIND_SOFTCAP) mul *= 2.f * LOG2E / a.softcap;  // 2^(2 log2e s / cap) = e^(2s/cap)
        if (KIND == KIND_ALIBI) mul *= LOG2E, slope[n][x] = hp[n][x] * LOG2E;
        if (KIND == KIND_SIGMOID) mul *= -LOG2E;
        rowmul[n][x] = mul;
      }
    }
    float o[MT][NT][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < MT; ++c) o[c][n][0] = o[c][n][1] = o[c][n][2] = o[c][n][3] = 0.f;
      m_run[n][0] = m_run[n][1] = SOFTMAX ? -INFINITY : -100.f;
      l_run[n][0] = l_run[n][1] = 0.f;
    }

    for (int i = 0; i < nt && !aborted; ++i) {
      const int kk = k + i, stage = kk % NST;
      if (!warp_all(paged_wait(bar0 + 8 * stage, (kk / NST) & 1, &abort_flag, a))) {
        // leave no copy in flight: the ring's memory is used again, and the CTA may exit
        PagedArgs d = a;
        d.timeout_ns = a.drain_ns;
        int none = 0;
        for (int j = kk; j < min(nk, kk + NST); ++j)
          paged_wait(bar0 + 8 * (j % NST), (j / NST) & 1, &none, d);
        aborted = true;
        break;
      }
      const int j0 = tl.key_tile(ut0 + i) * TK;
      float4 sc = scales[kk % C::SCALES];
      const uint32_t kst = ring + stage * C::STAGE, vst = kst + TK * D;
      const bool all =
          a.dil == 1 ? (j0 >= lo_max && j0 + TK - 1 <= hi_min) || j0 <= pf_all : j0 <= pf_all;
      int gone = 0;  // keys that are not there
      if (!all) {  // the scales of 16 keys that nobody sees may be anything
        const bool s0 = j0 < pf || (j0 <= hi_max && j0 + 15 >= lo_min);
        const bool s1 = j0 + 16 < pf || (j0 + 16 <= hi_max && j0 + 31 >= lo_min);
        if (!s0) sc.x = sc.y = 0.f;
        if (!s1) sc.z = sc.w = 0.f;
        // (so may their page, a window's left behind for one)
        if (any_lost) gone = s_lost[warp][kk % C::SCALES];
        if (lane == 0 && ((s0 && (gone & 1)) || (s1 && (gone & 2)))) report(a.status, kStatusBadIndex);
      }
      // ---------------- S^T = K Q^T
      float s[2][NT][4];
      uint4 kr[2][2][H];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = 16 * m + 8 * x + gid;
          const int sw = D == 128 ? row & 7 : (row >> 1) & 3;
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const uint32_t ad = kst + row * D + (((H * tig + h) ^ sw) << 4);
            uint4 &k4 = kr[m][x][h];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(k4.x), "=r"(k4.y), "=r"(k4.z), "=r"(k4.w)
                         : "r"(ad));
          }
        }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.f;
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int m = 0; m < 2; ++m) {  // (two chains of products side by side)
            auto word = [&](const uint4 &v) { return st == 0 ? v.x : st == 1 ? v.y : st == 2 ? v.z : v.w; };
            uint32_t ka[4];
            cache4_to_f16<CT>(word(kr[m][0][h]), ka[0], ka[2]);
            cache4_to_f16<CT>(word(kr[m][1][h]), ka[1], ka[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma_f16(s[m][n], ka, qf[n][h * 4 + st][0], qf[n][h * 4 + st][1]);
          }
      // V: the loads of the first VP parts of 16 keys go ahead of the softmax
      constexpr int VP = NT == 1 ? 2 : 1;
      uint32_t vr[2][MT / 2][4];
      auto load_v = [&](int m) {
#pragma unroll
        for (int c = 0; c < MT; c += 2) {
          const int key = 16 * m + (lane & 7) + ((lane >> 3) & 1) * 8, ch = c + (lane >> 4);
          const int sw = D == 128 ? key & 7 : (key >> 1) & 3;
          ldsm_x4_t(vst + key * D + ((ch ^ sw) << 4), vr[m][c / 2][0], vr[m][c / 2][1], vr[m][c / 2][2],
                    vr[m][c / 2][3]);
        }
      };
#pragma unroll
      for (int m = 0; m < VP; ++m) load_v(m);
      // ---------------- score modification, mask, normaliser
      // s[m][n][2 x + e]: key j0 + 16 m + 8 x + gid, row 8 n + 2 tig + e
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const float f = rowmul[n][e] * (m ? sc.z : sc.x), vf = m ? sc.w : sc.y;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float &v = s[m][n][2 * x + e];
              if (KIND == KIND_SOFTCAP) {
                // cap tanh(y) = cap - 2 cap / (e^(2y) + 1), to 2^-22 cap: the
                // approximate tanh instruction (2^-11) would show in P
                const float z = ptx::ex2(v * f);
                v = fmaf(a.softcap * LOG2E, fmaf(-2.f, ptx::rcp_fast(z + 1.f), 1.f), vf);
              } else if (KIND == KIND_ALIBI) {
                v = fmaf(slope[n][e], static_cast<float>(j0 + 16 * m + 8 * x + gid - posn[n][e]),
                         fmaf(v, f, vf));
              } else if (KIND == KIND_SIGMOID) {
                v = vf * ptx::rcp_fast(1.f + ptx::ex2(fmaf(v, f, -a.sig_bias * LOG2E)));
              } else if (KIND == KIND_RELU) {
                v *= f;
                v = v < 0.f ? 0.f : v * vf;  // (a NaN stays)
              } else {
                v = fmaf(v, f, vf);
              }
            }
          }
      if (!all) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i_pos = posn[n][e];
            int lo, hi;
            band32(a, i_pos, len, lo, hi);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int j = j0 + 16 * m + 8 * x + gid;
                const bool vis = ((real >> (2 * n + e)) & 1u) && !((gone >> m) & 1) &&
                                 (j < pf || (j >= lo && j <= hi &&
                                             (a.dil == 1 || divides(a.dil, i_pos - j))));
                if (!vis) s[m][n][2 * x + e] = SOFTMAX ? -INFINITY : 0.f;
              }
          }
      }
      {
        float mx[NT][2];
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mx[n][e] = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
            grow |= mx[n][e] > (SOFTMAX ? m_run[n][e] : ptx::ex2(m_run[n][e]));
          }
        if (__any_sync(0xffffffffu, grow)) {  // some row's maximum is exceeded
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v = mx[n][e];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
              if (!SOFTMAX)  // the power of two above it, as its logarithm
                v = static_cast<float>(static_cast<int>(__float_as_uint(v) >> 23) - 126);
              const float nm = fmaxf(m_run[n][e], v);
              const float al = ptx::ex2(m_run[n][e] - (nm == -INFINITY ? 0.f : nm));
              m_run[n][e] = nm;
              l_run[n][e] *= al;
#pragma unroll
              for (int c = 0; c < MT; ++c) {
                o[c][n][e] *= al;
                o[c][n][2 + e] *= al;
              }
            }
        }
      }
      const float il[2] = {SOFTMAX ? ptx::ex2(-sc.y) : 0.f, SOFTMAX ? ptx::ex2(-sc.w) : 0.f};
      // P as halves. Beside outputs of 8 bits (bf16) that rounding, 2^-12, is nothing;
      // outputs of 11 bits get what it left as halves too.
      uint32_t pb[2][NT][2], rest[2][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mu = m_run[n][e] == -INFINITY ? 0.f : m_run[n][e] - kPTop;
          const float down = SOFTMAX ? 0.f : ptx::ex2(-mu);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float &v = s[m][n][2 * x + e];
              if (SOFTMAX) {
                v = ptx::ex2(v - mu);
                sum += v;
              } else {
                v *= down;
              }
            }
            if (SOFTMAX) l_run[n][e] = fmaf(sum, il[m], l_run[n][e]);
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            pb[m][n][x] = movmatrix(ptx::pack_f16(s[m][n][2 * x], s[m][n][2 * x + 1]));
      }
      if (!BF16) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float p = s[m][n][2 * x], q = s[m][n][2 * x + 1];
              const float2 f = f16x2_to_float2(ptx::pack_f16(p, q));
              rest[m][n][x] = movmatrix(ptx::pack_f16(p - f.x, q - f.y));
            }
      }
      // ---------------- O^T += V^T P^T
      bool nan_seen = false;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (m + VP < 2) load_v(m + VP);
        if (CT == CACHE_E4M3 && !all) {  // NaN times a P of zero is not zero
          uint32_t some[2];  // bytes of keys 16 m + 8 x + 2 tig, + 1 that some row sees
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int j = j0 + 16 * m + 8 * x + 2 * tig;
            some[x] = (j < pf || (j >= lo_min && j <= hi_max) ? 0x0101u : 0u) |
                      (j + 1 < pf || (j + 1 >= lo_min && j + 1 <= hi_max) ? 0x01010000u : 0u);
            if ((gone >> m) & 1) some[x] = 0;
          }
#pragma unroll
          for (int c = 0; c < MT / 2; ++c)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t &v = vr[m][c][w];
              const uint32_t nan = (((v & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
              nan_seen |= (nan & some[w & 1]) != 0;
              v &= ~(nan * 0xffu);
            }
        }
        auto add_pv = [&](const uint32_t(&p)[NT][2]) {
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            uint32_t va[4];
            cache4_to_f16<CT>(__byte_perm(vr[m][c / 2][2 * (c & 1)], 0, 0x3120), va[0], va[1]);
            cache4_to_f16<CT>(__byte_perm(vr[m][c / 2][2 * (c & 1) + 1], 0, 0x3120), va[2], va[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(o[c][n], va, p[n][0], p[n][1]);
          }
        };
        add_pv(pb[m]);
        if (!BF16) add_pv(rest[m]);
      }
      if (CT == CACHE_E4M3 && !all && __any_sync(0xffffffffu, nan_seen)) {
        // The NaN values left out above go to the rows that do see their keys.
        for (int kk = 0; kk < TK; ++kk) {
          if ((gone >> (kk / 16)) & 1) continue;
          const int j = j0 + kk;
          const int sw = D == 128 ? kk & 7 : (kk >> 1) & 3;
          bool sees[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int i_pos = posn[n][e];
              int lo, hi;
              band32(a, i_pos, len, lo, hi);
              sees[n][e] = ((real >> (2 * n + e)) & 1u) &&
                           (j < pf || (j >= lo && j <= hi &&
                                       (a.dil == 1 || divides(a.dil, i_pos - j))));
            }
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            uint16_t two;
            asm volatile("ld.shared.u16 %0, [%1];"
                         : "=h"(two)
                         : "r"(vst + kk * D + ((c ^ sw) << 4) + 2 * gid));
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (((two >> (8 * y)) & 0x7f) == 0x7f)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (sees[n][e]) o[c][n][2 * y + e] = __int_as_float(0x7fffffff);
          }
        }
      }
      __syncwarp();  // all lanes are done with the stage
      issue(kk + NST);
    }
    k += nt;

    // ---------------- the unit's result, or this worker's part of it
    const bool begun = ut0 == 0, ended = ut0 + nt == tl.n;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
          l_run[n][e] += __shfl_xor_sync(0xffffffffu, l_run[n][e], d);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) m_run[n][e] -= kPTop;  // what O and the sum are relative to
    if (begun && ended) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * n + 2 * tig + e;
          const bool odd = gid & 1;
          float f;
          uint16_t *dst = row_out<KIND>(a, un, min(r, un.rows - 1), m_run[n][e], l_run[n][e],
                                        gid == 0 && r < un.rows, f) +
                          2 * (gid & ~1);
#pragma unroll
          for (int c = 0; c < MT; c += 2) {
            // neighbours in gid exchange, so that each has four channels of a row:
            // the even one of channel tile c, the odd one of the next
            const float x0 = __shfl_xor_sync(0xffffffffu, odd ? o[c][n][e] : o[c + 1][n][e], 4);
            const float x1 = __shfl_xor_sync(0xffffffffu, odd ? o[c][n][2 + e] : o[c + 1][n][2 + e], 4);
            if (r < un.rows) {
              if (odd)
                store4<BF16>(a, dst + 16 * (c + 1), f, x0, x1, o[c + 1][n][e], o[c + 1][n][2 + e]);
              else
                store4<BF16>(a, dst + 16 * c, f, o[c][n][e], o[c][n][2 + e], x0, x1);
            }
          }
        }
    } else {
      // A unit that goes on after this piece ends the worker's work: its part
      // waits for the other workers' in shared memory, in the rings once all
      // are spent. One that ended here began before: to the workspace.
      float *po = head_o(me), *pm = head_ml(me);
      int pitch = D;
      if (!ended) {
        has_end = true;
        if (lane == 0) s_end[warp] = un, s_has_end[warp] = begun ? 1 : 2;
        po = parts + warp * ROWS * PITCH;
        pm = &part_ml[warp][0][0];
        pitch = PITCH;
        rings_spent();
      } else if (lane == 0) {
        s_head[warp] = un, s_has_head[warp] = 1;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * n + 2 * tig + e;
#pragma unroll
          for (int c = 0; c < MT; ++c)
            *reinterpret_cast<float2 *>(po + r * pitch + 16 * c + 2 * gid) =
                make_float2(o[c][n][e], o[c][n][2 + e]);
          if (gid == 0) *reinterpret_cast<float2 *>(pm + 2 * r) = make_float2(m_run[n][e], l_run[n][e]);
        }
    }
    if (k < nk) begin_unit(k, line.entry_at(c0 + k));
  }
  if (!has_end) rings_spent();
  __syncthreads();

  // ================ the parts of this CTA's workers, in the order of the line
  if (t < 32) {
    const uint32_t heads = __ballot_sync(0xffffffffu, lane < kSplitWarps && s_has_head[lane & 7] != 0);
    const uint32_t ends = __ballot_sync(0xffffffffu, lane < kSplitWarps && s_has_end[lane & 7] != 0);
    const uint32_t mid = __ballot_sync(0xffffffffu, lane < kSplitWarps && s_has_end[lane & 7] == 2);
    if (lane == 0) {
      int n = 0;
      bool open = false;
      Group gr;
      for (int w = 0; w < kSplitWarps; ++w) {
        if ((heads >> w) & 1) {  // closes the open group, or one begun in an earlier CTA
          if (!open) gr.first = w, gr.before = true;
          gr.last = w, gr.last_is_head = true, gr.after = false;
          s_group[n++] = gr;
          open = false;
        }
        if ((ends >> w) & 1) {
          if (!open) gr.first = w, gr.before = (mid >> w) & 1;
          open = true;
          gr.last = w, gr.last_is_head = false, gr.after = true;
        }
      }
      if (open) s_group[n++] = gr;
      s_groups = n;
      s_ends = ends;
      s_last[0] = s_last[1] = 0;
    }
  }
  __syncthreads();
  const int groups = s_groups;
  auto unit_of = [&](const Group &gr) -> const Unit & {
    return gr.last_is_head ? s_head[gr.last] : s_end[gr.last];
  };
  auto add = [&](float4 &acc, float &L, float wt, const float4 &x, float l) {
    L = fmaf(wt, l, L);
    acc.x = fmaf(wt, x.x, acc.x);
    acc.y = fmaf(wt, x.y, acc.y);
    acc.z = fmaf(wt, x.z, acc.z);
    acc.w = fmaf(wt, x.w, acc.w);
  };
  constexpr int ITEMS = ROWS * (D / 4);  // of a unit: a row's four channels each
  for (int e = t; e < groups * ITEMS; e += kSplitThreads) {
    const Group &gr = s_group[e / ITEMS];
    const Unit &un = unit_of(gr);
    const int r = e % ITEMS / (D / 4), c4 = e % (D / 4);
    if (r >= un.rows) continue;
    // the workers' parts in shared memory, then the one in the workspace; all loads at once
    const uint32_t span = (2u << gr.last) - (1u << gr.first);
    const uint32_t in_smem = span & s_ends & ~(gr.last_is_head ? 1u << gr.last : 0u);
    float2 hml = make_float2(-INFINITY, 0.f);
    float4 hv = make_float4(0.f, 0.f, 0.f, 0.f);
    if (gr.last_is_head) {
      const int w = blockIdx.x * kSplitWarps + gr.last;
      hml = __ldcg(reinterpret_cast<const float2 *>(head_ml(w)) + r);
      hv = __ldcg(reinterpret_cast<const float4 *>(head_o(w) + r * D) + c4);
    }
    float2 x[kSplitWarps];
    float M = hml.x, L = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      x[w] = (in_smem >> w) & 1 ? make_float2(part_ml[w][r][0], part_ml[w][r][1])
                                : make_float2(-INFINITY, 0.f);
      M = fmaxf(M, x[w].x);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w)
      if ((in_smem >> w) & 1)
        add(acc, L, ptx::ex2(x[w].x - (M == -INFINITY ? 0.f : M)),
            *reinterpret_cast<const float4 *>(parts + (w * ROWS + r) * PITCH + 4 * c4), x[w].y);
    if (gr.last_is_head) add(acc, L, ptx::ex2(hml.x - (M == -INFINITY ? 0.f : M)), hv, hml.y);
    if (!gr.before && !gr.after) {
      float f;
      uint16_t *dst = row_out<KIND>(a, un, r, M, L, c4 == 0, f);
      store4<BF16>(a, dst + 4 * c4, f, acc.x, acc.y, acc.z, acc.w);
    } else {
      const int64_t slot = 2ll * blockIdx.x + (gr.before ? 0 : 1);
      *reinterpret_cast<float4 *>(a.part_o + (slot * ROWS + r) * D + 4 * c4) = acc;
      if (c4 == 0) *reinterpret_cast<float2 *>(a.part_ml + (slot * ROWS + r) * 2) = make_float2(M, L);
    }
  }
  if (groups == 0 || !(s_group[0].before || s_group[groups - 1].after)) return;

  // ================ the last CTA of a unit merges the CTAs' parts, in their order
  __syncthreads();
  if (t < 2 && (t == 0 ? s_group[0].before : s_group[groups - 1].after && !s_group[groups - 1].before)) {
    const Unit &un = unit_of(s_group[t == 0 ? 0 : groups - 1]);
    const int first = line.cta_of(un, 0), last = line.cta_of(un, un.n - 1);
    const unsigned parts_less_1 = last - first;
    s_first_cta[t] = first, s_last_cta[t] = last;
    __threadfence();  // (the CTA's parts, seen through the barrier, before the ticket)
    // counts the unit's CTAs and wraps to zero
    s_last[t] = atomicInc(reinterpret_cast<unsigned *>(a.tickets) + first, parts_less_1) == parts_less_1;
    __threadfence();
  }
  __syncthreads();
  for (int x = 0; x < 2; ++x) {
    if (!s_last[x]) continue;
    const Unit &un = unit_of(s_group[x == 0 ? 0 : groups - 1]);
    const int first = s_first_cta[x], last = s_last_cta[x];
    for (int e = t; e < un.rows * (D / 4); e += kSplitThreads) {
      const int r = e / (D / 4), c4 = e % (D / 4);
      float M = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      merge_parts<ROWS, D>(a, first, last, r, c4, M, L, acc);
      float f;
      uint16_t *dst = row_out<KIND>(a, un, r, M, L, c4 == 0, f);
      store4<BF16>(a, dst + 4 * c4, f, acc.x, acc.y, acc.z, acc.w);
    }
  }
}

// Launches of one head size and cache type; each has a source file of its own.
template <int D, int CT>
cudaError_t launch_split(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a, int kind,
                         int tiles, int grid, int device, cudaStream_t s);

template <int D, int CT, int NT, int KIND, bool BF16>
cudaError_t launch_split_one(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a,
                             int grid, int device, cudaStream_t s) {
  static std::atomic<uint64_t> set{0};
  constexpr int bytes = SplitConfig<D, NT>::SMEM;
  const cudaError_t e = allow_smem(
      reinterpret_cast<const void *>(&paged_split_kernel<D, CT, NT, KIND, BF16>), bytes, device, set);
  if (e != cudaSuccess) return e;
  return launch_after(paged_split_kernel<D, CT, NT, KIND, BF16>, dim3(grid), kSplitThreads, bytes, s, mk, mv, a);
}

template <int D, int CT, int NT, bool BF16>
cudaError_t launch_split_kind(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a,
                              int kind, int grid, int device, cudaStream_t s) {
  switch (kind) {
    case KIND_SOFTCAP: return launch_split_one<D, CT, NT, KIND_SOFTCAP, BF16>(mk, mv, a, grid, device, s);
    case KIND_ALIBI: return launch_split_one<D, CT, NT, KIND_ALIBI, BF16>(mk, mv, a, grid, device, s);
    case KIND_SIGMOID: return launch_split_one<D, CT, NT, KIND_SIGMOID, BF16>(mk, mv, a, grid, device, s);
    case KIND_RELU: return launch_split_one<D, CT, NT, KIND_RELU, BF16>(mk, mv, a, grid, device, s);
    default: return launch_split_one<D, CT, NT, KIND_SOFTMAX, BF16>(mk, mv, a, grid, device, s);
  }
}

#define CHIA_INSTANTIATE_SPLIT(D, CT)                                                           \
  template <>                                                                                   \
  cudaError_t chia::launch_split<D, CT>(const CUtensorMap &mk, const CUtensorMap &mv,           \
                                        const PagedArgs &a, int kind, int tiles, int grid,      \
                                        int device, cudaStream_t s) {                           \
    if (a.bf16)                                                                                 \
      return tiles == 1 ? launch_split_kind<D, CT, 1, true>(mk, mv, a, kind, grid, device, s)   \
                        : launch_split_kind<D, CT, 2, true>(mk, mv, a, kind, grid, device, s);  \
    return tiles == 1 ? launch_split_kind<D, CT, 1, false>(mk, mv, a, kind, grid, device, s)    \
                      : launch_split_kind<D, CT, 2, false>(mk, mv, a, kind, grid, device, s);   \
  }

}  // namespace chia
