// paged_split_sm100.cuh -- attention of few queries over the paged 8-bit K/V
// cache: decode steps and drafted tokens.
//
// Every key and value byte is read once and used by group * queries rows, so
// the work is bound by HBM as long as nothing else is in its way. The grid is
// one wave of CTAs; all (request, K/V head, block of rows) units with their
// 32-key tiles form one line of tiles, of which each CTA takes an equal piece,
// whatever the lengths. A unit that is cut by CTAs' borders leaves partial
// results, and the last CTA to finish merges them in a fixed order.
//
// A CTA: four compute warps and one that loads. The load warp looks up 32
// tiles' pages and scales at a time, a tile a lane, and keeps a ring of tiles
// in flight by TMA (tiled copies with a swizzle that keeps the reads below free
// of bank conflicts). A tile is consumed by one compute warp alone (or by one
// warp of each row group), with its own running maximum, sum and output: no
// barrier between warps until the unit ends.
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
// (11 bits) after it is multiplied by its page's value scale over the largest
// such scale seen: it stays within [0, 1] whatever the scales are.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "decode_sm100.cuh"
#include "paged_common.cuh"

namespace chia {

struct PagedArgs {
  const void *q;
  void *o;
  int64_t q_st, q_sh, o_st, o_sh;  // element strides: token, head
  const float *k_scale, *v_scale;
  const int32_t *block_table, *seq_lens, *cu_q;
  int64_t table_stride;
  float *lse;
  const float *head_param;
  int32_t left, right, block, prefix, dil;  // the mask, on positions (at most 2^30 each)
  float score_scale, softcap, sig_bias, out_scale;
  int32_t heads, heads_kv, group, batch, tokens, page, width;
  int32_t num_pages;
  int32_t q_each;     // queries of a request where cu_q is null
  int32_t token0;     // first token of request 0 where cu_q is null
  int32_t row_groups; // 1, 2 or 4: compute warps that share a tile
  int32_t bf16;       // type of q and o
  int32_t *tickets;   // [gridDim.x], zero between launches
  float *part_o;      // [2 gridDim.x][rows][D]
  float *part_ml;     // [2 gridDim.x][rows][2]
  int32_t *status;
  uint64_t timeout_ns, drain_ns;
};

constexpr int kSplitMaxBatch = 1024;  // requests of one launch (prefix sums in shared memory)
constexpr int kSplitThreads = 160;

// Queries and keys of request b, checked: [t0, t0 + n) of q, keys [0, len).
struct Request {
  int t0, n, len;
};
__device__ __forceinline__ Request request_of(const PagedArgs &a, int b, bool &bad) {
  Request r;
  if (a.cu_q != nullptr) {
    r.t0 = a.cu_q[b];
    const int t1 = a.cu_q[b + 1];
    if (r.t0 < 0 || t1 < r.t0 || t1 > a.tokens) {
      bad = true;
      r.t0 = r.n = 0;
    } else {
      r.n = t1 - r.t0;
    }
  } else {
    r.t0 = a.token0 + b * a.q_each;
    r.n = a.q_each;
  }
  r.len = a.seq_lens[b];
  const int most = a.width * a.page;
  if (r.len < 0 || r.len > most) {
    bad = true;
    r.len = r.len < 0 ? 0 : most;
  }
  return r;
}

// The keys position i sees beside the prefix (position_band in 32 bits).
__device__ __forceinline__ void band32(const PagedArgs &a, int i, int len, int &lo, int &hi) {
  lo = 0;
  hi = len - 1;
  if (a.left >= 0) lo = max(lo, i - a.left);
  if (a.right >= 0) hi = min(hi, i + a.right);
  if (a.block > 0) {
    const int b0 = (i >= 0 ? i / a.block : -((-i + a.block - 1) / a.block)) * a.block;
    lo = max(lo, b0);
    hi = min(hi, b0 + a.block - 1);
  }
}

// Tiles of TK keys that queries at positions [p0, p1] visit: `pre` tiles from
// key 0 on, then those from `lo` on; `n` in all, at least one (a unit whose
// rows see nothing still writes zeros).
struct Tiles {
  int pre, lo, n;
  __device__ __forceinline__ int key_tile(int t) const { return t < pre ? t : lo + (t - pre); }
};
template <int TK>
__device__ __forceinline__ Tiles tiles_of(const PagedArgs &a, int p0, int p1, int len) {
  Tiles r;
  int lo, hi, x;
  band32(a, p0, len, lo, x);
  band32(a, p1, len, x, hi);
  const int pf = min(a.prefix, len);
  r.pre = (pf + TK - 1) / TK;
  r.lo = r.pre;
  int n = r.pre;
  if (lo <= hi) {
    r.lo = max(lo / TK, r.pre);
    n += max(0, hi / TK + 1 - r.lo);
  }
  r.n = max(n, 1);
  return r;
}

// A wait of limited length. After one has run out (`abort`), all return at once.
__device__ __forceinline__ bool split_wait(uint32_t bar, uint32_t parity, volatile int *abort,
                                           const PagedArgs &a) {
  if (ptx::mbar_test_wait(bar, parity)) return true;
  const uint64_t t0 = ptx::globaltimer_ns();
  while (!ptx::mbar_try_wait(bar, parity, 20000u)) {
    if (*abort) return false;
    if (ptx::globaltimer_ns() - t0 > a.timeout_ns) {
      *abort = 1;
      report(a.status, 5);  // CHIA_ERR_DEVICE_TIMEOUT
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// 8x8 16-bit matrix, one row a quad of lanes: transposed
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void bar_compute() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int D, int NT>
struct SplitConfig {
  static constexpr int TK = 32;                     // keys of a tile
  static constexpr int STAGE = 2 * TK * D;          // bytes: K, then V
  static constexpr int NST = (NT == 1 ? 10 : 8) * (128 / D);  // 80 or 64 KB of tiles
  static constexpr int ROWS = 8 * NT;               // rows of a row group
  static constexpr int PITCH = D + 4;               // floats of a row in the merge buffer
  static constexpr int MERGE = 4 * ROWS * (PITCH + 2) * 4;
  static constexpr int SCALES = 64;                 // tiles whose scales are held
  static constexpr int SMEM = 1024 + NST * STAGE + MERGE + SCALES * 16;
};

// Grid: at most two CTAs an SM. KIND: score modification and normaliser.
template <int D, int CT, int NT, int KIND>
__global__ void __launch_bounds__(kSplitThreads, 2)
paged_split_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                   const PagedArgs a) {
  using C = SplitConfig<D, NT>;
  constexpr int TK = C::TK, NST = C::NST, ROWS = C::ROWS, PITCH = C::PITCH;
  constexpr int H = D / 64;   // 16-byte pieces of a key row a lane
  constexpr int MT = D / 16;  // channel tiles of the output
  constexpr bool SOFTMAX = KIND == KIND_SOFTMAX || KIND == KIND_SOFTCAP || KIND == KIND_ALIBI;
  constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
  extern __shared__ uint8_t dyn[];
  uint8_t *sm = dyn + ((1024u - (ptx::smem_u32(dyn) & 1023u)) & 1023u);
  float *mo = reinterpret_cast<float *>(sm + NST * C::STAGE);  // [4][ROWS][PITCH]
  float *mml = mo + 4 * ROWS * PITCH;                          // [4][ROWS][2]
  float4 *scales = reinterpret_cast<float4 *>(mml + 4 * ROWS * 2);  // ks, vs of keys 0-15, 16-31
  __shared__ long long pre[kSplitMaxBatch + 1];
  __shared__ long long wsum[5];
  __shared__ __align__(8) uint64_t bars[2 * NST];
  __shared__ volatile int abort_flag;
  __shared__ int s_last;

  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int RG = a.row_groups, KW = 4 / RG, RPB = ROWS * RG;
  const uint32_t ring = ptx::smem_u32(sm), bar0 = ptx::smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (NST + s); };
  if (t < NST) {
    ptx::mbar_init(full(t), 1);
    ptx::mbar_init(empty(t), RG);
  }
  if (t == 0) abort_flag = 0;
  if (t == 128) {
    ptx::tma_prefetch_desc(&mk);
    ptx::tma_prefetch_desc(&mv);
  }

  // ---- the line of tiles: pre[b] is where request b's begin
  {
    const int per = (a.batch + kSplitThreads - 1) / kSplitThreads;
    const int b0 = t * per, b1 = min(a.batch, b0 + per);
    long long sum = 0;
    bool bad = false;
    for (int b = b0; b < b1; ++b) {
      const Request r = request_of(a, b, bad);
      long long n = 0;
      if (r.n > 0)
        n = static_cast<long long>(tiles_of<TK>(a, r.len - r.n, r.len - 1, r.len).n) * a.heads_kv *
            ((static_cast<long long>(r.n) * a.group + RPB - 1) / RPB);
      pre[b + 1] = n;
      sum += n;
    }
    if (bad && blockIdx.x == 0) report(a.status, kStatusBadIndex);
    long long inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += u;
    }
    if (lane == 31) wsum[warp] = inc;
    ptx::fence_barrier_init();
    __syncthreads();
    long long at = inc - sum;
    for (int w = 0; w < warp; ++w) at += wsum[w];
    for (int b = b0; b < b1; ++b) {
      at += pre[b + 1];
      pre[b + 1] = at;
    }
    if (t == 0) pre[0] = 0;
    __syncthreads();
  }
  const long long total = pre[a.batch];
  // no more CTAs than give each compute warp a tile
  long long ctas = (total + KW - 1) / KW;
  if (ctas > gridDim.x) ctas = gridDim.x;
  if (blockIdx.x >= ctas) return;
  const long long c0 = total * blockIdx.x / ctas, c1 = total * (blockIdx.x + 1) / ctas;
  auto request_at = [&](long long g) {  // the request of tile g
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= g)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  };

  if (warp == 4) {
    // ================================================= the load warp
    long long seq = 0;  // tiles issued
    bool ok = true;
    for (long long base = c0; base < c1 && ok; base += 32) {
      const int n = static_cast<int>(min(32ll, c1 - base));
      int row0 = -1, row1 = -1, tok = 0;  // rows of the tensor map (page * heads_kv + head)
      float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane < n) {
        const long long g = base + lane;
        const int b = request_at(g);
        bool bad = false;
        const Request r = request_of(a, b, bad);
        const Tiles tl = tiles_of<TK>(a, r.len - r.n, r.len - 1, r.len);
        const long long in = g - pre[b];
        const int nrb = (r.n * a.group + RPB - 1) / RPB;
        const int hk = static_cast<int>(in / tl.n) / nrb;
        const int key = tl.key_tile(static_cast<int>(in % tl.n)) * TK;
        const int32_t *table = a.block_table + b * a.table_stride;
        tok = key % a.page;
        int p0 = -1, p1 = -1;
        if (key < r.len) p0 = table[key / a.page];
        if (a.page == 16 && key + 16 < r.len) p1 = table[key / 16 + 1];
        if (key < r.len) {
          if (p0 < 0 || p0 >= a.num_pages)
            bad = true, p0 = -1;
          else
            row0 = p0 * a.heads_kv + hk;
        }
        if (a.page == 16 && key + 16 < r.len) {
          if (p1 < 0 || p1 >= a.num_pages)
            bad = true, p1 = -1;
          else
            row1 = p1 * a.heads_kv + hk;
        }
        if (bad) report(a.status, kStatusBadIndex);
      }
      auto issue = [&](int i) {  // wait for the stage, start its copies
        const int stage = static_cast<int>((seq + i) % NST);
        const uint32_t par = static_cast<uint32_t>((seq + i) / NST) & 1u;
        if (!split_wait(empty(stage), par ^ 1u, &abort_flag, a)) return false;
        const int r0 = __shfl_sync(0xffffffffu, row0, i), r1 = __shfl_sync(0xffffffffu, row1, i);
        const int tk = __shfl_sync(0xffffffffu, tok, i);
        if (lane == 0) {
          const uint32_t dst = ring + stage * C::STAGE;
          const int rows = a.page == 16 ? 16 : TK;
          mbar_expect_tx(full(stage), ((r0 >= 0) + (r1 >= 0)) * 2 * rows * D);
          if (r0 >= 0) {
            tma_load_3d(dst, &mk, full(stage), 0, tk, r0);
            tma_load_3d(dst + TK * D, &mv, full(stage), 0, tk, r0);
          }
          if (r1 >= 0) {
            tma_load_3d(dst + 16 * D, &mk, full(stage), 0, 0, r1);
            tma_load_3d(dst + TK * D + 16 * D, &mv, full(stage), 0, 0, r1);
          }
        }
        return true;
      };
      // the first copies leave before the scales are here
      const int early = min(n, NST);
      int done = 0;
      for (; done < early && ok; ++done) ok = issue(done);
      if (row0 >= 0) sc.x = a.k_scale[row0], sc.y = a.v_scale[row0];
      if (a.page != 16)
        sc.z = sc.x, sc.w = sc.y;
      else if (row1 >= 0)
        sc.z = a.k_scale[row1], sc.w = a.v_scale[row1];
      scales[(seq + lane) % C::SCALES] = sc;
      __syncwarp();
      if (!ok) --done;
      if (lane == 0)
        for (int i = 0; i < done; ++i) ptx::mbar_arrive(full((seq + i) % NST));
      for (int i = early; i < n && ok; ++i) {
        ok = issue(i);
        if (ok) {
          if (lane == 0) ptx::mbar_arrive(full((seq + i) % NST));
          ++done;
        }
      }
      seq += done;
    }
    // no copy of this CTA is in flight when it exits
    PagedArgs d = a;
    d.timeout_ns = a.drain_ns;
    int none = 0;
    for (long long i = seq > NST ? seq - NST : 0; i < seq; ++i)
      split_wait(full(i % NST), static_cast<uint32_t>(i / NST) & 1u, &none, d);
    return;
  }

  // =================================================== compute warps
  const int gid = lane >> 2, tig = lane & 3;
  const int rg = warp % RG, kw = warp / RG;
  long long seq = 0;
  for (long long g = c0; g < c1;) {
    const int b = request_at(g);
    bool bad = false;
    const Request rq = request_of(a, b, bad);
    const int p0 = rq.len - rq.n;
    const Tiles tl = tiles_of<TK>(a, p0, rq.len - 1, rq.len);
    const long long in = g - pre[b];
    const int nrows_all = rq.n * a.group;
    const int nrb = (nrows_all + RPB - 1) / RPB;
    const int ut0 = static_cast<int>(in % tl.n), u = static_cast<int>(in / tl.n);
    const int hk = u / nrb, rb = u % nrb;
    const long long ustart = g - ut0, uend = ustart + tl.n;
    const int nt = static_cast<int>(min(uend, c1) - g);
    const int row_base = rb * RPB;                       // rows of this unit: [row_base, row_end)
    const int row_end = min(nrows_all, row_base + RPB);
    // all rows of the unit see keys [lo_max, hi_min]; none sees one outside [lo_min, hi_max]
    int lo_min, lo_max, hi_min, hi_max;
    band32(a, p0 + row_base / a.group, rq.len, lo_min, hi_min);
    band32(a, p0 + (row_end - 1) / a.group, rq.len, lo_max, hi_max);
    const int pf = min(a.prefix, rq.len);

    // ---- Q: row rg * ROWS + 8 n + gid, channels 16 (H tig + h) + 4 s .. + 3 of step (h, s)
    uint32_t qf[NT][H * 4][2];
    float rowmul[NT][2], slope[NT][2];  // rows 8 n + 2 tig + e, as in the columns of S^T
    int posn[NT][2];
    uint32_t real = 0;  // bit 2 n + e: that row exists
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row_base + rg * ROWS + 8 * n + gid;
      uint4 raw[H * 2];
      if (row < row_end) {
        const uint16_t *src = static_cast<const uint16_t *>(a.q) +
                              static_cast<int64_t>(rq.t0 + row / a.group) * a.q_st +
                              (hk * a.group + row % a.group) * a.q_sh + H * 16 * tig;
#pragma unroll
        for (int c = 0; c < H * 2; ++c) raw[c] = *reinterpret_cast<const uint4 *>(src + 8 * c);
      } else {
#pragma unroll
        for (int c = 0; c < H * 2; ++c) raw[c] = make_uint4(0, 0, 0, 0);
      }
      float mx = 0.f;
      auto get = [&](int w, float2 &x) {  // 32-bit word w of the lane's channels
        const uint4 &r4 = raw[w / 4];
        const uint32_t v = w % 4 == 0 ? r4.x : w % 4 == 1 ? r4.y : w % 4 == 2 ? r4.z : r4.w;
        x = a.bf16 ? in16x2_to_float2<true>(v) : in16x2_to_float2<false>(v);
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
      const int src_row = row_base + rg * ROWS + 8 * n + 2 * tig;
      const float down = pow2f(e - 14);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f = __shfl_sync(0xffffffffu, down, (2 * tig + x) * 4);
        const int r = min(src_row + x, row_end - 1);
        const float hp = a.head_param != nullptr ? a.head_param[hk * a.group + r % a.group] : 1.f;
        posn[n][x] = p0 + r / a.group;
        real |= (src_row + x < row_end ? 1u : 0u) << (2 * n + x);
        float mul = a.score_scale * f;
        slope[n][x] = 0.f;
        if (KIND == KIND_SOFTMAX) mul *= LOG2E * hp;
        if (KIND == KIND_SOFTCAP) mul *= 2.f * LOG2E / a.softcap;  // 2^(2 log2e s / cap) = e^(2s/cap)
        if (KIND == KIND_ALIBI) mul *= LOG2E, slope[n][x] = hp * LOG2E;
        if (KIND == KIND_SIGMOID) mul *= -LOG2E;
        rowmul[n][x] = mul;
      }
    }
    float o[MT][NT][4], m_run[NT][2], l_run[NT][2], vref = 0.f, inv_vref = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < MT; ++c) o[c][n][0] = o[c][n][1] = o[c][n][2] = o[c][n][3] = 0.f;
      m_run[n][0] = m_run[n][1] = SOFTMAX ? -INFINITY : KIND == KIND_RELU ? -120.f : 0.f;
      l_run[n][0] = l_run[n][1] = 0.f;
    }

    for (int i = (kw - static_cast<int>(seq % KW) + KW) % KW; i < nt; i += KW) {
      const int stage = static_cast<int>((seq + i) % NST);
      const uint32_t par = static_cast<uint32_t>((seq + i) / NST) & 1u;
      if (!split_wait(full(stage), par, &abort_flag, a)) break;
      __syncwarp();
      const int j0 = tl.key_tile(ut0 + i) * TK;
      float4 sc = scales[(seq + i) % C::SCALES];
      const uint32_t kst = ring + stage * C::STAGE, vst = kst + TK * D;
      const bool all = a.dil == 1 ? (j0 >= lo_max && j0 + TK - 1 <= hi_min) || j0 + TK <= pf
                                  : j0 + TK <= pf;
      if (!all) {  // the scales of 16 keys that nobody sees may be anything
        const bool s0 = j0 < pf || (j0 <= hi_max && j0 + 15 >= lo_min);
        const bool s1 = j0 + 16 < pf || (j0 + 16 <= hi_max && j0 + 31 >= lo_min);
        if (!s0) sc.x = sc.y = 0.f;
        if (!s1) sc.z = sc.w = 0.f;
      }
      // ---------------- S^T = K Q^T
      float s[2][NT][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.f;
        uint4 kr[2][H];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = 16 * m + 8 * x + gid;
          const int sw = D == 128 ? row & 7 : (row >> 1) & 3;
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const uint32_t ad = kst + row * D + (((H * tig + h) ^ sw) << 4);
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(kr[x][h].x), "=r"(kr[x][h].y), "=r"(kr[x][h].z), "=r"(kr[x][h].w)
                         : "r"(ad));
          }
        }
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int st = 0; st < 4; ++st) {
            auto word = [&](const uint4 &v) { return st == 0 ? v.x : st == 1 ? v.y : st == 2 ? v.z : v.w; };
            uint32_t ka[4];
            cache4_to_f16<CT>(word(kr[0][h]), ka[0], ka[2]);
            cache4_to_f16<CT>(word(kr[1][h]), ka[1], ka[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma16816<false>(s[m][n], ka, qf[n][h * 4 + st][0], qf[n][h * 4 + st][1]);
          }
      }
      // ---------------- score modification, mask, normaliser
      // s[m][n][2 x + e]: key j0 + 16 m + 8 x + gid, row 8 n + 2 tig + e
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const float f = rowmul[n][e] * (m ? sc.z : sc.x);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float &v = s[m][n][2 * x + e];
              if (KIND == KIND_SOFTCAP) {
                // cap tanh(y) = cap - 2 cap / (e^(2y) + 1), to 2^-22 cap: the
                // approximate tanh instruction (2^-11) would show in P
                const float z = ptx::ex2(v * f);
                v = a.softcap * LOG2E * fmaf(-2.f, ptx::rcp_fast(z + 1.f), 1.f);
              } else if (KIND == KIND_ALIBI) {
                v = fmaf(slope[n][e],
                         static_cast<float>(j0 + 16 * m + 8 * x + gid - posn[n][e]), v * f);
              } else if (KIND == KIND_SIGMOID) {
                v = ptx::rcp_fast(1.f + ptx::ex2(fmaf(v, f, -a.sig_bias * LOG2E)));
              } else if (KIND == KIND_RELU) {
                v *= f;
                v = v < 0.f ? 0.f : v;  // (a NaN stays)
              } else {
                v *= f;
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
            band32(a, i_pos, rq.len, lo, hi);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int j = j0 + 16 * m + 8 * x + gid;
                const bool vis = ((real >> (2 * n + e)) & 1u) &&
                                 (j < pf || (j >= lo && j <= hi &&
                                             (a.dil == 1 || (i_pos - j) % a.dil == 0)));
                if (!vis) s[m][n][2 * x + e] = SOFTMAX ? -INFINITY : 0.f;
              }
          }
      }
      if (SOFTMAX || KIND == KIND_RELU) {
        float mx[NT][2];
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mx[n][e] = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
            grow |= KIND == KIND_RELU ? mx[n][e] > ptx::ex2(m_run[n][e]) : mx[n][e] > m_run[n][e];
          }
        if (__any_sync(0xffffffffu, grow)) {  // some row's maximum is exceeded
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v = mx[n][e];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
              if (KIND == KIND_RELU)  // the power of two above it, as its logarithm
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
      // the values' scales, relative to the largest power of two above one so far
      {
        const float vm = fmaxf(sc.y, sc.w);
        if (vm > vref) {
          const uint32_t bits = __float_as_uint(vm);
          const float up = __uint_as_float(min((bits + 0x7fffffu) & 0xff800000u, 0x7f000000u));
          const float al = vref * __frcp_rn(up);  // (exact: powers of two)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < MT; ++c)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[c][n][x] *= al;
          vref = up;
          inv_vref = __frcp_rn(up);
        }
      }
      const float r0 = sc.y * inv_vref, r1 = sc.w * inv_vref;
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mu = m_run[n][e] == -INFINITY ? 0.f : m_run[n][e];
          const float down = KIND == KIND_RELU ? ptx::ex2(-mu) : 1.f;
          float sum = 0.f;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float &v = s[m][n][2 * x + e];
              if (SOFTMAX) {
                v = ptx::ex2(v - mu);
                sum += v;
              }
              v *= (m ? r1 : r0) * down;
            }
          l_run[n][e] += sum;
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            pb[m][n][x] = movmatrix(ptx::pack_f16(s[m][n][2 * x], s[m][n][2 * x + 1]));
      }
      // ---------------- O^T += V^T P^T
      bool nan_seen = false;
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c = 0; c < MT; c += 2) {
          const int key = 16 * m + (lane & 7) + ((lane >> 3) & 1) * 8, ch = c + (lane >> 4);
          const int sw = D == 128 ? key & 7 : (key >> 1) & 3;
          uint32_t v[4];
          ldsm_x4_t(vst + key * D + ((ch ^ sw) << 4), v[0], v[1], v[2], v[3]);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if (CT == CACHE_E4M3 && !all) {  // NaN times a P of zero is not zero
              const uint32_t nan = (((v[w] & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
              nan_seen |= nan != 0;
              v[w] &= ~(nan * 0xffu);
            }
            v[w] = __byte_perm(v[w], 0, 0x3120);
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t va[4];
            cache4_to_f16<CT>(v[2 * y], va[0], va[1]);
            cache4_to_f16<CT>(v[2 * y + 1], va[2], va[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<false>(o[c + y][n], va, pb[m][n][0], pb[m][n][1]);
          }
        }
      if (CT == CACHE_E4M3 && !all && __any_sync(0xffffffffu, nan_seen)) {
        // The NaN values left out above go to the rows that do see their keys.
        for (int kk = 0; kk < TK; ++kk) {
          const int j = j0 + kk;
          const int sw = D == 128 ? kk & 7 : (kk >> 1) & 3;
          bool sees[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int i_pos = posn[n][e];
              int lo, hi;
              band32(a, i_pos, rq.len, lo, hi);
              sees[n][e] = ((real >> (2 * n + e)) & 1u) &&
                           (j < pf || (j >= lo && j <= hi &&
                                       (a.dil == 1 || (i_pos - j) % a.dil == 0)));
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
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(empty(stage));
    }
    seq += nt;

    // ---------------- merge the key warps
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[n][e];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        const int r = 8 * n + 2 * tig + e;
        float *dst = mo + (warp * ROWS + r) * PITCH + 2 * gid;
#pragma unroll
        for (int c = 0; c < MT; ++c)
          *reinterpret_cast<float2 *>(dst + 16 * c) =
              make_float2(o[c][n][e] * vref, o[c][n][2 + e] * vref);
        if (gid == 0) {
          mml[(warp * ROWS + r) * 2] = m_run[n][e];
          mml[(warp * ROWS + r) * 2 + 1] = l;
        }
      }
    bar_compute();
    const bool whole = ustart >= c0 && uend <= c1;
    const int64_t slot = 2ll * blockIdx.x + (ustart < c0 ? 0 : 1);
    const int rows = row_end - row_base;
    auto store = [&](int r, int c4, float4 acc, float M, float L) {  // a row's four channels
      float f = 1.f;
      if (SOFTMAX) f = L > 0.f ? 1.f / L : L;  // (a NaN stays)
      if (KIND == KIND_RELU) f = a.out_scale * ptx::ex2(M);
      const int qi = (row_base + r) / a.group, hh = hk * a.group + (row_base + r) % a.group;
      const int64_t tok = rq.t0 + qi;
      uint16_t *dst = static_cast<uint16_t *>(a.o) + tok * a.o_st + hh * a.o_sh + 4 * c4;
      acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
      *reinterpret_cast<uint2 *>(dst) =
          a.bf16 ? make_uint2(ptx::pack_bf16(acc.x, acc.y), ptx::pack_bf16(acc.z, acc.w))
                 : make_uint2(ptx::pack_f16(acc.x, acc.y), ptx::pack_f16(acc.z, acc.w));
      if (SOFTMAX && a.lse != nullptr && c4 == 0)
        a.lse[tok * a.heads + hh] = L > 0.f ? (M + __log2f(L)) * LN2 : L == 0.f ? -INFINITY : L;
    };
    for (int e = t; e < rows * (D / 4); e += 128) {
      const int r = e / (D / 4), c4 = e % (D / 4);
      const int w0 = r / ROWS, rr = r % ROWS;  // warps w0, w0 + RG, ...
      float M = -INFINITY, L = 0.f;
      for (int k = 0; k < KW; ++k) M = fmaxf(M, mml[((w0 + k * RG) * ROWS + rr) * 2]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < KW; ++k) {
        const int w = (w0 + k * RG) * ROWS + rr;
        const float wt = ptx::ex2(mml[w * 2] - (M == -INFINITY ? 0.f : M));
        const float4 x = *reinterpret_cast<const float4 *>(mo + w * PITCH + 4 * c4);
        L = fmaf(wt, mml[w * 2 + 1], L);
        acc.x = fmaf(wt, x.x, acc.x);
        acc.y = fmaf(wt, x.y, acc.y);
        acc.z = fmaf(wt, x.z, acc.z);
        acc.w = fmaf(wt, x.w, acc.w);
      }
      if (whole) {
        store(r, c4, acc, M, L);
      } else {
        *reinterpret_cast<float4 *>(a.part_o + (slot * RPB + r) * D + 4 * c4) = acc;
        if (c4 == 0)
          *reinterpret_cast<float2 *>(a.part_ml + (slot * RPB + r) * 2) = make_float2(M, L);
      }
    }
    if (!whole) {
      // ---------------- the last of the unit's CTAs merges its parts, in their order
      auto cta_of = [&](long long x) { return static_cast<int>(((x + 1) * ctas - 1) / total); };
      const int first = cta_of(ustart), last = cta_of(uend - 1);
      __threadfence();
      bar_compute();
      if (t == 0)  // counts up to the number of parts and wraps to zero
        s_last = atomicInc(reinterpret_cast<unsigned *>(a.tickets) + first,
                           static_cast<unsigned>(last - first)) ==
                 static_cast<unsigned>(last - first);
      bar_compute();
      if (s_last) {
        __threadfence();
        for (int e = t; e < rows * (D / 4); e += 128) {
          const int r = e / (D / 4), c4 = e % (D / 4);
          auto part = [&](int c) { return (2ll * c + (c == first ? 1 : 0)) * RPB + r; };
          float M = -INFINITY, L = 0.f;
          for (int c = first; c <= last; ++c) M = fmaxf(M, __ldcg(a.part_ml + part(c) * 2));
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int c = first; c <= last; ++c) {
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(a.part_ml + part(c) * 2));
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(a.part_o + part(c) * D + 4 * c4));
            const float wt = ptx::ex2(ml.x - (M == -INFINITY ? 0.f : M));
            L = fmaf(wt, ml.y, L);
            acc.x = fmaf(wt, x.x, acc.x);
            acc.y = fmaf(wt, x.y, acc.y);
            acc.z = fmaf(wt, x.z, acc.z);
            acc.w = fmaf(wt, x.w, acc.w);
          }
          store(r, c4, acc, M, L);
        }
      }
    }
    bar_compute();  // the merge buffer is free again
    g += nt;
  }
}

// Launches of one head size and cache type; each has a source file of its own.
template <int D, int CT>
cudaError_t launch_split(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a, int kind,
                         int tiles, int grid, int device, cudaStream_t s);

// Once for each kernel and device.
inline cudaError_t allow_smem(const void *kernel, int bytes, int device, std::atomic<uint64_t> &set) {
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (set.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) set.fetch_or(bit, std::memory_order_release);
  return e;
}

template <int D, int CT, int NT, int KIND>
cudaError_t launch_split_one(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a,
                             int grid, int device, cudaStream_t s) {
  static std::atomic<uint64_t> set{0};
  constexpr int bytes = SplitConfig<D, NT>::SMEM;
  const cudaError_t e = allow_smem(
      reinterpret_cast<const void *>(&paged_split_kernel<D, CT, NT, KIND>), bytes, device, set);
  if (e != cudaSuccess) return e;
  paged_split_kernel<D, CT, NT, KIND><<<grid, kSplitThreads, bytes, s>>>(mk, mv, a);
  return cudaGetLastError();
}

template <int D, int CT, int NT>
cudaError_t launch_split_kind(const CUtensorMap &mk, const CUtensorMap &mv, const PagedArgs &a,
                              int kind, int grid, int device, cudaStream_t s) {
  switch (kind) {
    case KIND_SOFTCAP: return launch_split_one<D, CT, NT, KIND_SOFTCAP>(mk, mv, a, grid, device, s);
    case KIND_ALIBI: return launch_split_one<D, CT, NT, KIND_ALIBI>(mk, mv, a, grid, device, s);
    case KIND_SIGMOID: return launch_split_one<D, CT, NT, KIND_SIGMOID>(mk, mv, a, grid, device, s);
    case KIND_RELU: return launch_split_one<D, CT, NT, KIND_RELU>(mk, mv, a, grid, device, s);
    default: return launch_split_one<D, CT, NT, KIND_SOFTMAX>(mk, mv, a, grid, device, s);
  }
}

#define CHIA_INSTANTIATE_SPLIT(D, CT)                                                           \
  template <>                                                                                   \
  cudaError_t chia::launch_split<D, CT>(const CUtensorMap &mk, const CUtensorMap &mv,           \
                                        const PagedArgs &a, int kind, int tiles, int grid,      \
                                        int device, cudaStream_t s) {                           \
    return tiles == 1 ? launch_split_kind<D, CT, 1>(mk, mv, a, kind, grid, device, s)           \
                      : launch_split_kind<D, CT, 2>(mk, mv, a, kind, grid, device, s);          \
  }

}  // namespace chia
