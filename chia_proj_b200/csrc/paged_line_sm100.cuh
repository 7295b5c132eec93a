// paged_line_sm100.cuh -- the work of attention over the paged cache as a line
// of key tiles, and what its kernels share.
//
// All (request, K/V head, block of ROWS rows) units, each with the key tiles
// that its rows see, stand in one line; CTAs take equal pieces of it, whatever
// the lengths. A unit counts as COST tiles more than it has (its queries, its
// output). The lengths are on the device, so every CTA sums them up itself.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "fmha_sm100.cuh"
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
  int32_t left, right, block, prefix, dil;  // the mask, on positions
  float score_scale, softcap, sig_bias, out_scale;
  int32_t heads, heads_kv, group, batch, tokens, page, width;
  uint32_t group_magic;  // ceil(2^32 / group); 0: a group of one
  int32_t num_pages;
  int32_t q_each;     // queries of a request where cu_q is null
  int32_t token0;     // first token of request 0 where cu_q is null
  int32_t bf16;       // type of q and o
  int32_t *tickets;   // one a CTA, zero between launches
  float *part_o;      // [parts][rows][D]: two parts a CTA, then (split kernel) one a worker
  float *part_ml;     // [parts][rows][2]
  int32_t *status;
  uint64_t timeout_ns, drain_ns;
};

constexpr int kLineBatch = 512;  // requests of one launch (they are held in shared memory)

// Tiles of TK keys that queries at positions [p0, p1] visit: `pre` tiles from
// key 0 on, then those from `lo` on; `n` in all, at least one (a unit whose
// rows see nothing still writes zeros).
struct Tiles {
  int pre, lo, n;
  __device__ __forceinline__ int key_tile(int t) const { return t < pre ? t : lo + (t - pre); }
};
// Queries and keys of request b, checked: [t0, t0 + n) of q, keys [0, len).
struct Request {
  int t0, n, len;
  int b;           // its row of the block table
  int row0, row1;  // an entry of the line: these rows (queries x heads of a group) of the request
  Tiles tl;        // the tiles that they visit
};
__device__ __forceinline__ bool offsets_ok(int t0, int t1, int tokens) { return t0 >= 0 && t1 >= t0 && t1 <= tokens; }
// The requests before the first whose offsets are out of range or fall. Those behind it
// are not served: they could own rows that others own, and the line, whose length the
// host bounds by the number of rows, could pass 32 bits. (It takes no PagedArgs: a
// reference would have every call put a copy of them on the stack.)
static __device__ __noinline__ int requests_in_order(const int32_t *cu_q, int batch, int tokens) {
  int b = 0;
  while (b < batch && offsets_ok(cu_q[b], cu_q[b + 1], tokens)) ++b;
  return b;
}
// bad: what the status word is told; gap: the offsets are bad
__device__ __forceinline__ Request request_of(const PagedArgs &a, int b, bool &bad, bool &gap) {
  Request r;
  r.b = b;
  if (a.cu_q != nullptr) {
    r.t0 = a.cu_q[b];
    const int t1 = a.cu_q[b + 1];
    if (offsets_ok(r.t0, t1, a.tokens)) {
      r.n = t1 - r.t0;
    } else {
      bad = gap = true;
      r.t0 = r.n = 0;
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
  r.row0 = 0;
  r.row1 = r.n * a.group;
  return r;
}

// The rare divisions stand in functions of their own: a call that needs none
// of them fetches the less code, and its first pass over the code is most of
// the time of a small call.
static __device__ __noinline__ int block_start(int i, int block) {
  return (i >= 0 ? i / block : -(-(i + 1) / block + 1)) * block;
}
static __device__ __noinline__ bool divides(int d, int x) { return x % d == 0; }
// x / group for x * group < 2^32
__device__ __forceinline__ int div_group(const PagedArgs &a, int x) {
  return a.group_magic == 0 ? x : static_cast<int>(__umulhi(static_cast<uint32_t>(x), a.group_magic));
}

// The keys that the query at position i sees beside the prefix, of keys 0 to
// len - 1; a position may be negative (a request with more queries than keys).
// Position and width may each be near 2^31, so sums of them are not formed.
__device__ __forceinline__ void band32(const PagedArgs &a, int i, int len, int &lo, int &hi) {
  lo = 0;
  hi = len - 1;
  if (a.left >= 0 && a.left < i) lo = i - a.left;
  if (a.right >= 0 && a.right < hi - i) hi = i + a.right;
  if (a.block > 0) {
    const int b0 = block_start(i, a.block), more = a.block - 1;
    lo = max(lo, b0);
    if (b0 <= 0x7fffffff - more) hi = min(hi, b0 + more);
  }
}

template <int TK>
__device__ __forceinline__ Tiles tiles_of(const PagedArgs &a, int p0, int p1, int len) {
  Tiles r;
  int lo, hi, x;
  band32(a, p0, len, lo, x);
  band32(a, p1, len, x, hi);
  const int pf = min(a.prefix, len);
  r.pre = pf / TK + (pf % TK != 0);
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
// The answer is a lane's own: where lanes go on together the caller takes the
// warp's (warp_all), since lanes that gave up alone would leave the others waiting
// for them. Under a limit below a microsecond, what the clock and a suspended lane
// cannot tell apart, a wait that is not met at once runs out.
__device__ __forceinline__ bool paged_wait(uint32_t bar, uint32_t parity, volatile int *abort,
                                           const PagedArgs &a) {
  if (ptx::mbar_test_wait(bar, parity)) return true;
  const uint64_t t0 = ptx::globaltimer_ns();
  while (a.timeout_ns < 1000 || !ptx::mbar_try_wait(bar, parity, 20000u)) {
    if (*abort) return false;
    if (ptx::globaltimer_ns() - t0 > a.timeout_ns) {
      *abort = 1;
      report(a.status, 5);  // CHIA_ERR_DEVICE_TIMEOUT
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool warp_all(bool x) { return __all_sync(0xffffffffu, x); }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// A unit: rows [row0, row0 + rows) of a request's queries with one K/V head.
struct Unit {
  int t0, row0, rows, hk;  // first token of the request
  int cost;                // where it begins in the line, in cost
  int n;                   // its tiles
};

// Where a row's output goes, and what it is multiplied by; `lse`: its log-sum-exp is written here too.
template <int KIND>
__device__ __forceinline__ uint16_t *row_out(const PagedArgs &a, const Unit &u, int r, float M, float L,
                                             bool lse, float &f) {
  constexpr bool SOFTMAX = KIND <= KIND_ALIBI;
  f = 1.f;
  if (SOFTMAX) f = L > 0.f ? 1.f / L : L;  // (a NaN stays)
  if (KIND == KIND_RELU) f = a.out_scale * ptx::ex2(M);
  if (KIND == KIND_SIGMOID) f = ptx::ex2(M);
  const int qi = div_group(a, u.row0 + r), hh = u.hk * a.group + u.row0 + r - qi * a.group;
  const int64_t tok = u.t0 + qi;
  if (SOFTMAX && a.lse != nullptr && lse)
    a.lse[tok * a.heads + hh] =
        L > 0.f ? (M + __log2f(L)) * 0.6931471805599453f : L == 0.f ? -INFINITY : L;
  return static_cast<uint16_t *>(a.o) + tok * a.o_st + hh * a.o_sh;
}

template <bool BF16>
__device__ __forceinline__ void store4(const PagedArgs &a, uint16_t *dst, float f, float x0, float x1,
                                       float x2, float x3) {
  x0 *= f, x1 *= f, x2 *= f, x3 *= f;
  *reinterpret_cast<uint2 *>(dst) =
      BF16 ? make_uint2(ptx::pack_bf16(x0, x1), ptx::pack_bf16(x2, x3))
           : make_uint2(ptx::pack_f16(x0, x1), ptx::pack_f16(x2, x3));
}

// Channels 4 c4 .. + 3 of row r from the parts that CTAs first..last left of a
// unit (the first one's is its later part), eight in flight at once.
template <int ROWS, int D>
__device__ __forceinline__ void merge_parts(const PagedArgs &a, int first, int last, int r, int c4, float &M,
                                            float &L, float4 &acc) {
  for (int c0 = first; c0 <= last; c0 += 8) {
    float2 ml[8];
    float4 v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      ml[x] = make_float2(-INFINITY, 0.f);
      v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c0 + x <= last) {
        const int64_t part = (2ll * (c0 + x) + (c0 + x == first ? 1 : 0)) * ROWS + r;
        ml[x] = __ldcg(reinterpret_cast<const float2 *>(a.part_ml + part * 2));
        v[x] = __ldcg(reinterpret_cast<const float4 *>(a.part_o + part * D + 4 * c4));
      }
    }
    float top = M;
#pragma unroll
    for (int x = 0; x < 8; ++x) top = fmaxf(top, ml[x].x);
    const float base = top == -INFINITY ? 0.f : top, old = ptx::ex2(M - base);
    L *= old, acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
    M = top;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const float wt = ptx::ex2(ml[x].x - base);
      L = fmaf(wt, ml[x].y, L);
      acc.x = fmaf(wt, v[x].x, acc.x);
      acc.y = fmaf(wt, v[x].y, acc.y);
      acc.z = fmaf(wt, v[x].z, acc.z);
      acc.w = fmaf(wt, v[x].w, acc.w);
    }
  }
}

// The line of units of ROWS rows and tiles of TK keys, in shared memory: its
// entries in their order. An entry is a request, or with BLOCKS a block of ROWS
// rows of one (several, where there are more blocks than entries fit): blocks
// of a long run of queries see different keys. An entry's units visit the same
// tiles. WHOLE: units of up to this cost (with BLOCKS: and of no more than a CTA's
// share) are not cut between CTAs.
template <int TK, int ROWS, int THREADS, int COST, int WHOLE, bool BLOCKS>
struct Line {
  struct Shared {
    int tiles_pre[kLineBatch + 1], units_pre[kLineBatch + 1];  // before each entry
    Request req[kLineBatch];
    int wsum[THREADS / 32][2];
    int starts[BLOCKS ? kLineBatch + 1 : 1];  // first entry of each request
  };
  Shared &s;
  const PagedArgs &a;
  int entries, total, ctas, step, rest;

  // Sums over the block of x and y before this thread's; the totals in tx, ty. Whether any
  // thread's `flag` is set.
  __device__ __forceinline__ bool scan(int &x, int &y, int &tx, int &ty, bool flag = false) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int x0 = x, y0 = y;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
      if (lane >= d) x += u, y += v;
    }
    if (lane == 31) s.wsum[warp][0] = x, s.wsum[warp][1] = y;
    const bool any = __syncthreads_or(flag);
    x -= x0, y -= y0;
    tx = ty = 0;
#pragma unroll 4
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) x += s.wsum[w][0], y += s.wsum[w][1];
      tx += s.wsum[w][0], ty += s.wsum[w][1];
    }
    __syncthreads();
    return any;
  }

  // All threads of the CTA; per_cta: the least cost of a CTA's piece.
  __device__ __forceinline__ Line(Shared &sh, const PagedArgs &args, int per_cta) : s(sh), a(args) {
    const int t = threadIdx.x;
    bool bad = false, gap = false;
    entries = a.batch;
    if (BLOCKS) {
      // (a launch has fewer requests than entries) the blocks of each request,
      // `each` to an entry so that all fit
      static_assert(!BLOCKS || kLineBatch <= THREADS, "an entry a thread");
      int blocks = 0, none = 0, x, each = 1;
      if (t < a.batch) blocks = (request_of(a, t, bad, gap).row1 + ROWS - 1) / ROWS;
      int at = blocks;
      if (scan(at, none, entries, x, gap)) {
        if (t >= requests_in_order(a.cu_q, a.batch, a.tokens)) blocks = 0;
        at = blocks;
        scan(at, none, entries, x);
      }
      if (entries > kLineBatch) {
        each = (entries + kLineBatch - a.batch - 1) / max(1, kLineBatch - a.batch);
        at = (blocks + each - 1) / each;
        scan(at, none, entries, x);
      }
      if (t < a.batch) s.starts[t] = at;
      if (t == 0) s.starts[a.batch] = entries;
      __syncthreads();
      if (t < entries) {
        const int b = last_not_above(s.starts, a.batch, t);
        Request r = request_of(a, b, bad, gap);
        r.row0 = (t - s.starts[b]) * each * ROWS;
        r.row1 = min(r.row1, r.row0 + each * ROWS);
        r.tl = tiles_of<TK>(a, r.len - r.n + div_group(a, r.row0), r.len - r.n + div_group(a, r.row1 - 1), r.len);
        s.req[t] = r;
      }
    } else {
      for (int b = t; b < entries; b += THREADS) {
        Request r = request_of(a, b, bad, gap);
        if (r.n > 0) r.tl = tiles_of<TK>(a, r.len - r.n, r.len - 1, r.len);
        s.req[b] = r;
      }
    }
    if (bad && blockIdx.x == 0) report(a.status, kStatusBadIndex);
    if (BLOCKS) {
      __syncthreads();
    } else if (__syncthreads_or(gap)) {
      const int ordered = requests_in_order(a.cu_q, a.batch, a.tokens);
      for (int b = t; b < entries; b += THREADS)
        if (b >= ordered) s.req[b].row1 = 0;
      __syncthreads();
    }
    const int per = (entries + THREADS - 1) / THREADS;
    const int b0 = t * per, b1 = min(entries, b0 + per);
    auto units_of = [&](const Request &r) {
      return r.row1 > r.row0 ? (r.row1 - r.row0 + ROWS - 1) / ROWS * a.heads_kv : 0;
    };
    int it = 0, iu = 0, x, y;
    for (int b = b0; b < b1; ++b) {
      const int u = units_of(s.req[b]);
      iu += u;
      if (u > 0) it += s.req[b].tl.n * u;
    }
    scan(it, iu, x, y);
    for (int b = b0; b < b1; ++b) {
      const int u = units_of(s.req[b]);
      s.tiles_pre[b] = it, s.units_pre[b] = iu;
      iu += u;
      if (u > 0) it += s.req[b].tl.n * u;
    }
    if (t == 0) s.tiles_pre[entries] = x, s.units_pre[entries] = y;
    __syncthreads();
    total = cost_before(entries);
    ctas = min(static_cast<int>(gridDim.x), (total + per_cta - 1) / per_cta);
    step = ctas > 0 ? total / ctas : 0;
    rest = ctas > 0 ? total % ctas : 0;
  }
  __device__ __forceinline__ int cost_before(int b) const { return s.tiles_pre[b] + COST * s.units_pre[b]; }
  // Border c of the CTAs' pieces, in cost.
  __device__ __forceinline__ int even(int c) const { return step * c + rest * c / ctas; }
  // Cost x, as a cost and as a tile. `snap`: moved to the nearer end of the
  // unit that it cuts where the unit is short: a cut costs a round of the
  // workspace (some 4 us), whole units wait for nobody.
  // `entry`: the one that the tile is in.
  __device__ __forceinline__ int place(int x, bool snap, int &tile, int &entry) const {
    if (x >= total) {
      tile = s.tiles_pre[entries];
      entry = entries;
      return total;
    }
    int lo = 0, hi = entries;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cost_before(mid) <= x)
        lo = mid;
      else
        hi = mid;
    }
    const int units = s.units_pre[lo + 1] - s.units_pre[lo];
    const int n = s.req[lo].tl.n, cost = n + COST;
    int in = x - cost_before(lo), u = in / cost;
    in -= u * cost;
    if (snap && cost <= WHOLE && (!BLOCKS || cost <= step)) {
      u += 2 * in >= cost ? 1 : 0;
      in = 0;
    }
    // (a border within the cost of a unit's own counts as its first tile)
    tile = s.tiles_pre[lo] + u * n + max(0, in - COST);
    entry = u < units ? lo : entries;
    if (u == units && tile < s.tiles_pre[entries]) entry = entry_at(tile);
    return cost_before(lo) + u * cost + in;
  }
  // The CTA that has tile k of a unit that is cut: the last with a border not above it.
  __device__ __forceinline__ int cta_of(const Unit &u, int k) const {
    const int x = u.cost + COST + k;
    int c = static_cast<int>(static_cast<float>(x) / static_cast<float>(total) * ctas);
    c = max(0, min(ctas - 1, c));
    while (c + 1 < ctas && even(c + 1) <= x) ++c;
    while (even(c) > x) --c;
    return c;
  }
  // The entry of tile g of the line, and the unit: its tiles from ut0 on follow.
  __device__ __forceinline__ int entry_at(int g) const { return last_not_above(s.tiles_pre, entries, g); }
  __device__ __forceinline__ Unit unit_at(int g, int b, const Request &r, int &ut0) const {
    const int blocks = (r.row1 - r.row0 + ROWS - 1) / ROWS;
    const int in = g - s.tiles_pre[b], u = in / r.tl.n;
    ut0 = in - u * r.tl.n;
    Unit un;
    un.t0 = r.t0;
    un.hk = blocks == 1 ? u : u / blocks;
    un.row0 = r.row0 + (u - un.hk * blocks) * ROWS;
    un.rows = min(ROWS, r.row1 - un.row0);
    un.cost = cost_before(b) + u * (r.tl.n + COST);
    un.n = r.tl.n;
    return un;
  }
};

// Once for each kernel and device.
inline cudaError_t allow_smem(const void *kernel, int bytes, int device, std::atomic<uint64_t> &set) {
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (set.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) set.fetch_or(bit, std::memory_order_release);
  return e;
}

}  // namespace chia
