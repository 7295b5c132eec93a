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
  int32_t left, right, block, prefix, dil;  // the mask, on positions (at most 2^30 each)
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
  Tiles tl;
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

// The rare divisions stand in functions of their own: a call that needs none
// of them fetches the less code, and its first pass over the code is most of
// the time of a small call.
static __device__ __noinline__ int block_start(int i, int block) {
  return (i >= 0 ? i / block : -((-i + block - 1) / block)) * block;
}
static __device__ __noinline__ bool divides(int d, int x) { return x % d == 0; }
// x / group for x * group < 2^32
__device__ __forceinline__ int div_group(const PagedArgs &a, int x) {
  return a.group_magic == 0 ? x : static_cast<int>(__umulhi(static_cast<uint32_t>(x), a.group_magic));
}

// The keys that the query at position i sees beside the prefix, of keys 0 to
// len - 1; a position may be negative (a request with more queries than keys).
__device__ __forceinline__ void band32(const PagedArgs &a, int i, int len, int &lo, int &hi) {
  lo = 0;
  hi = len - 1;
  if (a.left >= 0) lo = max(lo, i - a.left);
  if (a.right >= 0) hi = min(hi, i + a.right);
  if (a.block > 0) {
    const int b0 = block_start(i, a.block);
    lo = max(lo, b0);
    hi = min(hi, b0 + a.block - 1);
  }
}

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
__device__ __forceinline__ bool paged_wait(uint32_t bar, uint32_t parity, volatile int *abort,
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
__device__ __forceinline__ void store4(const PagedArgs &a, uint16_t *dst, float f, float x0, float x1,
                                       float x2, float x3) {
  x0 *= f, x1 *= f, x2 *= f, x3 *= f;
  *reinterpret_cast<uint2 *>(dst) =
      a.bf16 ? make_uint2(ptx::pack_bf16(x0, x1), ptx::pack_bf16(x2, x3))
             : make_uint2(ptx::pack_f16(x0, x1), ptx::pack_f16(x2, x3));
}

// The line of units of ROWS rows and tiles of TK keys, in shared memory.
// WHOLE: units of up to this cost are not cut between CTAs.
template <int TK, int ROWS, int THREADS, int COST, int WHOLE>
struct Line {
  struct Shared {
    int tiles_pre[kLineBatch + 1], units_pre[kLineBatch + 1];  // before each request
    Request req[kLineBatch];
    int wsum[THREADS / 32][2];
  };
  Shared &s;
  const PagedArgs &a;
  int total, ctas, step, rest;

  // All threads of the CTA; per_cta: the least cost of a CTA's piece.
  __device__ __forceinline__ Line(Shared &sh, const PagedArgs &args, int per_cta) : s(sh), a(args) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int per = (a.batch + THREADS - 1) / THREADS;
    const int b0 = t * per, b1 = min(a.batch, b0 + per);
    int nt = 0, nu = 0;
    bool bad = false;
    for (int b = b0; b < b1; ++b) {
      Request r = request_of(a, b, bad);
      int n = 0, u = 0;
      if (r.n > 0) {
        r.tl = tiles_of<TK>(a, r.len - r.n, r.len - 1, r.len);
        u = (r.n * a.group + ROWS - 1) / ROWS * a.heads_kv;
        n = r.tl.n * u;
      }
      s.req[b] = r;
      s.tiles_pre[b + 1] = n;
      s.units_pre[b + 1] = u;
      nt += n;
      nu += u;
    }
    if (bad && blockIdx.x == 0) report(a.status, kStatusBadIndex);
    int it = nt, iu = nu;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, it, d), y = __shfl_up_sync(0xffffffffu, iu, d);
      if (lane >= d) it += x, iu += y;
    }
    if (lane == 31) s.wsum[warp][0] = it, s.wsum[warp][1] = iu;
    __syncthreads();
    it -= nt, iu -= nu;
    for (int w = 0; w < warp; ++w) it += s.wsum[w][0], iu += s.wsum[w][1];
    for (int b = b0; b < b1; ++b) {
      it += s.tiles_pre[b + 1], iu += s.units_pre[b + 1];
      s.tiles_pre[b + 1] = it, s.units_pre[b + 1] = iu;
    }
    if (t == 0) s.tiles_pre[0] = s.units_pre[0] = 0;
    __syncthreads();
    total = cost_before(a.batch);
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
  __device__ __forceinline__ int place(int x, bool snap, int &tile) const {
    if (x >= total) {
      tile = s.tiles_pre[a.batch];
      return total;
    }
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cost_before(mid) <= x)
        lo = mid;
      else
        hi = mid;
    }
    const int units = s.units_pre[lo + 1] - s.units_pre[lo];
    const int n = (s.tiles_pre[lo + 1] - s.tiles_pre[lo]) / units, cost = n + COST;
    int in = x - cost_before(lo), u = in / cost;
    in -= u * cost;
    if (snap && cost <= WHOLE) {
      u += 2 * in >= cost ? 1 : 0;
      in = 0;
    }
    // (a border within the cost of a unit's own counts as its first tile)
    tile = s.tiles_pre[lo] + u * n + max(0, in - COST);
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
  // The request of tile g of the line, and the unit: its tiles from ut0 on follow.
  __device__ __forceinline__ int request_at(int g) const {
    return last_not_above(s.tiles_pre, a.batch, g);
  }
  __device__ __forceinline__ Unit unit_at(int g, int b, const Request &r, int &ut0) const {
    const int rows = r.n * a.group, blocks = (rows + ROWS - 1) / ROWS;
    const int in = g - s.tiles_pre[b], u = in / r.tl.n;
    ut0 = in - u * r.tl.n;
    Unit un;
    un.t0 = r.t0;
    un.hk = blocks == 1 ? u : u / blocks;
    un.row0 = (u - un.hk * blocks) * ROWS;
    un.rows = min(ROWS, rows - un.row0);
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
