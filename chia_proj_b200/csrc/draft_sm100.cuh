// draft_sm100.cuh -- trees of drafted tokens over the paged 8-bit K/V cache: their
// tables, their verification, and the compaction of what was accepted.
#pragma once
#include "paged_common.cuh"

namespace chia {

// A request's rows [t0, t0 + n), n < 0 where its offsets are out of range or fall.
struct TreeRows {
  int t0, n;
};
__device__ __forceinline__ TreeRows tree_rows(const int32_t *cu_q, int b, int tokens) {
  const int t0 = cu_q[b], t1 = cu_q[b + 1];
  if (t0 < 0 || t1 < t0 || t1 > tokens) return {0, -1};
  return {t0, t1 - t0};
}

// ---------------------------------------------------------------------- tables
struct TreeArgs {
  const int32_t *parents, *cu_q, *seq_lens;
  int32_t *positions;
  unsigned long long *ancestors;
  int32_t *status;
  int32_t batch, tokens;
};

constexpr int kTreeThreads = 256;

// A warp a request, two nodes a lane. Words are completed by doubling: a node's word
// takes up that of the node 2^i above it, and then looks twice as far up; six rounds
// reach the root of any tree. The depth is the number of ancestors. Requests from an
// offset on that falls are not served, as everywhere; rows that nobody owns get zeros.
// A few KB: the time is latency (one tree of 13 nodes 2.4 us, 64 of up to 64 nodes 2.7, on the device).
static __global__ void __launch_bounds__(kTreeThreads) tree_tables_kernel(const TreeArgs a) {
  __shared__ int s_ordered;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) s_ordered = a.batch;
  follow();
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += kTreeThreads)
    if (tree_rows(a.cu_q, b, a.tokens).n < 0) atomicMin(&s_ordered, b);
  __syncthreads();
  const int ordered = s_ordered;
  bool bad = ordered < a.batch;
  for (int b = blockIdx.x * (kTreeThreads / 32) + warp; b < ordered; b += gridDim.x * (kTreeThreads / 32)) {
    const TreeRows r = tree_rows(a.cu_q, b, a.tokens);
    const int base = a.seq_lens[b] - r.n;
    if (r.n > kTreeNodes) {
      for (int i = lane; i < r.n; i += 32) a.positions[r.t0 + i] = base + i, a.ancestors[r.t0 + i] = 0;
      continue;
    }
    unsigned long long word[2];
    int up[2];  // the node that is looked at next, itself where there is none
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int i = lane + 32 * x;
      word[x] = 1ull << i, up[x] = i;
      if (i < r.n) {
        const int p = a.parents[r.t0 + i];
        if (p >= 0 && p < i)
          up[x] = p;
        else if (p != -1)
          bad = true;
      }
    }
#pragma unroll
    for (int round = 0; round < 6; ++round) {
      unsigned long long w[2];
      int u[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const unsigned long long w0 = __shfl_sync(0xffffffffu, word[0], up[x] & 31),
                                 w1 = __shfl_sync(0xffffffffu, word[1], up[x] & 31);
        const int u0 = __shfl_sync(0xffffffffu, up[0], up[x] & 31), u1 = __shfl_sync(0xffffffffu, up[1], up[x] & 31);
        w[x] = up[x] < 32 ? w0 : w1, u[x] = up[x] < 32 ? u0 : u1;
      }
      word[0] |= w[0], word[1] |= w[1], up[0] = u[0], up[1] = u[1];
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int i = lane + 32 * x;
      if (i < r.n) {
        a.positions[r.t0 + i] = base + __popcll(word[x]) - 1;
        a.ancestors[r.t0 + i] = word[x];
      }
    }
  }
  // rows before the first and behind the last request that is served
  const int first = ordered > 0 ? a.cu_q[0] : a.tokens, last = ordered > 0 ? a.cu_q[ordered] : 0;
  for (int t = blockIdx.x * kTreeThreads + threadIdx.x; t < a.tokens; t += gridDim.x * kTreeThreads)
    if (t < first || t >= last) a.positions[t] = 0, a.ancestors[t] = 0;
  if (bad) report(a.status, kStatusBadIndex);
}

// ---------------------------------------------------------------- verification
struct VerifyArgs {
  const void *p, *q;
  int64_t p_st, q_st;
  const int32_t *tokens, *parents, *cu_q;
  const float *u;
  int32_t *counts, *out, *path, *status;
  int32_t batch, rows, vocab, most, chunks;  // chunks: of kVerifyChunk entries, in all
};

constexpr int kVerifyMostThreads = 1024;
constexpr int kVerifyCtas = 8;  // of a request: a cluster
constexpr int kVerifyChunk = 512;  // entries that a warp sums at a time
constexpr int kVerifyMostChunks = 1024;  // of a CTA

// An entry; one that is no positive finite number is 0 (its bits are none of those up to infinity's).
__device__ __forceinline__ float verify_clean(float x) {
  return __float_as_uint(x) < 0x7f800000u ? x : 0.f;
}
template <int T>
__device__ __forceinline__ float verify_one(const void *p, int64_t e) {
  if (T == 2) return verify_clean(static_cast<const float *>(p)[e]);
  const uint32_t v = static_cast<const uint16_t *>(p)[e];
  return verify_clean(T == 0 ? in16x2_to_float2<true>(v).x : in16x2_to_float2<false>(v).x);
}

// Four entries from v on, of a row whose first one is e (VEC: rows are aligned for it); behind the
// row's end there are zeros.
template <int T, bool VEC>
__device__ __forceinline__ void verify_four(const void *p, int64_t e, int v, int vocab, float (&x)[4]) {
  if (VEC && v + 4 <= vocab) {
    if (T == 2) {
      const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + e + v);
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + e + v);
      const float2 a = in16x2_to_float2<T == 0>(w.x), b = in16x2_to_float2<T == 0>(w.y);
      x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = 0.f;
      if (v + i < vocab) {
        if (T == 2)
          x[i] = static_cast<const float *>(p)[e + v + i];
        else
          x[i] = in16x2_to_float2<T == 0>(static_cast<const uint16_t *>(p)[e + v + i]).x;
      }
    }
  }
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
// to the same place in the shared memory of CTA `rank` of the cluster
__device__ __forceinline__ void cluster_store(double *at, int rank, double v) {
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(ptx::smem_u32(at)), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(v) : "memory");
}
__device__ __forceinline__ double shfl_up(double x, int d) { return __shfl_up_sync(0xffffffffu, x, d); }

// A request's walk down its tree, by a cluster. What decides at a child is four numbers
// (u, p, q at its token, and the residual's mass), so the probabilities of all nodes'
// tokens are gathered at the start and the walk itself takes no memory. The rows are
// read only for a mass: the residual behind rejected children is
//   r = max(p - F q, 0),  F = sum of their Z / (1 - s)
// (max(max(x - a, 0) - b, 0) = max(x - a - b, 0) for a, b >= 0), a function of the two
// rows alone, so a pass keeps nothing but its sums: one for each chunk of 512 entries,
// in the order of the vocabulary, so the drawn token is found from the last pass's sums
// and one chunk that is read again. Without draft rows the mass is 1 minus what was
// rejected, and the only pass is the last. All CTAs walk alike.
//
// Measured, fp32: 64 trees of up to 25 nodes over 131,072 entries, drafts drawn at random, 28.5 us,
// where the rows that tokens are drawn from take 10 at the rate of a copy: some 4 us to the first pass
// (offsets, nodes, their probabilities), 3 to 4 a pass, up to five passes one behind another in a
// request; one chain of five drafts over 32,000 entries 5.0. An entry of a row costs a conversion, one of the
// target's two 64-bit operations beside; with single entries a load and a maximum in 64 bits the trees took
// 102 us. Rows whose width or address is no multiple of four entries are read entry by entry: 27.5 us over
// 131,072 entries are 35.9 over 131,073, and 15.5 over 50,256 are 17.7 over 50,257.
template <int T, bool DRAFTS, bool VEC>
__global__ void __launch_bounds__(kVerifyMostThreads, 1) verify_kernel(const VerifyArgs a) {
  __shared__ double s_sum[kVerifyMostChunks];  // of this CTA's chunks
  __shared__ double s_total[2][kVerifyCtas];   // of each CTA, two passes by turns
  __shared__ float s_p[kTreeNodes], s_q[kTreeNodes], s_u[kTreeNodes];
  __shared__ int s_parent[kTreeNodes], s_token[kTreeNodes];
  __shared__ double s_warp[kVerifyMostThreads / 32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x / 32;
  const int rank = cluster_rank(), b = blockIdx.x / kVerifyCtas;
  cluster_arrive();
  follow();
  cluster_wait();  // all CTAs of the cluster run: their shared memory may be written
  const TreeRows r = tree_rows(a.cu_q, b, a.rows);
  bool bad = r.n < 0 || r.n > kTreeNodes;
  int32_t *out = a.out + static_cast<int64_t>(b) * a.most, *path = a.path + static_cast<int64_t>(b) * a.most;
  if (r.n == 0 || bad) {
    if (rank == 0) {
      for (int i = t; i < a.most; i += blockDim.x) out[i] = path[i] = -1;
      if (t == 0) a.counts[b] = 0;
      if (t == 0 && bad) report(a.status, kStatusBadIndex);
    }
    return;  // (all CTAs of the cluster do)
  }
  const int per = (a.chunks + kVerifyCtas - 1) / kVerifyCtas;  // chunks of a CTA
  if (t < r.n) {
    const int x = a.tokens[r.t0 + t];
    int p = a.parents[r.t0 + t];
    s_u[t] = a.u[r.t0 + t];
    if (t == 0) {
      bad = p != -1;
      p = -1;
    } else if (p < -1 || p >= t || x < 0 || x >= a.vocab) {
      bad = true;
      p = -1;
    }
    s_parent[t] = p, s_token[t] = x;
    if (p >= 0) {
      s_p[t] = verify_one<T>(a.p, (r.t0 + p) * a.p_st + x);
      if (DRAFTS) s_q[t] = verify_one<T>(a.q, (r.t0 + p) * a.q_st + x);
    }
    if (bad && rank == 0) report(a.status, kStatusBadIndex);
  }
  __syncthreads();

  // Sums of the residual at `node`; returns the mass, the same in all CTAs.
  int turn = 0;
  const int c0 = rank * per, mine = max(0, min(per, a.chunks - c0));
  unsigned long long dropped = 0;  // (without draft rows) rejected children of the node
  // four entries of the residual, from the rows'
  auto residual = [&](double F, const float (&p)[4], const float (&q)[4], double (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = verify_clean(p[i]);
      if (DRAFTS) {
        x[i] = fma(-F, static_cast<double>(verify_clean(q[i])), x[i]);
        if (__double2hiint(x[i]) < 0) x[i] = 0.0;
      }
    }
  };
  // without draft rows: rejected tokens among the chunk's (few chunks have any)
  auto drop = [&](int c, int v, double (&x)[4]) {
    for (unsigned long long m = dropped; m != 0; m &= m - 1) {
      const int at = s_token[__ffsll(m) - 1];
      if (at / kVerifyChunk != c) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i == at) x[i] = 0.0;
    }
  };
  auto has_dropped = [&](int c) {
    bool any = false;
    if (!DRAFTS)
      for (unsigned long long m = dropped; m != 0; m &= m - 1) any |= s_token[__ffsll(m) - 1] / kVerifyChunk == c;
    return any;
  };
  auto chunk_sum = [&](int64_t pe, int64_t qe, double F, int c) {  // this lane's part of it
    constexpr int N = kVerifyChunk / 128;
    float p[N][4], q[N][4];
    const int v0 = (c0 + c) * kVerifyChunk + 4 * lane;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) verify_four<T, VEC>(a.p, pe, v0 + 128 * i, a.vocab, p[i]);  // (all loads at once)
    if (DRAFTS && F != 0.0) {
#pragma unroll
      for (int i = 0; i < N; ++i) verify_four<T, VEC>(a.q, qe, v0 + 128 * i, a.vocab, q[i]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        double x[4];
        residual(F, p[i], q[i], x);
        sum += (x[0] + x[1]) + (x[2] + x[3]);
      }
    } else {  // nothing was rejected, or there is no draft row
      const bool dropping = has_dropped(c0 + c);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        double x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = verify_clean(p[i][e]);
        if (dropping) drop(c0 + c, v0 + 128 * i, x);
        sum += (x[0] + x[1]) + (x[2] + x[3]);
      }
    }
    return sum;
  };
  auto warp_sum = [&](double x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
  };
  // `last`: the sums of chunks are kept (a mass that a sibling waits for is never the last)
  auto mass = [&](int node, double F, bool last) {
    const int64_t pe = (r.t0 + node) * a.p_st, qe = (r.t0 + node) * a.q_st;
    double sum = 0.0;
#pragma unroll 1
    for (int c = warp; c < mine; c += warps) {
      const double x = chunk_sum(pe, qe, F, c);
      if (last) {
        const double all = warp_sum(x);
        if (lane == 0) s_sum[c] = all;
        sum += all;
      } else {
        sum += x;
      }
    }
    if (!last) sum = warp_sum(sum);
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      sum = warp_sum(lane < warps ? s_warp[lane] : 0.0);
      if (lane < kVerifyCtas) cluster_store(&s_total[turn][rank], lane, sum);
    }
    cluster_sync();
    double z = 0.0;
#pragma unroll
    for (int x = 0; x < kVerifyCtas; ++x) z += s_total[turn][x];
    turn ^= 1;
    return z;
  };

  int node = 0, count = 1;
  double Z = 1.0, F = 0.0, sib = 0.0;
  bool known = true;  // Z is that of the residual
  if (rank == 0 && t == 0) path[0] = 0;
  for (int i = 1; i < r.n && count < a.most; ++i) {
    if (s_parent[i] != node) continue;
    const double u = s_u[i], p = s_p[i];
    bool yes;
    if (DRAFTS) {
      const double q = s_q[i];
      if (!known) Z = mass(node, F, false), known = true;
      double here = fmax(fma(-F, q, p), 0.0), qx = q;
      // (a token that an earlier sibling had is in neither)
      for (int j = node + 1; j < i; ++j)
        if (s_parent[j] == node && s_token[j] == s_token[i]) qx = 0.0;
      const double d = 1.0 - sib;
      yes = u * Z * qx < here * d;
      if (!yes) {
        if (d > 0.0) F += Z / d, known = false;
        sib += qx;
      }
    } else {
      double here = p;
      for (unsigned long long m = dropped; m != 0; m &= m - 1)
        if (s_token[__ffsll(m) - 1] == s_token[i]) here = 0.0;
      yes = u * Z < here;
      if (!yes) Z -= here, dropped |= 1ull << i;
    }
    if (yes) {
      if (rank == 0 && t == 0) path[count] = i, out[count - 1] = s_token[i];
      node = i, ++count, Z = 1.0, F = 0.0, sib = 0.0, known = true, dropped = 0;
    }
  }

  // the token behind the last accepted node
  Z = mass(node, F, true);
  if (!(Z > 0.0)) F = 0.0, dropped = 0, Z = mass(node, F, true);
  const double *total = s_total[turn ^ 1];
  const double target = static_cast<double>(s_u[0]) * Z;
  // the CTA whose chunks hold the place, or the last that holds anything
  int owner = -1;
  double before = 0.0, sum = 0.0;
#pragma unroll
  for (int x = 0; x < kVerifyCtas; ++x) {
    if (total[x] > 0.0 && (owner < 0 || !(sum > target))) owner = x, before = sum;
    sum += total[x];
  }
  if (rank == 0) {
    for (int i = count + t; i < a.most; i += blockDim.x) out[i] = path[i] = -1;
    if (t == 0) {
      a.counts[b] = count;
      if (owner < 0) out[count - 1] = -1;
    }
  }
  if (owner == rank && warp == 0) {
    // the chunk likewise, 32 at a time
    int chunk = -1;
    double base = before, in = before;  // the sum before the chunk
    for (int x0 = 0; x0 < mine; x0 += 32) {
      const double own = x0 + lane < mine ? s_sum[x0 + lane] : 0.0;
      double inc = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double y = shfl_up(inc, d);
        if (lane >= d) inc += y;
      }
      const unsigned over = __ballot_sync(0xffffffffu, own > 0.0 && base + inc > target);
      const unsigned some = __ballot_sync(0xffffffffu, own > 0.0);
      const int pick = over != 0 ? __ffs(over) - 1 : some != 0 ? 31 - __clz(some) : -1;
      if (pick >= 0) {
        chunk = x0 + pick;
        in = base + __shfl_sync(0xffffffffu, inc - own, pick);
      }
      if (over != 0) break;
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
    // the lane likewise, 16 entries each, and the entry
    if (chunk >= 0) {
      constexpr int N = kVerifyChunk / 128;
      const int64_t pe = (r.t0 + node) * a.p_st, qe = (r.t0 + node) * a.q_st;
      const int v0 = (c0 + chunk) * kVerifyChunk + 4 * N * lane;
      double x[N][4], own = 0.0;
      {
        float p[N][4], q[N][4];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          verify_four<T, VEC>(a.p, pe, v0 + 4 * i, a.vocab, p[i]);
          if (DRAFTS) verify_four<T, VEC>(a.q, qe, v0 + 4 * i, a.vocab, q[i]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          residual(F, p[i], q[i], x[i]);
          if (!DRAFTS) drop(c0 + chunk, v0 + 4 * i, x[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) own += x[i][e];
        }
      }
      double inc = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double y = shfl_up(inc, d);
        if (lane >= d) inc += y;
      }
      const unsigned over = __ballot_sync(0xffffffffu, own > 0.0 && in + inc > target);
      const unsigned some = __ballot_sync(0xffffffffu, own > 0.0);
      if (lane == (over != 0 ? __ffs(over) - 1 : 31 - __clz(some))) {
        int found = -1;
        double sum = in + (inc - own);
        bool done = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sum += x[i][e];
            if (!done && x[i][e] > 0.0) found = v0 + 4 * i + e, done = sum > target;
          }
        out[count - 1] = found;
      }
    }
  }
}

// ------------------------------------------------------------------ compaction
struct CompactArgs {
  const int32_t *path, *counts, *cu_q, *seq_lens, *block_table;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int32_t *keep_lens, *status;
  const int32_t *slots;  // [tokens] or null
  int64_t table_stride, num_pages, tokens;
  int32_t batch, most, heads_kv, page, width;
};

constexpr int kCompactThreads = 128;

// A CTA a request, K/V head, K or V. The path's nodes rise, so a token moves to a place
// before its own; all of them are read (and their pages' scales) before anything is
// written. Then page by page: the scale, where it grows what the page holds, and the
// tokens. A few KB a CTA: the time is latency (one path of a tree of 13 nodes 3.0 us, 128 of trees of
// up to 64 nodes 4.4, on the device).
template <int D, int CT>
__global__ void __launch_bounds__(kCompactThreads) cache_compact_kernel(const CompactArgs a) {
  constexpr int PIECES = D / 16;  // 16-byte pieces of a token
  __shared__ uint4 s_code[kTreeNodes * PIECES];
  __shared__ float s_scale[kTreeNodes];                 // of the page that token k comes from
  __shared__ float s_old[kTreeNodes];                   // of the one that it goes to
  __shared__ int s_from[kTreeNodes], s_to[kTreeNodes];  // slots; -1: it stays
  const int t = threadIdx.x, kinds = 2 * a.heads_kv;
  const int b = blockIdx.x / kinds, which = blockIdx.x % kinds, h = which >> 1;
  uint8_t *cache = which & 1 ? a.v_cache : a.k_cache;
  float *scale = which & 1 ? a.v_scale : a.k_scale;
  const int shift = 31 - __clz(a.page);
  follow();
  const int len = a.seq_lens[b], count = a.counts[b], t0 = a.cu_q[b], n = a.cu_q[b + 1] - t0;
  const int base = len - n;
  if (n > kTreeNodes && t0 >= 0) {  // a chunk: nothing of it was drafted
    if (which == 0 && t == 0) a.keep_lens[b] = len;
    return;
  }
  if (a.slots != nullptr) {  // a request without a place for its tokens: len has no tree in it
    const bool missing = t0 >= 0 && t < n && (static_cast<int64_t>(t0) + t >= a.tokens || a.slots[t0 + t] < 0);
    if (__syncthreads_or(missing)) {
      if (which == 0 && t == 0) a.keep_lens[b] = len;
      return;
    }
  }
  bool bad = t0 < 0 || n < 0 || len < n || count < 0 || count > n || count > a.most ||
             len > static_cast<int64_t>(a.width) * a.page;
  bool moves = false;
  if (!bad && t < count) {
    const int x = a.path[static_cast<int64_t>(b) * a.most + t];
    const int last = t > 0 ? a.path[static_cast<int64_t>(b) * a.most + t - 1] : -1;
    int from = -1, to = -1;
    if (x <= last || x >= n) {
      bad = true;
    } else if (x != t) {
      const int32_t *table = a.block_table + b * a.table_stride;
      const int fp = table[(base + x) >> shift], tp = table[(base + t) >> shift];
      if (fp < 0 || fp >= a.num_pages || tp < 0 || tp >= a.num_pages) {
        bad = true;
      } else {
        from = (fp << shift) + ((base + x) & (a.page - 1)), to = (tp << shift) + ((base + t) & (a.page - 1));
        moves = true;
      }
    }
    s_from[t] = from, s_to[t] = to;
  }
  bad = __syncthreads_or(bad);
  if (which == 0 && t == 0) {
    a.keep_lens[b] = bad ? len : base + count;
    if (bad) report(a.status, kStatusBadIndex);
  }
  const int moved = __syncthreads_count(moves && !bad);  // the last `moved` ones
  if (moved == 0) return;
  const int k0 = count - moved;
  auto token = [&](int slot) {  // a token's bytes
    return cache + ((static_cast<int64_t>(slot >> shift) * a.heads_kv + h) * a.page + (slot & (a.page - 1))) * D;
  };
  for (int e = t; e < moved * PIECES; e += kCompactThreads)
    s_code[e] = reinterpret_cast<const uint4 *>(token(s_from[k0 + e / PIECES]))[e % PIECES];
  if (t >= k0 && t < count) {
    s_scale[t] = scale[static_cast<int64_t>(s_from[t] >> shift) * a.heads_kv + h];
    s_old[t] = scale[static_cast<int64_t>(s_to[t] >> shift) * a.heads_kv + h];
  }
  __syncthreads();
  auto again = [&](uint4 v, float ratio) {
    auto one = [&](uint32_t w) {
      uint32_t p01, p23;
      cache4_to_f16<CT>(w, p01, p23);
      const float2 f = f16x2_to_float2(p01), g = f16x2_to_float2(p23);
      return to_cache4<CT>(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
    };
    return make_uint4(one(v.x), one(v.y), one(v.z), one(v.w));
  };
  for (int k = k0; k < count;) {
    const int page = s_to[k] >> shift;
    int end = k;
    float top = 0.f;
    for (; end < count && s_to[end] >> shift == page; ++end) top = fmaxf(top, s_scale[end]);
    const int64_t ph = static_cast<int64_t>(page) * a.heads_kv + h;
    // (read once, by one thread: a barrier stands in a branch on it)
    const float old = s_old[k], now = fmaxf(old, top);
    if (now > old) {
      if (t == 0) scale[ph] = now;
      uint4 *p = reinterpret_cast<uint4 *>(cache + ph * a.page * D);
      for (int e = t; e < a.page * PIECES; e += kCompactThreads) p[e] = again(p[e], old / now);
      __syncthreads();  // the tokens below go on top
    }
    for (int e = t; e < (end - k) * PIECES; e += kCompactThreads) {
      const int x = k + e / PIECES;
      const uint4 v = s_code[(x - k0) * PIECES + e % PIECES];
      const float own = s_scale[x];
      reinterpret_cast<uint4 *>(token(s_to[x]))[e % PIECES] = own == now ? v : again(v, own / now);
    }
    k = end;
  }
}

}  // namespace chia
