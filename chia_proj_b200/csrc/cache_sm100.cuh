// cache_sm100.cuh -- the tables of a serving step and the write of new tokens
// into the paged 8-bit K/V cache.
#pragma once
#include "paged_common.cuh"

namespace chia {

// ---------------------------------------------------------------------- tables
struct TablesArgs {
  const int32_t *seq_lens, *new_lens, *free_state;
  int32_t *block_table, *free_pages;
  int32_t *slots, *positions, *cu_q, *new_seq_lens, *new_free_state, *status;
  int64_t table_stride;
  int32_t batch, width, ring, max_tokens, page;
};

constexpr int kTablesThreads = 1024;

struct Scan2 {
  long long a, b;
};

// Inclusive sums over the block of two values a thread; `tot` gets the block's.
__device__ __forceinline__ Scan2 block_scan2(Scan2 v, Scan2 &tot, Scan2 *warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long ua = __shfl_up_sync(0xffffffffu, v.a, d);
    const long long ub = __shfl_up_sync(0xffffffffu, v.b, d);
    if (lane >= d) {
      v.a += ua;
      v.b += ub;
    }
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    Scan2 w = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long ua = __shfl_up_sync(0xffffffffu, w.a, d);
      const long long ub = __shfl_up_sync(0xffffffffu, w.b, d);
      if (lane >= d) {
        w.a += ua;
        w.b += ub;
      }
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  if (warp > 0) {
    v.a += warp_sums[warp - 1].a;
    v.b += warp_sums[warp - 1].b;
  }
  tot = warp_sums[31];
  __syncthreads();
  return v;
}

// One step's tables. Every CTA sums over all requests, kTablesThreads at a
// time (a few KB from L2), and then fills its share of each chunk's tokens:
// one launch, and no CTA waits for another. The token at a page's first slot
// enters the page in the block table.
__global__ void __launch_bounds__(kTablesThreads) page_tables_kernel(const TablesArgs a) {
  __shared__ Scan2 sums[32];
  __shared__ int32_t s_cu[kTablesThreads + 1], s_len[kTablesThreads], s_first[kTablesThreads];
  const int t = threadIdx.x;
  const bool first_cta = blockIdx.x == 0;
  int head = a.free_state[0], count = a.free_state[1];
  if (head < 0 || head >= a.ring || count < 0 || count > a.ring) {
    if (t == 0 && first_cta) report(a.status, kStatusBadIndex);
    head = 0;
    count = 0;
  }
  long long pages0 = 0, tokens0 = 0;
  long long taken = 0;  // pages handed out (thread 0's sum over the chunks)
  int bad = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kTablesThreads) {
    const int b = b0 + t;
    int len = 0, add = 0;
    if (b < a.batch) {
      len = a.seq_lens[b];
      add = a.new_lens[b];
      if (len < 0 || add < 0 || len > 0x7fffffff - add) {
        bad |= kStatusBadIndex;
        len = max(0, min(len, 0x3fffffff));
        add = 0;
      }
    }
    const int held = (len + a.page - 1) / a.page;
    int need = static_cast<int>((static_cast<long long>(len) + add + a.page - 1) / a.page) - held;
    const bool fits = static_cast<long long>(held) + need <= a.width;
    if (!fits) need = 0;
    Scan2 tot;
    const Scan2 sc = block_scan2(Scan2{need, add}, tot, sums);
    const long long upto = pages0 + sc.a;  // pages wanted by the requests up to this one
    const bool served = fits && (need == 0 || upto <= count);
    if (b < a.batch && !served) bad |= kStatusNoPages;
    const long long cu = tokens0 + sc.b - add;
    s_cu[t] = static_cast<int32_t>(cu < a.max_tokens ? cu : a.max_tokens);
    s_len[t] = len;
    s_first[t] = served ? static_cast<int32_t>(upto - need) : -1;
    if (t == kTablesThreads - 1) {
      const long long end = tokens0 + tot.b;
      s_cu[kTablesThreads] = static_cast<int32_t>(end < a.max_tokens ? end : a.max_tokens);
    }
    if (first_cta && b < a.batch) {
      a.cu_q[b] = static_cast<int32_t>(cu);
      a.new_seq_lens[b] = served ? len + add : len;
    }
    // pages handed out: the served requests with a need come first
    Scan2 got;
    block_scan2(Scan2{served ? need : 0, 0}, got, sums);
    taken += got.a;
    // (s_* are visible: block_scan2 ends with a barrier)
    const int n = min(kTablesThreads, a.batch - b0);
    const int c0 = s_cu[0], c1 = s_cu[kTablesThreads];
    for (int tile = c0 / kTablesThreads; tile * kTablesThreads < c1; ++tile) {
      if (tile % static_cast<int>(gridDim.x) != static_cast<int>(blockIdx.x)) continue;
      const int x = tile * kTablesThreads + t;
      if (x < c0 || x >= c1) continue;
      const int r = last_not_above(s_cu, n, x);
      const int row = b0 + r, l = s_len[r], first = s_first[r];
      const int pos = l + (x - s_cu[r]);
      const int pg = pos / a.page, off = pos % a.page, hp = (l + a.page - 1) / a.page;
      int slot = -1;
      if (first >= 0) {
        int32_t *entry = a.block_table + row * a.table_stride + pg;
        int page;
        if (pg < hp) {
          page = *entry;
        } else {
          page = a.free_pages[(static_cast<long long>(head) + first + (pg - hp)) % a.ring];
          if (off == 0) *entry = page;
        }
        if (page < 0 || page > 0x7fffffff / a.page - 1)
          bad |= kStatusBadIndex;
        else
          slot = page * a.page + off;
      }
      a.slots[x] = slot;
      a.positions[x] = pos;
    }
    pages0 += tot.a;
    tokens0 += tot.b;
    __syncthreads();  // s_* are rewritten by the next chunk
  }
  if (tokens0 > a.max_tokens) bad |= kStatusBadIndex;
  for (long long x = tokens0 + blockIdx.x * kTablesThreads + t; x < a.max_tokens;
       x += static_cast<long long>(gridDim.x) * kTablesThreads) {
    a.slots[x] = -1;
    a.positions[x] = 0;
  }
  if (first_cta && t == 0) {
    a.cu_q[a.batch] = static_cast<int32_t>(tokens0 < 0x7fffffff ? tokens0 : 0x7fffffff);
    a.new_free_state[0] = static_cast<int32_t>((head + taken) % a.ring);
    a.new_free_state[1] = static_cast<int32_t>(count - taken);
  }
  if (bad && (first_cta || (bad & kStatusBadIndex))) report(a.status, bad);
}

// Pages of finished requests to the ring's tail: the same sums, the pages of a
// chunk in the place of its tokens.
__global__ void __launch_bounds__(kTablesThreads) release_pages_kernel(const TablesArgs a) {
  __shared__ Scan2 sums[32];
  __shared__ int32_t s_at[kTablesThreads + 1];
  const int t = threadIdx.x;
  const bool first_cta = blockIdx.x == 0;
  int head = a.free_state[0], count = a.free_state[1];
  if (head < 0 || head >= a.ring || count < 0 || count > a.ring) {
    if (t == 0 && first_cta) report(a.status, kStatusBadIndex);
    head = 0;
    count = a.ring;  // nothing more is taken
  }
  long long pages0 = 0;
  int bad = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kTablesThreads) {
    const int b = b0 + t;
    int len = 0, done = 0;
    if (b < a.batch) {
      len = a.seq_lens[b];
      done = a.new_lens[b] != 0;
      if (len < 0) {
        bad |= kStatusBadIndex;
        len = 0;
      }
    }
    int pages = done ? (len + a.page - 1) / a.page : 0;
    if (pages > a.width) {
      bad |= kStatusBadIndex;
      pages = a.width;
    }
    Scan2 tot;
    const Scan2 sc = block_scan2(Scan2{pages, 0}, tot, sums);
    s_at[t] = static_cast<int32_t>(sc.a - pages);
    if (t == 0) s_at[kTablesThreads] = static_cast<int32_t>(tot.a);
    __syncthreads();
    if (first_cta && b < a.batch) a.new_seq_lens[b] = done ? 0 : len;
    const int n = min(kTablesThreads, a.batch - b0);
    const int end = s_at[kTablesThreads];
    for (int x = blockIdx.x * kTablesThreads + t; x < end; x += gridDim.x * kTablesThreads) {
      const int r = last_not_above(s_at, n, x);
      const int page = a.block_table[(b0 + r) * a.table_stride + (x - s_at[r])];
      const long long at = pages0 + x;  // among all released pages
      if (count + at < a.ring)
        a.free_pages[(head + count + at) % a.ring] = page;
      else
        bad |= kStatusBadIndex;  // more pages than the ring holds: given back twice
    }
    pages0 += tot.a;
    __syncthreads();
  }
  if (first_cta && t == 0) {
    const long long all = count + pages0;
    a.new_free_state[0] = head;
    a.new_free_state[1] = static_cast<int32_t>(all < a.ring ? all : a.ring);
  }
  if (bad) report(a.status, bad);
}

// ---------------------------------------------------------------------- append
struct AppendArgs {
  const void *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;  // element strides: token, head
  const int32_t *slots;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int32_t *status;
  int32_t tokens, heads_kv, page;
  int64_t num_pages;
};

// One CTA a token, K/V head and K or V (blockIdx.z); only the CTA of the first
// token of a page's run works, on the whole run.
template <int D, bool BF16, int CT>
__global__ void __launch_bounds__(128) cache_append_kernel(const AppendArgs a) {
  __shared__ float s_max[4];
  const int t0 = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int slot0 = a.slots[t0];
  if (slot0 < 0) return;
  const int page = slot0 / a.page;
  if (page >= a.num_pages) {
    if (tid == 0 && h == 0 && blockIdx.z == 0) report(a.status, kStatusBadIndex);
    return;
  }
  if (t0 > 0) {
    const int before = a.slots[t0 - 1];
    if (before >= 0 && before / a.page == page) return;
  }
  const uint16_t *src = static_cast<const uint16_t *>(blockIdx.z ? a.v : a.k) +
                        h * (blockIdx.z ? a.v_sh : a.k_sh);
  const int64_t st = blockIdx.z ? a.v_st : a.k_st;
  const int64_t ph = static_cast<int64_t>(page) * a.heads_kv + h;
  uint8_t *dst = (blockIdx.z ? a.v_cache : a.k_cache) + ph * a.page * D;
  float *scale = (blockIdx.z ? a.v_scale : a.k_scale) + ph;
  int n = 0;
  bool fresh = false;
  while (n < a.page && t0 + n < a.tokens) {
    const int s = a.slots[t0 + n];
    if (s < 0 || s / a.page != page) break;
    fresh |= s % a.page == 0;
    ++n;
  }
  float mx = 0.f;
  for (int e = tid; e < n * (D / 2); e += 128) {
    const int r = e / (D / 2), c = e % (D / 2);
    const float2 x = in16x2_to_float2<BF16>(
        *reinterpret_cast<const uint32_t *>(src + (t0 + r) * st + 2 * c));
    const float u = fabsf(x.x), w = fabsf(x.y);
    if (u <= 3.4028235e38f) mx = fmaxf(mx, u);
    if (w <= 3.4028235e38f) mx = fmaxf(mx, w);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  if ((tid & 31) == 0) s_max[tid >> 5] = mx;
  const float old = *scale;
  __syncthreads();
  mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  float sc = pow2f(scale_exp<CT>(mx));
  if (!fresh) sc = fmaxf(sc, old);
  const float inv = 1.f / sc;
  if (!fresh && sc != old) {  // the page's values in the larger scale
    const float ratio = old * inv;
    for (int e = tid; e < a.page * D / 4; e += 128) {
      uint32_t *p = reinterpret_cast<uint32_t *>(dst) + e;
      uint32_t p01, p23;
      cache4_to_f16<CT>(*p, p01, p23);
      const float2 x = f16x2_to_float2(p01), y = f16x2_to_float2(p23);
      *p = to_cache4<CT>(x.x * ratio, x.y * ratio, y.x * ratio, y.y * ratio);
    }
    __syncthreads();
  }
  if (tid == 0) *scale = sc;
  for (int e = tid; e < n * (D / 4); e += 128) {
    const int r = e / (D / 4), c = e % (D / 4);
    const uint2 raw = *reinterpret_cast<const uint2 *>(src + (t0 + r) * st + 4 * c);
    const float2 x = in16x2_to_float2<BF16>(raw.x), y = in16x2_to_float2<BF16>(raw.y);
    const int off = a.slots[t0 + r] % a.page;
    *reinterpret_cast<uint32_t *>(dst + off * D + 4 * c) =
        to_cache4<CT>(x.x * inv, x.y * inv, y.x * inv, y.y * inv);
  }
}

}  // namespace chia
