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
// enters the page in the block table. A few KB, so the time is latency: 64 decode
// steps 3.6 us, 512 prompts of up to 300 tokens 4.0 us, on the device.
__global__ void __launch_bounds__(kTablesThreads) page_tables_kernel(const TablesArgs a) {
  __shared__ Scan2 sums[32];
  __shared__ int32_t s_cu[kTablesThreads + 1], s_len[kTablesThreads], s_first[kTablesThreads];
  const int t = threadIdx.x, shift = 31 - __clz(a.page);
  const bool first_cta = blockIdx.x == 0;
  follow();
  int head = a.free_state[0], count = a.free_state[1];
  if (head < 0 || head >= a.ring || count < 0 || count > a.ring) {
    if (t == 0 && first_cta) report(a.status, kStatusBadIndex);
    head = 0;
    count = 0;
  }
  long long pages0 = 0, tokens0 = 0;
  int taken = 0;  // pages handed out, as far as this thread's requests know
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
    const int held = static_cast<int>((static_cast<long long>(len) + a.page - 1) >> shift);
    int need = static_cast<int>((static_cast<long long>(len) + add + a.page - 1) >> shift) - held;
    const bool fits = static_cast<long long>(held) + need <= a.width;
    if (!fits) need = 0;
    Scan2 tot;
    const Scan2 sc = block_scan2(Scan2{need, add}, tot, sums);
    const long long upto = pages0 + sc.a;  // pages wanted by the requests up to this one
    const bool served = fits && (need == 0 || upto <= count);
    if (b < a.batch && !served) bad |= kStatusNoPages;
    const long long cu = tokens0 + sc.b - add;
    // (tokens past max_tokens have no slot to be told, but their pages are entered all the same)
    constexpr long long kMost = 0x7fffffff;
    s_cu[t] = static_cast<int32_t>(min(cu, kMost));
    s_len[t] = len;
    s_first[t] = served ? static_cast<int32_t>(upto - need) : -1;
    if (t == kTablesThreads - 1) {
      const long long end = tokens0 + tot.b;
      s_cu[kTablesThreads] = static_cast<int32_t>(min(end, kMost));
    }
    if (first_cta && b < a.batch) {
      a.cu_q[b] = static_cast<int32_t>(min(cu, kMost));
      a.new_seq_lens[b] = served ? len + add : len;
    }
    if (served && need > 0) taken = static_cast<int>(upto);  // (those served come first)
    __syncthreads();
    const int n = min(kTablesThreads, a.batch - b0);
    const int c0 = s_cu[0], c1 = s_cu[kTablesThreads];
    // this CTA's tiles of kTablesThreads tokens: blockIdx.x, blockIdx.x + gridDim.x, ...
    const int g = static_cast<int>(gridDim.x);
    int tile = c0 / kTablesThreads;
    tile += (static_cast<int>(blockIdx.x) + g - tile % g) % g;
    for (; static_cast<long long>(tile) * kTablesThreads < c1; tile += g) {
      const int x = tile * kTablesThreads + t;
      if (x < c0 || x >= c1) continue;
      const int r = last_not_above(s_cu, n, x);
      const int l = s_len[r], first = s_first[r];
      const int pos = l + (x - s_cu[r]);
      const int pg = pos >> shift, off = pos & (a.page - 1), hp = (l + a.page - 1) >> shift;
      int slot = -1;
      if (first >= 0) {
        int32_t *entry = a.block_table + (b0 + r) * a.table_stride + pg;
        int page;
        if (pg < hp) {
          page = *entry;
        } else {
          unsigned at = static_cast<unsigned>(head) + first + (pg - hp);  // < 2 ring
          if (at >= static_cast<unsigned>(a.ring)) at -= a.ring;
          page = a.free_pages[at];
          if (off == 0) *entry = page;
        }
        if (page < 0 || page > (0x7fffffff >> shift) - 1)
          bad |= kStatusBadIndex;
        else
          slot = (page << shift) + off;
      }
      if (x < a.max_tokens) {
        a.slots[x] = slot;
        a.positions[x] = pos;
      }
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
  if (first_cta) {
    taken = __reduce_max_sync(0xffffffffu, taken);
    if ((t & 31) == 0) s_first[t >> 5] = taken;
    __syncthreads();
    if (t < 32) {
      taken = __reduce_max_sync(0xffffffffu, s_first[t]);
      if (t == 0) {
        a.cu_q[a.batch] = static_cast<int32_t>(tokens0 < 0x7fffffff ? tokens0 : 0x7fffffff);
        a.new_free_state[0] = static_cast<int32_t>((static_cast<long long>(head) + taken) % a.ring);
        a.new_free_state[1] = count - taken;
      }
    }
  }
  if (bad && (first_cta || (bad & kStatusBadIndex))) report(a.status, bad);
}

// Pages of finished requests (TRIM: those past the tokens that a request keeps) to the
// ring's tail: the same sums, the pages of a chunk in the place of its tokens. 64
// requests 3.5 us, 2048 of up to 128 pages 6.8, on the device.
template <bool TRIM>
__global__ void __launch_bounds__(kTablesThreads) release_pages_kernel(const TablesArgs a) {
  __shared__ Scan2 sums[32];
  __shared__ int32_t s_at[kTablesThreads + 1], s_kept[kTablesThreads];  // s_kept: pages
  const int t = threadIdx.x;
  const bool first_cta = blockIdx.x == 0;
  follow();
  int head = a.free_state[0], count = a.free_state[1];
  // In a ring that makes no sense there is no place for a page: nobody is released,
  // and the ring that goes on is empty, as page_tables leaves it then.
  const bool ring_ok = head >= 0 && head < a.ring && count >= 0 && count <= a.ring;
  if (!ring_ok) {
    if (t == 0 && first_cta) report(a.status, kStatusBadIndex);
    head = count = 0;
  }
  long long pages0 = 0;
  int bad = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kTablesThreads) {
    const int b = b0 + t;
    int len = 0, keep = 0;
    if (b < a.batch) {
      len = a.seq_lens[b];
      if (len < 0) {
        bad |= kStatusBadIndex;
        len = 0;
      }
      keep = TRIM ? a.new_lens[b] : a.new_lens[b] != 0 ? 0 : len;
      if (keep < 0 || keep > len) {
        bad |= kStatusBadIndex;
        keep = len;
      }
      if (!ring_ok) keep = len;
    }
    auto pages_of = [&](int n) { return (static_cast<long long>(n) + a.page - 1) / a.page; };
    if (keep < len && pages_of(len) > a.width) {  // which pages it holds is not known: it keeps them
      bad |= kStatusBadIndex;
      keep = len;
    }
    const long long kept = pages_of(keep), pages = pages_of(len) - kept;
    s_kept[t] = static_cast<int32_t>(kept);
    Scan2 tot;
    const Scan2 sc = block_scan2(Scan2{pages, 0}, tot, sums);
    // (of lengths that make no sense: pages past the 2^31st are in no ring)
    constexpr long long kMost = 0x7fffffff;
    s_at[t] = static_cast<int32_t>(min(sc.a - pages, kMost));
    if (t == 0) s_at[kTablesThreads] = static_cast<int32_t>(min(tot.a, kMost));
    __syncthreads();
    if (first_cta && b < a.batch) a.new_seq_lens[b] = keep;
    const int n = min(kTablesThreads, a.batch - b0);
    const int end = s_at[kTablesThreads];
    for (long long y = blockIdx.x * kTablesThreads + t; y < end; y += gridDim.x * kTablesThreads) {
      const int x = static_cast<int>(y), r = last_not_above(s_at, n, x);
      const int page = a.block_table[(b0 + r) * a.table_stride + s_kept[r] + (x - s_at[r])];
      const long long at = pages0 + x;  // among all released pages
      if (count + at < a.ring)
        a.free_pages[(static_cast<long long>(head) + count + at) % a.ring] = page;
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

// A page's tokens for one K/V head, K or V: 128 threads hold them in registers
// (16 bytes a load, all loads in flight at once), so the input is read once:
// the largest value decides the scale, then the values are rounded and stored.
// Bound by HBM: 2 bytes in and 1 out for each value. A CTA looks at `window`
// tokens and works on the runs of tokens of one page that begin there: a page's
// worth for prompts, one for decode steps, so that their few runs spread out. A run is
// what follows a page's first token within a page's number of rows, up to a token of
// another page; skipped tokens may lie between. The tokens before tell whether the run
// began earlier. A page that comes again behind another one, or goes on for more rows,
// would be rewritten by two CTAs at a time: that is seen a page's number of rows back,
// reported, and the later tokens are left out.
// Measured (8 K/V heads, D 128, bf16 to e4m3, pages of 64): 16 prompts of up to 4,099
// tokens 43 us, 5.1 TB/s, 78% of the copy rate; 64 single tokens 3.9 us, the launch and
// three dependent loads (slots, input, scale).
template <int D, bool BF16, int CT, int IT>
__global__ void __launch_bounds__(128, IT == 16 ? 4 : 8) cache_append_kernel(const AppendArgs a, int window) {
  constexpr int LANES = D / 8;       // threads of a row: 16 bytes each
  constexpr int STEP = 128 / LANES;  // rows of one load of the CTA
  constexpr int PAGE = IT * STEP;    // page_size
  constexpr int SHIFT = PAGE == 16 ? 4 : PAGE == 32 ? 5 : PAGE == 64 ? 6 : 7;
  __shared__ uint32_t s_max[2][4];
  __shared__ int s_slot[4 * PAGE];  // of the window, one page's number of rows before it and two behind it
  // Ballots of a run, one set for each of the warps whose lanes stand for a page's rows:
  // rows from its first token on that continue it; tokens of the page among them, of the
  // page's first slot; tokens in the rows before it, nearest first, of the page among them.
  struct __align__(16) Ballots {
    unsigned same, in, first, prev, prev_in;
  };
  constexpr int WORDS = (PAGE + 31) / 32;
  __shared__ Ballots s_run[2][WORDS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kinds = 2 * a.heads_kv;
  const int which = blockIdx.x % kinds, h = which >> 1;
  const bool is_v = which & 1;
  const int w0 = static_cast<int>(blockIdx.x / kinds) * window;
  const int w1 = min(w0 + window, a.tokens);
  const uint16_t *src = static_cast<const uint16_t *>(is_v ? a.v : a.k) + h * (is_v ? a.v_sh : a.k_sh) +
                        (tid % LANES) * 8;
  const int64_t st = is_v ? a.v_st : a.k_st;
  follow();
#pragma unroll
  for (int e = tid; e < 4 * PAGE; e += 128) {  // (all loads at once)
    const int x = w0 - PAGE + e;
    s_slot[e] = e < window + 3 * PAGE && x >= 0 && x < a.tokens ? a.slots[x] : -1;
  }
  __syncthreads();
  // Two sets of s_run and s_max by turns, one a run: a run has a barrier at least, so a set
  // is written again only behind the barrier of the run between.
  int par = 1;
  for (int t0 = w0; t0 < w1;) {
    const int at = t0 - w0 + PAGE, slot0 = s_slot[at];
    if (slot0 < 0) {  // skipped
      ++t0;
      continue;
    }
    // the run: the following tokens in the same page, and skipped ones between them
    par ^= 1;
    const int page = slot0 >> SHIFT;
    if (warp < WORDS) {
      const bool row = PAGE >= 32 || lane < PAGE;
      const int next = row ? s_slot[at + tid] : -1, last = row ? s_slot[at - 1 - tid] : -1;
      const int later = row ? s_slot[at + PAGE + tid] : -1;
      const bool in = (next >> SHIFT) == page;  // (that of a skipped one is negative)
      Ballots b;
      b.in = __ballot_sync(0xffffffffu, in);
      b.same = b.in | __ballot_sync(0xffffffffu, row && next < 0);
      b.first = __ballot_sync(0xffffffffu, in && (next & (PAGE - 1)) == 0);
      b.prev = __ballot_sync(0xffffffffu, last >= 0);
      b.prev_in = __ballot_sync(0xffffffffu, (last >> SHIFT) == page);
      if (lane == 0) s_run[par][warp] = b;
      if ((later >> SHIFT) == page && which == 0) report(a.status, kStatusBadIndex);  // more rows than a page's
    }
    __syncthreads();
    int n = 0;
    bool fresh = false;  // it holds the page's first slot
    bool begun = false;  // the token before is of this page, or one before that
    bool adjacent = false;
    bool holes = false;  // skipped tokens in the run
    unsigned before = 0;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const Ballots b = s_run[par][w];
      if (before == 0) {
        before = b.prev & -b.prev;
        adjacent = (b.prev_in & before) != 0;
      }
      begun |= b.prev_in != 0;
      if (n == 32 * w) {
        const int here = b.same == ~0u ? 32 : __ffs(~b.same) - 1;
        const unsigned rows = here == 32 ? ~0u : (1u << here) - 1;
        n += here;
        fresh |= (b.first & rows) != 0;
        holes |= (~b.in & rows) != 0;
      }
    }
    if (begun || page >= a.num_pages) {
      if (!adjacent && tid == 0 && which == 0) report(a.status, kStatusBadIndex);
      t0 += n;
      continue;
    }
    const int64_t ph = static_cast<int64_t>(page) * a.heads_kv + h;
    uint8_t *dst = (is_v ? a.v_cache : a.k_cache) + ph * PAGE * D;
    float *scale = (is_v ? a.v_scale : a.k_scale) + ph;
    unsigned skipped = 0;  // bits: this thread's rows
    if (holes) {
#pragma unroll 1
      for (int i = 0; i < IT; ++i) skipped |= (s_slot[at + i * STEP + tid / LANES] < 0 ? 1u : 0u) << i;
    }
    uint4 x[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = i * STEP + tid / LANES;
      x[i] = make_uint4(0, 0, 0, 0);
      if (r < n && !((skipped >> i) & 1)) x[i] = *reinterpret_cast<const uint4 *>(src + (t0 + r) * st);
    }
    const float old = *scale;
    // the largest value: 16-bit patterns without their signs order as the values do
    constexpr uint32_t INF = BF16 ? 0x7f80u : 0x7c00u;
    uint32_t m2 = 0;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) m2 = __vmaxu2(m2, w[j] & 0x7fff7fffu);
    }
    m2 = max(m2 & 0xffffu, m2 >> 16);
    if (m2 >= INF) {  // infinities and NaN do not count
      m2 = 0;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u = w[j] & 0x7fffu, v = (w[j] >> 16) & 0x7fffu;
          m2 = max(m2, max(u < INF ? u : 0u, v < INF ? v : 0u));
        }
      }
    }
    m2 = __reduce_max_sync(0xffffffffu, m2);
    if (lane == 0) s_max[par][warp] = m2;
    __syncthreads();
    m2 = max(max(s_max[par][0], s_max[par][1]), max(s_max[par][2], s_max[par][3]));
    const float mx = in16x2_to_float2<BF16>(m2).x;
    float sc = pow2f(scale_exp<CT>(mx));
    if (!fresh) sc = fmaxf(sc, old);
    const float inv = 1.f / sc;
    if (!fresh && sc != old) {  // the page's values in the larger scale
      const float ratio = old * inv;
      for (int e = tid; e < PAGE * D / 16; e += 128) {
        uint4 *p = reinterpret_cast<uint4 *>(dst) + e;
        uint4 v = *p;
        auto again = [&](uint32_t w) {
          uint32_t p01, p23;
          cache4_to_f16<CT>(w, p01, p23);
          const float2 f = f16x2_to_float2(p01), g = f16x2_to_float2(p23);
          return to_cache4<CT>(f.x * ratio, f.y * ratio, g.x * ratio, g.y * ratio);
        };
        v.x = again(v.x), v.y = again(v.y), v.z = again(v.z), v.w = again(v.w);
        *p = v;
      }
      __syncthreads();
    }
    if (tid == 0 && (fresh || sc != old)) *scale = sc;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = i * STEP + tid / LANES;
      if (r < n && !((skipped >> i) & 1)) {
        const float2 f0 = in16x2_to_float2<BF16>(x[i].x), f1 = in16x2_to_float2<BF16>(x[i].y);
        const float2 f2 = in16x2_to_float2<BF16>(x[i].z), f3 = in16x2_to_float2<BF16>(x[i].w);
        *reinterpret_cast<uint2 *>(dst + (s_slot[at + r] & (PAGE - 1)) * D + (tid % LANES) * 8) =
            make_uint2(to_cache4<CT>(f0.x * inv, f0.y * inv, f1.x * inv, f1.y * inv),
                       to_cache4<CT>(f2.x * inv, f2.y * inv, f3.x * inv, f3.y * inv));
      }
    }
    t0 += n;
  }
}

}  // namespace chia
