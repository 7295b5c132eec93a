// paged_attn_sm100.cuh -- attention over the paged 8-bit K/V cache.
#pragma once
#include "fmha_sm100.cuh"
#include "paged_common.cuh"

namespace chia {

struct PagedArgs {
  const void *q;
  void *o;
  int64_t q_st, q_sh, o_st, o_sh;  // element strides: token, head
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int32_t *block_table, *seq_lens, *cu_q;
  int64_t table_stride;
  float *lse;
  const float *head_param;
  MaskGeom mask;  // left, right, block, prefix, dil; positions
  float score_scale, softcap, sig_bias, out_scale;
  int32_t heads, heads_kv, group, batch, tokens, page, width;
  int64_t num_pages;
  int32_t *status;
};

// One warp a (query, head): the keys one after another, the head's channels
// over the lanes, an online softmax.
template <int D, bool BF16, int CT>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedArgs a, int kind) {
  constexpr int N = D / 32;  // channels a lane
  const int lane = threadIdx.x & 31;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x) >> 5;
  if (w >= static_cast<int64_t>(a.tokens) * a.heads) return;
  const int t = static_cast<int>(w / a.heads), h = static_cast<int>(w % a.heads);
  int b, i0, n;
  if (a.cu_q != nullptr) {
    if (t < a.cu_q[0] || t >= a.cu_q[a.batch]) return;
    b = last_not_above(a.cu_q, a.batch, t);
    i0 = a.cu_q[b];
    n = a.cu_q[b + 1] - i0;
    if (i0 < 0 || n < 1 || n > a.tokens - i0) {
      report(a.status, kStatusBadIndex);
      return;
    }
  } else {
    n = a.tokens / a.batch;
    b = t / n;
    i0 = b * n;
  }
  int len = a.seq_lens[b];
  if (len < 0 || len > a.width * a.page) {
    report(a.status, kStatusBadIndex);
    len = max(0, min(len, a.width * a.page));
  }
  const int64_t i = static_cast<int64_t>(len) - n + (t - i0);
  int64_t lo, hi;
  position_band(a.mask, i, len, lo, hi);
  const float hp = a.head_param != nullptr ? a.head_param[h] : 1.f;
  float q[N], o[N], m = -INFINITY, l = 0.f;
  const uint16_t *qp = static_cast<const uint16_t *>(a.q) + t * a.q_st + h * a.q_sh + lane * N;
#pragma unroll
  for (int c = 0; c < N; c += 2) {
    const float2 x = in16x2_to_float2<BF16>(*reinterpret_cast<const uint32_t *>(qp + c));
    q[c] = x.x;
    q[c + 1] = x.y;
    o[c] = o[c + 1] = 0.f;
  }
  const int hk = h / a.group;
  for (int64_t j = 0; j < len; ++j) {
    const bool vis = j < a.mask.prefix ||
                     (j >= lo && j <= hi && (a.mask.dil == 1 || (i - j) % a.mask.dil == 0));
    if (!vis) continue;
    const int page = a.block_table[b * a.table_stride + j / a.page];
    if (page < 0 || page >= a.num_pages) {
      report(a.status, kStatusBadIndex);
      continue;
    }
    const int64_t ph = static_cast<int64_t>(page) * a.heads_kv + hk;
    const int64_t at = (ph * a.page + j % a.page) * D + lane * N;
    float k[4], v[4];
    uint32_t kr, vr, p, r;
    if (N == 4) {
      kr = *reinterpret_cast<const uint32_t *>(a.k_cache + at);
      vr = *reinterpret_cast<const uint32_t *>(a.v_cache + at);
    } else {
      kr = *reinterpret_cast<const uint16_t *>(a.k_cache + at);
      vr = *reinterpret_cast<const uint16_t *>(a.v_cache + at);
    }
    cache4_to_f16<CT>(kr, p, r);
    float2 x = f16x2_to_float2(p), y = f16x2_to_float2(r);
    k[0] = x.x, k[1] = x.y, k[2] = y.x, k[3] = y.y;
    cache4_to_f16<CT>(vr, p, r);
    x = f16x2_to_float2(p), y = f16x2_to_float2(r);
    v[0] = x.x, v[1] = x.y, v[2] = y.x, v[3] = y.y;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) s = fmaf(q[c], k[c], s);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.k_scale[ph] * a.score_scale;
    float pr;
    if (kind == KIND_SIGMOID) {
      pr = 1.f / (1.f + expf(-(s + a.sig_bias)));
    } else if (kind == KIND_RELU) {
      pr = fmaxf(s, 0.f);
    } else {
      if (kind == KIND_SOFTCAP)
        s = a.softcap * tanhf(s / a.softcap);
      else if (kind == KIND_ALIBI)
        s = fmaf(hp, static_cast<float>(j - i), s);
      else
        s *= hp;
      const float mn = fmaxf(m, s);
      const float al = expf(m - mn);
      pr = expf(s - mn);
      l = l * al + pr;
      m = mn;
#pragma unroll
      for (int c = 0; c < N; ++c) o[c] *= al;
    }
    pr *= a.v_scale[ph];
#pragma unroll
    for (int c = 0; c < N; ++c) o[c] = fmaf(pr, v[c], o[c]);
  }
  const bool softmax = kind <= KIND_ALIBI;
  const float f = softmax ? (l > 0.f ? 1.f / l : 0.f) : (kind == KIND_RELU ? a.out_scale : 1.f);
  uint16_t *op = static_cast<uint16_t *>(a.o) + t * a.o_st + h * a.o_sh + lane * N;
#pragma unroll
  for (int c = 0; c < N; c += 2)
    *reinterpret_cast<uint32_t *>(op + c) =
        BF16 ? ptx::pack_bf16(o[c] * f, o[c + 1] * f) : ptx::pack_f16(o[c] * f, o[c + 1] * f);
  if (softmax && a.lse != nullptr && lane == 0)
    a.lse[static_cast<int64_t>(t) * a.heads + h] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace chia
