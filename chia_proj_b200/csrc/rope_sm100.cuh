// rope_sm100.cuh -- the norm of queries and keys, head by head, with the rotation
// to their positions in the same pass; forward and backward.
//
// A row is a token's query or key of one head. A group of D / 8 lanes holds it,
// eight channels a lane as four pairs that turn together: channels 4 l .. + 3 and
// those rot / 2 on, or (interleaved, and the channels that do not turn) 8 l .. + 7.
// So the rotation needs no exchange, and a lane's angles are pairs 4 l .. + 3 in
// either layout. A CTA takes a few tokens with all their heads: their angles' sines
// and cosines are computed once.
//
// An angle is pos * freq, in turns a product of whole numbers modulo 2^64, so the
// reduction is exact for any position; its upper 32 bits go to sincospi.
//
// Sums are in 32 bits; the output is rounded once. Bound by HBM.
#pragma once
#include "paged_common.cuh"

namespace chia {

enum RopeType : int { ROPE_BF16 = 0, ROPE_F16 = 1, ROPE_F32 = 2 };

struct RopeSide {  // queries or keys
  const void *x, *dy;  // input; gradient of the output (backward)
  void *y;             // output; gradient of the input (backward)
  const void *w;
  int64_t x_st[3], y_st[3], dy_st[3];  // element strides: batch, head, token
  int32_t heads;
  uint32_t magic;  // ceil(2^32 / heads); 0: one head
};
struct RopeArgs {
  RopeSide side[2];
  const uint64_t *freqs;
  const int32_t *positions;
  int64_t pos_stride;
  int32_t tokens, seqlen, rot, per_cta;  // tokens: of all batch entries
  int32_t w_type;
  float eps, w_offset;
  float *partial;  // backward: [CTAs][2][D] sums of the weights' gradients
};

constexpr int kRopeThreads = 256;
constexpr int kRopeTokens = 8;  // most tokens of a CTA at a time

template <int T>
struct RopeRaw {  // four channels
  using type = uint2;
};
template <>
struct RopeRaw<ROPE_F32> {
  using type = uint4;
};
template <int T>
__device__ __forceinline__ const typename RopeRaw<T>::type *rope_at(const void *p, int64_t e) {
  return reinterpret_cast<const typename RopeRaw<T>::type *>(static_cast<const uint8_t *>(p) +
                                                             e * (T == ROPE_F32 ? 4 : 2));
}
template <int T>
__device__ __forceinline__ float4 rope_values(const typename RopeRaw<T>::type &r) {
  if constexpr (T == ROPE_F32) {
    return make_float4(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w));
  } else {
    const float2 a = in16x2_to_float2<T == ROPE_BF16>(r.x), b = in16x2_to_float2<T == ROPE_BF16>(r.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
}
template <int T>
__device__ __forceinline__ void rope_store(void *p, int64_t e, const float *v) {
  auto *dst = const_cast<typename RopeRaw<T>::type *>(rope_at<T>(p, e));
  if constexpr (T == ROPE_F32)
    *dst = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else if constexpr (T == ROPE_BF16)
    *dst = make_uint2(ptx::pack_bf16(v[0], v[1]), ptx::pack_bf16(v[2], v[3]));
  else
    *dst = make_uint2(ptx::pack_f16(v[0], v[1]), ptx::pack_f16(v[2], v[3]));
}
__device__ __forceinline__ float rope_weight(const void *w, int type, int c) {
  if (type == ROPE_F32) return static_cast<const float *>(w)[c];
  const uint32_t v = static_cast<const uint16_t *>(w)[c];
  return type == ROPE_BF16 ? in16x2_to_float2<true>(v).x : in16x2_to_float2<false>(v).x;
}

// What both directions begin with: the angles of tokens [t0, t0 + n), where their rows are.
template <int D>
struct RopeShared {
  float cos[kRopeTokens][D / 2], sin[kRopeTokens][D / 2];
  int64_t x_at[2][kRopeTokens], y_at[2][kRopeTokens], dy_at[2][kRopeTokens];
};
template <int D, bool BACK>
__device__ __forceinline__ void rope_tokens(const RopeArgs &a, RopeShared<D> &s, int t0, int n) {
  for (int e = threadIdx.x; e < n * (D / 2); e += kRopeThreads) {
    const int j = e / (D / 2), i = e % (D / 2), t = t0 + j;
    float c = 1.f, sn = 0.f;
    if (i < a.rot / 2) {
      const int b = t / a.seqlen, at = t - b * a.seqlen;
      const int pos = a.positions != nullptr ? a.positions[b * a.pos_stride + at] : at;
      const uint64_t turn = static_cast<uint64_t>(static_cast<int64_t>(pos)) * a.freqs[i];
      // the upper 32 bits as -1/2 .. 1/2 of a turn, in half turns
      sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * 0x1p-31f, &sn, &c);
    }
    s.cos[j][i] = c, s.sin[j][i] = sn;
  }
  if (threadIdx.x < 2 * n) {
    const int j = threadIdx.x >> 1, t = t0 + j;
    const int64_t b = t / a.seqlen, at = t - b * a.seqlen;
    const int k = threadIdx.x & 1;
    const RopeSide &d = a.side[k];
    s.x_at[k][j] = b * d.x_st[0] + at * d.x_st[2];
    s.y_at[k][j] = b * d.y_st[0] + at * d.y_st[2];
    if (BACK) s.dy_at[k][j] = b * d.dy_st[0] + at * d.dy_st[2];
  }
}

// A lane's channels, of a row and of its angles.
struct RopeLane {
  int a, b;    // first channels of its two fours
  int pair;    // first pair
  bool turns;
  bool split;  // its pairs are (i, i + 4) of the eight, otherwise neighbours
};
template <int D, bool INTER>
__device__ __forceinline__ RopeLane rope_lane(int rot) {
  const int l = threadIdx.x % (D / 8);
  const bool turns = l < rot / 8, half = !INTER && turns;
  return {half ? 4 * l : 8 * l, half ? rot / 2 + 4 * l : 8 * l + 4, 4 * l, turns, half};
}
// (a, b) -> (a c - b s, b c + a s) of a lane's pairs
__device__ __forceinline__ void rope_turn(float (&v)[8], bool split, const float4 &c, const float4 &s) {
  const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = split ? v[i] : v[2 * i], b = split ? v[i + 4] : v[2 * i + 1];
    const float x = a * cc[i] - b * ss[i], y = b * cc[i] + a * ss[i];
    if (split)
      v[i] = x, v[i + 4] = y;
    else
      v[2 * i] = x, v[2 * i + 1] = y;
  }
}
template <int LANES>
__device__ __forceinline__ float rope_sum(float x) {
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
__device__ __forceinline__ int rope_div(uint32_t magic, int x) {
  return magic == 0 ? x : static_cast<int>(__umulhi(static_cast<uint32_t>(x), magic));
}

template <int T, int D, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int LANES = D / 8, GROUPS = kRopeThreads / LANES, U = 4;  // rows of a group at a time
  using Raw = typename RopeRaw<T>::type;
  __shared__ RopeShared<D> s;
  const RopeLane me = rope_lane<D, INTER>(a.rot);
  const int g = threadIdx.x / LANES;
  follow();
  const int t0 = blockIdx.x * a.per_cta, n = min(a.per_cta, a.tokens - t0);
  rope_tokens<D, false>(a, s, t0, n);
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const RopeSide &d = a.side[k];
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[i] = d.w != nullptr ? rope_weight(d.w, a.w_type, (i < 4 ? me.a : me.b - 4) + i) + a.w_offset : 1.f;
    const int rows = n * d.heads;
#pragma unroll 1
    for (int r0 = g; r0 - g < rows; r0 += U * GROUPS) {
      Raw raw[U][2];
      int tok[U], head[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * GROUPS;
        tok[u] = rope_div(d.magic, r), head[u] = r - tok[u] * d.heads;
        if (r < rows) {
          const int64_t at = s.x_at[k][tok[u]] + head[u] * d.x_st[1];
          raw[u][0] = *rope_at<T>(d.x, at + me.a);
          raw[u][1] = *rope_at<T>(d.x, at + me.b);
        } else {
          raw[u][0] = raw[u][1] = Raw{};
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float4 x0 = rope_values<T>(raw[u][0]), x1 = rope_values<T>(raw[u][1]);
        float v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
        const float rstd = rsqrtf(rope_sum<LANES>(sum) * (1.f / D) + a.eps);
        if (r0 + u * GROUPS < rows) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= rstd * w[i];
          if (me.turns)
            rope_turn(v, me.split, *reinterpret_cast<const float4 *>(&s.cos[tok[u]][me.pair]),
                      *reinterpret_cast<const float4 *>(&s.sin[tok[u]][me.pair]));
          const int64_t at = s.y_at[k][tok[u]] + head[u] * d.y_st[1];
          rope_store<T>(d.y, at + me.a, v);
          rope_store<T>(d.y, at + me.b, v + 4);
        }
      }
    }
  }
}

// Backward: with g the output's gradient turned back, xhat = x rstd,
//   dw = sum of g xhat,   dx = rstd (g w - xhat mean(g w xhat)).
// x and the gradient are read once, so the row's rstd is computed again. A CTA goes
// on over blocks of tokens and keeps its sums of dw in registers; they are added up
// by group, by CTA and in the kernel below in an order that is always the same.
template <int T, int D, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_bwd_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int LANES = D / 8, GROUPS = kRopeThreads / LANES, U = 2;
  using Raw = typename RopeRaw<T>::type;
  __shared__ RopeShared<D> s;
  __shared__ float s_dw[GROUPS][D];
  const RopeLane me = rope_lane<D, INTER>(a.rot);
  const int g = threadIdx.x / LANES;
  float dw[2][8] = {};
  follow();
  for (int t0 = blockIdx.x * a.per_cta; t0 < a.tokens; t0 += gridDim.x * a.per_cta) {
    const int n = min(a.per_cta, a.tokens - t0);
    rope_tokens<D, true>(a, s, t0, n);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const RopeSide &d = a.side[k];
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = d.w != nullptr ? rope_weight(d.w, a.w_type, (i < 4 ? me.a : me.b - 4) + i) + a.w_offset : 1.f;
      const int rows = n * d.heads;
#pragma unroll 1
      for (int r0 = g; r0 - g < rows; r0 += U * GROUPS) {
        Raw raw[U][2], grad[U][2];
        int tok[U], head[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * GROUPS;
          tok[u] = rope_div(d.magic, r), head[u] = r - tok[u] * d.heads;
          if (r < rows) {
            const int64_t at = s.x_at[k][tok[u]] + head[u] * d.x_st[1];
            const int64_t dat = s.dy_at[k][tok[u]] + head[u] * d.dy_st[1];
            raw[u][0] = *rope_at<T>(d.x, at + me.a);
            raw[u][1] = *rope_at<T>(d.x, at + me.b);
            grad[u][0] = *rope_at<T>(d.dy, dat + me.a);
            grad[u][1] = *rope_at<T>(d.dy, dat + me.b);
          } else {
            raw[u][0] = raw[u][1] = grad[u][0] = grad[u][1] = Raw{};
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bool real = r0 + u * GROUPS < rows;
          const float4 x0 = rope_values<T>(raw[u][0]), x1 = rope_values<T>(raw[u][1]);
          const float4 g0 = rope_values<T>(grad[u][0]), g1 = rope_values<T>(grad[u][1]);
          float v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
          float q[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
          const int j = real ? tok[u] : 0;
          const float4 sn = *reinterpret_cast<const float4 *>(&s.sin[j][me.pair]);
          if (me.turns)
            rope_turn(q, me.split, *reinterpret_cast<const float4 *>(&s.cos[j][me.pair]),
                      make_float4(-sn.x, -sn.y, -sn.z, -sn.w));
          float sum = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum), dot = fmaf(q[i] * w[i], v[i], dot);
          const float rstd = rsqrtf(rope_sum<LANES>(sum) * (1.f / D) + a.eps);
          dot = rope_sum<LANES>(dot) * (1.f / D) * rstd;  // mean(g w xhat)
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float xhat = v[i] * rstd;
            dw[k][i] = fmaf(q[i], xhat, dw[k][i]);
            o[i] = rstd * (q[i] * w[i] - xhat * dot);
          }
          if (real) {
            const int64_t at = s.y_at[k][tok[u]] + head[u] * d.y_st[1];
            rope_store<T>(d.y, at + me.a, o);
            rope_store<T>(d.y, at + me.b, o + 4);
          }
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (a.side[k].w == nullptr) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) s_dw[g][(i < 4 ? me.a : me.b - 4) + i] = dw[k][i];
    __syncthreads();
    if (threadIdx.x < D) {
      float sum = 0.f;
      for (int x = 0; x < GROUPS; ++x) sum += s_dw[x][threadIdx.x];
      a.partial[(static_cast<int64_t>(blockIdx.x) * 2 + k) * D + threadIdx.x] = sum;
    }
    __syncthreads();
  }
}

// The CTAs' sums of the weights' gradients, [parts][2][D], to dw[k][D]: a CTA 32
// channels, its 32 warps every 32nd part.
struct RopeSumArgs {
  const float *partial;
  void *dw[2];
  int32_t parts, dim, w_type;
};
static __global__ void __launch_bounds__(1024) rope_weight_sum_kernel(const RopeSumArgs a) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, k = c / a.dim;
  follow();
  float sum = 0.f;
#pragma unroll 4
  for (int p = warp; p < a.parts; p += 32) sum += a.partial[static_cast<int64_t>(p) * 2 * a.dim + c];
  s[warp][lane] = sum;
  __syncthreads();
  void *dw = k == 0 ? a.dw[0] : a.dw[1];
  if (warp == 0 && dw != nullptr) {
    sum = 0.f;
#pragma unroll
    for (int x = 0; x < 32; ++x) sum += s[x][lane];
    const int e = c - k * a.dim;
    if (a.w_type == ROPE_F32)
      static_cast<float *>(dw)[e] = sum;
    else
      static_cast<uint16_t *>(dw)[e] = static_cast<uint16_t>(
          a.w_type == ROPE_BF16 ? ptx::pack_bf16(sum, 0.f) : ptx::pack_f16(sum, 0.f));
  }
}

}  // namespace chia
