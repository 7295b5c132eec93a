// rope_sm100.cuh -- the norm of queries and keys, head by head, with the rotation
// to their positions in the same pass; forward and backward.
//
// A row is a token's query or key of one head. A group of D / 8 lanes holds it,
// eight channels a lane as four pairs that turn together: channels 4 l .. + 3 and
// those rot / 2 on, or (interleaved, and the channels that do not turn) 8 l .. + 7.
// So the rotation needs no exchange, and a lane's angles are pairs 4 l .. + 3 in
// either layout. A group stays with a token and goes over its heads (or each `parts`-th
// of them): its angles and their products with the weights are computed once, in
// registers, and the next row is a stride away. Groups have nothing in common, so there
// is no barrier.
//
// An angle is pos * freq, in turns a product of whole numbers modulo 2^64, so the
// reduction is exact for any position; of its upper 32 bits sine and cosine are computed.
//
// Sums are in 32 bits; the output is rounded once. Bound by HBM, and next to it by the
// number of instructions. Measured, bf16, D 128: 4 x 4,096 tokens of 16 + 16 heads forward 46.9 us
// (5.7 TB/s, 89% of the rate of a copy), backward 79.7 (5.1 TB/s); 16,421 tokens of 32 + 8 heads out
// of one projection, half of the channels turned, 60.1 (5.6 TB/s); one token 2.9. Tried: a block of
// tokens a CTA with the angles in shared memory, forward 53.2 and backward 114; rows through
// rings of asynchronous copies, 74.6 and 114 (240 instructions a warp and pair of rows where this has 124).
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
};
struct RopeArgs {
  RopeSide side[2];
  const uint64_t *freqs;
  const int32_t *positions;
  int64_t pos_stride;
  int32_t tokens, seqlen, rot, part_bits;  // tokens: of all batch entries; 2^part_bits groups share a token
  int32_t w_type;
  float eps, w_offset;
  float *partial;  // backward: [CTAs][2][D] sums of the weights' gradients
};

constexpr int kRopeThreads = 128;

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
// A lane's eight channels as four pairs (a_i, b_i), two to a register pair: packed
// arithmetic takes half the instructions, which are what bounds these kernels next to HBM.
struct RopeVals {
  uint64_t a[2], b[2];
};
// INTER: the channels are a0 b0 a1 b1 .., otherwise the first four and the second four
template <bool INTER>
__device__ __forceinline__ RopeVals rope_pairs(const float (&x)[8]) {
  if (INTER) return {{ptx::f2(x[0], x[2]), ptx::f2(x[4], x[6])}, {ptx::f2(x[1], x[3]), ptx::f2(x[5], x[7])}};
  return {{ptx::f2(x[0], x[1]), ptx::f2(x[2], x[3])}, {ptx::f2(x[4], x[5]), ptx::f2(x[6], x[7])}};
}
template <int T, bool INTER>
__device__ __forceinline__ RopeVals rope_values(const typename RopeRaw<T>::type (&r)[2]) {
  float x[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (T == ROPE_F32) {
      x[4 * h] = __uint_as_float(r[h].x), x[4 * h + 1] = __uint_as_float(r[h].y);
      x[4 * h + 2] = __uint_as_float(r[h].z), x[4 * h + 3] = __uint_as_float(r[h].w);
    } else {
      const float2 f = in16x2_to_float2<T == ROPE_BF16>(r[h].x), g = in16x2_to_float2<T == ROPE_BF16>(r[h].y);
      x[4 * h] = f.x, x[4 * h + 1] = f.y, x[4 * h + 2] = g.x, x[4 * h + 3] = g.y;
    }
  }
  return rope_pairs<INTER>(x);
}
// the channels in their order again
template <bool INTER>
__device__ __forceinline__ void rope_channels(const RopeVals &v, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float a0, a1, b0, b1;
    ptx::f2_split(v.a[h], a0, a1);
    ptx::f2_split(v.b[h], b0, b1);
    if (INTER)
      x[4 * h] = a0, x[4 * h + 1] = b0, x[4 * h + 2] = a1, x[4 * h + 3] = b1;
    else
      x[2 * h] = a0, x[2 * h + 1] = a1, x[4 + 2 * h] = b0, x[4 + 2 * h + 1] = b1;
  }
}
template <int T, bool INTER>
__device__ __forceinline__ void rope_store(uint8_t *p, int ab, const RopeVals &v) {  // ab: bytes between the fours
  float x[8];
  rope_channels<INTER>(v, x);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    auto *dst = reinterpret_cast<typename RopeRaw<T>::type *>(p + (h ? ab : 0));
    const float *y = x + 4 * h;
    if constexpr (T == ROPE_F32)
      *dst = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
    else if constexpr (T == ROPE_BF16)
      *dst = make_uint2(ptx::pack_bf16(y[0], y[1]), ptx::pack_bf16(y[2], y[3]));
    else
      *dst = make_uint2(ptx::pack_f16(y[0], y[1]), ptx::pack_f16(y[2], y[3]));
  }
}
__device__ __forceinline__ RopeVals rope_mul(const RopeVals &x, const RopeVals &y) {
  return {{ptx::mul2(x.a[0], y.a[0]), ptx::mul2(x.a[1], y.a[1])}, {ptx::mul2(x.b[0], y.b[0]), ptx::mul2(x.b[1], y.b[1])}};
}
__device__ __forceinline__ RopeVals rope_fma(const RopeVals &x, const RopeVals &y, const RopeVals &z) {
  return {{ptx::fma2(x.a[0], y.a[0], z.a[0]), ptx::fma2(x.a[1], y.a[1], z.a[1])},
          {ptx::fma2(x.b[0], y.b[0], z.b[0]), ptx::fma2(x.b[1], y.b[1], z.b[1])}};
}
__device__ __forceinline__ RopeVals rope_all(float f) {
  const uint64_t x = ptx::f2(f, f);
  return {{x, x}, {x, x}};
}
// sum of a lane's products
__device__ __forceinline__ float rope_dot(const RopeVals &x, const RopeVals &y) {
  const uint64_t s = ptx::fma2(x.b[1], y.b[1], ptx::fma2(x.b[0], y.b[0], ptx::fma2(x.a[1], y.a[1], ptx::mul2(x.a[0], y.a[0]))));
  float lo, hi;
  ptx::f2_split(s, lo, hi);
  return lo + hi;
}
// A lane's channels, of a row and of its angles.
struct RopeLane {
  int a, b;    // first channels of its two fours
  int pair;    // first pair
  bool turns;
};
template <int D, bool INTER>
__device__ __forceinline__ RopeLane rope_lane(int rot) {
  const int l = threadIdx.x % (D / 8);
  const bool turns = l < rot / 8, half = !INTER && turns;
  return {half ? 4 * l : 8 * l, half ? rot / 2 + 4 * l : 8 * l + 4, 4 * l, turns};
}
// (a, b) -> (a ca - b sb, b cb + a sa) of a lane's pairs; lanes that do not turn have no sines
struct RopeTurn {
  uint64_t ca[2], cb[2], sa[2], sb[2];  // sb: negative
};
__device__ __forceinline__ RopeVals rope_turn(const RopeVals &v, const RopeTurn &c, bool turns) {
  RopeVals r;
#pragma unroll
  for (int h = 0; h < 2; ++h) r.a[h] = ptx::mul2(v.a[h], c.ca[h]), r.b[h] = ptx::mul2(v.b[h], c.cb[h]);
  if (turns) {
#pragma unroll
    for (int h = 0; h < 2; ++h) r.a[h] = ptx::fma2(v.b[h], c.sb[h], r.a[h]), r.b[h] = ptx::fma2(v.a[h], c.sa[h], r.b[h]);
  }
  return r;
}
template <int LANES>
__device__ __forceinline__ float rope_sum(float x) {
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
// a lane's eight weights (ones where there are none)
template <bool INTER>
__device__ __forceinline__ RopeVals rope_weights(const RopeArgs &a, const void *w, const RopeLane &me) {
  if (w == nullptr) return rope_all(1.f);
  RopeVals v;
  if (a.w_type == ROPE_F32) {
    const uint4 r[2] = {*rope_at<ROPE_F32>(w, me.a), *rope_at<ROPE_F32>(w, me.b)};
    v = rope_values<ROPE_F32, INTER>(r);
  } else {
    const uint2 r[2] = {*rope_at<ROPE_BF16>(w, me.a), *rope_at<ROPE_BF16>(w, me.b)};
    v = a.w_type == ROPE_BF16 ? rope_values<ROPE_BF16, INTER>(r) : rope_values<ROPE_F16, INTER>(r);
  }
  const RopeVals o = rope_all(a.w_offset);
  return {{ptx::add2(v.a[0], o.a[0]), ptx::add2(v.a[1], o.a[0])}, {ptx::add2(v.b[0], o.a[0]), ptx::add2(v.b[1], o.a[0])}};
}
// Cosines and sines of four angles, turns in units of 2^-64. The nearest quarter turn goes to a
// choice of signs and sides; what is left, |x| <= pi / 4, to the Taylor polynomials
//   sin x = x - x^3/3! + .. + x^9/9!,  cos x = 1 - x^2/2! + .. + x^10/10!
// whose next terms are 2^-29 and 2^-33.
__device__ __forceinline__ void rope_angles(const uint64_t (&turn)[4], uint64_t (&cos)[2], uint64_t (&sin)[2]) {
  float c[4], s[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float x[2];
    uint32_t quarter[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t t = static_cast<uint32_t>(turn[2 * h + i] >> 32);
      quarter[i] = (t + 0x20000000u) >> 30;
      x[i] = static_cast<float>(static_cast<int32_t>(t - (quarter[i] << 30))) * 1.4629180792671596e-9f;  // pi / 2^31
    }
    auto all = [](float f) { return ptx::f2(f, f); };
    const uint64_t X = ptx::f2(x[0], x[1]), X2 = ptx::mul2(X, X);
    uint64_t S = ptx::fma2(X2, all(1.f / 362880.f), all(-1.f / 5040.f));
    S = ptx::fma2(X2, S, all(1.f / 120.f));
    S = ptx::fma2(X2, S, all(-1.f / 6.f));
    S = ptx::fma2(ptx::mul2(X, X2), S, X);
    uint64_t C = ptx::fma2(X2, all(-1.f / 3628800.f), all(1.f / 40320.f));
    C = ptx::fma2(X2, C, all(-1.f / 720.f));
    C = ptx::fma2(X2, C, all(1.f / 24.f));
    C = ptx::fma2(X2, C, all(-0.5f));
    C = ptx::fma2(X2, C, all(1.f));
    float sv[2], cv[2];
    ptx::f2_split(S, sv[0], sv[1]);
    ptx::f2_split(C, cv[0], cv[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // by q quarter turns: (c, s), (-s, c), (-c, -s), (s, -c)
      const uint32_t q = quarter[i];
      const float a = q & 1 ? sv[i] : cv[i], b = q & 1 ? cv[i] : sv[i];
      c[2 * h + i] = __uint_as_float(__float_as_uint(a) ^ (((q + 1) & 2) << 30));
      s[2 * h + i] = __uint_as_float(__float_as_uint(b) ^ ((q & 2) << 30));
    }
  }
  cos[0] = ptx::f2(c[0], c[1]), cos[1] = ptx::f2(c[2], c[3]);
  sin[0] = ptx::f2(s[0], s[1]), sin[1] = ptx::f2(s[2], s[3]);
}

// Forward: y = turn(x rstd w). Backward (BACK): with g the output's gradient turned back
// and xhat = x rstd,
//   dw = sum of g xhat,   dx = rstd (g w - xhat mean(g w xhat));
// x and the gradient are read once, so the row's rstd is computed again. Sums of dw stay in
// registers while a group goes on from token to token; they are added up by group, by CTA
// and in the kernel below in an order that is always the same. The backward kernel asks for the
// next rows before it computes these: 108 us without, and 80 at 128 registers a thread; forward,
// eight CTAs an SM of 64 registers do as much.
template <int T, int D, bool INTER, bool BACK>
__global__ void __launch_bounds__(kRopeThreads, BACK ? 4 : 8) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int LANES = D / 8, GROUPS = kRopeThreads / LANES, SIZE = T == ROPE_F32 ? 4 : 2;
  constexpr int U = (BACK ? 2 : 4) / (T == ROPE_F32 ? 2 : 1);  // rows on their way at a time
  using Raw = typename RopeRaw<T>::type;
  __shared__ float s_dw[BACK ? GROUPS : 1][D];
  const RopeLane me = rope_lane<D, INTER>(a.rot);
  const int ab = (me.b - me.a) * SIZE;  // bytes
  const int g = threadIdx.x / LANES, parts = 1 << a.part_bits;
  const int64_t tasks = static_cast<int64_t>(a.tokens) << a.part_bits;
  RopeVals dw[BACK ? 2 : 1] = {};
  follow();
  // (a warp's groups go on together, as its shuffles want)
  const int64_t warp0 = static_cast<int64_t>(blockIdx.x) * GROUPS + g / (32 / LANES) * (32 / LANES);
#pragma unroll 1
  for (int64_t task0 = warp0; task0 < tasks; task0 += static_cast<int64_t>(gridDim.x) * GROUPS) {
    const int64_t task = task0 + g % (32 / LANES);
    const bool there = task < tasks;
    const int token = there ? static_cast<int>(task >> a.part_bits) : 0, part = static_cast<int>(task) & (parts - 1);
    int b = 0, at = token;
    if (a.seqlen != a.tokens) b = token / a.seqlen, at = token - b * a.seqlen;
    uint64_t cos[2], sin[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const RopeSide &d = a.side[k];
      auto row = [&](const void *p, const int64_t(&st)[3]) {
        return static_cast<const uint8_t *>(p) + (b * st[0] + at * st[2] + part * st[1] + me.a) * SIZE;
      };
      const uint8_t *xp = row(d.x, d.x_st), *dp = BACK ? row(d.dy, d.dy_st) : nullptr;
      uint8_t *yp = const_cast<uint8_t *>(row(d.y, d.y_st));
      const int64_t xs = (d.x_st[1] << a.part_bits) * SIZE, ys = (d.y_st[1] << a.part_bits) * SIZE,
                    ds = BACK ? (d.dy_st[1] << a.part_bits) * SIZE : 0;
      const int trips = (d.heads + parts - 1) >> a.part_bits;
      const int have = there ? (d.heads - part + parts - 1) >> a.part_bits : 0;  // rows of this group
      Raw raw[U][2], grad[BACK ? U : 1][2];
      auto get = [](const uint8_t *p) { return *reinterpret_cast<const Raw *>(p); };
      auto load = [&](int left) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u < left) {
            raw[u][0] = get(xp), raw[u][1] = get(xp + ab);
            if (BACK) grad[u][0] = get(dp), grad[u][1] = get(dp + ab);
          }
          xp += xs, dp += ds;
        }
      };
      load(have);  // (the angles and weights are computed while the first rows are on their way)
      if (k == 0) {
        const int pos = a.positions != nullptr ? a.positions[b * a.pos_stride + at] : at;
        uint64_t turn[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          turn[i] = me.turns ? static_cast<uint64_t>(static_cast<int64_t>(pos)) * a.freqs[me.pair + i] : 0;
        rope_angles(turn, cos, sin);
      }
      const RopeVals w = rope_weights<INTER>(a, d.w, me);
      RopeTurn c;
      const uint64_t neg = ptx::f2(-1.f, -1.f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (BACK) {
          c.ca[h] = c.cb[h] = cos[h], c.sb[h] = sin[h], c.sa[h] = ptx::mul2(sin[h], neg);
        } else {
          c.ca[h] = ptx::mul2(w.a[h], cos[h]), c.cb[h] = ptx::mul2(w.b[h], cos[h]);
          c.sa[h] = ptx::mul2(w.a[h], sin[h]), c.sb[h] = ptx::mul2(ptx::mul2(w.b[h], sin[h]), neg);
        }
      }
      int left = have;
#pragma unroll 1
      for (int j = 0; j < trips; j += U, left -= U) {
        Raw x[U][2], dy[BACK ? U : 1][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u][0] = raw[u][0], x[u][1] = raw[u][1];
          if (BACK) dy[u][0] = grad[u][0], dy[u][1] = grad[u][1];
        }
        if (BACK && j + U < trips) load(left - U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const RopeVals v = rope_values<T, INTER>(x[u]);
          const float rstd = rsqrtf(rope_sum<LANES>(rope_dot(v, v)) * (1.f / D) + a.eps);
          if constexpr (BACK) {
            const RopeVals q = rope_turn(rope_values<T, INTER>(dy[u]), c, me.turns);
            const RopeVals gw = rope_mul(q, w);
            const float dot = rope_sum<LANES>(rope_dot(gw, v)) * (1.f / D) * rstd;  // mean(g w xhat)
            if (u < left) {
              const RopeVals xhat = rope_mul(v, rope_all(rstd));
              dw[k] = rope_fma(q, xhat, dw[k]);
              rope_store<T, INTER>(yp, ab, rope_mul(rope_fma(xhat, rope_all(-dot), gw), rope_all(rstd)));
            }
          } else {
            if (u < left) rope_store<T, INTER>(yp, ab, rope_turn(rope_mul(v, rope_all(rstd)), c, me.turns));
          }
          yp += ys;
        }
        if (!BACK && j + U < trips) load(left - U);
      }
    }
  }
  if constexpr (BACK) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (a.side[k].w == nullptr) continue;
      __syncthreads();
      float x[8];
      rope_channels<INTER>(dw[k], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) s_dw[g][(i < 4 ? me.a : me.b - 4) + i] = x[i];
      __syncthreads();
      if (threadIdx.x < D) {
        float sum = 0.f;
        for (int x = 0; x < GROUPS; ++x) sum += s_dw[x][threadIdx.x];
        a.partial[(static_cast<int64_t>(blockIdx.x) * 2 + k) * D + threadIdx.x] = sum;
      }
    }
  }
}

// The CTAs' sums of the weights' gradients, [parts][2][D], to dw[k][D]: a CTA 32 channels,
// its 32 warps every 32nd part.
struct RopeSumArgs {
  const float *partial;
  void *dw[2];
  int32_t parts, dim, w_type;
};
static __global__ void __launch_bounds__(1024) rope_weight_sum_kernel(const RopeSumArgs a) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane, k = c / a.dim, e = c - k * a.dim;
  follow();
  void *dw = k == 0 ? a.dw[0] : a.dw[1];
  if (dw == nullptr) return;
  float sum = 0.f;
#pragma unroll 4
  for (int p = warp; p < a.parts; p += 32) sum += a.partial[static_cast<int64_t>(p) * 2 * a.dim + c];
  s[warp][lane] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = 0.f;
#pragma unroll
    for (int x = 0; x < 32; ++x) sum += s[x][lane];
    if (a.w_type == ROPE_F32)
      static_cast<float *>(dw)[e] = sum;
    else
      static_cast<uint16_t *>(dw)[e] = static_cast<uint16_t>(
          a.w_type == ROPE_BF16 ? ptx::pack_bf16(sum, 0.f) : ptx::pack_f16(sum, 0.f));
  }
}

}  // namespace chia
