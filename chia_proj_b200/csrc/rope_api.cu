// rope_api.cu -- extern "C" entry points of the norm and rotation of queries and
// keys (include/chia_rope.h): argument checks, launch. No allocation, no
// synchronisation.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/chia_rope.h"
#include "rope_sm100.cuh"

namespace {

constexpr int64_t kI32 = 0x7fffffffLL;
constexpr int kMostHeads = 16384;

bool aligned(const void *p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int device_sms(int &sms) {
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
      major != 10 ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1)
    return CHIA_ERR_NO_DEVICE;
  return CHIA_OK;
}

bool type_ok(int t) { return t == CHIA_DTYPE_BF16 || t == CHIA_DTYPE_F16 || t == CHIA_DTYPE_F32; }

int check_strides(const int64_t *s) {
  for (int d = 0; d < 3; ++d) {
    if (s[d] < 0) return CHIA_ERR_INVALID_ARGUMENT;
    if (s[d] % 8 != 0) return CHIA_ERR_MISALIGNED;
  }
  return CHIA_OK;
}

int check(const chia_rope_params_t *p, bool outputs) {
  if (p == nullptr || p->abi_version != CHIA_ROPE_ABI_VERSION) return CHIA_ERR_INVALID_ARGUMENT;
  if (!type_ok(p->dtype) || !type_ok(p->weight_dtype)) return CHIA_ERR_UNSUPPORTED;
  if (p->head_dim != 64 && p->head_dim != 128) return CHIA_ERR_UNSUPPORTED;
  if (p->heads < 1 || p->heads_kv < 1 || p->heads > kMostHeads || p->heads_kv > kMostHeads || p->batch < 1 ||
      p->seqlen < 0 || p->rot < 0 || p->rot > p->head_dim || p->rot % 8 != 0 || p->position_stride < 0)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (p->batch > kI32 || p->seqlen > kI32 / p->batch) return CHIA_ERR_UNSUPPORTED;
  if (!std::isfinite(p->eps) || p->eps < 0.f || !std::isfinite(p->weight_offset)) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->rot > 0 && p->freqs == nullptr) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->seqlen > 0 && (!p->q || !p->k || (outputs && (!p->q_out || !p->k_out)))) return CHIA_ERR_INVALID_ARGUMENT;
  if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->q_out, 16) || !aligned(p->k_out, 16) ||
      !aligned(p->q_weight, 16) || !aligned(p->k_weight, 16) || !aligned(p->freqs, 8) || !aligned(p->positions, 4))
    return CHIA_ERR_MISALIGNED;
  for (const int64_t *s : {p->q_stride, p->k_stride, p->q_out_stride, p->k_out_stride}) {
    const int rc = check_strides(s);
    if (rc != CHIA_OK) return rc;
  }
  return CHIA_OK;
}

void set_side(chia::RopeSide &d, const void *x, void *y, const void *w, int heads, const int64_t *xs, const int64_t *ys) {
  d.x = x, d.y = y, d.w = w, d.heads = heads;
  for (int i = 0; i < 3; ++i) d.x_st[i] = xs[i], d.y_st[i] = ys[i];
}

void set_args(const chia_rope_params_t *p, chia::RopeArgs &a) {
  set_side(a.side[0], p->q, p->q_out, p->q_weight, p->heads, p->q_stride, p->q_out_stride);
  set_side(a.side[1], p->k, p->k_out, p->k_weight, p->heads_kv, p->k_stride, p->k_out_stride);
  a.freqs = p->freqs;
  a.positions = p->positions;
  a.pos_stride = p->position_stride;
  a.tokens = static_cast<int32_t>(p->batch * p->seqlen);
  a.seqlen = static_cast<int32_t>(p->seqlen);
  a.rot = p->rot;
  a.w_type = p->weight_dtype;
  a.eps = p->eps;
  a.w_offset = p->weight_offset;
}

// Groups that share a token: as many as make kTasks pieces of work for the GPU, a head at least
// to each.
constexpr int64_t kTasks = 32768;
// CTAs of the backward kernel, an SM: its groups go on from token to token and leave one sum of
// the weights' gradients a CTA.
constexpr int kBwdCtas = 4;
int set_grid(chia::RopeArgs &a, int dim, bool back, int sms) {
  const int heads = a.side[0].heads > a.side[1].heads ? a.side[0].heads : a.side[1].heads;
  a.part_bits = 0;
  while ((2 << a.part_bits) <= heads && (static_cast<int64_t>(a.tokens) << a.part_bits) < kTasks) ++a.part_bits;
  const int groups = chia::kRopeThreads / (dim / 8);
  const int64_t ctas = ((static_cast<int64_t>(a.tokens) << a.part_bits) + groups - 1) / groups;
  const int64_t most = back ? static_cast<int64_t>(kBwdCtas) * sms : kI32;
  return static_cast<int>(ctas < most ? ctas : most);
}

template <int T, int D, bool BACK>
int launch(const chia::RopeArgs &a, bool inter, int grid, cudaStream_t s) {
  const cudaError_t e =
      inter ? chia::launch_after(chia::qk_norm_rope_kernel<T, D, true, BACK>, dim3(grid), chia::kRopeThreads, 0, s, a)
            : chia::launch_after(chia::qk_norm_rope_kernel<T, D, false, BACK>, dim3(grid), chia::kRopeThreads, 0, s, a);
  return e == cudaSuccess ? CHIA_OK : CHIA_ERR_LAUNCH;
}
template <int T, int D>
int launch_fwd(const chia::RopeArgs &a, bool inter, int grid, cudaStream_t s) {
  return launch<T, D, false>(a, inter, grid, s);
}
template <int T, int D>
int launch_bwd(const chia::RopeArgs &a, bool inter, int grid, cudaStream_t s) {
  return launch<T, D, true>(a, inter, grid, s);
}
#define CHIA_ROPE_BY_TYPE(p, FN, ...)                                                             \
  ((p)->head_dim == 128 ? ((p)->dtype == CHIA_DTYPE_BF16  ? FN<chia::ROPE_BF16, 128>(__VA_ARGS__) \
                           : (p)->dtype == CHIA_DTYPE_F16 ? FN<chia::ROPE_F16, 128>(__VA_ARGS__)  \
                                                          : FN<chia::ROPE_F32, 128>(__VA_ARGS__)) \
                        : ((p)->dtype == CHIA_DTYPE_BF16  ? FN<chia::ROPE_BF16, 64>(__VA_ARGS__)  \
                           : (p)->dtype == CHIA_DTYPE_F16 ? FN<chia::ROPE_F16, 64>(__VA_ARGS__)   \
                                                          : FN<chia::ROPE_F32, 64>(__VA_ARGS__)))

}  // namespace

extern "C" {

int chia_qk_norm_rope(const chia_rope_params_t *p, void *stream) {
  int rc = check(p, true), sms = 0;
  if (rc != CHIA_OK || (rc = device_sms(sms)) != CHIA_OK) return rc;
  if (p->seqlen == 0) return CHIA_OK;
  chia::RopeArgs a{};
  set_args(p, a);
  const int grid = set_grid(a, p->head_dim, false, sms);
  return CHIA_ROPE_BY_TYPE(p, launch_fwd, a, p->interleaved != 0, grid, static_cast<cudaStream_t>(stream));
}

int64_t chia_qk_norm_rope_bwd_workspace_bytes(const chia_rope_params_t *p) {
  if (check(p, false) != CHIA_OK) return -1;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1)
    sms = 148;  // host-only callers (no GPU): size for a B200
  return static_cast<int64_t>(kBwdCtas) * sms * 2 * p->head_dim * 4;
}

int chia_qk_norm_rope_bwd(const chia_rope_params_t *p, const chia_rope_grads_t *g, void *workspace,
                          int64_t workspace_bytes, void *stream) {
  int rc = check(p, false), sms = 0;
  if (rc != CHIA_OK) return rc;
  if (g == nullptr) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->seqlen > 0 && (!g->dq_out || !g->dk_out || !g->dq || !g->dk)) return CHIA_ERR_INVALID_ARGUMENT;
  if ((g->dq_weight && !p->q_weight) || (g->dk_weight && !p->k_weight)) return CHIA_ERR_INVALID_ARGUMENT;
  const unsigned w = p->weight_dtype == CHIA_DTYPE_F32 ? 4 : 2;
  if (!aligned(g->dq_out, 16) || !aligned(g->dk_out, 16) || !aligned(g->dq, 16) || !aligned(g->dk, 16) ||
      !aligned(g->dq_weight, w) || !aligned(g->dk_weight, w) || !aligned(workspace, 16))
    return CHIA_ERR_MISALIGNED;
  if ((rc = check_strides(g->dq_out_stride)) != CHIA_OK || (rc = check_strides(g->dk_out_stride)) != CHIA_OK) return rc;
  const bool weights = p->q_weight != nullptr || p->k_weight != nullptr;
  if (weights && workspace == nullptr) return CHIA_ERR_INVALID_ARGUMENT;
  if ((rc = device_sms(sms)) != CHIA_OK) return rc;
  if (weights && workspace_bytes < static_cast<int64_t>(kBwdCtas) * sms * 2 * p->head_dim * 4)
    return CHIA_ERR_INVALID_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  chia::RopeArgs a{};
  set_args(p, a);
  a.side[0].y = g->dq, a.side[1].y = g->dk;
  a.side[0].dy = g->dq_out, a.side[1].dy = g->dk_out;
  for (int i = 0; i < 3; ++i) a.side[0].dy_st[i] = g->dq_out_stride[i], a.side[1].dy_st[i] = g->dk_out_stride[i];
  a.partial = static_cast<float *>(workspace);
  const int grid = set_grid(a, p->head_dim, true, sms);
  if (grid > 0) {
    rc = CHIA_ROPE_BY_TYPE(p, launch_bwd, a, p->interleaved != 0, grid, s);
    if (rc != CHIA_OK) return rc;
  }
  if (g->dq_weight == nullptr && g->dk_weight == nullptr) return CHIA_OK;
  // (no tokens: no parts, zeros)
  const chia::RopeSumArgs r{a.partial, {g->dq_weight, g->dk_weight}, grid, p->head_dim, p->weight_dtype};
  const cudaError_t e = chia::launch_after(chia::rope_weight_sum_kernel, dim3(2 * p->head_dim / 32), 1024, 0, s, r);
  return e == cudaSuccess ? CHIA_OK : CHIA_ERR_LAUNCH;
}

}  // extern "C"
