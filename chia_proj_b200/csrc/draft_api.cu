// draft_api.cu -- extern "C" entry points of the tables, the verification and the
// compaction of drafted tokens (include/chia_draft.h; its attention is in
// paged_api.cu): argument checks, launch. No allocation, no synchronisation.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/chia_draft.h"
#include "draft_sm100.cuh"

namespace {

constexpr int64_t kI32 = 0x7fffffffLL;

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

int launched(cudaError_t e) { return e == cudaSuccess ? CHIA_OK : CHIA_ERR_LAUNCH; }

// vec: rows are aligned so that four entries are one load
template <int T>
int launch_verify(const chia::VerifyArgs &a, bool vec, int sms, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch) * chia::kVerifyCtas);
  // A warp for each chunk of a CTA, but no more threads than the GPU holds at once (1024 an SM):
  // a request alone waits for one round of loads, a full batch runs side by side.
  int threads = 128;
  const int chunks = (a.chunks + chia::kVerifyCtas - 1) / chia::kVerifyCtas;
  while (threads < chia::kVerifyMostThreads && threads < 32 * chunks &&
         2ll * threads * chia::kVerifyCtas * a.batch <= 1024ll * sms)
    threads *= 2;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = chia::kVerifyCtas, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  auto run = [&](void (*kernel)(chia::VerifyArgs)) { return launched(cudaLaunchKernelEx(&cfg, kernel, a)); };
  if (a.q != nullptr) return vec ? run(chia::verify_kernel<T, true, true>) : run(chia::verify_kernel<T, true, false>);
  return vec ? run(chia::verify_kernel<T, false, true>) : run(chia::verify_kernel<T, false, false>);
}

}  // namespace

extern "C" {

int chia_tree_tables(const chia_tree_params_t *p, void *stream) {
  if (p == nullptr || p->abi_version != CHIA_DRAFT_ABI_VERSION) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->batch < 1 || p->batch > (1 << 24) || p->tokens < 0 || p->tokens > kI32 || !p->cu_q || !p->seq_lens ||
      (p->tokens > 0 && (!p->parents || !p->positions || !p->ancestors)))
    return CHIA_ERR_INVALID_ARGUMENT;
  if (!aligned(p->parents, 4) || !aligned(p->cu_q, 4) || !aligned(p->seq_lens, 4) || !aligned(p->positions, 4) ||
      !aligned(p->ancestors, 8) || !aligned(p->status, 4))
    return CHIA_ERR_MISALIGNED;
  int sms = 0;
  const int rc = device_sms(sms);
  if (rc != CHIA_OK) return rc;
  if (p->tokens == 0) return CHIA_OK;
  chia::TreeArgs a{};
  a.parents = p->parents;
  a.cu_q = p->cu_q;
  a.seq_lens = p->seq_lens;
  a.positions = p->positions;
  a.ancestors = reinterpret_cast<unsigned long long *>(p->ancestors);
  a.status = p->status;
  a.batch = static_cast<int32_t>(p->batch);
  a.tokens = static_cast<int32_t>(p->tokens);
  constexpr int per = chia::kTreeThreads / 32;
  const int64_t ctas = (p->batch + per - 1) / per;
  return launched(chia::launch_after(chia::tree_tables_kernel, dim3(static_cast<unsigned>(ctas < sms ? ctas : sms)),
                                     chia::kTreeThreads, 0, static_cast<cudaStream_t>(stream), a));
}

int chia_verify_drafts(const chia_verify_params_t *p, void *stream) {
  if (p == nullptr || p->abi_version != CHIA_DRAFT_ABI_VERSION) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->dtype != CHIA_DTYPE_BF16 && p->dtype != CHIA_DTYPE_F16 && p->dtype != CHIA_DTYPE_F32)
    return CHIA_ERR_UNSUPPORTED;
  if (p->batch < 1 || p->batch > (1 << 24) || p->tokens < 0 || p->tokens > kI32 || p->vocab < 1 ||
      p->max_tokens < 1 || p->max_tokens > kI32 || p->target_stride < p->vocab ||
      (p->draft_probs && p->draft_stride < p->vocab) || !p->cu_q || !p->counts || !p->out_tokens || !p->path ||
      (p->tokens > 0 && (!p->target_probs || !p->node_tokens || !p->parents || !p->uniforms)))
    return CHIA_ERR_INVALID_ARGUMENT;
  constexpr int64_t most = static_cast<int64_t>(chia::kVerifyMostChunks) * chia::kVerifyChunk * chia::kVerifyCtas;
  static_assert(most == 1 << 22, "as chia_draft.h says");
  if (p->vocab > most) return CHIA_ERR_UNSUPPORTED;
  const unsigned size = p->dtype == CHIA_DTYPE_F32 ? 4 : 2;
  if (!aligned(p->target_probs, size) || !aligned(p->draft_probs, size) || !aligned(p->node_tokens, 4) ||
      !aligned(p->parents, 4) || !aligned(p->cu_q, 4) || !aligned(p->uniforms, 4) || !aligned(p->counts, 4) ||
      !aligned(p->out_tokens, 4) || !aligned(p->path, 4) || !aligned(p->status, 4))
    return CHIA_ERR_MISALIGNED;
  int sms = 0;
  const int rc = device_sms(sms);
  if (rc != CHIA_OK) return rc;
  chia::VerifyArgs a{};
  a.p = p->target_probs;
  a.q = p->draft_probs;
  a.p_st = p->target_stride;
  a.q_st = p->draft_stride;
  a.tokens = p->node_tokens;
  a.parents = p->parents;
  a.cu_q = p->cu_q;
  a.u = p->uniforms;
  a.counts = p->counts;
  a.out = p->out_tokens;
  a.path = p->path;
  a.status = p->status;
  a.batch = static_cast<int32_t>(p->batch);
  a.rows = static_cast<int32_t>(p->tokens);
  a.vocab = static_cast<int32_t>(p->vocab);
  a.most = static_cast<int32_t>(p->max_tokens);
  a.chunks = static_cast<int32_t>((p->vocab + chia::kVerifyChunk - 1) / chia::kVerifyChunk);
  const bool vec = aligned(p->target_probs, 4 * size) && p->target_stride % 4 == 0 &&
                   (!p->draft_probs || (aligned(p->draft_probs, 4 * size) && p->draft_stride % 4 == 0));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p->dtype == CHIA_DTYPE_BF16  ? launch_verify<0>(a, vec, sms, s)
         : p->dtype == CHIA_DTYPE_F16 ? launch_verify<1>(a, vec, sms, s)
                                      : launch_verify<2>(a, vec, sms, s);
}

int chia_cache_compact(const chia_compact_params_t *p, void *stream) {
  if (p == nullptr || p->abi_version < 1 || p->abi_version > CHIA_COMPACT_ABI_VERSION) return CHIA_ERR_INVALID_ARGUMENT;
  const int32_t *slots = p->abi_version > 1 ? p->slots : nullptr;  // (the field is not there before)
  if (slots != nullptr && p->tokens < 0) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->cache_dtype != CHIA_CACHE_E4M3 && p->cache_dtype != CHIA_CACHE_INT8) return CHIA_ERR_UNSUPPORTED;
  if ((p->head_dim != 64 && p->head_dim != 128) ||
      (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128))
    return CHIA_ERR_UNSUPPORTED;
  if (p->heads_kv < 1 || p->heads_kv > 65535 || p->batch < 1 || p->batch > (1 << 24) || p->max_tokens < 1 ||
      p->max_tokens > kI32 || p->num_pages < 1 || p->num_pages > kI32 / p->page_size || p->table_width < 1 ||
      p->table_width > kI32 / p->page_size || p->table_stride < p->table_width)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (!p->path || !p->counts || !p->cu_q || !p->seq_lens || !p->block_table || !p->k_cache || !p->v_cache ||
      !p->k_scale || !p->v_scale || !p->keep_lens || p->keep_lens == p->seq_lens || p->keep_lens == p->counts)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (!aligned(p->k_cache, 16) || !aligned(p->v_cache, 16) || !aligned(p->k_scale, 4) || !aligned(p->v_scale, 4) ||
      !aligned(p->path, 4) || !aligned(p->counts, 4) || !aligned(p->cu_q, 4) || !aligned(p->seq_lens, 4) ||
      !aligned(p->block_table, 4) || !aligned(p->keep_lens, 4) || !aligned(p->status, 4) || !aligned(slots, 4))
    return CHIA_ERR_MISALIGNED;
  const int64_t grid = p->batch * 2 * p->heads_kv;
  if (grid > kI32) return CHIA_ERR_UNSUPPORTED;
  int sms = 0;
  const int rc = device_sms(sms);
  if (rc != CHIA_OK) return rc;
  chia::CompactArgs a{};
  a.path = p->path;
  a.counts = p->counts;
  a.cu_q = p->cu_q;
  a.seq_lens = p->seq_lens;
  a.block_table = p->block_table;
  a.k_cache = static_cast<uint8_t *>(p->k_cache);
  a.v_cache = static_cast<uint8_t *>(p->v_cache);
  a.k_scale = p->k_scale;
  a.v_scale = p->v_scale;
  a.keep_lens = p->keep_lens;
  a.status = p->status;
  a.slots = slots;
  a.tokens = slots != nullptr ? p->tokens : 0;
  a.table_stride = p->table_stride;
  a.num_pages = p->num_pages;
  a.batch = static_cast<int32_t>(p->batch);
  a.most = static_cast<int32_t>(p->max_tokens);
  a.heads_kv = p->heads_kv;
  a.page = p->page_size;
  a.width = static_cast<int32_t>(p->table_width);
  auto run = [&](void (*kernel)(chia::CompactArgs)) {
    return launched(chia::launch_after(kernel, dim3(static_cast<unsigned>(grid)), chia::kCompactThreads, 0,
                                       static_cast<cudaStream_t>(stream), a));
  };
  const bool e4m3 = p->cache_dtype == CHIA_CACHE_E4M3;
  if (p->head_dim == 128)
    return e4m3 ? run(chia::cache_compact_kernel<128, chia::CACHE_E4M3>) : run(chia::cache_compact_kernel<128, chia::CACHE_INT8>);
  return e4m3 ? run(chia::cache_compact_kernel<64, chia::CACHE_E4M3>) : run(chia::cache_compact_kernel<64, chia::CACHE_INT8>);
}

}  // extern "C"
