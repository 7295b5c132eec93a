// paged_api.cu -- extern "C" entry points of the paged 8-bit K/V cache
// (include/chia_paged.h): argument checks, choice of the kernel, launch. No
// allocation, no synchronisation.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <mutex>

#include "../../include/chia_paged.h"
#include "cache_sm100.cuh"
#include "paged_split_sm100.cuh"
#include "paged_tiled_sm100.cuh"

namespace {

constexpr int64_t kI32 = 0x7fffffffLL;
constexpr uint64_t kDefaultTimeoutNs = 2000000000ull;  // 2 s a wait

bool aligned(const void *p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

bool page_ok(int64_t p) { return p == 16 || p == 32 || p == 64 || p == 128; }

// The current device's number of SMs; CHIA_ERR_NO_DEVICE where it is no sm_100.
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

// ---------------------------------------------------------------------- tables
int tables_args(const chia_tables_params_t *p, bool release, chia::TablesArgs &a) {
  if (p == nullptr || p->abi_version != CHIA_PAGED_ABI_VERSION) return CHIA_ERR_INVALID_ARGUMENT;
  if (!page_ok(p->page_size)) return CHIA_ERR_UNSUPPORTED;
  if (p->batch < 1 || p->batch > (1 << 24) || p->table_width < 1 || p->table_width > kI32 ||
      p->table_stride < p->table_width || p->ring_size < 1 || p->ring_size > kI32 ||
      p->max_tokens < 0 || p->max_tokens > kI32)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (!p->seq_lens || !p->new_lens || !p->block_table || !p->free_pages || !p->free_state ||
      !p->new_seq_lens || !p->new_free_state)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (!release && (!p->cu_q || (p->max_tokens > 0 && (!p->slots || !p->positions))))
    return CHIA_ERR_INVALID_ARGUMENT;
  // the kernels read them while they write the new ones
  if (p->new_seq_lens == p->seq_lens || p->new_free_state == p->free_state)
    return CHIA_ERR_INVALID_ARGUMENT;
  for (const void *q : {static_cast<const void *>(p->seq_lens), static_cast<const void *>(p->new_lens),
                        static_cast<const void *>(p->block_table),
                        static_cast<const void *>(p->free_pages),
                        static_cast<const void *>(p->free_state), static_cast<const void *>(p->slots),
                        static_cast<const void *>(p->positions), static_cast<const void *>(p->cu_q),
                        static_cast<const void *>(p->new_seq_lens),
                        static_cast<const void *>(p->new_free_state),
                        static_cast<const void *>(p->status)})
    if (!aligned(q, 4)) return CHIA_ERR_MISALIGNED;
  a.seq_lens = p->seq_lens;
  a.new_lens = p->new_lens;
  a.free_state = p->free_state;
  a.block_table = p->block_table;
  a.free_pages = p->free_pages;
  a.slots = p->slots;
  a.positions = p->positions;
  a.cu_q = p->cu_q;
  a.new_seq_lens = p->new_seq_lens;
  a.new_free_state = p->new_free_state;
  a.status = p->status;
  a.table_stride = p->table_stride;
  a.batch = static_cast<int32_t>(p->batch);
  a.width = static_cast<int32_t>(p->table_width);
  a.ring = static_cast<int32_t>(p->ring_size);
  a.max_tokens = static_cast<int32_t>(p->max_tokens);
  a.page = p->page_size;
  return CHIA_OK;
}

// CTAs of the tables' kernels: one for each kTablesThreads items, one wave at most.
int tables_grid(int64_t items, int sms) {
  const int64_t n = (items + chia::kTablesThreads - 1) / chia::kTablesThreads;
  return static_cast<int>(n < 1 ? 1 : n > sms ? sms : n);
}

template <bool TRIM>
int give_back(const chia_tables_params_t *p, void *stream) {
  chia::TablesArgs a{};
  int rc = tables_args(p, true, a), sms = 0;
  if (rc != CHIA_OK || (rc = device_sms(sms)) != CHIA_OK) return rc;
  return launched(chia::launch_after(chia::release_pages_kernel<TRIM>, dim3(tables_grid(p->ring_size, sms)),
                                     chia::kTablesThreads, 0, static_cast<cudaStream_t>(stream), a));
}

// ---------------------------------------------------------------------- append
int check_append(const chia_append_params_t *p) {
  if (p == nullptr || p->abi_version != CHIA_PAGED_ABI_VERSION) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->dtype != CHIA_DTYPE_BF16 && p->dtype != CHIA_DTYPE_F16) return CHIA_ERR_UNSUPPORTED;
  if (p->cache_dtype != CHIA_CACHE_E4M3 && p->cache_dtype != CHIA_CACHE_INT8)
    return CHIA_ERR_UNSUPPORTED;
  if ((p->head_dim != 64 && p->head_dim != 128) || !page_ok(p->page_size))
    return CHIA_ERR_UNSUPPORTED;
  if (p->heads_kv < 1 || p->heads_kv > 65535 || p->tokens < 0 || p->tokens > kI32 ||
      p->num_pages < 1 || p->num_pages > kI32 / p->page_size)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (p->tokens > 0 && (!p->k || !p->v || !p->slots)) return CHIA_ERR_INVALID_ARGUMENT;
  if (!p->k_cache || !p->v_cache || !p->k_scale || !p->v_scale) return CHIA_ERR_INVALID_ARGUMENT;
  if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->k_cache, 16) ||
      !aligned(p->v_cache, 16) || !aligned(p->slots, 4) || !aligned(p->k_scale, 4) ||
      !aligned(p->v_scale, 4) || !aligned(p->status, 4))
    return CHIA_ERR_MISALIGNED;
  for (const int64_t *s : {p->k_stride, p->v_stride})
    for (int d = 0; d < 2; ++d) {
      if (s[d] < 0) return CHIA_ERR_INVALID_ARGUMENT;
      if (s[d] % 8 != 0) return CHIA_ERR_MISALIGNED;
    }
  return CHIA_OK;
}

// Tokens that a CTA of the append looks at: a page's, or as many fewer as give
// every SM eight CTAs. 16 prompts of some 4,100 tokens: 43 us by pages, 590 by single
// tokens (every CTA then reads its neighbours' slots); 64 single tokens: 62 and 3.9.
template <int D, bool BF16, int CT>
int launch_append(const chia::AppendArgs &a, int sms, cudaStream_t s) {
  const int64_t kinds = 2ll * a.heads_kv;
  int window = a.page;
  while (window > 1 && (a.tokens + window - 1) / window * kinds < 8 * sms) window /= 2;
  const int64_t grid = (a.tokens + window - 1) / window * kinds;
  if (grid > kI32) return CHIA_ERR_UNSUPPORTED;
  const unsigned g = static_cast<unsigned>(grid);
  auto run = [&](void (*kernel)(chia::AppendArgs, int)) {
    return launched(chia::launch_after(kernel, dim3(g), 128, 0, s, a, window));
  };
  switch (a.page * D / 1024) {
    case 1: return run(chia::cache_append_kernel<64, BF16, CT, 1>);
    case 2: return run(chia::cache_append_kernel<D, BF16, CT, 2>);
    case 4: return run(chia::cache_append_kernel<D, BF16, CT, 4>);
    case 8: return run(chia::cache_append_kernel<D, BF16, CT, 8>);
    default: return run(chia::cache_append_kernel<128, BF16, CT, 16>);
  }
}

// ------------------------------------------------------------------- attention
int check_paged(const chia_paged_params_t *p) {
  if (p == nullptr || p->abi_version != CHIA_PAGED_ABI_VERSION) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->dtype != CHIA_DTYPE_BF16 && p->dtype != CHIA_DTYPE_F16) return CHIA_ERR_UNSUPPORTED;
  if (p->cache_dtype != CHIA_CACHE_E4M3 && p->cache_dtype != CHIA_CACHE_INT8)
    return CHIA_ERR_UNSUPPORTED;
  if ((p->head_dim != 64 && p->head_dim != 128) || !page_ok(p->page_size))
    return CHIA_ERR_UNSUPPORTED;
  if (p->norm < CHIA_NORM_SOFTMAX || p->norm > CHIA_NORM_RELU) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->mod < CHIA_MOD_NONE || p->mod > CHIA_MOD_TEMP) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->norm != CHIA_NORM_SOFTMAX && p->mod != CHIA_MOD_NONE) return CHIA_ERR_UNSUPPORTED;
  if (p->heads < 1 || p->heads > (1 << 20) || p->heads_kv < 1 || p->heads % p->heads_kv != 0 ||
      p->max_q < 1 || p->batch < 1 || p->batch > (1 << 24) || p->tokens < 0 || p->tokens > kI32 ||
      p->num_pages < 1 || p->num_pages > kI32 / p->page_size || p->table_width < 1 ||
      p->table_width > kI32 / p->page_size || p->table_stride < p->table_width)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (p->cu_q == nullptr && p->tokens % p->batch != 0) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->num_pages * p->heads_kv > kI32) return CHIA_ERR_UNSUPPORTED;
  if (p->win_left < -1 || p->win_right < -1 || p->block < 0 || p->prefix < 0 || p->dilation < 1)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (p->tokens > 0 && (!p->q || !p->o)) return CHIA_ERR_INVALID_ARGUMENT;
  if (!p->k_cache || !p->v_cache || !p->k_scale || !p->v_scale || !p->block_table || !p->seq_lens)
    return CHIA_ERR_INVALID_ARGUMENT;
  if ((p->mod == CHIA_MOD_ALIBI || p->mod == CHIA_MOD_TEMP) && p->head_param == nullptr)
    return CHIA_ERR_INVALID_ARGUMENT;
  if (p->mod == CHIA_MOD_SOFTCAP && !(p->softcap > 0.f)) return CHIA_ERR_INVALID_ARGUMENT;
  if (!std::isfinite(p->scale) || !std::isfinite(p->sig_bias) || !std::isfinite(p->out_scale))
    return CHIA_ERR_INVALID_ARGUMENT;
  if (!aligned(p->q, 16) || !aligned(p->o, 16) || !aligned(p->k_cache, 16) ||
      !aligned(p->v_cache, 16) || !aligned(p->k_scale, 4) || !aligned(p->v_scale, 4) ||
      !aligned(p->block_table, 4) || !aligned(p->seq_lens, 4) || !aligned(p->cu_q, 4) ||
      !aligned(p->lse, 4) || !aligned(p->head_param, 4) || !aligned(p->status, 4))
    return CHIA_ERR_MISALIGNED;
  for (const int64_t *s : {p->q_stride, p->o_stride})
    for (int d = 0; d < 2; ++d) {
      if (s[d] < 0) return CHIA_ERR_INVALID_ARGUMENT;
      if (s[d] % 8 != 0) return CHIA_ERR_MISALIGNED;
    }
  return CHIA_OK;
}

int kind_of(const chia_paged_params_t *p) {
  if (p->norm == CHIA_NORM_SIGMOID) return chia::KIND_SIGMOID;
  if (p->norm == CHIA_NORM_RELU) return chia::KIND_RELU;
  switch (p->mod) {
    case CHIA_MOD_SOFTCAP: return chia::KIND_SOFTCAP;
    case CHIA_MOD_ALIBI: return chia::KIND_ALIBI;
    default: return chia::KIND_SOFTMAX;  // NONE and TEMP
  }
}

// Which kernel, and the workspace: the tickets, then the parts of two units a
// CTA and (split kernel) of one a worker.
constexpr int64_t kTicketBytes = 4096;
// Rows of a K/V head (queries x heads of a group) from which the tiled kernel is the
// faster one. Split and tiled, us, D 128, 8 K/V heads: 8 requests x 4096 keys, 48 rows 53, 57,
// 64 rows 65, 58, 256 rows 206, 69; 32 x 1024, 48 rows 63, 63, 64 rows 71, 63.
constexpr int64_t kTiledRows = 56;
struct SplitPlan {
  bool tiled;
  // split kernel: eights of rows of a unit. Two from 9 rows on: 64 requests x 8192 keys, 16
  // rows 208 us, and 363 in units of 8, which read the keys twice (24 x 1500, 20 rows: 35 and 27).
  int tiles;
  int rows;   // of a unit
  int grid;   // one CTA an SM
  int64_t off_ml, off_cuts, bytes;
};
int split_plan(const chia_paged_params_t *p, int sms, SplitPlan &pl) {
  const int64_t group = p->heads / p->heads_kv;
  pl.tiled = p->max_q * group >= kTiledRows;
  pl.tiles = p->max_q * group <= 8 ? 1 : 2;
  pl.rows = pl.tiled ? chia::TiledConfig<128>::ROWS : 8 * pl.tiles;
  pl.grid = sms;
  // the line of tiles is counted in 32 bits
  const int tk = pl.tiled ? 64 : 32;
  const double line = static_cast<double>(p->heads_kv) * (p->tokens * group / pl.rows + p->batch + 1) *
                      (p->table_width * p->page_size / tk + 2 + chia::kUnitCost);
  if (pl.grid * 4 > kTicketBytes || p->tokens * p->heads > kI32 ||
      p->tokens * group * group > 2 * kI32 || line > kI32)
    return CHIA_ERR_UNSUPPORTED;
  const int64_t slots = (2 + (pl.tiled ? 0 : chia::kSplitWarps)) * static_cast<int64_t>(pl.grid) * pl.rows;
  pl.off_ml = kTicketBytes + slots * p->head_dim * 4;
  pl.off_cuts = (pl.off_ml + slots * 8 + 255) / 256 * 256;
  pl.bytes = pl.off_cuts + (pl.tiled ? (pl.grid * sizeof(chia::CutUnit) + 255) / 256 * 256 : 0);
  return CHIA_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault,
                                         &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// A cache as (head_dim, page_size, pages * heads) bytes; a box is `rows` tokens
// of one page and head, swizzled over their own width or as they are.
bool encode_cache(CUtensorMap *map, const void *base, const chia_paged_params_t *p, int rows,
                  bool swizzle) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t D = p->head_dim, P = p->page_size;
  const cuuint64_t dims[3] = {D, P, static_cast<cuuint64_t>(p->num_pages) * p->heads_kv};
  const cuuint64_t strides[2] = {D, P * D};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(D), static_cast<cuuint32_t>(rows), 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(base), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE,
            !swizzle ? CU_TENSOR_MAP_SWIZZLE_NONE
            : D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// (no position is that large)
int32_t clamp32(int64_t v) { return static_cast<int32_t>(v > kI32 ? kI32 : v); }

// FN<D, BF16, CT>(...) for the call's types.
#define CHIA_BY_TYPE(p, FN, ...)                                                          \
  ((p)->head_dim == 128                                                                   \
       ? ((p)->dtype == CHIA_DTYPE_BF16                                                   \
              ? ((p)->cache_dtype == CHIA_CACHE_E4M3 ? FN<128, true, 0>(__VA_ARGS__)      \
                                                     : FN<128, true, 1>(__VA_ARGS__))     \
              : ((p)->cache_dtype == CHIA_CACHE_E4M3 ? FN<128, false, 0>(__VA_ARGS__)     \
                                                     : FN<128, false, 1>(__VA_ARGS__)))   \
       : ((p)->dtype == CHIA_DTYPE_BF16                                                   \
              ? ((p)->cache_dtype == CHIA_CACHE_E4M3 ? FN<64, true, 0>(__VA_ARGS__)       \
                                                     : FN<64, true, 1>(__VA_ARGS__))      \
              : ((p)->cache_dtype == CHIA_CACHE_E4M3 ? FN<64, false, 0>(__VA_ARGS__)      \
                                                     : FN<64, false, 1>(__VA_ARGS__))))

}  // namespace

extern "C" {

int chia_page_tables(const chia_tables_params_t *p, void *stream) {
  chia::TablesArgs a{};
  int rc = tables_args(p, false, a), sms = 0;
  if (rc != CHIA_OK || (rc = device_sms(sms)) != CHIA_OK) return rc;
  return launched(chia::launch_after(chia::page_tables_kernel, dim3(tables_grid(p->max_tokens, sms)), chia::kTablesThreads, 0,
                                     static_cast<cudaStream_t>(stream), a));
}

int chia_release_pages(const chia_tables_params_t *p, void *stream) { return give_back<false>(p, stream); }

int chia_trim_pages(const chia_tables_params_t *p, void *stream) { return give_back<true>(p, stream); }

int chia_cache_append(const chia_append_params_t *p, void *stream) {
  int rc = check_append(p), sms = 0;
  if (rc != CHIA_OK || (rc = device_sms(sms)) != CHIA_OK) return rc;
  if (p->tokens == 0) return CHIA_OK;
  chia::AppendArgs a{};
  a.k = p->k;
  a.v = p->v;
  a.k_st = p->k_stride[0], a.k_sh = p->k_stride[1];
  a.v_st = p->v_stride[0], a.v_sh = p->v_stride[1];
  a.slots = p->slots;
  a.k_cache = static_cast<uint8_t *>(p->k_cache);
  a.v_cache = static_cast<uint8_t *>(p->v_cache);
  a.k_scale = p->k_scale;
  a.v_scale = p->v_scale;
  a.status = p->status;
  a.tokens = static_cast<int32_t>(p->tokens);
  a.heads_kv = p->heads_kv;
  a.page = p->page_size;
  a.num_pages = p->num_pages;
  return CHIA_BY_TYPE(p, launch_append, a, sms, static_cast<cudaStream_t>(stream));
}

int64_t chia_paged_attn_workspace_bytes(const chia_paged_params_t *p) {
  if (check_paged(p) != CHIA_OK) return -1;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1)
    sms = 148;  // host-only callers (no GPU): size for a B200
  SplitPlan pl;
  return split_plan(p, sms, pl) == CHIA_OK ? pl.bytes : -1;
}

int chia_paged_attn(const chia_paged_params_t *p, void *stream) {
  int rc = check_paged(p), sms = 0, dev = 0;
  if (rc != CHIA_OK) return rc;
  if (p->workspace == nullptr) return CHIA_ERR_INVALID_ARGUMENT;
  if (!aligned(p->workspace, 256)) return CHIA_ERR_MISALIGNED;
  // (a workspace for no device is too small for any)
  if (p->workspace_bytes <= kTicketBytes) return CHIA_ERR_INVALID_ARGUMENT;
  if ((rc = device_sms(sms)) != CHIA_OK) return rc;
  if (cudaGetDevice(&dev) != cudaSuccess) return CHIA_ERR_NO_DEVICE;
  SplitPlan pl;
  if ((rc = split_plan(p, sms, pl)) != CHIA_OK) return rc;
  if (p->workspace_bytes < pl.bytes) return CHIA_ERR_INVALID_ARGUMENT;
  if (p->tokens == 0) return CHIA_OK;
  CUtensorMap mk, mv;
  const int most = pl.tiled ? 64 : 32, box = p->page_size < most ? p->page_size : most;
  if (!encode_cache(&mk, p->k_cache, p, box, !pl.tiled) ||
      !encode_cache(&mv, p->v_cache, p, box, !pl.tiled))
    return CHIA_ERR_LAUNCH;
  chia::PagedArgs a{};
  a.q = p->q;
  a.o = p->o;
  a.q_st = p->q_stride[0], a.q_sh = p->q_stride[1];
  a.o_st = p->o_stride[0], a.o_sh = p->o_stride[1];
  a.k_scale = p->k_scale;
  a.v_scale = p->v_scale;
  a.block_table = p->block_table;
  a.seq_lens = p->seq_lens;
  a.cu_q = p->cu_q;
  a.table_stride = p->table_stride;
  a.lse = p->norm == CHIA_NORM_SOFTMAX ? p->lse : nullptr;
  a.head_param = (p->mod == CHIA_MOD_ALIBI || p->mod == CHIA_MOD_TEMP) ? p->head_param : nullptr;
  a.left = clamp32(p->win_left);
  a.right = clamp32(p->win_right);
  a.block = clamp32(p->block);
  a.prefix = clamp32(p->prefix);
  a.dil = clamp32(p->dilation);
  a.score_scale = p->scale;
  a.softcap = p->softcap;
  a.sig_bias = p->sig_bias;
  a.out_scale = p->out_scale;
  a.heads = p->heads;
  a.heads_kv = p->heads_kv;
  a.group = p->heads / p->heads_kv;
  a.group_magic = a.group == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + a.group - 1) / a.group);
  a.tokens = static_cast<int32_t>(p->tokens);
  a.page = p->page_size;
  a.width = static_cast<int32_t>(p->table_width);
  a.num_pages = static_cast<int32_t>(p->num_pages);
  a.q_each = static_cast<int32_t>(p->tokens / p->batch);
  a.bf16 = p->dtype == CHIA_DTYPE_BF16;
  a.status = p->status;
  uint8_t *ws = static_cast<uint8_t *>(p->workspace);
  a.tickets = reinterpret_cast<int32_t *>(ws);
  a.part_o = reinterpret_cast<float *>(ws + kTicketBytes);
  a.part_ml = reinterpret_cast<float *>(ws + pl.off_ml);
  a.timeout_ns = p->wait_limit_ns > 0 ? p->wait_limit_ns : kDefaultTimeoutNs;
  a.drain_ns = kDefaultTimeoutNs;
  const int kind = kind_of(p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  for (int64_t b = 0; b < p->batch; b += chia::kLineBatch) {
    const int64_t n = p->batch - b < chia::kLineBatch ? p->batch - b : chia::kLineBatch;
    a.batch = static_cast<int32_t>(n);
    a.seq_lens = p->seq_lens + b;
    a.cu_q = p->cu_q != nullptr ? p->cu_q + b : nullptr;
    a.token0 = static_cast<int32_t>(b * a.q_each);
    a.block_table = p->block_table + b * p->table_stride;
    const uint8_t *v8 = static_cast<const uint8_t *>(p->v_cache);
#define CHIA_LAUNCH(D, CT)                                                                   \
  (pl.tiled ? chia::launch_tiled<D, CT>(mk, mv, a, v8, ws + pl.off_cuts, kind, pl.grid, dev, s)                \
            : chia::launch_split<D, CT>(mk, mv, a, kind, pl.tiles, pl.grid, dev, s))
    const bool e4m3 = p->cache_dtype == CHIA_CACHE_E4M3;
    const cudaError_t e =
        p->head_dim == 128
            ? (e4m3 ? CHIA_LAUNCH(128, chia::CACHE_E4M3) : CHIA_LAUNCH(128, chia::CACHE_INT8))
            : (e4m3 ? CHIA_LAUNCH(64, chia::CACHE_E4M3) : CHIA_LAUNCH(64, chia::CACHE_INT8));
#undef CHIA_LAUNCH
    if (e != cudaSuccess) return CHIA_ERR_LAUNCH;
  }
  return CHIA_OK;
}

}  // extern "C"
