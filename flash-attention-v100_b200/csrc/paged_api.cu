// C-ABI launch layer of the paged key/value cache (declared in include/fmha_b200.h): validate plain-pointer
// parameters, launch, return a status.  Nothing here allocates device memory or synchronises.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/fmha_b200.h"
#include "cache_kernels.cuh"
#include "host_common.cuh"
#include "paged_simple_kernel.cuh"

namespace {

// sizes and type that the three entry points share; seqlen is checked by each
int check_sizes(int batch, int heads, int head_dim, int dtype) {
  if (dtype != FMHA_DTYPE_FP16 && dtype != FMHA_DTYPE_BF16) return FMHA_ERR_BAD_DTYPE;
  if (head_dim != 64 && head_dim != 96 && head_dim != 128) return FMHA_ERR_BAD_HEAD_DIM;
  if (batch < 0 || heads <= 0) return FMHA_ERR_BAD_SHAPE;
  return FMHA_OK;
}

// strides of a pool in elements: multiples of 16 bytes where they are used
int check_pool_strides(const FmhaStrides& s, int pages, int rows, int heads, int unit) {
  if ((rows > 1 && (s.row % unit != 0 || s.row <= 0)) || (heads > 1 && (s.head % unit != 0 || s.head <= 0)) ||
      (pages > 1 && (s.batch % unit != 0 || s.batch <= 0)))
    return FMHA_ERR_BAD_STRIDE;
  return FMHA_OK;
}

int check_cache(const FmhaPagedCache& c, int heads) {
  if (c.k == nullptr || c.v == nullptr || c.block_table == nullptr) return FMHA_ERR_NULL_POINTER;
  if (c.format != FMHA_CACHE_16BIT && c.format != FMHA_CACHE_E4M3) return FMHA_ERR_BAD_DTYPE;
  const bool e4m3 = c.format == FMHA_CACHE_E4M3;
  if (e4m3 && (c.k_scale == nullptr || c.v_scale == nullptr)) return FMHA_ERR_NULL_POINTER;
  if (c.num_pages <= 0 || c.page_size <= 0 || c.page_size % 16 != 0 || c.max_pages <= 0) return FMHA_ERR_BAD_SHAPE;
  if ((long long)c.max_pages * c.page_size > (1ll << 30)) return FMHA_ERR_TOO_LARGE;
  if (!aligned16(c.k) || !aligned16(c.v)) return FMHA_ERR_BAD_ALIGNMENT;
  int rc;
  const int unit = e4m3 ? 16 : 8;
  if ((rc = check_pool_strides(c.k_strides, c.num_pages, c.page_size, heads, unit))) return rc;
  if ((rc = check_pool_strides(c.v_strides, c.num_pages, c.page_size, heads, unit))) return rc;
  if (c.block_table_stride < 0) return FMHA_ERR_BAD_STRIDE;
  if (e4m3 && ((rc = check_pool_strides(c.k_scale_strides, c.num_pages, c.page_size, heads, 1)) ||
               (rc = check_pool_strides(c.v_scale_strides, c.num_pages, c.page_size, heads, 1))))
    return rc;
  return FMHA_OK;
}

fmha::PagedCache device_cache(const FmhaPagedCache& c) {
  const int bytes = c.format == FMHA_CACHE_E4M3 ? 1 : 2;
  auto pool = [&](void* rows, uint8_t* scales, const FmhaStrides& s, const FmhaStrides& t) {
    return fmha::PagePool{static_cast<uint8_t*>(rows), scales,  s.batch * bytes, s.row * bytes,
                          s.head * bytes,              t.batch, t.row,           t.head};
  };
  return fmha::PagedCache{pool(c.k, c.k_scale, c.k_strides, c.k_scale_strides),
                          pool(c.v, c.v_scale, c.v_strides, c.v_scale_strides),
                          c.block_table,
                          c.block_table_stride,
                          c.num_pages,
                          c.page_size,
                          c.max_pages};
}

// DR, kBf16 and kE4m3 for a kernel of the cache
#define FMHA_DISPATCH_CACHE_FORMAT(dtype, format, ...)                 \
  if ((dtype) == FMHA_DTYPE_BF16) {                                    \
    constexpr bool kBf16 = true;                                       \
    if ((format) == FMHA_CACHE_E4M3) {                                 \
      constexpr bool kE4m3 = true;                                     \
      __VA_ARGS__                                                      \
    } else {                                                           \
      constexpr bool kE4m3 = false;                                    \
      __VA_ARGS__                                                      \
    }                                                                  \
  } else {                                                             \
    constexpr bool kBf16 = false;                                      \
    if ((format) == FMHA_CACHE_E4M3) {                                 \
      constexpr bool kE4m3 = true;                                     \
      __VA_ARGS__                                                      \
    } else {                                                           \
      constexpr bool kE4m3 = false;                                    \
      __VA_ARGS__                                                      \
    }                                                                  \
  }
#define FMHA_DISPATCH_CACHE(head_dim, dtype, format, ...)              \
  if ((head_dim) == 128) {                                             \
    constexpr int DR = 128;                                            \
    FMHA_DISPATCH_CACHE_FORMAT(dtype, format, __VA_ARGS__)             \
  } else if ((head_dim) == 96) {                                       \
    constexpr int DR = 96;                                             \
    FMHA_DISPATCH_CACHE_FORMAT(dtype, format, __VA_ARGS__)             \
  } else {                                                             \
    constexpr int DR = 64;                                             \
    FMHA_DISPATCH_CACHE_FORMAT(dtype, format, __VA_ARGS__)             \
  }

// (a 32-bit grid of blocks of 256 threads, 8 or 16 of them a row)
constexpr long long kMaxCacheRows = 1ll << 34;

}  // namespace

extern "C" {

int fmha_cache_write(const FmhaCacheWriteParams* p, void* stream) {
  if (p == nullptr) return FMHA_ERR_NULL_POINTER;
  int rc = check_sizes(p->batch, p->heads, p->head_dim, p->dtype);
  if (rc) return rc;
  if (p->seqlen < 0) return FMHA_ERR_BAD_SHAPE;
  if ((rc = check_cache(p->cache, p->heads))) return rc;
  const long long rows = (long long)p->batch * p->seqlen * p->heads;
  if (rows == 0) return FMHA_OK;
  if (rows > kMaxCacheRows) return FMHA_ERR_TOO_LARGE;
  if (p->k == nullptr || p->v == nullptr || p->seqlens == nullptr) return FMHA_ERR_NULL_POINTER;
  if (!aligned16(p->k) || !aligned16(p->v)) return FMHA_ERR_BAD_ALIGNMENT;
  if ((rc = check_strides(p->k_strides, p->seqlen, p->heads, p->batch))) return rc;
  if ((rc = check_strides(p->v_strides, p->seqlen, p->heads, p->batch))) return rc;
  fmha::CacheWriteArgs a;
  a.cache = device_cache(p->cache);
  a.k = static_cast<const uint8_t*>(p->k);
  a.v = static_cast<const uint8_t*>(p->v);
  a.k_batch = p->k_strides.batch * 2, a.k_row = p->k_strides.row * 2, a.k_head = p->k_strides.head * 2;
  a.v_batch = p->v_strides.batch * 2, a.v_row = p->v_strides.row * 2, a.v_head = p->v_strides.head * 2;
  a.seqlens = p->seqlens;
  a.seqused = p->seqused;
  a.heads = p->heads;
  a.seqlen = p->seqlen;
  a.rows = rows;
  const int per_block = 256 / (p->head_dim == 64 ? 8 : 16);
  const unsigned grid = (unsigned)((rows + per_block - 1) / per_block);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FMHA_DISPATCH_CACHE(p->head_dim, p->dtype, p->cache.format,
                      fmha::cache_write_kernel<DR, kBf16, kE4m3><<<grid, 256, 0, s>>>(a);)
  return cudaGetLastError() == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}

int fmha_cache_read(const FmhaCacheReadParams* p, void* stream) {
  if (p == nullptr) return FMHA_ERR_NULL_POINTER;
  int rc = check_sizes(p->batch, p->heads, p->head_dim, p->dtype);
  if (rc) return rc;
  if (p->seqlen < 0) return FMHA_ERR_BAD_SHAPE;
  if ((rc = check_cache(p->cache, p->heads))) return rc;
  const long long rows = (long long)p->batch * p->seqlen * p->heads;
  if (rows == 0) return FMHA_OK;
  if (rows > kMaxCacheRows) return FMHA_ERR_TOO_LARGE;
  if (p->k == nullptr || p->v == nullptr || p->seqused_k == nullptr) return FMHA_ERR_NULL_POINTER;
  if (!aligned16(p->k) || !aligned16(p->v)) return FMHA_ERR_BAD_ALIGNMENT;
  if ((rc = check_strides(p->k_strides, p->seqlen, p->heads, p->batch))) return rc;
  if ((rc = check_strides(p->v_strides, p->seqlen, p->heads, p->batch))) return rc;
  fmha::CacheReadArgs a;
  a.cache = device_cache(p->cache);
  a.k = static_cast<uint8_t*>(p->k);
  a.v = static_cast<uint8_t*>(p->v);
  a.k_batch = p->k_strides.batch * 2, a.k_row = p->k_strides.row * 2, a.k_head = p->k_strides.head * 2;
  a.v_batch = p->v_strides.batch * 2, a.v_row = p->v_strides.row * 2, a.v_head = p->v_strides.head * 2;
  a.seqused_k = p->seqused_k;
  a.heads = p->heads;
  a.seqlen = p->seqlen;
  a.rows = rows;
  const unsigned grid = (unsigned)((rows * (p->head_dim / 8) + 255) / 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FMHA_DISPATCH_CACHE(p->head_dim, p->dtype, p->cache.format,
                      fmha::cache_read_kernel<DR, kBf16, kE4m3><<<grid, 256, 0, s>>>(a);)
  return cudaGetLastError() == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}

size_t fmha_paged_fwd_workspace_bytes(const FmhaPagedFwdParams* p) {
  (void)p;
  return 0;
}

int fmha_paged_fwd(const FmhaPagedFwdParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (p == nullptr) return FMHA_ERR_NULL_POINTER;
  int rc = check_sizes(p->batch, p->heads_k, p->head_dim, p->dtype);
  if (rc) return rc;
  if (p->heads_q <= 0 || p->heads_q % p->heads_k != 0 || p->heads_q / p->heads_k > 128 || p->seqlen_q < 0 ||
      !std::isfinite(p->scale) || p->scale == 0.f)
    return FMHA_ERR_BAD_SHAPE;
  if ((rc = check_cache(p->cache, p->heads_k))) return rc;
  if (p->batch == 0 || p->seqlen_q == 0) return FMHA_OK;
  if ((long long)p->seqlen_q * p->heads_q >= (1ll << 31) ||
      (long long)p->batch * p->heads_q * (p->seqlen_q / 128 + 2ll) >= (1ll << 31)) return FMHA_ERR_TOO_LARGE;
  if (p->q == nullptr || p->o == nullptr || p->lse == nullptr || p->seqused_k == nullptr) return FMHA_ERR_NULL_POINTER;
  if (!aligned16(p->q) || !aligned16(p->o) || !aligned16(workspace)) return FMHA_ERR_BAD_ALIGNMENT;
  if ((rc = check_strides(p->q_strides, p->seqlen_q, p->heads_q, p->batch))) return rc;
  if ((rc = check_strides(p->o_strides, p->seqlen_q, p->heads_q, p->batch))) return rc;
  (void)workspace_bytes;
  fmha::PagedSimpleArgs a;
  a.cache = device_cache(p->cache);
  a.q = static_cast<const uint8_t*>(p->q);
  a.o = static_cast<uint8_t*>(p->o);
  a.lse = p->lse;
  a.q_batch = p->q_strides.batch * 2, a.q_row = p->q_strides.row * 2, a.q_head = p->q_strides.head * 2;
  a.o_batch = p->o_strides.batch * 2, a.o_row = p->o_strides.row * 2, a.o_head = p->o_strides.head * 2;
  a.seqused_k = p->seqused_k;
  a.seqused_q = p->seqused_q;
  a.heads_q = p->heads_q;
  a.group = p->heads_q / p->heads_k;
  a.seqlen_q = p->seqlen_q;
  a.causal = p->causal != 0;
  a.scale = p->scale;
  a.rows = (long long)p->batch * p->seqlen_q * p->heads_q;
  const unsigned grid = (unsigned)((a.rows + 3) / 4);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FMHA_DISPATCH_CACHE(p->head_dim, p->dtype, p->cache.format,
                      fmha::paged_simple_kernel<DR, kBf16, kE4m3><<<grid, 128, 0, s>>>(a);)
  return cudaGetLastError() == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}

}  // extern "C"
