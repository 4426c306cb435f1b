// C-ABI launch layer of the paged key/value cache (declared in include/fmha_b200.h): validate plain-pointer
// parameters, launch, return a status.  Nothing here allocates device memory or synchronises.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <numeric>
#include <type_traits>

#include "../../include/fmha_b200.h"
#include "cache_kernels.cuh"
#include "host_common.cuh"
#include "paged_few_kernel.cuh"
#include "paged_many_kernel.cuh"

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
  if ((long long)c.max_pages * c.page_size >= (1ll << 30)) return FMHA_ERR_TOO_LARGE;
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
  const unsigned unit = (unsigned)c.page_size / 16;
  unsigned l = 0;
  while ((1u << l) < unit) ++l;
  return fmha::PagedCache{pool(c.k, c.k_scale, c.k_strides, c.k_scale_strides),
                          pool(c.v, c.v_scale, c.v_strides, c.v_scale_strides),
                          c.block_table,
                          c.block_table_stride,
                          c.num_pages,
                          c.page_size,
                          c.max_pages,
                          (unsigned)((1ull << (26 + l)) / unit + 1),
                          26 + l};
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

// A pool as a 4-D map (D, page_size, H, num_pages), 128-byte swizzle, zeros outside; box 64 x box_rows x 1 x 1 of 16-bit
// elements, 128 x box_rows x 1 x 1 of codes
int make_pool_map(CUtensorMap* map, const void* base, const FmhaPagedCache& c, const FmhaStrides& s, int heads, int D,
                  int box_rows, bool bf16) {
  EncodeTiledFn encode = get_encode_fn();
  if (encode == nullptr) return FMHA_ERR_NO_DEVICE;
  const bool codes = c.format == FMHA_CACHE_E4M3;
  // a stride of a size-1 dimension is never used for addressing; make it well-formed
  const int64_t row = s.row, head = heads > 1 ? s.head : (D + 15) / 16 * 16;
  const int64_t page = c.num_pages > 1 ? s.batch : row * c.page_size;
  const cuuint64_t unit = codes ? 1 : 2;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)c.page_size, (cuuint64_t)heads, (cuuint64_t)c.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)row * unit, (cuuint64_t)head * unit, (cuuint64_t)page * unit};
  const cuuint32_t box[4] = {codes ? 128u : 64u, (cuuint32_t)box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
  // What a miss brings into the L2 is no more than a row has: the row behind it is another head's, which another block reads
  // at another time.
  const CUtensorMapL2promotion promotion = D * unit >= 256   ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                                           : D * unit >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                                             : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
  const CUresult r = encode(map,
                            codes  ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                            : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FMHA_OK : FMHA_ERR_TENSOR_MAP;
}

// Rows of one cache head's queries, (Z, N, H, D) as a 4-D map (D, H, N, Z), box 64 x heads x tokens x 1: the box's rows
// are tokens with a cache head's query heads inside
int make_rows_map(CUtensorMap* map, const void* base, int Z, int N, int H, int D, const FmhaStrides& s, int heads, int tokens,
                  bool bf16) {
  EncodeTiledFn encode = get_encode_fn();
  if (encode == nullptr) return FMHA_ERR_NO_DEVICE;
  const int64_t head = H > 1 ? s.head : D, row = N > 1 ? s.row : head * H;
  const int64_t batch = Z > 1 ? s.batch : row * N;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)N, (cuuint64_t)Z};
  const cuuint64_t strides[3] = {(cuuint64_t)head * 2, (cuuint64_t)row * 2, (cuuint64_t)batch * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)heads, (cuuint32_t)tokens, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FMHA_OK : FMHA_ERR_TENSOR_MAP;
}

// sizes of an attention call, which the size query and the call itself have to agree on
int check_paged_sizes(const FmhaPagedFwdParams* p) {
  if (const int rc = check_sizes(p->batch, p->heads_k, p->head_dim, p->dtype)) return rc;
  if (p->heads_q <= 0 || p->heads_q % p->heads_k != 0 || p->heads_q / p->heads_k > 128 || p->seqlen_q < 0)
    return FMHA_ERR_BAD_SHAPE;
  return FMHA_OK;
}
// items are counted in 32 bits, and so are the blocks that join them (eight rows each)
int check_paged_limits(const FmhaPagedFwdParams* p) {
  if ((long long)p->seqlen_q * p->heads_q >= (1ll << 31) ||
      (double)p->batch * p->heads_q * (p->seqlen_q / 128 + 2.0) >= 2147483648.0 ||
      (double)p->batch * p->heads_q * (p->seqlen_q + 256.0) >= 8 * 2147483648.0)
    return FMHA_ERR_TOO_LARGE;
  return FMHA_OK;
}

// How a call is cut (paged_work.cuh) and what that takes.
struct PagedPlan {
  int kernel_rows;       // rows of an item that the kernel has room for
  int tokens_per_block;  // new tokens of an item
  int rows_per_tile;     // rows in use of each of
  int tiles;             // its row tiles
  int blocks_per_entry;
  int min_share;
  int blocks;            // of the grid
  size_t part_bytes, lse_bytes, item_bytes;
  size_t bytes() const { return part_bytes + lse_bytes + item_bytes; }
};

// Rows (new tokens times query heads of a cache head) of up to 16, 32, 48 or 64 run the kernel of few rows, more the one of
// many.  us, on the GPU alone: 64 rows over 16384 keys, one entry of 8 heads, few 31.6 / many 34.4; 64 over 8192, 32 entries,
// 160 / 197; 40 rows of 8-bit caches of 8192, 8 entries of 4 heads, by 48 / 64 / many 33.6 / 37.3 / 46.2.
// The least share of a block: a tile, because a piece more costs less than a tile more on a block's way: with 1 / 2 / 4 / 8
// tiles, one row group of 8 heads over 512 keys 9.9 / 10.6 / 12.2 / 15.5, over 4096 keys 12.2 / 12.2 / 13.1 / 15.7.  Two with many
// rows, whose pieces leave 256 rows to be joined: 512 rows over 2048 keys, 8 heads, with 2 / 4 / 8 24.2 / 30.3 / 42.3.
PagedPlan plan_paged(const FmhaPagedFwdParams* p, int sms) {
  PagedPlan plan = {};
  const int group = p->heads_q / p->heads_k;
  const long long rows = (long long)p->seqlen_q * group;
  if (rows <= 64) {
    plan.kernel_rows = (int)(rows + 15) / 16 * 16;
    plan.tokens_per_block = p->seqlen_q;
    plan.rows_per_tile = (int)rows;
    plan.tiles = 1;
    plan.min_share = 1;
  } else {
    plan.kernel_rows = 256;
    plan.tokens_per_block = 128 / group * 2;
    plan.rows_per_tile = 128 / group * group;
    plan.tiles = 2;
    plan.min_share = 2;
  }
  plan.blocks_per_entry = (int)(((long long)p->seqlen_q + plan.tokens_per_block - 1) / plan.tokens_per_block);
  plan.blocks = sms;
  const size_t items = (size_t)p->batch * plan.blocks_per_entry * p->heads_k;
  plan.part_bytes = (size_t)2 * plan.blocks * plan.kernel_rows * p->head_dim * sizeof(float);
  plan.lse_bytes = ((size_t)2 * plan.blocks * plan.kernel_rows * sizeof(float) + 255) / 256 * 256;
  plan.item_bytes = items * sizeof(int2);
  return plan;
}

fmha::PagedParams kernel_params(const FmhaPagedFwdParams* p, const PagedPlan& plan, void* workspace) {
  fmha::PagedParams a;
  a.cache = device_cache(p->cache);
  a.seqused_k = p->seqused_k;
  a.seqused_q = p->seqused_q;
  a.batch = p->batch;
  a.heads_k = p->heads_k;
  a.group = p->heads_q / p->heads_k;
  a.group_mul = 65536u / a.group + 1;
  a.seqlen_q = p->seqlen_q;
  a.causal = p->causal ? 1 : 0;
  a.blocks_per_entry = plan.blocks_per_entry;
  a.tokens_per_block = plan.tokens_per_block;
  a.rows_per_tile = plan.rows_per_tile;
  a.box_rows = std::gcd(p->cache.page_size, 128);
  a.part_shift = 0;
  while (a.box_rows << a.part_shift < 128) ++a.part_shift;
  a.min_share = plan.min_share;
  a.scale_log2 = std::fabs(p->scale) * 1.4426950408889634f;
  a.negate = p->scale < 0.f;
  a.q = static_cast<const uint16_t*>(p->q);
  a.q_batch = p->q_strides.batch;
  a.q_row = p->q_strides.row;
  a.q_head = p->q_strides.head;
  a.o = static_cast<uint16_t*>(p->o);
  a.o_batch = p->o_strides.batch;
  a.o_row = p->o_strides.row;
  a.o_head = p->o_strides.head;
  a.lse = p->lse;
  char* ws = static_cast<char*>(workspace);
  a.o_part = reinterpret_cast<float*>(ws);
  a.lse_part = reinterpret_cast<float*>(ws + plan.part_bytes);
  a.item_blocks = reinterpret_cast<int2*>(ws + plan.part_bytes + plan.lse_bytes);
  a.status = p->status;
  return a;
}

// joins what was cut, launched as soon as no block of the kernel before is left to start or run (it waits for
// their writes itself)
template <bool kBf16, int DR, int kRows>
int launch_join(const fmha::PagedParams& a, const PagedPlan& plan, cudaStream_t stream) {
  using E = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
  const int items = a.batch * a.blocks_per_entry * a.heads_k, rows_per_item = plan.tiles * plan.rows_per_tile;
  const long long rows = (long long)items * rows_per_item;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)((rows + 7) / 8));
  config.blockDim = dim3(256);
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, fmha::paged_join_kernel<E, DR, kRows>, a, rows_per_item, items, plan.blocks) !=
      cudaSuccess) {
    (void)cudaGetLastError();
    return FMHA_ERR_LAUNCH;
  }
  return FMHA_OK;
}

template <int D, int DR, bool kBf16, bool kE4m3, int kRows>
int launch_few(const FmhaPagedFwdParams* p, const PagedPlan& plan, void* workspace, int dev, cudaStream_t stream) {
  using T = fmha::FewTraits<D, DR, kBf16, kE4m3, kRows>;
  const fmha::PagedParams a = kernel_params(p, plan, workspace);
  CUtensorMap tq, tk, tv;
  int rc;
  if ((rc = make_rows_map(&tq, p->q, p->batch, p->seqlen_q, p->heads_q, DR, p->q_strides, a.group, p->seqlen_q, kBf16)))
    return rc;
  if ((rc = make_pool_map(&tk, p->cache.k, p->cache, p->cache.k_strides, p->heads_k, DR, a.box_rows, kBf16)) ||
      (rc = make_pool_map(&tv, p->cache.v, p->cache, p->cache.v_strides, p->heads_k, DR, a.box_rows, kBf16)))
    return rc;
  if (!launch_with_smem<fmha::paged_few_kernel<D, DR, kBf16, kE4m3, kRows>>(dev, plan.blocks, T::kThreads, T::kSmemBytes,
                                                                            stream, tq, tk, tv, a))
    return FMHA_ERR_LAUNCH;
  return launch_join<kBf16, DR, kRows>(a, plan, stream);
}

template <int D, int DR, bool kBf16, bool kE4m3>
int launch_many(const FmhaPagedFwdParams* p, const PagedPlan& plan, void* workspace, int dev, cudaStream_t stream) {
  using T = fmha::ManyTraits<D, DR, kBf16, kE4m3>;
  const fmha::PagedParams a = kernel_params(p, plan, workspace);
  const int tokens = plan.tokens_per_block / 2;
  CUtensorMap tq, tk, tv, to;
  int rc;
  if ((rc = make_rows_map(&tq, p->q, p->batch, p->seqlen_q, p->heads_q, DR, p->q_strides, a.group, tokens, kBf16)) ||
      (rc = make_rows_map(&to, p->o, p->batch, p->seqlen_q, p->heads_q, DR, p->o_strides, a.group, tokens, kBf16)) ||
      (rc = make_pool_map(&tk, p->cache.k, p->cache, p->cache.k_strides, p->heads_k, DR, a.box_rows, kBf16)) ||
      (rc = make_pool_map(&tv, p->cache.v, p->cache, p->cache.v_strides, p->heads_k, DR, a.box_rows, kBf16)))
    return rc;
  if (!launch_with_smem<fmha::paged_many_kernel<D, DR, kBf16, kE4m3>>(dev, plan.blocks, T::kThreads, T::kSmemBytes, stream, tq,
                                                                      tk, tv, to, a))
    return FMHA_ERR_LAUNCH;
  return launch_join<kBf16, DR, 256>(a, plan, stream);
}

// rows of an entry (a thread's row is counted in 32 bits)
constexpr long long kMaxCacheRows = 1ll << 27;

// blocks of `per_block` rows for every entry
dim3 cache_grid(int rows, int per_block, int batch) {
  return dim3((unsigned)((rows + per_block - 1) / per_block), (unsigned)std::min(batch, 65535));
}

}  // namespace

extern "C" {

int fmha_cache_write(const FmhaCacheWriteParams* p, void* stream) {
  if (p == nullptr) return FMHA_ERR_NULL_POINTER;
  int rc = check_sizes(p->batch, p->heads, p->head_dim, p->dtype);
  if (rc) return rc;
  if (p->seqlen < 0) return FMHA_ERR_BAD_SHAPE;
  if (p->seqlen == 0 || p->batch == 0) return FMHA_OK;  // (empty tensors have no memory)
  if ((rc = check_cache(p->cache, p->heads))) return rc;
  const long long rows = (long long)p->seqlen * p->heads;
  if (rows > kMaxCacheRows || rows * p->batch > (1ll << 34)) return FMHA_ERR_TOO_LARGE;
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
  a.batch = p->batch;
  a.rows = (int)rows;
  const dim3 grid = cache_grid(a.rows, fmha::kWriteRows * (256 / (p->head_dim == 64 ? 8 : 16)), p->batch);
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
  if (p->seqlen == 0 || p->batch == 0) return FMHA_OK;  // (empty tensors have no memory)
  if ((rc = check_cache(p->cache, p->heads))) return rc;
  const long long rows = (long long)p->seqlen * p->heads;
  if (rows > kMaxCacheRows || rows * p->batch > (1ll << 34)) return FMHA_ERR_TOO_LARGE;
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
  a.batch = p->batch;
  a.rows = (int)rows;
  const dim3 grid = cache_grid(a.rows, fmha::kReadRows * (256 / (p->head_dim / 8)), p->batch);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FMHA_DISPATCH_CACHE(p->head_dim, p->dtype, p->cache.format,
                      fmha::cache_read_kernel<DR, kBf16, kE4m3><<<grid, 256, 0, s>>>(a);)
  return cudaGetLastError() == cudaSuccess ? FMHA_OK : FMHA_ERR_LAUNCH;
}

size_t fmha_paged_fwd_workspace_bytes(const FmhaPagedFwdParams* p) {
  if (p == nullptr || check_paged_sizes(p) != FMHA_OK || p->batch == 0 || p->seqlen_q == 0 ||
      check_paged_limits(p) != FMHA_OK)
    return 0;
  return plan_paged(p, sm_count(current_device())).bytes();
}

int fmha_paged_fwd(const FmhaPagedFwdParams* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (p == nullptr) return FMHA_ERR_NULL_POINTER;
  int rc = check_paged_sizes(p);
  if (rc) return rc;
  if (!std::isfinite(p->scale) || p->scale == 0.f) return FMHA_ERR_BAD_SHAPE;
  if (p->batch == 0 || p->seqlen_q == 0) return FMHA_OK;
  if ((rc = check_cache(p->cache, p->heads_k))) return rc;
  if ((rc = check_paged_limits(p))) return rc;
  if (p->q == nullptr || p->o == nullptr || p->lse == nullptr || p->seqused_k == nullptr) return FMHA_ERR_NULL_POINTER;
  if (!aligned16(p->q) || !aligned16(p->o) || !aligned16(workspace)) return FMHA_ERR_BAD_ALIGNMENT;
  if ((rc = check_strides(p->q_strides, p->seqlen_q, p->heads_q, p->batch))) return rc;
  if ((rc = check_strides(p->o_strides, p->seqlen_q, p->heads_q, p->batch))) return rc;
  const int dev = current_device();
  const PagedPlan plan = plan_paged(p, sm_count(dev));
  // the line of units (paged_work.cuh) is counted in 32 bits
  const double tiles = (double)p->cache.max_pages * p->cache.page_size / 128 + 2;
  if ((double)p->batch * p->heads_k * plan.blocks_per_entry * tiles >= 2147483648.0) return FMHA_ERR_TOO_LARGE;
  if (plan.bytes() > 0 && (workspace == nullptr || workspace_bytes < plan.bytes())) return FMHA_ERR_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  FMHA_DISPATCH_CACHE(p->head_dim, p->dtype, p->cache.format, {
    constexpr int D = DR == 64 ? 64 : 128;
    if (plan.kernel_rows == 16) return launch_few<D, DR, kBf16, kE4m3, 16>(p, plan, workspace, dev, s);
    if (plan.kernel_rows == 32) return launch_few<D, DR, kBf16, kE4m3, 32>(p, plan, workspace, dev, s);
    if (plan.kernel_rows == 48) return launch_few<D, DR, kBf16, kE4m3, 48>(p, plan, workspace, dev, s);
    if (plan.kernel_rows == 64) return launch_few<D, DR, kBf16, kE4m3, 64>(p, plan, workspace, dev, s);
    return launch_many<D, DR, kBf16, kE4m3>(p, plan, workspace, dev, s);
  })
}

}  // extern "C"
