// How attention over the paged cache is cut over the SMs, by lengths that only the device knows.
//
// An item is a block of new tokens of one entry with all query heads of one cache head; it has as many KV tiles of
// 128 keys as its last token sees.  All items' tiles in a row, plus kItemCost tiles for every item's own start and
// end, are one line of units, which is cut into equal shares: block c of the grid has units [c S, c S + S).  What a
// block does of one item is a piece.  A piece that is its whole item writes O and LSE; others leave fp32 rows, which
// paged_join_kernel joins.  So every SM has the same number of keys to read whatever the lengths are, a single long
// entry is spread over all of them, and an item is cut about as often as there are blocks to an item, no more.
// Every block works out the line's length and its own place on it from the lengths, a warp at a time.  (The line
// has less than 2^31 units: checked on the host.)
#pragma once
#include "cache_kernels.cuh"

namespace fmha {

struct PagedParams {
  PagedCache cache;
  const int32_t *seqused_k, *seqused_q;
  int batch, heads_k, group, seqlen_q, causal;
  unsigned group_mul;     // r / group = (r * group_mul) >> 16 for r < 256
  int blocks_per_entry;   // blocks of new tokens
  int tokens_per_block;
  int rows_per_tile;      // rows of a block that lie together in its partial rows: all (few rows), or each half (many)
  int box_rows;           // rows of a K or V box: what divides both a page and a tile, 128 >> part_shift
  int part_shift;
  int min_share;          // units a block has at least
  float scale_log2;       // |scale| * log2(e)
  int negate;             // scale < 0: the tensor cores form -Q K^T
  const uint16_t* q;
  long long q_batch, q_row, q_head;  // element strides
  uint16_t* o;
  long long o_batch, o_row, o_head;
  float* lse;
  // workspace: rows of pieces (slot, row, DR), their log-sum-exp (slot, row), blocks of every item
  float *o_part, *lse_part;
  int2* item_blocks;      // (first block, last block) of an item's tiles
  int* status;
};

// Units that an item costs beside its tiles.
constexpr int kItemCost = 1;

struct PagedPiece {
  int id;            // item, -1: no more
  int z, h, token0;  // entry, cache head, first new token
  int first, tiles;  // KV tiles [first, first + tiles); tiles = 0: the item sees no key at all
  int slot;          // of its partial rows, -1: the piece is the whole item
  int sq, sk;        // the entry's lengths
  int n0, n1;        // (many rows) of the tiles, those that the first and the second half of the block's rows see
};

__device__ __forceinline__ void paged_lengths(const PagedParams& p, int z, int& sq, int& sk) {
  sq = p.seqused_q == nullptr ? p.seqlen_q : max(0, min(p.seqlen_q, __ldg(p.seqused_q + z)));
  sk = max(0, min(__ldg(p.seqused_k + z), cache_capacity(p.cache)));
}
// the last key that token i of an entry sees (-1: none)
__device__ __forceinline__ int paged_last_key(const PagedParams& p, int i, int sq, int sk) {
  if (i >= sq) return -1;
  return p.causal ? max(-1, sk - sq + i) : sk - 1;
}
// KV tiles that `tokens` tokens from token0 on see
__device__ __forceinline__ int paged_tiles(const PagedParams& p, int token0, int tokens, int sq, int sk) {
  if (token0 >= sq) return 0;
  return (paged_last_key(p, min(token0 + tokens, sq) - 1, sq, sk) + 128) / 128;
}

__device__ __forceinline__ int row_token(const PagedParams& p, int r) { return (int)((unsigned)r * p.group_mul >> 16); }

// One block's share, walked in order by a converged warp (every lane has the same state).
struct PagedWork {
  int pos, end;     // units still to do
  int pair_start;   // first unit of the current (entry, block of tokens), all heads of which follow
  int pair, z, token0, tiles;
  int sq, sk;
  int share;

  __device__ __forceinline__ void enter_pair(const PagedParams& p) {
    z = pair / p.blocks_per_entry;
    token0 = (pair - z * p.blocks_per_entry) * p.tokens_per_block;
    paged_lengths(p, z, sq, sk);
    tiles = paged_tiles(p, token0, p.tokens_per_block, sq, sk);
  }

  __device__ __forceinline__ void start(const PagedParams& p, int block, int blocks) {
    const int lane = threadIdx.x & 31;
    const int pairs = p.batch * p.blocks_per_entry;
    auto units = [&](int f) {
      if (f >= pairs) return 0;
      pair = f;
      enter_pair(p);
      return p.heads_k * (tiles + kItemCost);
    };
    int total = 0;
#pragma unroll 1
    for (int f = lane; f < pairs; f += 32) total += units(f);
    total = __reduce_add_sync(0xffffffffu, total);
    share = max(p.min_share, (int)(((unsigned)total + blocks - 1) / blocks));
    pos = end = 0;
    if ((long long)block * share >= total) return;
    pos = block * share;
    end = share < total - pos ? pos + share : total;
    int before = 0;  // units of the pairs before this group of 32
#pragma unroll 1
    for (int f0 = 0;; f0 += 32) {
      const int mine = units(f0 + lane);
      int sum = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += up;
      }
      const uint32_t beyond = __ballot_sync(0xffffffffu, before + sum > pos);
      if (beyond != 0) {
        const int l = __ffs(beyond) - 1;
        pair = f0 + l;
        pair_start = __shfl_sync(0xffffffffu, before + sum - mine, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    enter_pair(p);
  }

  __device__ __forceinline__ PagedPiece next(const PagedParams& p, int block) {
    PagedPiece it = {};  // (the last one, which says that there is none, has no tiles for anybody)
    it.id = -1;
#pragma unroll 1
    while (pos < end) {
      const int w = tiles + kItemCost;
      const int h = (pos - pair_start) / w;
      if (h >= p.heads_k) {
        pair_start += p.heads_k * w;
        ++pair;
        enter_pair(p);
        continue;
      }
      const int u0 = pair_start + h * w;
      const int first = pos - u0, last = min(tiles, end - u0);
      pos = u0 + w;
      if (first >= tiles && !(tiles == 0 && first == 0)) continue;  // only the item's end: nothing to do for it
      it.id = pair * p.heads_k + h;
      it.z = z;
      it.h = h;
      it.token0 = token0;
      it.first = first;
      it.tiles = last - first;
      it.slot = first == 0 && last == tiles ? -1 : 2 * block + (first > 0 ? 0 : 1);
      it.sq = sq;
      it.sk = sk;
      const int half = p.tokens_per_block / 2;
      it.n0 = max(0, min(it.tiles, paged_tiles(p, token0, half, sq, sk) - first));
      it.n1 = max(0, min(it.tiles, paged_tiles(p, token0 + half, half, sq, sk) - first));
      if (first == 0 && (threadIdx.x & 31) == 0)
        p.item_blocks[it.id] = make_int2(u0 / share, tiles > 0 ? (u0 + tiles - 1) / share : u0 / share);
      break;
    }
    return it;
  }
};

// Pages of a piece's tiles, in parts of box_rows rows, 32 parts at a time, a lane each, and the next 32 while these are used:
// a lookup takes microseconds when all of HBM's rate is used.  For a converged warp.
struct PagedPages {
  const PagedParams& p;
  struct Window {
    int now, next;
  };
  __device__ __forceinline__ int parts() const { return 1 << p.part_shift; }  // of a tile

  // the table's entry for part 32 * batch + lane (not looked at before it is used)
  __device__ __forceinline__ int lookup(const PagedPiece& it, int batch) const {
    const int part = 32 * batch + (threadIdx.x & 31), key = it.first * 128 + part * p.box_rows;
    int entry = -1;
    if (part < it.tiles << p.part_shift && key < it.sk) entry = cache_entry(p.cache, it.z, key);
    return entry;
  }
  // page and row of a part of tile j, j in ascending order (num_pages, outside the pool, where there is none)
  __device__ __forceinline__ int page_of(const PagedPiece& it, Window& w, int j, int part, int& row) const {
    const int first = j << p.part_shift;
    if (j > 0 && (first & 31) == 0) {
      w.now = w.next;
      w.next = lookup(it, first / 32 + 1);
    }
    const int page = __shfl_sync(0xffffffffu, w.now, (first + part) & 31);
    row = cache_page_row(p.cache, it.first * 128 + (first + part) * p.box_rows);
    return (unsigned)page < (unsigned)p.cache.num_pages ? page : p.cache.num_pages;
  }
  // Scales of a tile's K and V rows into their stages of the ring of codes: four rows a lane, which lie in one page.  What is
  // copied is words, each the one that a row's byte is in (a word that holds a byte of an allocation is in it), and beside
  // them which of a word's bytes it is.
  __device__ __forceinline__ bool copy_scales(const PagedPiece& it, Window& w, int j, uint32_t* words, uint8_t* selects,
                                              uint64_t* full, uint64_t* empty, uint32_t stages, uint32_t& slot,
                                              uint32_t& phase, volatile int* abort_word) const {
    const int lane = threadIdx.x & 31;
    int row;
    const int page = page_of(it, w, j, lane >> (5 - p.part_shift), row);
    row += lane * 4 & (p.box_rows - 1);
#pragma unroll 1
    for (int n = 0; n < 2; ++n) {
      const PagePool& pool = n ? p.cache.v : p.cache.k;
      const uint8_t* src = pool.scales + page * pool.scale_page + row * pool.scale_row + it.h * pool.scale_head;
      if (!rolled_wait_warp(smem_u32(&empty[slot]), phase, abort_word, 19)) return false;
      const uint32_t to = smem_u32(words + slot * 128 + lane * 4);
      uint32_t select = 0;
      if (page < p.cache.num_pages) {
#pragma unroll
        for (int i = 0; i < 4; ++i, src += pool.scale_row) {
          const size_t at = reinterpret_cast<size_t>(src);
          copy_async4(to + 4 * i, reinterpret_cast<const void*>(at & ~size_t(3)));
          select |= (uint32_t)(at & 3) << (2 * i);
        }
      } else {
        sts128(to, 127, 127, 127, 127);
      }
      selects[slot * 32 + lane] = (uint8_t)select;
      copy_async_arrive(smem_u32(&full[slot]));
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&full[slot]));
      if (++slot == stages) {
        slot = 0;
        phase ^= 1;
      }
    }
    return true;
  }
};
// the scale byte of a row in a stage
__device__ __forceinline__ uint32_t staged_scale(const uint32_t* words, const uint8_t* selects, uint32_t stage, int row) {
  return words[stage * 128 + row] >> ((selects[stage * 32 + (row >> 2)] >> (row % 4 * 2) & 3) * 8) & 0xffu;
}

// Joins the pieces of the items that were cut: a warp per row.  Every partial row is normalised by its own row
// sum; its weight is exp(lse_part - lse).
template <typename E, int DR, int kRows>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedParams p, int rows_per_item, int items, int blocks_of_grid) {
  grid_dependency_wait();
  if (p.status != nullptr && *reinterpret_cast<const volatile int*>(p.status) != 0) return;
  const int lane = threadIdx.x & 31;
  const long long n = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int item = (int)(n / rows_per_item), row = (int)(n % rows_per_item);
  if (item >= items) return;
  const int2 blocks = p.item_blocks[item];
  // (where a wait ran out and nobody keeps a status word, this may be anything)
  if (blocks.x < 0 || blocks.x >= blocks.y || blocks.y >= blocks_of_grid) return;
  const int h = item % p.heads_k, pair = item / p.heads_k;
  const int z = pair / p.blocks_per_entry;
  const int half = row >= p.rows_per_tile ? 1 : 0, in_tile = row - half * p.rows_per_tile, t = row_token(p, in_tile);
  const int token = pair % p.blocks_per_entry * p.tokens_per_block + half * (p.rows_per_tile / p.group) + t;
  const int hq = h * p.group + in_tile - t * p.group;
  if (token >= p.seqlen_q) return;
  // part i: of block blocks.x + i.  Lane i has the weight of part i (of 32 at a time); rows are asked for eight at a time,
  // and before the weights are there: one after the other, 17 parts took 14 us.
  const int parts = blocks.y - blocks.x + 1;
  auto part_at = [&](int i) { return (long long)(2 * (blocks.x + i) + (i == 0 ? 1 : 0)) * kRows + half * 128 + in_tile; };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f, base = -CUDART_INF_F;
  const int col = lane * 4;
#pragma unroll 1
  for (int i0 = 0; i0 < parts; i0 += 32) {
    const float lp = i0 + lane < parts ? p.lse_part[part_at(i0 + lane)] : -CUDART_INF_F;
    float4 v[2][8];
    auto ask = [&](int buf, int i1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[buf][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i1 + i < 32 && i0 + i1 + i < parts && col < DR)
          v[buf][i] = *reinterpret_cast<const float4*>(p.o_part + part_at(i0 + i1 + i) * DR + col);
      }
    };
    ask(0, 0);
    ask(1, 8);
    // a part that is NaN makes the row NaN
    float mx = max_nan(lp, base);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    if (mx != base && base != -CUDART_INF_F) {  // more than 32 parts, and a larger one among the later ones
      const float a = expf(base - mx);
      sum *= a;
      acc.x *= a, acc.y *= a, acc.z *= a, acc.w *= a;
    }
    base = mx;
    // nothing visible in a part (-inf): its weight is 0, and its row may be anything; (inf - inf would be NaN)
    const float mine = lp == -CUDART_INF_F ? 0.f : lp == base ? 1.f : expf(lp - base);
#pragma unroll
    for (int i1 = 0; i1 < 32; i1 += 8) {
      if (i0 + i1 >= parts) break;
      float4(&x)[8] = v[i1 / 8 % 2];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = __shfl_sync(0xffffffffu, mine, i1 + i);
        if (w != 0.f) {
          sum += w;
          acc.x += w * x[i].x, acc.y += w * x[i].y, acc.z += w * x[i].z, acc.w += w * x[i].w;
        }
      }
      if (i1 < 16) ask(i1 / 8 % 2, i1 + 16);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (lane == 0)
    p.lse[((long long)z * p.heads_k * p.group + hq) * p.seqlen_q + token] = sum == 0.f ? -CUDART_INF_F : base + logf(sum);
  if (col < DR) {
    constexpr bool kBf16 = std::is_same<E, __nv_bfloat16>::value;
    uint2 v;
    v.x = pack16x2<kBf16>(acc.x * inv, acc.y * inv);
    v.y = pack16x2<kBf16>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(p.o + z * p.o_batch + token * p.o_row + hq * p.o_head + col) = v;
  }
}

}  // namespace fmha
