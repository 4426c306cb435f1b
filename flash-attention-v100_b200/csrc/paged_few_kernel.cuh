// Attention of few rows over the paged cache: single new tokens, drafted ones.  An item's rows (its new tokens
// times the query heads of one cache head) are kRows at most.
//
// Such a call reads the cache once and computes next to nothing, so everything is arranged around reading: the
// tensor cores get the CACHE as the 128-row operand and the few rows as the narrow one,
//   S^T (128 keys x rows) = K Q^T,     O^T (head_dim x rows) += V^T P^T,
// and a thread has one key: its scores of all rows are `rows` columns of tensor memory, a tile's softmax is a
// few dozen instructions, and what belongs to a key (is it visible) is worked out once per thread.  Row sums stay
// partial per thread until the item ends.  The reference of a row's exponentials is its maximum over the first tile; a
// later tile replaces it only where an exponential would exceed 2^10, so that an ordinary tile needs no maximum
// across threads, only a vote.
//
//   warps 0-3   softmax: thread = key; P^T to shared memory; O^T (thread = element of the head) at the end
//   warp 4      MMA issuer
//   warp 5      TMA producer of Q
//   warp 6      source of pieces; 16-bit caches: TMA producer of K and V, a box per page (or per part of one)
//   warps 8-15  8-bit caches: K and V through registers, codes times scale to 16 bits, into the ring
//
// Shared memory, 128-byte swizzle: ring of K and V tiles (128 x D, boxes of 64 columns), Q (kRows x D, the same
// boxes), P^T (kRows x 128 keys, two boxes of 64 keys).  Rows of V behind an entry's last token are set to
// zero before they are multiplied: the page may hold anything there, and 0 * NaN is NaN.
// Tensor memory: S^T twice, O^T twice, kRows columns each.
#pragma once
#include <cuda.h>

#include "paged_work.cuh"

namespace fmha {

template <int D, int DR, bool kBf16, bool kE4m3, int kRows>
struct FewTraits {
  static constexpr int kBoxes = D / 64;
  static constexpr int kBoxBytes = 128 * 128;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kQBoxBytes = kRows * 128;
  static constexpr int kQBytes = kBoxes * kQBoxBytes;
  static constexpr int kPBytes = 2 * kRows * 128;
  static constexpr int kStages = D == 128 ? (kRows == 64 ? 5 : 6) : (kRows == 64 ? 9 : 12);
  static constexpr int kQBufs = D == 128 && kRows == 64 ? 1 : 2;
  static constexpr int kItemStages = 4;
  static constexpr int kThreads = kE4m3 ? 512 : 224;
  static constexpr int kSmemBytes = 1024 + kStages * kTileBytes + kQBufs * kQBytes + 2 * kPBytes;
  static constexpr int kTmemCols = 4 * kRows;
  static constexpr uint32_t kIdescQK = umma_idesc_f16(128, kRows, 0, 0, kBf16);
  static constexpr uint32_t kIdescPV = umma_idesc_f16(128, kRows, 1, 0, kBf16);
  // V^T has D rows; with D = 64 the upper 64 of the 128 repeat the lower ones, unused
  static constexpr uint32_t kLboV = D == 128 ? kBoxBytes : 0;
  // 16-byte chunks of a row of codes, and how many of a tile's a converting thread has
  static constexpr int kChunks = DR / 16;
  static constexpr int kPerThread = 128 * kChunks / 256;
};

__device__ __forceinline__ bool vote_any(uint32_t id, uint32_t count, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)mine), "r"(id), "r"(count)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(addr), "h"((unsigned short)v) : "memory");
}

// Sums over the 32 lanes of N values each; lane l ends up with the total of value (l * N / 32) (N <= 32: of lanes
// that share a value, each has it).  Every step exchanges half of the values that a lane still has.
template <int N>
__device__ __forceinline__ float warp_totals(float (&v)[N], int lane) {
  int have = N;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    if (have > 1) {
      const bool upper = (lane & off) != 0;
      have /= 2;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
        if (i < have) {
          const float give = upper ? v[i] : v[i + have], keep = upper ? v[i + have] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    }
  }
  return v[0];
}

template <int D, int DR, bool kBf16, bool kE4m3, int kRows>
__global__ void __launch_bounds__(FewTraits<D, DR, kBf16, kE4m3, kRows>::kThreads, 1)
    paged_few_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const PagedParams p) {
  using T = FewTraits<D, DR, kBf16, kE4m3, kRows>;
  constexpr int kStages = T::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PagedPiece items[T::kItemStages];
  __shared__ uint64_t bar_item_full[T::kItemStages], bar_item_empty[T::kItemStages];
  __shared__ uint64_t bar_kv_full[kStages], bar_kv_empty[kStages];
  __shared__ uint64_t bar_q_full[2], bar_q_free[2], bar_s_full[2], bar_s_free[2], bar_p_full[2], bar_p_free[2],
      bar_o_full[2], bar_o_free[2];
  __shared__ float warp_part[4][kRows];   // per warp: a row's maximum, or its sum
  __shared__ __align__(16) float row_neg[kRows];    // -m * c, 0 where there is no finite reference
  __shared__ __align__(16) float row_scale[kRows];  // what O is multiplied by
  __shared__ __align__(16) int row_last[kRows];     // last key a row sees
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_word;
  __shared__ int skip_cta;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    skip_cta = (p.status != nullptr && *reinterpret_cast<volatile int*>(p.status) != 0) ? 1 : 0;
    abort_word = 0;
  }
  __syncthreads();
  if (skip_cta) return;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring_smem = smem_base;
  const uint32_t q_smem = ring_smem + kStages * T::kTileBytes;
  const uint32_t p_smem = q_smem + T::kQBufs * T::kQBytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::kItemStages; ++s) {
      mbar_init(smem_u32(&bar_item_full[s]), 1);
      mbar_init(smem_u32(&bar_item_empty[s]), kE4m3 ? 14 : 6);  // MMA, Q, four softmax (and eight converting) warps
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_kv_full[s]), kE4m3 ? 8 : 1);
      mbar_init(smem_u32(&bar_kv_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bar_q_full[b]), 1);
      mbar_init(smem_u32(&bar_q_free[b]), 1);
      mbar_init(smem_u32(&bar_s_full[b]), 1);
      mbar_init(smem_u32(&bar_s_free[b]), 4);
      mbar_init(smem_u32(&bar_p_full[b]), 4);
      mbar_init(smem_u32(&bar_p_free[b]), 1);
      mbar_init(smem_u32(&bar_o_full[b]), 1);
      mbar_init(smem_u32(&bar_o_free[b]), 4);
    }
    fence_barrier_init();
  }
  if (warp == 4) {
    tmem_alloc(smem_u32(&tmem_base_slot), T::kTmemCols);
    tmem_relinquish();
  }
  // rows of Q that no load fills stay zero: their scores are 0
  for (uint32_t at = threadIdx.x * 16; at < T::kQBufs * T::kQBytes; at += blockDim.x * 16) sts128(q_smem + at, 0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);

  uint32_t item_cnt = 0;
  auto take_item = [&]() -> PagedPiece {
    const uint32_t s = item_cnt % T::kItemStages;
    PagedPiece it;
    if (mbar_wait_warp(smem_u32(&bar_item_full[s]), (item_cnt / T::kItemStages) & 1, &abort_word, 1)) {
      it = items[s];
      it.id = __shfl_sync(0xffffffffu, it.id, 0);
      it.tiles = __shfl_sync(0xffffffffu, it.tiles, 0);
    } else {
      it.id = -1;
      it.tiles = 0;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bar_item_empty[s]));
    ++item_cnt;
    return it;
  };

  if (warp == 6) {
    // =========================== source of pieces, K and V producer ===========================
    PagedWork work;
    work.start(p, blockIdx.x, gridDim.x);
    bool ok = true;
    uint32_t published = 0, loaded = 0;
    [[maybe_unused]] const int subs = 128 / p.box_rows;
    while (ok) {
      const PagedPiece it = work.next(p, blockIdx.x);
      const uint32_t s = published % T::kItemStages, round = published / T::kItemStages;
      if (round > 0 && !mbar_wait_warp(smem_u32(&bar_item_empty[s]), (round - 1) & 1, &abort_word, 2)) break;
      if (lane == 0) {
        items[s] = it;
        mbar_arrive(smem_u32(&bar_item_full[s]));
      }
      __syncwarp();
      ++published;
      if (it.id < 0) break;
      if constexpr (!kE4m3) {
        // a lane per box: 128 / box_rows parts of the tile, kBoxes column blocks of each
        const int sub = lane / T::kBoxes, box = lane % T::kBoxes;
        const bool mine = sub < subs;
        const uint32_t dst = box * T::kBoxBytes + sub * p.box_rows * 128;
        auto place = [&](int tile, int& row) {  // page of this lane's part (num_pages, outside the pool: zeros)
          const int key = (it.first + tile) * 128 + sub * p.box_rows;
          row = key % p.cache.page_size;
          if (!mine || key >= it.sk) return p.cache.num_pages;
          const int page = cache_page(p.cache, it.z, key);
          return page < 0 ? p.cache.num_pages : page;
        };
        int row, page = place(0, row);
#pragma unroll 1
        for (int j = 0; ok && j < it.tiles; ++j) {
          int row_next = 0, page_next = 0;
          if (j + 1 < it.tiles) page_next = place(j + 1, row_next);
#pragma unroll 1
          for (int n = 0; n < 2; ++n) {
            const uint32_t slot = loaded % kStages;
            if (!(ok = mbar_wait_warp(smem_u32(&bar_kv_empty[slot]), (loaded / kStages & 1) ^ 1, &abort_word, 3))) break;
            if (lane == 0) mbar_arrive_expect_tx(smem_u32(&bar_kv_full[slot]), T::kTileBytes);
            __syncwarp();
            if (mine)
              tma_load_4d(ring_smem + slot * T::kTileBytes + dst, n ? &tm_v : &tm_k, smem_u32(&bar_kv_full[slot]), box * 64,
                          row, it.h, page);
            __syncwarp();
            ++loaded;
          }
          row = row_next;
          page = page_next;
        }
      }
    }
  } else if (warp == 5) {
    // =========================== Q producer ===========================
    const uint32_t bytes = T::kBoxes * p.seqlen_q * p.group * 128;
    uint32_t used = 0;
    for (;;) {
      const PagedPiece it = take_item();
      if (it.id < 0) break;
      if (it.tiles == 0) continue;
      const uint32_t b = used % T::kQBufs, round = used / T::kQBufs;
      if (round > 0 && !mbar_wait_warp(smem_u32(&bar_q_free[b]), (round - 1) & 1, &abort_word, 4)) break;
      if (elect_one()) {
        const uint32_t bar = smem_u32(&bar_q_full[b]);
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int box = 0; box < T::kBoxes; ++box)
          tma_load_4d(q_smem + b * T::kQBytes + box * T::kQBoxBytes, &tm_q, bar, box * 64, it.h * p.group, it.token0, it.z);
      }
      __syncwarp();
      ++used;
    }
  } else if (warp == 4) {
    // =========================== MMA issuer (converged warp, elected issue) ===================
    // S^T of a tile is issued before O^T of the one before it, so that the tensor pipe has work while the softmax
    // warps have the tile.  K of tile n is slot 2n of the ring, V slot 2n + 1.
    const uint32_t idesc_qk = T::kIdescQK | (p.negate ? kIdescNegateA : 0u);
    uint32_t n = 0, piece = 0;
    bool ok = true;
    bool pending = false, pending_first = false, pending_last = false;
    uint32_t pending_piece = 0;
    auto issue_pv = [&]() {
      const uint32_t m = n - 1, b = m & 1, at = 2 * m + 1, slot = at % kStages;
      ok = mbar_wait_warp(smem_u32(&bar_p_full[b]), (m >> 1) & 1, &abort_word, 5) &&
           mbar_wait_warp(smem_u32(&bar_kv_full[slot]), at / kStages & 1, &abort_word, 6);
      const uint32_t ob = pending_piece & 1;
      if (ok && pending_first && pending_piece >= 2)
        ok = mbar_wait_warp(smem_u32(&bar_o_free[ob]), ((pending_piece >> 1) - 1) & 1, &abort_word, 7);
      if (!ok) return;
      tc_fence_after();
      const uint32_t a_lo = umma_desc_lo(ring_smem + slot * T::kTileBytes, T::kLboV);
      const uint32_t b_lo = umma_desc_lo(p_smem + b * T::kPBytes, kLboKMajor);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
        umma_ss_elect(tmem_base + (2 + ob) * kRows, a_lo + ((ks * 2048) >> 4),
                      b_lo + (((ks >> 2) * kRows * 128 + (ks & 3) * 32) >> 4), T::kIdescPV,
                      (!pending_first || ks > 0) ? 1u : 0u);
      umma_commit_elect(smem_u32(&bar_kv_empty[slot]));
      umma_commit_elect(smem_u32(&bar_p_free[b]));
      if (pending_last) umma_commit_elect(smem_u32(&bar_o_full[ob]));
      pending = false;
    };
    while (ok) {
      const PagedPiece it = take_item();
      if (it.id < 0) break;
#pragma unroll 1
      for (int j = 0; j < it.tiles; ++j) {
        const uint32_t b = n & 1, at = 2 * n, slot = at % kStages, qb = piece % T::kQBufs;
        if (j == 0) ok = mbar_wait_warp(smem_u32(&bar_q_full[qb]), piece / T::kQBufs & 1, &abort_word, 8);
        ok = ok && mbar_wait_warp(smem_u32(&bar_kv_full[slot]), at / kStages & 1, &abort_word, 9);
        if (ok && n >= 2) ok = mbar_wait_warp(smem_u32(&bar_s_free[b]), ((n >> 1) - 1) & 1, &abort_word, 10);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a_lo = umma_desc_lo(ring_smem + slot * T::kTileBytes, kLboKMajor);
        const uint32_t b_lo = umma_desc_lo(q_smem + qb * T::kQBytes, kLboKMajor);
#pragma unroll
        for (int ks = 0; ks < DR / 16; ++ks)
          umma_ss_elect(tmem_base + b * kRows, a_lo + (((ks >> 2) * T::kBoxBytes + (ks & 3) * 32) >> 4),
                        b_lo + (((ks >> 2) * T::kQBoxBytes + (ks & 3) * 32) >> 4), idesc_qk, ks > 0 ? 1u : 0u);
        umma_commit_elect(smem_u32(&bar_kv_empty[slot]));
        umma_commit_elect(smem_u32(&bar_s_full[b]));
        if (j == it.tiles - 1) umma_commit_elect(smem_u32(&bar_q_free[qb]));
        if (pending) issue_pv();
        if (!ok) break;
        ++n;
        pending = true;
        pending_first = j == 0;
        pending_last = j == it.tiles - 1;
        pending_piece = piece;
      }
      if (it.tiles > 0) ++piece;
    }
    if (ok && pending) issue_pv();
  } else if (warp < 4) {
    // =========================== softmax, O ===========================
    const int tid = threadIdx.x;  // key of the tile, element of the head
    const uint32_t lane_addr = uint32_t(warp * 32) << 16;
    const float c = p.scale_log2;
    const int rows = p.seqlen_q * p.group;
    // P^T: row r at r * 128 bytes, keys 64 and up in a second box, 16-byte chunks swizzled by the row
    const uint32_t p_key = (tid >> 6) * (kRows * 128) + (tid & 7) * 2;
    const uint32_t p_chunk = (tid >> 3) & 7;
    float ref = -CUDART_INF_F;  // (threads below kRows) reference of row tid
    uint32_t n = 0, piece = 0;
    for (;;) {
      const PagedPiece it = take_item();
      if (it.id < 0) break;
      const int token_of_row = tid / p.group;
      const bool row_here = tid < kRows && tid < rows;
      const int my_token = it.token0 + token_of_row, my_head = it.h * p.group + tid % p.group;
      float* const my_lse = it.slot >= 0 ? p.lse_part + (long long)it.slot * kRows + tid
                                         : p.lse + ((long long)it.z * p.heads_k * p.group + my_head) * p.seqlen_q + my_token;
      if (it.tiles == 0) {  // nobody sees anything: O = 0, LSE = -inf
        if (row_here) *my_lse = -CUDART_INF_F;
        if (tid < DR)
          for (int r = 0; r < rows; ++r)
            p.o[it.z * p.o_batch + (it.token0 + r / p.group) * p.o_row + (it.h * p.group + r % p.group) * p.o_head + tid] = 0;
        continue;
      }
      // rows that do not exist have scores of 0 and see every key there is
      const int least = it.token0 + p.seqlen_q > it.sq ? -1 : paged_last_key(p, it.token0, it.sq, it.sk);
      if (tid < kRows) {
        row_last[tid] = row_here ? paged_last_key(p, my_token, it.sq, it.sk) : it.sk - 1;
        ref = -CUDART_INF_F;
      }
      float l[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) l[r] = 0.f;
      bool force = true;  // some row has no reference yet
#pragma unroll 1
      for (int j = 0; j < it.tiles; ++j, ++n) {
        const uint32_t b = n & 1;
        const int key0 = (it.first + j) * 128, key = key0 + tid;
        const uint32_t tS = tmem_base + lane_addr + b * kRows, tO = tmem_base + lane_addr + (2 + (piece & 1)) * kRows;
        mbar_wait(smem_u32(&bar_s_full[b]), (n >> 1) & 1, &abort_word, 11);
        tc_fence_after();
        if (j > 0) {
          // would an exponential be too large?  (2^10: P has to stay far from the 65504 of fp16)
          float top = -CUDART_INF_F;
#pragma unroll
          for (int r0 = 0; r0 < kRows; r0 += 16) {
            uint32_t s[16];
            tmem_ld16(tS + r0, s);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 g = *reinterpret_cast<const float4*>(&row_neg[r0 + i]);
              top = max3_nan(top, fmaf(__uint_as_float(s[i]), c, g.x), fmaf(__uint_as_float(s[i + 1]), c, g.y));
              top = max3_nan(top, fmaf(__uint_as_float(s[i + 2]), c, g.z), fmaf(__uint_as_float(s[i + 3]), c, g.w));
            }
          }
          force = vote_any(1, 128, force || (key < it.sk && !(top <= 10.f)));
        }
        const bool all_seen = key0 + 127 <= least;
        if (force) {
          // a new reference for every row: its largest score so far
#pragma unroll 1
          for (int r0 = 0; r0 < kRows; r0 += 16) {
            uint32_t s[16];
            tmem_ld16(tS + r0, s);
            tmem_wait_ld();
            float mine = -CUDART_INF_F;
            if (r0 == 0 && j == 0) named_bar_sync(1, 128);  // row_last is there
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float m = warp_max(key <= row_last[r0 + i] ? __uint_as_float(s[i]) : -CUDART_INF_F);
              mine = lane == i ? m : mine;
            }
            if (lane < 16) warp_part[warp][r0 + lane] = mine;
          }
          named_bar_sync(1, 128);
          bool unset = false;
          if (tid < kRows) {
            const float m = fmaxf(fmaxf(fmaxf(warp_part[0][tid], warp_part[1][tid]),
                                        fmaxf(warp_part[2][tid], warp_part[3][tid])), ref);
            row_scale[tid] = isinf(m) || isinf(ref) ? 1.f : fast_exp2((ref - m) * c);
            row_neg[tid] = isinf(m) ? 0.f : -m * c;
            ref = m;
            unset = m == -CUDART_INF_F && row_last[tid] > key0 + 127;
          }
          force = vote_any(1, 128, unset);
          if (j > 0) {
            // O^T of the tiles before is complete
            mbar_wait(smem_u32(&bar_p_free[b ^ 1]), ((n - 1) >> 1) & 1, &abort_word, 12);
            tc_fence_after();
#pragma unroll
            for (int r0 = 0; r0 < kRows; r0 += 16) {
              uint32_t o[16];
              tmem_ld16(tO + r0, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float a = row_scale[r0 + i];
                o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
                l[r0 + i] *= a;
              }
              tmem_st16(tO + r0, o);
            }
            tmem_wait_st();
          }
        }
        if (!kE4m3 && key0 + 128 > it.sk) {
          // rows of V behind the entry's end
          const uint32_t at = 2 * n + 1, slot = at % kStages;
          mbar_wait(smem_u32(&bar_kv_full[slot]), at / kStages & 1, &abort_word, 13);
          if (key >= it.sk) {
#pragma unroll
            for (int box = 0; box < T::kBoxes; ++box)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                sts128(ring_smem + slot * T::kTileBytes + box * T::kBoxBytes + tid * 128 + i * 16, 0, 0, 0, 0);
          }
        }
        if (n >= 2) mbar_wait(smem_u32(&bar_p_free[b]), ((n >> 1) - 1) & 1, &abort_word, 14);
        const uint32_t dst = p_smem + b * T::kPBytes + p_key;
#pragma unroll
        for (int r0 = 0; r0 < kRows; r0 += 16) {
          uint32_t s[16];
          tmem_ld16(tS + r0, s);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float4 g = *reinterpret_cast<const float4*>(&row_neg[r0 + i]);
            float e[4] = {fast_exp2(fmaf(__uint_as_float(s[i]), c, g.x)), fast_exp2(fmaf(__uint_as_float(s[i + 1]), c, g.y)),
                          fast_exp2(fmaf(__uint_as_float(s[i + 2]), c, g.z)), fast_exp2(fmaf(__uint_as_float(s[i + 3]), c, g.w))};
            if (!all_seen) {
              const int4 last = *reinterpret_cast<const int4*>(&row_last[r0 + i]);
              e[0] = key <= last.x ? e[0] : 0.f;
              e[1] = key <= last.y ? e[1] : 0.f;
              e[2] = key <= last.z ? e[2] : 0.f;
              e[3] = key <= last.w ? e[3] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 4; u += 2) {
              l[r0 + i + u] += e[u];
              l[r0 + i + u + 1] += e[u + 1];
              const uint32_t w = pack16x2<kBf16>(e[u], e[u + 1]);
              const int r = r0 + i + u;
              sts16(dst + r * 128 + ((p_chunk ^ (r & 7)) << 4), w);
              sts16(dst + (r + 1) * 128 + ((p_chunk ^ ((r + 1) & 7)) << 4), w >> 16);
            }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&bar_s_free[b]));
          mbar_arrive(smem_u32(&bar_p_full[b]));
        }
      }
      // ---- the piece's end: row sums over the threads, O^T / l
#pragma unroll
      for (int r0 = 0; r0 < kRows; r0 += 16) {
        float part[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) part[i] = l[r0 + i];
        const float sum = warp_totals(part, lane);
        if ((lane & 1) == 0) warp_part[warp][r0 + (lane >> 1)] = sum;
      }
      named_bar_sync(1, 128);
      if (tid < kRows) {
        const float sum = (warp_part[0][tid] + warp_part[1][tid]) + (warp_part[2][tid] + warp_part[3][tid]);
        row_scale[tid] = sum == 0.f ? 0.f : 1.f / sum;
        if (row_here) *my_lse = sum == 0.f ? -CUDART_INF_F : (ref * c + log2f(sum)) * 0.6931471805599453f;
      }
      named_bar_sync(1, 128);
      const uint32_t ob = piece & 1;
      mbar_wait(smem_u32(&bar_o_full[ob]), (piece >> 1) & 1, &abort_word, 15);
      tc_fence_after();
      uint16_t* const out = p.o + it.z * p.o_batch + it.token0 * p.o_row + it.h * p.group * p.o_head + tid;
      float* const part = p.o_part + (long long)it.slot * kRows * DR + tid;
#pragma unroll 1
      for (int r0 = 0; r0 < kRows && r0 < rows; r0 += 16) {
        uint32_t o[16];
        tmem_ld16(tmem_base + lane_addr + (2 + ob) * kRows + r0, o);
        tmem_wait_ld();
        if (tid < DR) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = r0 + i;
            if (r >= rows) break;
            // (a row without a visible key: P was 0, but 0 times what V holds need not be)
            const float v = row_scale[r] == 0.f ? 0.f : __uint_as_float(o[i]) * row_scale[r];
            if (it.slot >= 0)
              part[r * DR] = v;
            else
              out[r / p.group * p.o_row + r % p.group * p.o_head] = (uint16_t)pack16x2<kBf16>(v, 0.f);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_o_free[ob]));
      ++piece;
    }
  } else if (kE4m3 && warp >= 8) {
    // =========================== 8-bit K and V into the ring ===========================
    // A thread has the same chunks (row, 16 codes) of every tile.  Two tiles are in flight in registers, 64 KB per SM,
    // while a third is converted.
    constexpr int kPer = T::kPerThread, kDepth = 2;
    const int t = threadIdx.x - 256;
    struct Chunk {
      uint4 codes[2][kPer];
      uint32_t scale[2][kPer];
    };
    Chunk buf[kDepth];
    PagedPiece it;
    it.id = 0;
    it.tiles = 0;
    int j = 0;
    // the next tile of this block's pieces -> registers; false: there is none
    auto fetch = [&](Chunk& x) -> bool {
      while (j >= it.tiles) {
        if (it.id < 0) return false;
        it = take_item();
        j = 0;
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int idx = t + 256 * i, row = idx / T::kChunks, chunk = idx % T::kChunks;
        const int key = (it.first + j) * 128 + row;
        const int page = key < it.sk ? cache_page(p.cache, it.z, key) : -1;
        const int slot = key % p.cache.page_size;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const PagePool& pool = n ? p.cache.v : p.cache.k;
          x.codes[n][i] = make_uint4(0, 0, 0, 0);
          x.scale[n][i] = 127;
          if (page >= 0) {
            x.codes[n][i] = __ldg(reinterpret_cast<const uint4*>(pool.rows + page * pool.page + slot * pool.row + it.h * pool.head) + chunk);
            x.scale[n][i] = __ldg(pool.scales + page * pool.scale_page + slot * pool.scale_row + it.h * pool.scale_head);
          }
        }
      }
      ++j;
      return true;
    };
    uint32_t done = 0;
    bool ok = true;
    auto store = [&](const Chunk& x) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t slot = done % kStages;
        ok = ok && mbar_wait_warp(smem_u32(&bar_kv_empty[slot]), (done / kStages & 1) ^ 1, &abort_word, 16);
        if (!ok) return;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int idx = t + 256 * i, row = idx / T::kChunks, chunk = idx % T::kChunks;
          const float s = scale_value(x.scale[n][i]);
          const uint2 a = e4m3x4_to_16<kBf16>(x.codes[n][i].x, s), b = e4m3x4_to_16<kBf16>(x.codes[n][i].y, s);
          const uint2 e = e4m3x4_to_16<kBf16>(x.codes[n][i].z, s), f = e4m3x4_to_16<kBf16>(x.codes[n][i].w, s);
          const uint32_t base = ring_smem + slot * T::kTileBytes + (chunk >> 2) * T::kBoxBytes + row * 128;
          const uint32_t q = (chunk & 3) * 2;
          // (threads of the second box start with their second half: the two boxes have the same banks)
          const bool swap = (chunk >> 2) != 0;
          const uint32_t first = base + (((q + (swap ? 1 : 0)) ^ (row & 7)) << 4);
          const uint32_t second = base + (((q + (swap ? 0 : 1)) ^ (row & 7)) << 4);
          sts128(first, swap ? e.x : a.x, swap ? e.y : a.y, swap ? f.x : b.x, swap ? f.y : b.y);
          sts128(second, swap ? a.x : e.x, swap ? a.y : e.y, swap ? b.x : f.x, swap ? b.y : f.y);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_kv_full[slot]));
        ++done;
      }
    };
    bool have[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) have[d] = fetch(buf[d]);
    while (ok && have[0]) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        if (!ok || !have[d]) continue;
        store(buf[d]);
        have[d] = ok && fetch(buf[d]);
      }
    }
  }

  // ---- teardown
  tc_fence_before();
  __syncthreads();
  if (abort_word != 0) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, 0, abort_word);
    // let copies that may still be in flight land before the shared memory is released
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem_base, T::kTmemCols);
  }
}

}  // namespace fmha
