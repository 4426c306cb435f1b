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
// across threads, only a vote.  P in fp16 is 2^5 times the exponential, 2^15 at most: its least step, 2^-24, is then 2^-29 of
// the reference's weight, and a long tail of small weights is not lost.  The row sum has the factor, too.
//
//   warps 0-3   softmax: thread = key; P^T to shared memory; O^T (thread = element of the head) at the end
//   warps 4, 7  MMA issuers, of S^T and of O^T
//   warp 5      producer of Q; 8-bit caches: of the scales
//   warp 6      source of pieces; TMA producer of K and V, a box per page (or per part of one)
// 8-bit caches, whose codes and scales arrive in a ring of their own:
//   warps 8-11  K: codes -> fp16, into tensor memory (a thread has a key there, as in the softmax)
//   warps 12 up V: codes times scale -> 16 bits, into the ring that 16-bit caches load directly
//
// Shared memory, 128-byte swizzle: ring of K and V tiles (128 x D, boxes of 64 columns; 8-bit caches: of V tiles), Q (kRows
// x D, the same boxes), P^T (kRows x 128 keys, two boxes of 64 keys), codes (128 rows of 128 bytes).  Rows of V behind
// an entry's last token are set to zero before they are multiplied: the page may hold anything there, and 0 * NaN is NaN.
// Tensor memory: S^T twice, O^T twice, kRows columns each; 8-bit caches: K twice, 64 columns each.
//
// 8-bit caches are multiplied in fp16, in which a code is exact and a conversion is one instruction for two of them.
// K goes in without its scale, which the key's softmax thread has as a factor of its scores; Q of bf16 tensors is
// brought to fp16 under a power of two (see there).  V is multiplied by its scale: exact for exponents of -15 to 7 (a row's
// largest value between 0.007 and 57344).  Where one of 16 rows has another exponent, bf16 tensors have these rows of V, and
// P of these keys, in bf16, exactly; fp16 tensors have them rounded to fp16.  The codes come in by TMA, not through
// registers.
//
// The code is kept small: the roles share an instruction cache, and a miss waits in the same queues as HBM's data.
// With 135 KB of code (everything unrolled, waits among it) warps waited for instructions most of the time, and 64 entries
// of 2048 to 16384 keys in 8 bits took three times as long as their bytes.
//
// What bounds it.  16 bits, head dimension 128: HBM (32 entries of 2048 to 16384 keys, 32 query heads over 8: 182 us for 1.21
// GB, 6.6 TB/s, the rate of a copy).  Otherwise a tile's way through the softmax warps: 1470 clk at head dimension 64, 16
// bits, where 32 KB come in 1370 (16 entries of 16 heads: 4.3 TB/s), and 2200 to 2800 clk beside the converting warps, which
// wait for it (64 entries in 8 bits: 311 us, 3.9 TB/s).  Short calls: 10 us of start, first loads, last tile and join.
// A second group of softmax warps, which takes every other tile, was tried twice and taken back: 16 bits no faster, 8 bits
// 309 -> 359 (four warps for V) and 393 (eight; 80 registers a thread), only head dimension 64 in 8 bits gained (296 -> 270).
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
  // ring of K and V (16 bits), or of V alone and of codes (8 bits)
  static constexpr int kStages = kE4m3 ? (D == 128 ? 3 : 4) : D == 128 ? (kRows == 16 ? 6 : 5) : (kRows >= 48 ? 9 : 12);
  static constexpr int kCodeStages = !kE4m3 ? 0 : D == 128 && kRows >= 48 ? 4 : 6;
  static constexpr int kCodeBytes = 128 * 128;
  static constexpr int kQBufs = D == 128 && (kRows >= 48 || (kE4m3 && kRows == 32)) ? 1 : 2;
  static constexpr int kItemStages = 8;
  // warps that convert V: as many as the registers of the softmax's row sums leave room for
  static constexpr int kVWarps = kRows == 16 ? 8 : 4, kVRows = 128 / kVWarps;
  static constexpr int kThreads = kE4m3 ? 32 * (12 + kVWarps) : 256;
  static constexpr int kSmemBytes =
      1024 + kStages * kTileBytes + kCodeStages * kCodeBytes + kQBufs * kQBytes + 2 * kPBytes;
  static_assert(kSmemBytes <= 230400, "the rest of the 227 KB is for what is declared in the kernel");
  static constexpr int kTmemCols = !kE4m3 ? (kRows == 48 ? 256 : 4 * kRows) : kRows >= 48 ? 512 : 256;
  // 8-bit caches are multiplied in fp16 (see the converting warps)
  static constexpr uint32_t kIdescQK = umma_idesc_f16(128, kRows, 0, 0, kBf16 && !kE4m3);
  static constexpr uint32_t kIdescPV = umma_idesc_f16(128, kRows, 1, 0, kBf16 && !kE4m3);
  static constexpr uint32_t kIdescPVBf16 = umma_idesc_f16(128, kRows, 1, 0, true);
  // V^T has D rows; with D = 64 the upper 64 of the 128 repeat the lower ones, unused
  static constexpr uint32_t kLboV = D == 128 ? kBoxBytes : 0;
  static constexpr int kChunks = DR / 16;  // 16-byte chunks of a row of codes
  // P is 2^kLift times the exponential over the reference
  static constexpr float kLift = kBf16 && !kE4m3 ? 0.f : 5.f;
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

// 2^(byte - 127 + e), byte a scale (255 is NaN) and e the exponent of queries: the sum of the two is ordinary where each alone need
// not be.  (At 2^-126 scores are nothing, at 2^126 they are beyond fp32: beyond these it stays what it is.)
__device__ __forceinline__ float scale_power(uint32_t byte, int e) {
  const int sum = max(1, min(253, (int)byte + e));
  return __uint_as_float(byte == 255 ? 0x7fc00000u : (uint32_t)sum << 23);
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
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedParams p) {
  using T = FewTraits<D, DR, kBf16, kE4m3, kRows>;
  constexpr int kStages = T::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PagedPiece items[T::kItemStages];
  __shared__ uint64_t bar_item_full[T::kItemStages], bar_item_empty[T::kItemStages];
  // bar_kv_empty: of a slot.  bar_k_full, bar_v_full: K, V of tile n have landed, n modulo kStages.  Not of a slot: with an odd
  // number of slots one holds K and V by turns, each of which another warp waits for.  The issuer of S^T would come to wait for K(n)
  // in a slot before V(n - 3) had landed there, and the parity it waits for would be that of the phase before.
  __shared__ uint64_t bar_k_full[kE4m3 ? 1 : kStages], bar_v_full[kStages], bar_kv_empty[kStages];
  __shared__ uint64_t bar_q_full[2], bar_q_free[2], bar_s_full[2], bar_s_free[2], bar_p_full[2], bar_p_free[2],
      bar_o_full[2], bar_o_free[2];
  __shared__ float warp_part[4][kRows];   // per warp: a row's maximum, or its sum
  // kLift minus the reference, 0 where there is no finite one, -inf for rows that see no key
  __shared__ __align__(16) float row_neg[kRows];
  __shared__ __align__(16) float row_scale[kRows];  // what O is multiplied by
  __shared__ __align__(16) int row_last[kRows];     // last key a row sees
  __shared__ long long row_out[kRows];              // where a row of O lies, from its block's first row on
  // 8-bit caches: codes and scale bytes of a stage; K in tensor memory, and its scale bytes (a tile's are read after the
  // next two may have been converted); whether 16 rows of V in a slot are bf16; the power of two that a piece's Q was divided
  // by (Q is three pieces ahead at most), or each row's where they are too unequal for one
  __shared__ uint64_t bar_code_full[kE4m3 ? T::kCodeStages : 1], bar_code_empty[kE4m3 ? T::kCodeStages : 1];
  __shared__ uint64_t bar_kt_full[2], bar_kt_free[2];
  __shared__ __align__(16) uint32_t code_scale[kE4m3 ? T::kCodeStages : 1][128];  // the aligned word around a row's byte
  __shared__ uint8_t code_select[kE4m3 ? T::kCodeStages : 1][32];    // which byte of it, two bits for each of four rows
  __shared__ uint8_t k_scale[kE4m3 ? 4 : 1][128];
  __shared__ __align__(8) uint8_t v_bf16[kE4m3 ? kStages : 1][8];
  constexpr int kUnequal = 1 << 20;  // in place of an exponent
  __shared__ int q_exponent[4], q_row_exponent[kE4m3 && kBf16 ? 4 : 1][kRows];
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
  [[maybe_unused]] const uint32_t code_smem = p_smem + 2 * T::kPBytes;
  // position of V of tile n in the ring
  auto v_at = [](uint32_t n) { return kE4m3 ? n : 2 * n + 1; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::kItemStages; ++s) {
      mbar_init(smem_u32(&bar_item_full[s]), 1);
      mbar_init(smem_u32(&bar_item_empty[s]), kE4m3 ? 11 + T::kVWarps : 7);  // two MMA, Q, four softmax (eight converting) warps
    }
    for (int s = 0; s < kStages; ++s) {
      if (!kE4m3) mbar_init(smem_u32(&bar_k_full[s]), 1);
      mbar_init(smem_u32(&bar_v_full[s]), kE4m3 ? T::kVWarps : 1);
      mbar_init(smem_u32(&bar_kv_empty[s]), 1);
    }
    for (int s = 0; s < T::kCodeStages; ++s) {
      mbar_init(smem_u32(&bar_code_full[s]), 34);  // TMA's thread, a warp's copies of scales, its word on which byte
      mbar_init(smem_u32(&bar_code_empty[s]), s & 1 ? T::kVWarps : 4);  // (K has the even stages, V the odd ones)
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
      mbar_init(smem_u32(&bar_kt_full[b]), 4);
      mbar_init(smem_u32(&bar_kt_free[b]), 1);
    }
    fence_barrier_init();
  }
  // The first piece and its pages are worked out beside the rest of the set-up (2 us of loads that depend on one another).
  const PagedPages pages{p};
  PagedWork work;
  PagedPiece first_piece = {};
  int first_pages = -1;
  if (warp == 6) {
    if (elect_one()) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      tma_prefetch_desc(&tm_q);
    }
    __syncwarp();
    work.start(p, blockIdx.x, gridDim.x);
    first_piece = work.next(p, blockIdx.x);
    first_pages = pages.lookup(first_piece, 0);
  }
  if (warp == 4) {
    tmem_alloc(smem_u32(&tmem_base_slot), T::kTmemCols);
    tmem_relinquish();
  }
  // rows of Q that no load fills stay zero: their scores are 0
  for (uint32_t at = threadIdx.x * 16; at < T::kQBufs * T::kQBytes; at += blockDim.x * 16) sts128(q_smem + at, 0, 0, 0, 0);
  if (threadIdx.x < kRows) {
    const int t = row_token(p, threadIdx.x);
    row_out[threadIdx.x] = t * p.o_row + ((int)threadIdx.x - t * p.group) * p.o_head;
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);
  grid_dependents_may_start();  // the joining kernel, which then need not be launched when this one ends

  uint32_t item_cnt = 0;
  auto take_item = [&]() -> PagedPiece {
    const uint32_t s = item_cnt % T::kItemStages;
    PagedPiece it;
    if (rolled_wait_warp(smem_u32(&bar_item_full[s]), (item_cnt / T::kItemStages) & 1, &abort_word, 1)) {
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
    // A lane per box: 128 / box_rows parts of a tile, kBoxes column blocks of each (codes: one); lanes 0-15 K's, 16-31 V's.
    // One pass of the loop for both, because the pass, not what it asks for, is what takes the time (500 clk).  The next
    // piece is worked out while the last tiles of this one are asked for.
    constexpr int kCols = kE4m3 ? 1 : T::kBoxes;
    constexpr uint32_t kRing = kE4m3 ? T::kCodeStages : kStages;
    constexpr uint32_t kBytes = kE4m3 ? T::kCodeBytes : T::kTileBytes;
    const bool is_v = lane >= 16;
    const int sub = (lane & 15) / kCols, box = lane % kCols;
    const bool mine = sub < pages.parts();
    const uint32_t dst = (kE4m3 ? code_smem : ring_smem) + box * T::kBoxBytes + sub * p.box_rows * 128;
    const CUtensorMap* const tm = is_v ? &tm_v : &tm_k;
    uint64_t* const fulls = kE4m3 ? bar_code_full : is_v ? bar_v_full : bar_k_full;
    uint64_t* const empties = kE4m3 ? bar_code_empty : bar_kv_empty;
    bool ok = true;
    uint32_t slot = 0, phase = 1, published = 0, tile = 0;  // tile: modulo kStages
    auto next_item = [&]() -> PagedPiece {
      const PagedPiece it = published == 0 ? first_piece : work.next(p, blockIdx.x);
      const uint32_t s = published % T::kItemStages, round = published / T::kItemStages;
      if (round > 0) ok = rolled_wait_warp(smem_u32(&bar_item_empty[s]), (round - 1) & 1, &abort_word, 2);
      if (ok && lane == 0) {
        items[s] = it;
        mbar_arrive(smem_u32(&bar_item_full[s]));
      }
      __syncwarp();
      ++published;
      return it;
    };
    PagedPiece it = next_item();
    while (ok && it.id >= 0) {
      PagedPiece after = it;
      int first_pages_after = 0;
      PagedPages::Window window{first_pages, pages.lookup(it, 1)};
#pragma unroll 1
      for (int j = 0; ok && j < max(it.tiles, 1); ++j) {
        if (j + 2 >= it.tiles && after.id == it.id) {
          after = next_item();
          first_pages_after = pages.lookup(after, 0);
        }
        if (j >= it.tiles) break;  // (no tiles at all)
        int row;
        const int page = pages.page_of(it, window, j, sub, row);
        // K's slot and V's, the one behind it
        const uint32_t slot_v = slot + 1 == kRing ? 0 : slot + 1, phase_v = slot + 1 == kRing ? phase ^ 1 : phase;
        ok = ok && rolled_wait_warp(smem_u32(&empties[slot]), phase, &abort_word, 3) &&
             rolled_wait_warp(smem_u32(&empties[slot_v]), phase_v, &abort_word, 4);
        if (!ok) break;
        const uint32_t to = is_v ? slot_v : slot, full = smem_u32(&fulls[kE4m3 ? to : tile]);
        if ((lane & 15) == 0) mbar_arrive_expect_tx(full, kBytes);
        __syncwarp();
        if (mine) tma_load_4d(dst + to * kBytes, tm, full, box * 64, row, it.h, page);
        __syncwarp();
        phase = slot + 2 >= kRing ? phase ^ 1 : phase;
        slot = slot + 2 >= kRing ? slot + 2 - kRing : slot + 2;
        tile = tile + 1 == (uint32_t)kStages ? 0 : tile + 1;
      }
      it = after;
      first_pages = first_pages_after;
    }
  } else if (warp == 5) {
    // =========================== Q producer; scales of codes ===========================
    const uint32_t bytes = T::kBoxes * p.seqlen_q * p.group * 128;
    uint32_t used = 0;
    [[maybe_unused]] uint32_t slot = 0, phase = 1;
    for (;;) {
      const PagedPiece it = take_item();
      if (it.id < 0) break;
      if (it.tiles == 0) continue;
      [[maybe_unused]] PagedPages::Window window = {};
      if constexpr (kE4m3) window = {pages.lookup(it, 0), pages.lookup(it, 1)};
      const uint32_t b = used % T::kQBufs, round = used / T::kQBufs;
      if (round > 0 && !rolled_wait_warp(smem_u32(&bar_q_free[b]), (round - 1) & 1, &abort_word, 24)) break;
      if constexpr (kE4m3 && kBf16) {
        // Q in fp16, like K: divided by the power of two that brings its largest value to [2^14, 2^15).  What is less
        // than 2^-28 of that value loses bits, nothing is off by more than 2^-39 of it.  So rows whose largest values are within
        // 2^13 of one another share one power (off by 2^-26 of a row's own at most, less than an fp32 sum is); others have one
        // each, which the softmax multiplies their scores by.  Rows behind the entry's new tokens may hold anything: they have
        // no say in it, and become zeros.
        const int total = p.seqlen_q * p.group * (DR / 8);  // chunks of 8 elements
        const int real = min(p.seqlen_q, it.sq - it.token0) * p.group * (DR / 8);
        const uint16_t* src = p.q + it.z * p.q_batch + it.token0 * p.q_row + it.h * p.group * p.q_head;
        auto chunk_of = [&](int n) {
          const int r = n / (DR / 8), t = row_token(p, r);
          return __ldg(reinterpret_cast<const uint4*>(src + t * p.q_row + (r - t * p.group) * p.q_head) + n % (DR / 8));
        };
        auto top_of = [](const uint4& x) {  // largest exponent field of a finite value
          uint32_t top = 0;
          for (uint32_t w : {x.x, x.y, x.z, x.w})
            for (uint32_t ex : {w >> 7 & 0xffu, w >> 23 & 0xffu}) top = ex == 255 ? top : max(top, ex);
          return top;
        };
        // (Four loads at a time where there are more than a few: 40 rows, 49.3 -> 43.7 us a call.  With 16 rows the code costs
        // more than they take: 64 entries 311 -> 319.)
        uint32_t most = 0, least = 255;
#pragma unroll(kRows == 16 ? 1 : 4)
        for (int n = lane; n < real; n += 32) {
          const uint32_t top = top_of(chunk_of(n));
          most = max(most, top);
          least = top == 0 ? least : min(least, top);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        least = __reduce_min_sync(0xffffffffu, least);
        const int e = most == 0 ? 0 : (int)most - 127 - 14;  // (-140 to 113)
        // (chunks within 2^13 of one another are of rows that are; where they are not, the rows may be)
        bool unequal = most > least + 13;
        int* const exponents = q_row_exponent[used & 3];
        if (unequal) {
          least = 255;
          for (int r = lane; r < kRows; r += 32) exponents[r] = e;
          __syncwarp();
#pragma unroll 1
          for (int n = 0; n < real; n += DR / 8) {
            const uint32_t top = __reduce_max_sync(0xffffffffu, lane < DR / 8 ? top_of(chunk_of(n + lane)) : 0u);
            least = top == 0 ? least : min(least, top);
            if (lane == 0 && top != 0) exponents[n / (DR / 8)] = (int)top - 127 - 14;
          }
          unequal = most > least + 13;
          __syncwarp();
        }
        // 2^-e in two factors: one alone need not be a normal number
        auto factor = [](int half) { return __uint_as_float((uint32_t)(127 - half) << 23); };
        float s0 = factor(e / 2), s1 = factor(e - e / 2);
#pragma unroll 1
        for (int n = lane; n < total; n += 32) {
          float f[8];
          unpack8<__nv_bfloat16>(n < real ? chunk_of(n) : make_uint4(0, 0, 0, 0), f);
          const int r = n / (DR / 8), c = n % (DR / 8);
          if (unequal) s0 = factor(exponents[r] / 2), s1 = factor(exponents[r] - exponents[r] / 2);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = f[i] * s0 * s1;
          sts128(q_smem + b * T::kQBytes + (c >> 3) * T::kQBoxBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4), pack_half2(f[0], f[1]),
                 pack_half2(f[2], f[3]), pack_half2(f[4], f[5]), pack_half2(f[6], f[7]));
        }
        if (lane == 0) q_exponent[used & 3] = unequal ? kUnequal : e;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_q_full[b]));
      } else if (elect_one()) {
        const uint32_t bar = smem_u32(&bar_q_full[b]);
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int box = 0; box < T::kBoxes; ++box)
          tma_load_4d(q_smem + b * T::kQBytes + box * T::kQBoxBytes, &tm_q, bar, box * 64, it.h * p.group, it.token0, it.z);
      }
      __syncwarp();
      ++used;
      if constexpr (kE4m3) {
        bool ok = true;
#pragma unroll 1
        for (int j = 0; ok && j < it.tiles; ++j)
          ok = pages.copy_scales(it, window, j, code_scale[0], code_select[0], bar_code_full, bar_code_empty, T::kCodeStages, slot,
                                 phase, &abort_word);
        if (!ok) break;
      }
    }
  } else if (warp == 4) {
    // =========================== MMA issuer of S^T = K Q^T ===================
    // Each product has a warp of its own: issuing, the commits most of all, takes longer than the products themselves.
    uint32_t n = 0, piece = 0, slot = 0, tile = 0, phase = 0;  // tile: n modulo kStages, and the parity of its round
    bool ok = true;
    while (ok) {
      const PagedPiece it = take_item();
      if (it.id < 0) break;
#pragma unroll 1
      for (int j = 0; j < it.tiles; ++j, ++n) {
        const uint32_t b = n & 1, qb = piece % T::kQBufs;
        if (j == 0) ok = rolled_wait_warp(smem_u32(&bar_q_full[qb]), piece / T::kQBufs & 1, &abort_word, 8);
        if (kE4m3)
          ok = ok && rolled_wait_warp(smem_u32(&bar_kt_full[b]), (n >> 1) & 1, &abort_word, 18);
        else
          ok = ok && rolled_wait_warp(smem_u32(&bar_k_full[tile]), phase, &abort_word, 9);
        if (ok && n >= 2) ok = rolled_wait_warp(smem_u32(&bar_s_free[b]), ((n >> 1) - 1) & 1, &abort_word, 10);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a_lo = umma_desc_lo(ring_smem + slot * T::kTileBytes, kLboKMajor);
        const uint32_t b_lo = umma_desc_lo(q_smem + qb * T::kQBytes, kLboKMajor);
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < DR / 16; ++ks) {
            const uint32_t q_lo = b_lo + (((ks >> 2) * T::kQBoxBytes + (ks & 3) * 32) >> 4);
            if (kE4m3)
              umma_ts(tmem_base + b * kRows, tmem_base + 4 * kRows + b * 64 + ks * 8, q_lo, T::kIdescQK, ks > 0 ? 1u : 0u);
            else
              umma_ss(tmem_base + b * kRows, a_lo + (((ks >> 2) * T::kBoxBytes + (ks & 3) * 32) >> 4), q_lo, T::kIdescQK,
                      ks > 0 ? 1u : 0u);
          }
          umma_commit(smem_u32(&bar_s_full[b]));
          umma_commit(smem_u32(kE4m3 ? &bar_kt_free[b] : &bar_kv_empty[slot]));
          if (j == it.tiles - 1) umma_commit(smem_u32(&bar_q_free[qb]));
        }
        __syncwarp();
        if ((slot += 2) >= (uint32_t)kStages) slot -= kStages;
        if (++tile == (uint32_t)kStages) {
          tile = 0;
          phase ^= 1;
        }
      }
      if (it.tiles > 0) ++piece;
    }
  } else if (warp == 7) {
    // =========================== MMA issuer of O^T += V^T P^T ===================
    uint32_t n = 0, piece = 0, slot = kE4m3 ? 0 : 1, tile = 0, phase = 0;
    bool ok = true;
    while (ok) {
      const PagedPiece it = take_item();
      if (it.id < 0) break;
      const uint32_t ob = piece & 1;
#pragma unroll 1
      for (int j = 0; j < it.tiles; ++j, ++n) {
        const uint32_t b = n & 1;
        if (j == 0 && piece >= 2) ok = rolled_wait_warp(smem_u32(&bar_o_free[ob]), ((piece >> 1) - 1) & 1, &abort_word, 7);
        ok = ok && rolled_wait_warp(smem_u32(&bar_v_full[tile]), phase, &abort_word, 6) &&
             rolled_wait_warp(smem_u32(&bar_p_full[b]), (n >> 1) & 1, &abort_word, 5);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a_lo = umma_desc_lo(ring_smem + slot * T::kTileBytes, T::kLboV);
        const uint32_t b_lo = umma_desc_lo(p_smem + b * T::kPBytes, kLboKMajor);
        uint2 in_bf16 = make_uint2(0, 0);  // a byte for each 16 keys
        if constexpr (kE4m3 && kBf16) {
          in_bf16 = *reinterpret_cast<const uint2*>(v_bf16[slot]);
          in_bf16.x = __shfl_sync(0xffffffffu, in_bf16.x, 0);
          in_bf16.y = __shfl_sync(0xffffffffu, in_bf16.y, 0);
        }
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const bool bf = ((ks < 4 ? in_bf16.x : in_bf16.y) >> (ks % 4 * 8) & 1) != 0;
            umma_ss(tmem_base + (2 + ob) * kRows, a_lo + ((ks * 2048) >> 4),
                    b_lo + (((ks >> 2) * kRows * 128 + (ks & 3) * 32) >> 4), bf ? T::kIdescPVBf16 : T::kIdescPV,
                    (j > 0 || ks > 0) ? 1u : 0u);
          }
          umma_commit(smem_u32(&bar_kv_empty[slot]));
          umma_commit(smem_u32(&bar_p_free[b]));
          if (j == it.tiles - 1) umma_commit(smem_u32(&bar_o_full[ob]));
        }
        __syncwarp();
        if ((slot += kE4m3 ? 1 : 2) >= (uint32_t)kStages) slot -= kStages;
        if (++tile == (uint32_t)kStages) {
          tile = 0;
          phase ^= 1;
        }
      }
      if (it.tiles > 0) ++piece;
    }
  } else if (warp < 4) {
    // =========================== softmax, O ===========================
    const int tid = threadIdx.x;  // key of the tile, element of the head
    const uint32_t lane_addr = uint32_t(warp * 32) << 16;
    const int rows = p.seqlen_q * p.group;
    // P^T: row r at r * 128 bytes, keys 64 and up in a second box, 16-byte chunks swizzled by the row
    const uint32_t p_key = (tid >> 6) * (kRows * 128) + (tid & 7) * 2;
    const uint32_t p_chunk = (tid >> 3) & 7;
    float ref = -CUDART_INF_F;  // (threads below kRows) reference of row tid: a score times log2(e)
    uint32_t n = 0, piece = 0;
    for (;;) {
      const PagedPiece it = take_item();
      if (it.id < 0) break;
      const int token_of_row = row_token(p, tid);
      const bool row_here = tid < kRows && tid < rows;
      const int my_token = it.token0 + token_of_row, my_head = it.h * p.group + tid - token_of_row * p.group;
      float* const my_lse = it.slot >= 0 ? p.lse_part + (long long)it.slot * kRows + tid
                                         : p.lse + ((long long)it.z * p.heads_k * p.group + my_head) * p.seqlen_q + my_token;
      if (it.tiles == 0) {  // nobody sees anything: O = 0, LSE = -inf
        if (row_here) *my_lse = -CUDART_INF_F;
        if (tid < DR)
#pragma unroll 1
          for (int r = 0; r < rows; ++r)
            p.o[it.z * p.o_batch + it.token0 * p.o_row + it.h * p.group * p.o_head + row_out[r] + tid] = 0;
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
      bool force = true;  // some row has no reference yet, or a very large one
#pragma unroll 1
      for (int j = 0; j < it.tiles; ++j, ++n) {
        const uint32_t b = n & 1;
        const int key0 = (it.first + j) * 128, key = key0 + tid;
        const uint32_t tS = tmem_base + lane_addr + b * kRows, tO = tmem_base + lane_addr + (2 + (piece & 1)) * kRows;
        rolled_wait(smem_u32(&bar_s_full[b]), (n >> 1) & 1, &abort_word, 11);
        tc_fence_after();
        float c = p.negate ? -p.scale_log2 : p.scale_log2;
        [[maybe_unused]] const int eq = kE4m3 && kBf16 ? q_exponent[piece & 3] : 0;
        if constexpr (kE4m3) c *= scale_power(k_scale[n & 3][tid], eq);
        // The exponentials' arguments: with 16 rows they stay in registers between the vote and the exponentials, with more
        // they are formed twice.
        float x[16];
        auto arguments = [&](int r0) {
          uint32_t s[16];
          tmem_ld16(tS + r0, s);
          tmem_wait_ld();
          const uint64_t c2 = pack2f(c, c);
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float4 g = *reinterpret_cast<const float4*>(&row_neg[r0 + i]);
            uint32_t a, b;
            unpack2(fma2(pack2(s[i], s[i + 1]), c2, pack2f(g.x, g.y)), a, b);
            x[i] = __uint_as_float(a), x[i + 1] = __uint_as_float(b);
            unpack2(fma2(pack2(s[i + 2], s[i + 3]), c2, pack2f(g.z, g.w)), a, b);
            x[i + 2] = __uint_as_float(a), x[i + 3] = __uint_as_float(b);
          }
        };
        if (j > 0) {
          // Would an exponential be too large?  (2^10 over the reference: P has to stay below the 65504 of fp16.)  Rows that see
          // no key, padding among them, have no say: their arguments are -inf, or NaN, which the maximum passes over.  (A NaN of
          // a row that does see the key makes P and the row sum NaN whatever the reference is.)
          float top = -CUDART_INF_F;
#pragma unroll
          for (int r0 = 0; r0 < kRows; r0 += 16) {
            arguments(r0);
#pragma unroll
            for (int i = 0; i < 16; i += 2) top = max3(top, x[i], x[i + 1]);
          }
          force = vote_any(1, 128, force || (key < it.sk && !(top <= 10.f + T::kLift)));
        }
        const bool all_seen = key0 + 127 <= least;
        const bool renewed = force;
        if (force) {
          // A new reference for every row: its largest score so far.  It is a rounded product, so this tile's scores become
          // rounded products, too, before it is taken off: in one step, a score of 2^28 could come out at 2^4 over itself, or
          // under.  Where a reference exceeds 2^20, every tile takes new ones; and where rows have a power of two each, which a
          // score of theirs is multiplied by here.
          if constexpr (kE4m3 && kBf16) {
            if (eq == kUnequal) {
              const float base = p.negate ? -p.scale_log2 : p.scale_log2;
              c = 1.f;
#pragma unroll 1
              for (int r = 0; r < kRows; ++r) {
                const float s = tmem_ld1(tS + r);
                tmem_st1(tS + r, s * (base * scale_power(k_scale[n & 3][tid], q_row_exponent[piece & 3][r])));
              }
              tmem_wait_st();
            }
          }
#pragma unroll 1
          for (int r0 = 0; r0 < kRows; r0 += 16) {
            uint32_t s[16];
            tmem_ld16(tS + r0, s);
            tmem_wait_ld();
            float mine = -CUDART_INF_F;
            if (r0 == 0 && j == 0) named_bar_sync(1, 128);  // row_last is there
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float product = __uint_as_float(s[i]) * c;
              s[i] = __float_as_uint(product);
              const float m = warp_max(key <= row_last[r0 + i] ? product : -CUDART_INF_F);
              mine = lane == i ? m : mine;
            }
            tmem_st16(tS + r0, s);
            if (lane < 16) warp_part[warp][r0 + lane] = mine;
          }
          tmem_wait_st();
          c = 1.f;
          named_bar_sync(1, 128);
          bool unset = false;  // the next tile has to take references again
          if (tid < kRows) {
            const float m = fmaxf(fmaxf(fmaxf(warp_part[0][tid], warp_part[1][tid]),
                                        fmaxf(warp_part[2][tid], warp_part[3][tid])), ref);
            row_scale[tid] = isinf(m) || isinf(ref) ? 1.f : fast_exp2(ref - m);
            row_neg[tid] = row_last[tid] < 0 ? -CUDART_INF_F : isinf(m) ? 0.f : T::kLift - m;
            ref = m;
            unset = m == -CUDART_INF_F ? row_last[tid] > key0 + 127 : fabsf(m) > 1048576.f;
          }
          force = vote_any(1, 128, unset || (kE4m3 && kBf16 && eq == kUnequal));
          if (j > 0) {
            // O^T of the tiles before is complete
            rolled_wait(smem_u32(&bar_p_free[b ^ 1]), ((n - 1) >> 1) & 1, &abort_word, 12);
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
          const uint32_t slot = v_at(n) % kStages;
          rolled_wait(smem_u32(&bar_v_full[n % kStages]), n / kStages & 1, &abort_word, 13);
          if (key >= it.sk) {
#pragma unroll
            for (int box = 0; box < T::kBoxes; ++box)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                sts128(ring_smem + slot * T::kTileBytes + box * T::kBoxBytes + tid * 128 + i * 16, 0, 0, 0, 0);
          }
        }
        [[maybe_unused]] bool bf = false;
        if constexpr (kE4m3 && kBf16) {
          const uint32_t slot = n % kStages;
          rolled_wait(smem_u32(&bar_v_full[slot]), n / kStages & 1, &abort_word, 17);
          bf = v_bf16[slot][tid >> 4] != 0;
        }
        if (n >= 2) rolled_wait(smem_u32(&bar_p_free[b]), ((n >> 1) - 1) & 1, &abort_word, 14);
        const uint32_t dst = p_smem + b * T::kPBytes + p_key;
#pragma unroll
        for (int r0 = 0; r0 < kRows; r0 += 16) {
          if (kRows > 16 || renewed) arguments(r0);
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            float e[4] = {fast_exp2(x[i]), fast_exp2(x[i + 1]), fast_exp2(x[i + 2]), fast_exp2(x[i + 3])};
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
              uint32_t w = pack16x2<kBf16 && !kE4m3>(e[u], e[u + 1]);
              if (kE4m3 && kBf16 && bf) w = pack_bf16x2(e[u], e[u + 1]);
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
        constexpr float kUnlift = T::kLift == 0.f ? 1.f : 1.f / 32.f;
        const float sum = (warp_part[0][tid] + warp_part[1][tid]) + (warp_part[2][tid] + warp_part[3][tid]);
        // (a score of infinity: inf / inf is NaN, and 1 / inf would be the 0 of a row without a key)
        row_scale[tid] = sum == 0.f ? 0.f : isinf(sum) ? CUDART_NAN_F : 1.f / sum;
        if (row_here) *my_lse = sum == 0.f ? -CUDART_INF_F : (ref + log2f(sum * kUnlift)) * 0.6931471805599453f;
      }
      named_bar_sync(1, 128);
      const uint32_t ob = piece & 1;
      rolled_wait(smem_u32(&bar_o_full[ob]), (piece >> 1) & 1, &abort_word, 15);
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
            const float a = row_scale[r], v = a == 0.f ? 0.f : __uint_as_float(o[i]) * a;
            if (it.slot >= 0)
              part[r * DR] = v;
            else
              out[row_out[r]] = (uint16_t)pack16x2<kBf16>(v, 0.f);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_o_free[ob]));
      ++piece;
    }
  } else if constexpr (kE4m3) {
    if (warp >= 8 && warp < 12) {
      // =========================== K: codes -> fp16 in tensor memory, thread = key ===========================
      const int tid = threadIdx.x - 256;
      const uint32_t tK = tmem_base + (uint32_t(tid & ~31) << 16) + 4 * kRows;
      uint32_t n = 0;
      bool ok = true;
      while (ok) {
        const PagedPiece it = take_item();
        if (it.id < 0) break;
#pragma unroll 1
        for (int j = 0; j < it.tiles; ++j, ++n) {
          const uint32_t b = n & 1, at = 2 * n, slot = at % T::kCodeStages;
          ok = rolled_wait_warp(smem_u32(&bar_code_full[slot]), at / T::kCodeStages & 1, &abort_word, 20);
          if (ok && n >= 2) ok = rolled_wait_warp(smem_u32(&bar_kt_free[b]), ((n >> 1) - 1) & 1, &abort_word, 21);
          if (!ok) break;
          tc_fence_after();
          const uint32_t src = code_smem + slot * T::kCodeBytes + tid * 128;
          k_scale[n & 3][tid] = (uint8_t)staged_scale(code_scale[0], code_select[0], slot, tid);
#pragma unroll 2
          for (int i = 0; i < T::kChunks; i += 2) {  // 32 elements, 16 columns of tensor memory
            uint32_t w[16];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float4 f = lds128(src + (((i + half) ^ (tid & 7)) << 4));
              const uint32_t codes[4] = {__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w)};
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                w[half * 8 + 2 * u] = e4m3x2_to_half2(codes[u] & 0xffffu);
                w[half * 8 + 2 * u + 1] = e4m3x2_to_half2(codes[u] >> 16);
              }
            }
            tmem_st16(tK + b * 64 + i * 8, w);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(smem_u32(&bar_kt_full[b]));
            mbar_arrive(smem_u32(&bar_code_empty[slot]));
          }
        }
      }
    } else if (warp >= 12) {
      // =========================== V: codes times scale -> 16 bits in the ring ===========================
      // A warp has 16 or 32 rows, that is one or two steps of O^T += V^T P^T.
      static_assert(T::kCodeStages % 2 == 0, "K has the even stages, V the odd ones");
      const int row0 = T::kVRows * (warp - 12);
      uint32_t n = 0;
      bool ok = true;
      while (ok) {
        const PagedPiece it = take_item();
        if (it.id < 0) break;
#pragma unroll 1
        for (int j = 0; j < it.tiles; ++j, ++n) {
          const uint32_t slot = n % kStages, at = 2 * n + 1, from = at % T::kCodeStages;
          ok = rolled_wait_warp(smem_u32(&bar_code_full[from]), at / T::kCodeStages & 1, &abort_word, 22) &&
               rolled_wait_warp(smem_u32(&bar_kv_empty[slot]), (n / kStages & 1) ^ 1, &abort_word, 23);
          if (!ok) break;
          const int rows = min(T::kVRows, it.sk - (it.first + j) * 128 - row0);  // of the warp's that exist
          const uint32_t my_scale = lane < rows ? staged_scale(code_scale[0], code_select[0], from, row0 + lane) : 127u;
          const uint32_t fits = __ballot_sync(0xffffffffu, my_scale >= 112 && my_scale <= 134);
          // Four lanes have the four chunks of 16 codes that make a row of a box, and the eight lanes of a shared-memory
          // phase rows r and r ^ 5: then neither their loads nor their stores, which are swizzled by the row, meet in a bank.
          const uint32_t from_smem = code_smem + from * T::kCodeBytes, to_smem = ring_smem + slot * T::kTileBytes;
          const int in8 = lane & 4 ? lane >> 3 ^ 5 : lane >> 3, quarter = lane & 3;
          const uint32_t ld = row0 * 128 + in8 * 128 + ((quarter ^ in8) << 4), st = row0 * 128 + in8 * 128 + ((quarter * 2 ^ in8) << 4);
#pragma unroll 2
          for (int k = 0; k < T::kVRows / 8; ++k) {  // rows 8 k to 8 k + 7 of the warp's
            const uint32_t byte = __shfl_sync(0xffffffffu, my_scale, 8 * k + in8);
            const uint32_t h = (byte == 112 ? 0x0200u : (byte - 112) << 10) * 0x10001u;  // 2^(byte - 127) in fp16, twice
            const bool plain = (fits >> (k & 2) * 8 & 0xffffu) == 0xffffu;
#pragma unroll
            for (int box = 0; box < T::kBoxes; ++box) {
              if (DR == 96 && box == 1 && quarter >= 2) continue;
              const float4 f = lds128(from_smem + k * 1024 + (ld ^ box * 64));
              const uint32_t codes[4] = {__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w)};
              uint32_t w[8];
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                w[2 * u] = e4m3x2_to_half2(codes[u] & 0xffffu);
                w[2 * u + 1] = e4m3x2_to_half2(codes[u] >> 16);
              }
              if (plain) {
#pragma unroll
                for (int u = 0; u < 8; ++u) w[u] = mul_half2(w[u], h);
              } else {
                const float s = scale_value(byte);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                  const float2 v = __half22float2(*reinterpret_cast<__half2*>(&w[u]));
                  w[u] = pack16x2<kBf16>(v.x * s, v.y * s);
                }
              }
              const uint32_t to = to_smem + box * T::kBoxBytes + k * 1024 + st;
              sts128(to, w[0], w[1], w[2], w[3]);
              sts128(to ^ 16, w[4], w[5], w[6], w[7]);
            }
          }
          // rows behind the entry's end: zeros, whatever the page holds there
          __syncwarp();
          if (lane >= rows && lane < T::kVRows) {
            for (int i = 0; i < 8 * T::kBoxes; ++i)
              sts128(to_smem + (i >> 3) * T::kBoxBytes + (row0 + lane) * 128 + (i & 7) * 16, 0, 0, 0, 0);
          }
          if (lane < T::kVRows / 16) v_bf16[slot][T::kVRows / 16 * (warp - 12) + lane] = (fits >> (16 * lane) & 0xffffu) != 0xffffu;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(smem_u32(&bar_v_full[slot]));
            mbar_arrive(smem_u32(&bar_code_empty[from]));
          }
        }
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
