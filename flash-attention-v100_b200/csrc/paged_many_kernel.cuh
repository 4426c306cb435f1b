// Attention of many rows over the paged cache: a chunk of new tokens.  The mathematics, the roles and the order of the
// turns are those of fmha_fwd_kernel (fwd_kernel.cuh, which says why); what differs is where rows and keys lie and how
// work is cut:
//
//   - An item is 256 rows, two tiles of 128: new tokens times the query heads of one cache head, so that K and V are
//     read once for all of them.  A tile has as many whole tokens as fit (128 / group; rows that are left over are idle).
//   - K and V come out of pages, a TMA box per page (or per part of one).
//   - What a block does of an item is a piece of its keys (paged_work.cuh); partial rows are joined afterwards.
//   - Rows of V behind an entry's last token are set to zero before they are multiplied (0 * NaN is NaN).
//
//   warps 0-3, 4-7  softmax, epilogue of the two row tiles
//   warp 8          source of pieces; TMA producer of K and V
//   warp 9          MMA issuer
//   warp 10         TMA producer of Q
//   warp 11         passes V on, with zeros in the rows behind an entry's last token
// 8-bit caches, whose codes and scales arrive in a ring of their own (warp 11: scales):
//   warps 12-15     codes times scale -> the tensors' type, into the ring that 16-bit caches load directly
//
// What bounds it: the turns of tensor pipe and softmax, as in fwd_kernel.cuh.  2048 tokens over 16384 keys, 32 query heads over 8,
// head dimension 128, bf16, causal: 560 to 617 us on different GPUs, 835 to 918 TFLOP/s; keys of unequal size, as these
// were, make a new reference of the softmax more often than N(0, 1) does.  8-bit caches: the four converting warps take as long as a
// round (six entries of 1024 to 8192 keys, 1 to 512 new tokens each: 306 us, in 16 bits 219).
#pragma once
#include <cuda.h>

#include <type_traits>

#include "fwd_kernel.cuh"
#include "paged_few_kernel.cuh"
#include "paged_work.cuh"

namespace fmha {

template <int D, int DR, bool kBf16, bool kE4m3>
struct ManyTraits {
  static constexpr int kBoxes = D / 64;
  static constexpr int kBoxBytes = 128 * 128;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kStages = D == 128 ? (kE4m3 ? 3 : 4) : (kE4m3 ? 5 : 8);
  static constexpr int kCodeStages = !kE4m3 ? 0 : D == 128 ? 2 : 4;
  static constexpr int kCodeBytes = 128 * 128;
  static constexpr int kItemStages = 4;
  static constexpr int kThreads = kE4m3 ? 512 : 384;
  // two tiles of Q, ring, codes, one box of output per softmax group
  static constexpr int kSmemBytes = 1024 + (2 + kStages) * kTileBytes + kCodeStages * kCodeBytes + 2 * kBoxBytes;
  static_assert(kSmemBytes <= 230400, "the rest of the 227 KB is for what is declared in the kernel");
  static constexpr uint32_t kIdescQK = umma_idesc_f16(128, 128, 0, 0, kBf16);
  static constexpr uint32_t kIdescPV = umma_idesc_f16(128, DR, 0, 1, kBf16);
  // registers of the launch: 168 (384 threads) or 128 (512); of the groups, whose sum is no more than the launch's
  static constexpr int kRegsLaunch = kE4m3 ? 128 : 168;
  static constexpr int kRegsOther = kE4m3 ? 64 : 88;
  static constexpr int kRegsSoftmax = kE4m3 ? 192 : 208;
  static_assert(kRegsOther <= kRegsLaunch && kRegsSoftmax >= kRegsLaunch &&
                    2 * kRegsSoftmax + (kThreads / 128 - 2) * kRegsOther <= kThreads / 128 * kRegsLaunch,
                "setmaxnreg.dec must not raise, .inc must not lower the launch's registers, nor ask for more than it has");
};

template <int D, int DR, bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(ManyTraits<D, DR, kBf16, kE4m3>::kThreads, 1)
    paged_many_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                      const __grid_constant__ PagedParams p) {
  using T = ManyTraits<D, DR, kBf16, kE4m3>;
  constexpr uint32_t kStages = T::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PagedPiece items[T::kItemStages];
  __shared__ uint64_t bar_item_full[T::kItemStages], bar_item_empty[T::kItemStages];
  __shared__ uint64_t bar_q_full[2];   // Q_t of the current piece has landed
  __shared__ uint64_t bar_q_free[2];   // the last S_t = Q_t K^T of the piece is done: Q_t reusable
  __shared__ uint64_t bar_kv_full[kStages], bar_kv_empty[kStages];
  __shared__ uint64_t bar_s_full[2];     // S_t(j) is there, and so is the result of O_t += of round j - 1
  __shared__ uint64_t bar_p_full[2][2];  // [tile][half]: P_t for 64 keys is there
  __shared__ uint64_t bar_pv_half[2];    // O_t += of the first 64 keys of the round has completed
  __shared__ uint64_t bar_o_full[2];
  __shared__ uint64_t bar_o_read[2];     // the softmax group has O_t in registers: O_t reusable
  __shared__ uint64_t bar_v_raw[kStages];  // (16-bit caches) V has landed; bar_kv_full of its slot: and ends where the entry does
  __shared__ uint64_t bar_code_full[kE4m3 ? T::kCodeStages : 1], bar_code_empty[kE4m3 ? T::kCodeStages : 1];
  __shared__ __align__(16) uint32_t code_scale[kE4m3 ? T::kCodeStages : 1][128];  // the aligned word around a row's byte
  __shared__ uint8_t code_select[kE4m3 ? T::kCodeStages : 1][32];   // which byte of it, two bits for each of four rows
  // The softmax warps' pieces, the one at work and the one whose epilogue is due: their threads have 128 scores in
  // registers and no room for them
  struct Held {
    int slot, z, h, token0, n;
  };
  __shared__ Held held[8][2];
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
  const uint32_t q_smem = smem_base;
  const uint32_t ring_smem = smem_base + 2 * T::kTileBytes;
  const uint32_t ostage_smem = ring_smem + kStages * T::kTileBytes;
  [[maybe_unused]] const uint32_t code_smem = ostage_smem + 2 * T::kBoxBytes;
  const int tokens_per_tile = p.tokens_per_block / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::kItemStages; ++s) {
      mbar_init(smem_u32(&bar_item_full[s]), 1);
      mbar_init(smem_u32(&bar_item_empty[s]), kE4m3 ? 15 : 11);  // MMA, Q, eight softmax, warp 11 (and four converting) warps
    }
    for (uint32_t s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_kv_full[s]), kE4m3 ? 4 : 1);
      mbar_init(smem_u32(&bar_v_raw[s]), 1);
      mbar_init(smem_u32(&bar_kv_empty[s]), 1);
    }
    for (int s = 0; s < T::kCodeStages; ++s) {
      mbar_init(smem_u32(&bar_code_full[s]), 34);  // TMA's thread, a warp's copies of scales, its word on which byte
      mbar_init(smem_u32(&bar_code_empty[s]), 4);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&bar_q_full[t]), 1);
      mbar_init(smem_u32(&bar_q_free[t]), 1);
      mbar_init(smem_u32(&bar_s_full[t]), 1);
      mbar_init(smem_u32(&bar_p_full[t][0]), 4);
      mbar_init(smem_u32(&bar_p_full[t][1]), 4);
      mbar_init(smem_u32(&bar_pv_half[t]), 1);
      mbar_init(smem_u32(&bar_o_full[t]), 1);
      mbar_init(smem_u32(&bar_o_read[t]), 4);
    }
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&tmem_base_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);
  grid_dependents_may_start();  // the joining kernel (see paged_few_kernel.cuh)

  uint32_t item_cnt = 0;
  auto take_item = [&]() -> PagedPiece {
    const uint32_t s = item_cnt % T::kItemStages;
    PagedPiece it;
    if (rolled_wait_warp(smem_u32(&bar_item_full[s]), (item_cnt / T::kItemStages) & 1, &abort_word, 12)) {
      it = items[s];
      it.id = __shfl_sync(0xffffffffu, it.id, 0);
      it.tiles = __shfl_sync(0xffffffffu, it.tiles, 0);
      it.n0 = __shfl_sync(0xffffffffu, it.n0, 0);
      it.n1 = __shfl_sync(0xffffffffu, it.n1, 0);
    } else {
      it.id = -1;
      it.tiles = it.n0 = it.n1 = 0;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&bar_item_empty[s]));
    ++item_cnt;
    return it;
  };

  if (warp >= 8) {
    reg_dealloc<T::kRegsOther>();
    const PagedPages pages{p};
    if (warp == 8) {
      // =========================== source of pieces, K and V producer ===========================
      // A lane per box; lanes 0-15 K's, 16-31 V's (see paged_few_kernel.cuh).
      constexpr int kCols = kE4m3 ? 1 : T::kBoxes;
      constexpr uint32_t kRing = kE4m3 ? T::kCodeStages : T::kStages;
      constexpr uint32_t kBytes = kE4m3 ? T::kCodeBytes : T::kTileBytes;
      const bool is_v = lane >= 16;
      const int sub = (lane & 15) / kCols, box = lane % kCols;
      const bool mine = sub < pages.parts();
      const uint32_t dst = (kE4m3 ? code_smem : ring_smem) + box * T::kBoxBytes + sub * p.box_rows * 128;
      const CUtensorMap* const tm = is_v ? &tm_v : &tm_k;
      uint64_t* const fulls = kE4m3 ? bar_code_full : bar_kv_full;
      uint64_t* const empties = kE4m3 ? bar_code_empty : bar_kv_empty;
      PagedWork work;
      work.start(p, blockIdx.x, gridDim.x);
      bool ok = true;
      uint32_t slot = 0, phase = 1, published = 0;
      auto next_item = [&]() -> PagedPiece {
        PagedPiece it = work.next(p, blockIdx.x);
        const uint32_t s = published % T::kItemStages, round = published / T::kItemStages;
        if (round > 0) ok = rolled_wait_warp(smem_u32(&bar_item_empty[s]), (round - 1) & 1, &abort_word, 13);
        if (ok && lane == 0) {
          items[s] = it;
          mbar_arrive(smem_u32(&bar_item_full[s]));
        }
        __syncwarp();
        ++published;
        return it;
      };
      PagedPiece it = next_item();
      int first_pages = pages.lookup(it, 0);
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
          const uint32_t slot_v = slot + 1 == kRing ? 0 : slot + 1, phase_v = slot + 1 == kRing ? phase ^ 1 : phase;
          ok = ok && rolled_wait_warp(smem_u32(&empties[slot]), phase, &abort_word, 2);
          if (!ok) break;
          // (K is asked for before V's slot is waited for: the round that gives it back may need this K)
          if (lane == 0) mbar_arrive_expect_tx(smem_u32(&fulls[slot]), kBytes);
          __syncwarp();
          if (mine && !is_v) tma_load_4d(dst + slot * kBytes, tm, smem_u32(&fulls[slot]), box * 64, row, it.h, page);
          __syncwarp();
          ok = rolled_wait_warp(smem_u32(&empties[slot_v]), phase_v, &abort_word, 20);
          if (!ok) break;
          const uint32_t full_v = smem_u32(kE4m3 ? &bar_code_full[slot_v] : &bar_v_raw[slot_v]);
          if (lane == 16) mbar_arrive_expect_tx(full_v, kBytes);
          __syncwarp();
          if (mine && is_v) tma_load_4d(dst + slot_v * kBytes, tm, full_v, box * 64, row, it.h, page);
          __syncwarp();
          phase = slot + 2 >= kRing ? phase ^ 1 : phase;
          slot = slot + 2 >= kRing ? slot + 2 - kRing : slot + 2;
        }
        it = after;
        first_pages = first_pages_after;
      }
    } else if (warp == 10) {
      // =========================== Q producer ===========================
      const uint32_t bytes = T::kBoxes * tokens_per_tile * p.group * 128;
      uint32_t phase = 0;  // bit t: Q_t tiles loaded so far, modulo 2
      uint32_t used = 0;   // bit t: Q_t has been loaded before
      bool ok = true;
      while (ok) {
        const PagedPiece it = take_item();
        if (it.id < 0) break;
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          if ((t == 0 ? it.n0 : it.n1) == 0) continue;
          if ((used >> t) & 1) {
            if (!(ok = rolled_wait_warp(smem_u32(&bar_q_free[t]), ((phase >> t) & 1) ^ 1, &abort_word, 1))) break;
          }
          if (elect_one()) {
            const uint32_t bar = smem_u32(&bar_q_full[t]);
            mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
            for (int b = 0; b < T::kBoxes; ++b)
              tma_load_4d(q_smem + t * T::kTileBytes + b * T::kBoxBytes, &tm_q, bar, b * 64, it.h * p.group,
                          it.token0 + t * tokens_per_tile, it.z);
          }
          __syncwarp();
          phase ^= 1u << t;
          used |= 1u << t;
        }
      }
    } else if (warp == 9) {
      // =========================== MMA issuer (converged warp, elected issue) ===================
      const uint32_t q_lo0 = umma_desc_lo(q_smem, kLboKMajor);
      const uint32_t idesc_qk = T::kIdescQK | (p.negate ? kIdescNegateA : 0u);
      uint32_t slot = 0, slot_phase = 0;
      uint32_t phase_q = 0;  // bit t: parity of the next q_full[t]
      uint32_t phase_p = 0;  // bit t: parity of the next p_full[t]
      uint32_t phase_o = 0;  // bit t: parity of the next o_read[t], of the first one already waited for
      uint32_t used_o = 0;   // bit t: O_t has been written before
      auto slot_next = [&]() {
        umma_commit_elect(smem_u32(&bar_kv_empty[slot]));
        if (++slot == kStages) {
          slot = 0;
          slot_phase ^= 1u;
        }
      };
      PagedPiece cur = take_item();
      int j = -1;
      bool ok = true;
      // One pass per round: V(j) of cur (j = -1: none) and K(j+1), which after the last round is K(0) of
      // the piece behind it (nxt).
      while (ok && cur.id >= 0) {
        const int n = cur.tiles;
        if (n == 0) {
          cur = take_item();
          continue;
        }
        const bool last = j == n - 1;
        PagedPiece nxt = cur;
        if (last) nxt = take_item();
        const bool has_k = !last || nxt.tiles > 0;
        const int jk = last ? 0 : j + 1;
        // V(j) sits in the current slot, K(jk) in the one behind it
        const uint32_t v_addr = ring_smem + slot * T::kTileBytes;
        const uint32_t k_slot = j < 0 ? slot : (slot + 1 == kStages ? 0 : slot + 1);
        const uint32_t k_addr = ring_smem + k_slot * T::kTileBytes;
        const uint32_t k_phase = k_slot < slot ? slot_phase ^ 1u : slot_phase;
        if (j >= 0 && !(ok = rolled_wait_warp(smem_u32(&bar_kv_full[slot]), slot_phase, &abort_word, 4))) break;
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          const int nt = t == 0 ? cur.n0 : cur.n1;
          if (j >= 0 && j < nt) {
            // ---- O_t (+)= P_t V(j), as the two halves of P_t come in
            if (j == 0) {
              if ((used_o >> t) & 1) {
                ok = rolled_wait_warp(smem_u32(&bar_o_read[t]), (phase_o >> t) & 1, &abort_word, 7);
                phase_o ^= 1u << t;
              }
              used_o |= 1u << t;
            }
            const uint32_t v_lo = umma_desc_lo(v_addr, kLboMnMajor);
            const uint32_t d = tmem_base + 256 + t * D, a = tmem_base + t * 128;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && rolled_wait_warp(smem_u32(&bar_p_full[t][half]), (phase_p >> t) & 1, &abort_word, 6);
              tc_fence_after();
#pragma unroll
              for (int ks = half * 4; ks < half * 4 + 4; ++ks)
                umma_ts_elect(d, a + ks * 8, v_lo + ((ks * 2048) >> 4), T::kIdescPV, (j > 0 || ks > 0) ? 1u : 0u);
              if (half == 0) umma_commit_elect(smem_u32(&bar_pv_half[t]));
            }
            phase_p ^= 1u << t;
            if (j == nt - 1) umma_commit_elect(smem_u32(&bar_o_full[t]));
            if (!ok) break;
          }
          if (t == 1 && j >= 0) slot_next();
          // ---- S_t = Q_t K^T of the round after, which may be the first of the next piece
          if (t == 0 && has_k && !(ok = rolled_wait_warp(smem_u32(&bar_kv_full[k_slot]), k_phase, &abort_word, 5))) break;
          const int nk = t == 0 ? nxt.n0 : nxt.n1;
          if (jk < nk) {
            if (jk == 0) {
              ok = rolled_wait_warp(smem_u32(&bar_q_full[t]), (phase_q >> t) & 1, &abort_word, 3);
              phase_q ^= 1u << t;
              if (!ok) break;
            }
            tc_fence_after();
            const uint32_t a_lo = q_lo0 + ((t * T::kTileBytes) >> 4);
            const uint32_t b_lo = umma_desc_lo(k_addr, kLboKMajor);
#pragma unroll
            for (int ks = 0; ks < DR / 16; ++ks) {
              const uint32_t off = ((ks >> 2) * T::kBoxBytes + (ks & 3) * 32) >> 4;
              umma_ss_elect(tmem_base + t * 128, a_lo + off, b_lo + off, idesc_qk, ks > 0 ? 1u : 0u);
            }
            umma_commit_elect(smem_u32(&bar_s_full[t]));
            if (jk == nk - 1) umma_commit_elect(smem_u32(&bar_q_free[t]));
          }
        }
        if (!ok) break;
        if (has_k) slot_next();
        ++j;
        if (last) {
          cur = nxt;
          j = has_k ? 0 : -1;
        }
      }
    } else if constexpr (!kE4m3) {
      // =========================== V ends where the entry does ===========================
      // Every V tile is passed on, the last one of an entry with zeros in the rows behind its last token.
      static_assert(kStages % 2 == 0, "V has the odd slots");
      uint32_t at = 1;
      bool ok = true;
      while (ok) {
        const PagedPiece it = take_item();
        if (it.id < 0) break;
#pragma unroll 1
        for (int j = 0; j < it.tiles; ++j, at += 2) {
          const uint32_t slot = at % kStages;
          if (!(ok = rolled_wait_warp(smem_u32(&bar_v_raw[slot]), at / kStages & 1, &abort_word, 17))) break;
          const int rows = it.sk - (it.first + j) * 128;
          if (rows < 128) {
#pragma unroll 1
            for (int i = lane; i < (128 - rows) * 8 * T::kBoxes; i += 32) {
              const int row = rows + i / (8 * T::kBoxes), chunk = i % (8 * T::kBoxes);
              sts128(ring_smem + slot * T::kTileBytes + (chunk >> 3) * T::kBoxBytes + row * 128 + (chunk & 7) * 16, 0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_kv_full[slot]));
        }
      }
    } else {
      if (warp == 11) {
        // =========================== scales ===========================
        uint32_t slot = 0, phase = 1;
        bool ok = true;
        while (ok) {
          const PagedPiece it = take_item();
          if (it.id < 0) break;
          PagedPages::Window window{pages.lookup(it, 0), pages.lookup(it, 1)};
#pragma unroll 1
          for (int j = 0; ok && j < it.tiles; ++j)
            ok = pages.copy_scales(it, window, j, code_scale[0], code_select[0], bar_code_full, bar_code_empty, T::kCodeStages,
                                   slot, phase, &abort_word);
        }
      } else {
        // =========================== codes times scale -> 16 bits in the ring ===========================
        // A warp has 32 rows; lanes and rows as in paged_few_kernel.cuh.  Every value is exact in the type that the cache was
        // written from.
        const int row0 = 32 * (warp - 12);
        const int in8 = lane & 4 ? lane >> 3 ^ 5 : lane >> 3, quarter = lane & 3;
        const uint32_t ld = row0 * 128 + in8 * 128 + ((quarter ^ in8) << 4), st = row0 * 128 + in8 * 128 + ((quarter * 2 ^ in8) << 4);
        uint32_t at = 0, slot = 0, slot_phase = 1, from = 0, from_phase = 0;
        bool ok = true;
        while (ok) {
          const PagedPiece it = take_item();
          if (it.id < 0) break;
#pragma unroll 1
          for (int j = 0; j < 2 * it.tiles; ++j, ++at) {  // K, V, K, V ...
            ok = rolled_wait_warp(smem_u32(&bar_code_full[from]), from_phase, &abort_word, 15) &&
                 rolled_wait_warp(smem_u32(&bar_kv_empty[slot]), slot_phase, &abort_word, 16);
            if (!ok) break;
            const int rows = it.sk - (it.first + (j >> 1)) * 128 - row0;  // of the 32 that exist
            const uint32_t from_smem = code_smem + from * T::kCodeBytes, to_smem = ring_smem + slot * T::kTileBytes;
#pragma unroll 2
            for (int k = 0; k < 4; ++k) {
              const int row = row0 + 8 * k + in8;
              const float s = scale_value(staged_scale(code_scale[0], code_select[0], from, row));
#pragma unroll
              for (int box = 0; box < T::kBoxes; ++box) {
                if (DR == 96 && box == 1 && quarter >= 2) continue;
                const float4 f = lds128(from_smem + k * 1024 + (ld ^ box * 64));
                const uint2 a = e4m3x4_to_16<kBf16>(__float_as_uint(f.x), s), b = e4m3x4_to_16<kBf16>(__float_as_uint(f.y), s);
                const uint2 c = e4m3x4_to_16<kBf16>(__float_as_uint(f.z), s), d = e4m3x4_to_16<kBf16>(__float_as_uint(f.w), s);
                const uint32_t to = to_smem + box * T::kBoxBytes + k * 1024 + st;
                sts128(to, a.x, a.y, b.x, b.y);
                sts128(to ^ 16, c.x, c.y, d.x, d.y);
              }
            }
            // rows behind the entry's end: zeros, whatever the page holds there
            __syncwarp();
            if (lane >= rows) {
              for (int i = 0; i < 8 * T::kBoxes; ++i)
                sts128(to_smem + (i >> 3) * T::kBoxBytes + (row0 + lane) * 128 + (i & 7) * 16, 0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(smem_u32(&bar_kv_full[slot]));
              mbar_arrive(smem_u32(&bar_code_empty[from]));
            }
            if (++slot == kStages) {
              slot = 0;
              slot_phase ^= 1;
            }
            if (++from == (uint32_t)T::kCodeStages) {
              from = 0;
              from_phase ^= 1;
            }
          }
        }
      }
    }
  } else {
    // =========================== softmax / epilogue ===========================
    reg_alloc<T::kRegsSoftmax>();
    const int t = warp >> 2;    // row tile of this warpgroup
    const int quad = warp & 3;  // TMEM lane quadrant of this warp
    const int row_in_tile = quad * 32 + lane;
    const uint32_t lane_addr = uint32_t(quad * 32) << 16;
    const uint32_t tS = tmem_base + lane_addr + t * 128;
    const uint32_t tO = tmem_base + lane_addr + 256 + t * D;
    const uint32_t o_stage = ostage_smem + t * T::kBoxBytes;
    const float c = p.scale_log2;
    const int my_token = row_token(p, row_in_tile);
    const bool my_row = my_token < tokens_per_tile;  // (what does not make a whole token is idle)
    uint32_t phase_s = 0, phase_o = 0;  // parities of the next s_full[t], o_full[t]
    bool stored = false;  // a TMA store of this group may still be reading the staging box

    // The reference is a rounded product.  Taken off in one step (fma), a key's own product is not rounded, and a score of 2^28
    // could come out at 2^4 over itself, or under.  So beyond 2^20 the reference is NaN to the ordinary way, which then sends
    // every round the other way, where a warp that has such a row rounds products first.  (Rounding them always: 3 % of a call.)
    auto one_step = [](float neg) { return fabsf(neg) > 1048576.f ? CUDART_NAN_F : neg; };

    // The epilogue of a piece is done after the first round of the next one (see fwd_kernel.cuh).
    bool pending = false;
    float done_m = 0.f, done_l = 0.f;

    for (uint32_t piece = 0;; ++piece) {
      int id, n, lim;  // lim: last visible column of this row in the round
      {
        const PagedPiece it = take_item();
        id = it.id;
        n = t == 0 ? it.n0 : it.n1;
        if (lane == 0) held[warp][piece & 1] = Held{it.slot, it.z, it.h, it.token0 + t * tokens_per_tile, n};
        __syncwarp();
        lim = id >= 0 && my_row ? paged_last_key(p, it.token0 + t * tokens_per_tile + my_token, it.sq, it.sk) : -1;
        lim -= it.first * 128;
      }
      float m_ref = -CUDART_INF_F;  // reference score of the running softmax (raw, unscaled)
      float neg_mc = 0.f;           // -m_ref * c, 0 while there is no reference, NaN where that is too large for one step
      float l = 0.f;                // running sum of exp2((s - m_ref) * c)

      for (int j = 0; j < n || j == 0; ++j, lim -= 128) {
        if (j < n) {
          rolled_wait(smem_u32(&bar_s_full[t]), phase_s, &abort_word, 9);
          phase_s ^= 1u;
          tc_fence_after();
          uint32_t s[4][32];
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) tmem_ld32(tS + cc * 32, s[cc]);
          tmem_wait_ld();
          if (lim < 127) {
#pragma unroll
            for (int cc = 0; cc < 4; ++cc)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (cc * 32 + i > lim) s[cc][i] = __float_as_uint(-CUDART_INF_F);
          }
          // P of 64 keys -> tensor memory; the reference stays what it was unless an exponential comes out too large
          // (fwd_kernel.cuh has the whole of it)
          auto half_round = [&](auto half_tag) {
            constexpr int half = decltype(half_tag)::value;
            const uint64_t c2 = pack2f(c, c), nm2 = pack2f(neg_mc, neg_mc);
            uint64_t la = pack2f(0.f, 0.f), lb = pack2f(0.f, 0.f);
            uint32_t pk[32];
            float top = 0.f;
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
              const int cc = half * 2 + ch;
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const uint64_t x2 = fma2(pack2(s[cc][i], s[cc][i + 1]), c2, nm2);
                uint64_t p2;
                if (((i >> 1) & 7) < kFwdPolyPairs) {
                  p2 = poly_exp2_pair(x2, top);
                } else {
                  uint32_t x0, x1;
                  unpack2(x2, x0, x1);
                  p2 = pack2f(fast_exp2(__uint_as_float(x0)), fast_exp2(__uint_as_float(x1)));
                }
                if (i & 2) lb = add2(lb, p2); else la = add2(la, p2);
                uint32_t p0, p1;
                unpack2(p2, p0, p1);
                pk[ch * 16 + (i >> 1)] = pack16x2<kBf16>(__uint_as_float(p0), __uint_as_float(p1));
              }
            }
            uint32_t a0, a1;
            unpack2(add2(la, lb), a0, a1);
            float sum = __uint_as_float(a0) + __uint_as_float(a1);
            const bool need = !(sum <= kRescaleSum) || !(top <= kPolyExp2Top) ||
                              (m_ref == -CUDART_INF_F && lim >= half * 64);
            if (!__any_sync(0xffffffffu, need)) {
              tmem_st32(tS + half * 32, pk);
            } else {
              float m_new = m_ref;
#pragma unroll 1
              for (int ch = 0; ch < 2; ++ch) {
                uint32_t x[32];
                tmem_ld32(tS + half * 64 + ch * 32, x);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (half * 64 + ch * 32 + i <= lim) m_new = fmaxf(m_new, __uint_as_float(x[i]));
              }
              if (j > 0) {
                if (half == 1) rolled_wait(smem_u32(&bar_pv_half[t]), phase_s ^ 1u, &abort_word, 11);
                tc_fence_after();
                const float alpha = isinf(m_new) ? 1.f : fast_exp2((m_ref - m_new) * c);
                l *= alpha;
#pragma unroll 1
                for (int cc = 0; cc < DR / 16; ++cc) {
                  uint32_t o[16];
                  tmem_ld16(tO + cc * 16, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                  tmem_st16(tO + cc * 16, o);
                }
              }
              m_ref = m_new;
              const float neg = isinf(m_ref) ? 0.f : -m_ref * c;
              neg_mc = one_step(neg);
              float factor = c;
              if (__any_sync(0xffffffffu, isnan(neg_mc))) {
                factor = 1.f;
#pragma unroll 1
                for (int ch = 0; ch < 4; ++ch) {
                  uint32_t x[16];
                  tmem_ld16(tS + half * 64 + ch * 16, x);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * c);
                  tmem_st16(tS + half * 64 + ch * 16, x);
                }
                tmem_wait_st();
              }
              sum = 0.f;
#pragma unroll 1
              for (int ch = 0; ch < 2; ++ch) {
                uint32_t x[32], h[16];
                tmem_ld32(tS + half * 64 + ch * 32, x);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  const int col = half * 64 + ch * 32 + i;
                  const float e0 = col <= lim ? fast_exp2(fmaf(__uint_as_float(x[i]), factor, neg)) : 0.f;
                  const float e1 = col + 1 <= lim ? fast_exp2(fmaf(__uint_as_float(x[i + 1]), factor, neg)) : 0.f;
                  sum += e0 + e1;
                  h[i >> 1] = pack16x2<kBf16>(e0, e1);
                }
                tmem_st16(tS + half * 32 + ch * 16, h);
              }
            }
            l += sum;
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar_p_full[t][half]));
          };
          if (j == 0) {
            // over all 128 keys, so that half 1 never has to rescale in round 0
            float mx[4];
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
              mx[cc] = fmaxf(__uint_as_float(s[cc][0]), __uint_as_float(s[cc][1]));
#pragma unroll
              for (int i = 2; i < 32; i += 2)
                mx[cc] = max3(mx[cc], __uint_as_float(s[cc][i]), __uint_as_float(s[cc][i + 1]));
            }
            m_ref = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
            neg_mc = one_step(isinf(m_ref) ? 0.f : -m_ref * c);
          }
          half_round(std::integral_constant<int, 0>{});
          half_round(std::integral_constant<int, 1>{});
        }

        if (j > 0 || !pending) continue;
        // ---- epilogue of the piece before: O_t / l -> registers (tensor memory released) -> 16 bit -> staging box -> TMA
        //      store; LSE.  A part of an item leaves fp32 rows instead.
        pending = false;
        const Held& done = held[warp][(piece & 1) ^ 1];
        const int done_n = done.n, done_slot = done.slot;
        const int token = done.token0 + my_token;
        const bool row_here = my_row && token < p.seqlen_q;
        const float inv_l = (done_l == 0.f) ? 0.f : 1.f / done_l;
        if (row_here) {
          const float lse = (done_l == 0.f) ? -CUDART_INF_F : (done_m * c + log2f(done_l)) * 0.6931471805599453f;
          if (done_slot >= 0)
            p.lse_part[(size_t)done_slot * 256 + t * 128 + row_in_tile] = lse;
          else
            p.lse[((size_t)done.z * p.heads_k * p.group + done.h * p.group + row_in_tile - my_token * p.group) * p.seqlen_q + token] = lse;
        }
        if (done_n > 0) {
          rolled_wait(smem_u32(&bar_o_full[t]), phase_o, &abort_word, 10);
          phase_o ^= 1u;
          tc_fence_after();
        }
        if (done_slot >= 0) {
          if (done_n == 0) continue;  // LSE = -inf: the join reads no row
          float* dst = p.o_part + ((size_t)done_slot * 256 + t * 128 + row_in_tile) * DR;
#pragma unroll 1
          for (int cc = 0; cc < DR / 16; ++cc) {
            uint32_t o[16];
            tmem_ld16(tO + cc * 16, o);
            tmem_wait_ld();
            if (row_here) {
#pragma unroll
              for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4*>(dst + cc * 16 + i) =
                    make_float4(__uint_as_float(o[i]) * inv_l, __uint_as_float(o[i + 1]) * inv_l,
                                __uint_as_float(o[i + 2]) * inv_l, __uint_as_float(o[i + 3]) * inv_l);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_o_read[t]));
          continue;
        }
#pragma unroll
        for (int b = 0; b < T::kBoxes; ++b) {
          constexpr int kLast = DR % 64 == 0 ? 2 : 1;  // 32-column parts of the last box
          uint32_t o[2][32];
          if (done_n > 0) {
            tmem_ld32(tO + b * 64, o[0]);
            tmem_ld32(tO + b * 64 + 32, o[1]);  // (head dimension 96: of its last box nothing, unused)
            tmem_wait_ld();
            if (b == T::kBoxes - 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_u32(&bar_o_read[t]));
            }
          } else {  // (left undefined, the registers would be taken for live all around the loop)
#pragma unroll
            for (int i = 0; i < 64; ++i) o[i >> 5][i & 31] = 0u;
          }
          if (row_in_tile == 0 && stored) tma_wait_group_read<0>();  // the box's last store has been read
          named_bar_sync(1 + t, 128);
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {  // 16-byte chunk of this row
            if (b == T::kBoxes - 1 && ch >= kLast * 4) break;
            const uint32_t* w = &o[ch >> 2][(ch & 3) * 8];
            uint32_t h4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              h4[i] = pack16x2<kBf16>(__uint_as_float(w[2 * i]) * inv_l, __uint_as_float(w[2 * i + 1]) * inv_l);
            // (a row without a visible key: P was 0, but 0 times what V holds need not be)
            if (done_l == 0.f) h4[0] = h4[1] = h4[2] = h4[3] = 0u;
            sts128(o_stage + row_in_tile * 128 + ((ch ^ (row_in_tile & 7)) << 4), h4[0], h4[1], h4[2], h4[3]);
          }
          fence_proxy_async_smem();
          named_bar_sync(1 + t, 128);
          if (row_in_tile == 0) {
            tma_store_4d(&tm_o, o_stage, b * 64, done.h * p.group, done.token0, done.z);
            tma_commit_group();
          }
          stored = true;
        }
      }
      if (id < 0) break;
      // (a tile behind the last token there is has nothing to write)
      pending = held[warp][piece & 1].token0 < p.seqlen_q;
      done_m = m_ref;
      done_l = l;
    }
    if (row_in_tile == 0) tma_wait_group<0>();
  }

  // ---- teardown
  tc_fence_before();
  __syncthreads();
  if (abort_word != 0) {
    if (threadIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, 0, abort_word);
    // let copies that may still be in flight land before the shared memory is released
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace fmha
