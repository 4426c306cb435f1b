// The paged key/value cache: where a token's row lies, the e4m3 format, and the two kernels that write rows
// and read them back.  The attention over it is in paged_few_kernel.cuh and paged_many_kernel.cuh.
#pragma once
#include <cuda_fp8.h>

#include <type_traits>

#include "aux_kernels.cuh"
#include "ptx.cuh"

namespace fmha {

// One pool (K or V) on the device.  Byte strides; E4M3 pools have a byte of scale per row.
struct PagePool {
  uint8_t* rows;
  uint8_t* scales;
  long long page, row, head;                    // strides of rows, bytes
  long long scale_page, scale_row, scale_head;  // of scales, bytes
};
struct PagedCache {
  PagePool k, v;
  const int32_t* table;
  long long table_stride;
  int num_pages, page_size, max_pages;
  // t / page_size for 0 <= t < 2^30 as a product: both are counted in units of 16, so that n < 2^26; with 2^l the power
  // of two at or above the divisor, m = floor(2^(26 + l) / divisor) + 1 fits 28 bits, and n / divisor is
  // (n * m) >> (26 + l)
  unsigned page_mul, page_shift;
};
__device__ __forceinline__ int cache_page_index(const PagedCache& c, int t) {
  return (int)(((unsigned long long)((unsigned)t >> 4) * c.page_mul) >> c.page_shift);
}
__device__ __forceinline__ int cache_page_row(const PagedCache& c, int t) {
  return t - cache_page_index(c, t) * c.page_size;
}

// tokens an entry can hold at most (fits: checked on the host)
__device__ __forceinline__ int cache_capacity(const PagedCache& c) { return c.max_pages * c.page_size; }

// what the table has for token `t` of entry z: a page, where it is less than num_pages (as an unsigned number)
__device__ __forceinline__ int cache_entry(const PagedCache& c, int z, int t) {
  return __ldg(c.table + z * c.table_stride + cache_page_index(c, t));
}

// 2^(byte - 127), the value of a scale byte (255 is NaN; 0 is 2^-127, a subnormal)
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}
// 2^-e for e in [-126, 126]
__device__ __forceinline__ float exp2_neg_int(int e) { return __uint_as_float((uint32_t)(127 - e) << 23); }

// Two codes (low byte first) as fp16, exactly, and as fp32
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)codes));
  return h;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t codes) {
  const uint32_t h = e4m3x2_to_half2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// fp32 pair -> codes, rounded to nearest even; a NaN is the code of NaN
__device__ __forceinline__ uint32_t float2_to_e4m3x2(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Four codes times 2^(scale byte - 127) -> two words of the 16-bit type.  In the type that the row was written
// from every product is exact; in another it is rounded to nearest.
template <bool kBf16>
__device__ __forceinline__ uint2 e4m3x4_to_16(uint32_t codes, float scale) {
  const float2 a = e4m3x2_to_float2(codes & 0xffffu), b = e4m3x2_to_float2(codes >> 16);
  return make_uint2(pack16x2<kBf16>(a.x * scale, a.y * scale), pack16x2<kBf16>(b.x * scale, b.y * scale));
}

// The exponent of a row's scale from its largest finite magnitude: the least e with top <= 448 * 2^e.
// 448 is 1.75 * 2^8, so it is the exponent of top minus 8, one more where its significand is above 1.75.
template <bool kBf16>
__device__ __forceinline__ int scale_exponent(float top) {
  constexpr int kLow = kBf16 ? -120 : -15, kHigh = kBf16 ? 120 : 8;
  const uint32_t bits = __float_as_uint(top);  // (subnormals, zero among them, end at kLow either way)
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(kLow, min(kHigh, e));
}
// at the highest exponent the codes above 240 would stand for values that the type does not have
template <bool kBf16>
__device__ __forceinline__ float code_limit(int e) {
  return e == (kBf16 ? 120 : 8) ? 240.f : 448.f;
}

struct CacheWriteArgs {
  PagedCache cache;
  const uint8_t *k, *v;                                   // 16-bit rows
  long long k_batch, k_row, k_head, v_batch, v_row, v_head;  // byte strides
  const int32_t *seqlens, *seqused;
  int heads, batch;
  int rows;  // of an entry: seqlen * heads
};

// K's and V's row of a token, 8 elements a thread, to its place in the pools
template <int DR, bool kBf16, bool kE4m3, int kLanes>
__device__ __forceinline__ void write_row(const PagedCache& c, int page, int slot, int h, int sub, bool in_row,
                                          const uint4 (&x)[2]) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const PagePool& pool = n ? c.v : c.k;
    uint8_t* dst = pool.rows + page * pool.page + slot * pool.row + h * pool.head;
    if constexpr (!kE4m3) {
      if (in_row) reinterpret_cast<uint4*>(dst)[sub] = x[n];
    } else {
      using E = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
      // The largest magnitude by its bits, whose order is the values' (infinity and NaN above all others)
      constexpr uint32_t kAbs = 0x7fff7fffu, kInfinity = kBf16 ? 0x7f80u : 0x7c00u;
      const uint32_t m2 = __vmaxu2(__vmaxu2(x[n].x & kAbs, x[n].y & kAbs), __vmaxu2(x[n].z & kAbs, x[n].w & kAbs));
      uint32_t m = max(m2 >> 16, m2 & 0xffffu);
      const uint32_t group = (kLanes == 8 ? 0xffu : 0xffffu) << (threadIdx.x % 32 / kLanes * kLanes);
#pragma unroll
      for (int off = kLanes / 2; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(group, m, off));
      float f[8];
      unpack8<E>(x[n], f);
      if (m >= kInfinity) {  // rare: what is not finite becomes NaN, and the scale is the others'
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!isfinite(f[j])) f[j] = CUDART_NAN_F;
          top = fmaxf(top, fabsf(f[j]));  // (a NaN operand leaves the other)
        }
#pragma unroll
        for (int off = kLanes / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(group, top, off));
        m = kBf16 ? __float_as_uint(top) >> 16 : (uint32_t)__half_as_ushort(__float2half_rn(top));
      }
      const int e = scale_exponent<kBf16>(kBf16 ? __uint_as_float(m << 16) : __half2float(__ushort_as_half((unsigned short)m)));
      const float s = exp2_neg_int(e), most = code_limit<kBf16>(e);
      if (most < 448.f) {  // rare, too
#pragma unroll
        for (int j = 0; j < 8; ++j)  // (minimum and maximum would drop a NaN)
          if (fabsf(f[j] * s) > most) f[j] = copysignf(most / s, f[j]);
      }
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; j += 2) w[j / 4] |= float2_to_e4m3x2(f[j] * s, f[j + 1] * s) << (j % 4 * 8);
      if (in_row) reinterpret_cast<uint2*>(dst)[sub] = make_uint2(w[0], w[1]);
      if (sub == 0)
        pool.scales[page * pool.scale_page + slot * pool.scale_row + h * pool.scale_head] = (uint8_t)(e + 127);
    }
  }
}

// Rows that a thread has: what bounds both kernels is the chain of loads from an entry's length by its table to the row's
// place, and then, in 8 bits, the conversion (ALU 47 and 63 % busy); more rows side by side hide the chain, more registers
// leave room for fewer threads.  On the GPU alone, 1 / 2 / 4 rows, us: four chunks of up to 4096 tokens into an 8-bit cache (50 MB)
// 18.5 / 17.3 / 17.7, three of 1000 in 16 bits (37 MB) 8.0 / 7.5 / 7.5; eight conversations of 1024 to 8192 tokens out of an
// 8-bit cache (345 MB) 78.9 / 66.1 / 59.3 (5.8 TB/s, 89 % of a copy's rate), five of 252 to 2016 in 16 bits (65 MB) 11.7 / 12.1 /
// 12.3.  (The magnitudes by their bits instead of as numbers: 22.5 -> 20.0 with the launch.)
constexpr int kWriteRows = 2, kReadRows = 4;

// New rows into their pages.  kLanes threads a row (8 elements each), K and V of the same row by the same threads, so
// that the place is worked out once.
template <int DR, bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheWriteArgs a) {
  constexpr int kLanes = DR == 64 ? 8 : 16;  // (96: four of sixteen idle)
  constexpr int kStep = 256 / kLanes;
  const int r0 = (int)(blockIdx.x * (kStep * kWriteRows) + threadIdx.x / kLanes), sub = threadIdx.x % kLanes;
  const bool in_row = sub * 8 < DR;
#pragma unroll 1
  for (int z = blockIdx.y; z < a.batch; z += gridDim.y) {
    const int held = __ldg(a.seqlens + z), used = a.seqused == nullptr ? 0x7fffffff : __ldg(a.seqused + z);
    uint4 x[kWriteRows][2];
    int page[kWriteRows];
#pragma unroll
    for (int k = 0; k < kWriteRows; ++k) {
      const int r = r0 + k * kStep, i = (int)((unsigned)r / (unsigned)a.heads), h = r - i * a.heads;
      const long long t = (long long)held + i;
      x[k][0] = x[k][1] = make_uint4(0, 0, 0, 0);
      page[k] = -1;
      if (r < a.rows && i < used && t >= 0 && t < cache_capacity(a.cache)) {
        page[k] = cache_entry(a.cache, z, (int)t);
        if (in_row) {
          x[k][0] = __ldg(reinterpret_cast<const uint4*>(a.k + z * a.k_batch + i * a.k_row + h * a.k_head) + sub);
          x[k][1] = __ldg(reinterpret_cast<const uint4*>(a.v + z * a.v_batch + i * a.v_row + h * a.v_head) + sub);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kWriteRows; ++k) {
      if ((unsigned)page[k] >= (unsigned)a.cache.num_pages) continue;  // (the threads of a row share a shuffle, and skip it together)
      const int r = r0 + k * kStep, i = (int)((unsigned)r / (unsigned)a.heads), h = r - i * a.heads;
      write_row<DR, kBf16, kE4m3, kLanes>(a.cache, page[k], cache_page_row(a.cache, held + i), h, sub, in_row, x[k]);
    }
  }
}

struct CacheReadArgs {
  PagedCache cache;
  uint8_t *k, *v;
  long long k_batch, k_row, k_head, v_batch, v_row, v_head;  // byte strides
  const int32_t* seqused_k;
  int heads, batch;
  int rows;  // of an entry: seqlen * heads
};

// Rows out of their pages, zeros behind an entry's end.  A thread has 8 elements of a row of K and of V.
template <int DR, bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheReadArgs a) {
  constexpr unsigned kLanes = DR / 8, kBlockRows = 256 / kLanes;  // (96: 4 of 256 threads idle)
  const int in_block = (int)(threadIdx.x / kLanes), sub = (int)(threadIdx.x % kLanes);
  if (in_block >= (int)kBlockRows) return;
  const int r0 = (int)(blockIdx.x * (kBlockRows * kReadRows)) + in_block;
#pragma unroll 1
  for (int z = blockIdx.y; z < a.batch; z += gridDim.y) {
    const int sk = min(__ldg(a.seqused_k + z), cache_capacity(a.cache));
    int page[kReadRows];
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
      const int r = r0 + k * (int)kBlockRows, t = (int)((unsigned)r / (unsigned)a.heads);
      page[k] = -1;
      if (r < a.rows && t < sk) page[k] = cache_entry(a.cache, z, t);
    }
    uint4 x[kReadRows][2] = {};
    uint32_t scale[kReadRows][2] = {};
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
      if ((unsigned)page[k] >= (unsigned)a.cache.num_pages) continue;
      const int r = r0 + k * (int)kBlockRows, t = (int)((unsigned)r / (unsigned)a.heads), h = r - t * a.heads;
      const int slot = cache_page_row(a.cache, t);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const PagePool& pool = n ? a.cache.v : a.cache.k;
        const uint8_t* src = pool.rows + page[k] * pool.page + slot * pool.row + h * pool.head;
        if constexpr (kE4m3) {
          const uint2 codes = __ldg(reinterpret_cast<const uint2*>(src) + sub);
          x[k][n].x = codes.x;
          x[k][n].y = codes.y;
          scale[k][n] = __ldg(pool.scales + page[k] * pool.scale_page + slot * pool.scale_row + h * pool.scale_head);
        } else {
          x[k][n] = __ldg(reinterpret_cast<const uint4*>(src) + sub);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
      const int r = r0 + k * (int)kBlockRows, t = (int)((unsigned)r / (unsigned)a.heads), h = r - t * a.heads;
      if (r >= a.rows) break;
      if constexpr (kE4m3) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float s = scale_value(scale[k][n]);
          const uint2 lo = e4m3x4_to_16<kBf16>(x[k][n].x, s), hi = e4m3x4_to_16<kBf16>(x[k][n].y, s);
          x[k][n] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      }
      // (written once, read by somebody else: not to push the cache's lines out)
      __stcs(reinterpret_cast<uint4*>(a.k + z * a.k_batch + t * a.k_row + h * a.k_head) + sub, x[k][0]);
      __stcs(reinterpret_cast<uint4*>(a.v + z * a.v_batch + t * a.v_row + h * a.v_head) + sub, x[k][1]);
    }
  }
}

}  // namespace fmha
