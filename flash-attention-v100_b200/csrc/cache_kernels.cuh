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

// what the table has for token `t` of entry z; its page, -1 where the table names none
__device__ __forceinline__ int cache_entry(const PagedCache& c, int z, int t) {
  return __ldg(c.table + z * c.table_stride + cache_page_index(c, t));
}
__device__ __forceinline__ int cache_page(const PagedCache& c, int z, int t) {
  const int page = cache_entry(c, z, t);
  return (unsigned)page < (unsigned)c.num_pages ? page : -1;
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
      float f[8];
      unpack8<E>(x[n], f);
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!isfinite(f[j])) f[j] = CUDART_NAN_F;
        top = fmaxf(top, fabsf(f[j]));  // (a NaN operand leaves the other)
      }
      const uint32_t group = (kLanes == 8 ? 0xffu : 0xffffu) << (threadIdx.x % 32 / kLanes * kLanes);
#pragma unroll
      for (int off = kLanes / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(group, top, off));
      const int e = scale_exponent<kBf16>(top);
      const float s = exp2_neg_int(e), most = code_limit<kBf16>(e);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        // minimum and maximum would drop a NaN: the limits are applied to what is one of the numbers
        float lo = f[j] * s, hi = f[j + 1] * s;
        lo = fabsf(lo) > most ? copysignf(most, lo) : lo;
        hi = fabsf(hi) > most ? copysignf(most, hi) : hi;
        w[j / 4] |= float2_to_e4m3x2(lo, hi) << (j % 4 * 8);
      }
      if (in_row) reinterpret_cast<uint2*>(dst)[sub] = make_uint2(w[0], w[1]);
      if (sub == 0)
        pool.scales[page * pool.scale_page + slot * pool.scale_row + h * pool.scale_head] = (uint8_t)(e + 127);
    }
  }
}

// New rows into their pages.  kLanes threads a row (8 elements each), K and V of the same row by the same threads, so
// that two loads are in flight and the place is worked out once.  What bounds it is HBM for chunks of a prompt and
// the launch for single tokens.
template <int DR, bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheWriteArgs a) {
  constexpr int kLanes = DR == 64 ? 8 : 16;  // (96: four of sixteen idle)
  const int r = (int)(blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes), sub = threadIdx.x % kLanes;
  if (r >= a.rows) return;  // (the threads of a row share a shuffle below, and return together)
  const int i = (int)((unsigned)r / (unsigned)a.heads), h = r - i * a.heads;
  const bool in_row = sub * 8 < DR;
#pragma unroll 1
  for (int z = blockIdx.y; z < a.batch; z += gridDim.y) {
    const long long t = (long long)__ldg(a.seqlens + z) + i;
    if (a.seqused != nullptr && i >= __ldg(a.seqused + z)) continue;
    if (t < 0 || t >= cache_capacity(a.cache)) continue;
    // (the row is asked for before its place is known)
    uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (in_row) {
      x[0] = __ldg(reinterpret_cast<const uint4*>(a.k + z * a.k_batch + i * a.k_row + h * a.k_head) + sub);
      x[1] = __ldg(reinterpret_cast<const uint4*>(a.v + z * a.v_batch + i * a.v_row + h * a.v_head) + sub);
    }
    const int page = cache_page(a.cache, z, (int)t);
    if (page < 0) continue;
    const int slot = cache_page_row(a.cache, (int)t);
    write_row<DR, kBf16, kE4m3, kLanes>(a.cache, page, slot, h, sub, in_row, x);
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

// Rows out of their pages, zeros behind an entry's end.  A thread has 16 elements of a row of K and of V.
template <int DR, bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheReadArgs a) {
  constexpr int kLanes = DR / 16;
  const unsigned n = blockIdx.x * 256 + threadIdx.x;
  const int r = (int)(n / kLanes), sub = (int)(n % kLanes);
  if (r >= a.rows) return;
  const int t = (int)((unsigned)r / (unsigned)a.heads), h = r - t * a.heads;
#pragma unroll 1
  for (int z = blockIdx.y; z < a.batch; z += gridDim.y) {
    const int sk = min(__ldg(a.seqused_k + z), cache_capacity(a.cache));
    const int page = t < sk ? cache_page(a.cache, z, t) : -1;
    uint4 x[2][2] = {};
    if (page >= 0) {
      const int slot = cache_page_row(a.cache, t);
      uint32_t scale[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const PagePool& pool = n ? a.cache.v : a.cache.k;
        const uint4* src = reinterpret_cast<const uint4*>(pool.rows + page * pool.page + slot * pool.row + h * pool.head);
        if constexpr (kE4m3) {
          x[n][0] = __ldg(src + sub);
          scale[n] = __ldg(pool.scales + page * pool.scale_page + slot * pool.scale_row + h * pool.scale_head);
        } else {
          x[n][0] = __ldg(src + 2 * sub);
          x[n][1] = __ldg(src + 2 * sub + 1);
        }
      }
      if constexpr (kE4m3) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float s = scale_value(scale[n]);
          const uint4 codes = x[n][0];
          const uint2 w0 = e4m3x4_to_16<kBf16>(codes.x, s), w1 = e4m3x4_to_16<kBf16>(codes.y, s);
          const uint2 w2 = e4m3x4_to_16<kBf16>(codes.z, s), w3 = e4m3x4_to_16<kBf16>(codes.w, s);
          x[n][0] = make_uint4(w0.x, w0.y, w1.x, w1.y);
          x[n][1] = make_uint4(w2.x, w2.y, w3.x, w3.y);
        }
      }
    }
    // (written once, read by somebody else: not to push the cache's lines out)
    uint4* const k = reinterpret_cast<uint4*>(a.k + z * a.k_batch + t * a.k_row + h * a.k_head) + 2 * sub;
    uint4* const v = reinterpret_cast<uint4*>(a.v + z * a.v_batch + t * a.v_row + h * a.v_head) + 2 * sub;
    __stcs(k, x[0][0]);
    __stcs(k + 1, x[0][1]);
    __stcs(v, x[1][0]);
    __stcs(v + 1, x[1][1]);
  }
}

}  // namespace fmha
