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
  int heads, seqlen;
  long long rows;  // batch * seqlen * heads
};

// New rows into their pages.  kLanes threads a row (8 elements each), K and V of the same row by the same threads, so
// that two loads are in flight and the place is worked out once.  What bounds it is HBM for chunks of a prompt and
// the launch for single tokens.
template <int DR, bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(256) cache_write_kernel(const CacheWriteArgs a) {
  constexpr int kLanes = DR == 64 ? 8 : 16;  // (96: four of sixteen idle)
  const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / kLanes;
  const int sub = threadIdx.x % kLanes;
  if (r >= a.rows) return;  // (rows of a warp share a shuffle below: masked by groups of kLanes, which return together)
  const int h = (int)(r % a.heads);
  const long long zi = r / a.heads;
  const int z = (int)(zi / a.seqlen), i = (int)(zi % a.seqlen);
  if (a.seqused != nullptr && i >= __ldg(a.seqused + z)) return;
  const long long t = (long long)__ldg(a.seqlens + z) + i;
  if (t < 0 || t >= cache_capacity(a.cache)) return;
  const int page = cache_page(a.cache, z, (int)t);
  if (page < 0) return;
  const int slot = cache_page_row(a.cache, (int)t);
  const bool in_row = sub * 8 < DR;
  uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (in_row) {
    x[0] = __ldg(reinterpret_cast<const uint4*>(a.k + z * a.k_batch + i * a.k_row + h * a.k_head) + sub);
    x[1] = __ldg(reinterpret_cast<const uint4*>(a.v + z * a.v_batch + i * a.v_row + h * a.v_head) + sub);
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const PagePool& pool = n ? a.cache.v : a.cache.k;
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

struct CacheReadArgs {
  PagedCache cache;
  uint8_t *k, *v;
  long long k_batch, k_row, k_head, v_batch, v_row, v_head;  // byte strides
  const int32_t* seqused_k;
  int heads, seqlen;
  long long rows;  // batch * seqlen * heads
};

// Rows out of their pages, zeros behind an entry's end.
template <int DR, bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheReadArgs a) {
  constexpr int kLanes = DR / 8;
  const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long r = n / kLanes;
  const int sub = (int)(n % kLanes);
  if (r >= a.rows) return;
  const int h = (int)(r % a.heads);
  const long long zi = r / a.heads;
  const int z = (int)(zi / a.seqlen), t = (int)(zi % a.seqlen);
  const int sk = min(__ldg(a.seqused_k + z), cache_capacity(a.cache));
  const int page = t < sk ? cache_page(a.cache, z, t) : -1;
  uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (page >= 0) {
    const int slot = cache_page_row(a.cache, t);
    const uint8_t* src[2];
    float s[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const PagePool& pool = n ? a.cache.v : a.cache.k;
      src[n] = pool.rows + page * pool.page + slot * pool.row + h * pool.head;
      if constexpr (kE4m3)
        s[n] = scale_value(__ldg(pool.scales + page * pool.scale_page + slot * pool.scale_row + h * pool.scale_head));
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if constexpr (kE4m3) {
        const uint2 codes = __ldg(reinterpret_cast<const uint2*>(src[n]) + sub);
        const uint2 lo = e4m3x4_to_16<kBf16>(codes.x, s[n]), hi = e4m3x4_to_16<kBf16>(codes.y, s[n]);
        x[n] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      } else {
        x[n] = __ldg(reinterpret_cast<const uint4*>(src[n]) + sub);
      }
    }
  }
  reinterpret_cast<uint4*>(a.k + z * a.k_batch + t * a.k_row + h * a.k_head)[sub] = x[0];
  reinterpret_cast<uint4*>(a.v + z * a.v_batch + t * a.v_row + h * a.v_head)[sub] = x[1];
}

}  // namespace fmha
