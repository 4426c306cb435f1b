// Attention over the paged cache, the plain way: a warp per query row, 32 keys at a time, one per lane.
#pragma once
#include "cache_kernels.cuh"

namespace fmha {

struct PagedSimpleArgs {
  PagedCache cache;
  const uint8_t* q;
  uint8_t* o;
  float* lse;
  long long q_batch, q_row, q_head, o_batch, o_row, o_head;  // byte strides
  const int32_t *seqused_k, *seqused_q;
  int heads_q, group, seqlen_q, causal;
  float scale;
  long long rows;  // batch * seqlen_q * heads_q
};

template <int DR, bool kBf16, bool kE4m3>
__device__ __forceinline__ void load8(const PagePool& pool, int page, int slot, int h, int c, float (&f)[8]) {
  using E = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
  const uint8_t* src = pool.rows + page * pool.page + slot * pool.row + h * pool.head;
  uint4 x;
  if constexpr (kE4m3) {
    const float s = scale_value(pool.scales[page * pool.scale_page + slot * pool.scale_row + h * pool.scale_head]);
    const uint2 codes = reinterpret_cast<const uint2*>(src)[c];
    const uint2 lo = e4m3x4_to_16<kBf16>(codes.x, s), hi = e4m3x4_to_16<kBf16>(codes.y, s);
    x = make_uint4(lo.x, lo.y, hi.x, hi.y);
  } else {
    x = reinterpret_cast<const uint4*>(src)[c];
  }
  unpack8<E>(x, f);
}

template <int DR, bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(128) paged_simple_kernel(const PagedSimpleArgs a) {
  using E = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
  __shared__ float sq_[4][DR];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long r = (long long)blockIdx.x * 4 + warp;
  if (r >= a.rows) return;
  const int hq = (int)(r % a.heads_q);
  const long long zi = r / a.heads_q;
  const int z = (int)(zi / a.seqlen_q), i = (int)(zi % a.seqlen_q);
  const int sk = max(0, min(a.seqused_k[z], cache_capacity(a.cache)));
  const int sq = a.seqused_q ? max(0, min(a.seqused_q[z], a.seqlen_q)) : a.seqlen_q;
  const int h = hq / a.group;
  const uint8_t* q = a.q + z * a.q_batch + i * a.q_row + hq * a.q_head;
  if (lane < DR / 8) {
    float f[8];
    unpack8<E>(reinterpret_cast<const uint4*>(q)[lane], f);
    for (int j = 0; j < 8; ++j) sq_[warp][lane * 8 + j] = f[j] * a.scale;
  }
  __syncwarp();
  const int end = i >= sq ? 0 : a.causal ? min(sk, sk - sq + i + 1) : sk;
  float m = -CUDART_INF_F, l = 0.f, o[8] = {};
  for (int k0 = 0; k0 < end; k0 += 32) {
    const int key = k0 + lane;
    float s = -CUDART_INF_F;
    if (key < end) {
      const int page = cache_page(a.cache, z, key);
      s = 0.f;
      if (page >= 0)
        for (int c = 0; c < DR / 8; ++c) {
          float f[8];
          load8<DR, kBf16, kE4m3>(a.cache.k, page, key % a.cache.page_size, h, c, f);
          for (int j = 0; j < 8; ++j) s += f[j] * sq_[warp][c * 8 + j];
        }
    }
    float top = s;
    for (int off = 16; off > 0; off >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float m_new = max_nan(m, top), base = m_new == -CUDART_INF_F ? 0.f : m_new;
    const float alpha = expf(m - base), p = expf(s - base);
    float sum = p;
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    l = l * alpha + sum;
    for (int j = 0; j < 8; ++j) o[j] *= alpha;
    for (int kk = 0; kk < 32 && k0 + kk < end; ++kk) {
      const float pk = __shfl_sync(0xffffffffu, p, kk);
      const int page = cache_page(a.cache, z, k0 + kk);
      if (page >= 0 && lane < DR / 8) {
        float f[8];
        load8<DR, kBf16, kE4m3>(a.cache.v, page, (k0 + kk) % a.cache.page_size, h, lane, f);
        for (int j = 0; j < 8; ++j) o[j] += pk * f[j];
      }
    }
    m = m_new;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane < DR / 8) {
    for (int j = 0; j < 8; ++j) o[j] *= inv;
    reinterpret_cast<uint4*>(a.o + z * a.o_batch + i * a.o_row + hq * a.o_head)[lane] = pack8<E>(o);
  }
  if (lane == 0)
    a.lse[((long long)z * a.heads_q + hq) * a.seqlen_q + i] = l == 0.f ? -CUDART_INF_F : m + logf(l);
}

}  // namespace fmha
