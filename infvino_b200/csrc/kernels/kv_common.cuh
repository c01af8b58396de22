// Device helpers of the language-model kernels: 16-bit rows and the paged cache.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "kv.cuh"

namespace ivb {

// Status words of these kernels (KernelStatus continues).
enum KvStatus : int {
  kStatusKvPage = 16,      // a page number outside the cache
  kStatusKvSeqs = 17,      // offsets, starts or lengths that do not fit
  kStatusKvPosition = 18,  // a position outside the rotary table
};

__device__ __forceinline__ void kv_flag(int *status, int code) { atomicCAS(status, 0, code); }

// Two 16-bit values as f32 and back (round to nearest even).
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  if (BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Eight consecutive 16-bit elements; element by element (a small loop, so that
// every use does not carry eight copies) where the row is not on 16 bytes.
template <bool L2 = false>  // (past the SM's own cache)
__device__ __forceinline__ uint4 load8(const uint16_t *p, bool vec) {
  if (vec) return L2 ? __ldcg(reinterpret_cast<const uint4 *>(p)) : *reinterpret_cast<const uint4 *>(p);
  uint64_t lo = 0, hi = 0;
#pragma unroll 1
  for (int i = 7; i >= 0; --i) {
    hi = (hi << 16) | (lo >> 48);
    lo = (lo << 16) | (L2 ? __ldcg(p + i) : p[i]);
  }
  return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}
__device__ __forceinline__ void store8(uint16_t *p, uint4 u, bool vec) {
  if (vec) {
    *reinterpret_cast<uint4 *>(p) = u;
    return;
  }
  uint64_t lo = u.x | ((uint64_t)u.y << 32), hi = u.z | ((uint64_t)u.w << 32);
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    p[i] = (uint16_t)lo;
    lo = (lo >> 16) | (hi << 48);
    hi >>= 16;
  }
}
template <bool BF16>
__device__ __forceinline__ void unpack8(uint4 u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = unpack2<BF16>(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]),
                    pack2<BF16>(f[6], f[7]));
}

// Offset in codes of slot `slot` of a page and head.  64 bits: a cache passes 2^31 bytes.
__device__ __forceinline__ long long kv_code_at(const KvCache &c, int page, int head, int slot) {
  return (((long long)page * c.heads + head) * c.page + slot) * c.dim;
}
__device__ __forceinline__ long long kv_scale_at(const KvCache &c, int page, int head, int slot) {
  return ((long long)page * c.heads + head) * (c.page / kKvBlock) + slot / kKvBlock;
}

// The page of position `pos` of sequence `b`, or -1 (status set) if the table has none for it.
__device__ __forceinline__ int kv_page_of(const KvCache &c, const KvSeqs &s, int b, int pos, int *status) {
  const int i = pos / c.page;
  if (pos < 0 || i >= s.pps) {
    kv_flag(status, kStatusKvSeqs);
    return -1;
  }
  const int page = s.pages[(long long)b * s.pps + i];
  if ((unsigned)page >= (unsigned long long)c.pages) {
    kv_flag(status, kStatusKvPage);
    return -1;
  }
  return page;
}

__device__ __forceinline__ int fast_div(int n, FastDiv f) {  // (0 <= n < 2^31)
  return (int)(((uint64_t)(uint32_t)n * f.m) >> (31u + f.s));
}

// How many sequences end at or before packed token t (= the sequence t is in),
// counted by the whole block: one round of loads instead of a search's chain.
__device__ __forceinline__ int kv_seq_of(const KvSeqs &s, long long t) {
  int n = 0;
  for (int b0 = 0; b0 < s.batch; b0 += blockDim.x) {
    const int b = b0 + (int)threadIdx.x;
    n += __syncthreads_count(b < s.batch && s.offsets[b + 1] <= t);
  }
  return n;
}

}  // namespace ivb
