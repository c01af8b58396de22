// What the attention kernels share: which keys a sequence's queries see.
#pragma once

#include "kv_common.cuh"

namespace ivb {

constexpr float kLog2e = 1.4426950408889634f;

// 2^x (relative error about 2^-22; 0 for -inf).
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float log2_of(float x) {  // (-inf for 0; exact for powers of two)
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's reference m is the largest s + lv of the keys that it sees, where lv is
// log2 (vs / vref): the largest weight times value scale, and not the largest
// weight, sets what the halves can hold.  m lags behind by up to a slack; a row's
// largest weight times value scale is from 2^bits to 2^(bits + slack) as a half
// (bits, slack: 12, 3.5 and 8, 7.5 in the two kernels; halves end at 2^16), so that
// halves keep their 11 bits down to 2^-26 and 2^-22 of it.  vref, the largest value scale so far, is
// common to the rows of an item; where it grows m is lowered with it, so that
// keys that are hidden from a row do not count for it.  s - m can be as large as
// -lv then, so sums of 2^(s - m) are kept in units of 2^-kSumBits.
constexpr float kSumBits = 64.f;
constexpr float kFarBelow = -150.f;  // lv is taken as at least this
// l 2^d, d far below the range of f32's exponents or not.
__device__ __forceinline__ float kv_scaled(float l, float d) {
  const float half = fast_exp2(0.5f * d);
  return l * half * half;
}
// How far a row's m may be lowered when its sum is l: until the sum is 2^96.
__device__ __forceinline__ float kv_room(float l) {
  return fmaxf(0.f, (float)(96 + 127 - (int)(__float_as_uint(l) >> 23)));
}
// vref / (l 2^kSumBits) as a product that stays inside f32's range; 0 for no sum (a NaN sum stays NaN).
__device__ __forceinline__ float2 kv_norm(float vref, float l) {
  if (l == 0.f) return make_float2(0.f, 0.f);
  return l < 1.f ? make_float2(vref / (l * 0x1p64f), 1.f) : make_float2(vref / l, 0x1p-64f);
}

// What a part's accumulators count beside the largest: t = m + log2 vref of either.
__device__ __forceinline__ float kv_share(float t, float top) { return t == -INFINITY ? 0.f : fast_exp2(t - top); }

// One sequence of a call: its packed tokens, cache length, and the key blocks
// (of kKvBlock keys) that its queries see: `sink_blocks` from 0, then the rest
// from `first_block`.  blocks is at least 1 where there are queries, so that
// rows without keys are visited and written.
struct KvSpan {
  int first;          // packed token
  int n, len;         // new tokens; tokens in the cache, those included
  int sink_blocks, first_block, blocks;
  __device__ __forceinline__ int block(int i) const { return i < sink_blocks ? i : i - sink_blocks + first_block; }
};

__device__ __forceinline__ KvSpan kv_span(const KvAttend &a, int b) {
  KvSpan s;
  const int o = a.seqs.offsets[b], e = a.seqs.offsets[b + 1];
  s.first = o;
  s.len = a.seqs.at[b];
  s.n = e - o;
  s.sink_blocks = s.first_block = s.blocks = 0;
  if (o < 0 || e < o || e > a.seqs.tokens || s.n > a.max_new || s.len < 0 ||
      s.len > (long long)a.seqs.pps * a.cache.page) {
    kv_flag(a.status, kStatusKvSeqs);
    s.n = 0;
    return s;
  }
  if (s.n == 0) return s;
  const int all = (s.len + kKvBlock - 1) / kKvBlock;
  if (a.window > 0) {
    // the first query's first window key; blocks before it only for the sinks
    const long long lo = (long long)s.len - s.n - a.window + 1;
    s.first_block = lo > 0 ? (int)(lo / kKvBlock) : 0;
    s.sink_blocks = min(s.first_block, a.sinks / kKvBlock + (a.sinks % kKvBlock != 0));
  }
  s.blocks = max(1, s.sink_blocks + all - s.first_block);
  return s;
}

// Whether the query at position p sees key j (which is in the cache).
__device__ __forceinline__ bool kv_sees(const KvAttend &a, int p, int j) {
  return j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
}

}  // namespace ivb
