// What the attention kernels share: which keys a sequence's queries see.
#pragma once

#include "kv_common.cuh"

namespace ivb {

constexpr float kLog2e = 1.4426950408889634f;

// Weights are 2^(s - m + kWeightBits), at most 2^14: as halves they keep their
// 11 bits down to 2^-28 of the row's largest, and sums of them fit as well.
constexpr float kWeightBits = 14.f;

// 2^x (relative error about 2^-22; 0 for -inf).
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

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
