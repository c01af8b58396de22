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

// What a launch works on: whole sequences; or, of sequences in groups with a common
// beginning, first the groups (all queries of a group over the beginning, whose
// results wait in the scratch: kv_part below), then each sequence's own keys, with
// those results joined in.
enum KvMode { kWhole = 0, kBegin = 1, kRest = 2 };

// The first sequence of a group, the one behind its last, and how many tokens are common; false (status set) if that does not fit.
__device__ __forceinline__ bool kv_group(const KvAttend &a, int g, int &s0, int &s1, int &len) {
  s0 = a.first[g], s1 = a.first[g + 1], len = a.shared[g];
  const bool fits = s0 >= 0 && s1 >= s0 && s1 <= a.sequences && len >= 0 && len <= (long long)a.seqs.pps * a.cache.page &&
                    len == fast_div(len, a.by_page) * a.cache.page;
  if (!fits) kv_flag(a.status, kStatusKvSeqs);
  return fits;
}

// Sequence b (kBegin: group b, as a sequence of all its queries over its first sequence's pages).
template <int MODE>
__device__ __forceinline__ KvSpan kv_span(const KvAttend &a, int b) {
  KvSpan s;
  s.sink_blocks = s.first_block = s.blocks = 0;
  if (MODE == kBegin) {
    int s0, s1, len;
    s.first = s.n = s.len = 0;
    if (!kv_group(a, b, s0, s1, len) || s0 == s1 || len == 0) return s;
    const int o = a.seqs.offsets[s0], e = a.seqs.offsets[s1];
    if (o < 0 || e < o || e > a.seqs.tokens) {
      kv_flag(a.status, kStatusKvSeqs);
      return s;
    }
    s.first = o;
    s.n = e - o;
    s.len = len;
    s.blocks = max(1, len / kKvBlock);
    return s;
  }
  const int o = a.seqs.offsets[b], e = a.seqs.offsets[b + 1];
  s.first = o;
  s.len = a.seqs.at[b];
  s.n = e - o;
  if (o < 0 || e < o || e > a.seqs.tokens || s.n > a.max_new || s.len < 0 ||
      s.len > (long long)a.seqs.pps * a.cache.page) {
    kv_flag(a.status, kStatusKvSeqs);
    s.n = 0;
    return s;
  }
  if (s.n == 0) return s;
  const int all = (s.len + kKvBlock - 1) / kKvBlock;
  if (MODE == kRest) {
    int g = 0, end = a.groups;  // the last group that begins at or before b
    while (end - g > 1) {
      const int mid = (g + end) / 2;
      if (a.first[mid] <= b)
        g = mid;
      else
        end = mid;
    }
    int s0, s1, len;
    if (!kv_group(a, g, s0, s1, len) || b < s0 || b >= s1 || s.len - s.n < len) {
      kv_flag(a.status, kStatusKvSeqs);
      s.n = 0;
      return s;
    }
    s.first_block = len / kKvBlock;
  } else if (a.window > 0) {
    // the first query's first window key; blocks before it only for the sinks
    const long long lo = (long long)s.len - s.n - a.window + 1;
    s.first_block = lo > 0 ? (int)(lo / kKvBlock) : 0;
    s.sink_blocks = min(s.first_block, a.sinks / kKvBlock + (a.sinks % kKvBlock != 0));
  }
  s.blocks = max(1, s.sink_blocks + all - s.first_block);
  return s;
}

// The row of the page table that b's pages are in.
template <int MODE>
__device__ __forceinline__ long long kv_page_row(const KvAttend &a, int b) {
  return (long long)(MODE == kBegin ? a.first[b] : b) * a.seqs.pps;
}
// The last key that query i of s sees.
template <int MODE>
__device__ __forceinline__ int kv_position(const KvSpan &s, int i) {
  return MODE == kBegin ? s.len - 1 : s.len - s.n + i;
}

// Whether the query at position p sees key j (which is in the cache).
__device__ __forceinline__ bool kv_sees(const KvAttend &a, int p, int j) {
  return j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
}

// ---- results over a common beginning, for every packed token and head: DIM floats
// each, then each one's m and l (the sum of weights 2^(s - m), in units of
// 2^(kPartBits - kSumBits)).  An item that was cut over CTAs has l = -1: its first
// words say which CTAs' slots have its parts, and its row in them.
constexpr float kPartBits = 12.f;
struct PromptSlot {  // one M tile of a cut item: accumulators [DIM / 4][128 rows][4] in units of 2^m vref, row's m and sum
  float acc[128 * 128];
  float m[128], l[128];
  float vref;
  float pad[31];
};
constexpr float kPromptToPart = 16.f;  // (sums of the prompt kernel are in units of 2^(8 - kSumBits))

__device__ __forceinline__ float *kv_part(const KvAttend &a, long long row) { return a.scratch + row * a.cache.dim; }
__device__ __forceinline__ float2 *kv_part_sums(const KvAttend &a, long long row) {
  return reinterpret_cast<float2 *>(a.scratch + a.seqs.tokens * a.q_heads * a.cache.dim) + row;
}

// x, eight elements from d0 on of a row's result over its own keys (with its m, and l in
// units as above), becomes the result over these and the beginning.
__device__ __forceinline__ void kv_join(const KvAttend &a, const PromptSlot *slots, long long row, int d0, float (&x)[8], float m, float l) {
  const float2 ml = __ldcg(kv_part_sums(a, row));
  float m1 = ml.x, l1 = ml.y, o[8];
  const float4 *at = reinterpret_cast<const float4 *>(kv_part(a, row));
  if (l1 == -1.f) {
    const int4 where = __ldcg(reinterpret_cast<const int4 *>(at));
    const int i = where.z >> 7, r = where.z & 127;
    float t = -INFINITY;
    m1 = -INFINITY, l1 = 0.f;
#pragma unroll 8
    for (int z = where.x; z <= where.y; ++z) {
      const PromptSlot &sl = slots[2 * (2 * z + (z == where.x ? 1 : 0)) + i];
      const float zm = __ldcg(&sl.m[r]);
      m1 = fmaxf(m1, zm);
      t = fmaxf(t, zm + log2_of(__ldcg(&sl.vref)));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll 4
    for (int z = where.x; z <= where.y; ++z) {
      const PromptSlot &sl = slots[2 * (2 * z + (z == where.x ? 1 : 0)) + i];
      const float zm = __ldcg(&sl.m[r]), zl = __ldcg(&sl.l[r]), wv = kv_share(zm + log2_of(__ldcg(&sl.vref)), t);
      const float4 u = __ldcg(reinterpret_cast<const float4 *>(&sl.acc[(d0 / 4 * 128 + r) * 4])),
                   v = __ldcg(reinterpret_cast<const float4 *>(&sl.acc[((d0 / 4 + 1) * 128 + r) * 4]));
      if (zm != -INFINITY || zl != 0.f) l1 += kv_scaled(zl, zm - m1);
      o[0] += u.x * wv, o[1] += u.y * wv, o[2] += u.z * wv, o[3] += u.w * wv;
      o[4] += v.x * wv, o[5] += v.y * wv, o[6] += v.z * wv, o[7] += v.w * wv;
    }
    const float2 y = kv_norm(fast_exp2(t - m1), l1);
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = o[k] * y.x * y.y;
    l1 *= kPromptToPart;
  } else {
    const float4 u = __ldcg(at + d0 / 4), v = __ldcg(at + d0 / 4 + 1);
    o[0] = u.x, o[1] = u.y, o[2] = u.z, o[3] = u.w, o[4] = v.x, o[5] = v.y, o[6] = v.z, o[7] = v.w;
  }
  const float top = fmaxf(m, m1);
  const float w1 = l1 != 0.f ? kv_scaled(l1, m1 - top) : 0.f, w = l != 0.f ? kv_scaled(l, m - top) : 0.f;
  const float sum = w1 + w, f1 = sum != 0.f ? w1 / sum : 0.f, f = sum != 0.f ? w / sum : 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = (f1 != 0.f ? o[k] * f1 : 0.f) + (f != 0.f ? x[k] * f : 0.f);
}

}  // namespace ivb
