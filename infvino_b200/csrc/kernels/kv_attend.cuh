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
  int lead, common;   // of kOne: the sequence whose pages have the first `common` tokens
  __device__ __forceinline__ int block(int i) const { return i < sink_blocks ? i : i - sink_blocks + first_block; }
};

// What a launch works on: whole sequences; or, of sequences in groups with a common
// beginning, first the groups (all queries of a group over the beginning, whose
// results wait in the scratch: kv_part below), then each sequence's own keys, with
// those results joined in; or both in one pass, each sequence reading the beginning.
enum KvMode { kWhole = 0, kBegin = 1, kRest = 2, kOne = 3 };

// What a launch reads.  The step kernel of kRest begins while the launch before it, of
// the same call, still works on the beginning: what was written before that launch is in
// the L2 by then, but an SM's own cache may hold it as it was earlier.
template <int MODE, class T>
__device__ __forceinline__ T kv_get(const T *p) {
  return MODE == kRest ? __ldcg(p) : *p;
}

// A group's sequences s0 .. s1 - 1, its packed tokens o .. e - 1, and how many are common; false (status set) if that does not fit.
struct KvGroup {
  int s0, s1, o, e, len;
};
template <int MODE>
__device__ __forceinline__ bool kv_group(const KvAttend &a, int g, KvGroup &r) {
  r.s0 = kv_get<MODE>(a.first + g), r.s1 = kv_get<MODE>(a.first + g + 1), r.len = kv_get<MODE>(a.shared + g);
  bool fits = r.s0 >= 0 && r.s1 >= r.s0 && r.s1 <= a.sequences && r.len >= 0 && r.len <= (long long)a.seqs.pps * a.cache.page &&
              r.len == fast_div(r.len, a.by_page) * a.cache.page;
  if (fits) {
    r.o = kv_get<MODE>(a.seqs.offsets + r.s0), r.e = kv_get<MODE>(a.seqs.offsets + r.s1);
    fits = r.o >= 0 && r.e >= r.o && r.e <= a.seqs.tokens;
  }
  if (!fits) kv_flag(a.status, kStatusKvSeqs);
  return fits;
}

// Sequence b (kBegin: group b, as a sequence of all its queries over its first sequence's pages).
template <int MODE>
__device__ __forceinline__ KvSpan kv_span(const KvAttend &a, int b) {
  KvSpan s;
  s.sink_blocks = s.first_block = s.blocks = 0;
  s.lead = s.common = 0;
  if (MODE == kBegin) {
    KvGroup r;
    s.first = s.n = s.len = 0;
    if (!kv_group<MODE>(a, b, r) || r.o == r.e || r.len == 0) return s;
    s.first = r.o;
    s.n = r.e - r.o;
    s.lead = r.s0;
    s.len = r.len;
    s.blocks = r.len / kKvBlock;
    return s;
  }
  const int o = kv_get<MODE>(a.seqs.offsets + b), e = kv_get<MODE>(a.seqs.offsets + b + 1);
  s.first = o;
  s.len = kv_get<MODE>(a.seqs.at + b);
  s.n = e - o;
  if (o < 0 || e < o || e > a.seqs.tokens || s.n > a.max_new || s.len < 0 ||
      s.len > (long long)a.seqs.pps * a.cache.page) {
    kv_flag(a.status, kStatusKvSeqs);
    s.n = 0;
    return s;
  }
  if (s.n == 0) return s;
  const int all = (s.len + kKvBlock - 1) / kKvBlock;
  if (MODE == kRest || MODE == kOne) {
    int g = 0, end = a.groups;  // the last group that begins at or before b
    while (end - g > 1) {
      const int mid = (g + end) / 2;
      if (kv_get<MODE>(a.first + mid) <= b)
        g = mid;
      else
        end = mid;
    }
    // (its tokens are the group's: their results over the beginning are there)
    KvGroup r;
    if (!kv_group<MODE>(a, g, r) || b < r.s0 || b >= r.s1 || o < r.o || e > r.e || s.len - s.n < r.len) {
      kv_flag(a.status, kStatusKvSeqs);
      s.n = 0;
      return s;
    }
    if (MODE == kRest) s.first_block = r.len / kKvBlock;
    s.lead = r.s0;
    s.common = r.len;
  } else if (a.window > 0) {
    // the first query's first window key; blocks before it only for the sinks
    const long long lo = (long long)s.len - s.n - a.window + 1;
    s.first_block = lo > 0 ? (int)(lo / kKvBlock) : 0;
    s.sink_blocks = min(s.first_block, a.sinks / kKvBlock + (a.sinks % kKvBlock != 0));
  }
  s.blocks = max(1, s.sink_blocks + all - s.first_block);
  return s;
}

// Where the page of block `at` (from 0) of sequence b's pages is named, for key `key`.
template <int MODE>
__device__ __forceinline__ long long kv_page_at(const KvAttend &a, const KvSpan &s, int b, int key, int at) {
  const int row = MODE == kBegin ? s.lead : MODE == kOne && key < s.common ? s.lead : b;
  return (long long)row * a.seqs.pps + at;
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
// 2^(12 - kSumBits)).  An item of the prompt kernel that was cut over CTAs has
// l = -1 at first: its first words say which CTAs' slots have its parts, and its row
// in them, for kv_parts_k.
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

// How much a row's result over the beginning and that over its own keys (with its m,
// and l in units as above) count.
__device__ __forceinline__ float2 kv_join(const KvAttend &a, long long row, float m, float l) {
  const float2 ml = __ldcg(kv_part_sums(a, row));
  const float m1 = ml.x, l1 = ml.y, top = fmaxf(m, m1);
  const float w1 = l1 != 0.f ? kv_scaled(l1, m1 - top) : 0.f, w = l != 0.f ? kv_scaled(l, m - top) : 0.f;
  const float sum = w1 + w;
  return sum != 0.f ? make_float2(w1 / sum, w / sum) : make_float2(0.f, 0.f);
}
// x, eight elements of a row's result over its own keys, becomes the result over these and the beginning (u, v).
__device__ __forceinline__ void kv_joined(float2 f, float4 u, float4 v, float (&x)[8]) {
  const float o[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = (f.x != 0.f ? o[k] * f.x : 0.f) + (f.y != 0.f ? x[k] * f.y : 0.f);
}

}  // namespace ivb
