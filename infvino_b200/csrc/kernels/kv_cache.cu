// Rotary positions and the paged 8-bit key/value cache: the table, the rotation,
// the append (rotation, block scales and codes in one pass) and the read.
//
// All four move bytes: a few operations for each element that is read and
// written once, so memory bounds long calls and the chain of dependent loads
// (sequence, page, position, angles) short ones.  Sixteen elements (eight
// pairs) of a row are a thread's share; a warp reads whole 128-byte lines of
// the two halves of a head.  Whether rows can be read 16 bytes at a time is
// settled for a whole launch: a branch at each load cost 9 %.
#include <algorithm>
#include <type_traits>

#include "kv_common.cuh"

namespace ivb {

namespace {

// A token's positions, on the axes that pairs turn by.  If one is outside the
// table nothing of the token is written.
struct Positions {
  int p[kKvMaxAxes];
};
__device__ __forceinline__ Positions load_positions(const KvRotary &r, long long token) {
  Positions x;
#pragma unroll
  for (int axis = 0; axis < kKvMaxAxes; ++axis) x.p[axis] = __ldg(r.pos[axis] + token);
  return x;
}
__device__ __forceinline__ bool in_table(const KvRotary &r, int p) { return p >= 0 && p < r.positions; }
__device__ __forceinline__ bool in_table(const KvRotary &r, const Positions &x) {
  bool ok = true;
#pragma unroll
  for (int axis = 0; axis < kKvMaxAxes; ++axis) ok = ok & in_table(r, x.p[axis]);
  return ok;
}
__device__ __forceinline__ int on_axis(const Positions &x, int axis) {
  const int lo = axis & 1 ? x.p[1] : x.p[0], hi = axis & 1 ? x.p[3] : x.p[2];
  return axis & 2 ? hi : lo;
}

// cos and sin of the eight pairs 8g.. at positions x (of position 0 for one outside the table).
struct Turn {
  float c[8], s[8];
};
__device__ __forceinline__ void load_turn(const KvRotary &r, int g, const Positions &x, Turn &t) {
  if ((r.one_axis >> g) & 1u) {
    const int p = on_axis(x, r.axis[8 * g]);
    const float4 *row = reinterpret_cast<const float4 *>(r.table + (in_table(r, p) ? (long long)p : 0) * r.pairs + 8 * g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = __ldg(row + i);
      t.c[2 * i] = v.x, t.s[2 * i] = v.y, t.c[2 * i + 1] = v.z, t.s[2 * i + 1] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = on_axis(x, r.axis[8 * g + i]);
      const float2 v = __ldg(r.table + (in_table(r, p) ? (long long)p : 0) * r.pairs + 8 * g + i);
      t.c[i] = v.x, t.s[i] = v.y;
    }
  }
}

// Where the two vectors of group g of a row begin: the halves of eight pairs
// (side by side when they are interleaved), or sixteen elements behind the
// rotated ones.
template <bool INTER>
__device__ __forceinline__ void group_at(int g, int pairs, int &a, int &b) {
  if (!INTER && 8 * g < pairs) {
    a = 8 * g;
    b = pairs + 8 * g;
  } else {
    a = 16 * g;
    b = 16 * g + 8;
  }
}

// Turns eight pairs in place.  Products and sums are rounded one by one (no
// fused multiply-add), so any IEEE evaluation of the formula gives the same
// bits, and with them the same codes in the cache.
template <bool INTER>
__device__ __forceinline__ void turn8(float (&a)[8], float (&b)[8], const Turn &t) {
  if (INTER) {  // a: pairs 0..3, b: pairs 4..7, each (x, y) side by side
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float(&h)[8] = i < 4 ? a : b;
      const int j = 2 * (i & 3);
      const float x = h[j], y = h[j + 1];
      h[j] = __fsub_rn(__fmul_rn(x, t.c[i]), __fmul_rn(y, t.s[i]));
      h[j + 1] = __fadd_rn(__fmul_rn(y, t.c[i]), __fmul_rn(x, t.s[i]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = __fsub_rn(__fmul_rn(x, t.c[i]), __fmul_rn(y, t.s[i]));
      b[i] = __fadd_rn(__fmul_rn(y, t.c[i]), __fmul_rn(x, t.s[i]));
    }
  }
}

__global__ void kv_rope_table_k(const __grid_constant__ KvRopeFreq f, int pairs, long long n, float2 *table) {
  pdl_wait_and_release();
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    const long long p = i / pairs;
    double s, c;
    sincos((double)p * f.inv[i - p * pairs], &s, &c);
    table[i] = make_float2((float)c, (float)s);
  }
}

// Heads a thread turns by the same angles at once: what hides the chain from
// position to table row is the rows in flight meanwhile, 2 x 16 bytes a head,
// more than the number of warps.  16381 tokens, 28 heads of 128: 44.5 us, 5.3
// TB/s (floor 36); 4 heads and three CTAs an SM 47, 2 heads and four 50.
constexpr int kRopeThreads = 256;
constexpr int kRopeHeads = 8;

// Turns the rows of token tile `tile`.  A token takes hs * (dim / 16) threads;
// thread (head h0, group g) turns heads h0, h0 + hs, ...
template <bool BF16, bool INTER, bool VEC, int HEADS>
__device__ __forceinline__ void rope_tile(long long tile, long long tokens, int heads, int dim, int hs, int per_block,
                                          const KvRows &x, const KvRows &out, const KvRotary &rot, int *status) {
  const int groups = dim / 16, upt = hs * groups;
  for (int u = threadIdx.x; u < upt * per_block; u += (int)blockDim.x) {
    const int tl = u / upt, r = u - tl * upt, h0 = r / groups, g = r - h0 * groups;
    const long long token = tile * per_block + tl;
    if (token >= tokens) break;
    const bool turned = 8 * g < rot.pairs;
    int ea, eb;
    group_at<INTER>(g, rot.pairs, ea, eb);
    const uint16_t *xr = static_cast<const uint16_t *>(x.p) + token * x.ts;
    uint16_t *yr = static_cast<uint16_t *>(out.p) + token * out.ts;
    Turn t;
    bool ok = true;
    for (int h = h0; h < heads; h += HEADS * hs) {
      // the rows are on their way before the angles' chain (position, then table) begins
      uint4 ua[HEADS], ub[HEADS];
#pragma unroll
      for (int i = 0; i < HEADS; ++i)
        if (h + i * hs < heads) {
          ua[i] = load8(xr + (h + i * hs) * x.hs + ea, VEC);
          ub[i] = load8(xr + (h + i * hs) * x.hs + eb, VEC);
        }
      if (h == h0) {
        const Positions at = load_positions(rot, token);
        ok = in_table(rot, at);
        if (turned) load_turn(rot, g, at, t);
        if (!ok) kv_flag(status, kStatusKvPosition);
      }
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < HEADS; ++i)
        if (h + i * hs < heads) {
          if (turned) {
            float a[8], b[8];
            unpack8<BF16>(ua[i], a);
            unpack8<BF16>(ub[i], b);
            turn8<INTER>(a, b, t);
            ua[i] = pack8<BF16>(a);
            ub[i] = pack8<BF16>(b);
          }
          store8(yr + (h + i * hs) * out.hs + ea, ua[i], VEC);
          store8(yr + (h + i * hs) * out.hs + eb, ub[i], VEC);
        }
    }
  }
}

template <bool BF16, bool INTER, bool VEC>
__global__ void __launch_bounds__(kRopeThreads, 2)
    kv_rope_k(long long tokens, int heads, int dim, int hs, int per_block, const __grid_constant__ KvRows x,
              const __grid_constant__ KvRows out, const __grid_constant__ KvRotary rot, int *status) {
  pdl_wait_and_release();
  rope_tile<BF16, INTER, VEC, kRopeHeads>(blockIdx.x, tokens, heads, dim, hs, per_block, x, out, rot, status);
}

// ---------------------------------------------------------------- append

struct AppendArgs {
  KvCache c;
  KvSeqs s;
  KvRows k, v, q, q_out;
  KvRotary rot;
  int q_heads, q_hs, q_per_block;
  int window;             // packed tokens an append CTA looks at
  int slices, append_ctas;
  int *status;
};

// The least e with m <= 127 * 2^e, m >= 0 finite: m = f * 2^x with f in [1, 2),
// and 127 = 1.984375 * 2^6.
__device__ __forceinline__ int scale_exponent(float m) {
  const uint32_t u = __float_as_uint(m);
  const int x = (int)(u >> 23) - 127;
  const int e = x - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return max(kKvMinExp, min(kKvMaxExp, e));  // (zero and subnormals: below the range)
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Four codes.  x * inv is exact (a power of two) and at most 127, so adding
// 1.5 * 2^23 rounds it to the nearest integer, ties to even, in the low byte.
__device__ __forceinline__ uint32_t quantise4(const float *x, float inv) {
  uint32_t t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = __float_as_uint(fmaf(x[i], inv, 12582912.f));
  return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}
// NaN to 0, infinities (and what the largest scale cannot hold) to the largest code.
__device__ __forceinline__ float tame(float x, float most) { return x == x ? fminf(fmaxf(x, -most), most) : 0.f; }
// The larger magnitude; NaN if one is.
__device__ __forceinline__ float max_abs(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}
__device__ __forceinline__ uint32_t requantise4(uint32_t w, float ratio) {
  uint32_t o = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (int)(int8_t)(w >> (8 * i));
    o |= ((uint32_t)__float2int_rn((float)c * ratio) & 0xffu) << (8 * i);
  }
  return o;
}

constexpr int kAppendThreads = 256;
constexpr int kAppendHeads = 4;  // query heads a thread turns at once: more would cost every CTA its registers
// Warps that share a block: with DIM / 32 of them a lane has sixteen elements
// of one of its rows, with half as many of two.
template <int TEAM>
__device__ __forceinline__ void team_sync(int team) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * TEAM) : "memory");
}
constexpr int append_ctas(int dim, int team) { return team == dim / 32 ? 3 : 2; }  // an SM, by registers

// TEAM warps: the new tokens of one block (rows r0 .. r1 - 1 of its 16, packed
// tokens from t0), keys or values (`codes`, `scales`: head 0's), of heads
// head, head + step, ...  A warp takes 16 / TEAM of the rows; lane (row l /
// groups, group l % groups) holds sixteen elements of every (32 / groups)-th.
// A token's angles are loaded once for all heads, and a head's rows while the
// one before is worked on.
template <bool BF16, bool INTER, int DIM, bool VEC, int TEAM>
__device__ __forceinline__ void append_block(const AppendArgs &a, const KvRows &x, bool turn, int8_t *codes,
                                             float *scales, int head, int step, int r0, int r1, long long t0,
                                             float *shared) {
  constexpr int kGroups = DIM / 16, kRows = 32 / kGroups, kSteps = kKvBlock / kRows / TEAM;
  const int lane = threadIdx.x & 31, g = lane % kGroups, warp = threadIdx.x >> 5, team = warp / TEAM;
  const int row0 = warp % TEAM * (kKvBlock / TEAM) + lane / kGroups;
  const int pairs = turn ? a.rot.pairs : 0;
  int ea, eb;
  group_at<INTER>(g, pairs, ea, eb);
  const uint16_t *xt = static_cast<const uint16_t *>(x.p) + t0 * x.ts;
  uint4 ua[kSteps], ub[kSteps];
  float before = 0.f;
  uint32_t rows = (1u << r1) - (1u << r0);  // bit r: row r is written
  auto load = [&](int h) {
    if (h >= a.c.heads) return;
    if (r0 > 0) before = scales[(long long)h * (a.c.page / kKvBlock)];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int r = row0 + i * kRows;
      ua[i] = ub[i] = make_uint4(0, 0, 0, 0);
      if ((rows >> r) & 1u) {
        const uint16_t *row = xt + (r - r0) * x.ts + h * x.hs;
        ua[i] = load8(row + ea, VEC);
        ub[i] = load8(row + eb, VEC);
      }
    }
  };
  // the largest magnitude of the block
  auto join = [&](float m) {
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) shared[warp] = m;
    team_sync<TEAM>(team);
#pragma unroll
    for (int w = 0; w < TEAM; ++w) m = max_abs(m, shared[team * TEAM + w]);
    team_sync<TEAM>(team);
    return m;
  };
  // lane l looks at the positions of row l % 16 on axes l / 16 and l / 16 + 2
  int p01 = 0, p23 = 0;
  if (a.rot.table && ((rows >> (lane & 15)) & 1u)) {
    const long long token = t0 + (lane & 15) - r0;
    p01 = __ldg((lane < 16 ? a.rot.pos[0] : a.rot.pos[1]) + token);
    p23 = __ldg((lane < 16 ? a.rot.pos[2] : a.rot.pos[3]) + token);
  }
  load(head);
  Turn t[kSteps];
  bool turned[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int r = row0 + i * kRows;
    Positions at;
#pragma unroll
    for (int axis = 0; axis < kKvMaxAxes; ++axis) at.p[axis] = __shfl_sync(0xffffffffu, axis < 2 ? p01 : p23, 16 * (axis & 1) + r);
    turned[i] = ((rows >> r) & 1u) && 8 * g < pairs;
    if (turned[i]) load_turn(a.rot, g, at, t[i]);
  }
  const uint32_t bad = a.rot.table ? __ballot_sync(0xffffffffu, !in_table(a.rot, p01) || !in_table(a.rot, p23)) : 0;
  if (bad) {
    if (lane == 0) kv_flag(a.status, kStatusKvPosition);
    rows &= ~(bad | bad >> 16);
    if (rows == 0) return;  // (for all warps of the team)
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      if (!((rows >> (row0 + i * kRows)) & 1u)) {
        ua[i] = ub[i] = make_uint4(0, 0, 0, 0);
        turned[i] = false;
      }
  }
#pragma unroll 1
  for (; head < a.c.heads; head += step) {
    float f[kSteps][2][8], most = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      unpack8<BF16>(ua[i], f[i][0]);
      unpack8<BF16>(ub[i], f[i][1]);
      if (turned[i]) turn8<INTER>(f[i][0], f[i][1], t[i]);
#pragma unroll
      for (int j = 0; j < 16; ++j) most = max_abs(most, f[i][j >> 3][j & 7]);
    }
    const float old = before;
    load(head + step);
    most = join(most);
    const bool odd = !(most <= 3.402823466e38f);  // an infinity or a NaN: the scale goes by the others
    if (odd) {
      most = 0.f;
#pragma unroll
      for (int j = 0; j < 16 * kSteps; ++j) {
        const float v = fabsf(f[j >> 4][j >> 3 & 1][j & 7]);
        if (v <= 3.402823466e38f) most = fmaxf(most, v);
      }
      most = join(most);
    }
    int8_t *ch = codes + (long long)head * a.c.page * DIM;
    int e = scale_exponent(most);
    if (r0 > 0) {  // tokens before: their codes follow the scale if it grows
      const int eo = max(kKvMinExp, min(kKvMaxExp, (int)((__float_as_uint(old) >> 23) & 0xffu) - 127));
      if (e > eo) {
        const float ratio = e - eo > 60 ? 0.f : exp2i(eo - e);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int r = row0 + i * kRows;
          if (r < r0) {
            uint4 *p = reinterpret_cast<uint4 *>(ch + r * DIM + 16 * g);
            const uint4 w = *p;
            *p = make_uint4(requantise4(w.x, ratio), requantise4(w.y, ratio), requantise4(w.z, ratio),
                            requantise4(w.w, ratio));
          }
        }
      }
      e = max(e, eo);
    }
    if (warp % TEAM == 0 && lane == 0) scales[(long long)head * (a.c.page / kKvBlock)] = exp2i(e);  // (all have read the old one)
    const float inv = exp2i(-e);
    if (odd || e == kKvMaxExp) {
      const float top = 127.f * exp2i(e);
#pragma unroll
      for (int j = 0; j < 16 * kSteps; ++j) {
        float &v = f[j >> 4][j >> 3 & 1][j & 7];
        v = tame(v, top);
      }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int r = row0 + i * kRows;
      if ((rows >> r) & 1u) {
        *reinterpret_cast<uint2 *>(ch + r * DIM + ea) = make_uint2(quantise4(f[i][0], inv), quantise4(f[i][0] + 4, inv));
        *reinterpret_cast<uint2 *>(ch + r * DIM + eb) = make_uint2(quantise4(f[i][1], inv), quantise4(f[i][1] + 4, inv));
      }
    }
  }
}

// Where a packed token is: its sequence's end, and its page and slot (-1: nowhere).
struct Place {
  long long first, end;  // the sequence's packed tokens
  int pos, page, slot;
};

// The places of packed tokens first .. first + window - 1, one thread each.
__device__ __forceinline__ void find_places(const KvCache &c, const KvSeqs &s, long long first, int window, int *status,
                                            Place *places) {
  int seq = kv_seq_of(s, first);
  const int i = threadIdx.x;
  const long long t = first + i;
  if (i < window) {
    Place p{0, 0, -1, -1, 0};
    if (t < s.tokens) {
      while (seq < s.batch && s.offsets[seq + 1] <= t) ++seq;
      if (seq < s.batch) {  // (tokens behind the last sequence are not the call's)
        p.first = s.offsets[seq];
        p.end = min((long long)s.offsets[seq + 1], s.tokens);
        const long long pos = (long long)s.at[seq] + (t - p.first);
        if (t < p.first || p.first < 0 || s.at[seq] < 0 || pos >= 0x7fffffffLL) {
          kv_flag(status, kStatusKvSeqs);
        } else {
          p.pos = (int)pos;
          p.page = kv_page_of(c, s, seq, p.pos, status);
          p.slot = p.pos % c.page;
        }
      }
    }
    places[i] = p;
  }
  __syncthreads();
}

// Of the first `append_ctas` CTAs each takes the blocks whose first new token
// is among `window` packed tokens, and every `slices`-th set of heads of
// them: a team of warps for a head's keys, one for its values.  A block is one
// team's alone, so nothing is atomic and the result does not depend on any
// order.  The other CTAs turn queries.
//
// Latency bounds it: two joins and a block's loads for each head in turn.  9375
// tokens, 8 heads of 128 beside 32 of queries: 45 us, 4.7 TB/s (floor 32); 64
// conversations, a token each: 4.3 us.
template <bool BF16, bool INTER, int DIM, bool VEC, int TEAM>
__global__ void __launch_bounds__(kAppendThreads, append_ctas(DIM, TEAM)) kv_append_k(const __grid_constant__ AppendArgs a) {
  __shared__ Place places[kKvBlock];
  __shared__ float most[kAppendThreads / 32];
  pdl_wait_and_release();
  if ((int)blockIdx.x >= a.append_ctas) {
    rope_tile<BF16, INTER, VEC, kAppendHeads>((int)blockIdx.x - a.append_ctas, a.s.tokens, a.q_heads, DIM, a.q_hs,
                                              a.q_per_block, a.q, a.q_out, a.rot, a.status);
    return;
  }
  const long long first = (long long)(blockIdx.x / a.slices) * a.window;
  find_places(a.c, a.s, first, a.window, a.status, places);
  constexpr int kTeams = kAppendThreads / 32 / TEAM, step = kTeams / 2;  // heads a CTA works on at once
  const int team = (threadIdx.x >> 5) / TEAM, head = (blockIdx.x % a.slices) * step + (team >> 1);
  for (int i = 0; i < a.window; ++i) {
    const Place p = places[i];
    const long long t = first + i;
    const int r0 = p.slot % kKvBlock;
    if (p.page < 0 || (t != p.first && r0 != 0)) continue;
    const int r1 = (int)min((long long)kKvBlock, r0 + (p.end - t));  // a block begins here
    const long long ca = kv_code_at(a.c, p.page, 0, p.slot - r0), sa = kv_scale_at(a.c, p.page, 0, p.slot - r0);
    const bool keys = (team & 1) == 0;
    append_block<BF16, INTER, DIM, VEC, TEAM>(a, keys ? a.k : a.v, keys && a.rot.table != nullptr, (keys ? a.c.k : a.c.v) + ca,
                                        (keys ? a.c.ks : a.c.vs) + sa, head, a.slices * step, r0, r1, t, most);
  }
}

// ---------------------------------------------------------------- read

// A CTA takes `window` packed tokens, all heads.  A thread keeps its place in
// the rows (keys or values, head, eight elements: 16 bytes out, so that a warp
// writes whole lines) and goes over the tokens, kReadAhead of them on their way
// at once.  9375 tokens, 8 heads of 128: 10.4 us with the codes in the L2, 14.6
// after a flush of it (floor 8.9); sixteen elements a thread, in two stores, 17.4.
constexpr int kReadAhead = 4, kReadThreads = 256;
template <bool BF16, int DIM>
__global__ void __launch_bounds__(kReadThreads)
    kv_read_k(const __grid_constant__ KvCache c, const __grid_constant__ KvSeqs s, const __grid_constant__ KvRows k,
              const __grid_constant__ KvRows v, int window, int *status) {
  __shared__ Place places[kKvBlock];
  pdl_wait_and_release();
  constexpr int kGroups = DIM / 8;
  const long long first = (long long)blockIdx.x * window;
  const int each = ((k.p ? 1 : 0) + (v.p ? 1 : 0)) * c.heads * kGroups;
  const int lanes = min(each, kReadThreads), step = kReadThreads / lanes;
  const int i0 = threadIdx.x / lanes;
  find_places(c, s, first, window, status, places);
  if (i0 >= step) return;
  for (int u = threadIdx.x - i0 * lanes; u < each; u += lanes) {
    const int g = u % kGroups, hh = u / kGroups;
    const bool val = hh >= c.heads || !k.p;
    const int head = hh >= c.heads ? hh - c.heads : hh;
    const int8_t *codes = (val ? c.v : c.k) + kv_code_at(c, 0, head, 0) + 8 * g;
    const float *scales = (val ? c.vs : c.ks) + kv_scale_at(c, 0, head, 0);
    const KvRows &y = val ? v : k;
    uint16_t *rows = static_cast<uint16_t *>(y.p) + first * y.ts + head * y.hs + 8 * g;
    for (int i = i0; i < window; i += kReadAhead * step) {
      uint2 w[kReadAhead];
      float sc[kReadAhead];
#pragma unroll
      for (int n = 0; n < kReadAhead; ++n) {
        const int j = i + n * step;
        if (j >= window || places[j].page < 0) continue;
        w[n] = *reinterpret_cast<const uint2 *>(codes + kv_code_at(c, places[j].page, 0, places[j].slot));
        sc[n] = scales[kv_scale_at(c, places[j].page, 0, places[j].slot)];
      }
#pragma unroll
      for (int n = 0; n < kReadAhead; ++n) {
        const int j = i + n * step;
        if (j >= window || places[j].page < 0) continue;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)((e < 4 ? w[n].x : w[n].y) >> (8 * (e & 3))) * sc[n];
        store8(rows + j * y.ts, pack8<BF16>(f), y.vec);
      }
    }
  }
}

// Tokens a CTA looks at: one while there are few (decoding: each begins a
// block), up to a block's sixteen where that still gives every SM some.
int window_of(long long tokens) {
  int w = 1;
  while (w < kKvBlock && tokens / w > 148 * 4) w *= 2;
  return w;
}

// Head groups of the rotation: one head a thread while that leaves SMs free,
// up to `most` (angles loaded once for them) from there on.
void rope_shape(long long tokens, int heads, int dim, int most, int threads, int &hs, int &per_block) {
  const int groups = dim / 16;
  const long long work = tokens * heads * groups / 148;
  const int each = work < 2048 ? 1 : work < 8192 ? std::min(4, most) : most;
  hs = (heads + each - 1) / each;
  per_block = std::max(1, threads / (hs * groups));
}

}  // namespace

cudaError_t launch_kv_rope_table(const KvRopeFreq &f, int pairs, long long positions, float2 *table, cudaStream_t st) {
  const long long n = positions * pairs;
  const int grid = (int)std::min<long long>((n + 255) / 256, 148 * 8);
  return launch_kernel(kv_rope_table_k, dim3(grid), dim3(256), 0, st, f, pairs, n, table);
}

cudaError_t launch_kv_rope(bool bf16, long long tokens, int heads, int dim, const KvRows &x, const KvRows &out,
                           const KvRotary &rot, int *status, cudaStream_t st) {
  int hs, per_block;
  rope_shape(tokens, heads, dim, kRopeHeads, kRopeThreads, hs, per_block);
  const dim3 grid((unsigned)((tokens + per_block - 1) / per_block));
  auto types = [&](auto inter, auto vec) {
    constexpr bool kInter = decltype(inter)::value, kVec = decltype(vec)::value;
    return bf16 ? kv_rope_k<true, kInter, kVec> : kv_rope_k<false, kInter, kVec>;
  };
  auto pick = [&](auto inter) {
    return x.vec && out.vec ? types(inter, std::true_type{}) : types(inter, std::false_type{});
  };
  auto kern = rot.interleaved ? pick(std::true_type{}) : pick(std::false_type{});
  return launch_kernel(kern, grid, dim3(kRopeThreads), 0, st, tokens, heads, dim,
                       hs, per_block, x, out, rot, status);
}

cudaError_t launch_kv_append(bool bf16, const KvCache &c, const KvSeqs &s, const KvRows &k, const KvRows &v,
                             const KvRotary &rot, int q_heads, const KvRows &q, const KvRows &q_out, int *status,
                             cudaStream_t st) {
  AppendArgs a{c, s, k, v, q, q_out, rot, q_heads, 1, 1, 0, 0, 0, status};
  a.window = window_of(s.tokens);
  // Two warps a block where most blocks get a token or two (64 conversations, 8
  // heads: 4.3 us; four warps 5.0), one row a lane where they are filled (9375
  // tokens, when it was compared: 47 us; two warps 53).
  const int team = a.window == 1 ? 2 : c.dim / 32, teams = kAppendThreads / 32 / team;
  // A CTA loops over the heads where there are blocks enough for two CTAs an
  // SM; fewer take the heads side by side.
  const int windows = (int)((s.tokens + a.window - 1) / a.window), most = (2 * c.heads + teams - 1) / teams;
  a.slices = std::max(1, std::min(most, 2 * 148 / windows));
  a.append_ctas = windows * a.slices;
  long long grid = a.append_ctas;
  if (q_heads) {
    rope_shape(s.tokens, q_heads, c.dim, kAppendHeads, kAppendThreads, a.q_hs, a.q_per_block);
    grid += (s.tokens + a.q_per_block - 1) / a.q_per_block;
  }
  auto dims = [&](auto inter, auto vec, auto type) {
    constexpr bool kInter = decltype(inter)::value, kVec = decltype(vec)::value, kBf16 = decltype(type)::value;
    return c.dim == 64 ? kv_append_k<kBf16, kInter, 64, kVec, 2>
           : team == 2 ? kv_append_k<kBf16, kInter, 128, kVec, 2>
                       : kv_append_k<kBf16, kInter, 128, kVec, 4>;
  };
  auto types = [&](auto inter, auto vec) { return bf16 ? dims(inter, vec, std::true_type{}) : dims(inter, vec, std::false_type{}); };
  auto pick = [&](auto inter) {
    return k.vec && v.vec && (!q_heads || (q.vec && q_out.vec)) ? types(inter, std::true_type{}) : types(inter, std::false_type{});
  };
  auto kern = rot.interleaved ? pick(std::true_type{}) : pick(std::false_type{});
  return launch_kernel(kern, dim3((unsigned)grid), dim3(kAppendThreads), 0, st, a);
}

cudaError_t launch_kv_read(bool bf16, const KvCache &c, const KvSeqs &s, const KvRows &k, const KvRows &v, int *status,
                           cudaStream_t st) {
  const int window = window_of(s.tokens);
  const dim3 grid((unsigned)((s.tokens + window - 1) / window));
  auto kern = c.dim == 64 ? (bf16 ? kv_read_k<true, 64> : kv_read_k<false, 64>)
                          : (bf16 ? kv_read_k<true, 128> : kv_read_k<false, 128>);
  return launch_kernel(kern, grid, dim3(kReadThreads), 0, st, c, s, k, v, window, status);
}

}  // namespace ivb
