// Attention over the paged 8-bit cache for few queries a sequence (decoding,
// checking drafted tokens).
//
// For a query at position p and the visible keys j (codes kc, vc; scales ks, vs):
//   s_j = scale * ks_j * (q . kc_j),  o = sum_j e^(s_j - m) vs_j vc_j / sum_j e^(s_j - m)
// in one pass with a running reference m (the largest weight times value scale).
// A decode step reads every visible code once and does a few operations for each,
// so the cache's bytes bound it.
//
// An item is a tile of 8 or 16 query rows (token, head of the group) of one
// sequence and kv head; its units are the key blocks (16 keys that share a
// scale).  All units of the launch are divided evenly over the CTAs, whatever
// the sequences' lengths: a CTA's share is the rest of one item, some whole
// ones and the beginning of another.  Where an item is cut, each CTA leaves
// its partial sums in its own slots, and the last of the item's CTAs to arrive
// adds them up in the order of the keys, so the result does not depend on who
// is last.  Counters return to zero by themselves.
//
// A warp takes whole blocks: it copies 16 rows of key and value codes to its
// ring in shared memory (cp.async, swizzled so that the reads below do not
// conflict), and multiplies with m16n8k16 tensor instructions, transposed
// (keys, then head elements, are the 16 rows; queries the 8 columns), so that
// a handful of queries fills an instruction and a code is converted once for
// all of them.  Value codes become halves exactly (1024 + code + 128 by a byte
// permutation, minus 1152); key codes stay code + 128, and 128 times the
// query's sum comes off the score (16 sequences of 131072: 660 us, 688 with exact
// codes).  A score's rounding error then goes by 2^-24 scale ks sum |q| (|code| +
// 128) and not |q code|: below 1 / 1000 of what rounding the keys to codes has
// cost, unless a query element is some 2^14 times the others where codes are small.
// The order of head elements and keys inside the products is chosen so that every
// lane reads whole 16-byte (64-wide heads: 8-byte) pieces of a row; the weights turn
// into the second product's operand by transposing 8 x 8 pieces in registers.
//
// 16 sequences of 131072 tokens, 8 heads of 128: 650 to 720 us, 6.0 to 6.6 TB/s
// (a copy reaches 6.5); 48 of up to 16384: 165 us, 6.1 TB/s (186 after a flush of
// the L2, which else holds a fifth of them).  Sliding windows of 1024 over 128
// sequences (64 wide): 23 us (floor 10), the start of the shares and their joins;
// six drafted tokens for 24 sequences, 30 rows: 50 us (floor 14), the latency of
// conversion, products and softmax in turn, at twelve warps an SM and for two row
// tiles.
#include <algorithm>

#include "kv_attend.cuh"

namespace ivb {

namespace {

constexpr int kStepWarps = 4, kStepThreads = 32 * kStepWarps;
constexpr unsigned kStepItemCost = 8;  // of items that are not cut: start and join, in blocks
constexpr int kStepStages = 4;  // blocks of a warp's ring; two are worked on at once
// A CTA's share is at least this: four blocks for each warp (777 keys, 4 kv
// heads: 12.2 us; one block 14.1, two 12.6, eight 15.3: joining against reading).
constexpr int kStepMinBlocks = 4 * kStepWarps;
// A row's maximum follows its scores only when one is kStepSlack above it: the
// sums are rescaled rarely, and weights stay below 2^(kStepBits + kStepSlack).
constexpr float kNoValue = -1000.f;  // log2 of a value scale of 0
constexpr float kStepSlack = 3.5f, kStepBits = 12.f;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of halves, a row's two halves a lane, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Two codes (+ 128, in bytes of w) as halves 2^-24 (code + 128): the bytes are
// the last bits of subnormal halves, which the tensor cores multiply exactly.
template <int SEL>
__device__ __forceinline__ uint32_t tiny2(uint32_t w) {
  return __byte_perm(w, 0u, SEL);
}
constexpr float kTiny = 0x1p-24f;

// Two codes (+ 128, in bytes of w) as halves.
template <int SEL>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  const uint32_t m = __byte_perm(w, 0x64646464u, SEL);
  const uint32_t bias = 0x64806480u;  // 1152
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(bias));
  return r;
}

// Offset in a 16-row tile of codes of byte o: 128-byte lines whose 16-byte
// pieces are exchanged so that neither the key reads (8 rows x 4 pieces a
// warp) nor the value reads (4 row pairs x 8 pieces) meet in a bank.
template <int DIM>
__device__ __forceinline__ uint32_t tile_swizzle(uint32_t o) {
  const uint32_t line = o >> 7;
  const uint32_t f = DIM == 128 ? ((line & 6u) ^ ((line & 1u) << 2)) : ((line & 3u) << 1);
  return o ^ (f << 4);
}

// CTAs an SM, by registers (and, for wide heads, the rings).  16 rows of 128-wide
// heads take 240 registers, three CTAs leave 168: 24 sequences of up to 6001
// tokens, 8 kv heads, at 16, 32, 64 rows 78, 130, 241 us, two CTAs 66, 115, 209.
constexpr int step_ctas(int dim, int nt) { return dim == 128 ? (nt == 1 ? 3 : 2) : (nt == 1 ? 4 : 3); }

template <int DIM, int NT>
struct StepSlot {  // a part of a cut item: accumulators lane by lane in units of 2^t, then each row's m, sum and t
  float acc[NT * DIM / 4 * 32];
  float m[8 * NT], l[8 * NT], t[8 * NT];
};

template <int DIM, int NT>
struct StepShared {
  alignas(128) uint8_t ring[kStepWarps][kStepStages][2][kKvBlock * DIM];
  float2 scales[kStepWarps][kStepStages];  // key scale, log2 of the value scale (-inf: no block)
  float m[kStepWarps][8 * NT], l[kStepWarps][8 * NT], lref[kStepWarps];
  long long scan[kStepWarps];
  long long base;
  int seq;
  int last;
  long long scan_items[kStepWarps];  // of kRest
  int most[kStepWarps];
};

// Of kRest: what sequences are, behind the above, where there is one for each thread
// at most.  (Looked up again, each has a chain of three loads: 98 us for a call of 96
// sequences in 6 groups, 94 so.)
struct StepKept {
  int first, n, len, first_block, blocks;
};

// NT: 8-row tiles of queries that share the codes of an item.
template <bool BF16, int DIM, int NT, int MODE>
__global__ void __launch_bounds__(kStepThreads, step_ctas(DIM, NT))
    kv_step_k(const __grid_constant__ KvAttend a, StepSlot<DIM, NT> *slots, unsigned *counters) {
  extern __shared__ uint8_t smem_raw[];
  StepShared<DIM, NT> &sh = *reinterpret_cast<StepShared<DIM, NT> *>(smem_raw);
  constexpr int kRows = 8 * NT;
  constexpr int kTiles = DIM / 16;      // 16-row tiles of head elements (output), 16-deep steps (scores)
  constexpr int kPiece = DIM / 8;       // head elements of a lane's piece
  constexpr int kAcc = NT * DIM / 4;    // accumulators a lane
  constexpr int kTile = kKvBlock * DIM;  // bytes of a block's keys or values
  constexpr int kZ = 2;                  // blocks worked on at once
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  // (kRest: its launch begins when every CTA of the one before, which works on the
  // beginning, has; that one's results are wanted, and its place in the workspace is free,
  // only at a segment's end)
  if (MODE != kRest) pdl_wait_and_release();

  // ---- all units, and the sequence where this CTA's share begins
  const int per = (a.seqs.batch + kStepThreads - 1) / kStepThreads;
  long long mine = 0;
  const int b_lo = min(a.seqs.batch, (int)threadIdx.x * per), b_hi = min(a.seqs.batch, b_lo + per);
  long long my_items = 0;
  int most = 0;
  StepKept *const kept = reinterpret_cast<StepKept *>(smem_raw + sizeof(StepShared<DIM, NT>));
  auto span_of = [&](int b) {
    if (MODE != kRest || per > 1) return kv_span<MODE>(a, b);
    const StepKept k = kept[b];
    KvSpan s;
    s.first = k.first, s.n = k.n, s.len = k.len, s.first_block = k.first_block, s.blocks = k.blocks;
    s.sink_blocks = s.lead = s.common = 0;
    return s;
  };
  for (int b = b_lo; b < b_hi; ++b) {
    const KvSpan s = kv_span<MODE>(a, b);
    if (MODE == kRest && per == 1) kept[b] = StepKept{s.first, s.n, s.len, s.first_block, s.blocks};
    const long long items = (long long)((s.n * a.group + kRows - 1) / kRows) * a.cache.heads;
    mine += s.blocks * items;
    if (MODE == kRest) my_items += items, most = max(most, s.blocks);
  }
  long long incl = mine, incl_items = my_items;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    const long long w = MODE == kRest ? __shfl_up_sync(0xffffffffu, incl_items, o) : 0;
    if (lane >= o) incl += v, incl_items += w;
  }
  if (lane == 31) sh.scan[warp] = incl;
  if (MODE == kRest) {
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 31) sh.scan_items[warp] = incl_items, sh.most[warp] = most;
  }
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kStepWarps; ++w) {
    if (w < warp) before += sh.scan[w];
    total += sh.scan[w];
  }
  // (no CTA ends before the launch before: what follows relies on that)
  if (total == 0) {
    if (MODE == kRest) pdl_wait_and_release();
    return;
  }
  if (total > 0x7fffffffLL) {  // (hours of work; units are counted in 32 bits from here)
    if (threadIdx.x == 0) kv_flag(a.status, kStatusKvSeqs);
    if (MODE == kRest) pdl_wait_and_release();
    return;
  }
  uint32_t at_least = kStepMinBlocks;
  bool by_item = false;  // a share is the items that begin in it, whole
  long long excl = before + incl - mine;
  uint32_t cost = 0;  // units of an item beside its blocks
  if (MODE == kRest) {
    // What sequences have of their own is often a few blocks.  Where no item is much more
    // than a share, nothing is cut (64 sequences of up to 500 keys of their own, 8 heads:
    // 25 us for this launch alone against 28); else a share is no more than an item.
    long long items_before = 0, items = 0;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) {
      if (w < warp) items_before += sh.scan_items[w];
      items += sh.scan_items[w];
      most = max(most, sh.most[w]);
    }
    by_item = most <= (total + gridDim.x - 1) / gridDim.x + 24 && total + kStepItemCost * items <= 0x7fffffffLL;
    at_least = by_item ? 1u : (uint32_t)min(total / max(items, 1ll) + 1, (long long)kStepMinBlocks);
    if (by_item) {
      cost = kStepItemCost;
      total += cost * items, mine += cost * my_items, excl += cost * (items_before + incl_items - my_items);
    }
  }
  auto units_of = [&](const KvSpan &s) { return MODE == kRest ? (uint32_t)s.blocks + cost : (uint32_t)s.blocks; };
  const uint32_t size = max(at_least, ((uint32_t)total + gridDim.x - 1) / gridDim.x);  // units of a share
  uint32_t u = blockIdx.x * size;
  if (u >= (uint32_t)total) {
    if (MODE == kRest) pdl_wait_and_release();
    return;
  }
  const uint32_t u_end = min((uint32_t)total, u + size);
  if (u >= excl && u < excl + mine) {
    long long at = excl;
    int b = b_lo;
    for (;; ++b) {
      const KvSpan s = span_of(b);
      const long long w = (long long)units_of(s) * ((s.n * a.group + kRows - 1) / kRows) * a.cache.heads;
      if (u < at + w) break;
      at += w;
    }
    sh.seq = b;
    sh.base = at;
  }
  __syncthreads();
  int b = sh.seq;
  uint32_t base = (uint32_t)sh.base;  // first unit of sequence b
  KvSpan s = span_of(b);
  int row_tiles = (s.n * a.group + kRows - 1) / kRows;
  if (MODE == kRest && by_item) {  // from the first item that begins here
    const uint32_t into = (u - base) % units_of(s);
    if (into) u += units_of(s) - into;
    if (u >= u_end) {
      pdl_wait_and_release();
      return;
    }
  }

  // ---- this lane's places in a tile of codes
  const uint32_t ring = smem_u32(&sh.ring[warp][0][0][0]);
  const uint32_t put0 = tile_swizzle<DIM>((uint32_t)lane * 16u), put1 = tile_swizzle<DIM>(512u + (uint32_t)lane * 16u);
  const uint32_t key_at = tile_swizzle<DIM>((uint32_t)(g * DIM + 16 * t4));  // row g, its second half: ^ 64
  const uint32_t val_at0 = tile_swizzle<DIM>((uint32_t)(2 * t4 * DIM + g * kPiece)),
                 val_at1 = tile_swizzle<DIM>((uint32_t)((2 * t4 + 1) * DIM + g * kPiece));

  // ---- the segment at u: blocks k0 .. k1 - 1 of item (b, head, row tile), and
  // this warp's of them, k0 + warp, + kStepWarps, ...
  int head = 0, rt = 0, k0 = 0, k1 = 0, count = 0, looked = 0;
  uint32_t item_begin = 0;
  long long where = -1;  // lane i: where the i-th of the next 32 blocks' codes are, -1: none
  float2 sc_mine = make_float2(0.f, -INFINITY);
  auto locate = [&]() {
    for (;;) {
      const uint32_t units = units_of(s) * (uint32_t)row_tiles * (uint32_t)a.cache.heads;
      if (u < base + units) break;
      base += units;
      s = span_of(++b);  // (units are left, so there is a next sequence)
      row_tiles = (s.n * a.group + kRows - 1) / kRows;
    }
    const uint32_t item = (u - base) / units_of(s);
    head = (int)(item / (uint32_t)row_tiles);
    rt = (int)item - head * row_tiles;
    item_begin = base + item * units_of(s);
    k0 = (int)(u - item_begin);
    k1 = MODE == kRest && by_item ? s.blocks : (int)(min(u_end, item_begin + (uint32_t)s.blocks) - item_begin);
    count = k1 - k0 > warp ? (k1 - k0 - warp + kStepWarps - 1) / kStepWarps : 0;
    looked = 0;
  };
  // A block is looked up 32 at a time and copied kStepStages ahead of the
  // products; its scales wait beside its codes (a value scale below 0:
  // nothing to see).
  auto fetch = [&](int it) {
    if (it < count) {
      if (it == looked) {
        looked += 32;
        where = -1;
        sc_mine = make_float2(0.f, -INFINITY);
        if (it + lane < count) {
          const int key = s.block(k0 + warp + (it + lane) * kStepWarps) * kKvBlock;
          if (key < s.len) {
            const int at = fast_div(key, a.by_page), page = kv_get<MODE>(a.seqs.pages + kv_page_at<MODE>(a, s, b, key, at));
            if ((unsigned)page < (unsigned long long)a.cache.pages) {
              const int slot = key - at * a.cache.page;
              where = kv_code_at(a.cache, page, head, slot);
              const long long sa = kv_scale_at(a.cache, page, head, slot);
              sc_mine = make_float2(kv_get<MODE>(a.cache.ks + sa), fmaxf(log2_of(kv_get<MODE>(a.cache.vs + sa)), kNoValue));
            } else {
              kv_flag(a.status, kStatusKvPage);
            }
          }
        }
      }
      const long long from = __shfl_sync(0xffffffffu, where, it & 31);
      if (lane == (it & 31)) sh.scales[warp][it % kStepStages] = sc_mine;
      if (from >= 0) {
        const uint32_t dst = ring + (uint32_t)(it % kStepStages) * (2u * kTile);
        const int8_t *kp = a.cache.k + from + lane * 16, *vp = a.cache.v + from + lane * 16;
#pragma unroll
        for (int i = 0; i < kTile / 512; ++i)
          cp_async16(dst + (uint32_t)(i >> 1) * 1024u + (i & 1 ? put1 : put0), kp + i * 512);
#pragma unroll
        for (int i = 0; i < kTile / 512; ++i)
          cp_async16(dst + kTile + (uint32_t)(i >> 1) * 1024u + (i & 1 ? put1 : put0), vp + i * 512);
      }
    }
    cp_async_commit();
  };
  // The join at a segment's end uses the last NT places of the ring; the first
  // ones hold the next segment's first blocks by then.
  constexpr int kAhead = kStepStages - NT;
  locate();
#pragma unroll
  for (int i = 0; i < kAhead; ++i) fetch(i);

  for (;;) {
#pragma unroll
    for (int i = kAhead; i < kStepStages; ++i) fetch(i);
    const int first_block = k0 + warp;

    // ---- queries: column g of tile t for the products, columns 2 t4, + 1 for the scores
    uint32_t q[NT][kTiles][2];
    int pos[NT][2];
    float rs[NT][2], qo[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = rt * kRows + 8 * t + g, i = fast_div(r, a.by_group);
      const uint16_t *row = static_cast<const uint16_t *>(a.q.p) + (long long)(s.first + i) * a.q.ts +
                            (long long)(head * a.group + r - i * a.group) * a.q.hs;
      uint32_t w[2 * kTiles];
#pragma unroll
      for (int c = 0; c < DIM / 64; ++c) {
        const uint4 x = i < s.n ? load8<MODE == kRest>(row + 64 * c + 16 * t4, a.q.vec) : make_uint4(0, 0, 0, 0);
        const uint4 y = i < s.n ? load8<MODE == kRest>(row + 64 * c + 16 * t4 + 8, a.q.vec) : make_uint4(0, 0, 0, 0);
        w[8 * c] = x.x, w[8 * c + 1] = x.y, w[8 * c + 2] = x.z, w[8 * c + 3] = x.w;
        w[8 * c + 4] = y.x, w[8 * c + 5] = y.y, w[8 * c + 6] = y.z, w[8 * c + 7] = y.w;
      }
      float up = a.scale * kLog2e / kTiny;
      if (BF16) {
        // bf16 queries become halves: the row is scaled by a power of two so
        // that its largest element lies in 2^15 .. 2^16 (eight bits are exact
        // down to 2^-32 of it)
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < 2 * kTiles; ++k) {
          const float2 f = unpack2<true>(w[k]);
          most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = min(max((int)(__float_as_uint(most) >> 23), 16), 254);  // biased
        const float down = __uint_as_float((uint32_t)(269 - e) << 23);
        up *= __uint_as_float((uint32_t)(e - 15) << 23);
#pragma unroll
        for (int k = 0; k < 2 * kTiles; ++k) {
          const float2 f = unpack2<true>(w[k]);
          w[k] = pack2<false>(f.x * down, f.y * down);
        }
      }
#pragma unroll
      for (int k = 0; k < kTiles; ++k) q[t][k][0] = w[2 * k], q[t][k][1] = w[2 * k + 1];
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 2 * kTiles; ++k) {
        const float2 f = unpack2<false>(w[k]);
        sum += f.x + f.y;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int rc = rt * kRows + 8 * t + 2 * t4 + c, ic = fast_div(rc, a.by_group);
        pos[t][c] = ic < s.n ? kv_position<MODE>(s, ic) : -1;
        rs[t][c] = BF16 ? __shfl_sync(0xffffffffu, up, (2 * t4 + c) * 4) : up;  // (lane of column 2 t4 + c)
        qo[t][c] = __shfl_sync(0xffffffffu, sum, (2 * t4 + c) * 4) * (-128.f * kTiny);
      }
    }
    const int p_lo = kv_position<MODE>(s, fast_div(rt * kRows, a.by_group));                               // first row's position
    const int p_hi = kv_position<MODE>(s, min(s.n - 1, fast_div(rt * kRows + kRows - 1, a.by_group)));  // last row's

    float acc[NT][kTiles][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int j = 0; j < kTiles; ++j) acc[t][j][0] = acc[t][j][1] = acc[t][j][2] = acc[t][j][3] = 0.f;
    }
    float lref = -INFINITY;  // acc is in units of vref, the largest value scale so far: log2 of it

    for (int it = 0; it < count; it += kZ) {
      cp_async_wait<kStepStages - kZ>();
      __syncwarp();
      const int st = it % kStepStages;  // (a multiple of kZ)
      // scores of keys g, g + 8 of each block
      float sc[kZ][NT][4];
      float lv[kZ];
#pragma unroll
      for (int z = 0; z < kZ; ++z) {
        const float2 scales = sh.scales[warp][st + z];
        lv[z] = z == 0 || it + z < count ? scales.y : -INFINITY;
        if (lv[z] == -INFINITY) {
#pragma unroll
          for (int t = 0; t < NT; ++t) sc[z][t][0] = sc[z][t][1] = sc[z][t][2] = sc[z][t][3] = -INFINITY;
          continue;
        }
        const uint8_t *kt = sh.ring[warp][st + z][0];
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[z][t][0] = sc[z][t][1] = sc[z][t][2] = sc[z][t][3] = 0.f;
#pragma unroll
        for (int c = 0; c < DIM / 64; ++c) {
          const uint4 x = *reinterpret_cast<const uint4 *>(kt + (key_at ^ (64u * c)));
          const uint4 y = *reinterpret_cast<const uint4 *>(kt + (key_at ^ (64u * c)) + 8 * DIM);
          const uint32_t xw[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
          const uint32_t yw[4] = {y.x ^ 0x80808080u, y.y ^ 0x80808080u, y.z ^ 0x80808080u, y.w ^ 0x80808080u};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a0 = tiny2<0x4140>(xw[i]), a1 = tiny2<0x4140>(yw[i]), a2 = tiny2<0x4342>(xw[i]),
                           a3 = tiny2<0x4342>(yw[i]);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma16816(sc[z][t], a0, a1, a2, a3, q[t][4 * c + i][0], q[t][4 * c + i][1]);
          }
        }
        const int key0 = s.block(first_block + (it + z) * kStepWarps) * kKvBlock;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          // (q . (code + 128) - 128 sum q, in the units of the products)
          const float f0 = rs[t][0] * scales.x, f1 = rs[t][1] * scales.x, o0 = qo[t][0] * f0, o1 = qo[t][1] * f1;
          sc[z][t][0] = fmaf(sc[z][t][0], f0, o0);
          sc[z][t][1] = fmaf(sc[z][t][1], f1, o1);
          sc[z][t][2] = fmaf(sc[z][t][2], f0, o0);
          sc[z][t][3] = fmaf(sc[z][t][3], f1, o1);
        }
        if (key0 + kKvBlock - 1 > p_lo || (a.window > 0 && p_hi - key0 >= a.window && key0 + kKvBlock > a.sinks)) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!kv_sees(a, pos[t][e & 1], key0 + g + 8 * (e >> 1))) sc[z][t][e] = -INFINITY;
        }
      }
      // the value scale, and the rows' maxima of s + log2 (vs / vref), where one is well above
      const float lnew = fmaxf(lref, fmaxf(lv[0], lv[kZ - 1]));
      const bool there[2] = {lv[0] != -INFINITY, lv[kZ - 1] != -INFINITY};
#pragma unroll
      for (int z = 0; z < kZ; ++z) lv[z] = fmaxf(lv[z] - lnew, kFarBelow);
      float mx[NT][2];
      bool above = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          mx[t][c] = fmaxf(sc[0][t][c], sc[0][t][c + 2]) + lv[0];
          if (kZ == 2) mx[t][c] = fmaxf(mx[t][c], fmaxf(sc[kZ - 1][t][c], sc[kZ - 1][t][c + 2]) + lv[kZ - 1]);
          above = above || mx[t][c] > m[t][c] + kStepSlack;
        }
      if (__any_sync(0xffffffffu, above) || lnew > lref) {
        const float lvr = lnew > lref ? lref - lnew : 0.f;  // in units of the new vref the largest so far is lower by this
        float most = 0.f;  // (fmaxf passes over NaN)
#pragma unroll
        for (int t = 0; t < NT; ++t) most = fmaxf(most, fmaxf(l[t][0], l[t][1]));
        const float room = kv_room(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))));
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = mx[t][c];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            // (a row's m goes by its own scores alone, whichever row brought the warp here)
            const float md = fmaxf(m[t][c] + lvr, m[t][c] - room);
            x = x > md + kStepSlack ? x : md;
            const float d = x != m[t][c] ? m[t][c] - x : 0.f, f = fast_exp2(d + lvr);
            l[t][c] = kv_scaled(l[t][c], d);
            m[t][c] = x;
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              acc[t][j][c] *= f;
              acc[t][j][c + 2] *= f;
            }
          }
        lref = lnew;
      }
#pragma unroll
      for (int z = 0; z < kZ; ++z) {
        if (!there[z]) continue;
        const float vf = fast_exp2(lv[z] + kSumBits);
        uint32_t p[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float w[4];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float shift = m[t][c] == -INFINITY ? 0.f : m[t][c] - (kStepBits - kSumBits);
            w[c] = fast_exp2(sc[z][t][c] - shift);
            w[c + 2] = fast_exp2(sc[z][t][c + 2] - shift);
            l[t][c] += w[c] + w[c + 2];
          }
          // rounded to 11 bits; summed in 32
          p[t][0] = transpose8x8(pack2<false>(w[0] * vf, w[1] * vf));
          p[t][1] = transpose8x8(pack2<false>(w[2] * vf, w[3] * vf));
        }
        // values of keys 2 t4, + 1, + 8, + 9; rows g, g + 8 of tile j are bytes 2j, 2j + 1 of the lane's piece
        const uint8_t *vt = sh.ring[warp][st + z][1];
        uint32_t vw[4][DIM / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t *at = vt + (i & 1 ? val_at1 : val_at0) + (i >> 1) * 8 * DIM;
          if (DIM == 128) {
            const uint4 x = *reinterpret_cast<const uint4 *>(at);
            vw[i][0] = x.x, vw[i][1] = x.y, vw[i][DIM / 32 - 2] = x.z, vw[i][DIM / 32 - 1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(at);
            vw[i][0] = x.x, vw[i][1] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < DIM / 32; ++w) {
          const uint32_t x0 = vw[0][w] ^ 0x80808080u, x1 = vw[1][w] ^ 0x80808080u, x2 = vw[2][w] ^ 0x80808080u,
                         x3 = vw[3][w] ^ 0x80808080u;
          const uint32_t lo = __byte_perm(x0, x1, 0x5140), hi = __byte_perm(x0, x1, 0x7362);
          const uint32_t lo8 = __byte_perm(x2, x3, 0x5140), hi8 = __byte_perm(x2, x3, 0x7362);
          const uint32_t a0 = codes2<0x4140>(lo), a1 = codes2<0x4342>(lo), a2 = codes2<0x4140>(lo8),
                         a3 = codes2<0x4342>(lo8);
          const uint32_t b0 = codes2<0x4140>(hi), b1 = codes2<0x4342>(hi), b2 = codes2<0x4140>(hi8),
                         b3 = codes2<0x4342>(hi8);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma16816(acc[t][2 * w], a0, a1, a2, a3, p[t][0], p[t][1]);
            mma16816(acc[t][2 * w + 1], b0, b1, b2, b3, p[t][0], p[t][1]);
          }
        }
      }
      __syncwarp();  // their places have been read
#pragma unroll
      for (int z = 0; z < kZ; ++z) fetch(it + kStepStages + z);
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- what the join needs of this segment, then the next one's blocks on their way
    const int n = s.n, first = s.first, head_now = head, rt_now = rt;
    const bool begins = k0 == 0, whole = begins && k1 == s.blocks, joins = MODE == kRest && s.first_block > 0;
    const int first_cta = (int)(item_begin / size), last_cta = (int)((item_begin + (uint32_t)s.blocks - 1u) / size);
    u += (uint32_t)(k1 - k0) + cost;
    const bool more = u < u_end;
    if (more) {
      locate();
#pragma unroll
      for (int i = 0; i < kAhead; ++i) fetch(i);
    }

    if (MODE == kRest) pdl_wait_and_release();

    // ---- join the warps: row maxima, then sums in a common scale
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[t][c] += __shfl_xor_sync(0xffffffffu, l[t][c], o);
        if (g == 0) {
          sh.m[warp][8 * t + 2 * t4 + c] = m[t][c];
          sh.l[warp][8 * t + 2 * t4 + c] = l[t][c];
        }
      }
    if (lane == 0) sh.lref[warp] = lref;
    __syncthreads();
    // accumulators lane by lane, [row tile][row of two][head element of the
    // piece]: eight neighbours of a lane are eight neighbouring outputs
    float *part = reinterpret_cast<float *>(&sh.ring[warp][kAhead][0][0]);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w) top = fmaxf(top, sh.m[w][8 * t + 2 * t4 + c] + sh.lref[w]);
        const float f = kv_share(m[t][c] + lref, top);
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) part[((2 * t + c) * kPiece + 2 * j + h) * 32 + lane] = acc[t][j][2 * h + c] * f;
      }
    __syncthreads();
    const int slot = 2 * (int)blockIdx.x + (begins ? 1 : 0);
    if (!whole) {
      for (int e = threadIdx.x; e < kAcc * 32; e += kStepThreads) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w) x += reinterpret_cast<const float *>(&sh.ring[w][kAhead][0][0])[e];
        __stcg(&slots[slot].acc[e], x);
      }
      if (threadIdx.x < kRows) {
        const int r = threadIdx.x;
        float top = -INFINITY, x = 0.f, t = -INFINITY;
        for (int w = 0; w < kStepWarps; ++w) top = fmaxf(top, sh.m[w][r]), t = fmaxf(t, sh.m[w][r] + sh.lref[w]);
        for (int w = 0; w < kStepWarps; ++w)
          if (sh.m[w][r] != -INFINITY || sh.l[w][r] != 0.f) x += kv_scaled(sh.l[w][r], sh.m[w][r] - top);
        __stcg(&slots[slot].m[r], top);
        __stcg(&slots[slot].l[r], x);
        __stcg(&slots[slot].t[r], t);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        __threadfence();  // (the CTA's writes, which the barrier has put before this)
        const unsigned parts = (unsigned)(last_cta - first_cta + 1);
        const bool last = atomicAdd(&counters[first_cta], 1u) == parts - 1;
        if (last) {
          atomicExch(&counters[first_cta], 0u);
          __threadfence();
        }
        sh.last = last;
      }
      __syncthreads();
    }
    if (whole || sh.last) {
      // eight neighbouring outputs a thread
      for (int e = threadIdx.x; e < kAcc / 8 * 32; e += kStepThreads) {
        const int ln = e & 31, i0 = (e >> 5) * 8;  // accumulators i0 .. i0 + 7 of lane ln
        const int rc = i0 / kPiece, d0 = i0 % kPiece;
        const int r = 8 * (rc >> 1) + 2 * (ln & 3) + (rc & 1);
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f, top = -INFINITY, t = -INFINITY;
        if (whole) {
          for (int w = 0; w < kStepWarps; ++w) top = fmaxf(top, sh.m[w][r]), t = fmaxf(t, sh.m[w][r] + sh.lref[w]);
          for (int w = 0; w < kStepWarps; ++w) {
            if (sh.m[w][r] != -INFINITY || sh.l[w][r] != 0.f) sum += kv_scaled(sh.l[w][r], sh.m[w][r] - top);
            const float *src = reinterpret_cast<const float *>(&sh.ring[w][kAhead][0][0]) + i0 * 32 + ln;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] += src[32 * k];
          }
        } else {
          // (four parts' loads at once: there can be many)
#pragma unroll 4
          for (int z = first_cta; z <= last_cta; ++z) {
            const StepSlot<DIM, NT> &sl = slots[2 * z + (z == first_cta ? 1 : 0)];
            top = fmaxf(top, __ldcg(&sl.m[r]));
            t = fmaxf(t, __ldcg(&sl.t[r]));
          }
#pragma unroll 4
          for (int z = first_cta; z <= last_cta; ++z) {
            const StepSlot<DIM, NT> &sl = slots[2 * z + (z == first_cta ? 1 : 0)];
            const float zm = __ldcg(&sl.m[r]), zl = __ldcg(&sl.l[r]), wv = kv_share(__ldcg(&sl.t[r]), t);
            // (a part of the keys that was hidden from the row: 0)
            if (zm != -INFINITY || zl != 0.f) sum += kv_scaled(zl, zm - top);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] += __ldcg(&sl.acc[(i0 + k) * 32 + ln]) * wv;
          }
        }
        const int row = rt_now * kRows + r, i = fast_div(row, a.by_group);
        if (i < n) {
          const float2 y = kv_norm(fast_exp2(t - top), sum);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = x[k] * y.x * y.y;
          const int d = (ln >> 2) * kPiece + d0, h = head_now * a.group + row - i * a.group;
          const long long at = (long long)(first + i) * a.q_heads + h;
          if (MODE == kBegin) {
            float4 *o = reinterpret_cast<float4 *>(kv_part(a, at) + d);
            __stcg(o, make_float4(x[0], x[1], x[2], x[3]));
            __stcg(o + 1, make_float4(x[4], x[5], x[6], x[7]));
            if (d == 0) __stcg(kv_part_sums(a, at), make_float2(top, sum));
            continue;
          }
          if (joins) {
            const float4 *o = reinterpret_cast<const float4 *>(kv_part(a, at) + d);
            const float4 v0 = __ldcg(o), v1 = __ldcg(o + 1);
            kv_joined(kv_join(a, at, top, sum), v0, v1, x);
          }
          uint16_t *o = static_cast<uint16_t *>(a.out.p) + (long long)(first + i) * a.out.ts + (long long)h * a.out.hs;
          store8(o + d, pack8<BF16>(x), a.out.vec);
        }
      }
    }
    if (!more) break;
    __syncthreads();  // the ring and the joins are free again
  }
}

template <bool BF16, int DIM, int NT, int MODE>
cudaError_t launch_step(const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  static std::atomic<bool> attr_set[kAttrMaxDevices];
  const int bytes = (int)(sizeof(StepShared<DIM, NT>) + (MODE == kRest ? sizeof(StepKept) * kStepThreads : 0));
  const cudaError_t e = ensure_dynamic_smem(kv_step_k<BF16, DIM, NT, MODE>, bytes, attr_set);
  if (e != cudaSuccess) return e;
  const int grid = sms * step_ctas(DIM, NT);
  return launch_kernel(kv_step_k<BF16, DIM, NT, MODE>, dim3(grid), dim3(kStepThreads), (size_t)bytes, st, a,
                       reinterpret_cast<StepSlot<DIM, NT> *>(static_cast<uint8_t *>(workspace) + kKvCounterBytes),
                       static_cast<unsigned *>(workspace));
}

template <bool BF16, int DIM, int MODE = kWhole>
cudaError_t launch_step_rows(const KvAttend &a, long long rows, void *workspace, int sms, cudaStream_t st) {
  // Rows beyond 16 come as further items: their codes are read again, from L2
  // (24 sequences of 6001, 30 rows of 64 wide heads: 58 us when it was compared,
  // 50 now; tiles of 32 rows, which read them once but leave room for half the
  // warps, 65 us).
  if (rows <= 8) return launch_step<BF16, DIM, 1, MODE>(a, workspace, sms, st);
  return launch_step<BF16, DIM, 2, MODE>(a, workspace, sms, st);
}

constexpr long long kOnePass = 48 << 20;  // bytes of codes

template <bool BF16, int DIM>
cudaError_t launch_shared(const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  // Rows of a group: of all sequences, one group like another.
  KvAttend b = a;
  b.seqs.batch = a.groups;
  const long long rows = (a.seqs.tokens + a.groups - 1) / a.groups * a.group;
  const long long own = (long long)a.max_new * a.group;
  // Few keys: every sequence reads the beginning for itself, in one launch (8 sequences
  // of some 60 keys behind 784, 4 heads of 128: 16 us a call against 34 in two passes).
  const long long keys = (long long)a.sequences * a.seqs.pps * a.cache.page;
  if (own <= 64 && keys * a.cache.heads * 2 * DIM <= kOnePass) return launch_step_rows<BF16, DIM, kOne>(a, own, workspace, sms, st);
  cudaError_t e;
  if (rows > 64 && kv_prompt_takes(b)) {
    // Items of 256 rows: fewer than CTAs, and an item is cut over several of them.
    b.many_parts = (a.seqs.tokens * a.group + 255) / 256 * a.cache.heads < sms;
    e = launch_kv_prompt(BF16, kBegin, b, workspace, sms, st);
    if (e == cudaSuccess && b.many_parts) e = launch_kv_parts(a, workspace, sms, st);
  } else {
    e = launch_step_rows<BF16, DIM, kBegin>(b, rows, workspace, sms, st);
  }
  if (e != cudaSuccess) return e;
  if (own > 64 && kv_prompt_takes(a)) return launch_kv_prompt(BF16, kRest, a, workspace, sms, st);
  return launch_step_rows<BF16, DIM, kRest>(a, own, workspace, sms, st);
}

}  // namespace

// Counters (zero before the first call and after each), then two slots a CTA.
size_t kv_workspace_bytes(int sms) {
  const size_t step = sizeof(StepSlot<128, 2>) * 2 * 4 * (size_t)sms;  // (the largest slot, the most CTAs)
  return kKvCounterBytes + std::max(step, kv_prompt_workspace_bytes(sms));
}

cudaError_t launch_kv_attend(bool bf16, const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  // Rows of one sequence and kv head (max_new has to do for all sequences).  Us in
  // this kernel / in the one for many queries, 8 kv heads, at 32, 48, 64 rows:
  //   24 sequences of up to 6001 tokens   64 wide   74/119  106/118  134/118
  //                                      128 wide  115/180  163/180  210/181
  //   one of 8192                         64 wide   26/27    21/28    23/28
  //                                      128 wide   29/38    29/38    30/38
  //   4 of 2000                           64 wide   19/22    19/22    20/22
  //                                      128 wide   23/28    26/29    28/29
  // At 96 and 128 rows (64 wide, 24 sequences) it was 125/98 and 173/109: few
  // sequences gain from this one up to 64 rows and beyond, many up to some 50.
  const long long rows = (long long)a.max_new * a.group;
  if (rows > 64 && kv_prompt_takes(a)) return launch_kv_prompt(bf16, kWhole, a, workspace, sms, st);
  if (a.cache.dim == 64)
    return bf16 ? launch_step_rows<true, 64>(a, rows, workspace, sms, st) : launch_step_rows<false, 64>(a, rows, workspace, sms, st);
  return bf16 ? launch_step_rows<true, 128>(a, rows, workspace, sms, st) : launch_step_rows<false, 128>(a, rows, workspace, sms, st);
}

cudaError_t launch_kv_attend_shared(bool bf16, const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  if (a.cache.dim == 64) return bf16 ? launch_shared<true, 64>(a, workspace, sms, st) : launch_shared<false, 64>(a, workspace, sms, st);
  return bf16 ? launch_shared<true, 128>(a, workspace, sms, st) : launch_shared<false, 128>(a, workspace, sms, st);
}

}  // namespace ivb
