// Attention over the paged 8-bit cache for many queries a sequence (prompts,
// chunks of prompts): the same formula as the step kernel's, on tcgen05.
//
// A key serves hundreds of query rows here, so arithmetic bounds it: 4 * DIM
// operations for each visible (row, key) pair on the tensor cores, and one
// exponential on the special function units, which takes as long (at DIM 128:
// 16 exponentials and 8192 operations a clock and SM).
//
// An item is 256 query rows (token, head of the group) of one sequence and kv
// head, two M tiles of 128; its units are tiles of 128 keys (8 blocks of 16,
// the sinks' blocks first where there is a window).  Units are divided evenly
// over the CTAs, one an SM; items that the division cuts are joined by the
// last of their CTAs to arrive, in the order of the keys.
//
// Sixteen warps a CTA:
//   0-3, 4-7  softmax of M tile 0 and 1, a thread a row: scores from TMEM, the
//             weights back into the scores' columns as the next product's
//             operand; O is rescaled in TMEM, rarely (a row's reference follows
//             only what is kSlack above it); at the end O goes out
//   8-11      key and value codes from the cache through registers into shared
//             memory as halves (exact), one tile ahead in registers and two in
//             shared memory; the blocks' scales beside them
//   12        issues the products: S_i = Q_i K^T (operands K-major in shared
//             memory) and O_i += P_i V (P_i from TMEM, V row-major as it lies
//             in the cache), i alternating, so that one tile's softmax runs
//             under the other tile's products
//   13        walks the CTA's share and publishes its segments, ahead of the rest
//
// A causal prompt of 8191 tokens, 32 heads of 128 over 8 of the cache: 722 us by
// itself, 0.76 PFLOP/s of visible pairs (floor 335), 750 back to back, where the
// card's power counts.  Rows that go by their own scores and value scales cost
// 2 to 3 % of it.  Measured before that: the products of 64 keys and 128 rows take
// 512 clocks by the pipe's rate, 572 when nothing else runs and 650 to 720 from
// issue to end here; their exponentials another 512; a CTA ends such a part every
// 1250 or so.  Without exponentials 14 % of the time goes, without seven of eight
// products another 10 %, without operand stores another 16 %: the hand-over between
// the roles is the rest, and no one of them bounds it.  An item costs some 8 us of
// filling and emptying the pipeline, which short and windowed prompts feel.
//
// Every wait is bounded: a timeout sets the status word and an abort flag, all
// roles run out, TMEM is released, and parts of cut items that the CTA has not come
// to are counted, so that the next call finds the counters at zero.
#include <algorithm>

#include "kv_attend.cuh"

namespace ivb {

namespace {

constexpr int kKeys = 128, kTileBlocks = kKeys / kKvBlock;
constexpr int kRows = 256;
constexpr int kThreads = 512;
constexpr int kSegments = 4;      // ring of segments
constexpr int kMeta = 4;          // rings: scales of a tile live until both softmaxes are done
constexpr int kSub = 64;          // keys of a score tile: two in turn for each M tile and key tile
// (slack 6: windowed chunks 182 us, 7.5: 180.5; every row rescales its sums by itself)
constexpr float kSlack = 7.5f, kBits = 8.f;
constexpr float kFar = -80.f;     // blocks with a lower lv (below) are looked at row by row
constexpr int kNoKey = 0x3fffffff;
constexpr int kItemCost = 2;      // what an item costs besides its tiles, in tiles: queries in, outputs out
constexpr int kMaxSeqs = 8192;    // sequences of a call that the start-up scan has room for

struct alignas(16) TileMeta {
  float kc[kTileBlocks];    // ks * |scale| * log2 e
  float lvf[kTileBlocks];   // lv = log2 (vs / vref)
  float ivf[kTileBlocks];   // 2^(-lv - kSumBits)
  int key0[kTileBlocks];    // first key, kNoKey behind the end
  float vref, lvr;          // vref: the largest value scale so far; log2 (vref before / vref)
  uint32_t rare[2];         // of half h: bit 4: vref grew; bit j: the lv of its block j is below kFar
};

// The key blocks that an item's rows see, for rows 256 rt and on of a sequence.
struct RowSpan {
  int sink_blocks, first_block, blocks, tiles;
};
template <int MODE>
__device__ __forceinline__ RowSpan row_span(const KvAttend &a, int n, int len, int first_block, int rt) {
  RowSpan s;
  if (MODE == kBegin) {  // every row sees all
    s.first_block = s.sink_blocks = 0;
    s.blocks = len / kKvBlock;
    s.tiles = max(1, (s.blocks + kTileBlocks - 1) / kTileBlocks);
    return s;
  }
  const int i0 = fast_div(rt * kRows, a.by_group), i1 = min(n - 1, fast_div(rt * kRows + kRows - 1, a.by_group));
  const int p_lo = len - n + i0, p_hi = len - n + i1;
  const int all = p_hi >= 0 ? p_hi / kKvBlock + 1 : 0;
  s.first_block = MODE == kRest ? first_block : 0;
  s.sink_blocks = 0;
  if (MODE == kWhole && a.window > 0) {
    const long long lo = (long long)p_lo - a.window + 1;
    s.first_block = lo > 0 ? (int)(lo / kKvBlock) : 0;
    s.sink_blocks = min(s.first_block, a.sinks / kKvBlock + (a.sinks % kKvBlock != 0));
  }
  s.blocks = max(0, s.sink_blocks + all - s.first_block);
  s.tiles = max(1, (s.blocks + kTileBlocks - 1) / kTileBlocks);
  return s;
}

// A piece of an item: tiles k0 .. k1 - 1 of rows 256 rt .. of sequence b, one kv head.
struct Segment {
  int more;                  // 0: there is none, the share is done
  int b, rt, head, k0, k1;
  int first_cta, last_cta;   // the CTAs that have tiles of the item
  KvSpan s;
  RowSpan r;
  __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == r.tiles; }
};

// A CTA's share of the units, segment by segment.
template <int MODE>
struct Walk {
  uint32_t u, end, base;  // next unit, the share's end, first unit of (b, rt)
  int b, rt, row_tiles;
  KvSpan s;
  RowSpan r;

  // The share begins at unit `from`, in row tile `rt0` (first unit `at`) of sequence b0; it may be empty.
  __device__ __forceinline__ void begin(const KvAttend &a, uint32_t from, uint32_t to, uint32_t at, int b0, int rt0) {
    u = from, end = to, base = at, b = b0, rt = rt0;
    if (u >= end) return;
    s = kv_span<MODE>(a, b);
    row_tiles = (s.n * a.group + kRows - 1) / kRows;
    r = row_span<MODE>(a, s.n, s.len, s.first_block, rt);
  }

  // The next segment into g (all but `more`); false where the share ends.
  __device__ __forceinline__ bool next(const KvAttend &a, uint32_t size, Segment &g) {
    while (u < end) {
      if (s.n > 0) {
        const uint32_t each = (uint32_t)r.tiles + kItemCost, units = each * (uint32_t)a.cache.heads;
        if (u < base + units) {
          const uint32_t head = (u - base) / each, item = base + head * each, to = min(end, item + each);
          g.k0 = max(0, (int)(u - item) - kItemCost);
          g.k1 = (int)(to - item) - kItemCost;
          u = to;
          if (g.k1 <= g.k0) continue;  // (the share ends before the item's first tile)
          g.b = b, g.rt = rt, g.head = (int)head;
          g.first_cta = (int)((item + kItemCost) / size);
          g.last_cta = (int)((item + each - 1) / size);
          g.s = s;
          g.r = r;
          return true;
        }
        base += units;
        if (++rt < row_tiles) {
          r = row_span<MODE>(a, s.n, s.len, s.first_block, rt);
          continue;
        }
      }
      rt = 0;
      s = kv_span<MODE>(a, ++b);  // (units are left, so there is a next sequence)
      row_tiles = (s.n * a.group + kRows - 1) / kRows;
      if (s.n > 0) r = row_span<MODE>(a, s.n, s.len, s.first_block, 0);
    }
    return false;
  }
};

template <int DIM>
struct PromptShared {
  static constexpr int kSlabs = DIM / 64;
  uint8_t q[2][kSlabs][128 * 128];  // 128 rows of 64 halves, 16-byte pieces exchanged by row % 8
  uint8_t k[2][kSlabs][kKeys * 128];
  uint8_t v[2][kSlabs][kKeys * 128];
  TileMeta meta[kMeta];
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2][2], pready[2][2], odone[2][2], qfull[2], drained, never;
  uint32_t tmem;
  volatile int abort;
  int last[2];
  int counted[2][2];  // M tile i's part of the item that the share begins in / ends in
  Segment seg[kSegments];  // written by warp 13, read by the 13 warps that work
  uint64_t segfull[kSegments], segempty[kSegments];
  long long scan[kThreads / 32];
  long long base;
  int seq, rt;
  uint32_t u_begin, u_end, size;  // the share, and how many units one has
};

// Whether the last CTA of a cut item adds its parts up.  Of kBegin items with many, kv_parts_k does.
template <int MODE>
__device__ __forceinline__ bool few_parts(const KvAttend &a, int first_cta, int last_cta) {
  return MODE != kBegin || !a.many_parts || last_cta - first_cta < 3;
}

// Counts a part of an item that CTAs first .. last share; the last one to come sets the counter back.
__device__ __forceinline__ bool count_part(unsigned *counter, int first, int last) {
  const bool done = atomicAdd(counter, 1u) == (unsigned)(last - first);
  if (done) atomicExch(counter, 0u);
  return done;
}

// The lowest n of 16 bits.
__device__ __forceinline__ uint32_t low_bits(int n) { return (1u << min(max(n, 0), kKvBlock)) - 1u; }

__device__ __forceinline__ void wg_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
// Whether all 128 threads say so.
__device__ __forceinline__ bool wg_all(int id, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %2, 0;\n\t"
      "barrier.cta.red.and.pred p, %1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)x)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

#define KV_R8(r, o) "=f"(r[o]), "=f"(r[o + 1]), "=f"(r[o + 2]), "=f"(r[o + 3]), "=f"(r[o + 4]), "=f"(r[o + 5]), "=f"(r[o + 6]), "=f"(r[o + 7])
#define KV_W8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])

// 32 columns of the thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : KV_R8(r, 0), KV_R8(r, 8), KV_R8(r, 16), KV_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      KV_W8(r, 0), KV_W8(r, 8)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// O (+)= P V with P from TMEM.
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 bd;\n\t"
      "mov.b64 bd, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], bd, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Two codes (+ 128, in bytes of w) as halves: 1024 + u, minus 1152.
template <int SEL>
__device__ __forceinline__ uint32_t halves(uint32_t w) {
  const uint32_t m = __byte_perm(w, 0x64646464u, SEL);
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(0x64806480u));
  return r;
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Sixteen codes as halves, to two 16-byte pieces of a row.
__device__ __forceinline__ void put_codes(uint32_t lo_at, uint32_t hi_at, uint4 w4) {
  const uint32_t w[4] = {w4.x ^ 0x80808080u, w4.y ^ 0x80808080u, w4.z ^ 0x80808080u, w4.w ^ 0x80808080u};
  st_shared16(lo_at, halves<0x4140>(w[0]), halves<0x4342>(w[0]), halves<0x4140>(w[1]), halves<0x4342>(w[1]));
  st_shared16(hi_at, halves<0x4140>(w[2]), halves<0x4342>(w[2]), halves<0x4140>(w[3]), halves<0x4342>(w[3]));
}

// Counts the parts of cut items that a CTA has not come to, so that the counters
// are zero again after a launch in which it gave up.  (Not inline: this is rarely run.)
template <int MODE, class Shared>
__device__ __noinline__ void count_rest(const KvAttend &a, Shared &sh, unsigned *counters) {
  Walk<MODE> walk;
  walk.begin(a, sh.u_begin, sh.u_end, (uint32_t)sh.base, sh.seq, sh.rt);
  Segment &g = sh.seg[0];
  while (walk.next(a, sh.size, g))
    for (int i = 0; i < 2; ++i)
      if (!g.whole() && few_parts<MODE>(a, g.first_cta, g.last_cta) && g.s.n * a.group > g.rt * kRows + 128 * i && !sh.counted[i][g.k0 == 0])
        count_part(&counters[2 * g.first_cta + i], g.first_cta, g.last_cta);
}

// (128 registers a thread; kRest, which holds the join's shares too, spills up to 112 bytes, the others up to 52.)
template <bool BF16, int DIM, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    kv_prompt_k(const __grid_constant__ KvAttend a, PromptSlot *slots, unsigned *counters) {
  extern __shared__ uint8_t smem_raw[];
  using Shared = PromptShared<DIM>;
  Shared &sh = *reinterpret_cast<Shared *>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  constexpr int kSlabs = DIM / 64;
  constexpr long long kLimit = kConvWaitLimitDefault;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh.kfull[i]), 4);
      mbar_init(smem_u32(&sh.vfull[i]), 4);
      mbar_init(smem_u32(&sh.kempty[i]), 1);
      mbar_init(smem_u32(&sh.vempty[i]), 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(smem_u32(&sh.sfull[i][h]), 1);
        mbar_init(smem_u32(&sh.pready[i][h]), 4);
        mbar_init(smem_u32(&sh.odone[i][h]), 1);
      }
      mbar_init(smem_u32(&sh.qfull[i]), 4);
    }
    for (int i = 0; i < kSegments; ++i) {
      mbar_init(smem_u32(&sh.segfull[i]), 1);
      mbar_init(smem_u32(&sh.segempty[i]), 13);
    }
    mbar_init(smem_u32(&sh.drained), 1);
    mbar_init(smem_u32(&sh.never), 1);
    sh.abort = 0;
    for (int i = 0; i < 4; ++i) sh.counted[i >> 1][i & 1] = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(&sh.tmem), 512);
    tmem_relinquish();
  }
  pdl_wait_and_release();

  // ---- all units, and where this CTA's share begins.  A warp adds up a
  // sequence's row tiles; the sequences' sums wait where the tiles will be.
  long long *sums = reinterpret_cast<long long *>(&sh.q[0][0][0]);
#pragma unroll 1
  for (int b0 = warp * 32; b0 < a.seqs.batch; b0 += kThreads) {
    int n = 0, len = 0, block = 0;
    if (b0 + lane < a.seqs.batch) {
      const KvSpan s = kv_span<MODE>(a, b0 + lane);
      n = s.n, len = s.len, block = s.first_block;
    }
#pragma unroll 1
    for (int j = 0; j < min(32, a.seqs.batch - b0); ++j) {
      const int nj = __shfl_sync(0xffffffffu, n, j), lj = __shfl_sync(0xffffffffu, len, j);
      const int bj = MODE == kRest ? __shfl_sync(0xffffffffu, block, j) : 0;
      const int rts = (nj * a.group + kRows - 1) / kRows;
      long long sum = 0;
#pragma unroll 1
      for (int rt = lane; rt < rts; rt += 32) sum += row_span<MODE>(a, nj, lj, bj, rt).tiles + kItemCost;
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) sums[b0 + j] = sum * a.cache.heads;
    }
  }
  __syncthreads();
  const int per = (a.seqs.batch + kThreads - 1) / kThreads;
  const int b_lo = min(a.seqs.batch, (int)threadIdx.x * per), b_hi = min(a.seqs.batch, b_lo + per);
  long long mine = 0;
#pragma unroll 1
  for (int b = b_lo; b < b_hi; ++b) mine += sums[b];
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.scan[warp] = incl;
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sh.scan[w];
    total += sh.scan[w];
  }
  // (2^31 units would be hours of work; they are counted in 32 bits from here)
  if (total == 0 || total > 0x7fffffffLL) {
    if (threadIdx.x == 0 && total) kv_flag(a.status, kStatusKvSeqs);
  }
  const bool sane = total > 0 && total <= 0x7fffffffLL;
  // (a share is more than an item's cost, or no CTA would have the tiles between two of them)
  const uint32_t size = sane ? max((uint32_t)kItemCost + 1, ((uint32_t)total + gridDim.x - 1) / gridDim.x) : 1u;
  const bool works = sane && blockIdx.x * size < (uint32_t)total;
  const uint32_t u_begin = works ? blockIdx.x * size : 0u;
  if (threadIdx.x == 0) {
    sh.u_begin = u_begin;
    sh.u_end = works ? min((uint32_t)total, u_begin + size) : 0u;
    sh.size = size;
  }
  const long long u = u_begin;
  const long long excl = before + incl - mine;
  if (works && u >= excl && u < excl + mine) {
    long long at = excl;
    int b = b_lo;
    while (u >= at + sums[b]) at += sums[b++];
    sh.seq = b;
    sh.base = at;
  }
  __syncthreads();
  if (works && warp == 0) {  // the row tile: 32 at a time
    const KvSpan s = kv_span<MODE>(a, sh.seq);
    const int rts = (s.n * a.group + kRows - 1) / kRows;
    long long at = sh.base;
#pragma unroll 1
    for (int r0 = 0; r0 < rts; r0 += 32) {
      long long w = r0 + lane < rts ? (long long)(row_span<MODE>(a, s.n, s.len, s.first_block, r0 + lane).tiles + kItemCost) * a.cache.heads : 0;
      long long in = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += v;
      }
      const bool here = u >= at + in - w && u < at + in;
      const unsigned vote = __ballot_sync(0xffffffffu, here);
      if (here) {
        sh.rt = r0 + lane;
        sh.base = at + in - w;
      }
      if (vote) break;
      at += __shfl_sync(0xffffffffu, in, 31);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  __syncthreads();  // the sums' room is the tiles' from here on

  // Waits as a warp.  A wait that is over already costs one test.
  bool ok = true;
  auto wait = [&](uint32_t bar, uint32_t parity, int code) {
    if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
      ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, &sh.abort, a.status, code, kLimit));
    return ok;
  };
  // A working warp's next segment: leaves the one it has (what it still needs
  // of it is in registers) and waits for the next.
  int seg_n = 0;
  auto next_segment = [&]() -> const Segment * {
    __syncwarp();
    if (seg_n > 0 && lane == 0) mbar_arrive(smem_u32(&sh.segempty[(seg_n - 1) % kSegments]));
    const int at = seg_n % kSegments;
    wait(smem_u32(&sh.segfull[at]), (seg_n / kSegments) & 1, kStatusTimeoutFull);
    ++seg_n;
    return ok && sh.seg[at].more ? &sh.seg[at] : nullptr;
  };

  if (warp < 8) {
    // ------------------------------------------------------------ softmax of M tile i
    reg_inc<184>();
    const int i = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_at = tmem + lanes + 256u + 128u * i;
    int done = 0;   // tiles so far, all segments
    int tile = 0;   // tiles of both M tiles so far: the place of the scales
    const Segment *g = nullptr;
    // ---- the warp's 32 query rows of the segment: halves, K-major.
    // DIM / 8 lanes a row; rf of a row's owner is what its halves were divided by.
    float rf = 1.f;
    auto load_q = [&]() {
      constexpr int kLanes = DIM / 8, kAtOnce = 32 / kLanes;
      const int c = lane % kLanes, first_row = g->rt * kRows + 128 * i + 32 * (warp & 3);
      const int all_rows = g->s.n * a.group, head0 = g->head * a.group;
      const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // |scale| is in the keys' factor
      const uint16_t *src = static_cast<const uint16_t *>(a.q.p) + (long long)g->s.first * a.q.ts + 8 * c;
#pragma unroll 1
      for (int e0 = 0; e0 < kLanes; e0 += 8) {
        uint4 w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int r = first_row + (e0 + e) * kAtOnce + lane / kLanes, tok = fast_div(r, a.by_group);
          w[e] = r < all_rows ? load8(src + (long long)tok * a.q.ts + (long long)(head0 + r - tok * a.group) * a.q.hs, a.q.vec)
                              : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int rw = (e0 + e) * kAtOnce + lane / kLanes;  // of the warp's rows
          w[e].x ^= flip, w[e].y ^= flip, w[e].z ^= flip, w[e].w ^= flip;
          if (BF16) {
            // bf16 queries become halves: scaled by a power of two so that the
            // row's largest element lies in 2^15 .. 2^16 (eight bits are exact
            // down to 2^-32 of it)
            float f[8], most = 0.f;
            unpack8<true>(w[e], f);
#pragma unroll
            for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(f[k]));
#pragma unroll
            for (int o = kLanes / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int x = min(max((int)(__float_as_uint(most) >> 23), 16), 254);  // biased
            const float down = __uint_as_float((uint32_t)(269 - x) << 23);
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] *= down;
            w[e] = pack8<false>(f);
            const int own = (lane % kAtOnce) * kLanes;  // (lane / kAtOnce = (e0 + e): the row is this lane's)
            const float up = __shfl_sync(0xffffffffu, __uint_as_float((uint32_t)(x - 15) << 23), own);
            if (lane / kAtOnce == e0 + e) rf = up;
          }
          const int row = 32 * (warp & 3) + rw;
          *reinterpret_cast<uint4 *>(&sh.q[i][c >> 3][row * 128 + (((c & 7) ^ (row & 7)) << 4)]) = w[e];
        }
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.qfull[i]));
    };
    // the next segment with rows for this M tile; its queries follow at once,
    // before the outputs of the one that is ending
    auto advance = [&]() {
      for (;;) {
        g = next_segment();
        // (the four warps end together, also where a bounded wait ran out: they share barriers)
        if (!wg_all(1 + i, g != nullptr)) return false;
        if (g->s.n * a.group > g->rt * kRows + 128 * i) {
          load_q();
          return true;
        }
        tile += g->k1 - g->k0;
      }
    };
    bool more = advance();
    while (more) {
      const int first_row = g->rt * kRows + 128 * i, rows = min(128, g->s.n * a.group - first_row);
      const int tiles = g->k1 - g->k0;
      const int tok = fast_div(first_row + row, a.by_group);
      const bool real = row < rows;
      const int p = real ? kv_position<MODE>(g->s, tok) : -1;
      const int p_lo = kv_position<MODE>(g->s, fast_div(first_row, a.by_group));
      const int p_hi = kv_position<MODE>(g->s, fast_div(first_row + rows - 1, a.by_group));
      const bool whole = g->whole(), head_part = g->k0 == 0;
      const int first_cta = g->first_cta, last_cta = g->last_cta;
      uint16_t *out = static_cast<uint16_t *>(a.out.p) + (long long)(g->s.first + tok) * a.out.ts +
                      (long long)(g->head * a.group + first_row + row - tok * a.group) * a.out.hs;
      // (of kBegin and kRest: the row's place in the scratch, and whether there is a beginning)
      const long long at = (long long)(g->s.first + tok) * a.q_heads + g->head * a.group + first_row + row - tok * a.group;
      const bool joins = MODE == kRest && g->s.first_block > 0;
      // parts (of four blocks) that need no look at single keys: up to part_hi
      // every row sees the end of it, from part_lo on every row its beginning
      // (or, before part_sink, all of it are sinks)
      const RowSpan &rs = g->r;
      const int part_hi = ((p_lo + 1) / kKvBlock + rs.sink_blocks - rs.first_block) / 4 - 1;
      int part_lo = 0, part_sink = 0;
      if (MODE == kWhole && a.window > 0 && p_hi >= a.window) {
        part_lo = ((p_hi - a.window) / kKvBlock + 1 - rs.first_block + rs.sink_blocks + 3) / 4;
        part_sink = min(rs.sink_blocks, a.sinks / kKvBlock) / 4;
      }
      int part = 2 * g->k0;
      float m = -INFINITY, l = 0.f, vref = 0.f;
#pragma unroll 1
      for (int t = 0; t < tiles; ++t, ++done, ++tile) {
        const TileMeta &me = sh.meta[tile % kMeta];
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (!wait(smem_u32(&sh.sfull[i][h]), done & 1, kStatusTimeoutAcc)) continue;
          tc_fence_after();
          const uint32_t s_at = tmem + lanes + (uint32_t)(2 * i + h) * kSub;
          const int b0 = 4 * h;  // its blocks
          // Hidden keys (behind the row, before its window, behind the end)
          // are put out in TMEM, block by block, before the scores are read:
          // few parts need it, and the code that all parts run stays straight.
          if (part > part_hi || (part < part_lo && part >= part_sink)) {
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {
              const int hi = p - me.key0[b0 + b];
              uint32_t seen = low_bits(hi + 1);
              if (MODE == kWhole && a.window > 0) seen &= ~low_bits(hi - a.window + 1) | low_bits(a.sinks - me.key0[b0 + b]);
              if (__all_sync(0xffffffffu, seen == 0xffffu)) continue;
              uint32_t w[16];
              tmem_ld16(s_at + 16 * b, w);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < kKvBlock; ++k) {
                asm volatile("" : "+r"(w[k]));
                if (!(seen >> k & 1)) w[k] = 0xff800000u;  // -inf
              }
              tmem_st16(s_at + 16 * b, w);
            }
            tmem_st_wait();
          }
          ++part;
          float s[kSub];
          tmem_ld32(s_at, s);
          tmem_ld32(s_at + 32, s + 32);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < kSub; ++k) asm volatile("" : "+f"(s[k]));  // uses stay after the wait
          const float4 kc4 = *reinterpret_cast<const float4 *>(&me.kc[b0]);
          const float4 lv4 = *reinterpret_cast<const float4 *>(&me.lvf[b0]), iv4 = *reinterpret_cast<const float4 *>(&me.ivf[b0]);
          float c[4] = {kc4.x, kc4.y, kc4.z, kc4.w}, mx = -INFINITY;
          float lvf[4] = {lv4.x, lv4.y, lv4.z, lv4.w}, ivf[4] = {iv4.x, iv4.y, iv4.z, iv4.w};
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if (BF16) c[b] = fmaxf(c[b] * rf, 0x1p-120f);  // (never 0: hidden keys stay at -inf)
            float x = s[kKvBlock * b];
#pragma unroll
            for (int k = 1; k < kKvBlock; ++k) x = fmaxf(x, s[kKvBlock * b + k]);
            mx = fmaxf(mx, fmaf(x, c[b], lvf[b]));
          }
          const uint32_t rare = me.rare[h];
          if (__any_sync(0xffffffffu, mx > m + kSlack) || rare != 0) {
            float lvr = 0.f;
            if (rare & 16u) {  // in units of the new vref the largest so far is lower by lvr
              lvr = me.lvr;
              vref = me.vref;
            }
            // (a row's m goes by its own scores alone, whichever row brought the warp here)
            const float md = fmaxf(m + lvr, m - kv_room(l)), top = mx > md + kSlack ? mx : md;
            const float d = top != m ? m - top : 0.f;
            l = kv_scaled(l, d);
            m = top;
            if (t > 0 || h > 0) {
              // the products before: the other half of the keys, of this tile or the last
              if (!wait(smem_u32(&sh.odone[i][h ^ 1]), (h == 0 ? done - 1 : done) & 1, kStatusTimeoutDrain)) continue;
              tc_fence_after();
              const float fo = fast_exp2(d + lvr);
#pragma unroll 1
              for (int d = 0; d < DIM / 32; ++d) {
                float o[32];
                tmem_ld32(o_at + 32 * d, o);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; ++k) asm volatile("" : "+f"(o[k]));
                uint32_t w[32];
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                  const float2 x = mul2(make_float2(o[k], o[k + 1]), make_float2(fo, fo));
                  w[k] = __float_as_uint(x.x);
                  w[k + 1] = __float_as_uint(x.y);
                }
                tmem_st16(o_at + 32 * d, w);
                tmem_st16(o_at + 32 * d + 16, w + 16);
              }
            }
          }
          if (rare & 15u) {
            // Weights may be too small for numbers here and yet count in the
            // sum, which has no 2^lv: lv is raised where the values count for
            // nothing all the same (2^-70 of the row's largest).
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              float x = s[kKvBlock * b];
#pragma unroll
              for (int k = 1; k < kKvBlock; ++k) x = fmaxf(x, s[kKvBlock * b + k]);
              if (lvf[b] == -INFINITY) continue;  // (no block)
              lvf[b] = fmaxf(lvf[b], fminf(kFar, m - x * c[b] - 70.f));
              ivf[b] = fast_exp2(-lvf[b] - kSumBits);
            }
          }
          // weights 2^(s c + lv - m + kBits), sums without 2^lv and in units of 2^-kSumBits
          const float shift = m == -INFINITY ? 0.f : kBits - m;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t w[16];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int b = 2 * q + z;
              const float f = c[b], add = shift + lvf[b];
              float2 sum = make_float2(0.f, 0.f);
#pragma unroll
              for (int k = 0; k < kKvBlock; k += 2) {
                float2 x = fma2(make_float2(s[kKvBlock * b + k], s[kKvBlock * b + k + 1]), make_float2(f, f), make_float2(add, add));
                x.x = fast_exp2(x.x);
                x.y = fast_exp2(x.y);
                sum = add2(sum, x);
                w[8 * z + k / 2] = pack2<false>(x.x, x.y);
              }
              l = fmaf(sum.x + sum.y, ivf[b], l);
            }
            tmem_st16(s_at + 16 * q, w);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.pready[i][h]));
        }
      }

      // ---- O
      more = advance();
      wait(smem_u32(&sh.odone[i][1]), (done - 1) & 1, kStatusTimeoutDrain);
      tc_fence_after();
      if (!ok) {  // (the slot keeps whatever it holds: the status word says that the result is not valid)
      } else if (whole) {
        const float2 y = kv_norm(vref, l);
        float2 shares = make_float2(0.f, 1.f);
        if (joins && real) shares = kv_join(a, at, m, l * kPromptToPart);
#pragma unroll 1
        for (int h = 0; h < DIM / 32; ++h) {
          float4 u[8];
          if (joins && real) {
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = __ldcg(reinterpret_cast<const float4 *>(kv_part(a, at) + 32 * h) + k);
          }
          float o[32];
          tmem_ld32(o_at + 32 * h, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) asm volatile("" : "+f"(o[k]));
          if (real) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              float f[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) f[j] = l != 0.f ? o[k + j] * y.x * y.y : 0.f;
              if (MODE == kBegin) {
                float4 *to = reinterpret_cast<float4 *>(kv_part(a, at) + 32 * h + k);
                __stcg(to, make_float4(f[0], f[1], f[2], f[3]));
                __stcg(to + 1, make_float4(f[4], f[5], f[6], f[7]));
                continue;
              }
              if (joins) kv_joined(shares, u[k / 4], u[k / 4 + 1], f);
              store8(out + 32 * h + k, pack8<BF16>(f), a.out.vec);
            }
          }
        }
        if (MODE == kBegin && real) __stcg(kv_part_sums(a, at), make_float2(m, l * kPromptToPart));
      } else {
        PromptSlot &slot = slots[2 * (2 * (int)blockIdx.x + (head_part ? 1 : 0)) + i];
#pragma unroll 1
        for (int h = 0; h < DIM / 32; ++h) {
          float o[32];
          tmem_ld32(o_at + 32 * h, o);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) asm volatile("" : "+f"(o[k]));
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            __stcg(reinterpret_cast<float4 *>(&slot.acc[((32 * h + k) / 4 * 128 + row) * 4]),
                   make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
        }
        __stcg(&slot.m[row], m);
        __stcg(&slot.l[row], l);
        if (row == 0) __stcg(&slot.vref, vref);
        if (MODE == kBegin && !few_parts<MODE>(a, first_cta, last_cta) && head_part && real) {
          __stcg(reinterpret_cast<int4 *>(kv_part(a, at)), make_int4(first_cta, last_cta, 128 * i + row, 0));
          __stcg(kv_part_sums(a, at), make_float2(0.f, -1.f));
        }
      }
      if (!whole && few_parts<MODE>(a, first_cta, last_cta)) {
        wg_sync(1 + i);
        if (row == 0) {
          __threadfence();  // (the four warps' writes, which the barrier has put before this)
          const bool last = count_part(&counters[2 * first_cta + i], first_cta, last_cta);
          if (last) __threadfence();
          sh.last[i] = last;
          sh.counted[i][head_part] = 1;
        }
        wg_sync(1 + i);
        if (sh.last[i] && real && ok) {
          float top = -INFINITY, t = -INFINITY, sum = 0.f;
          float2 shares = make_float2(0.f, 1.f);
          // (several parts' loads at once: a short call over a long cache has many)
#pragma unroll 4
          for (int z = first_cta; z <= last_cta; ++z) {
            const PromptSlot &sl = slots[2 * (2 * z + (z == first_cta ? 1 : 0)) + i];
            const float zm = __ldcg(&sl.m[row]);
            top = fmaxf(top, zm);
            t = fmaxf(t, zm + log2_of(__ldcg(&sl.vref)));
          }
#pragma unroll 1
          for (int h = 0; h < DIM / 64; ++h) {
            float x[64];
#pragma unroll
            for (int k = 0; k < 64; ++k) x[k] = 0.f;
            sum = 0.f;
#pragma unroll 1
            for (int z = first_cta; z <= last_cta; ++z) {
              const PromptSlot &sl = slots[2 * (2 * z + (z == first_cta ? 1 : 0)) + i];
              const float zm = __ldcg(&sl.m[row]), zl = __ldcg(&sl.l[row]), wv = kv_share(zm + log2_of(__ldcg(&sl.vref)), t);
              // (a part of the keys that was hidden from the row: 0)
              if (zm != -INFINITY || zl != 0.f) sum += kv_scaled(zl, zm - top);
#pragma unroll
              for (int k = 0; k < 64; k += 4) {
                const float4 v = __ldcg(reinterpret_cast<const float4 *>(&sl.acc[((64 * h + k) / 4 * 128 + row) * 4]));
                x[k] += v.x * wv, x[k + 1] += v.y * wv, x[k + 2] += v.z * wv, x[k + 3] += v.w * wv;
              }
            }
            const float2 y = kv_norm(fast_exp2(t - top), sum);
            if (joins && h == 0) shares = kv_join(a, at, top, sum * kPromptToPart);
            if (MODE == kBegin && h == 0) __stcg(kv_part_sums(a, at), make_float2(top, sum * kPromptToPart));
#pragma unroll
            for (int k = 0; k < 64; k += 8) {
              float f[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) f[j] = x[k + j] * y.x * y.y;
              float4 *part = reinterpret_cast<float4 *>(kv_part(a, at) + 64 * h + k);
              if (MODE == kBegin) {
                __stcg(part, make_float4(f[0], f[1], f[2], f[3]));
                __stcg(part + 1, make_float4(f[4], f[5], f[6], f[7]));
                continue;
              }
              if (joins) kv_joined(shares, __ldcg(part), __ldcg(part + 1), f);
              store8(out + 64 * h + k, pack8<BF16>(f), a.out.vec);
            }
          }
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------ codes to halves
    reg_dec<96>();
    // A warp takes 32 rows (two blocks): eight rows of 64 elements at once, a
    // lane sixteen codes of one.  (Eight lanes, two rows, meet eight different
    // 16-byte banks when they store.)
    constexpr int kEach = 4 * kSlabs;
    const int w = warp - 8, c = lane & 3, r8 = lane >> 2;
    const uint32_t put_lo = (uint32_t)((32 * w + r8) * 128 + (((2 * c) ^ r8) << 4)),
                   put_hi = (uint32_t)((32 * w + r8) * 128 + (((2 * c + 1) ^ r8) << 4));
    const float kc_all = fabsf(a.scale) * kLog2e;
    uint4 kreg[kEach], vreg[kEach];
    int tile = 0;
    const Segment *g = nullptr;
    float vref = 0.f;
    // Lane j < 8 knows block j of a tile: where its codes are, its scales.  The
    // page number is asked for a tile before the place and the scales, and
    // those a tile before the codes, so that no look-up waits for another.
    struct Blocks {
      long long at;
      int key0;
      float ks, vs;
    };
    int key_next = kNoKey, page_next = -1;
    auto ask_page = [&](int t) {
      const int bi = t * kTileBlocks + lane;
      key_next = kNoKey;
      if (lane < kTileBlocks && t < g->k1 && bi < g->r.blocks) {
        key_next = (bi < g->r.sink_blocks ? bi : bi - g->r.sink_blocks + g->r.first_block) * kKvBlock;
        page_next = a.seqs.pages[kv_page_at<MODE>(a, g->s, g->b, key_next, fast_div(key_next, a.by_page))];  // (in the row: kv_span has checked)
      }
    };
    auto look_up = [&]() {
      Blocks x{-1, kNoKey, 0.f, 0.f};
      if (key_next != kNoKey) {
        if ((unsigned)page_next < (unsigned long long)a.cache.pages) {
          const int slot = key_next - fast_div(key_next, a.by_page) * a.cache.page;
          x.key0 = key_next;
          x.at = kv_code_at(a.cache, page_next, g->head, slot);
          const long long sa = kv_scale_at(a.cache, page_next, g->head, slot);
          x.ks = a.cache.ks[sa];
          x.vs = a.cache.vs[sa];
        } else {
          kv_flag(a.status, kStatusKvPage);
        }
      }
      return x;
    };
    auto load = [&](const int8_t *codes, const Blocks &x, uint4(&reg)[kEach]) {
      const long long at0 = __shfl_sync(0xffffffffu, x.at, 2 * w), at1 = __shfl_sync(0xffffffffu, x.at, 2 * w + 1);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {  // rows 8 (e % 4).., slab e / 4
        const long long at = e % 4 < 2 ? at0 : at1;
        reg[e] = at >= 0 ? __ldg(reinterpret_cast<const uint4 *>(codes + at + (8 * (e % 2) + r8) * DIM + 64 * (e / 4) + 16 * c))
                         : make_uint4(0, 0, 0, 0);
      }
    };
    while ((g = next_segment())) {
      vref = 0.f;
      ask_page(g->k0);
      Blocks now = look_up();
      ask_page(g->k0 + 1);
      Blocks ahead = look_up();
      ask_page(g->k0 + 2);
      load(a.cache.k, now, kreg);
      load(a.cache.v, now, vreg);
#pragma unroll 1
      for (int t = g->k0; t < g->k1; ++t, ++tile) {
        const int st = tile & 1;
        const bool reused = tile >= 2;
        const uint32_t k_at = smem_u32(&sh.k[0][0][0]) + (uint32_t)(st * sizeof(sh.k[0])), v_at = smem_u32(&sh.v[0][0][0]) + (uint32_t)(st * sizeof(sh.v[0]));
        if (reused) wait(smem_u32(&sh.kempty[st]), ((tile >> 1) - 1) & 1, kStatusTimeoutEmpty);
        if (w == 0) {  // the scales
          float vmax = now.vs;
#pragma unroll
          for (int o = 4; o; o >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
          vmax = fmaxf(vref, __shfl_sync(0xffffffffu, vmax, 0));
          TileMeta &me = sh.meta[tile % kMeta];
          const float lv = vmax > 0.f && now.vs > 0.f ? fmaxf(log2_of(now.vs) - log2_of(vmax), kFarBelow) : kFarBelow;
          if (lane < kTileBlocks) {
            me.kc[lane] = fmaxf(now.ks * kc_all, 0x1p-120f);
            // (a block in a page outside the cache: weights and sums of 0)
            const bool none = now.key0 == kNoKey;
            me.lvf[lane] = none ? -INFINITY : lv;
            me.ivf[lane] = none ? 0.f : fast_exp2(-fmaxf(lv, kFar) - kSumBits);
            me.key0[lane] = now.key0;
          }
          const uint32_t far = __ballot_sync(0xffffffffu, lane < kTileBlocks && now.key0 != kNoKey && lv < kFar);
          if (lane == 0) {
            me.lvr = vmax > vref ? log2_of(vref) - log2_of(vmax) : 0.f;
            me.vref = vmax;
            me.rare[0] = (far & 15u) | (vmax > vref ? 16u : 0u);
            me.rare[1] = far >> 4;
          }
          vref = vmax;
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          put_codes(k_at + put_lo + 16384 * (e / 4) + 1024 * (e % 4), k_at + put_hi + 16384 * (e / 4) + 1024 * (e % 4), kreg[e]);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.kfull[st]));
        load(a.cache.k, ahead, kreg);
        if (reused) wait(smem_u32(&sh.vempty[st]), ((tile >> 1) - 1) & 1, kStatusTimeoutEmpty);
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          put_codes(v_at + put_lo + 16384 * (e / 4) + 1024 * (e % 4), v_at + put_hi + 16384 * (e / 4) + 1024 * (e % 4), vreg[e]);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.vfull[st]));
        load(a.cache.v, ahead, vreg);
        now = ahead;
        ahead = look_up();
        ask_page(t + 3);
      }
    }
  } else {
    reg_dec<40>();
    if (warp == 12) {
      // ---------------------------------------------------------- products
      const bool leader = elect_one();
      const uint32_t idesc_s = idesc_f16_f32(128, kSub);
      const uint32_t idesc_o = idesc_f16_f32(128, DIM) | (1u << 16);  // V: rows are keys (its N side is dense)
      const uint64_t qd = smem_desc_kmajor(smem_u32(&sh.q[0][0][0]), 128), kd = smem_desc_kmajor(smem_u32(&sh.k[0][0][0]), 128);
      // V: 64 head elements a row of 128 bytes; 8 keys 1024 bytes on, the next 64 elements a slab on
      const uint64_t vd = (uint64_t)((smem_u32(&sh.v[0][0][0]) & 0x3FFFFu) >> 4) | ((uint64_t)(128 * 128 >> 4) << 16) |
                          ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
      constexpr uint32_t kTileUnits = kSlabs * 128 * 128 / 16, kSlabUnits = 128 * 128 / 16;
      int tile = 0, seg[2] = {0, 0}, done[2] = {0, 0};
      const Segment *g = nullptr;
      if (a.probe > 0 && blockIdx.x % 2 == 1)
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&sh.never), 0, &sh.abort, a.status, kStatusTimeoutProbe, a.probe));
      // One lane issues, in one stretch for each part, with every operand
      // worked out before: between two parts the tensor cores have only a few
      // products queued.  (64 keys are 8192 bytes on in a tile.)
      const uint32_t q_hi = (uint32_t)(qd >> 32), k_hi = (uint32_t)(kd >> 32), v_hi = (uint32_t)(vd >> 32);
      auto scores = [&](int i, int h, uint32_t k_lo) {
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          const uint32_t o = (uint32_t)(k >> 2) * kSlabUnits + 2u * (k & 3);
          umma_f16_lh(tmem + (uint32_t)(2 * i + h) * kSub, (uint32_t)qd + (uint32_t)i * kTileUnits + o, q_hi, k_lo + 512u * h + o, k_hi,
                      idesc_s, k > 0);
        }
        umma_commit(smem_u32(&sh.sfull[i][h]));
      };
      // O_i += P_i V over part h, then the scores of the next tile's part h into its place
      // (the next tile may not be there yet: the products do not wait for it)
      auto part = [&](int i, int h, uint32_t v_lo, uint32_t k_lo, bool begin, bool more, bool keys_late, bool last, int st) {
        if (!wait(smem_u32(&sh.pready[i][h]), done[i] & 1, kStatusTimeoutAccEmpty)) return;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int k = 0; k < kSub / 16; ++k)
            umma_f16_ts(tmem + 256u + 128u * i, tmem + (uint32_t)(2 * i + h) * kSub + 8u * k, v_lo + 512u * h + (2048u / 16u) * k, v_hi,
                        idesc_o, !begin || k > 0);
          umma_commit(smem_u32(&sh.odone[i][h]));
          if (last) umma_commit(smem_u32(&sh.vempty[st]));
          if (more && !keys_late) {
            scores(i, h, k_lo);
            if (last) umma_commit(smem_u32(&sh.kempty[st ^ 1]));
          }
        }
        __syncwarp();
        if (keys_late && more) {
          if (!wait(smem_u32(&sh.kfull[st ^ 1]), ((tile + 1) >> 1) & 1, kStatusTimeoutFull)) return;
          tc_fence_after();
          if (leader) scores(i, h, k_lo);
          __syncwarp();
        }
      };
      while ((g = next_segment())) {
        const int tiles = g->k1 - g->k0;
        const bool two = g->s.n * a.group - g->rt * kRows > 128;
        const int st0 = tile & 1;
        wait(smem_u32(&sh.kfull[st0]), (tile >> 1) & 1, kStatusTimeoutFull);
        const uint32_t k0_lo = (uint32_t)kd + (uint32_t)st0 * kTileUnits;
        wait(smem_u32(&sh.qfull[0]), seg[0]++ & 1, kStatusTimeoutFull);
        tc_fence_after();
        if (ok && leader) {
          scores(0, 0, k0_lo);
          scores(0, 1, k0_lo);
        }
        __syncwarp();
        if (two) {
          wait(smem_u32(&sh.qfull[1]), seg[1]++ & 1, kStatusTimeoutFull);
          tc_fence_after();
          if (ok && leader) {
            scores(1, 0, k0_lo);
            scores(1, 1, k0_lo);
          }
          __syncwarp();
        }
        if (ok && leader) umma_commit(smem_u32(&sh.kempty[st0]));
        __syncwarp();
#pragma unroll 1
        for (int t = 0; t < tiles && ok; ++t, ++tile) {
          const int st = tile & 1;
          const bool more = t + 1 < tiles;
          const uint32_t v_lo = (uint32_t)vd + (uint32_t)st * kTileUnits, k_lo = (uint32_t)kd + (uint32_t)(st ^ 1) * kTileUnits;
          wait(smem_u32(&sh.vfull[st]), (tile >> 1) & 1, kStatusTimeoutFull);
          if (!ok) break;
          const bool late = more && !__all_sync(0xffffffffu, mbar_try_wait(smem_u32(&sh.kfull[st ^ 1]), ((tile + 1) >> 1) & 1));
          part(0, 0, v_lo, k_lo, t == 0, more, late, false, st);
          if (two) part(1, 0, v_lo, k_lo, t == 0, more, false, false, st);
          part(0, 1, v_lo, k_lo, false, more, false, !two, st);
          if (two) part(1, 1, v_lo, k_lo, false, more, false, true, st);
          ++done[0];
          if (two) ++done[1];
        }
      }
      // every product retires before TMEM is released
      volatile int no_abort = 0;
      if (leader) umma_commit(smem_u32(&sh.drained));
      __syncwarp();
      mbar_wait_bounded(smem_u32(&sh.drained), 0, &no_abort, a.status, kStatusTimeoutDrain, 400000000LL);
    } else if (warp == 13 && lane == 0) {
      // ---------------------------------------------------------- segments
      Walk<MODE> walk;
      const uint32_t size = sh.size;
      walk.begin(a, sh.u_begin, sh.u_end, (uint32_t)sh.base, sh.seq, sh.rt);
      for (int n = 0;; ++n) {
        Segment &g = sh.seg[n % kSegments];
        if (n >= kSegments && !mbar_wait_bounded(smem_u32(&sh.segempty[n % kSegments]), (n / kSegments - 1) & 1, &sh.abort, a.status,
                                                 kStatusTimeoutEmpty, kLimit))
          break;
        const bool found = walk.next(a, size, g);
        g.more = found;
        mbar_arrive(smem_u32(&sh.segfull[n % kSegments]));
        if (!found) break;
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  } else if (threadIdx.x == 0 && sh.abort) {
    count_rest<MODE>(a, sh, counters);
  }
}

// The parts of items that kBegin cut among many CTAs, added up in the order of their
// keys: eight rows a block, a thread four elements of one.  (A few rows over long
// beginnings have a part in every CTA; with 18 parts of 256 rows, the last CTA alone
// took as long for them as for the keys.)
constexpr int kPartsMost = 256;  // CTAs that a launch has at most
template <int DIM>
__global__ void __launch_bounds__(2 * DIM) kv_parts_k(const __grid_constant__ KvAttend a, const PromptSlot *slots, int ctas) {
  __shared__ float ms[8][kPartsMost + 1], ls[8][kPartsMost + 1], ts[8][kPartsMost + 1];
  constexpr int kThreadsRow = DIM / 4, kAtOnce = 8;
  const int rr = threadIdx.x & 7, c = threadIdx.x >> 3;
  const long long row = (long long)blockIdx.x * 8 + rr;
  pdl_wait_and_release();
  const bool marked = row < a.seqs.tokens * a.q_heads && __ldcg(kv_part_sums(a, row)).y == -1.f;
  if (!__syncthreads_or(marked)) return;
  const int4 w = marked ? __ldcg(reinterpret_cast<const int4 *>(kv_part(a, row))) : make_int4(0, -1, 0, 0);
  // (rows of no group are as the caller left them)
  const bool there = marked && w.x >= 0 && w.y >= w.x && w.y < ctas && (unsigned)w.z < kRows;
  const int i = w.z >> 7, r = w.z & 127, parts = there ? w.y - w.x + 1 : 0;
  auto slot = [&](int k) -> const PromptSlot & { return slots[2 * (2 * (w.x + k) + (k == 0 ? 1 : 0)) + i]; };
  auto load = [&](int k) {
    return k < parts ? __ldcg(reinterpret_cast<const float4 *>(&slot(k).acc[(c * 128 + r) * 4])) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  float4 u[kAtOnce];
#pragma unroll
  for (int k = 0; k < kAtOnce; ++k) u[k] = load(k);
  for (int k = c; k < parts; k += kThreadsRow) {
    const float zm = __ldcg(&slot(k).m[r]);
    ms[rr][k] = zm;
    ls[rr][k] = __ldcg(&slot(k).l[r]);
    ts[rr][k] = zm + log2_of(__ldcg(&slot(k).vref));
  }
  __syncthreads();  // (also: every thread has read the row's marks)
  if (!there) return;
  float m = -INFINITY, t = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < parts; ++k) {
    m = fmaxf(m, ms[rr][k]);
    t = fmaxf(t, ts[rr][k]);
  }
  for (int k0 = 0; k0 < parts; k0 += kAtOnce) {
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (k0 + k < parts) {
        const float zm = ms[rr][k0 + k], zl = ls[rr][k0 + k], wv = kv_share(ts[rr][k0 + k], t);
        if (zm != -INFINITY || zl != 0.f) l += kv_scaled(zl, zm - m);
        o[0] += u[k].x * wv, o[1] += u[k].y * wv, o[2] += u[k].z * wv, o[3] += u[k].w * wv;
      }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) u[k] = load(k0 + kAtOnce + k);
  }
  const float2 y = kv_norm(fast_exp2(t - m), l);
  __stcg(reinterpret_cast<float4 *>(kv_part(a, row) + 4 * c),
         make_float4(o[0] * y.x * y.y, o[1] * y.x * y.y, o[2] * y.x * y.y, o[3] * y.x * y.y));
  if (c == 0) __stcg(kv_part_sums(a, row), make_float2(m, l * kPromptToPart));
}

template <bool BF16, int DIM, int MODE>
cudaError_t launch_prompt(const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  static std::atomic<bool> attr_set[kAttrMaxDevices];
  const int bytes = (int)sizeof(PromptShared<DIM>) + 1024;
  const cudaError_t e = ensure_dynamic_smem(kv_prompt_k<BF16, DIM, MODE>, bytes, attr_set);
  if (e != cudaSuccess) return e;
  PromptSlot *const slots = reinterpret_cast<PromptSlot *>(static_cast<uint8_t *>(workspace) + kKvCounterBytes);
  return launch_kernel(kv_prompt_k<BF16, DIM, MODE>, dim3(sms), dim3(kThreads), (size_t)bytes, st, a, slots,
                       static_cast<unsigned *>(workspace));
}

template <int MODE>
cudaError_t launch_mode(bool bf16, const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  if (a.cache.dim == 64)
    return bf16 ? launch_prompt<true, 64, MODE>(a, workspace, sms, st) : launch_prompt<false, 64, MODE>(a, workspace, sms, st);
  return bf16 ? launch_prompt<true, 128, MODE>(a, workspace, sms, st) : launch_prompt<false, 128, MODE>(a, workspace, sms, st);
}

}  // namespace

size_t kv_prompt_workspace_bytes(int sms) { return sizeof(PromptSlot) * 4 * (size_t)sms; }

cudaError_t launch_kv_parts(const KvAttend &a, const void *workspace, int sms, cudaStream_t st) {
  if (sms > kPartsMost) return cudaErrorInvalidValue;
  const PromptSlot *slots = reinterpret_cast<const PromptSlot *>(static_cast<const uint8_t *>(workspace) + kKvCounterBytes);
  const unsigned grid = (unsigned)((a.seqs.tokens * a.q_heads + 7) / 8);
  if (a.cache.dim == 64) return launch_kernel(kv_parts_k<64>, dim3(grid), dim3(128), 0, st, a, slots, sms);
  return launch_kernel(kv_parts_k<128>, dim3(grid), dim3(256), 0, st, a, slots, sms);
}

bool kv_prompt_takes(const KvAttend &a) { return a.seqs.batch <= kMaxSeqs; }

cudaError_t launch_kv_prompt(bool bf16, int mode, const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  if (mode == kBegin) return launch_mode<kBegin>(bf16, a, workspace, sms, st);
  if (mode == kRest) return launch_mode<kRest>(bf16, a, workspace, sms, st);
  return launch_mode<kWhole>(bf16, a, workspace, sms, st);
}

}  // namespace ivb
