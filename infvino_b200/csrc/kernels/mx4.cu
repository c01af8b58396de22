// Matrices of microscaled 4-bit numbers (OCP MXFP4): quantisation, reading back,
// and the product out = X W^T.
//
// Blocks of 32 values of a row share the scale 2^e, e = floor(log2 of the largest
// magnitude) - 2, so that the largest code is 4 or 6; codes are x 2^-e rounded to
// the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even mantissa.  Both steps
// are exact but for that rounding.
#include <algorithm>

#include <cooperative_groups.h>

#include "../tma.h"
#include "kv_common.cuh"
#include "mx4.cuh"

namespace ivb {

namespace {

namespace cg = cooperative_groups;

// Eight values as codes, the first in the lowest four bits.
__device__ __forceinline__ uint32_t mx4_codes(const float (&f)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}
// Two codes as halves.
__device__ __forceinline__ float2 mx4_pair(uint32_t byte) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(r) : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2 *>(&r));
}
__device__ __forceinline__ float mx4_scale(uint32_t e) {  // 2^(e - 127)
  return e == 255 ? __uint_as_float(0x7fc00000u) : e == 0 ? 0x1p-127f : __uint_as_float(e << 23);
}

// Eight values of a block of 32, four neighbouring lanes each, as codes; the scale's
// byte is returned.  Maxima go by the bits, two values an instruction; a block with a
// NaN or an infinity takes another path.
template <bool BF16>
__device__ __forceinline__ int mx4_block(uint4 w, uint32_t &codes) {
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  uint32_t two = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
  two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, 1));
  two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, 2));
  uint32_t top = max(two & 0xffffu, two >> 16);
  float f[8];
  unpack8<BF16>(w, f);
  if (__any_sync(0xffffffffu, top >= kInf)) {  // (the largest finite one; NaN is 0)
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(f[i]);
      most = fmaxf(most, a < INFINITY ? a : 0.f);
      f[i] = f[i] != f[i] ? 0.f : f[i];
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    top = pack2<BF16>(most, 0.f) & 0xffffu;
  }
  const float most = BF16 ? __uint_as_float(top << 16) : __half2float(__ushort_as_half((unsigned short)top));
  const int e = max((int)(__float_as_uint(most) >> 23) - 2, 0);
  const float by = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= by;
  codes = mx4_codes(f);
  return e;
}

constexpr int kQuantThreads = 256, kQuantRows = kQuantThreads / 32;

// A warp takes N pieces of 256 of a row (one after another in a launch's x), a thread eight
// values of each, four lanes a block of 32; a CTA eight rows.  Memory bounds it (2 + 17 /
// 32 bytes a value), if few instructions are spent on a value (8191 x 8192: 33 us, 5.2
// TB/s; with maxima in f32 and a row and column for each piece 61).
template <bool BF16, int N>
__global__ void __launch_bounds__(kQuantThreads) mx4_quantize_k(const uint16_t *x, long long rows, long long padded,
                                                               long long stride, int vec, Mx4 m) {
  const int lane = threadIdx.x & 31, width = (int)m.width, chunks = (width + 127) / 128;
  const int c0 = blockIdx.x * (256 * N) + lane * 8;
  pdl_wait_and_release();
  for (long long r = (long long)blockIdx.y * kQuantRows + (threadIdx.x >> 5); r < padded; r += (long long)gridDim.y * kQuantRows) {
    uint4 w[N];
#pragma unroll
    for (int q = 0; q < N; ++q) w[q] = r < rows && c0 + 256 * q < width ? load8(x + r * stride + c0 + 256 * q, vec) : make_uint4(0, 0, 0, 0);
    uint32_t *const codes = reinterpret_cast<uint32_t *>(m.codes + r * (width / 2) + c0 / 2);
    uint8_t *const scales = m.scales + mx4_scale_at(r, c0 / 32, chunks);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      uint32_t word;
      const int e = mx4_block<BF16>(w[q], word);
      if (r < rows && c0 + 256 * q < width) codes[32 * q] = word;
      // four blocks' bytes in one word
      word = (uint32_t)e << (8 * ((lane >> 2) & 3));
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      word |= __shfl_xor_sync(0xffffffffu, word, 8);
      // (0 where there is no row; the matrix's rows behind the call's keep theirs)
      if ((lane & 15) == 0 && (r < rows || r >= m.rows) && c0 + 256 * q < chunks * 128) *reinterpret_cast<uint32_t *>(scales + 1024 * q) = word;
    }
  }
}

template <bool BF16, int N>
__global__ void __launch_bounds__(kQuantThreads) mx4_read_k(Mx4 m, long long rows, uint16_t *out, long long stride, int vec) {
  const int lane = threadIdx.x & 31, width = (int)m.width, chunks = (width + 127) / 128;
  const int c0 = blockIdx.x * (256 * N) + lane * 8;
  pdl_wait_and_release();
  for (long long r = (long long)blockIdx.y * kQuantRows + (threadIdx.x >> 5); r < rows; r += (long long)gridDim.y * kQuantRows) {
    const uint32_t *const codes = reinterpret_cast<const uint32_t *>(m.codes + r * (width / 2) + c0 / 2);
    const uint8_t *const scales = m.scales + mx4_scale_at(r, c0 / 32, chunks);
    uint32_t w[N], e[N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const bool there = c0 + 256 * q < width;
      w[q] = there ? codes[32 * q] : 0u;
      e[q] = there ? scales[1024 * q] : 0u;
    }
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const float s = mx4_scale(e[q]);
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = mx4_pair(w[q] >> (8 * i));
        f[2 * i] = p.x * s;
        f[2 * i + 1] = p.y * s;
      }
      if (c0 + 256 * q < width) store8(out + r * stride + c0 + 256 * q, pack8<BF16>(f), vec);
    }
  }
}

bool rows_vec(const void *p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

// ---------------------------------------------------------------- out = X W^T
//
// On the tensor cores in 4 bits: tcgen05.mma kind::mxf4 multiplies codes and
// applies the blocks' scales itself, 128 weight rows (a lane of TMEM each) by TN
// tokens (a column each) by 64 of the width an instruction, sums in f32.
//
// A tile is 128 weight rows (or twice that) x TN tokens, in stages of 256 of the width.  A
// CTA, one an SM, has some tiles; or, where tiles are fewer than SMs, the CTAs of a
// cluster have a part of one's stages each, and add the parts up out of one another's
// shared memory.  (Parts left in global memory for the last CTA: 38 us for 50 tokens x
// 4096 -> 6144, two weight tiles, against 13 without parts; an SM reads too slowly.)
//   warp 0     brings a stage's codes (TMA, 128-byte swizzled lines) and scales (as they
//              lie in memory: 512 bytes for 128 rows x 128 of the width)
//   warp 1     copies a stage's scales into TMEM and issues its products
//   warps 2 .. take a finished tile out of TMEM: a thread a weight row
// Where TMEM has two sets of accumulators a tile's products run while the one before it goes out.
//
// Every wait is bounded: a timeout sets the status word and an abort flag, all
// roles run out.
constexpr int kMm = 128;             // weight rows of an instruction
constexpr int kStageK = 256;         // of the width
constexpr int kFuseWarps = 4, kFuseTokens = 6;  // (warps that quantise tokens on the way, and how many tokens there may be)
constexpr int kMostSplit = 8;          // CTAs of a cluster that share a tile

// MT: weight tiles of 128 rows that share a stage's tokens.  What an SM gets from the L2 in
// a clock (some 38 bytes when all ask) bounds products with many tokens, and weights,
// from memory, queue up behind tokens in the copies of those with some: two weight tiles
// halve the tokens' part.  (4001 tokens x 4096 -> 14336: 121 us with 256 x 192 tiles, 1.18 GB
// into the SMs, the tensor cores 45 % of the time at work; the loads alone 93.)
template <int TN, int MT>
struct Tile {
  static constexpr int kRows = 128 * MT;                   // weight rows of a tile
  static constexpr int kRowTiles = (TN + 127) / 128;       // 128-row scale pieces of the tokens that a stage may touch
  static constexpr uint32_t kA = kRows * 128, kB = TN * 128, kSa = 1024 * MT, kSb = 1024 * kRowTiles;
  static constexpr uint32_t kStage = kA + kB + kSa + kSb;
  // Up to 64 tokens two CTAs fit on an SM: the next launch's CTAs set themselves up, and ask for
  // their weights, while this one's end.
  static constexpr int kCtas = TN <= 64 && MT == 1 ? 2 : 1;
  static constexpr int kStages = MT == 2 ? (TN > 64 ? 3 : 5) : TN == 16 ? 5 : TN <= 64 ? 4 : TN == 128 ? 6 : 5;
  static constexpr int kD = TN < 32 ? 32 : TN;             // columns of an accumulator
  // Two sets of accumulators where they fit.  (256 x 192: one; the loads go on while it is emptied.)
  static constexpr int kBufs = MT == 2 && TN > 64 ? 1 : 2;
  static constexpr int kScaleCols = 8 * (MT + kRowTiles);  // columns of a stage's scales
  static constexpr int kTmem = 512 / kCtas;
  static constexpr int kSmem = kStage * kStages + 1024;
  static constexpr int kThreads = 64 + 128 * MT;           // loads, products, and four warps for each weight tile's results
  // Many tokens: X and W change places (X's rows are the lanes), so that a thread has
  // neighbouring outputs of a token and stores 32 bytes at once.
  static constexpr bool kSwap = MT == 2 && TN > 64;
  static_assert(kBufs * MT * kD + kStages * kScaleCols <= kTmem, "TMEM");
  static_assert(kSmem * kCtas <= 224 << 10, "shared memory");
  static_assert(kSwap || kRows * TN * 4 <= kStage * kStages, "a part fits into the ring");
};

struct LinearArgs {
  CUtensorMap wmap, xmap;   // of the lanes' matrix (W, or X where they change places), of the columns'
  const uint16_t *x;        // FUSED: rows that are quantised on the way
  long long x_stride;
  int x_vec;
  const uint8_t *ws, *xs;   // their scales
  uint16_t *out;
  long long stride;
  int out_vec;              // rows of outputs on 32 bytes
  long long chunks;         // 128-wide scale pieces of a row
  int rows, outputs, width;
  int m_tiles, ks;          // tiles of lanes; stages of a tile
  uint32_t tiles, each;     // in all; of a CTA (or cluster)
  int split;                // CTAs of a cluster that share a tile
  int fresh;
  int *status;
};

// A CTA's tiles (m, t), one after the other; or, where `split` CTAs of a cluster have a
// tile, the CTA's part of its stages: k0 .. k1 - 1.
struct LinearWalk {
  uint32_t i, end;
  int m, t, k0, k1;
  __device__ __forceinline__ LinearWalk(const LinearArgs &a) {
    i = blockIdx.x / (uint32_t)a.split * a.each;
    end = min(a.tiles, i + a.each);
    const int rank = (int)(blockIdx.x % (uint32_t)a.split);
    k0 = rank * a.ks / a.split;
    k1 = (rank + 1) * a.ks / a.split;
  }
  __device__ __forceinline__ bool next(const LinearArgs &a) {
    if (i >= end) return false;
    m = (int)(i % (uint32_t)a.m_tiles);
    t = (int)(i / (uint32_t)a.m_tiles);
    ++i;
    return true;
  }
};

__device__ __forceinline__ void prefetch_2d(const void *map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// Scales of 128 rows x 128 of the width: 32 lanes x 16 bytes, to four columns (of all four lane quarters).
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t saddr) {
  const uint64_t desc = (uint64_t)((saddr & 0x3FFFFu) >> 4) | (8ull << 16) | (8ull << 32) | (1ull << 46);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
      : "memory");
}

// Sixteen outputs of a token, the first n of them.
template <bool BF16>
__device__ __forceinline__ void store_outputs(uint16_t *out, const float (&v)[16], int n, bool vec) {
  if (n >= 16 && vec) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pack2<BF16>(v[2 * i], v[2 * i + 1]);
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < n) out[i] = (uint16_t)pack2<BF16>(v[i], v[i]);
}

// FUSE: 0: X comes from memory in 4 bits; 1, 2: from halves / bf16 rows, which the CTA
// quantises itself, with kFuseWarps more warps.  Few rows: every CTA does it for its
// stages again, but a launch is saved, and the weights are on their way meanwhile.
template <int TN, int MT, bool BF16, int FUSE>
__global__ void __launch_bounds__(Tile<TN, MT>::kThreads + (FUSE ? 32 * kFuseWarps : 0), Tile<TN, MT>::kCtas)
    mx4_linear_k(const __grid_constant__ LinearArgs a) {
  using S = Tile<TN, MT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], accfull[2], accempty[2], drained;
  __shared__ uint32_t tmem_sh;
  __shared__ volatile int abort_sh;
  constexpr long long kLimit = kConvWaitLimitDefault;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float *const parts = reinterpret_cast<float *>(smem_raw + (ring - smem_u32(smem_raw)));  // [columns][128 rows], where a cluster has a tile
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(smem_u32(&full[i]), FUSE ? 2 : 1), mbar_init(smem_u32(&empty[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&accfull[i]), 1), mbar_init(smem_u32(&accempty[i]), 4 * MT);
    mbar_init(smem_u32(&drained), 1);
    abort_sh = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_sh), S::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh;

  if (warp == 0) {
    // ---- loads
    if (!a.fresh) {
      // (into the L2 for now, which is no reading: what comes before this launch may still write them)
      LinearWalk w(a);
      int left = S::kStages;
      while (left > 0 && w.next(a))
        for (int k = w.k0; k < w.k1 && left > 0; ++k, --left)
          if (elect_one()) prefetch_2d(&a.wmap, k * 128, w.m * S::kRows);
      pdl_wait();
    }
    // (after a fresh quantisation the weights are there already: their first stages come before it has ended)
    bool waited = !a.fresh;
    if (waited) pdl_release();
    uint32_t n = 0, pending = 0;  // stages begun; those whose tokens are still to be asked for
    LinearWalk w(a), tokens(a);
    bool more = tokens.next(a);
    int tk = tokens.k0;
    auto load_tokens = [&](uint32_t i) {
      if (FUSE) return;
      const uint32_t s = i % S::kStages, at = ring + s * S::kStage, bar = smem_u32(&full[s]);
      const int chunks = (int)min(2ll, a.chunks - 2 * tk);
      const long long rt = (long long)tokens.t * TN / 128;
      if (elect_one()) {
        tma_load_2d(at + S::kA, &a.xmap, bar, tk * 128, tokens.t * TN);
#pragma unroll
        for (int r = 0; r < S::kRowTiles; ++r)
          if ((rt + r) * 128 < (S::kSwap ? a.outputs : a.rows))
            bulk_load(at + S::kA + S::kB + S::kSa + 1024u * r, a.xs + ((rt + r) * a.chunks + 2 * tk) * 512, 512u * chunks, bar);
      }
      if (++tk == tokens.k1 && (more = tokens.next(a))) tk = tokens.k0;
    };
    bool ok = true;
    while (ok && w.next(a)) {
      for (int k = w.k0; k < w.k1 && ok; ++k, ++n) {
        const uint32_t s = n % S::kStages, wrap = n / S::kStages;
        if (wrap > 0 && !waited) {
          pdl_wait();
          pdl_release();
          waited = true;
          for (uint32_t i = n - pending; i < n; ++i) load_tokens(i);
          pending = 0;
        }
        if (wrap > 0) ok = mbar_wait_bounded(smem_u32(&empty[s]), (wrap - 1u) & 1u, &abort_sh, a.status, kStatusTimeoutEmpty, kLimit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t at = ring + s * S::kStage, bar = smem_u32(&full[s]);
        const int chunks = (int)min(2ll, a.chunks - 2 * k);
        const long long rt = (long long)w.t * TN / 128;
        const long long mt0 = (long long)w.m * MT;
        const int mts = MT == 1 || (mt0 + 1) * kMm < (S::kSwap ? a.rows : a.outputs) ? MT : 1;
        uint32_t pieces = (uint32_t)mts;
#pragma unroll
        for (int r = 0; r < S::kRowTiles; ++r) pieces += !FUSE && (rt + r) * 128 < (S::kSwap ? a.outputs : a.rows);
        if (elect_one()) {
          mbar_expect_tx(bar, S::kA + (FUSE ? 0 : S::kB) + 512u * chunks * pieces);
#pragma unroll
          for (int m = 0; m < MT; ++m) tma_load_2d(at + m * (kMm * 128), &a.wmap, bar, k * 128, w.m * S::kRows + m * kMm);
          for (int m = 0; m < mts; ++m) bulk_load(at + S::kA + S::kB + 1024u * m, a.ws + ((mt0 + m) * a.chunks + 2 * k) * 512, 512u * chunks, bar);
        }
        __syncwarp();
        if (waited)
          load_tokens(n);
        else
          ++pending;
      }
    }
    if (!waited) {
      pdl_wait();
      pdl_release();
      for (uint32_t i = n - pending; i < n; ++i) load_tokens(i);
    }
    if (abort_sh) {
      // copies in flight end before the CTA does
      for (uint32_t i = n > S::kStages ? n - S::kStages : 0; i < n; ++i)
        (void)mbar_wait_poll(smem_u32(&full[i % S::kStages]), (i / S::kStages) & 1u, kLimit);
    }
  } else if (warp == 1) {
    // ---- products
    constexpr uint32_t kIdesc = (1u << 7) | (1u << 10)         // A, B: e2m1
                                | ((uint32_t)(TN >> 3) << 17)  // N / 8
                                | (1u << 23)                   // scales: powers of two in 8 bits
                                | (1u << 27);                  // M / 128
    uint32_t n = 0, tile = 0;
    LinearWalk w(a);
    bool ok = true;
    while (ok && w.next(a)) {
      const uint32_t buf = tile % S::kBufs, use = tile / S::kBufs;
      if (use > 0) ok = mbar_wait_bounded(smem_u32(&accempty[buf]), (use - 1u) & 1u, &abort_sh, a.status, kStatusTimeoutAccEmpty, kLimit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d = tmem + buf * (MT * S::kD);
      const uint32_t group = (uint32_t)(((long long)w.t * TN % 128) / 32);  // first 32 tokens of the tile in their scale piece
      for (int k = w.k0; k < w.k1; ++k, ++n) {
        const uint32_t s = n % S::kStages;
        ok = mbar_wait_bounded(smem_u32(&full[s]), (n / S::kStages) & 1u, &abort_sh, a.status, kStatusTimeoutFull, kLimit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t at = ring + s * S::kStage;
        const uint32_t sa = tmem + S::kBufs * MT * S::kD + s * S::kScaleCols, sb = sa + 8 * MT;  // (four columns for each 128 rows and 128 of the width)
        const int steps = min(kStageK / 64, (a.width - k * kStageK + 63) / 64);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int m = 0; m < MT; ++m) scales_to_tmem(sa + 8 * m + 4 * c, at + S::kA + S::kB + 1024 * m + 512 * c);
#pragma unroll
            for (int r = 0; r < S::kRowTiles; ++r)
              scales_to_tmem(sb + 4 * S::kRowTiles * c + 4 * r, at + S::kA + S::kB + S::kSa + 1024 * r + 512 * c);
          }
          const uint64_t ad = smem_desc_kmajor(at, 128), bd = smem_desc_kmajor(at + S::kA, 128);
          for (int i = 0; i < steps; ++i) {
            const uint32_t id = (uint32_t)(i & 1) * 2u, c = (uint32_t)i >> 1;  // which two of the four scales of 128
#pragma unroll
            for (int m = 0; m < MT; ++m)
              umma_mxf4(d + m * S::kD, ad + m * (kMm * 128 / 16) + 2 * i, bd + 2 * i, kIdesc | (id << 29) | (id << 4), sa + 8 * m + 4 * c,
                        sb + 4 * S::kRowTiles * c + group, k > w.k0 || i > 0);
          }
          umma_commit(smem_u32(&empty[s]));
          if (k == w.k1 - 1) umma_commit(smem_u32(&accfull[buf]));
        }
        __syncwarp();
      }
      ++tile;
    }
    // what was issued ends before TMEM is given back
    if (elect_one()) umma_commit(smem_u32(&drained));
    __syncwarp();
    (void)mbar_wait_poll(smem_u32(&drained), 0, kLimit);
  } else if (FUSE && warp >= 2 + 4 * MT) {
    // ---- tokens: a warp every kFuseWarps-th stage, its rows as mx4_quantize_k takes them.
    // (A wait tells one phase of a barrier from the next, not from the one after that.
    // The warp has waited for the place of the stage kFuseWarps before, so that with at
    // most kStages warps the phase before the one that it waits for is over.)
    static_assert(!FUSE || kFuseWarps <= S::kStages, "phases");
    constexpr bool XB = FUSE == 2;
    constexpr int kEach = 8;  // rows in flight
    const uint32_t mine = (uint32_t)warp - (2 + 4 * MT);
    pdl_wait();
    uint32_t n = 0;
    LinearWalk w(a);
    bool ok = true;
    while (ok && w.next(a)) {
      for (int k = w.k0; k < w.k1; ++k, ++n) {
        if (n % kFuseWarps != mine) continue;
        const uint32_t s = n % S::kStages, wrap = n / S::kStages;
        uint8_t *const at = smem_raw + (ring - smem_u32(smem_raw)) + s * S::kStage + S::kA;
        const int c = k * kStageK + lane * 8;
        for (int r0 = 0; r0 < a.rows; r0 += kEach) {
          uint4 now[kEach];
#pragma unroll
          for (int i = 0; i < kEach; ++i)
            now[i] = r0 + i < a.rows && c < a.width ? load8(a.x + (r0 + i) * a.x_stride + c, a.x_vec) : make_uint4(0, 0, 0, 0);
          if (r0 == 0 && wrap > 0) {
            ok = mbar_wait_bounded(smem_u32(&empty[s]), (wrap - 1u) & 1u, &abort_sh, a.status, kStatusTimeoutEmpty, kLimit);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            const int r = r0 + i;
            if (r >= a.rows) break;
            uint32_t codes;
            const int e = mx4_block<XB>(now[i], codes);
            *reinterpret_cast<uint32_t *>(at + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = codes;
            uint32_t word = (uint32_t)e << (8 * ((lane >> 2) & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            if ((lane & 15) == 0) *reinterpret_cast<uint32_t *>(at + S::kB + S::kSa + (lane >> 4) * 512 + r * 16) = word;
          }
        }
        if (!ok) break;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&full[s]));
      }
    }
  } else {
    // ---- results: thread = weight row, four warps the four lane quarters
    const int quarter = warp & 3, row = quarter * 32 + lane, mt = (warp - 2) >> 2;
    pdl_wait();
    uint32_t tile = 0;
    LinearWalk w(a);
    bool ok = true;
    constexpr int kStep = 16;
    while (w.next(a)) {
      const uint32_t buf = tile % S::kBufs, use = tile / S::kBufs;
      if (ok) ok = mbar_wait_bounded(smem_u32(&accfull[buf]), use & 1u, &abort_sh, a.status, kStatusTimeoutAcc, kLimit);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const uint32_t d = tmem + (buf * MT + mt) * S::kD + ((uint32_t)quarter << 21);
      const int t0 = w.t * TN, count = min(TN, (S::kSwap ? a.outputs : a.rows) - t0);
      const long long n = (long long)w.m * S::kRows + mt * kMm + row;
      // (swapped: the lanes are tokens, the columns outputs)
      const long long lanes = S::kSwap ? a.rows : a.outputs;
      uint16_t *out = S::kSwap ? a.out + n * a.stride + t0 : a.out + (long long)t0 * a.stride + n;
      if (ok) {
#pragma unroll 1
        for (int c = 0; c < count; c += kStep) {
          uint32_t r[16];
          tmem_ld16(d + c, r);
          tmem_ld_wait();
          float v[kStep];
#pragma unroll
          for (int i = 0; i < kStep; ++i) v[i] = __uint_as_float(r[i]);
          if (a.split > 1) {  // (all products have read their operands: the ring is free)
#pragma unroll
            for (int i = 0; i < kStep; ++i) parts[(mt * TN + c + i) * kMm + row] = v[i];
          } else if (n < lanes) {
            if constexpr (S::kSwap) {
              store_outputs<BF16>(out + c, v, count - c, a.out_vec);
            } else {
#pragma unroll
              for (int i = 0; i < kStep; ++i)
                if (c + i < count) out[(c + i) * a.stride] = (uint16_t)pack2<BF16>(v[i], v[i]);
            }
          }
        }
      }
      // the accumulator is free again
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&accempty[buf]));
      ++tile;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, S::kTmem);
  if constexpr (!S::kSwap) {
    if (a.split > 1) {
      // the cluster's parts, added up in the order of their stages: a CTA some of the columns
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      if (warp >= 2 && warp < 2 + 4 * MT) {
        const int row = (warp & 3) * 32 + lane, mt = (warp - 2) >> 2;
        LinearWalk w(a);
        w.next(a);
        const int t0 = w.t * TN, count = min(TN, a.rows - t0), per = (count + a.split - 1) / a.split;
        const int c0 = (int)(blockIdx.x % (uint32_t)a.split) * per, c1 = min(count, c0 + per);
        const long long n = (long long)w.m * S::kRows + mt * kMm + row;
        const float *from[kMostSplit];
#pragma unroll
        for (int q = 0; q < kMostSplit; ++q) from[q] = cluster.map_shared_rank(parts, min(q, a.split - 1)) + mt * TN * kMm + row;
        constexpr int kCols = TN <= 32 ? 2 : 8;  // columns whose parts are asked for together
        for (int c = c0; c < c1; c += kCols) {
          float v[kCols][kMostSplit];
#pragma unroll
          for (int q = 0; q < kMostSplit; ++q)
            if (q < a.split)
#pragma unroll
              for (int i = 0; i < kCols; ++i) v[i][q] = c + i < c1 ? from[q][(c + i) * kMm] : 0.f;
#pragma unroll
          for (int i = 0; i < kCols; ++i) {
            float sum = v[i][0];
#pragma unroll
            for (int q = 1; q < kMostSplit; ++q)
              if (q < a.split) sum += v[i][q];
            if (c + i < c1 && n < a.outputs) a.out[(t0 + c + i) * a.stride + n] = (uint16_t)pack2<BF16>(sum, sum);
          }
        }
      }
      cluster.sync();  // (the parts have been read)
    }
  }
}

// How a product is divided: tokens and weight tiles of a tile, CTAs that share one (or tiles that one CTA has).
struct LinearPlan {
  int tn, mt, split;
  uint32_t tiles, each;
};

// How many clusters of `split` CTAs run at a time (asked once for a device: SMs come in
// groups, and a cluster lies in one of them).
int linear_clusters(int device, int mt, int split) {
  static std::atomic<int> known[kAttrMaxDevices][2][kMostSplit + 1];
  const bool tracked = device >= 0 && device < kAttrMaxDevices;
  int n = tracked ? known[device][mt - 1][split].load(std::memory_order_relaxed) : 0;
  if (n) return n - 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)split);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto ask = [&](auto kernel, int threads, int bytes) {
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)bytes;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
  };
  if (mt == 2)
    ask(mx4_linear_k<64, 2, false, 0>, Tile<64, 2>::kThreads, Tile<64, 2>::kSmem);
  else  // (alone on its SM, as if others' blocks had the second places)
    ask(mx4_linear_k<128, 1, false, 0>, Tile<128, 1>::kThreads, Tile<128, 1>::kSmem);
  if (tracked) known[device][mt - 1][split].store(n + 1, std::memory_order_relaxed);
  return n;
}

LinearPlan linear_plan(const Mx4Linear &l) {
  const long long ks = (l.w.width + kStageK - 1) / kStageK;
  LinearPlan best{};
  double least = 1e300;
  const double memory = l.w.rows * l.w.width * 17.0 / 32 / 6.2e6;
  struct Form {
    int tn, mt;
  };
  for (const Form f : {Form{16, 1}, Form{16, 2}, Form{32, 1}, Form{32, 2}, Form{64, 1}, Form{64, 2}, Form{128, 1}, Form{192, 1}, Form{192, 2}}) {
    const int tn = f.tn, mt = f.mt;
    if (tn < 64 && l.x.rows > tn) continue;
    if (tn > 16 && tn / 2 >= l.x.rows) continue;
    const bool swap = mt == 2 && tn > 64;  // (Tile::kSwap)
    const long long lanes = swap ? l.x.rows : l.w.rows, columns = swap ? l.w.rows : l.x.rows;
    const long long tiles = (lanes + 128 * mt - 1) / (128 * mt) * ((columns + tn - 1) / tn);
    if (tiles > 0x7fffffffLL) continue;
    // Us, from measurements at 1 to 4001 tokens (within some 10 %): a stage's bytes into an
    // SM, weights slower than tokens, or all weights out of memory; starting and ending; a
    // tile's results where nothing else runs meanwhile, or a cluster's gathering.
    const double weights = mt * kMm * 136.0, tokens = tn * 136.0;
    for (int split = 1; split <= (swap ? 1 : kMostSplit); ++split) {
      if (split > 1 && (split > ks || tiles > linear_clusters(l.device, mt, split))) continue;
      const long long each = split > 1 ? 1 : (tiles + l.sms - 1) / l.sms;
      const double stages = each * ((ks + split - 1) / split) * (weights / (mt == 2 ? 85e3 : 64e3) + tokens / 100e3);
      const double us = 4.0 + std::max(stages, memory) + each * (swap ? 2.0 : 0.0) + (each - 1) * 1.5 + (split > 1 ? 1.0 + 0.03 * tn * mt : 0.0);
      if (us < least) {
        least = us;
        best = LinearPlan{tn, mt, split, (uint32_t)tiles, (uint32_t)each};
      }
    }
  }
  return best;
}

template <int TN, int MT, bool BF16, int FUSE>
cudaError_t linear_tiles(const Mx4Linear &l, const LinearPlan &plan, cudaStream_t st) {
  using S = Tile<TN, MT>;
  LinearArgs a;
  std::string err;
  const uint64_t pitch = (uint64_t)l.w.width / 2;
  const Mx4 &lanes = S::kSwap ? l.x : l.w, &columns = S::kSwap ? l.w : l.x;
  if (!encode_tiled_bytes(&a.wmap, lanes.codes, pitch, (uint64_t)lanes.rows, pitch, kMm, &err)) return cudaErrorInvalidValue;
  if (!FUSE && !encode_tiled_bytes(&a.xmap, columns.codes, pitch, (uint64_t)columns.rows, pitch, TN, &err)) return cudaErrorInvalidValue;
  a.x = static_cast<const uint16_t *>(l.rows);
  a.x_stride = l.x_stride;
  a.x_vec = rows_vec(l.rows, l.x_stride);
  a.ws = lanes.scales, a.xs = columns.scales;
  a.out = static_cast<uint16_t *>(l.out);
  a.stride = l.stride;
  a.out_vec = reinterpret_cast<uintptr_t>(l.out) % 32 == 0 && l.stride % 16 == 0;
  a.chunks = (l.w.width + 127) / 128;
  a.rows = (int)l.x.rows, a.outputs = (int)l.w.rows, a.width = (int)l.w.width;
  a.m_tiles = (int)((lanes.rows + S::kRows - 1) / S::kRows);
  a.ks = (int)((l.w.width + kStageK - 1) / kStageK);
  a.tiles = plan.tiles;
  a.each = plan.each;
  a.split = plan.split;
  a.fresh = l.rows && !FUSE && !S::kSwap;
  a.status = l.status;
  static std::atomic<bool> attr_set[kAttrMaxDevices];
  const cudaError_t e = ensure_dynamic_smem(mx4_linear_k<TN, MT, BF16, FUSE>, S::kSmem, attr_set);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((plan.tiles + plan.each - 1) / plan.each * (unsigned)plan.split);
  cfg.blockDim = dim3(S::kThreads + (FUSE ? 32 * kFuseWarps : 0));
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (plan.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)plan.split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (g_launch_pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = (unsigned)n;
  return cudaLaunchKernelEx(&cfg, mx4_linear_k<TN, MT, BF16, FUSE>, a);
}

template <bool BF16>
cudaError_t linear_rows(const Mx4Linear &l, cudaStream_t st) {
  const LinearPlan p = linear_plan(l);
  if (!p.tn) return cudaErrorInvalidValue;
  // (one launch / two: 4096 -> 6144, 1 token 7.4 / 8.9 us, 4 8.0 / 9.4, 8 9.6 / 9.7, 16 13.8 / 10.3;
  // 8192 -> 28672, 1 22.6 / 24.6, 4 23.3 / 24.5, 8 27.2 / 24.6)
  if (p.tn == 16 && l.rows && l.x.rows <= kFuseTokens) {
    if (p.mt == 2) return l.x_bf16 ? linear_tiles<16, 2, BF16, 2>(l, p, st) : linear_tiles<16, 2, BF16, 1>(l, p, st);
    return l.x_bf16 ? linear_tiles<16, 1, BF16, 2>(l, p, st) : linear_tiles<16, 1, BF16, 1>(l, p, st);
  }
  if (l.rows) {
    const cudaError_t e = launch_mx4_quantize(l.x_bf16, l.rows, l.x.rows, l.x_stride, l.x, l.sms, st);
    if (e != cudaSuccess) return e;
  }
  switch (p.tn * 4 + p.mt) {
    case 16 * 4 + 1: return linear_tiles<16, 1, BF16, 0>(l, p, st);
    case 16 * 4 + 2: return linear_tiles<16, 2, BF16, 0>(l, p, st);
    case 32 * 4 + 1: return linear_tiles<32, 1, BF16, 0>(l, p, st);
    case 32 * 4 + 2: return linear_tiles<32, 2, BF16, 0>(l, p, st);
    case 64 * 4 + 1: return linear_tiles<64, 1, BF16, 0>(l, p, st);
    case 64 * 4 + 2: return linear_tiles<64, 2, BF16, 0>(l, p, st);
    case 128 * 4 + 1: return linear_tiles<128, 1, BF16, 0>(l, p, st);
    case 192 * 4 + 1: return linear_tiles<192, 1, BF16, 0>(l, p, st);
    default: return linear_tiles<192, 2, BF16, 0>(l, p, st);
  }
}

// Pieces of a warp, and the grid: few values go to many warps.
dim3 quant_grid(long long width, long long rows, int sms, bool &four) {
  const long long blocks = (rows + kQuantRows - 1) / kQuantRows;
  four = width > 256 && blocks * ((width + 1023) / 1024) >= sms * 2;
  const long long x = (width + (four ? 1023 : 255)) / (four ? 1024 : 256);
  return dim3((unsigned)x, (unsigned)std::min(blocks, std::max(1ll, sms * 8 / x)));
}

template <bool BF16>
cudaError_t quantize(const void *x, long long rows, long long stride, const Mx4 &m, int sms, cudaStream_t st) {
  const long long padded = (rows + 127) / 128 * 128;  // (scale bytes of rows that are not there are 0)
  bool four;
  const dim3 grid = quant_grid(m.width, padded, sms, four);
  const uint16_t *p = static_cast<const uint16_t *>(x);
  if (four) return launch_kernel(mx4_quantize_k<BF16, 4>, grid, dim3(kQuantThreads), 0, st, p, rows, padded, stride, (int)rows_vec(x, stride), m);
  return launch_kernel(mx4_quantize_k<BF16, 1>, grid, dim3(kQuantThreads), 0, st, p, rows, padded, stride, (int)rows_vec(x, stride), m);
}
template <bool BF16>
cudaError_t read(const Mx4 &m, long long rows, void *out, long long stride, int sms, cudaStream_t st) {
  bool four;
  const dim3 grid = quant_grid(m.width, rows, sms, four);
  uint16_t *p = static_cast<uint16_t *>(out);
  if (four) return launch_kernel(mx4_read_k<BF16, 4>, grid, dim3(kQuantThreads), 0, st, m, rows, p, stride, (int)rows_vec(out, stride));
  return launch_kernel(mx4_read_k<BF16, 1>, grid, dim3(kQuantThreads), 0, st, m, rows, p, stride, (int)rows_vec(out, stride));
}

}  // namespace

cudaError_t launch_mx4_quantize(bool bf16, const void *x, long long rows, long long stride, const Mx4 &m, int sms,
                                cudaStream_t st) {
  return bf16 ? quantize<true>(x, rows, stride, m, sms, st) : quantize<false>(x, rows, stride, m, sms, st);
}

cudaError_t launch_mx4_read(bool bf16, const Mx4 &m, long long rows, void *out, long long stride, int sms, cudaStream_t st) {
  return bf16 ? read<true>(m, rows, out, stride, sms, st) : read<false>(m, rows, out, stride, sms, st);
}

cudaError_t launch_mx4_linear(const Mx4Linear &a, cudaStream_t st) {
  return a.bf16 ? linear_rows<true>(a, st) : linear_rows<false>(a, st);
}

}  // namespace ivb
