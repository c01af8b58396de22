// Matrices of microscaled 4-bit numbers (OCP MXFP4): quantisation, reading back,
// and the product out = X W^T.
//
// Blocks of 32 values of a row share the scale 2^e, e = floor(log2 of the largest
// magnitude) - 2, so that the largest code is 4 or 6; codes are x 2^-e rounded to
// the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even mantissa.  Both steps
// are exact but for that rounding.
#include <algorithm>

#include "../tma.h"
#include "kv_common.cuh"
#include "mx4.cuh"

namespace ivb {

namespace {

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

constexpr int kQuantThreads = 256, kQuantRows = kQuantThreads / 32;

// A warp takes N pieces of 256 of a row (one after another in a launch's x), a thread eight
// values of each, four lanes a block of 32; a CTA eight rows.  Memory bounds it (2 + 17 /
// 32 bytes a value), if few instructions are spent on a value: maxima go by the bits,
// two values an instruction, and a block with a NaN or an infinity takes another path.
// (8191 x 8192: TODO us.)
template <bool BF16, int N>
__global__ void __launch_bounds__(kQuantThreads) mx4_quantize_k(const uint16_t *x, long long rows, long long padded,
                                                               long long stride, int vec, Mx4 m) {
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
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
      uint32_t two = __vmaxu2(__vmaxu2(w[q].x & 0x7fff7fffu, w[q].y & 0x7fff7fffu), __vmaxu2(w[q].z & 0x7fff7fffu, w[q].w & 0x7fff7fffu));
      two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, 1));
      two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, 2));
      uint32_t top = max(two & 0xffffu, two >> 16);
      float f[8];
      unpack8<BF16>(w[q], f);
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
      if (r < rows && c0 + 256 * q < width) codes[32 * q] = mx4_codes(f);
      // four blocks' bytes in one word
      uint32_t word = (uint32_t)e << (8 * ((lane >> 2) & 3));
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      word |= __shfl_xor_sync(0xffffffffu, word, 8);
      if ((lane & 15) == 0 && c0 + 256 * q < chunks * 128) *reinterpret_cast<uint32_t *>(scales + 1024 * q) = word;
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
// A tile is 128 weight rows x TN tokens; its units are stages of 256 of the width.
// The units are divided over the CTAs, one an SM, evenly (few tiles: a tile is cut
// over CTAs, its parts are joined by the last of them to arrive, in their order) or
// by whole tiles.
//   warp 0     brings a stage's codes (TMA, 128-byte swizzled lines) and scales (as they
//              lie in memory: 512 bytes for 128 rows x 128 of the width)
//   warp 1     copies a stage's scales into TMEM and issues its products
//   warps 2-5  take a finished tile out of TMEM: a thread a weight row
// Two accumulators: a tile's products run while the one before it goes out.
//
// Every wait is bounded: a timeout sets the status word and an abort flag, all
// roles run out, and parts of cut tiles are counted all the same.
constexpr int kMm = 128;             // weight rows of a tile
constexpr int kStageK = 256;         // of the width
constexpr int kLinearThreads = 192;
constexpr int kMaxTokens = 192;      // of a tile

template <int TN>
struct Tile {
  static constexpr int kRowTiles = (TN + 127) / 128;       // 128-row scale pieces a stage may touch
  static constexpr uint32_t kA = kMm * 128, kB = TN * 128, kSa = 1024, kSb = 1024 * kRowTiles;
  static constexpr uint32_t kStage = kA + kB + kSa + kSb;
  static constexpr int kStages = TN == 16 ? 10 : TN == 32 ? 9 : TN == 64 ? 8 : TN == 128 ? 6 : 5;
  static constexpr int kD = TN < 32 ? 32 : TN;             // columns of an accumulator
  static constexpr int kScaleCols = 8 + 8 * kRowTiles;     // columns of a stage's scales
  static constexpr int kSmem = kStage * kStages + 1024;
  static_assert(2 * kD + kStages * kScaleCols <= 512, "TMEM");
};

struct LinearArgs {
  CUtensorMap wmap, xmap;
  const uint8_t *ws, *xs;   // scales
  uint16_t *out;
  long long stride;
  long long chunks;         // 128-wide scale pieces of a row
  int rows, outputs, width;
  int m_tiles, ks;          // weight tiles; stages of a tile
  uint32_t units, size;     // in all; of a CTA's share
  int fresh;
  float *slots;
  unsigned *counters;
  int *status;
};

// A CTA's share, tile by tile: stages k0 .. k1 - 1 of tile (m, t).
struct LinearWalk {
  uint32_t u, end;
  int m, t, k0, k1;
  int first_cta, last_cta;
  __device__ __forceinline__ LinearWalk(const LinearArgs &a) {
    u = min(a.units, blockIdx.x * a.size);
    end = min(a.units, u + a.size);
  }
  __device__ __forceinline__ bool next(const LinearArgs &a) {
    if (u >= end) return false;
    const uint32_t ks = (uint32_t)a.ks, tile = u / ks, begin = tile * ks;
    m = (int)(tile % (uint32_t)a.m_tiles);
    t = (int)(tile / (uint32_t)a.m_tiles);
    k0 = (int)(u - begin);
    k1 = (int)(min(end, begin + ks) - begin);
    first_cta = (int)(begin / a.size);
    last_cta = (int)((begin + ks - 1) / a.size);
    u = begin + (uint32_t)k1;
    return true;
  }
};

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

template <int TN, bool BF16>
__global__ void __launch_bounds__(kLinearThreads, 1) mx4_linear_k(const __grid_constant__ LinearArgs a) {
  using S = Tile<TN>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], accfull[2], accempty[2], drained;
  __shared__ uint32_t tmem_sh;
  __shared__ volatile int abort_sh;
  __shared__ int last_sh;
  constexpr long long kLimit = kConvWaitLimitDefault;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(smem_u32(&full[i]), 1), mbar_init(smem_u32(&empty[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&accfull[i]), 1), mbar_init(smem_u32(&accempty[i]), 4);
    mbar_init(smem_u32(&drained), 1);
    abort_sh = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_sh), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh;

  if (warp == 0) {
    // ---- loads
    if (!a.fresh) pdl_wait();
    // (after a fresh quantisation the weights are there already: their first stages come before it has ended)
    bool waited = !a.fresh;
    if (waited) pdl_release();
    uint32_t n = 0, pending = 0;  // stages begun; those whose tokens are still to be asked for
    LinearWalk w(a), tokens(a);
    bool more = tokens.next(a);
    int tk = tokens.k0;
    auto load_tokens = [&](uint32_t i) {
      const uint32_t s = i % S::kStages, at = ring + s * S::kStage, bar = smem_u32(&full[s]);
      const int chunks = (int)min(2ll, a.chunks - 2 * tk);
      const long long rt = (long long)tokens.t * TN / 128;
      if (elect_one()) {
        tma_load_2d(at + S::kA, &a.xmap, bar, tk * 128, tokens.t * TN);
#pragma unroll
        for (int r = 0; r < S::kRowTiles; ++r)
          if ((rt + r) * 128 < a.rows)
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
        uint32_t pieces = 1;
#pragma unroll
        for (int r = 0; r < S::kRowTiles; ++r) pieces += (rt + r) * 128 < a.rows;
        if (elect_one()) {
          mbar_expect_tx(bar, S::kA + S::kB + 512u * chunks * pieces);
          tma_load_2d(at, &a.wmap, bar, k * 128, w.m * kMm);
          bulk_load(at + S::kA + S::kB, a.ws + ((long long)w.m * a.chunks + 2 * k) * 512, 512u * chunks, bar);
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
      const uint32_t buf = tile & 1u, use = tile >> 1;
      if (use > 0) ok = mbar_wait_bounded(smem_u32(&accempty[buf]), (use - 1u) & 1u, &abort_sh, a.status, kStatusTimeoutAccEmpty, kLimit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d = tmem + buf * S::kD;
      const uint32_t group = (uint32_t)(((long long)w.t * TN % 128) / 32);  // first 32 tokens of the tile in their scale piece
      for (int k = w.k0; k < w.k1; ++k, ++n) {
        const uint32_t s = n % S::kStages;
        ok = mbar_wait_bounded(smem_u32(&full[s]), (n / S::kStages) & 1u, &abort_sh, a.status, kStatusTimeoutFull, kLimit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t at = ring + s * S::kStage;
        const uint32_t sc = tmem + 2 * S::kD + s * S::kScaleCols;
        const int steps = min(kStageK / 64, (a.width - k * kStageK + 63) / 64);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            scales_to_tmem(sc + 4 * c, at + S::kA + S::kB + 512 * c);
#pragma unroll
            for (int r = 0; r < S::kRowTiles; ++r)
              scales_to_tmem(sc + 8 + 4 * S::kRowTiles * c + 4 * r, at + S::kA + S::kB + S::kSa + 1024 * r + 512 * c);
          }
          const uint64_t ad = smem_desc_kmajor(at, 128), bd = smem_desc_kmajor(at + S::kA, 128);
          for (int i = 0; i < steps; ++i) {
            const uint32_t id = (uint32_t)(i & 1) * 2u, c = (uint32_t)i >> 1;  // which two of the four scales of 128
            umma_mxf4(d, ad + 2 * i, bd + 2 * i, kIdesc | (id << 29) | (id << 4), sc + 4 * c, sc + 8 + 4 * S::kRowTiles * c + group,
                      k > w.k0 || i > 0);
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
  } else {
    // ---- results: thread = weight row, four warps the four lane quarters
    const int quarter = warp & 3, row = quarter * 32 + lane;
    pdl_wait();
    uint32_t tile = 0;
    LinearWalk w(a);
    bool ok = true;
    constexpr int kStep = 16;
    while (w.next(a)) {
      const uint32_t buf = tile & 1u, use = tile >> 1;
      if (ok) ok = mbar_wait_bounded(smem_u32(&accfull[buf]), use & 1u, &abort_sh, a.status, kStatusTimeoutAcc, kLimit);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const uint32_t d = tmem + buf * S::kD + ((uint32_t)quarter << 21);
      const int t0 = w.t * TN, count = min(TN, a.rows - t0);
      const long long n = (long long)w.m * kMm + row;
      const bool whole = w.k0 == 0 && w.k1 == a.ks;
      uint16_t *out = a.out + (long long)t0 * a.stride + n;
      bool last = false;
      if (!whole) {
        float *slot = a.slots + (size_t)(2 * blockIdx.x + (w.k0 == 0)) * (kMm * TN);
        if (ok) {
#pragma unroll 1
          for (int c = 0; c < count; c += kStep) {
            uint32_t r[16];
            tmem_ld16(d + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < kStep; ++i)
              if (c + i < count) __stcg(&slot[(c + i) * kMm + row], __uint_as_float(r[i]));
          }
        }
        __threadfence();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (threadIdx.x == 64) {
          __threadfence();
          const unsigned parts = (unsigned)(w.last_cta - w.first_cta + 1);
          const bool done = atomicAdd(&a.counters[w.first_cta], 1u) == parts - 1;
          if (done) {
            atomicExch(&a.counters[w.first_cta], 0u);
            __threadfence();
          }
          last_sh = done;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        last = last_sh != 0;
      }
      if (ok && (whole || last)) {
#pragma unroll 1
        for (int c = 0; c < count; c += kStep) {
          float v[kStep];
          if (whole) {
            uint32_t r[16];
            tmem_ld16(d + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < kStep; ++i) v[i] = __uint_as_float(r[i]);
          } else {
#pragma unroll
            for (int i = 0; i < kStep; ++i) v[i] = 0.f;
            for (int z = w.first_cta; z <= w.last_cta; ++z) {
              const float *slot = a.slots + (size_t)(2 * z + (z == w.first_cta)) * (kMm * TN);
#pragma unroll
              for (int i = 0; i < kStep; ++i)
                if (c + i < count) v[i] += __ldcg(&slot[(c + i) * kMm + row]);
            }
          }
          if (n < a.outputs) {
#pragma unroll
            for (int i = 0; i < kStep; ++i)
              if (c + i < count) out[(c + i) * a.stride] = (uint16_t)pack2<BF16>(v[i], v[i]);
          }
        }
      }
      // the accumulator is free again
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&accempty[buf]));
      if (!whole) asm volatile("bar.sync 1, 128;" ::: "memory");  // (last_sh has been read)
      ++tile;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

template <int TN, bool BF16>
cudaError_t linear_tiles(const Mx4Linear &l, cudaStream_t st) {
  using S = Tile<TN>;
  LinearArgs a;
  std::string err;
  const uint64_t pitch = (uint64_t)l.w.width / 2;
  if (!encode_tiled_bytes(&a.wmap, l.w.codes, pitch, (uint64_t)l.w.rows, pitch, kMm, &err) ||
      !encode_tiled_bytes(&a.xmap, l.x.codes, pitch, (uint64_t)l.x.rows, pitch, TN, &err))
    return cudaErrorInvalidValue;
  a.ws = l.w.scales, a.xs = l.x.scales;
  a.out = static_cast<uint16_t *>(l.out);
  a.stride = l.stride;
  a.chunks = (l.w.width + 127) / 128;
  a.rows = (int)l.x.rows, a.outputs = (int)l.w.rows, a.width = (int)l.w.width;
  a.m_tiles = (int)((l.w.rows + kMm - 1) / kMm);
  a.ks = (int)((l.w.width + kStageK - 1) / kStageK);
  const long long tiles = (long long)a.m_tiles * ((l.x.rows + TN - 1) / TN);
  if (tiles * a.ks > 0x7fffffffLL) return cudaErrorInvalidValue;
  a.units = (uint32_t)(tiles * a.ks);
  // whole tiles where they fill the CTAs evenly enough
  const long long turns = (tiles + l.sms - 1) / l.sms;
  if (tiles * 10 >= turns * l.sms * 9)
    a.size = (uint32_t)(turns * a.ks);
  else
    a.size = (uint32_t)((a.units + l.sms - 1) / l.sms);
  const int grid = (int)((a.units + a.size - 1) / a.size);
  a.fresh = l.fresh;
  a.counters = static_cast<unsigned *>(l.workspace);
  a.slots = reinterpret_cast<float *>(static_cast<uint8_t *>(l.workspace) + kKvCounterBytes);
  a.status = l.status;
  static std::atomic<bool> attr_set[kAttrMaxDevices];
  const cudaError_t e = ensure_dynamic_smem(mx4_linear_k<TN, BF16>, S::kSmem, attr_set);
  if (e != cudaSuccess) return e;
  return launch_kernel(mx4_linear_k<TN, BF16>, dim3((unsigned)grid), dim3(kLinearThreads), (size_t)S::kSmem, st, a);
}

template <bool BF16>
cudaError_t linear_rows(const Mx4Linear &l, cudaStream_t st) {
  if (l.x.rows <= 16) return linear_tiles<16, BF16>(l, st);
  if (l.x.rows <= 32) return linear_tiles<32, BF16>(l, st);
  if (l.x.rows <= 64) return linear_tiles<64, BF16>(l, st);
  if (l.x.rows <= 128) return linear_tiles<128, BF16>(l, st);
  return linear_tiles<192, BF16>(l, st);
}

// Pieces of a warp, and the grid: few values go to many warps.
dim3 quant_grid(long long width, long long rows, bool &four) {
  const long long blocks = (rows + kQuantRows - 1) / kQuantRows;
  four = width > 256 && blocks * ((width + 1023) / 1024) >= 148 * 2;
  const long long x = (width + (four ? 1023 : 255)) / (four ? 1024 : 256);
  return dim3((unsigned)x, (unsigned)std::min(blocks, std::max(1ll, 148 * 8 / x)));
}

template <bool BF16>
cudaError_t quantize(const void *x, long long rows, long long stride, const Mx4 &m, cudaStream_t st) {
  const long long padded = (rows + 127) / 128 * 128;  // (scale bytes of rows that are not there are 0)
  bool four;
  const dim3 grid = quant_grid(m.width, padded, four);
  const uint16_t *p = static_cast<const uint16_t *>(x);
  if (four) return launch_kernel(mx4_quantize_k<BF16, 4>, grid, dim3(kQuantThreads), 0, st, p, rows, padded, stride, (int)rows_vec(x, stride), m);
  return launch_kernel(mx4_quantize_k<BF16, 1>, grid, dim3(kQuantThreads), 0, st, p, rows, padded, stride, (int)rows_vec(x, stride), m);
}
template <bool BF16>
cudaError_t read(const Mx4 &m, long long rows, void *out, long long stride, cudaStream_t st) {
  bool four;
  const dim3 grid = quant_grid(m.width, rows, four);
  uint16_t *p = static_cast<uint16_t *>(out);
  if (four) return launch_kernel(mx4_read_k<BF16, 4>, grid, dim3(kQuantThreads), 0, st, m, rows, p, stride, (int)rows_vec(out, stride));
  return launch_kernel(mx4_read_k<BF16, 1>, grid, dim3(kQuantThreads), 0, st, m, rows, p, stride, (int)rows_vec(out, stride));
}

}  // namespace

cudaError_t launch_mx4_quantize(bool bf16, const void *x, long long rows, long long stride, const Mx4 &m,
                                cudaStream_t st) {
  return bf16 ? quantize<true>(x, rows, stride, m, st) : quantize<false>(x, rows, stride, m, st);
}

cudaError_t launch_mx4_read(bool bf16, const Mx4 &m, long long rows, void *out, long long stride, cudaStream_t st) {
  return bf16 ? read<true>(m, rows, out, stride, st) : read<false>(m, rows, out, stride, st);
}

// Counters (zero before the first call and after each), then two parts of tiles a CTA.
size_t mx4_workspace_bytes(int sms) { return kKvCounterBytes + sizeof(float) * 2 * (size_t)sms * kMm * kMaxTokens; }

cudaError_t launch_mx4_linear(const Mx4Linear &a, cudaStream_t st) {
  return a.bf16 ? linear_rows<true>(a, st) : linear_rows<false>(a, st);
}

}  // namespace ivb
