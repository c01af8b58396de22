// Attention over the paged 8-bit cache for few queries a sequence (decoding,
// checking drafted tokens).
//
// For a query at position p and the visible keys j (codes kc, vc; scales ks, vs):
//   s_j = scale * ks_j * (q . kc_j),  o = sum_j e^(s_j - m) vs_j vc_j / sum_j e^(s_j - m)
// in one pass with a running maximum m.  A decode step reads every visible
// code once and does a few operations for each, so the cache's bytes bound it.
//
// An item is a tile of 16 query rows (token, head of the group) of one
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
// conflict), and multiplies with m16n8k16 tensor instructions: codes become
// halves exactly (1024 + code + 128 by a byte permutation, minus 1152), the
// order of head elements and keys inside the products is chosen so that every
// lane reads whole 16-byte (64-wide heads: 8-byte) pieces of a row and the
// scores leave one product in the registers that the next one wants.
#include "kv_attend.cuh"

namespace ivb {

namespace {

constexpr int kStepWarps = 4, kStepThreads = 32 * kStepWarps;
constexpr int kStepRows = 16;
constexpr int kStepStages = 4;
constexpr int kStepCtasPerSm = 3;
constexpr int kStepMinBlocks = kStepWarps;  // of a CTA's share: a block for each warp

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

// Two codes (+ 128, in bytes LO, LO + 1 of w) as halves.
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

template <int DIM>
struct StepSlot {  // partial sums of a cut item: accumulators lane by lane, then per row maximum and sum
  float acc[DIM / 2 * 32];
  float m[kStepRows], l[kStepRows];
  float vref;
  float pad[31];
};

template <int DIM>
struct StepShared {
  alignas(128) uint8_t ring[kStepWarps][kStepStages][2][kKvBlock * DIM];
  float2 scales[kStepWarps][kStepStages];
  float m[kStepWarps][kStepRows], l[kStepWarps][kStepRows], vref[kStepWarps];
  long long scan[kStepWarps];
  long long total, base;
  int seq;
  int last;
};

template <bool BF16, int DIM>
__global__ void __launch_bounds__(kStepThreads, kStepCtasPerSm)
    kv_step_k(const __grid_constant__ KvAttend a, StepSlot<DIM> *slots, unsigned *counters) {
  extern __shared__ uint8_t smem_raw[];
  StepShared<DIM> &sh = *reinterpret_cast<StepShared<DIM> *>(smem_raw);
  constexpr int kAcc = DIM / 2;         // accumulators a lane (16 x DIM over 32 lanes)
  constexpr int kTiles = DIM / 8;       // 8-wide column tiles of the output
  constexpr int kSteps = DIM / 16;      // 16-deep steps of the score product
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  pdl_wait_and_release();

  // ---- all units, and the sequence where this CTA's share begins
  const int per = (a.seqs.batch + kStepThreads - 1) / kStepThreads;
  long long mine = 0;
  const int b_lo = min(a.seqs.batch, (int)threadIdx.x * per), b_hi = min(a.seqs.batch, b_lo + per);
  for (int b = b_lo; b < b_hi; ++b) {
    const KvSpan s = kv_span(a, b);
    mine += (long long)s.blocks * ((s.n * a.group + kStepRows - 1) / kStepRows) * a.cache.heads;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh.scan[warp] = incl;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kStepWarps; ++w) {
    if (w < warp) before += sh.scan[w];
    total += sh.scan[w];
  }
  if (total == 0) return;
  const long long want = (total + kStepMinBlocks - 1) / kStepMinBlocks;
  const int ctas = (int)(want < (long long)gridDim.x ? want : (long long)gridDim.x);
  if ((int)blockIdx.x >= ctas) return;
  long long u = share_begin(total, ctas, blockIdx.x);
  const long long u_end = share_begin(total, ctas, blockIdx.x + 1);
  const long long excl = before + incl - mine;
  if (u >= excl && u < excl + mine) {
    long long at = excl;
    int b = b_lo;
    for (;; ++b) {
      const KvSpan s = kv_span(a, b);
      const long long w = (long long)s.blocks * ((s.n * a.group + kStepRows - 1) / kStepRows) * a.cache.heads;
      if (u < at + w) break;
      at += w;
    }
    sh.seq = b;
    sh.base = at;
  }
  __syncthreads();
  int b = sh.seq;
  long long base = sh.base;  // first unit of sequence b

  const float qscale = a.scale * kLog2e;
  while (u < u_end) {
    // ---- the segment: blocks k0 .. k1 - 1 of item (b, head, row tile)
    const KvSpan s = kv_span(a, b);
    const int row_tiles = (s.n * a.group + kStepRows - 1) / kStepRows;
    const long long units = (long long)s.blocks * row_tiles * a.cache.heads;
    if (u >= base + units) {
      base += units;
      ++b;
      continue;
    }
    const long long item = (u - base) / s.blocks;
    const int head = (int)(item / row_tiles), rt = (int)(item - (long long)head * row_tiles);
    const long long item_begin = base + item * s.blocks, item_end = item_begin + s.blocks;
    const int k0 = (int)(u - item_begin), k1 = (int)(min(u_end, item_end) - item_begin);

    // ---- this lane's rows g and g + 8: positions and queries
    int pos[2];
    float rs[2];
    uint32_t q[kSteps][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = rt * kStepRows + g + 8 * h, i = r / a.group;
      pos[h] = i < s.n ? s.len - s.n + i : -1;
      const uint16_t *row = static_cast<const uint16_t *>(a.q.p) + (long long)(s.first + i) * a.q.ts +
                            (long long)(head * a.group + r - i * a.group) * a.q.hs;
      uint32_t w[2 * kSteps];
#pragma unroll
      for (int c = 0; c < DIM / 64; ++c) {
        const uint4 x = pos[h] >= 0 ? load8(row + 64 * c + 16 * t4, a.q.vec) : make_uint4(0, 0, 0, 0);
        const uint4 y = pos[h] >= 0 ? load8(row + 64 * c + 16 * t4 + 8, a.q.vec) : make_uint4(0, 0, 0, 0);
        w[8 * c] = x.x, w[8 * c + 1] = x.y, w[8 * c + 2] = x.z, w[8 * c + 3] = x.w;
        w[8 * c + 4] = y.x, w[8 * c + 5] = y.y, w[8 * c + 6] = y.z, w[8 * c + 7] = y.w;
      }
      rs[h] = qscale;
      if (BF16) {
        // bf16 queries become halves: the row is scaled by a power of two so
        // that its largest element lies in 2^0 .. 2^1 (its eight bits stay)
        float most = 0.f;
#pragma unroll
        for (int i2 = 0; i2 < 2 * kSteps; ++i2) {
          const float2 f = unpack2<true>(w[i2]);
          most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = min(max((int)(__float_as_uint(most) >> 23), 1), 253);  // biased
        const float down = __uint_as_float((uint32_t)(254 - e) << 23);
        rs[h] *= __uint_as_float((uint32_t)e << 23);
#pragma unroll
        for (int i2 = 0; i2 < 2 * kSteps; ++i2) {
          const float2 f = unpack2<true>(w[i2]);
          w[i2] = pack2<false>(f.x * down, f.y * down);
        }
      }
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        q[k][h] = w[2 * k];
        q[k][2 + h] = w[2 * k + 1];
      }
    }
    const int p_lo = s.len - s.n + rt * kStepRows / a.group;                              // first row's position
    const int p_hi = s.len - s.n + min(s.n - 1, (rt * kStepRows + kStepRows - 1) / a.group);  // last row's

    float acc[kTiles][4];
#pragma unroll
    for (int j = 0; j < kTiles; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float vref = 0.f, vinv = 0.f;  // acc is in units of vref, the largest value scale so far

    // ---- blocks k0 + warp, + kStepWarps, ...; lane i knows the i-th of the next 32
    const int count = k1 - k0 > warp ? (k1 - k0 - warp + kStepWarps - 1) / kStepWarps : 0;
    const uint32_t ring = smem_u32(&sh.ring[warp][0][0][0]);
    long long where = -1;  // this lane's block's codes, -1: none
    float ksc = 0.f, vsc = 0.f;
    int looked = 0;
    auto look_up = [&](int it) {  // for iterations it .. it + 31
      where = -1;
      ksc = vsc = 0.f;
      if (it + lane < count) {
        const int key = s.block(k0 + warp + (it + lane) * kStepWarps) * kKvBlock;
        if (key < s.len) {
          const int page = kv_page_of(a.cache, a.seqs, b, key, a.status);
          if (page >= 0) {
            const int slot = key % a.cache.page;
            where = kv_code_at(a.cache, page, head, slot);
            const long long sa = kv_scale_at(a.cache, page, head, slot);
            ksc = a.cache.ks[sa];
            vsc = a.cache.vs[sa];
          }
        }
      }
    };
    auto copy = [&](int it, long long from) {
      if (from >= 0) {
        const uint32_t dst = ring + (uint32_t)(it % kStepStages) * (2u * kKvBlock * DIM);
#pragma unroll
        for (int i = 0; i < kKvBlock * DIM / 512; ++i) {
          const uint32_t o = (uint32_t)(i * 32 + lane) * 16u;
          cp_async16(dst + tile_swizzle<DIM>(o), a.cache.k + from + o);
        }
#pragma unroll
        for (int i = 0; i < kKvBlock * DIM / 512; ++i) {
          const uint32_t o = (uint32_t)(i * 32 + lane) * 16u;
          cp_async16(dst + kKvBlock * DIM + tile_swizzle<DIM>(o), a.cache.v + from + o);
        }
      }
      cp_async_commit();
    };
    // the look-up runs kStepStages - 1 blocks ahead of the products: a block's
    // scales wait beside its codes (a value scale below 0: nothing to see)
    auto fetch = [&](int it) {
      long long from = -1;
      if (it < count) {
        if (it == looked) {
          look_up(it);
          looked += 32;
        }
        from = __shfl_sync(0xffffffffu, where, it & 31);
        if (lane == (it & 31)) sh.scales[warp][it % kStepStages] = make_float2(ksc, where >= 0 ? vsc : -1.f);
      }
      copy(it, from);
    };
#pragma unroll
    for (int i = 0; i < kStepStages - 1; ++i) fetch(i);
    for (int it = 0; it < count; ++it) {
      cp_async_wait<kStepStages - 2>();
      __syncwarp();
      const int st = it % kStepStages;
      const float2 scales = sh.scales[warp][st];
      const float bk = scales.x, bv = scales.y;
      if (bv >= 0.f) {
        const uint8_t *kt = sh.ring[warp][st][0], *vt = sh.ring[warp][st][1];
        // scores of keys 8j + 2 t4, + 1 (j = 0, 1) for rows g, g + 8
        float sc[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
#pragma unroll
          for (int c = 0; c < DIM / 64; ++c) {
            const uint4 w4 =
                *reinterpret_cast<const uint4 *>(kt + tile_swizzle<DIM>((uint32_t)((8 * j + g) * DIM + 64 * c + 16 * t4)));
            const uint32_t w[4] = {w4.x ^ 0x80808080u, w4.y ^ 0x80808080u, w4.z ^ 0x80808080u, w4.w ^ 0x80808080u};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int k = 4 * c + i;
              mma16816(sc[j], q[k][0], q[k][1], q[k][2], q[k][3], codes2<0x4140>(w[i]), codes2<0x4342>(w[i]));
            }
          }
        }
        const int key0 = s.block(k0 + warp + it * kStepWarps) * kKvBlock;
        const bool masked = key0 + kKvBlock - 1 > p_lo ||
                            (a.window > 0 && p_hi - key0 >= a.window && key0 + kKvBlock > a.sinks);
        float mx[2] = {m[0], m[1]};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = e >> 1;
            float x = sc[j][e] * (rs[h] * bk);
            if (masked && !kv_sees(a, pos[h], key0 + 8 * j + 2 * t4 + (e & 1))) x = -INFINITY;
            sc[j][e] = x;
            mx[h] = fmaxf(mx[h], x);
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        }
        const float vnew = fmaxf(vref, bv);
        if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1]) || vnew > vref) {
          const float vr = vref > 0.f ? __fdividef(vref, vnew) : 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float f = mx[h] > m[h] ? fast_exp2(m[h] - mx[h]) : 1.f;
            l[h] *= f;
            m[h] = mx[h];
            const float fo = f * vr;
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              acc[j][2 * h] *= fo;
              acc[j][2 * h + 1] *= fo;
            }
          }
          vref = vnew;
          vinv = vref > 0.f ? 1.f / vref : 0.f;
        }
        const float bf = bv * vinv;
        uint32_t p[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float base_m = m[h] == -INFINITY ? 0.f : m[h] - kWeightBits;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x = fast_exp2(sc[j][2 * h] - base_m), y = fast_exp2(sc[j][2 * h + 1] - base_m);
            l[h] += x + y;
            p[2 * j + h] = pack2<false>(x * bf, y * bf);  // rounded to 11 bits; summed in 32
          }
        }
        // values: keys 2 t4, + 1, + 8, + 9; column tile j is byte j of the lane's piece of a row
        uint32_t vw[4][DIM / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t o = (uint32_t)((8 * (i >> 1) + 2 * t4 + (i & 1)) * DIM + g * (DIM / 8));
          if (DIM == 128) {
            const uint4 x = *reinterpret_cast<const uint4 *>(vt + tile_swizzle<DIM>(o));
            vw[i][0] = x.x, vw[i][1] = x.y, vw[i][DIM / 32 - 2] = x.z, vw[i][DIM / 32 - 1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(vt + tile_swizzle<DIM>(o));
            vw[i][0] = x.x, vw[i][1] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < DIM / 32; ++w) {
          const uint32_t x0 = vw[0][w] ^ 0x80808080u, x1 = vw[1][w] ^ 0x80808080u, x2 = vw[2][w] ^ 0x80808080u,
                         x3 = vw[3][w] ^ 0x80808080u;
          const uint32_t a0 = __byte_perm(x0, x1, 0x5140), a1 = __byte_perm(x0, x1, 0x7362);
          const uint32_t c0 = __byte_perm(x2, x3, 0x5140), c1 = __byte_perm(x2, x3, 0x7362);
          mma16816(acc[4 * w], p[0], p[1], p[2], p[3], codes2<0x4140>(a0), codes2<0x4140>(c0));
          mma16816(acc[4 * w + 1], p[0], p[1], p[2], p[3], codes2<0x4342>(a0), codes2<0x4342>(c0));
          mma16816(acc[4 * w + 2], p[0], p[1], p[2], p[3], codes2<0x4140>(a1), codes2<0x4140>(c1));
          mma16816(acc[4 * w + 3], p[0], p[1], p[2], p[3], codes2<0x4342>(a1), codes2<0x4342>(c1));
        }
      }
      __syncwarp();  // the slot that the next copy overwrites has been read
      fetch(it + kStepStages - 1);
    }
    cp_async_wait<0>();

    // ---- join the warps: row maxima, then sums in a common scale
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t4 == 0) {
        sh.m[warp][g + 8 * h] = m[h];
        sh.l[warp][g + 8 * h] = l[h];
      }
    }
    if (lane == 0) sh.vref[warp] = vref;
    __syncthreads();
    float all_m[2], all_v = 0.f, f[2];
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) all_v = fmaxf(all_v, sh.vref[w]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      all_m[h] = -INFINITY;
#pragma unroll
      for (int w = 0; w < kStepWarps; ++w) all_m[h] = fmaxf(all_m[h], sh.m[w][g + 8 * h]);
      f[h] = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - all_m[h]) * (all_v > 0.f ? __fdividef(vref, all_v) : 0.f);
    }
    // accumulators lane by lane: [row half][column half][tile], so that eight
    // neighbours of a lane are eight neighbouring outputs
    float *part = reinterpret_cast<float *>(&sh.ring[warp][0][0][0]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < kTiles; ++j) part[((2 * h + c) * kTiles + j) * 32 + lane] = acc[j][2 * h + c] * f[h];
    __syncthreads();
    const bool whole = k0 == 0 && k1 == s.blocks;
    const int first_cta = share_of(total, ctas, item_begin), last_cta = share_of(total, ctas, item_end - 1);
    const int slot = 2 * (int)blockIdx.x + (k0 == 0 ? 1 : 0);
    if (!whole) {
      for (int e = threadIdx.x; e < kAcc * 32; e += kStepThreads) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kStepWarps; ++w) x += reinterpret_cast<const float *>(&sh.ring[w][0][0][0])[e];
        __stcg(&slots[slot].acc[e], x);
      }
      if (threadIdx.x < kStepRows) {
        const int r = threadIdx.x;
        float am = -INFINITY, x = 0.f;
        for (int w = 0; w < kStepWarps; ++w) am = fmaxf(am, sh.m[w][r]);
        for (int w = 0; w < kStepWarps; ++w)
          if (sh.m[w][r] != -INFINITY || sh.l[w][r] != 0.f) x += sh.l[w][r] * fast_exp2(sh.m[w][r] - am);
        __stcg(&slots[slot].m[r], am);
        __stcg(&slots[slot].l[r], x);
        if (r == 0) __stcg(&slots[slot].vref, all_v);
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const unsigned parts = (unsigned)(last_cta - first_cta + 1);
        const unsigned old = atomicAdd(&counters[first_cta], 1u);
        sh.last = old == parts - 1;
        if (sh.last) atomicExch(&counters[first_cta], 0u);
        __threadfence();
      }
      __syncthreads();
    }
    if (whole || sh.last) {
      // eight neighbouring outputs a thread
      for (int e = threadIdx.x; e < kAcc / 8 * 32; e += kStepThreads) {
        const int ln = e & 31, i0 = (e >> 5) * 8;  // accumulators i0 .. i0 + 7 of lane ln
        const int h = i0 / (2 * kTiles), c = i0 / kTiles % 2, j0 = i0 % kTiles;
        const int r = (ln >> 2) + 8 * h;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f, top = -INFINITY, vr = 0.f;
        if (whole) {
          for (int w = 0; w < kStepWarps; ++w) top = fmaxf(top, sh.m[w][r]);
          vr = all_v;
          for (int w = 0; w < kStepWarps; ++w) {
            if (sh.m[w][r] != -INFINITY || sh.l[w][r] != 0.f) sum += sh.l[w][r] * fast_exp2(sh.m[w][r] - top);
            const float *src = reinterpret_cast<const float *>(&sh.ring[w][0][0][0]) + i0 * 32 + ln;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] += src[32 * k];
          }
        } else {
          for (int z = first_cta; z <= last_cta; ++z) {
            const StepSlot<DIM> &sl = slots[2 * z + (z == first_cta ? 1 : 0)];
            top = fmaxf(top, __ldcg(&sl.m[r]));
            vr = fmaxf(vr, __ldcg(&sl.vref));
          }
          for (int z = first_cta; z <= last_cta; ++z) {
            const StepSlot<DIM> &sl = slots[2 * z + (z == first_cta ? 1 : 0)];
            const float zm = __ldcg(&sl.m[r]), zl = __ldcg(&sl.l[r]);
            if (zm == -INFINITY && zl == 0.f) continue;  // this part of the keys was hidden from the row
            const float w = fast_exp2(zm - top), wv = vr > 0.f ? w * __fdividef(__ldcg(&sl.vref), vr) : 0.f;
            sum += zl * w;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] += __ldcg(&sl.acc[(i0 + k) * 32 + ln]) * wv;
          }
        }
        const int row = rt * kStepRows + r, i = row / a.group;
        if (i < s.n) {
          const float y = sum != 0.f ? vr / sum : 0.f;  // (a NaN sum stays NaN)
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] *= y;
          uint16_t *o = static_cast<uint16_t *>(a.out.p) + (long long)(s.first + i) * a.out.ts +
                        (long long)(head * a.group + row - i * a.group) * a.out.hs;
          store8(o + (2 * (ln & 3) + c) * kTiles + j0, pack8<BF16>(x), a.out.vec);
        }
      }
    }
    __syncthreads();  // the ring and the joins are free again
    u += k1 - k0;
  }
}

template <bool BF16, int DIM>
cudaError_t launch_step(const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  static std::atomic<bool> attr_set[kAttrMaxDevices];
  const int bytes = (int)sizeof(StepShared<DIM>);
  const cudaError_t e = ensure_dynamic_smem(kv_step_k<BF16, DIM>, bytes, attr_set);
  if (e != cudaSuccess) return e;
  const int grid = sms * kStepCtasPerSm;
  return launch_kernel(kv_step_k<BF16, DIM>, dim3(grid), dim3(kStepThreads), (size_t)bytes, st, a,
                       reinterpret_cast<StepSlot<DIM> *>(static_cast<uint8_t *>(workspace) + kKvCounterBytes),
                       static_cast<unsigned *>(workspace));
}

}  // namespace

// Counters (zero before the first call and after each), then two slots a CTA.
size_t kv_workspace_bytes(int sms) { return kKvCounterBytes + sizeof(StepSlot<128>) * 2 * (size_t)sms * kStepCtasPerSm; }

cudaError_t launch_kv_attend(bool bf16, const KvAttend &a, void *workspace, int sms, cudaStream_t st) {
  if (a.cache.dim == 64)
    return bf16 ? launch_step<true, 64>(a, workspace, sms, st) : launch_step<false, 64>(a, workspace, sms, st);
  return bf16 ? launch_step<true, 128>(a, workspace, sms, st) : launch_step<false, 128>(a, workspace, sms, st);
}

}  // namespace ivb
