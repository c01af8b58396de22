// The next token from a row of logits: temperature, top k, top p, min p, and a
// random number.
//
// Token i weighs w_i = e^((x_i - max) / T).  In the order of falling logits, equal
// ones by their numbers, each filter keeps a beginning, so that together they are
// a cut: the last (logit, number) that is kept.  The token is then the first, by
// number, where the running sum of kept weights passes u times their sum.  Which
// one that is goes by sums next to a border, so weights and sums are in 64 bits,
// added in an order that is fixed for a size, a number of rows, a device and a row's
// address (modulo 16 bytes): a token next to a border may be another one elsewhere.
//
// Two kernels.  sample_count_k, for logits in 16 bits: a CTA a row counts how often
// each of the 65536 values occurs, in shared memory.  A value's weight is then worked
// out once for all its tokens, every cut follows from the counts, and only tokens
// that are kept are weighed one by one, where the running sums need them.
// sample_k, for the others and for few long rows: a cluster of CTAs a row, each with
// a slice of it in shared memory.  It counts logits in bins of equal width, up to the
// bin where the cut must be; if these are at most kList, one CTA puts them in order
// and does the rest; if not, the bin is binned again, equal logits by their numbers.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "sample.cuh"

namespace ivb {

namespace {

namespace cg = cooperative_groups;

constexpr int kClusterThreads = 512;
constexpr int kMostWarps = 32;
constexpr int kBins = 2048, kList = 1024;
constexpr int kMaxRanks = 8;
constexpr int kWindow = 16;  // bins around a guess
constexpr double kFar = 41.588830833596715;  // 60 ln 2: what is further below the largest has no weight

// 2^(j / 256), j below 256.
constexpr int kPowers = 256;
__device__ __forceinline__ void fill_powers(double *powers) {
  for (int j = threadIdx.x; j < kPowers; j += blockDim.x) powers[j] = exp2(j / (double)kPowers);
}
// e^((v - top) / T) = 2^(n / 256) 2^(r / 256), |r| at most a half: the first from the
// table, of the second the first terms of its series (the rest is below 2^-54 of it).
struct Weights {
  float top;
  // Whether a weight is 0 is asked in 32 bits: (v times - top_times) by32, where neither
  // the difference of the largest numbers nor a division by the smallest runs over.
  float times, top_times, by32;
  double by;  // 256 log2(e) / T
  const double *powers;
  __device__ __forceinline__ void set(float t, float temperature) {
    top = t;
    by = kPowers * 1.4426950408889634 / (double)temperature;
    const bool small = by > 0x1p126 && fabsf(top) < 0x1p27f;  // (a larger one is by more than 60 bits above the next)
    times = small ? 0x1p100f : 0.5f;
    top_times = top * times;
    by32 = (float)(by / (double)times);
  }
  __device__ __forceinline__ double operator()(float v) const {
    if (!(fmaf(v, times, -top_times) * by32 > -60.f * kPowers)) return v == top ? 1.0 : 0.0;  // (the largest may be +inf)
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: what is added to it is rounded to a whole number
    constexpr double c = 0.6931471805599453 / kPowers;
    const double d = (double)v - (double)top, s = fma(d, by, kRound), r = fma(d, by, kRound - s);
    const int n = __double2loint(s);
    const double w = fma(fma(fma(fma(c * c * c * c / 24.0, r, c * c * c / 6.0), r, c * c / 2.0), r, c), r, 1.0) * powers[n & (kPowers - 1)];
    return __hiloint2double(__double2hiint(w) + (n >> 8) * (1 << 20), __double2loint(w));
  }
};

struct Cut {  // kept: x > this one's, or x equal and number at most this one's
  float x;
  int i;
};

// Weights summed up in kWindow bins as whole numbers of 2^-63, so that their order does not
// matter: in six pieces of 11 bits (a row has less than 2^19 tokens), since shared memory
// adds 32 bits at once, and 64 by trying until nobody interferes.  A sum is off by 2^-45 at
// most.  top_p, in 32 bits, leaves 2^-24 of the weight or more behind a cut, so that where
// one lies tokens weigh 2^-43 and more.  (With numbers of 2^-44 a cut at the end of 60000
// equal tokens of e^-20 came out past it.)
struct Window {
  static constexpr int kPieces = 6, kBits = 11;
  unsigned piece[kPieces][kWindow];
  __device__ __forceinline__ void clear() {
    if (threadIdx.x < kPieces * kWindow) (&piece[0][0])[threadIdx.x] = 0;
  }
  __device__ __forceinline__ void add(unsigned k, double w) {
    const unsigned long long f = __double2ull_rn(w * 0x1p63);
#pragma unroll
    for (int q = 0; q < kPieces; ++q) atomicAdd(&piece[q][k], (unsigned)(f >> (kBits * q)) & ((1u << kBits) - 1u));
  }
  __device__ __forceinline__ double sum(unsigned k) const {
    double f = 0;
#pragma unroll
    for (int q = 0; q < kPieces; ++q) f = f * 0x1p-11 + (double)piece[q][k];
    return f * 0x1p-8;  // (the last piece counts 2^55)
  }
};
static_assert(kSampleMaxVocab < 1 << 19, "pieces of a sum");

struct SampleShared {
  double powers[kPowers];
  alignas(16) unsigned hist[kBins];
  unsigned long long key[kList];  // (order of x, number), rising
  double mass[kList], wt[kList];  // running sums, weights
  double part[2][kMaxRanks][2];   // what CTAs tell one another, two exchanges in turn
  double red[2][kMostWarps];
  unsigned cnt[kMostWarps];
  unsigned listed, staged, place;
  int found, kept, reached;
  unsigned before, in_bin;
  Cut cut;
  double seg[kMostWarps];
  Window window;
};

// Order of floats as unsigned numbers, falling (no NaN, no -0).
__device__ __forceinline__ uint32_t falling(float x) {
  const uint32_t b = __float_as_uint(x);
  return (int)b < 0 ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float from_falling(uint32_t k) { return __uint_as_float((int)k < 0 ? k : ~k & 0x7fffffffu); }

template <class T>
__device__ __forceinline__ float logit(T v) {
  float x = (float)v;
  return x != x ? -INFINITY : x + 0.f;  // (-0 is 0)
}
// What a row asks for.
struct Want {
  int k;               // 0: all
  float t, p, min_p, u;
  __device__ __forceinline__ Want(const Sample &a, long long r) {
    t = a.temperature ? a.temperature[r] : 1.f;
    k = a.top_k ? a.top_k[r] : 0;
    k = !(t > 0.f) ? 1 : k > 0 && k < a.vocab ? k : 0;
    p = a.top_p && t > 0.f ? fmaxf(a.top_p[r], 0.f) : 1.f;
    if (!(a.top_p && a.top_p[r] < 1.f)) p = 1.f;
    min_p = a.min_p ? a.min_p[r] : 0.f;
    if (min_p > 1.f && a.vocab > 1) k = 1;  // (no weight is as large: the first alone)
    u = a.u[r];
    u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  }
  // Logits below this weigh less than min_p, by more than any rounding.
  __device__ __forceinline__ float floor(float top) const {
    if (!(min_p > 0.f) || !(t > 0.f)) return -INFINITY;
    if (top == INFINITY) return top;  // (the others weigh nothing)
    const double x = (double)top + (fmin(log((double)min_p), 0.0) - 1e-6) * (double)t;
    return (float)(x - 2e-7 * fabs(x));
  }
  __device__ __forceinline__ bool enough(double w, bool top) const { return !(min_p > 0.f) || top || w >= (double)min_p; }
};

template <class T, int THREADS>
struct Row {
  static constexpr int kThreads = THREADS, kWarps = THREADS / 32, kPer = kList / THREADS;
  SampleShared &sh;
  const T *x;      // this CTA's slice
  bool vec;        // on 16 bytes
  int n, first;    // its length, the number of its first token
  int ranks, rank;
  float top;       // the largest logit
  Weights weight;
  Cut cut;
  int turn = 0;    // of `part`

  __device__ Row(SampleShared &s) : sh(s) { weight.powers = s.powers; }

  __device__ __forceinline__ void sync() {
    if (ranks > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  template <class V>
  __device__ __forceinline__ V *at(V *p, int r) {
    return ranks > 1 ? cg::this_cluster().map_shared_rank(p, r) : p;
  }

  __device__ __forceinline__ bool keeps(float v, int i) const { return v > cut.x || (v == cut.x && i <= cut.i); }

  // Sum (or maximum) of a and b over the cluster, to all its threads.
  template <bool MAX>
  __device__ void reduce(double &a, double &b) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const double c = __shfl_xor_sync(0xffffffffu, a, o), d = __shfl_xor_sync(0xffffffffu, b, o);
      a = MAX ? fmax(a, c) : a + c;
      b = MAX ? fmax(b, d) : b + d;
    }
    if (lane == 0) sh.red[0][warp] = a, sh.red[1][warp] = b;
    __syncthreads();
    double s = sh.red[0][0], t = sh.red[1][0];
    for (int w = 1; w < kWarps; ++w) {
      s = MAX ? fmax(s, sh.red[0][w]) : s + sh.red[0][w];
      t = MAX ? fmax(t, sh.red[1][w]) : t + sh.red[1][w];
    }
    turn ^= 1;
    if ((int)threadIdx.x < ranks) {
      double *p = at(&sh.part[turn][rank][0], (int)threadIdx.x);
      p[0] = s, p[1] = t;
    }
    sync();
    a = sh.part[turn][0][0], b = sh.part[turn][0][1];
    for (int r = 1; r < ranks; ++r) {
      a = MAX ? fmax(a, sh.part[turn][r][0]) : a + sh.part[turn][r][0];
      b = MAX ? fmax(b, sh.part[turn][r][1]) : b + sh.part[turn][r][1];
    }
  }

  // Four logits from j on (a multiple of 4; -inf behind the slice's end).
  __device__ __forceinline__ void load4(int j, float (&v)[4]) const {
    T t[4];
    if (vec && j + 3 < n) {
      if (sizeof(T) == 4)
        *reinterpret_cast<uint4 *>(t) = *reinterpret_cast<const uint4 *>(x + j);
      else
        *reinterpret_cast<uint2 *>(t) = *reinterpret_cast<const uint2 *>(x + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = logit(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = j + i < n ? logit(x[j + i]) : -INFINITY;
    }
  }
  // f(logit, number) for each of the slice (and for some -inf behind it).
  template <class F>
  __device__ __forceinline__ void each(F &&f) {
#pragma unroll 2
    for (int j = 4 * threadIdx.x; j < n; j += 4 * kThreads) {
      float v[4];
      load4(j, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) f(v[i], first + j + i);
    }
  }

  // Counts into sh.hist, over the cluster, what bin(logit, number) says (below 0: nothing).
  template <class F>
  __device__ void count(F &&bin) {
    clear();
    each([&](float v, int i) {
      const int b = bin(v, i);
      if (b >= 0) atomicAdd(&sh.hist[b], 1u);
    });
    merge();
  }
  __device__ void clear() {
    for (int b = threadIdx.x; b < kBins; b += kThreads) sh.hist[b] = 0;
    __syncthreads();
  }
  // The CTAs' counts become the cluster's.
  __device__ void merge() {
    if (ranks == 1) {
      __syncthreads();
      return;
    }
    sync();
    // A CTA adds up its part of the bins, and gives it to all (all parts in every CTA: 64 rows
    // of 131072 78 us, 75 so).
    static_assert(kBins % (4 * kMaxRanks) == 0 && kBins / 8 <= kClusterThreads, "bins");
    const int part = kBins / 4 / ranks;  // (fours)
    uint4 sum = make_uint4(0, 0, 0, 0);
    const int four = rank * part + (int)threadIdx.x;
    const bool mine = (int)threadIdx.x < part;
    if (mine) {
      uint4 u[kMaxRanks];
#pragma unroll
      for (int r = 0; r < kMaxRanks; ++r) u[r] = r < ranks ? reinterpret_cast<const uint4 *>(at(sh.hist, r))[four] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < kMaxRanks; ++r) sum.x += u[r].x, sum.y += u[r].y, sum.z += u[r].z, sum.w += u[r].w;
    }
    sync();
    if (mine)
      for (int r = 0; r < ranks; ++r) reinterpret_cast<uint4 *>(at(sh.hist, r))[four] = sum;
    sync();
  }

  // The first bin where value(b) summed up to it reaches `target` (the last one, if none),
  // into sh.found; counts before it into sh.before.  With `more`, the target is higher by
  // what all values are beyond that.
  template <class F>
  __device__ void find(double target, F &&value, double more = -1) {
    constexpr int kEach = kBins / kThreads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double v[kEach], mine = 0;
    unsigned c = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      v[k] = value((int)threadIdx.x * kEach + k);
      mine += v[k];
      c += sh.hist[threadIdx.x * kEach + k];
    }
    double incl = mine;
    unsigned ci = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, incl, o);
      const unsigned u = __shfl_up_sync(0xffffffffu, ci, o);
      if (lane >= o) incl += t, ci += u;
    }
    if (lane == 31) sh.red[0][warp] = incl, sh.cnt[warp] = ci;
    if (threadIdx.x == 0) sh.found = kBins - 1;
    __syncthreads();
    double before = 0, all = 0;
    unsigned cb = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.red[0][w], cb += sh.cnt[w];
      all += sh.red[0][w];
    }
    if (more >= 0) target += all - more;
    before += incl - mine;
    cb += ci - c;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      before += v[k];
      if (before >= target) {
        atomicMin(&sh.found, (int)threadIdx.x * kEach + k);
        break;
      }
    }
    __syncthreads();
    const int b = sh.found;
    if (b / kEach == (int)threadIdx.x) {
      for (int k = 0; k < b % kEach; ++k) cb += sh.hist[threadIdx.x * kEach + k];
      sh.before = cb;
      sh.in_bin = sh.hist[b];
    }
    __syncthreads();
  }

  // The sum of f over the first n bins.
  template <class F>
  __device__ double guessed(int n, F &&f) {
    double m = 0;
    for (int k = threadIdx.x; k < n; k += kThreads) m += f(k);
#pragma unroll
    for (int o = 16; o; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.red[0][threadIdx.x >> 5] = m;
    __syncthreads();
    m = sh.red[0][0];
    for (int w = 1; w < kWarps; ++w) m += sh.red[0][w];
    __syncthreads();
    return m;
  }

  // Collects those of which in(logit, number) holds, in CTA 0's sh.key and sh.listed (more
  // than kList: not all).  A CTA collects its own first (all counting in CTA 0: up to 6000
  // clocks more for 1000 of 131072).
  template <class F>
  __device__ void collect(F &&in) {
    if (threadIdx.x == 0) sh.listed = 0, sh.staged = 0;
    sync();
    unsigned long long *const stage = ranks > 1 ? reinterpret_cast<unsigned long long *>(sh.mass) : sh.key;
    unsigned *const counter = ranks > 1 ? &sh.staged : &sh.listed;
    each([&](float v, int i) {
      if (!in(v, i)) return;
      const unsigned p = atomicAdd(counter, 1u);
      if (p < kList) stage[p] = ((unsigned long long)falling(v) << 32) | (unsigned)i;
    });
    __syncthreads();
    if (ranks == 1) return;
    if (threadIdx.x == 0 && sh.staged) sh.place = atomicAdd(at(&sh.listed, 0), sh.staged);
    __syncthreads();
    unsigned long long *const key = at(sh.key, 0);
    for (unsigned e = threadIdx.x; e < min(sh.staged, (unsigned)kList) && sh.place + e < kList; e += kThreads) key[sh.place + e] = stage[e];
    sync();
  }
  // Those, at most kList, in order; how many there are is returned in CTA 0.
  template <class F>
  __device__ unsigned gather(F &&in) {
    collect(in);
    const unsigned n = min(sh.listed, (unsigned)kList);
    if (rank == 0) sort(n);
    return n;
  }

  // The n keys in rising order: two neighbours a thread, exchanged in registers but for steps
  // of 64 and more.  (All steps in shared memory: some 6000 clocks more for 1024 keys.)
  __device__ void sort(unsigned n) {
    using Key = unsigned long long;
    unsigned size = 2;
    while (size < n) size <<= 1;
    const unsigned e = 2 * threadIdx.x;
    const bool works = 2 * (threadIdx.x & ~31u) < size;
    Key a = works && e < n ? sh.key[e] : ~0ull, b = works && e + 1 < n ? sh.key[e + 1] : ~0ull;
    auto keep = [](Key &x, Key y, bool less) { x = (y < x) == less ? y : x; };
    for (unsigned k = 2; k <= size; k <<= 1) {
      const bool up = (e & k) == 0;
      unsigned j = k >> 1;
      for (; j >= 64; j >>= 1) {
        if (works) sh.key[e] = a, sh.key[e + 1] = b;
        __syncthreads();
        if (works) {
          const bool less = ((e & j) == 0) == up;
          keep(a, sh.key[e ^ j], less);
          keep(b, sh.key[(e + 1) ^ j], less);
        }
        __syncthreads();
      }
      if (!works) continue;
      for (; j >= 2; j >>= 1) {
        const bool less = ((e & j) == 0) == up;
        keep(a, __shfl_xor_sync(0xffffffffu, a, j >> 1), less);
        keep(b, __shfl_xor_sync(0xffffffffu, b, j >> 1), less);
      }
      if ((a > b) == up) {
        const Key t = a;
        a = b, b = t;
      }
    }
    if (works) sh.key[e] = a, sh.key[e + 1] = b;
    __syncthreads();
  }

  // Running sums of kPer doubles a thread over the block, and their total.
  __device__ __forceinline__ double scan(double (&x)[kPer]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 1; i < kPer; ++i) x[i] += x[i - 1];
    const double mine = x[kPer - 1];
    double s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    __syncthreads();
    if (lane == 31) sh.red[0][warp] = s;
    __syncthreads();
    double before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) before = all;
      all += sh.red[0][w];
    }
    before += s - mine;
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] += before;
    return all;
  }

  // Of the n logits in sh.key, in order: what is kept, and the token; CTA 0.  mass: of
  // all tokens (top_p of them is meant where there is no top_k).  False: top_p is not reached.
  __device__ bool finish(unsigned n, const Want &want, double mass, const Sample &a, long long r) {
    const int e0 = kPer * threadIdx.x;
    double w[kPer], c[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      w[i] = e0 + i < (int)n ? weight(from_falling((uint32_t)(sh.key[e0 + i] >> 32))) : 0.0;
      sh.wt[e0 + i] = w[i];
      c[i] = w[i];
    }
    scan(c);
#pragma unroll
    for (int i = 0; i < kPer; ++i) sh.mass[e0 + i] = c[i];
    const int m = want.k ? min(want.k, (int)n) : (int)n;
    if (threadIdx.x == 0) sh.kept = m, sh.reached = 0;
    __syncthreads();
    if (want.p < 1.f) {
      const double target = (double)want.p * (want.k ? sh.mass[m - 1] : mass);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (e0 + i < (int)n && c[i] >= target) {
          atomicMin(&sh.kept, e0 + i + 1);
          sh.reached = 1;
          break;
        }
    }
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i)
      if (e0 + i < (int)n && !want.enough(w[i], from_falling((uint32_t)(sh.key[e0 + i] >> 32)) == top)) atomicMin(&sh.kept, e0 + i);
    __syncthreads();
    if (want.p < 1.f && !want.k && !sh.reached) return false;
    const unsigned kept = (unsigned)sh.kept;
    // by number
    unsigned long long by_number[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) by_number[i] = (sh.key[e0 + i] << 32) | (unsigned)(e0 + i);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (e0 + i < (int)kept) sh.key[e0 + i] = by_number[i];
    if (threadIdx.x == 0) sh.found = (int)kept - 1;
    __syncthreads();
    sort(kept);
#pragma unroll
    for (int i = 0; i < kPer; ++i) c[i] = e0 + i < (int)kept ? sh.wt[(uint32_t)sh.key[e0 + i]] : 0.0;
    const double all = scan(c), target = (double)want.u * all;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (e0 + i < (int)kept && c[i] > target) {
        atomicMin(&sh.found, e0 + i);
        break;
      }
    __syncthreads();
    if (threadIdx.x == 0) {
      const unsigned long long key = sh.key[sh.found];
      a.tokens[r] = (int)(key >> 32);
      if (a.probs) a.probs[r] = (float)(sh.wt[(uint32_t)key] / all);
    }
    return true;
  }

  // Of the n logits in sh.key, in order, behind others that weigh `base`: the first where
  // the sum reaches the target; n, if none.
  __device__ unsigned reach(unsigned n, double base, double target) {
    double c[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const unsigned e = kPer * threadIdx.x + i;
      c[i] = e < n ? weight(from_falling((uint32_t)(sh.key[e] >> 32))) : 0.0;
    }
    if (threadIdx.x == 0) sh.found = (int)n;
    scan(c);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (kPer * threadIdx.x + i < n && base + c[i] >= target) {
        atomicMin(&sh.found, (int)(kPer * threadIdx.x) + i);
        break;
      }
    __syncthreads();
    return (unsigned)sh.found;
  }

  static constexpr int kMissed = -7;  // as a cut's number: there is none
  // CTA 0's choice becomes every CTA's cut.
  __device__ void publish(bool chooses, Cut c) {
    if (rank == 0 && chooses)
      for (int r = 0; r < ranks; ++r) *at(&sh.cut, r) = c;
    sync();
    cut = sh.cut;
    sync();
  }

  __device__ void cut_at(unsigned long long k) { publish(true, Cut{from_falling((uint32_t)(k >> 32)), (int)(uint32_t)k}); }

  // The r-th (from 1) by number of those that are kept and equal v.
  __device__ void cut_equal(float v, unsigned r, int vocab) {
    const int width = (vocab + kBins - 1) / kBins;  // (at most kList / 2)
    count([&](float x, int i) { return x == v && keeps(x, i) ? i / width : -1; });
    find((double)r, [&](int b) { return (double)sh.hist[b]; });
    const int b = sh.found;
    const unsigned before = sh.before;
    if (before + sh.in_bin < r) {  // all of them
      if (cut.x < v) cut = Cut{v, 0x7fffffff};
      __syncthreads();
      return;
    }
    const unsigned listed = gather([&](float x, int i) { return x == v && keeps(x, i) && i / width == b; });
    const unsigned at = min(r - before, max(listed, 1u)) - 1;
    cut_at(sh.key[at]);
  }

  // Bins of equal width from hi down to lo; -1 for what is outside, or not kept.
  struct Bins {
    float hi, lo, fscale;
    double scale;
    bool wide;
    __device__ __forceinline__ Bins(float h, float l) : hi(h), lo(l) {
      scale = kBins * 0.99999 / ((double)h - (double)l);
      fscale = (float)scale;
      wide = !(fscale < 1e30f && fscale > 1e-30f && h - l < 1e30f);
    }
    __device__ __forceinline__ int operator()(float v) const {
      if (v > hi || v < lo) return -1;
      const float b = wide ? (float)(((double)hi - (double)v) * scale) : (hi - v) * fscale;
      return min(kBins - 1, (int)b);
    }
    __device__ __forceinline__ float middle(int k) const { return (float)fmin((double)hi - (k + 0.5) / scale, (double)hi); }
  };

  // Cuts where `target` is reached: of how many are kept (COUNT) or of what they weigh.
  template <bool COUNT>
  // counted: the bins from the largest logit down to `least` have been; guessed_bin: and the guess is this one (below 0: not made).
  __device__ void select(double target, float least, int vocab, bool counted, int guessed_bin) {
    float hi = top, lo = least;
    double base = 0;
    for (;; counted = false, guessed_bin = -1) {
      if (!(lo < hi)) {
        // equal ones: as many as it takes
        const double w = COUNT ? 1.0 : weight(hi);
        const double r = ceil((target - base) / w);
        cut_equal(hi, (unsigned)fmin(fmax(r, 1.0), 2147483647.0), vocab);
        return;
      }
      const Bins bins(hi, lo);
      auto bin = [&](float v, int i) { return keeps(v, i) ? bins(v) : -1; };
      if (!counted) count(bin);
      int b;
      if (COUNT) {
        find(target - base, [&](int k) { return (double)sh.hist[k]; });
        b = sh.found;
        if (base + sh.before + sh.in_bin < target) return;  // there are not so many
        base += sh.before;
      } else {
        // a guess by the weights of the bins' middles; then the weights up to a window
        // around it are added up one by one
        auto guess = [&](int k) { return sh.hist[k] ? sh.hist[k] * weight(bins.middle(k)) : 0.0; };
        b = guessed_bin;
        if (b < 0) {
          find(target - base, guess);
          b = sh.found;
        }
        // (what comes before some bins around it is added up, and these are listed, in one pass;
        // mostly the sum is reached in the list)
        if (sh.hist[b] <= kList) {
          int w0 = b, w1 = b;
          unsigned many = sh.hist[b];
          for (int more = 0; more < kWindow / 2; ++more) {
            if (w1 + 1 < kBins && many + sh.hist[w1 + 1] <= kList) many += sh.hist[++w1];
            if (w0 > 0 && many + sh.hist[w0 - 1] <= kList) many += sh.hist[--w0];
          }
          double a = 0, none = 0;
          collect([&](float v, int i) {
            const int k = bin(v, i);
            if (k >= 0 && k < w0) a += weight(v);
            return k >= w0 && k <= w1;
          });
          reduce<false>(a, none);
          if (rank == 0) {
            const unsigned listed = min(sh.listed, (unsigned)kList);
            sort(listed);
            unsigned at = listed ? reach(listed, base + a, target) : 0u;
            const bool ends = w1 == kBins - 1 && listed;  // (sums in another order may fall short by a rounding)
            if (at == listed && ends) at = listed - 1;
            Cut c{0.f, kMissed};
            if (at < listed && (w0 == 0 || base + a < target)) {
              const unsigned long long k = sh.key[at];
              c = Cut{from_falling((uint32_t)(k >> 32)), (int)(uint32_t)k};
            }
            const Cut before = cut;
            publish(threadIdx.x == 0, c);
            if (c.i != kMissed) return;
            cut = before;
          } else {
            const Cut before = cut;
            publish(false, Cut{});
            if (cut.i != kMissed) return;
            cut = before;
          }
        }
        int from = 0, to = kBins - 1;  // the bin is one of these
        for (;;) {
          const int w0 = max(from, min(b - kWindow / 2, to + 1 - kWindow));
          __syncthreads();
          sh.window.clear();
          __syncthreads();
          double a = 0, none = 0;
          each([&](float v, int i) {
            const int k = bin(v, i) - w0;
            if (k >= kWindow || k + w0 < 0) return;
            const double w = weight(v);
            if (k < 0)
              a += w;
            else
              sh.window.add(k, w);
          });
          reduce<false>(a, none);  // (and the windows are complete)
          if (threadIdx.x < kWindow) {
            double u = 0;
            for (int r = 0; r < ranks; ++r) u += at(&sh.window, r)->sum(threadIdx.x);
            sh.mass[threadIdx.x] = u;
          }
          __syncthreads();
          double sum = base + a;
          int hit = -1;
          for (int k = 0; k < kWindow && hit < 0; ++k) {
            const double m = sh.mass[k];
            if (sum + m >= target || w0 + k == to)
              hit = k;
            else
              sum += m;
          }
          sync();  // (the windows have been read)
          // (the next guess begins at the window's edge, where the sum is known)
          if (base + a >= target && w0 > from) {
            to = w0 - 1;
            find(guessed(w0, guess) - (base + a - target), guess);
            b = sh.found;
          } else if (hit < 0) {
            from = w0 + kWindow;
            find(guessed(from, guess) + (target - sum), guess);
            b = sh.found;
          } else {
            b = w0 + hit;
            base = sum;
            break;
          }
        }
      }
      // (a sum in another order may be short of what one before it has shown, or above it, by a
      // rounding: of no tokens then, and what comes before them is kept whole)
      if (!COUNT && sh.hist[b] == 0) {
        while (b > 0 && sh.hist[b] == 0) --b;
        target = INFINITY;
      }
      const unsigned in_bin = sh.hist[b];
      __syncthreads();
      if (in_bin == 0) return;
      if (in_bin <= kList) {
        const unsigned listed = gather([&](float v, int i) { return bin(v, i) == b; });
        if (rank == 0) {
          unsigned at;
          if (COUNT) {
            at = (unsigned)(target - base) - 1;
          } else {
            at = reach(listed, base, target);
          }
          const unsigned long long k = sh.key[min(at, listed - 1)];
          publish(threadIdx.x == 0, Cut{from_falling((uint32_t)(k >> 32)), (int)(uint32_t)k});
        } else {
          publish(false, Cut{});
        }
        return;
      }
      double l = -INFINITY, h = -INFINITY;
      each([&](float v, int i) {
        if (bin(v, i) != b) return;
        h = fmax(h, (double)v);
        l = fmax(l, -(double)v);
      });
      reduce<true>(h, l);
      hi = (float)h, lo = (float)-l;
    }
  }

  // The row's token.  x, n, first, ranks and rank are set, sh.powers filled, high the
  // largest logit and low the smallest above -inf negated, of the whole row.
  // mine: the largest that this thread has seen, of logits that no other one has seen.
  __device__ void run(const Sample &a, long long r, double high, double low, float mine) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    top = (float)high;
    const bool writes = rank == 0 && threadIdx.x == 0;
    if (high == -INFINITY) {
      if (writes) {
        a.tokens[r] = -1;
        if (a.probs) a.probs[r] = 0.f;
      }
      return;
    }
    const Want want(a, r);
    if (!(want.t > 0.f)) {
      double best = -INFINITY, none = 0;
      each([&](float v, int i) {
        if (v == top) best = fmax(best, -(double)i);
      });
      reduce<true>(best, none);
      if (writes) {
        a.tokens[r] = (int)-best;
        if (a.probs) a.probs[r] = 1.f;
      }
      return;
    }
    weight.set(top, want.t);
    cut = Cut{-INFINITY, -1};  // (-inf weighs nothing)
    // logits below this have no weight
    const float least = high == INFINITY ? top : (float)fmax(-low, high - kFar * (double)want.t);
    double mass = 0, none = 0;
    bool counted = false;
    int guess = -1;
    if (want.p < 1.f && !want.k) {
      if (least < top) {  // (with the count that follows)
        const Bins bins(top, least);
        count([&](float v, int) {
          const int b = bins(v);
          if (b >= 0) mass += weight(v);
          return b;
        });
        counted = true;
      } else {
        each([&](float v, int) { mass += v > -INFINITY ? weight(v) : 0.0; });
      }
      reduce<false>(mass, none);
    }
    if ((want.p < 1.f || want.k) && want.k <= kList && least < top) {
      // what is kept, if it is not much, goes through one list
      const Bins bins(top, least);
      // At least k logits are no smaller than the k-th of the threads' largest, and of n
      // threads' mostly no more than n log(1 / (1 - k / n)).  That k-th is found with one
      // count a thread (a row of 131072, k = 50: 46000 clocks in all, against 53000 or more
      // with a count of every logit).
      const float threads = (float)(ranks * kThreads);
      if (want.k && want.k < threads && -threads * log1pf(-want.k / threads) < 0.85f * kList) {
        clear();
        const int own = bins(mine);
        if (own >= 0) atomicAdd(&sh.hist[own], 1u);
        merge();
        find((double)want.k, [&](int b) { return (double)sh.hist[b]; });
        const int b = sh.found;
        const bool there = sh.before + sh.in_bin >= (unsigned)want.k;
        __syncthreads();
        if (there) {
          collect([&](float v, int) { return (unsigned)bins(v) <= (unsigned)b; });
          const unsigned n = *at(&sh.listed, 0);
          sync();  // (all have read it)
          if (n <= kList) {
            if (rank == 0) {
              sort(n);
              finish(n, want, mass, a, r);
            }
            return;
          }
        }
      }
      if (want.k) count([&](float v, int) { return bins(v); });
      counted = true;
      if (want.k)
        find((double)want.k, [&](int b) { return (double)sh.hist[b]; });
      else  // by the bins' middles: that their sum is not the logits' comes from the first bins above all, before the cut
        find((double)want.p * mass, [&](int b) { return sh.hist[b] ? sh.hist[b] * weight(bins.middle(b)) : 0.0; }, mass);
      int b = sh.found;
      unsigned many = sh.before + sh.in_bin;
      if (!want.k) {  // (the bins' middles are a guess: two more)
        guess = b;
        for (int more = 0; more < 2 && b + 1 < kBins; ++more) many += sh.hist[++b];
      }
      __syncthreads();
      if (many <= kList) {
        const unsigned n = gather([&](float v, int) { return (unsigned)bins(v) <= (unsigned)b; });
        bool done = true;
        if (rank == 0) done = finish(n, want, mass, a, r);
        if (want.k) return;
        if (rank == 0 && threadIdx.x < ranks) *at(&sh.reached, (int)threadIdx.x) = done;
        sync();
        if (sh.reached) return;
      }
    }
    if (want.k) select<true>((double)want.k, least, a.vocab, counted, -1);
    if (want.p < 1.f) {
      if (want.k) {
        mass = 0;
        each([&](float v, int i) { mass += keeps(v, i) ? weight(v) : 0.0; });
        reduce<false>(mass, none);
      }
      select<false>((double)want.p * mass, least, a.vocab, counted && !want.k, guess);
    }
    // ---- running sums, by number: a warp has a piece of the slice, in steps of 128
    const float lowest = want.floor(top);
    auto kept = [&](float v, int i) {
      if (!keeps(v, i) || v < lowest) return 0.0;
      const double w = weight(v);
      return want.enough(w, v == top) ? w : 0.0;
    };
    const int piece = (a.slice + 128 * kWarps - 1) / (128 * kWarps) * 128;
    const int j0 = min(warp * piece, n), j1 = min(j0 + piece, n);
    double weighs = 0;
    for (int j = j0 + 4 * lane; j < j1; j += 128) {
      float v[4];
      load4(j, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) weighs += kept(v[i], first + j + i);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) weighs += __shfl_xor_sync(0xffffffffu, weighs, o);
    if (lane == 0) sh.seg[warp] = weighs;
    __syncthreads();
    mass = threadIdx.x < kWarps ? sh.seg[threadIdx.x] : 0.0;
    reduce<false>(mass, none);
    const double target = (double)want.u * mass;
    // the CTA, then the warp, where the sum passes the target
    double before = 0;
    int q = 0;
    for (; q + 1 < ranks; ++q) {
      const double s = sh.part[turn][q][0];
      if (before + s > target) break;
      before += s;
    }
    // (a last CTA without weight, by a rounding: the last one with some)
    while (q > 0 && sh.part[turn][q][0] == 0) --q;
    if (q != rank) return;
    int w = 0;
    for (; w + 1 < kWarps; ++w) {
      if (before + sh.seg[w] > target) break;
      before += sh.seg[w];
    }
    while (w > 0 && sh.seg[w] == 0) --w;
    if (w != warp) return;
    int token = -1;
    double share = 0;
    for (int j = j0; j < j1; j += 128) {
      float v[4];
      double c[4], s = 0;
      load4(j + 4 * lane, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = j + 4 * lane < j1 ? kept(v[i], first + j + 4 * lane + i) : 0.0, s += c[i];
      const double sum = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      const unsigned some = __ballot_sync(0xffffffffu, sum > 0), over = __ballot_sync(0xffffffffu, sum > 0 && before + s > target);
      if (some) {
        const int l = over ? __ffs(over) - 1 : 31 - __clz(some);
        // the last of the lane's that weighs something, or the first that passes
        double run = before + (s - sum);
        int at = -1;
        double sh_at = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (c[i] > 0 && (at < 0 || !(run > target))) at = i, sh_at = c[i];
          run += c[i];
        }
        token = __shfl_sync(0xffffffffu, first + j + 4 * lane + at, l);
        share = __shfl_sync(0xffffffffu, sh_at, l);
      }
      if (over) break;
      before += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) {
      a.tokens[r] = token;
      if (a.probs) a.probs[r] = (float)(share / mass);
    }
  }
};

// (Two CTAs an SM, so 64 registers a thread: some 340 bytes spill.)
template <class T>
__global__ void __launch_bounds__(kClusterThreads, 2) sample_k(const __grid_constant__ Sample a) {
  extern __shared__ __align__(16) uint8_t slice_raw[];
  __shared__ SampleShared sh;
  constexpr int kThreads = kClusterThreads;
  Row<T, kThreads> row(sh);
  row.ranks = a.ranks;
  row.rank = a.ranks > 1 ? (int)(blockIdx.x % a.ranks) : 0;
  const long long r = blockIdx.x / a.ranks;
  row.first = min(row.rank * a.slice, a.vocab);
  row.n = min(a.slice, a.vocab - row.first);
  // (a CTA's shared memory is there for others once it runs: the wait for that is below,
  // before the first exchange, so that it passes under the loads)
  if (a.ranks > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  fill_powers(sh.powers);
  pdl_wait_and_release();
  const T *x = static_cast<const T *>(a.x) + r * a.stride + row.first;
  row.x = x;
  row.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0;
  float high = -INFINITY, low = -INFINITY;  // the largest logit, and the smallest above -inf negated
  T *const slice = reinterpret_cast<T *>(slice_raw);
  constexpr int kEach = 16 / sizeof(T);
  auto look = [&](T v) {
    const float f = logit(v);
    high = fmaxf(high, f);
    if (f > -INFINITY) low = fmaxf(low, -f);
  };
  if (row.vec && a.resident) {
    constexpr int kAtOnce = 4;
    for (int j0 = threadIdx.x * kEach; j0 < row.n; j0 += kAtOnce * kThreads * kEach) {
      uint4 w[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q)
        if (j0 + q * kThreads * kEach + kEach <= row.n) w[q] = __ldg(reinterpret_cast<const uint4 *>(x + j0 + q * kThreads * kEach));
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int j = j0 + q * kThreads * kEach;
        if (j + kEach <= row.n) {
          *reinterpret_cast<uint4 *>(slice + j) = w[q];
          T t[kEach];
          *reinterpret_cast<uint4 *>(t) = w[q];
#pragma unroll
          for (int i = 0; i < kEach; ++i) look(t[i]);
        } else {
          for (int i = j; i < row.n; ++i) {
            const T v = x[i];
            slice[i] = v;
            look(v);
          }
        }
      }
    }
  } else {
    for (int j = threadIdx.x; j < row.n; j += kThreads) {
      const T v = x[j];
      if (a.resident) slice[j] = v;
      look(v);
    }
  }
  if (a.resident) row.x = slice, row.vec = true;
  double h = high, l = low;
  if (a.ranks > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  row.template reduce<true>(h, l);  // (and the slice is in place)
  row.run(a, r, h, l, high);
}

// ---------------------------------------------------------------- by counting values
//
// Keys are the bits of a logit, turned so that larger logits come first: 16 bits, or
// the upper 16 of 32.  Counters are 16 bits too, two a word; their sum tells whether
// one of them ran over (more than 65535 equal logits), and such a row goes the other
// kernel's way.  A cut of 32-bit logits lies inside a bin: the bin's logits are
// counted again by their lower 16 bits.
constexpr int kCountThreads = 1024, kCountWarps = kCountThreads / 32;
constexpr int kWords = 32768, kGroups = 2048;     // two counters a word; 32 counters a group
constexpr int kSpan = 256;                        // tokens of a running sum's entry

struct CountShared {
  union {
    unsigned hist[kWords];
    SampleShared other;
  };
  double sum[kGroups];
  unsigned cnt[kGroups];
  double powers[kPowers];
  Window window;
  double red[kCountWarps];
  unsigned redc[kCountWarps];
  unsigned bin, before;
  double mass;
};

template <class T>
struct Key;
template <>
struct Key<float> {
  static constexpr uint32_t kInf = 0;
  static __device__ __forceinline__ float value(uint32_t k) { return from_falling(k); }
};
template <int MANTISSA>
struct Key16 {
  static constexpr uint32_t kInf = 0x7fffu & ~((1u << MANTISSA) - 1u);
  static __device__ __forceinline__ uint32_t bits(uint32_t k) { return k >> 31 ? k >> 16 : 0x7fffu ^ (k >> 16); }
};
template <>
struct Key<__half> : Key16<10> {
  static __device__ __forceinline__ float value(uint32_t k) { return __half2float(__ushort_as_half((unsigned short)bits(k))); }
};
template <>
struct Key<__nv_bfloat16> : Key16<7> {
  static __device__ __forceinline__ float value(uint32_t k) { return __uint_as_float(bits(k) << 16); }
};
constexpr uint32_t kDead = 0xffffffffu;  // -inf, NaN

// The key of a logit given by its bits (16-bit ones in the lower half).
template <class T>
__device__ __forceinline__ uint32_t key_of(uint32_t b) {
  if (sizeof(T) == 4) {
    const float x = __uint_as_float(b) + 0.f;
    return x > -INFINITY ? falling(x) : kDead;
  }
  constexpr uint32_t inf = Key<T>::kInf;
  uint32_t k = b >> 15 ? b : 0x7fffu ^ b;
  k -= k == 0x8000u;                                   // -0 is 0
  return k - (0x7fffu ^ inf) < 0x8000u + inf - (0x7fffu ^ inf) ? k << 16 : kDead;
}

template <class T>
struct Counter {
  static constexpr int kEach = 16 / sizeof(T);
  static constexpr bool kWide = sizeof(T) == 4;
  CountShared &sh;
  const T *x;
  int vocab, skip;            // skip: how many elements before the row its first 16-byte piece begins
  float top;
  Weights weight;
  uint32_t cut = kDead - 1;   // kept: smaller keys, and the first `room` (by number) of this one
  unsigned room = 0xffffffffu;

  __device__ Counter(CountShared &s) : sh(s) { weight.powers = s.powers; }

  __device__ __forceinline__ double weight_at(uint32_t k) const { return weight(Key<T>::value(k)); }

  // The keys of piece c of the row (16 bytes, in order).
  __device__ __forceinline__ void keys(int c, uint32_t (&k)[kEach]) const {
    const int j0 = c * kEach - skip;
    if (j0 >= 0 && j0 + kEach <= vocab) {
      unpack(__ldg(reinterpret_cast<const uint4 *>(x + j0)), k);
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        k[i] = kDead;
        if (j0 + i >= 0 && j0 + i < vocab)
          k[i] = key_of<T>(sizeof(T) == 4 ? __float_as_uint(*reinterpret_cast<const float *>(x + j0 + i)) : *reinterpret_cast<const uint16_t *>(x + j0 + i));
      }
    }
  }
  // Piece c as it lies in memory, with NaN where it is not the row's.
  __device__ __forceinline__ uint4 piece(int c) const {
    const int j0 = c * kEach - skip;
    if (j0 >= 0 && j0 + kEach <= vocab) return __ldg(reinterpret_cast<const uint4 *>(x + j0));
    uint32_t w[4] = {kDead, kDead, kDead, kDead};
    if (!kWide)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + i >= 0 && j0 + i < vocab) {
          const uint32_t b = *reinterpret_cast<const uint16_t *>(x + j0 + i);
          w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | b << 16 : (w[i / 2] & 0xffff0000u) | b;
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ void unpack(uint4 u, uint32_t (&k)[kEach]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (kWide) {
        k[i] = key_of<T>(w[i]);
      } else {
        k[2 * i % kEach] = key_of<T>(w[i] & 0xffffu);
        k[(2 * i + 1) % kEach] = key_of<T>(w[i] >> 16);
      }
    }
  }
  __device__ __forceinline__ int pieces() const { return (skip + vocab + kEach - 1) / kEach; }
  // f(keys of a piece) for every piece, several in flight.
  template <class F>
  __device__ __forceinline__ void each(F &&f) const {
    constexpr int kAtOnce = 4;
    const int n = pieces();
    for (int c0 = threadIdx.x; c0 < n; c0 += kAtOnce * kCountThreads) {
      uint4 u[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int j0 = (c0 + q * kCountThreads) * kEach - skip;
        if (j0 >= 0 && j0 + kEach <= vocab) u[q] = __ldg(reinterpret_cast<const uint4 *>(x + j0));
      }
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int c = c0 + q * kCountThreads, j0 = c * kEach - skip;
        if (c >= n) break;
        uint32_t k[kEach];
        if (j0 >= 0 && j0 + kEach <= vocab)
          unpack(u[q], k);
        else
          keys(c, k);
        f(k);
      }
    }
  }

  __device__ double total(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.red[0];
    for (int w = 1; w < kCountWarps; ++w) v += sh.red[w];
    return v;
  }
  __device__ unsigned total(unsigned v) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.redc[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kCountWarps; ++w) v += sh.redc[w];
    return v;
  }

  __device__ __forceinline__ void clear() {
    __syncthreads();
    for (int i = threadIdx.x; i < kWords / 4; i += kCountThreads) reinterpret_cast<uint4 *>(sh.hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  __device__ __forceinline__ void add(uint32_t b) { atomicAdd(&sh.hist[b >> 1], 1u << (16 * (b & 1))); }
  __device__ __forceinline__ unsigned counter(uint32_t b) const { return sh.hist[b >> 1] >> (16 * (b & 1)) & 0xffffu; }

  // Counts of the groups of 32 counters: their sum.
  __device__ unsigned group_counts() {
    __syncthreads();
    unsigned all = 0;
#pragma unroll
    for (int z = 0; z < kGroups / kCountThreads; ++z) {
      const int g = threadIdx.x + z * kCountThreads;
      unsigned n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // (the lanes begin at different quarters: no two meet in a bank)
        const uint4 u = reinterpret_cast<const uint4 *>(sh.hist)[4 * g + ((i + (threadIdx.x >> 1)) & 3)];
        n += (u.x & 0xffffu) + (u.x >> 16) + (u.y & 0xffffu) + (u.y >> 16) + (u.z & 0xffffu) + (u.z >> 16) + (u.w & 0xffffu) + (u.w >> 16);
      }
      sh.cnt[g] = n;
      all += n;
    }
    return total(all);  // (barriers: the counts are in place)
  }
  // Weights of the groups; key(b) stands for counter b.
  template <class F>
  __device__ void group_weights(F &&key) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g0 = 0; g0 < kGroups; g0 += 32 * kCountWarps) {
      const int mine = g0 + warp + kCountWarps * lane;
      unsigned some = __ballot_sync(0xffffffffu, sh.cnt[mine] != 0);
      if (!(some >> lane & 1)) sh.sum[mine] = 0.0;
      for (; some; some &= some - 1) {
        const int g = g0 + warp + kCountWarps * (__ffs(some) - 1);
        const unsigned c = counter(32 * g + lane);
        double w = c ? (double)c * weight_at(key(32 * g + lane)) : 0.0;
#pragma unroll
        for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        if (lane == 0) sh.sum[g] = w;
      }
    }
    __syncthreads();
  }

  // What the counters before counter b weigh.
  template <class F>
  __device__ double weight_before(uint32_t b, F &&key) {
    double m = 0;
    for (uint32_t g = threadIdx.x; g < b / 32; g += kCountThreads) m += sh.sum[g];
    if (threadIdx.x < b % 32) {
      const uint32_t k = (b & ~31u) + threadIdx.x;
      if (counter(k)) m += (double)counter(k) * weight_at(key(k));
    }
    return total(m);
  }

  // Running sums over the groups, two a thread: of counts and (MASS) of weights; the
  // first counter where they reach the target into sh.bin, what lies before it into
  // sh.before and sh.mass.  False: they do not reach it.
  template <bool MASS, class F>
  __device__ bool locate(double target, F &&key) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g0 = 2 * threadIdx.x;
    unsigned c[2] = {sh.cnt[g0], sh.cnt[g0 + 1]};
    double m[2] = {MASS ? sh.sum[g0] : (double)c[0], MASS ? sh.sum[g0 + 1] : (double)c[1]};
    double s = m[0] + m[1];
    unsigned n = c[0] + c[1];
    const double s0 = s;
    const unsigned n0 = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, s, o);
      const unsigned u = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) s += t, n += u;
    }
    __syncthreads();
    if (lane == 31) sh.red[warp] = s, sh.redc[warp] = n;
    if (threadIdx.x == 0) sh.bin = kGroups;
    __syncthreads();
    double before = 0;
    unsigned nb = 0;
    for (int w = 0; w < warp; ++w) before += sh.red[w], nb += sh.redc[w];
    before += s - s0;
    nb += n - n0;
    // (an empty group may seem to be the first: what is before it is added up in another order
    // than by the threads before this one)
    const int at = c[0] && before + m[0] >= target ? 0 : c[1] && before + m[0] + m[1] >= target ? 1 : 2;
    if (at < 2) atomicMin(&sh.bin, (unsigned)(g0 + at));
    __syncthreads();
    const unsigned g = sh.bin;
    __syncthreads();
    if (g == kGroups) return false;
    if (g / 2 == threadIdx.x) {
      sh.mass = before + (at ? m[0] : 0.0);
      sh.before = nb + (at ? c[0] : 0u);
    }
    __syncthreads();
    if (warp == 0) {  // inside the group
      const unsigned k = counter(32 * g + lane);
      double v = MASS ? (k ? (double)k * weight_at(key(32 * g + lane)) : 0.0) : (double)k;
      const double v0 = v;
      unsigned q = k;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, v, o);
        const unsigned u = __shfl_up_sync(0xffffffffu, q, o);
        if (lane >= o) v += t, q += u;
      }
      // (the last counter that is not empty, where the sums in this order fall short by a rounding)
      const unsigned some = __ballot_sync(0xffffffffu, k > 0), over = __ballot_sync(0xffffffffu, k > 0 && sh.mass + v >= target);
      const int l = over ? __ffs(over) - 1 : 31 - __clz(some);
      const double base = sh.mass;
      const unsigned nbase = sh.before;
      __syncwarp();
      if (lane == l) {
        sh.bin = 32 * g + lane;
        sh.mass = base + (v - v0);
        sh.before = nbase + (q - k);
      }
    }
    __syncthreads();
    return true;
  }

  // How many of n equal ones, weighing w each, it takes from `base` to the target.
  static __device__ __forceinline__ unsigned enough(double target, double base, double w, unsigned n) {
    const double r = ceil((target - base) / w);
    return r > 1.0 ? (unsigned)fmin(r, (double)n) : 1u;
  }

  // Counts the lower halves of the keys of bin b.  False: a counter ran over.
  __device__ bool count_inside(uint32_t b, unsigned n) {
    clear();
    each([&](const uint32_t(&k)[kEach]) {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (k[i] >> 16 == b && k[i] != kDead) add(k[i] & 0xffffu);
    });
    return group_counts() == n;
  }

  static __device__ __forceinline__ float2 values2(uint32_t w) {
    if (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  // Two 16-bit keys from two logits (-0 is not 0 here).
  static __device__ __forceinline__ uint32_t keys2(uint32_t w) {
    return w ^ 0x7fff7fffu ^ ((w >> 15 & 0x00010001u) * 0x7fffu);
  }
  // The same with -0 as 0.
  static __device__ __forceinline__ uint32_t keys2_zero(uint32_t w) {
    const uint32_t k = keys2(w);
    return k - (__vcmpeq2(k, 0x80008000u) & 0x00010001u);
  }
  static constexpr uint32_t kInf = Key<T>::kInf, kFirst16 = 0x7fffu - kInf, kEnd16 = 0x8000u + kInf;  // keys of logits: kFirst16 .. kEnd16 - 1

  // Counts the upper halves of all keys; how many logits there are, and the first key.
  __device__ bool count_all(unsigned &live, uint32_t &first) {
    clear();
    unsigned n = 0;
    uint32_t least = kDead;
    if constexpr (kWide) {
      each([&](const uint32_t(&k)[kEach]) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (k[i] != kDead) {
            add(k[i] >> 16);
            least = min(least, k[i]);
            ++n;
          }
      });
    } else {
      auto two = [&](uint32_t w) {
        const uint32_t k = keys2(w), lo = k & 0xffffu, hi = k >> 16;
        // (NaN with the sign bit and -inf are left out here, the other NaN and -0 below)
        if (lo < kEnd16) add(lo), ++n;
        if (hi < kEnd16) add(hi), ++n;
      };
      constexpr int kAtOnce = 4;
      const int c1 = pieces() - 1;
      for (int c0 = threadIdx.x; c0 <= c1; c0 += kAtOnce * kCountThreads) {
        uint4 u[kAtOnce];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) u[q] = piece(c0 + q * kCountThreads);
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q)
          if (c0 + q * kCountThreads <= c1) two(u[q].x), two(u[q].y), two(u[q].z), two(u[q].w);
      }
      __syncthreads();
      unsigned out = 0;
      for (uint32_t b = threadIdx.x; b < kFirst16; b += kCountThreads) out += counter(b);
      out = total(out);  // (a barrier: all have looked)
      for (uint32_t b = threadIdx.x; b < kFirst16 / 2; b += kCountThreads) sh.hist[b] = 0;
      if (threadIdx.x == 0) {
        if (kFirst16 & 1) sh.hist[kFirst16 / 2] &= 0xffff0000u;
        const unsigned zero = counter(0x8000u);
        sh.hist[0x4000] -= zero;
        // (should the sum run over, the total tells)
        sh.hist[0x3fff] += zero << 16;
      }
      if (threadIdx.x == 1) n -= out;
    }
    live = total(n);
    if constexpr (kWide) {
      least = __reduce_min_sync(0xffffffffu, least);
      __syncthreads();
      if ((threadIdx.x & 31) == 0) sh.redc[threadIdx.x >> 5] = least;
      __syncthreads();
      first = sh.redc[0];
      for (int w = 1; w < kCountWarps; ++w) first = min(first, sh.redc[w]);
    }
    const bool fits = group_counts() == live;
    if constexpr (!kWide) {
      // the first counter that is not empty
      __syncthreads();
      if (threadIdx.x == 0) sh.bin = kGroups;
      __syncthreads();
      for (int g = threadIdx.x; g < kGroups; g += kCountThreads)
        if (sh.cnt[g]) {
          atomicMin(&sh.bin, (unsigned)g);
          break;
        }
      __syncthreads();
      const unsigned g = min(sh.bin, (unsigned)kGroups - 1);
      const unsigned some = __ballot_sync(0xffffffffu, counter(32 * g + (threadIdx.x & 31)) != 0);
      first = (32 * g + __ffs(some) - 1) << 16;
    }
    return fits;
  }

  // The first key alone (kDead: there are no logits).
  __device__ uint32_t first_key() {
    uint32_t least = kDead;
    if constexpr (kWide) {
      each([&](const uint32_t(&k)[kEach]) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) least = min(least, k[i]);
      });
    } else {
      constexpr int kAtOnce = 4;
      constexpr uint32_t kBefore = kFirst16 * 0x10001u;  // (NaN without the sign bit goes behind all others)
      const int c1 = pieces() - 1;
      uint32_t two = kDead;
      for (int c0 = threadIdx.x; c0 <= c1; c0 += kAtOnce * kCountThreads) {
        uint4 u[kAtOnce];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) u[q] = c0 + q * kCountThreads <= c1 ? piece(c0 + q * kCountThreads) : make_uint4(kDead, kDead, kDead, kDead);
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q)
          two = __vminu2(two, __vminu2(__vminu2(__vsub2(keys2_zero(u[q].x), kBefore), __vsub2(keys2_zero(u[q].y), kBefore)),
                                       __vminu2(__vsub2(keys2_zero(u[q].z), kBefore), __vsub2(keys2_zero(u[q].w), kBefore))));
      }
      const uint32_t k = min(two & 0xffffu, two >> 16);
      least = k < kEnd16 - kFirst16 ? (k + kFirst16) << 16 : kDead;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.redc[threadIdx.x >> 5] = least;
    __syncthreads();
    least = sh.redc[0];
    for (int w = 1; w < kCountWarps; ++w) least = min(least, sh.redc[w]);
    return least;
  }

  // All of bin b is kept, and nothing behind it (b < 0xffff).
  __device__ __forceinline__ void cut_behind(uint32_t b) { cut = b << 16 | 0xffffu, room = 0xffffffffu; }

  // The cut.  False: a counter ran over, or a guess was too far off.
  __device__ bool select(const Want &want, unsigned live, uint32_t first) {
    auto upper = [](uint32_t b) { return b << 16; };
    // (of a bin of 32-bit logits the middle, but no more than the largest logit)
    auto middle = [first](uint32_t b) { return kWide ? max(b << 16 | 0x8000u, first) : b << 16; };
    if (want.k && (unsigned)want.k < live) {
      locate<false>((double)want.k, upper);
      const uint32_t b = sh.bin;
      unsigned need = want.k - sh.before;
      const unsigned in_bin = counter(b);
      if (kWide) {
        if (!count_inside(b, in_bin)) return false;
        locate<false>((double)need, upper);
        need -= sh.before;
        cut = b << 16 | sh.bin;
        if (want.p < 1.f) {
          unsigned n;
          uint32_t f;
          if (!count_all(n, f)) return false;
        }
      } else {
        cut = b << 16;
      }
      room = need;
    }
    if (!(want.p < 1.f)) return true;
    group_weights(middle);
    const double wc = cut < kDead - 1 ? weight_at(cut) : 0.0;
    double mass;
    // (the cut's own bin: as much as there is room for)
    mass = cut < kDead - 1 ? weight_before(cut >> 16, middle) + room * wc : weight_before(0x10000u, middle);
    constexpr double kLeast = 1e-300;  // (something is kept, also with top_p 0)
    double target = fmax((double)want.p * mass, kLeast);
    if (!kWide) {
      if (!locate<true>(target, middle)) return true;  // (p is 1, but for a rounding)
      const uint32_t b = sh.bin;
      if ((b << 16) > cut) return true;
      const unsigned r = enough(target, sh.mass, weight_at(b << 16), counter(b));
      room = (b << 16) < cut ? r : min(room, r);
      cut = b << 16;
      return true;
    }
    // The middles gave a guess of the bin; the weights up to a window around it are added up one by one.
    uint32_t b = locate<true>(target, middle) ? sh.bin : 0xffffu;
    // (top_k's cut lies in the last of them: its bin is in the window or behind it, so that what
    // there is room for counts)
    uint32_t lo = 0, hi = cut >> 16;  // the bin is one of these
    for (;;) {
      const uint32_t from = min(max(b > kWindow / 2 ? b - kWindow / 2 : 0u, lo), max(lo, hi + 1 > kWindow ? hi + 1 - kWindow : 0u));
      __syncthreads();
      sh.window.clear();
      __syncthreads();
      double below = 0, above = 0;
      each([&](const uint32_t(&k)[kEach]) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (k[i] < cut) {
            const double w = weight_at(k[i]);
            const uint32_t at = (k[i] >> 16) - from;
            if (k[i] >> 16 < from)
              below += w;
            else if (at >= kWindow)
              above += w;
            else
              sh.window.add(at, w);
          }
      });
      below = total(below);
      above = total(above);
      double in[kWindow], all = below + above + room * wc;
      if (!(cut < kDead - 1)) all = below + above;
#pragma unroll
      for (int i = 0; i < kWindow; ++i) in[i] = sh.window.sum(i), all += in[i];
      const uint32_t at = (cut >> 16) - from;
      target = fmax((double)want.p * all, kLeast);
      if (target <= below && from > lo) {  // (the next guess begins at the window's edge, where the sum is known)
        hi = from - 1;
        b = locate<true>(fmax(weight_before(from, middle) - (below - target), kLeast), middle) ? sh.bin : hi;
        continue;
      }
      double base = below;
      int hit = -1;
#pragma unroll
      for (int i = 0; i < kWindow; ++i) {
        const double m = in[i] + ((uint32_t)i == at && cut < kDead - 1 ? room * wc : 0.0);
        if (hit < 0 && base + m >= target) hit = i;
        if (hit < 0) base += m;
      }
      if (hit < 0) {
        lo = from + kWindow;
        if (lo > hi) {
          // (sums in another order have shown that it is no later than hi)
          if (hi < cut >> 16) cut_behind(hi);
          return true;
        }
        b = locate<true>(weight_before(lo, middle) + (target - base), middle) ? sh.bin : hi;
        continue;
      }
      const uint32_t bin = from + hit;
      const unsigned in_bin = counter(bin);
      if (in_bin == 0 || !count_inside(bin, in_bin)) return false;
      auto inside = [bin](uint32_t l) { return bin << 16 | l; };
      group_weights(inside);
      if (!locate<true>(target - base, inside)) {  // (short of it by a rounding)
        if (bin < cut >> 16) cut_behind(bin);
        return true;
      }
      const uint32_t key = bin << 16 | sh.bin;
      if (key > cut) return true;
      const unsigned r = enough(target - base, sh.mass, weight_at(key), counter(sh.bin));
      room = key < cut ? r : min(room, r);
      cut = key;
      return true;
    }
  }

  // The running sums of the kept tokens, by number, and the token where they pass u of them all.
  __device__ void choose(const Want &want, const Sample &a, long long r, uint32_t first) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float lowest = want.floor(top);
    const double wc = weight_at(cut);
    const bool cut_counts = cut < kDead - 1 && want.enough(wc, Key<T>::value(cut) == top);
    constexpr int kLanePieces = kSpan / 32 / kEach;  // pieces of a lane in an entry
    const int n = pieces(), entries = (n + 32 * kLanePieces - 1) / (32 * kLanePieces);
    auto before_cut = [&](uint32_t k) {
      if (k >= cut) return 0.0;
      const float v = Key<T>::value(k);
      if (v < lowest) return 0.0;
      const double w = weight(v);
      return want.enough(w, v == top) ? w : 0.0;
    };
    const uint32_t k0 = first >> 16, end = cut >> 16;
    const bool table = !kWide && end - k0 <= sizeof(sh.hist) / sizeof(double);
    __syncthreads();
    for (int e = threadIdx.x; e < kGroups; e += kCountThreads) sh.sum[e] = 0.0, sh.cnt[e] = 0;
    if constexpr (kWide) {
      __syncthreads();
      constexpr int kAtOnce = 2;
      for (int e0 = warp; e0 < entries; e0 += kAtOnce * kCountWarps) {
        uint32_t k[kAtOnce][kLanePieces][kEach];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
          for (int z = 0; z < kLanePieces; ++z) {
            const int c = ((e0 + q * kCountWarps) * 32 + lane) * kLanePieces + z;
#pragma unroll
            for (int i = 0; i < kEach; ++i) k[q][z][i] = kDead;
            if (e0 + q * kCountWarps < entries && c < n) keys(c, k[q][z]);
          }
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          uint32_t least = kDead;
#pragma unroll
          for (int z = 0; z < kLanePieces; ++z)
#pragma unroll
            for (int i = 0; i < kEach; ++i) least = min(least, k[q][z][i]);
          if (!__any_sync(0xffffffffu, least <= cut)) continue;
          double s = 0;
          unsigned equal = 0;
          if (least <= cut) {
#pragma unroll
            for (int z = 0; z < kLanePieces; ++z)
#pragma unroll
              for (int i = 0; i < kEach; ++i) {
                s += before_cut(k[q][z][i]);
                equal += k[q][z][i] == cut;
              }
          }
          equal = __reduce_add_sync(0xffffffffu, equal);
#pragma unroll
          for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if (lane == 0) sh.sum[e0 + q * kCountWarps] = s, sh.cnt[e0 + q * kCountWarps] = cut_counts ? equal : 0u;
        }
      }
    } else if (!table) {
      // more values than a table holds (or everything) is kept: weights from the logits as they are
      __syncthreads();
      constexpr int kAtOnce = 4;
      const bool bounded = want.min_p > 0.f, all_kept = cut == kDead - 1;
      const float last = all_kept ? -INFINITY : Key<T>::value(cut);
      for (int e0 = warp; e0 < entries; e0 += kAtOnce * kCountWarps) {
        uint4 u[kAtOnce];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const int c = (e0 + q * kCountWarps) * 32 + lane;
          u[q] = c < n ? piece(c) : make_uint4(kDead, kDead, kDead, kDead);
        }
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          if (e0 + q * kCountWarps >= entries) break;
          const uint32_t w[4] = {u[q].x, u[q].y, u[q].z, u[q].w};
          double s = 0;
          unsigned equal = 0;
          auto weigh = [&](float v) {
            if (!(v > last)) {
              equal += v == last;
            } else if (!(v < lowest)) {
              const double w = weight(v);
              s += !bounded || want.enough(w, v == top) ? w : 0.0;
            }
          };
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = values2(w[i]);
            weigh(f.x);
            weigh(f.y);
          }
          equal = __reduce_add_sync(0xffffffffu, equal);
#pragma unroll
          for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if (lane == 0) sh.sum[e0 + q * kCountWarps] = s, sh.cnt[e0 + q * kCountWarps] = cut_counts ? equal : 0u;
        }
      }
    } else {
      // the weights of the kept values, in the counters' place
      double *const weights = reinterpret_cast<double *>(sh.hist);
      for (uint32_t i = threadIdx.x; k0 + i < end; i += kCountThreads) weights[i] = before_cut((k0 + i) << 16);
      __syncthreads();
      auto weigh = [&](uint32_t k, double &s, unsigned &equal) {
        if (k < end) s += weights[k - k0];
        equal += k == end;
      };
      constexpr int kAtOnce = 4;
      for (int e0 = warp; e0 < entries; e0 += kAtOnce * kCountWarps) {
        uint4 u[kAtOnce];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const int c = (e0 + q * kCountWarps) * 32 + lane;
          u[q] = c < n ? piece(c) : make_uint4(kDead, kDead, kDead, kDead);
        }
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const uint32_t k[4] = {keys2_zero(u[q].x), keys2_zero(u[q].y), keys2_zero(u[q].z), keys2_zero(u[q].w)};
          const uint32_t m = __vminu2(__vminu2(k[0], k[1]), __vminu2(k[2], k[3])), least = min(m & 0xffffu, m >> 16);
          // (a NaN without the sign bit has a smaller key than any logit: it passes here, and weighs nothing below)
          if (!__any_sync(0xffffffffu, least <= end)) continue;
          double s = 0;
          unsigned equal = 0;
          if (least <= end) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t lo = k[i] & 0xffffu, hi = k[i] >> 16;
              if (lo >= k0) weigh(lo, s, equal);
              if (hi >= k0) weigh(hi, s, equal);
            }
          }
          equal = __reduce_add_sync(0xffffffffu, equal);
#pragma unroll
          for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if (lane == 0 && e0 + q * kCountWarps < entries) sh.sum[e0 + q * kCountWarps] = s, sh.cnt[e0 + q * kCountWarps] = cut_counts ? equal : 0u;
        }
      }
    }
    __syncthreads();
    // two entries a thread: how many equal to the cut come before, then sums
    const int e0 = 2 * threadIdx.x;
    const unsigned c[2] = {sh.cnt[e0], sh.cnt[e0 + 1]};
    unsigned nq = c[0] + c[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned t = __shfl_up_sync(0xffffffffu, nq, o);
      if (lane >= o) nq += t;
    }
    if (lane == 31) sh.redc[warp] = nq;
    __syncthreads();
    unsigned have = nq - c[0] - c[1];
    for (int w = 0; w < warp; ++w) have += sh.redc[w];
    const unsigned have0 = min(have, room), have1 = min(have + c[0], room), have2 = min(have + c[0] + c[1], room);
    const double v0 = sh.sum[e0] + (have1 > have0 ? (have1 - have0) * wc : 0.0), v1 = sh.sum[e0 + 1] + (have2 > have1 ? (have2 - have1) * wc : 0.0);
    double s = v0 + v1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    if (lane == 31) sh.red[warp] = s;
    if (threadIdx.x == 0) sh.bin = kGroups, sh.before = 0;
    __syncthreads();
    double start = 0, all = 0;
    for (int w = 0; w < kCountWarps; ++w) {
      if (w == warp) start = all;
      all += sh.red[w];
    }
    start += s - v0 - v1;
    const double target = (double)want.u * all;
    const int at = v0 > 0 && start + v0 > target ? 0 : v1 > 0 && start + v0 + v1 > target ? 1 : 2;
    if (at < 2) atomicMin(&sh.bin, (unsigned)(e0 + at));
    if (v0 > 0 || v1 > 0) atomicMax(&sh.before, (unsigned)(v1 > 0 ? e0 + 1 : e0));  // the last with some weight
    __syncthreads();
    const unsigned e = sh.bin < kGroups ? sh.bin : sh.before;
    __syncthreads();
    if (e / 2 == threadIdx.x) {
      sh.mass = e & 1 ? start + v0 : start;
      sh.before = e & 1 ? have1 : have0;
    }
    __syncthreads();
    if (warp != 0) return;
    // the entry, a lane's tokens one after the other
    uint32_t k[kLanePieces * kEach];
#pragma unroll
    for (int z = 0; z < kLanePieces; ++z) {
      const int p = ((int)e * 32 + lane) * kLanePieces + z;
      uint32_t t[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) t[i] = kDead;
      if (p < n) keys(p, t);
#pragma unroll
      for (int i = 0; i < kEach; ++i) k[z * kEach + i] = t[i];
    }
    unsigned equal = 0;
#pragma unroll
    for (int i = 0; i < kLanePieces * kEach; ++i) equal += cut_counts && k[i] == cut;
    unsigned eq = equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned t = __shfl_up_sync(0xffffffffu, eq, o);
      if (lane >= o) eq += t;
    }
    unsigned used = sh.before + eq - equal;
    double w[kLanePieces * kEach], mine = 0;
#pragma unroll
    for (int i = 0; i < kLanePieces * kEach; ++i) {
      w[i] = before_cut(k[i]);
      if (cut_counts && k[i] == cut && used++ < room) w[i] = wc;
      mine += w[i];
    }
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    const double base = sh.mass;
    const unsigned some = __ballot_sync(0xffffffffu, mine > 0), over = __ballot_sync(0xffffffffu, mine > 0 && base + incl > target);
    const int l = over ? __ffs(over) - 1 : 31 - __clz(some);
    if (lane == l) {
      double run = base + (incl - mine), share = 0;
      int hit = -1;
#pragma unroll
      for (int i = 0; i < kLanePieces * kEach; ++i) {
        if (w[i] > 0 && (hit < 0 || !(run > target))) hit = i, share = w[i];
        run += w[i];
      }
      a.tokens[r] = ((int)e * 32 + lane) * kLanePieces * kEach + hit - skip;
      if (a.probs) a.probs[r] = (float)(share / all);
    }
  }
};

template <class T>
__global__ void __launch_bounds__(kCountThreads, 1) sample_count_k(const __grid_constant__ Sample a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  CountShared &sh = *reinterpret_cast<CountShared *>(smem_raw);
  Counter<T> c(sh);
  const long long r = blockIdx.x;
  fill_powers(sh.powers);
  pdl_wait_and_release();
  c.x = static_cast<const T *>(a.x) + r * a.stride;
  c.vocab = a.vocab;
  c.skip = (int)(reinterpret_cast<uintptr_t>(c.x) % 16 / sizeof(T));
  const Want want(a, r);
  const bool filtered = want.t > 0.f && (want.k || want.p < 1.f);
  unsigned live = 0;
  uint32_t first;
  bool fits = true;
  if (filtered) {
    fits = c.count_all(live, first);
  } else {
    first = c.first_key();
    live = first != kDead;
  }
  if (live == 0) {
    if (threadIdx.x == 0) {
      a.tokens[r] = -1;
      if (a.probs) a.probs[r] = 0.f;
    }
    return;
  }
  c.top = Key<T>::value(first);
  c.weight.set(c.top, want.t > 0.f ? want.t : 1.f);
  if (!(want.t > 0.f)) {  // the first of the largest
    c.cut = first;
    c.room = 1;
  } else if (fits && filtered) {
    fits = c.select(want, live, first);
  }
  if (fits) {
    c.choose(want, a, r, first);
    return;
  }
  // the other kernel's way, from global memory
  __syncthreads();
  Row<T, kCountThreads> row(sh.other);
  row.ranks = 1, row.rank = 0;
  row.x = c.x, row.n = a.vocab, row.first = 0;
  row.vec = c.skip == 0;
  fill_powers(sh.other.powers);
  __syncthreads();
  double high = -INFINITY, low = -INFINITY;
  row.each([&](float v, int) {
    if (v > -INFINITY) high = fmax(high, (double)v), low = fmax(low, -(double)v);
  });
  const float mine = (float)high;
  row.template reduce<true>(high, low);
  row.run(a, r, high, low, mine);
}

template <class T>
cudaError_t launch_count(const Sample &a, cudaStream_t st) {
  static std::atomic<bool> attr_set[kAttrMaxDevices];
  const cudaError_t e = ensure_dynamic_smem(sample_count_k<T>, (int)sizeof(CountShared), attr_set);
  if (e != cudaSuccess) return e;
  Sample s = a;
  s.ranks = 1;
  s.slice = a.vocab;
  return launch_kernel(sample_count_k<T>, dim3((unsigned)a.rows), dim3(kCountThreads), sizeof(CountShared), st, s);
}

template <class T>
cudaError_t launch(const Sample &a, int sms, cudaStream_t st) {
  constexpr int kResident = 184 << 10;  // bytes of a slice that is kept
  // A CTA a row is enough where there are many.  (Measured at one width; top p alone is faster
  // by counting from fewer rows on, which this does not look at.)  Us in a cluster / by
  // counting, rows of 131072, with top p / with top k, top p and min p: 16-bit logits, 1 row 25/43 and 25/43,
  // 32 rows 66/72 and 61/54, 48 rows 113/73 and 84/55; 32 bits, 16 rows 59/190 and 53/131,
  // 100 rows 175/156 and 100/190, 148 rows 234/158 and 132/154.
  if (a.rows >= (sizeof(T) == 2 ? 40 : 148)) return launch_count<T>(a, st);
  Sample s = a;
  const long long bytes = (long long)a.vocab * sizeof(T);
  s.ranks = 1;
  while (s.ranks < kMaxRanks && (bytes / s.ranks > (96 << 10) || (a.rows * s.ranks < sms && bytes / s.ranks > (8 << 10)))) s.ranks *= 2;
  s.slice = ((a.vocab + s.ranks - 1) / s.ranks + 7) / 8 * 8;
  const long long need = (long long)s.slice * sizeof(T);
  s.resident = need <= kResident;
  static std::atomic<bool> attr_set[kAttrMaxDevices];
  const cudaError_t e = ensure_dynamic_smem(sample_k<T>, kResident, attr_set);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * s.ranks));
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = s.resident ? (size_t)need : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)s.ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_launch_pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, sample_k<T>, s);
}

}  // namespace

cudaError_t launch_sample(Sample a, int sms, cudaStream_t st) {
  if (a.dtype == 0) return launch<__half>(a, sms, st);
  if (a.dtype == 1) return launch<__nv_bfloat16>(a, sms, st);
  return launch<float>(a, sms, st);
}

}  // namespace ivb
