// The next token from a row of logits: temperature, top k, top p, min p, and a
// random number.
//
// Token i weighs w_i = e^((x_i - max) / T).  In the order of falling logits, equal
// ones by their numbers, each filter keeps a beginning, so that together they are
// a cut: the last (logit, number) that is kept.  The token is then the first, by
// number, where the running sum of kept weights passes u times their sum.  Which
// one that is goes by sums next to a border, so weights and sums are in 64 bits,
// added in an order that is fixed for a size and a number of rows.
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

#include "common.cuh"
#include "sample.cuh"

namespace ivb {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kList = 1024;
constexpr int kMaxRanks = 8;
constexpr double kFar = 41.588830833596715;  // 60 ln 2: what is further below the largest has no weight

// 2^(j / 64), j below 64, by the first threads of a block.
constexpr int kPowers = 64;
__device__ __forceinline__ void fill_powers(double *powers) {
  if (threadIdx.x < kPowers) powers[threadIdx.x] = exp2(threadIdx.x / (double)kPowers);
}
// e^((v - top) / T) with by = 64 log2(e) / T: 2^(n / 64) from the table, and the first
// terms of the series of 2^(r / 64), r at most a half (the rest is below 2^-44 of it).
__device__ __forceinline__ double weight_of(float v, float top, double by, const double *powers) {
  if (v == top) return 1.0;
  const double t = ((double)v - (double)top) * by;
  if (!(t > -60.0 * kPowers)) return 0.0;
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: what is added to it is rounded to a whole number
  const double s = t + kRound;
  const double r = t - (s - kRound);
  const int n = __double2loint(s);
  constexpr double c = 0.6931471805599453 / kPowers;
  double p = c * c * c * c / 24.0;
  p = fma(p, r, c * c * c / 6.0);
  p = fma(p, r, c * c / 2.0);
  p = fma(p, r, c);
  p = fma(p, r, 1.0);
  const double w = p * powers[n & (kPowers - 1)];
  return __hiloint2double(__double2hiint(w) + (n >> 6) * (1 << 20), __double2loint(w));
}

struct Cut {  // kept: x > this one's, or x equal and number at most this one's
  float x;
  int i;
};

struct SampleShared {
  double powers[kPowers];
  unsigned hist[kBins];
  unsigned long long key[kList];  // (order of x, number), rising
  double mass[kList], wt[kList];  // running sums, weights
  double part[2][kMaxRanks][2];   // what CTAs tell one another, two exchanges in turn
  double red[2][kWarps];
  unsigned cnt[kWarps];
  unsigned listed;
  int found, kept, reached;
  unsigned before, in_bin;
  Cut cut;
  double seg[kWarps];
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
    u = a.u[r];
    u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  }
  // Logits below this weigh less than min_p, by more than any rounding.
  __device__ __forceinline__ float floor(float top) const {
    if (!(min_p > 0.f) || !(t > 0.f)) return -INFINITY;
    const double x = (double)top + (fmin(log((double)min_p), 0.0) - 1e-6) * (double)t;
    return (float)(x - 2e-7 * fabs(x));
  }
  __device__ __forceinline__ bool enough(double w, bool top) const { return !(min_p > 0.f) || top || w >= (double)min_p; }
};

template <class T>
struct Row {
  SampleShared &sh;
  const T *x;      // this CTA's slice
  bool vec;        // on 16 bytes
  int n, first;    // its length, the number of its first token
  int ranks, rank;
  float top;       // the largest logit
  double by;       // 64 log2(e) / T
  Cut cut;
  int turn = 0;    // of `part`

  __device__ Row(SampleShared &s) : sh(s) {}

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

  __device__ __forceinline__ double weight(float v) const { return weight_of(v, top, by, sh.powers); }
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
    for (int b = threadIdx.x; b < kBins; b += kThreads) sh.hist[b] = 0;
    __syncthreads();
    each([&](float v, int i) {
      const int b = bin(v, i);
      if (b >= 0) atomicAdd(&sh.hist[b], 1u);
    });
    if (ranks == 1) {
      __syncthreads();
      return;
    }
    sync();
    unsigned sum[kBins / kThreads];
#pragma unroll
    for (int k = 0; k < kBins / kThreads; ++k) {
      sum[k] = 0;
      for (int r = 0; r < ranks; ++r) sum[k] += at(sh.hist, r)[threadIdx.x + k * kThreads];
    }
    sync();
#pragma unroll
    for (int k = 0; k < kBins / kThreads; ++k) sh.hist[threadIdx.x + k * kThreads] = sum[k];
    __syncthreads();
  }

  // The first bin where value(b) summed up to it reaches `target` (the last one, if none), into sh.found; counts before it into sh.before.
  template <class F>
  __device__ void find(double target, F &&value) {
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
    double before = 0;
    unsigned cb = 0;
    for (int w = 0; w < warp; ++w) before += sh.red[0][w], cb += sh.cnt[w];
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

  // Puts those of which in(logit, number) holds (at most kList) in order, in CTA 0: sh.key; how many there are is returned there.
  template <class F>
  __device__ unsigned gather(F &&in) {
    if (threadIdx.x == 0) sh.listed = 0;
    sync();
    unsigned *listed = at(&sh.listed, 0);
    unsigned long long *key = at(sh.key, 0);
    each([&](float v, int i) {
      if (!in(v, i)) return;
      const unsigned p = atomicAdd(listed, 1u);
      if (p < kList) key[p] = ((unsigned long long)falling(v) << 32) | (unsigned)i;
    });
    sync();
    const unsigned n = min(sh.listed, (unsigned)kList);
    if (rank == 0) sort(n);
    return n;
  }

  // Rising, padded with ~0 to a power of two.  Steps over at most 32 stay inside a warp's 64 keys.
  __device__ void sort(unsigned n) {
    unsigned size = 2;
    while (size < n) size <<= 1;
    for (unsigned e = n + threadIdx.x; e < size; e += kThreads) sh.key[e] = ~0ull;
    __syncthreads();
    for (unsigned k = 2; k <= size; k <<= 1)
      for (unsigned j = k >> 1; j; j >>= 1) {
        for (unsigned e = threadIdx.x; e < size / 2; e += kThreads) {
          const unsigned a = 2 * e - (e & (j - 1)), b = a + j;
          const unsigned long long s = sh.key[a], t = sh.key[b];
          if ((s > t) == ((a & k) == 0)) sh.key[a] = t, sh.key[b] = s;
        }
        if (j > 32 || (j == 1 && k >= 64))
          __syncthreads();
        else
          __syncwarp();
      }
    __syncthreads();
  }

  // Running sums of two doubles a thread over the block, and their total.
  __device__ __forceinline__ double scan(double &x0, double &x1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double s = x0 + x1;
    const double mine = s;
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
    const double a0 = x0;
    x0 = before + (s - mine) + a0;
    x1 = before + s;
    return all;
  }

  // Of the n logits in sh.key, in order: what is kept, and the token; CTA 0.  mass: of
  // all tokens (top_p of them is meant where there is no top_k).  False: top_p is not reached.
  __device__ bool finish(unsigned n, const Want &want, double mass, const Sample &a, long long r) {
    static_assert(kList == 2 * kThreads, "two a thread");
    const int e0 = 2 * threadIdx.x;
    double w[2], c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = e0 + i < (int)n ? weight(from_falling((uint32_t)(sh.key[e0 + i] >> 32))) : 0.0;
      sh.wt[e0 + i] = w[i];
      c[i] = w[i];
    }
    scan(c[0], c[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) sh.mass[e0 + i] = c[i];
    const int m = want.k ? min(want.k, (int)n) : (int)n;
    if (threadIdx.x == 0) sh.kept = m, sh.reached = 0;
    __syncthreads();
    if (want.p < 1.f) {
      const double target = (double)want.p * (want.k ? sh.mass[m - 1] : mass);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (e0 + i < (int)n && c[i] >= target) {
          atomicMin(&sh.kept, e0 + i + 1);
          sh.reached = 1;
          break;
        }
    }
#pragma unroll
    for (int i = 1; i >= 0; --i)
      if (e0 + i < (int)n && !want.enough(w[i], from_falling((uint32_t)(sh.key[e0 + i] >> 32)) == top)) atomicMin(&sh.kept, e0 + i);
    __syncthreads();
    if (want.p < 1.f && !want.k && !sh.reached) return false;
    const unsigned kept = (unsigned)sh.kept;
    // by number
    unsigned long long by_number[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) by_number[i] = (sh.key[e0 + i] << 32) | (unsigned)(e0 + i);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (e0 + i < (int)kept) sh.key[e0 + i] = by_number[i];
    if (threadIdx.x == 0) sh.found = (int)kept - 1;
    __syncthreads();
    sort(kept);
#pragma unroll
    for (int i = 0; i < 2; ++i) c[i] = e0 + i < (int)kept ? sh.wt[(uint32_t)sh.key[e0 + i]] : 0.0;
    const double all = scan(c[0], c[1]), target = (double)want.u * all;
#pragma unroll
    for (int i = 0; i < 2; ++i)
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
  __device__ void select(double target, float least, int vocab) {
    float hi = top, lo = least;
    double base = 0;
    for (;;) {
      if (!(lo < hi)) {
        // equal ones: as many as it takes
        const double w = COUNT ? 1.0 : weight(hi);
        const double r = ceil((target - base) / w);
        cut_equal(hi, (unsigned)fmin(fmax(r, 1.0), 2147483647.0), vocab);
        return;
      }
      const Bins bins(hi, lo);
      auto bin = [&](float v, int i) { return keeps(v, i) ? bins(v) : -1; };
      count(bin);
      int b;
      if (COUNT) {
        find(target - base, [&](int k) { return (double)sh.hist[k]; });
        b = sh.found;
        if (base + sh.before + sh.in_bin < target) return;  // there are not so many
        base += sh.before;
      } else {
        // a guess by the weights of the bins' middles, then sums
        find(target - base, [&](int k) { return sh.hist[k] ? sh.hist[k] * weight(bins.middle(k)) : 0.0; });
        b = sh.found;
        int from = 0, to = kBins - 1;
        for (int tries = 0;; ++tries) {
          double a = 0, in = 0;
          each([&](float v, int i) {
            const int k = bin(v, i);
            if (k < 0 || k > b) return;
            const double w = weight(v);
            if (k < b)
              a += w;
            else
              in += w;
          });
          reduce<false>(a, in);
          if (base + a >= target && b > from) {
            to = b - 1;
            b = tries < 2 ? to : (from + to) / 2;
          } else if (base + a + in < target && b < to) {
            from = b + 1;
            b = tries < 2 ? from : (from + to) / 2;
          } else {
            base += a;
            break;
          }
        }
      }
      const unsigned in_bin = sh.hist[b];
      __syncthreads();
      if (in_bin == 0) return;  // (sums in another order fell short by a rounding)
      if (in_bin <= kList) {
        const unsigned listed = gather([&](float v, int i) { return bin(v, i) == b; });
        if (rank == 0) {
          unsigned at;
          if (COUNT) {
            at = (unsigned)(target - base) - 1;
          } else {
            for (unsigned e = threadIdx.x; e < listed; e += kThreads) sh.mass[e] = weight(from_falling((uint32_t)(sh.key[e] >> 32)));
            __syncthreads();
            if (threadIdx.x == 0) {
              double s = base;
              unsigned e = 0;
              while (e + 1 < listed && (s += sh.mass[e]) < target) ++e;
              sh.found = (int)e;
            }
            __syncthreads();
            at = (unsigned)sh.found;
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
  __device__ void run(const Sample &a, long long r, double high, double low) {
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
    by = kPowers * 1.4426950408889634 / (double)want.t;
    cut = Cut{-INFINITY, -1};  // (-inf weighs nothing)
    // logits below this have no weight
    const float least = high == INFINITY ? top : (float)fmax(-low, high - kFar * (double)want.t);
    double mass = 0, none = 0;
    if (want.p < 1.f && !want.k) {
      each([&](float v, int) { mass += v > -INFINITY ? weight(v) : 0.0; });
      reduce<false>(mass, none);
    }
    if ((want.p < 1.f || want.k) && want.k <= kList && least < top) {
      // what is kept, if it is not much, goes through one list
      const Bins bins(top, least);
      count([&](float v, int) { return bins(v); });
      if (want.k)
        find((double)want.k, [&](int b) { return (double)sh.hist[b]; });
      else
        find((double)want.p * mass, [&](int b) { return sh.hist[b] ? sh.hist[b] * weight(bins.middle(b)) : 0.0; });
      int b = sh.found;
      unsigned many = sh.before + sh.in_bin;
      if (!want.k) {  // (the bins' middles are a guess: two more)
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
    if (want.k) select<true>((double)want.k, least, a.vocab);
    if (want.p < 1.f) {
      if (want.k) {
        mass = 0;
        each([&](float v, int i) { mass += keeps(v, i) ? weight(v) : 0.0; });
        reduce<false>(mass, none);
      }
      select<false>((double)want.p * mass, least, a.vocab);
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
    double mine = 0;
    for (int j = j0 + 4 * lane; j < j1; j += 128) {
      float v[4];
      load4(j, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) mine += kept(v[i], first + j + i);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) sh.seg[warp] = mine;
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

template <class T>
__global__ void __launch_bounds__(kThreads) sample_k(const __grid_constant__ Sample a) {
  extern __shared__ __align__(16) uint8_t slice_raw[];
  __shared__ SampleShared sh;
  Row<T> row(sh);
  row.ranks = a.ranks;
  row.rank = a.ranks > 1 ? (int)(blockIdx.x % a.ranks) : 0;
  const long long r = blockIdx.x / a.ranks;
  row.first = min(row.rank * a.slice, a.vocab);
  row.n = min(a.slice, a.vocab - row.first);
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
  row.template reduce<true>(h, l);  // (and the slice is in place)
  row.run(a, r, h, l);
}

template <class T>
cudaError_t launch(const Sample &a, int sms, cudaStream_t st) {
  constexpr int kResident = 184 << 10;  // bytes of a slice that is kept
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
  cfg.blockDim = dim3(kThreads);
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
