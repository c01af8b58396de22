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
// A row belongs to a cluster of CTAs, each with a slice of it in shared memory.
// A cut is found by counting logits in bins of equal width and looking closer at
// the bin where it must be: up to kList of them are put in order, more of them are
// binned again, equal ones by their numbers.
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

struct Cut {  // kept: x > this one's, or x equal and number at most this one's
  float x;
  int i;
};

struct SampleShared {
  unsigned hist[kBins];
  unsigned long long key[kList];  // (order of x, number), rising
  double mass[kList];
  double part[2][kMaxRanks][2];   // what CTAs tell one another, two exchanges in turn
  double red[2][kWarps];
  unsigned cnt[kWarps];
  unsigned listed;
  int found;
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

template <class T>
struct Row {
  SampleShared &sh;
  const T *x;      // this CTA's slice
  int n, first;    // its length, the number of its first token
  int ranks, rank;
  float top;       // the largest logit
  double inv_t;
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

  __device__ __forceinline__ double weight(float v) const {
    if (v == top) return 1.0;
    const double z = ((double)v - (double)top) * inv_t;
    return z > -kFar ? exp(z) : 0.0;
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

  // f(logit, number) for each of the slice.
  template <class F>
  __device__ __forceinline__ void each(F &&f) {
    for (int j = threadIdx.x; j < n; j += kThreads) f(logit(x[j]), first + j);
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
        __syncthreads();
      }
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
      const double scale = kBins * 0.99999 / ((double)hi - (double)lo);
      const float fhi = hi, fscale = (float)scale;
      const bool wide = !(fscale < 1e30f && fscale > 1e-30f && hi - lo < 1e30f);
      auto bin = [&](float v, int i) {
        if (v > hi || v < lo || !keeps(v, i)) return -1;
        const float b = wide ? (float)(((double)hi - (double)v) * scale) : (fhi - v) * fscale;
        return min(kBins - 1, (int)b);
      };
      count(bin);
      int b;
      if (COUNT) {
        find(target - base, [&](int k) { return (double)sh.hist[k]; });
        b = sh.found;
        if (base + sh.before + sh.in_bin < target) return;  // there are not so many
        base += sh.before;
      } else {
        // a guess by the weights of the bins' middles, then sums
        find(target - base, [&](int k) { return sh.hist[k] ? sh.hist[k] * exp(fmax(((double)hi - (k + 0.5) / scale - top) * inv_t, -kFar)) : 0.0; });
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
};

template <class T>
__global__ void __launch_bounds__(kThreads) sample_k(const __grid_constant__ Sample a) {
  extern __shared__ __align__(16) uint8_t slice_raw[];
  __shared__ SampleShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Row<T> row(sh);
  row.ranks = a.ranks;
  row.rank = a.ranks > 1 ? (int)(blockIdx.x % a.ranks) : 0;
  const long long r = blockIdx.x / a.ranks;
  row.first = min(row.rank * a.slice, a.vocab);
  row.n = min(a.slice, a.vocab - row.first);
  pdl_wait_and_release();
  const T *x = static_cast<const T *>(a.x) + r * a.stride + row.first;
  row.x = x;
  double high = -INFINITY, low = -INFINITY;  // the largest logit, and the smallest above -inf negated
  for (int j = threadIdx.x; j < row.n; j += kThreads) {
    const T v = x[j];
    if (a.resident) reinterpret_cast<T *>(slice_raw)[j] = v;
    const float f = logit(v);
    high = fmax(high, (double)f);
    if (f > -INFINITY) low = fmax(low, -(double)f);
  }
  if (a.resident) row.x = reinterpret_cast<const T *>(slice_raw);
  row.template reduce<true>(high, low);  // (and the slice is in place)
  row.top = (float)high;
  const bool writes = row.rank == 0 && threadIdx.x == 0;
  if (high == -INFINITY) {
    if (writes) {
      a.tokens[r] = -1;
      if (a.probs) a.probs[r] = 0.f;
    }
    return;
  }
  const float t = a.temperature ? a.temperature[r] : 1.f;
  if (!(t > 0.f)) {
    double best = -INFINITY, none = 0;
    row.each([&](float v, int i) {
      if (v == row.top) best = fmax(best, -(double)i);
    });
    row.template reduce<true>(best, none);
    if (writes) {
      a.tokens[r] = (int)-best;
      if (a.probs) a.probs[r] = 1.f;
    }
    return;
  }
  row.inv_t = 1.0 / (double)t;
  row.cut = Cut{-INFINITY, -1};  // (-inf weighs nothing)
  // logits below this have no weight
  const float least = high == INFINITY ? row.top : (float)fmax(-low, high - kFar * (double)t);
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f, min_p = a.min_p ? a.min_p[r] : 0.f;
  if (k > 0 && k < a.vocab) row.template select<true>((double)k, least, a.vocab);
  if (p < 1.f) {
    double z = 0, none = 0;
    row.each([&](float v, int i) { z += row.keeps(v, i) ? row.weight(v) : 0.0; });
    row.template reduce<false>(z, none);
    row.template select<false>(fmax((double)p, 0.0) * z, least, a.vocab);
  }
  // ---- running sums, by number: a warp has a piece of the slice
  auto kept = [&](float v, int i) {
    if (!row.keeps(v, i)) return 0.0;
    const double w = row.weight(v);
    return w >= (double)min_p || v == row.top || !(min_p > 0.f) ? w : 0.0;
  };
  const int piece = (a.slice + kThreads - 1) / kThreads * 32;
  const int j0 = min(warp * piece, row.n), j1 = min(j0 + piece, row.n);
  double mine = 0;
  for (int j = j0 + lane; j < j1; j += 32) mine += kept(logit(row.x[j]), row.first + j);
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) sh.seg[warp] = mine;
  __syncthreads();
  double mass = threadIdx.x < kWarps ? sh.seg[threadIdx.x] : 0.0, none = 0;
  row.template reduce<false>(mass, none);
  float u = a.u[r];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  const double target = (double)u * mass;
  // the CTA, then the warp, where the sum passes the target
  double before = 0;
  int rank = 0;
  for (; rank + 1 < a.ranks; ++rank) {
    const double s = sh.part[row.turn][rank][0];
    if (before + s > target) break;
    before += s;
  }
  // (a last CTA without weight, by a rounding: the last one with some)
  while (rank > 0 && sh.part[row.turn][rank][0] == 0) --rank;
  if (rank != row.rank) return;
  int w = 0;
  for (; w + 1 < kWarps; ++w) {
    if (before + sh.seg[w] > target) break;
    before += sh.seg[w];
  }
  while (w > 0 && sh.seg[w] == 0) --w;
  if (w != warp) return;
  int token = -1;
  double share = 0;
  for (int j = j0; j < j1; j += 32) {
    const double v = j + lane < j1 ? kept(logit(row.x[j + lane]), row.first + j + lane) : 0.0;
    double s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double q = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += q;
    }
    const unsigned some = __ballot_sync(0xffffffffu, v > 0), over = __ballot_sync(0xffffffffu, v > 0 && before + s > target);
    if (some) {
      const int l = over ? __ffs(over) - 1 : 31 - __clz(some);
      token = row.first + j + l;
      share = __shfl_sync(0xffffffffu, v, l);
    }
    if (over) break;
    before += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) {
    a.tokens[r] = token;
    if (a.probs) a.probs[r] = (float)(share / mass);
  }
}

template <class T>
cudaError_t launch(const Sample &a, int sms, cudaStream_t st) {
  constexpr int kResident = 200 << 10;  // bytes of a slice that is kept
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
