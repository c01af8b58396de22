// Attention over the paged 8-bit cache.
//
// For a query at position p and the visible keys j (codes kc, vc; scales ks, vs):
//   s_j = scale * ks_j * (q . kc_j),  o = sum_j e^(s_j - m) vs_j vc_j / sum_j e^(s_j - m)
// in one pass with a running maximum m (f32 throughout).
#include "kv_common.cuh"

namespace ivb {

namespace {

// One warp per (packed token, query head); lane l holds elements l * DIM / 32 ...
template <bool BF16, int DIM>
__global__ void __launch_bounds__(256) kv_attend_k(const __grid_constant__ KvAttend a) {
  pdl_wait_and_release();
  constexpr int kE = DIM / 32;
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long t = w / a.q_heads;
  const int qh = (int)(w - t * a.q_heads), head = qh / a.group;
  if (t >= a.seqs.tokens) return;
  int lo = 0, hi = a.seqs.batch;  // first sequence that ends behind t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.seqs.offsets[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= a.seqs.batch) return;
  const int o = a.seqs.offsets[lo], end = a.seqs.offsets[lo + 1], len = a.seqs.at[lo];
  if (o < 0 || t < o || end - o > a.max_new) {
    kv_flag(a.status, kStatusKvSeqs);
    return;
  }
  const int p = len - (end - (int)t);
  float q[kE], acc[kE], m = -INFINITY, l = 0.f;
  const uint16_t *qr = static_cast<const uint16_t *>(a.q.p) + t * a.q.ts + qh * a.q.hs + lane * kE;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    q[i] = unpack2<BF16>(qr[i]).x;
    acc[i] = 0.f;
  }
  int page = -1, page_at = -1;
  for (int j = 0; j <= p; ++j) {
    if (a.window && p - j >= a.window && j >= a.sinks) {
      j = p - a.window;
      continue;
    }
    if (j / a.cache.page != page_at) {
      page_at = j / a.cache.page;
      page = kv_page_of(a.cache, a.seqs, lo, j, a.status);
    }
    if (page < 0) break;
    const int slot = j % a.cache.page;
    const long long ca = kv_code_at(a.cache, page, head, slot) + lane * kE, sa = kv_scale_at(a.cache, page, head, slot);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kE; ++i) s += q[i] * (float)a.cache.k[ca + i];
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.scale * a.cache.ks[sa];
    const float m2 = fmaxf(m, s), f = __expf(m - m2), e = __expf(s - m2), ev = e * a.cache.vs[sa];
    m = m2;
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < kE; ++i) acc[i] = acc[i] * f + ev * (float)a.cache.v[ca + i];
  }
  uint16_t *yr = static_cast<uint16_t *>(a.out.p) + t * a.out.ts + qh * a.out.hs + lane * kE;
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < kE; ++i) yr[i] = (uint16_t)pack2<BF16>(acc[i] * inv, 0.f);
}

}  // namespace

cudaError_t launch_kv_attend(bool bf16, const KvAttend &a, cudaStream_t st) {
  const long long warps = a.seqs.tokens * a.q_heads;
  const dim3 grid((unsigned)((warps + 7) / 8));
  auto kern = a.cache.dim == 64 ? (bf16 ? kv_attend_k<true, 64> : kv_attend_k<false, 64>)
                                : (bf16 ? kv_attend_k<true, 128> : kv_attend_k<false, 128>);
  return launch_kernel(kern, grid, dim3(256), 0, st, a);
}

}  // namespace ivb
