// Matrices of microscaled 4-bit numbers (OCP MXFP4): quantisation, reading back,
// and the product out = X W^T.
//
// Blocks of 32 values of a row share the scale 2^e, e = floor(log2 of the largest
// magnitude) - 2, so that the largest code is 4 or 6; codes are x 2^-e rounded to
// the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even mantissa.  Both steps
// are exact but for that rounding.
#include <algorithm>

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

constexpr int kQuantThreads = 256;

// A thread takes eight values, four lanes a block of 32, a warp 256 of a row.
// Memory bounds it: 2 + 17 / 32 bytes a value.
template <bool BF16>
__global__ void __launch_bounds__(kQuantThreads) mx4_quantize_k(const uint16_t *x, long long rows, long long stride,
                                                               int vec, Mx4 m, int pieces, long long units) {
  const int lane = threadIdx.x & 31;
  const long long chunks = (m.width + 127) / 128;
  pdl_wait_and_release();
  for (long long u = (long long)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); u < units;
       u += (long long)gridDim.x * (kQuantThreads / 32)) {
    const long long r = u / pieces;
    const long long c0 = (u - r * pieces) * 256 + lane * 8;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const bool there = r < rows && c0 < m.width;
    if (there) unpack8<BF16>(load8(x + r * stride + c0, vec), f);
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (f[i] != f[i]) f[i] = 0.f;
      if (fabsf(f[i]) < INFINITY) most = fmaxf(most, fabsf(f[i]));
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = max((int)(__float_as_uint(most) >> 23) - 2, 0);
    const float by = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= by;
    if (there) *reinterpret_cast<uint32_t *>(m.codes + r * (m.width / 2) + c0 / 2) = mx4_codes(f);
    // four blocks' bytes in one word
    uint32_t word = (uint32_t)e << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if ((lane & 15) == 0 && c0 < chunks * 128)
      *reinterpret_cast<uint32_t *>(m.scales + mx4_scale_at(r, c0 / 32, chunks)) = word;
  }
}

template <bool BF16>
__global__ void __launch_bounds__(kQuantThreads) mx4_read_k(Mx4 m, long long rows, uint16_t *out, long long stride,
                                                           int vec, int pieces, long long units) {
  const int lane = threadIdx.x & 31;
  const long long chunks = (m.width + 127) / 128;
  pdl_wait_and_release();
  for (long long u = (long long)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5); u < units;
       u += (long long)gridDim.x * (kQuantThreads / 32)) {
    const long long r = u / pieces;
    const long long c0 = (u - r * pieces) * 256 + lane * 8;
    if (c0 >= m.width) continue;
    const uint32_t w = *reinterpret_cast<const uint32_t *>(m.codes + r * (m.width / 2) + c0 / 2);
    const float s = mx4_scale(m.scales[mx4_scale_at(r, c0 / 32, chunks)]);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = mx4_pair(w >> (8 * i));
      f[2 * i] = p.x * s;
      f[2 * i + 1] = p.y * s;
    }
    store8(out + r * stride + c0, pack8<BF16>(f), vec);
  }
}

bool rows_vec(const void *p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

// A thread an output.
template <bool BF16>
__global__ void __launch_bounds__(128) mx4_linear_k(Mx4 x, Mx4 w, uint16_t *out, long long stride) {
  pdl_wait_and_release();
  const long long n = (long long)blockIdx.x * 128 + threadIdx.x, t = blockIdx.y;
  if (n >= w.rows) return;
  const long long chunks = (w.width + 127) / 128;
  float sum = 0.f;
  for (long long b = 0; b < w.width / 32; ++b) {
    const uint4 cx = *reinterpret_cast<const uint4 *>(x.codes + t * (w.width / 2) + b * 16);
    const uint4 cw = *reinterpret_cast<const uint4 *>(w.codes + n * (w.width / 2) + b * 16);
    const uint32_t ax[4] = {cx.x, cx.y, cx.z, cx.w}, aw[4] = {cw.x, cw.y, cw.z, cw.w};
    float part = 0.f;
    for (int i = 0; i < 16; ++i) {
      const float2 p = mx4_pair(ax[i >> 2] >> (8 * (i & 3))), q = mx4_pair(aw[i >> 2] >> (8 * (i & 3)));
      part += p.x * q.x + p.y * q.y;
    }
    sum += part * mx4_scale(x.scales[mx4_scale_at(t, b, chunks)]) * mx4_scale(w.scales[mx4_scale_at(n, b, chunks)]);
  }
  const uint32_t r = pack2<BF16>(sum, sum);
  out[t * stride + n] = (uint16_t)r;
}

template <bool BF16>
cudaError_t quantize(const void *x, long long rows, long long stride, const Mx4 &m, cudaStream_t st) {
  const int pieces = (int)((m.width + 255) / 256);
  const long long units = (rows + 127) / 128 * 128 * pieces;  // (scale bytes of rows that are not there are 0)
  const long long grid = std::min<long long>((units + kQuantThreads / 32 - 1) / (kQuantThreads / 32), 148 * 8);
  return launch_kernel(mx4_quantize_k<BF16>, dim3((unsigned)grid), dim3(kQuantThreads), 0, st, static_cast<const uint16_t *>(x), rows,
                       stride, (int)rows_vec(x, stride), m, pieces, units);
}
template <bool BF16>
cudaError_t read(const Mx4 &m, long long rows, void *out, long long stride, cudaStream_t st) {
  const int pieces = (int)((m.width + 255) / 256);
  const long long units = rows * pieces;
  const long long grid = std::min<long long>((units + kQuantThreads / 32 - 1) / (kQuantThreads / 32), 148 * 8);
  return launch_kernel(mx4_read_k<BF16>, dim3((unsigned)grid), dim3(kQuantThreads), 0, st, m, rows, static_cast<uint16_t *>(out), stride,
                       (int)rows_vec(out, stride), pieces, units);
}

}  // namespace

cudaError_t launch_mx4_quantize(bool bf16, const void *x, long long rows, long long stride, const Mx4 &m,
                                cudaStream_t st) {
  return bf16 ? quantize<true>(x, rows, stride, m, st) : quantize<false>(x, rows, stride, m, st);
}

cudaError_t launch_mx4_read(bool bf16, const Mx4 &m, long long rows, void *out, long long stride, cudaStream_t st) {
  return bf16 ? read<true>(m, rows, out, stride, st) : read<false>(m, rows, out, stride, st);
}

size_t mx4_workspace_bytes(int) { return 0; }

cudaError_t launch_mx4_linear(const Mx4Linear &a, cudaStream_t st) {
  const dim3 grid((unsigned)((a.w.rows + 127) / 128), (unsigned)a.x.rows);
  if (a.bf16) return launch_kernel(mx4_linear_k<true>, grid, dim3(128), 0, st, a.x, a.w, static_cast<uint16_t *>(a.out), a.stride);
  return launch_kernel(mx4_linear_k<false>, grid, dim3(128), 0, st, a.x, a.w, static_cast<uint16_t *>(a.out), a.stride);
}

}  // namespace ivb
