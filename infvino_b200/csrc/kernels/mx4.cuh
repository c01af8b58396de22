// Host-visible declarations of the kernels for matrices of microscaled 4-bit numbers.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace ivb {

constexpr int kMx4Block = 32;  // values that share a scale

// codes [rows][width / 2], the lower four bits first; scale bytes
// [ceil(rows / 128)][ceil(width / 128)][32][4][4] (mx4_scale_at).
struct Mx4 {
  uint8_t *codes, *scales;
  long long rows, width;
};

// Where the scale byte of block b of row r is; `chunks` = ceil(width / 128).
__host__ __device__ inline long long mx4_scale_at(long long r, long long b, long long chunks) {
  return ((r >> 7) * chunks + (b >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

cudaError_t launch_mx4_quantize(bool bf16, const void *x, long long rows, long long stride, const Mx4 &m, int sms,
                                cudaStream_t st);
cudaError_t launch_mx4_read(bool bf16, const Mx4 &m, long long rows, void *out, long long stride, int sms, cudaStream_t st);
struct Mx4Linear {
  Mx4 x, w;         // x.rows: the rows that are used
  const void *rows;  // if not null: 16-bit rows that X is quantised from, x is room for it
  long long x_stride;
  bool x_bf16;
  void *out;
  long long stride;
  bool bf16;
  int *status;
  int sms, device;
};
cudaError_t launch_mx4_linear(const Mx4Linear &a, cudaStream_t st);

}  // namespace ivb
