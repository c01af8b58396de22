// Host-side TMA tensor-map encoding through the driver entry point (no link
// dependency on libcuda).
#pragma once

#include <cstdint>
#include <cuda.h>
#include <string>

namespace ivb {

// Encodes a tiled fp16 tensor map.  dims/box/elem_strides have `rank` entries,
// byte_strides has rank-1 entries (dimension 1..rank-1).  Returns false and fills
// `err` if the driver rejects the description.
bool encode_tiled_f16(CUtensorMap *map, int rank, const void *base, const uint64_t *dims,
                      const uint64_t *byte_strides, const uint32_t *box, const uint32_t *elem_strides,
                      CUtensorMapSwizzle swizzle, std::string *err);

// A tiled map of bytes [rows][row_bytes] (rows `pitch` bytes apart, a multiple of
// 16), boxes of 128 bytes x box_rows rows in 128-byte swizzled lines.
bool encode_tiled_bytes(CUtensorMap *map, const void *base, uint64_t row_bytes, uint64_t rows, uint64_t pitch,
                        uint32_t box_rows, std::string *err);

CUtensorMapSwizzle swizzle_for_row_bytes(int row_bytes);

}  // namespace ivb
