// The packed cache: keys and values of one layer in 4 or 8 bits.
//
// pages: uint8 [num_pages, nkv, page_bytes].  The block of one page and kv head holds, for P tokens of d channels:
//   the codes of the keys    P rows of d * bits / 8 bytes (4 bits: channel 2i is the low half of byte i, 2i + 1 the high one),
//   the codes of the values  P rows of the same,
//   the pairs of the keys    P x groups x (scale, offset) in bfloat16,
//   the pairs of the values  the same.
// A group is 64 channels where that divides d, else 32, else 16.  A code c stands for scale * c + offset.  Keys and values of a
// page and head lie in one block so that one run of copies brings both (2304 bytes: 16 tokens of 128 channels in 4 bits).
// The offset is the group's smallest value rounded down to bfloat16 and the scale the smallest bfloat16 that is not below
// (largest - offset) / (2^bits - 1): every value lies inside the codes' range, so none is clipped, and a value is off by at
// most half a scale.  A group that holds an infinity or a NaN has NaN for both (one with a value below bfloat16's range an infinity, and
// reads as NaN).
#pragma once
#include "common.cuh"

__host__ __device__ __forceinline__ int packed_group(int d) { return d % 64 == 0 ? 64 : d % 32 == 0 ? 32 : 16; }

struct PackedRows {
  int bits, d, page_size, group;
  __host__ __device__ PackedRows(int bits_, int d_, int page_size_) : bits(bits_), d(d_), page_size(page_size_), group(packed_group(d_)) {}
  __host__ __device__ int row() const { return d * bits / 8; }                     // bytes of a token's codes
  __host__ __device__ int groups() const { return d / group; }
  __host__ __device__ int page_bytes() const { return 2 * page_size * (row() + 4 * groups()); }
  // offsets inside a block: codes and pairs of token `place`; which = 0 keys, 1 values
  __host__ __device__ int codes(int which, int place) const { return (which * page_size + place) * row(); }
  __host__ __device__ int pairs(int which, int place) const { return 2 * page_size * row() + (which * page_size + place) * groups() * 4; }
};
// pages of a size whose blocks and rows of pairs start on 16 bytes
__host__ __device__ __forceinline__ bool packed_sizes_ok(int bits, int d, int page_size) {
  return (bits == 4 || bits == 8) && d >= 16 && d <= 256 && d % 16 == 0 && page_size >= 4 && page_size <= 256 && (page_size & (page_size - 1)) == 0;
}
