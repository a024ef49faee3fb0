// Rows in four bits, shared by the kernels that make them (gn_four.cu) and multiply them (gn_linear4.cu): e2m1 codes, two a byte, the first
// one low, and block scales in tiles.
//
//   block 16: scale s in e4m3, d = s * g with the tensor's own scale g in fp32:  s = e4m3(max |y| / (6 g)), in 2^-9 .. 448
//   block 32: scale d = 2^(floor(log2 max |y|) - 2) in e8m0, no g
//   code = e2m1(y / d), nearest, ties to the even code, at most 6 in magnitude; a block with a NaN or an infinity has a NaN for its scale
//
// A row has whole blocks of 32 codes; those behind its channels are zeros.  Scales: tiles of 128 rows and 4 blocks, 512 bytes each, in which row r,
// block b is byte (r % 32) * 16 + r % 128 / 32 * 4 + b % 4 - the order in which a matrix product takes them into tensor memory, 16 bytes a lane.  The
// tiles of 128 rows lie one behind the other along the blocks; scales of rows and blocks that are not there are zeros.
#pragma once
#include <cuda_fp4.h>

#include "gn_tokens.cuh"

namespace gnb200 {

constexpr int kFourUnit = 32;  // channels that a row is filled up to
constexpr int kScaleTile = 512;

__host__ __device__ inline int64_t four_wide(int64_t C) { return (C + kFourUnit - 1) / kFourUnit * kFourUnit; }
// tiles along a row
__host__ __device__ inline int64_t four_tiles(int64_t C, int block) { return (four_wide(C) / block + 3) / 4; }
__host__ __device__ inline int64_t four_scale_bytes(int64_t rows, int64_t C, int block) { return (rows + 127) / 128 * four_tiles(C, block) * kScaleTile; }

// where the four scales of row r in tile t begin
__device__ __forceinline__ long long four_scale_at(long long r, long long t, int tiles) {
  return ((r >> 7) * tiles + t) * kScaleTile + (r & 31) * 16 + (r >> 5 & 3) * 4;
}

}  // namespace gnb200
