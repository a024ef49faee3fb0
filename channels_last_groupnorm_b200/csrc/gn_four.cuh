// Rows in four bits, shared by the kernels that make them (gn_four.cu) and multiply them (gn_linear4.cu): e2m1 codes, two a byte, the first
// one low, and block scales in tiles.
//
//   block 16: scale s in e4m3, d = s * g with the tensor's own scale g in fp32, 2^-100 .. 2^117:  s = e4m3(max |y| / (6 g)), in 2^-9 .. 448
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

// ---------------------------------------------------------------------------------------------
// Codes and scales
// ---------------------------------------------------------------------------------------------
// Quotients are those of a division: with 16-bit inputs y / d lies midway between two codes often enough that a quotient one unit off shows.  The
// reciprocal is the correctly rounded one (a Newton step from the hardware's), a quotient is corrected by its remainder (Markstein's theorem).
__device__ __forceinline__ float reciprocal(float d) {
  float near;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(near) : "f"(d));
  return fmaf(fmaf(-d, near, 1.f), near, near);
}
__device__ __forceinline__ float scale_value(uint32_t byte, int block) {
  if (block == 16) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
  return byte == 0xff ? __uint_as_float(0x7fc00000u) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);  // (2^-127 is subnormal)
}
// the largest magnitude of three, or NaN where one is
__device__ __forceinline__ float largest(float a, float b, float c) {
  float m;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// The tensor's scale and what is made of it once
struct TensorScale {
  float g, six, inverse;  // 6 g and its reciprocal
  __device__ __forceinline__ TensorScale(const float* at) {
    g = at ? *at : 1.f;
    six = 6.f * g;
    inverse = reciprocal(six);
  }
};
struct FourStep {
  float value, inverse;
  uint32_t byte;
  bool cut;  // the scale is the largest there is, so that quotients may be infinite, or NaN
};
template <int BLOCK>
__device__ __forceinline__ FourStep four_step(float most, const TensorScale& t) {
  FourStep step;
  const bool finite = most < __uint_as_float(0x7f800000u);  // (no NaN either)
  if constexpr (BLOCK == 16) {
    const float q = most * t.inverse;
    const float s = q >= 448.f ? 448.f : fmaxf(fmaf(-t.inverse, fmaf(q, t.six, -most), q), 0.001953125f);
    step.byte = finite ? __nv_cvt_float_to_fp8(s, __NV_SATFINITE, __NV_E4M3) : 0x7fu;
    step.value = scale_value(step.byte, 16) * t.g;
    step.inverse = reciprocal(step.value);
    step.cut = !(q < 448.f);
  } else {
    const int e = max((int)(__float_as_uint(most) >> 23) - 2, 0);
    step.byte = finite ? (uint32_t)e : 0xffu;
    step.value = 0.f;  // (a product with the inverse, a power of two, is the quotient)
    step.inverse = __uint_as_float((uint32_t)(254 - min(e, 252)) << 23);
    step.cut = false;
  }
  return step;
}
// 8 codes
template <int BLOCK>
__device__ __forceinline__ uint32_t codes8(const float* y, const FourStep& step) {
  // (block 16: of the negative quotient, so that its correction takes the remainder y - q d with no sign to be turned for each, and a zero keeps its own)
  float value = step.value, inverse = BLOCK == 16 ? -step.inverse : step.inverse;
  float q[8], x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = y[e];
  if (BLOCK == 16 && step.cut) {  // one branch for all that is unusual: selects in its place cost 3 % of 30000 x 640
    const float most = 8.f * value;  // what is beyond has the largest code; an infinite quotient would have a NaN for its correction
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fminf(fmaxf(x[e], -most), most);
    if (isnan(value)) value = 0.f, inverse = -0.f;  // zeros behind a row's channels stay zeros
  }
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    mul2(q[e], q[e + 1], x[e], x[e + 1], inverse, inverse);
    if constexpr (BLOCK == 16) {
      float r0, r1;
      fma2(r0, r1, q[e], q[e + 1], value, value, x[e], x[e + 1]);
      fma2(q[e], q[e + 1], r0, r1, inverse, inverse, q[e], q[e + 1]);
    }
  }
  uint32_t word;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(word)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return BLOCK == 16 ? word ^ 0x88888888u : word;
}
// The scales of four blocks, one word, of row `row` and tile `tile`; zeros for the rows of its 16 bytes that are not there.
__device__ __forceinline__ void put_scales(uint8_t* scales, long long row, long long rows, int tile, int tiles, uint32_t word) {
  uint32_t* const at = reinterpret_cast<uint32_t*>(scales + four_scale_at(row, tile, tiles));
  at[0] = word;
  if (row + 32 >= rows)
    for (int k = 1; k < 4 - (int)(row >> 5 & 3); ++k) at[k] = 0;
}
// The scales of the lanes of the last tile that have no row at all, by all threads of the grid.
__device__ __forceinline__ void clear_behind(uint8_t* scales, long long all_rows, int tiles, unsigned thread, unsigned threads) {
  const unsigned rows = (unsigned)(all_rows & 127);
  if (rows == 0 || rows >= 32) return;
  uint8_t* const last = scales + (all_rows >> 7) * tiles * kScaleTile;
  const unsigned lanes = 32 - rows, all = lanes * (unsigned)tiles;
  for (unsigned i = thread; i < all; i += threads) *reinterpret_cast<uint4*>(last + (size_t)(i / lanes) * kScaleTile + (rows + i % lanes) * 16) = make_uint4(0, 0, 0, 0);
}

// gnb200_rms_fwd_4bit on the kernels of gn_rms.cu; cudaErrorInvalidValue: rows without a common frame or longer than these hold
struct FourNorm {
  const void *x, *residual, *weight;
  void* sum;
  uint8_t *codes, *scales;
  const float* tensor_scale;
  long long rows, x_stride, r_stride;
  int C, block, dtype, residual_dtype, weight_dtype;
  double eps, offset;
};
cudaError_t launch_rms_4bit(const FourNorm& n, cudaStream_t stream);

}  // namespace gnb200
