// Rows to four bits and back, and the root-mean-square norm with the residual's addition straight into four bits (formulas and layout:
// gn_four.cuh; the norm is that of gn_rms.cu: s = x + r in fp32, y = s * rsqrt(mean(s^2) + eps) * (offset + w), y not rounded before its codes).
//
// A lane holds 16 channels: a block of 16, or half of one of 32, whose largest magnitude a shuffle completes; 8 bytes of codes a lane; the scales
// of four blocks become one word.  To four bits bound by HBM and instructions (12 to 14 for 32 elements): 16384 x 8192 bf16 55 us in blocks of 32, 63 of 16 (the scales' words, which go to
// tiles of their own, take most of the difference), floor 52; back by the writes: 71 us, where filling the output alone takes 69.  The norm runs on the kernels of gn_rms.cu, which
// hand a row's 16-byte vectors out; here are the rows that these do not take.
#include <algorithm>

#include "../../include/gnb200.h"
#include "gn_four.cuh"
#include "gn_kernels.h"

namespace gnb200 {
namespace {

constexpr int VE = 16;  // channels of a lane
template <int BLOCK>
constexpr int kLanes = BLOCK / VE;  // lanes of a block

struct FourRows {
  uint8_t *codes, *scales;
  const float* tensor_scale;  // g, or NULL for one
  long long rows;
  int C, wide, tiles;
};

// Codes of the 16 channels y of vector v of a row (zeros where it has none) and the scales that its lanes share; by whole warps.
template <int BLOCK>
__device__ __forceinline__ void put(const FourRows& p, long long row, int v, bool live, const float (&y)[VE], const TensorScale& t) {
  constexpr int LANES = kLanes<BLOCK>;
  float most = 0.f;
#pragma unroll
  for (int e = 0; e < VE; e += 2) most = largest(most, y[e], y[e + 1]);
  if constexpr (LANES > 1) most = larger(most, __shfl_xor_sync(0xffffffffu, most, 1));
  const FourStep step = four_step<BLOCK>(most, t);
  const uint2 words = make_uint2(codes8<BLOCK>(y, step), codes8<BLOCK>(y + 8, step));
  const bool inside = v * VE < p.wide;
  if (live && inside) *reinterpret_cast<uint2*>(p.codes + (row * (p.wide / VE) + v) * 8) = words;
  const int block = v / LANES;
  uint32_t scales = inside ? step.byte << (8 * (block & 3)) : 0;
  scales |= __shfl_xor_sync(0xffffffffu, scales, LANES);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 2 * LANES);
  if (live && v % (4 * LANES) == 0) put_scales(p.scales, row, p.rows, block >> 2, p.tiles, scales);
}
// ---------------------------------------------------------------------------------------------
// 16 channels of a row
// ---------------------------------------------------------------------------------------------
// A tensor's bytes: vectors that reach beyond a row may be read as long as they stay in these.
struct Bounds {
  const char *begin, *end;
};
// Aligned (VEC, rows of whole 8 channels), or from any address: then the 16-byte vectors that the channels lie in are read whole and shifted into place,
// three of them for 16 bits where element by element it were 16 loads (9001 x 1111 bf16 to four bits 66 us so); element by element at the ends of a
// row and where a vector would reach out of the tensor.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* row, int v, int C, const Bounds& bounds, float (&f)[VE]) {
  constexpr int N = VE * (int)sizeof(T) / 16;  // vectors
  const T* at = row + v * VE;
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float part[16 / sizeof(T)];
      if (v * VE + k * (int)(16 / sizeof(T)) < C) {
        unpack16<T, 16 / sizeof(T)>(reinterpret_cast<const uint4*>(at)[k], part);
      } else {
#pragma unroll
        for (int e = 0; e < (int)(16 / sizeof(T)); ++e) part[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < (int)(16 / sizeof(T)); ++e) f[k * (16 / sizeof(T)) + e] = part[e];
    }
  } else {
    const uintptr_t a = reinterpret_cast<uintptr_t>(at);
    const char* const from = reinterpret_cast<const char*>(a & ~(uintptr_t)15);
    if (v * VE + VE <= C && from >= bounds.begin && from + 16 * (N + 1) <= bounds.end) {
      uint32_t w[4 * (N + 1)];
#pragma unroll
      for (int k = 0; k <= N; ++k) {
        const uint4 q = reinterpret_cast<const uint4*>(from)[k];
        w[4 * k] = q.x, w[4 * k + 1] = q.y, w[4 * k + 2] = q.z, w[4 * k + 3] = q.w;
      }
      const bool two = a & 8, one = a & 4, half = a & 2;
#pragma unroll
      for (int k = 0; k < 4 * N + 2; ++k) w[k] = two ? w[k + 2] : w[k];
#pragma unroll
      for (int k = 0; k < 4 * N + 1; ++k) w[k] = one ? w[k + 1] : w[k];
#pragma unroll
      for (int k = 0; k < 4 * N; ++k) {
        if constexpr (sizeof(T) == 4) {
          f[k] = __uint_as_float(w[k]);
        } else {
          const uint32_t pair = __funnelshift_r(w[k], w[k + 1], half ? 16 : 0);
          float part[2];
          unpack<T, 2>(*reinterpret_cast<const Pack<T, 2>*>(&pair), part);
          f[2 * k] = part[0], f[2 * k + 1] = part[1];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) f[e] = v * VE + e < C ? load_param<T>(at, e) : 0.f;
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store16(T* row, int v, int C, const float (&f)[VE]) {
  constexpr int W = 16 / sizeof(T);
  T* at = row + v * VE;
#pragma unroll
  for (int k = 0; k < VE / W; ++k) {
    float part[W];
#pragma unroll
    for (int e = 0; e < W; ++e) part[e] = f[k * W + e];
    if constexpr (VEC) {
      if (v * VE + k * W < C) store_vec<T, W>(at + k * W, pack<T, W>(part));
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (v * VE + k * W + e < C) at[k * W + e] = store_param<T>(part[e]);
    }
  }
}
__device__ __forceinline__ void zero(float (&f)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) f[e] = 0.f;
}

// 16 channels as they lie in an aligned row
template <typename T>
struct Raw {
  uint4 q[sizeof(T)];
  __device__ __forceinline__ void load(const T* row, int v, int C) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(T); ++k) {
      q[k] = make_uint4(0, 0, 0, 0);
      if (v * VE + k * (int)(16 / sizeof(T)) < C) q[k] = reinterpret_cast<const uint4*>(row + v * VE)[k];
    }
  }
  __device__ __forceinline__ void unpack(float (&f)[VE]) const {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < (int)sizeof(T); ++k) {
      float part[W];
      unpack16<T, W>(q[k], part);
#pragma unroll
      for (int e = 0; e < W; ++e) f[k * W + e] = part[e];
    }
  }
};

// ---------------------------------------------------------------------------------------------
// Rows to four bits and back
// ---------------------------------------------------------------------------------------------
constexpr int kThreads = 256;

// Work in units: 2^shift lanes a row, one vector a lane.  A row has `pieces` of these; the units of all rows are dealt out one by one, so that CTAs have the
// same number of them but for one (whole rows to a warp: 8192 x 8192 on 740 CTAs, one row or two a warp, 36 us).
struct Units {
  int shift, pieces;
  int over, rest;  // what a step of the whole grid is: rows of CTAs, pieces
};
struct Unit {
  long long base;  // rows of CTAs
  int piece;
  __device__ __forceinline__ Unit(const Units& u) {
    base = blockIdx.x / u.pieces;
    piece = blockIdx.x % u.pieces;
  }
  __device__ __forceinline__ void step(const Units& u) {
    base += u.over;
    piece += u.rest;
    if (piece >= u.pieces) piece -= u.pieces, ++base;
  }
};

// Aligned rows: a lane asks for its next 16 channels before it works on these.
template <typename T, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const T* x, long long x_stride, const Bounds bounds, const FourRows p, const Units u) {
  grid_dep_launch_dependents();
  const int per_cta = kThreads >> u.shift, own_row = threadIdx.x >> u.shift, lane = threadIdx.x & ((1 << u.shift) - 1), vectors = p.tiles * 4 * kLanes<BLOCK>;
  const TensorScale t(BLOCK == 16 ? p.tensor_scale : nullptr);
  Unit unit(u);
  Raw<T> next;
  const auto ask = [&]() {
    const long long row = unit.base * per_cta + own_row;
    const int v = (unit.piece << u.shift) + lane;
    if (VEC && row < p.rows && v * VE < p.C) next.load(x + row * x_stride, v, p.C);
  };
  ask();
  while (unit.base * per_cta < p.rows) {
    const long long row = unit.base * per_cta + own_row;
    const int v = (unit.piece << u.shift) + lane;
    const bool live = row < p.rows;
    float y[VE];
    zero(y);
    if (live && v * VE < p.C) {
      if constexpr (VEC)
        next.unpack(y);
      else
        load16<T, false>(x + row * x_stride, v, p.C, bounds, y);
    }
    unit.step(u);
    ask();
    put<BLOCK>(p, row, v, live && v < vectors, y, t);
  }
  clear_behind(p.scales, p.rows, p.tiles, blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads);
}

__device__ __forceinline__ void values_of(uint32_t word, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 two = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(word >> (4 * e)), __NV_E2M1)));
    f[e] = two.x, f[e + 1] = two.y;
  }
}
// VEC: output rows of whole 16-byte vectors on their boundaries; a vector a lane, so that a warp's stores lie side by side (16 codes a lane: 16384 x 8192 bf16
// 90 us).
template <typename T, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const FourRows p, T* out, const Units u) {
  constexpr int W = 16 / sizeof(T), AT_ONCE = VEC ? 4 : 1;
  const int per_cta = kThreads >> u.shift, own_row = threadIdx.x >> u.shift, lane = threadIdx.x & ((1 << u.shift) - 1);
  const float g = BLOCK == 16 && p.tensor_scale ? *p.tensor_scale : 1.f;
  const auto scale_at = [&](long long row, int channel) {
    const int block = channel / BLOCK;
    return scale_value(p.scales[four_scale_at(row, block >> 2, p.tiles) + (block & 3)], BLOCK);
  };
  Unit unit(u);
  while (unit.base * per_cta < p.rows) {
    if constexpr (VEC) {
      uint32_t word[AT_ONCE];
      float scale[AT_ONCE];
      T* to[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const long long row = unit.base * per_cta + own_row;
        const int at = ((unit.piece << u.shift) + lane) * W;
        to[k] = row < p.rows && at < p.C ? out + row * p.C + at : nullptr;
        if (to[k]) {
          const uint8_t* const from = p.codes + row * (p.wide / 2) + at / 2;
          word[k] = W == 8 ? *reinterpret_cast<const uint32_t*>(from) : *reinterpret_cast<const uint16_t*>(from);
          scale[k] = scale_at(row, at);
        }
        unit.step(u);
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        if (to[k]) {
          float f[8], o[W];
          values_of(word[k], f);
#pragma unroll
          for (int e = 0; e < W; ++e) o[e] = f[e];
          scale_each(o, scale[k]);
          if constexpr (BLOCK == 16) scale_each(o, g);
          store_vec<T, W>(to[k], pack<T, W>(o));
        }
      }
    } else {
      // in the frame of the output's 16-byte vectors, whose first and last have elements of the rows beside this one; 8 codes from any one on
      const long long row = unit.base * per_cta + own_row;
      if (row < p.rows) {
        T* const to = out + row * p.C;
        const int skew = (int)(reinterpret_cast<uintptr_t>(to) / sizeof(T) % W), words = p.wide / 8;
        const int c = ((unit.piece << u.shift) + lane) * W - skew, at = c < 0 ? -1 : c / 8;
        if (c < p.C) {
          const uint32_t* const w = reinterpret_cast<const uint32_t*>(p.codes + row * (p.wide / 2));
          const uint32_t below = at >= 0 ? w[at] : 0, above = at + 1 < words ? w[at + 1] : 0;
          float f[8];
          values_of(__funnelshift_r(below, above, 4 * (c & 7)), f);
          const int border = ((c + W - 1) / BLOCK) * BLOCK;  // channels from here on have the last one's scale
          const float last = scale_at(row, min(c + W - 1, p.C - 1)), first = c >= 0 && c < border ? scale_at(row, c) : last;
          float o[W];
#pragma unroll
          for (int e = 0; e < W; ++e) o[e] = f[e] * (c + e < border ? first : last) * g;
          if (c >= 0 && c + W <= p.C) {
            store_vec<T, W>(to + c, pack<T, W>(o));
          } else {
#pragma unroll
            for (int e = 0; e < W; ++e)
              if ((unsigned)(c + e) < (unsigned)p.C) to[c + e] = store_param<T>(o[e]);
          }
        }
      }
      unit.step(u);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Norm
// ---------------------------------------------------------------------------------------------
struct NormArgs {
  const void *x, *residual, *weight;
  void* sum;
  long long x_stride, r_stride;
  Bounds x_bounds, r_bounds;
  int w_dtype;
  float eps, offset, inv_c;
};

// Rows that the kernels of gn_rms.cu do not take: tensors without a common frame, rows of more channels than a CTA holds.  A CTA to a row, which it
// reads twice.
constexpr int kNormThreads = 512;
template <typename Tx, typename Ts, int BLOCK, bool VEC>
__global__ void __launch_bounds__(kNormThreads) norm_any_kernel(const NormArgs a, const FourRows p) {
  __shared__ TeamSlots slots;
  grid_dep_launch_dependents();
  const int at = threadIdx.x, vectors = p.tiles * 4 * kLanes<BLOCK>;
  const TensorScale t(BLOCK == 16 ? p.tensor_scale : nullptr);
  clear<false>(slots, kNormThreads, 0, at);
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const Tx* x = static_cast<const Tx*>(a.x) + row * a.x_stride;
    const Ts* r = a.residual ? static_cast<const Ts*>(a.residual) + row * a.r_stride : nullptr;
    auto sum_of = [&](int v, float (&s)[VE]) {
      zero(s);
      if (v * VE < p.C) {
        load16<Tx, VEC>(x, v, p.C, a.x_bounds, s);
        if (r) {
          float f[VE];
          load16<Ts, VEC>(r, v, p.C, a.r_bounds, f);
          add_each(s, f);
        }
      }
    };
    float s[VE], sq[2] = {0.f, 0.f};
    for (int v = at; v * VE < p.C; v += kNormThreads) {
      sum_of(v, s);
      dot_each(sq, s, s);
    }
    const float rstd = __frsqrt_rn(fmaf(team_sum<false>(sq[0] + sq[1], slots, turn, kNormThreads, 0), a.inv_c, a.eps));
    for (int first = 0; first < vectors; first += kNormThreads) {
      const int v = first + at;
      sum_of(v, s);  // (the last look at these: the sum may be the residual's own buffer)
      if (v * VE < p.C) {
        if (r) store16<Ts, VEC>(static_cast<Ts*>(a.sum) + row * p.C, v, p.C, s);
        scale_each(s, rstd);
#pragma unroll
        for (int e = 0; e < VE; ++e)  // (behind the row a NaN rstd would leave NaN in the zeros)
          s[e] = v * VE + e >= p.C ? 0.f : a.weight ? s[e] * (a.offset + param_at(a.weight, a.w_dtype, v * VE + e, 1.f)) : s[e];
      }
      put<BLOCK>(p, row, v, v < vectors, s, t);
    }
  }
  clear_behind(p.scales, p.rows, p.tiles, blockIdx.x * kNormThreads + threadIdx.x, gridDim.x * kNormThreads);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
template <typename F>
cudaError_t with_type(int dtype, F&& f) {
  if (dtype == GNB200_F32) return f(float());
  if (dtype == GNB200_F16) return f(__half());
  return f(__nv_bfloat16());
}
template <typename F>
cudaError_t with_flag(bool flag, F&& f) {
  return flag ? f(std::true_type()) : f(std::false_type());
}
template <typename F>
cudaError_t with_block(int block, F&& f) {
  return block == 16 ? f(std::integral_constant<int, 16>()) : f(std::integral_constant<int, 32>());
}
bool dtype_ok(int d) { return d == GNB200_F32 || d == GNB200_F16 || d == GNB200_BF16; }
int size_of(int dtype) { return dtype == GNB200_F32 ? 4 : 2; }
bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
Bounds bounds_of(const void* p, int64_t rows, int64_t stride, int64_t C, int size) {
  const char* const begin = static_cast<const char*>(p);
  return p && stride >= 0 ? Bounds{begin, begin + ((rows - 1) * stride + C) * size} : Bounds{};
}

// `vectors` a row, at least `least` lanes (a power of two) to it; `waves` times the CTAs that are resident, which evens out what the SMs differ in (to four bits 16384 x 8192
// bf16 in blocks of 16 72 us with one, 65 with three, 66 with eight; back one is the best).  A row's vectors go to as many lanes, up to a warp's; more where the call is too small for all CTAs.
cudaError_t share_out(int64_t rows, int64_t vectors, int least, int waves, const void* kernel, Units* u, unsigned* grid) {
  Residency r = {};
  const cudaError_t err = residency(kernel, kThreads, 0, &r);
  if (err != cudaSuccess) return err;
  const int64_t resident = (int64_t)r.per_sm * r.sms;
  int shift = 0;
  while (1 << shift < least || (shift < 5 && 1 << shift < vectors)) ++shift;
  // (few rows leave lanes of a CTA without one)
  while (shift < 8 && rows < kThreads >> shift && 1 << shift < vectors) ++shift;
  const int64_t high = (rows + (kThreads >> shift) - 1) / (kThreads >> shift);
  u->shift = shift;
  u->pieces = (int)((vectors + (1 << shift) - 1) >> shift);
  *grid = (unsigned)std::min<int64_t>(high * u->pieces, waves * resident);
  u->over = (int)(*grid / u->pieces);
  u->rest = (int)(*grid % u->pieces);
  return cudaSuccess;
}

int launched(const char* name, cudaError_t err) {
  if (err == cudaSuccess) return GNB200_OK;
  return report_error(GNB200_ERR_CUDA, "%s: CUDA error: %s", name, cudaGetErrorString(err));
}

int check_four(const char* name, int64_t rows, int64_t C, int block, const float* tensor_scale) {
  if (block != 16 && block != 32) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: block is 16 or 32 channels (got %d)", name, block);
  if (block == 32 && tensor_scale) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: blocks of 32 have no scale of the whole tensor", name);
  if (rows < 0 || C < 1)
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: rows must not be negative and channels be positive (got %lld, %lld)", name, (long long)rows,
                        (long long)C);
  if (C > (1 << 30) || rows >= (int64_t)1 << 31)
    return report_error(GNB200_ERR_UNSUPPORTED, "%s: 2^31 rows or more than 2^30 channels are not supported (got %lld, %lld)", name, (long long)rows, (long long)C);
  return GNB200_OK;
}
FourRows four_rows(int64_t rows, int64_t C, int block, const float* tensor_scale, const void* codes, const void* scales) {
  FourRows p = {};
  p.codes = static_cast<uint8_t*>(const_cast<void*>(codes)), p.scales = static_cast<uint8_t*>(const_cast<void*>(scales)), p.tensor_scale = tensor_scale;
  p.rows = rows, p.C = (int)C, p.wide = (int)four_wide(C), p.tiles = (int)four_tiles(C, block);
  return p;
}

}  // namespace
}  // namespace gnb200

using namespace gnb200;

extern "C" {

size_t gnb200_4bit_code_bytes(int64_t rows, int64_t C) { return rows < 0 || C < 1 ? 0 : (size_t)rows * (size_t)(four_wide(C) / 2); }
size_t gnb200_4bit_scale_bytes(int64_t rows, int64_t C, int block) {
  return rows < 0 || C < 1 || (block != 16 && block != 32) ? 0 : (size_t)four_scale_bytes(rows, C, block);
}

int gnb200_quantize_4bit(const void* x, int64_t x_stride, int64_t rows, int64_t C, int dtype, int block, const float* tensor_scale, void* codes,
                         void* scales, void* stream) {
  const char* name = "gnb200_quantize_4bit";
  if (!dtype_ok(dtype)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if (int rc = check_four(name, rows, C, block, tensor_scale)) return rc;
  if (rows == 0) return GNB200_OK;
  if (!x || !codes || !scales) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!on16(codes) || !on16(scales)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: codes and scales begin on 16 bytes", name);
  const FourRows p = four_rows(rows, C, block, tensor_scale, codes, scales);
  const int width = 16 / size_of(dtype);
  const bool vec = on16(x) && C % width == 0 && (rows == 1 || x_stride % width == 0);
  return launched(name, with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_block(block, [&](auto b) {
      return with_flag(vec, [&](auto v) {
        constexpr int BLOCK = decltype(b)::value;
        auto kernel = &quantize_kernel<T, BLOCK, decltype(v)::value>;
        Units u;
        unsigned grid = 0;
        const cudaError_t err = share_out(rows, (int64_t)p.tiles * 4 * kLanes<BLOCK>, 4 * kLanes<BLOCK>, 3, (const void*)kernel, &u, &grid);
        if (err != cudaSuccess) return err;
        kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const T*>(x), x_stride, bounds_of(x, rows, x_stride, C, sizeof(T)), p, u);
        return cudaGetLastError();
      });
    });
  }));
}

int gnb200_dequantize_4bit(const void* codes, const void* scales, int64_t rows, int64_t C, int block, const float* tensor_scale, int dtype, void* out,
                           void* stream) {
  const char* name = "gnb200_dequantize_4bit";
  if (!dtype_ok(dtype)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if (int rc = check_four(name, rows, C, block, tensor_scale)) return rc;
  if (rows == 0) return GNB200_OK;
  if (!out || !codes || !scales) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!on16(codes) || !on16(scales)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: codes and scales begin on 16 bytes", name);
  const FourRows p = four_rows(rows, C, block, tensor_scale, codes, scales);
  const int width = 16 / size_of(dtype);
  const bool vec = on16(out) && C % width == 0;
  return launched(name, with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_block(block, [&](auto b) {
      return with_flag(vec, [&](auto v) {
        auto kernel = &dequantize_kernel<T, decltype(b)::value, decltype(v)::value>;
        Units u;
        unsigned grid = 0;
        const cudaError_t err = share_out(rows, vec ? C / width : (C + 2 * width - 2) / width, 4, 1, (const void*)kernel, &u, &grid);
        if (err != cudaSuccess) return err;
        kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p, static_cast<T*>(out), u);
        return cudaGetLastError();
      });
    });
  }));
}

int gnb200_rms_fwd_4bit(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, int64_t rows, int64_t C,
                        double eps, double offset, int dtype, int residual_dtype, int weight_dtype, int block, const float* tensor_scale, void* codes,
                        void* scales, void* sum, void* stream) {
  const char* name = "gnb200_rms_fwd_4bit";
  if (!residual) residual_dtype = dtype;
  if (!weight) weight_dtype = dtype;
  if (!dtype_ok(dtype) || !dtype_ok(residual_dtype) || !dtype_ok(weight_dtype))
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype code (0=f32, 1=f16, 2=bf16)", name);
  if ((residual_dtype != dtype && residual_dtype != GNB200_F32) || (weight_dtype != dtype && weight_dtype != GNB200_F32))
    return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: the residual and the weight have the type of x or float32", name);
  if (int rc = check_four(name, rows, C, block, tensor_scale)) return rc;
  if (rows == 0) return GNB200_OK;
  if (!x || !codes || !scales || (residual && !sum)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!on16(codes) || !on16(scales)) return report_error(GNB200_ERR_INVALID_ARGUMENT, "%s: codes and scales begin on 16 bytes", name);
  const FourRows p = four_rows(rows, C, block, tensor_scale, codes, scales);
  const FourNorm n = {x, residual, weight, sum, p.codes, p.scales, tensor_scale, rows, x_stride, residual_stride, (int)C, block, dtype, residual_dtype, weight_dtype, eps, offset};
  const cudaError_t how = launch_rms_4bit(n, static_cast<cudaStream_t>(stream));
  if (how != cudaErrorInvalidValue) return launched(name, how);
  NormArgs a = {};
  a.x = x, a.residual = residual, a.weight = weight, a.sum = sum, a.x_stride = x_stride, a.r_stride = residual_stride, a.w_dtype = weight_dtype;
  a.eps = (float)eps, a.offset = (float)offset, a.inv_c = (float)(1.0 / (double)C);
  a.x_bounds = bounds_of(x, rows, x_stride, C, size_of(dtype)), a.r_bounds = bounds_of(residual, rows, residual_stride, C, size_of(residual_dtype));
  const bool vec = C % 8 == 0 && on16(x) && on16(residual) && on16(sum) &&
                   (rows == 1 || (x_stride * size_of(dtype) % 16 == 0 && (!residual || residual_stride * size_of(residual_dtype) % 16 == 0)));
  return launched(name, with_type(dtype, [&](auto t) {
    using Tx = decltype(t);
    const auto typed = [&](auto u) {
      using Ts = decltype(u);
      return with_block(block, [&](auto b) {
        return with_flag(vec, [&](auto is_vec) {
          auto kernel = &norm_any_kernel<Tx, Ts, decltype(b)::value, decltype(is_vec)::value>;
          Residency r = {};
          const cudaError_t err = residency((const void*)kernel, kNormThreads, 0, &r);
          if (err != cudaSuccess) return err;
          kernel<<<(unsigned)std::min<int64_t>(rows, (int64_t)r.per_sm * r.sms), kNormThreads, 0, static_cast<cudaStream_t>(stream)>>>(a, p);
          return cudaGetLastError();
        });
      });
    };
    if constexpr (!std::is_same<Tx, float>::value)
      if (residual && residual_dtype == GNB200_F32) return typed(float());
    return typed(Tx());
  }));
}

}  // extern "C"
